"""GPU tests of the step operators at the ends of their ranges: counts, scales and queries far
apart, long contexts, every sequence of many.

An output row (all heads of a token) is held to 2.5e-3 of its norm. With x its values and steps of 2^-7
2^floor(log2 |x|), rounding to BF16 alone gives sqrt(sum step^2 / 12 / sum x^2), 1.6e-3 where the x are spread over
their binades (at most 2^-7 / sqrt 12 = 2.3e-3, at 1, 2, 4, ...). Beside it a probability times its value scale is
rounded to 11 bits: 2^-11 at most, 1.7e-4 where many keys count. Scores are off by some 2^-16 of their size.
Rows have at least 128 values, so that the norm of the rounding errors stays within 30 % of its mean.
"""

import numpy as np
import pytest
import torch

from oracle import step as oracle
from oracle.packed_q6 import bf16_round
from q6moe import paged_tree_attention, plan_pages, write_tokens

from .test_gpu_step import FEW_AND_MANY, _attn, _cache, _case, _dev, _sees

pytestmark = pytest.mark.gpu

NORM = 2.5e-3


@pytest.mark.parametrize("batch,rows,paths", [(4, 100, "one workgroup"), (4, 6000, "two"), (2, 9000, "three"),
                                              (1025, 50, "two, many")])
@pytest.mark.parametrize("most", [2**30, 2**31 - 1])
def test_missing_of_huge_counts(device, batch, rows, paths, most):
    # every sequence asks for more than fits: what is missing is never read as none, whichever launches run
    pps, page = 3, 64
    counts = np.full(batch, most, np.int32)
    table = _dev(np.arange(batch * pps, dtype=np.int32).reshape(batch, pps), device)
    kw = {} if paths == "three" else dict(max_count=4000)
    plan = plan_pages(table, _dev(np.zeros(batch, np.int32), device), _dev(counts, device),
                      _dev(np.array([5], np.int32), device), _dev(np.array([0], np.int32), device), page_size=page,
                      rows=rows, **kw)
    fits, placed, lost = rows, 0, 0
    for b in range(batch):
        got = min(kw.get("max_count", rows), fits)
        fits -= got
        placed += min(got, pps * page)
        lost += min(most - got, (2**31 - 1 - rows) // batch)
    assert plan.missing.item() == lost + (rows - fits - placed) > 2**30


@pytest.mark.parametrize("r,most", [(4, 6), (20, 6), (4, 3)])
def test_attention_without_out_gives_zeros_where_nothing_is_computed(device, r, most):
    # rows behind the last sequence, and those from max_count on, whatever the memory held
    case = (*_case(38, [50, 3], [6, 5], 16, 2, r, 128, extra=9)[:10], most)
    rows = case[9].shape
    for _ in range(3):
        dirty = torch.full(rows, float("nan"), dtype=torch.bfloat16, device=device)
        torch.cuda.synchronize()
        del dirty
        got = _attn(device, case, None)
        want = _attn(device, case, None, fill=7.0)
        idle = np.ones(len(got), bool)
        for first, end in ((0, 6), (6, 11)):
            idle[first:min(end, first + most)] = False
        assert (got[idle] == 0).all() and (want[idle] == 7.0).all()
        np.testing.assert_array_equal(got[~idle], want[~idle])


def test_write_refuses_pools_that_overlap(device):
    both = torch.zeros(5, 4, 64, dtype=torch.int8, device=device)
    scales, apart = torch.ones(5, 4, 1, device=device), torch.ones(3, 4, 1, device=device)
    x, slots = torch.zeros(2, 64, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    other = torch.zeros(3, 4, 64, dtype=torch.int8, device=device)
    kw = dict(kv_heads=1, head_dim=64)
    for k, ks, v, vs in ((both[:3], scales[:3], both[2:], apart), (both[2:], scales[:3], both[:3], apart),
                         (both[:3], scales[:3], other, scales[2:]), (both[:3], scales[2:], other, scales[:3])):
        with pytest.raises(ValueError, match="same memory"):
            write_tokens(k, ks, v, vs, x, x, slots, **kw)
    write_tokens(both[:2], scales[:2], both[2:4], scales[2:4], x, x, slots, **kw)  # side by side


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _hold(got, want, rows=None):
    """Every row that is not NaN in ``want`` (of ``rows``) is within NORM of its norm."""
    live = ~np.isnan(want).any((1, 2))
    if rows is not None:
        live &= np.isin(np.arange(len(want)), rows)
    assert live.any() and want[live][0].size >= 128
    error = np.linalg.norm((got - want)[live].reshape(live.sum(), -1), axis=1)
    size = np.linalg.norm(want[live].reshape(live.sum(), -1), axis=1)
    ratio = error / np.maximum(size, 1e-300)
    over = np.nonzero(live)[0][~(ratio <= NORM)].tolist()
    assert not over, (over, ratio.max())


def _exact(case, sees):
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = case
    return oracle.attention(q, k, ks, v, vs, table, lengths, starts, sees, page, most)[0]


@pytest.mark.parametrize("lengths,counts,page,kvh,r,dim,kind,room", [
    ([65533, 40000], [3, 2], 64, 1, 2, 64, "chain", False),           # a long context in few rows
    ([65500], [30], 256, 1, 4, 64, "tree", False),                    # several tiles of it
    ([65500], [30], 256, 1, 4, 64, "tree", True),                     # tiles of 128 rows
    ([30000, 7, 12345, 0, 511], [16, 16, 3, 16, 1], 16, 2, 8, 128, "tree", False),
    ([9000, 20000, 64], [40, 0, 60], 64, 1, 8, 128, "chain", True),
    ([5000, 3001], [50, 20], 128, 1, 6, 256, "tree", True),
    ([5000, 3001], [50, 20], 128, 1, 6, 256, "chain", False),
    ([30000] + [50] * 70, [2] * 71, 64, 1, 4, 64, "chain", False),    # items found in a launch of their own
    ([15000] * 8, [13] * 8, 256, 2, 8, 64, "tree", True),
])
def test_attention_counts_every_key_once(device, lengths, counts, page, kvh, r, dim, kind, room):
    """All keys are equal, so every seen one has the same weight, and the value of token t is 1 in channel t / 16 % D
    alone: an output is the number of a channel's seen tokens over that of all. Codes and scales (powers of two) are
    exact, and so are sums over the values, whole numbers below 2^24. A weight is 2 to the power of a score of at most
    2^4 less itself, off by half a step of it, 2^-21: with the exponential's step, and 11 bits that round it to 1
    for the values, a quotient is off by less than 2^-16 before it is rounded to BF16. A run of 16 keys that is lost or
    counted twice changes a channel by 16 D / n, at least 1.5 %."""
    rng = np.random.default_rng(len(lengths) + page)
    k, ks, v, vs, table, _, starts, page, kvh, q, most = _case(5, lengths, counts, page, kvh, r, dim, qscale=0.5, room=room)
    k[:] = rng.integers(-127, 128, (1, 1, kvh, dim))
    ks[:], vs[:], v[:] = 2.0**-7, 2.0**-6, 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        t = np.arange(n + c)
        v[table[b, t // page], t % page, :, t // 16 % dim] = 64
    sees = None if kind == "chain" else _sees(rng, counts, 0)
    got = _attn(device, (k, ks, v, vs, table, lengths, starts, page, kvh, q, most), sees)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        whole = np.bincount(np.arange(n) // 16 % dim, minlength=dim)
        for j in range(c):
            new = n + np.array(sorted(range(j + 1) if sees is None else sees[starts[b] + j]))
            count = whole + np.bincount(new // 16 % dim, minlength=dim)
            want = count / count.sum()
            assert (np.abs(got[starts[b] + j] - want) <= want * (2.0**-8 + 2.0**-16)).all(), (b, j)


def test_attention_long_contexts_by_the_norm(device):
    # what an elementwise bound that grows with the number of keys cannot see
    rng = np.random.default_rng(18)
    k, ks = _cache(rng, 64, 64, 1, 64)
    v, vs = _cache(rng, 64, 64, 1, 64)
    table = rng.integers(0, 64, (2, 1024)).astype(np.int32)
    q = bf16_round(rng.standard_normal((5, 4, 64)).astype(np.float32) * 2)
    case = (k, ks, v, vs, table, [65533, 40000], np.array([0, 3, 5]), 64, 1, q, 3)
    _hold(_attn(device, case, None), _exact(case, None))


def _chain_exact(device, case):
    """The oracle's chain in 64 bits on the GPU, all sequences at once."""
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = case
    batch, cap, (rows, hq, dim) = table.shape[0], table.shape[1] * page, q.shape
    n, first = (_dev(np.asarray(t, np.int64), device) for t in (lengths, starts))
    t = torch.arange(cap, device=device)
    slot = _dev(table.astype(np.int64), device)[:, t // page] * page + t % page
    x = _dev(q, device, torch.float64)
    row = first[:-1, None] + torch.arange(most, device=device)
    live = row < first[1:, None]
    sees = t <= n[:, None, None] + torch.arange(most, device=device)[:, None]  # [batch, most, cap]
    out = torch.full((rows, hq, dim), float("nan"), dtype=torch.float64, device=device)
    for h in range(kvh):
        kk, vv = (_dev(c[:, :, h].reshape(-1, dim), device)[slot].double()
                  * _dev(s[:, :, h].reshape(-1), device)[slot].double()[..., None] for c, s in ((k, ks), (v, vs)))
        kk = kk.transpose(1, 2).contiguous()
        for g in range(h * hq // kvh, (h + 1) * hq // kvh):
            s = torch.matmul(x[:, g][row.clamp(max=rows - 1)], kk) / dim**0.5
            p = torch.softmax(s.masked_fill(~sees, -float("inf")), -1)
            out[row[live], g] = torch.matmul(p, vv)[live]
    return out.cpu().numpy()


@pytest.mark.parametrize("batch,kvh,r,dim,count,most_len,spare_count", [
    (300, 2, 2, 64, 1, 400, 0), (520, 4, 1, 128, 1, 30, 0), (70, 4, 9, 64, 12, 300, 5), (390, 8, 25, 64, 4, 20, 0),
    (64, 2, 3, 128, 3, 700, 0), (65, 2, 3, 128, 3, 700, 1), (1023, 2, 2, 64, 2, 60, 0), (1024, 2, 2, 64, 1, 60, 0),
    (1025, 2, 2, 64, 2, 60, 0), (2100, 2, 4, 256, 1, 15, 0), (80, 1, 4, 128, 2, 9000, 0), (3, 2, 4, 128, 700, 500, 0),
])
def test_attention_of_every_sequence_of_many(device, batch, kvh, r, dim, count, most_len, spare_count):
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, most_len + 1, batch)
    counts = rng.integers(0, count + 1, batch)
    counts[[0, -1]] = count
    k, ks, v, vs, table, _, starts, page, kvh, q, _ = _case(batch, lengths, counts, 16, kvh, r, dim, 2)
    case = (k, ks, v, vs, table, lengths, starts, page, kvh, q, count + spare_count)
    got = _attn(device, case, None, fill=9.0)
    assert (got[starts[-1]:] == 9.0).all()
    _hold(got, _chain_exact(device, case))


DIMS = pytest.mark.parametrize("dim", [64, 128, 256])


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [104, 108, 112, -112])
def test_attention_values_near_the_ends_of_fp32(device, dim, r, room, power):
    # value scales of 2^power and 2^-7 of that; sums over 100 keys stay below 2^128
    case = _case(36, [90, 3], [8, 5], 16, 1, r, dim, qscale=0.5, room=room)
    case[3][:] = (case[3] * np.float32(2.0**power) if power < 0 else np.float32(2.0**power) * (case[3] / case[3].max()))
    _hold(_attn(device, case, None), _exact(case, None))


def _near(rng, case, spread=0.05):
    """Queries of all rows and heads near one direction, which is returned."""
    q = case[9]
    base = rng.standard_normal(q.shape[2]).astype(np.float32) * 2
    q[:] = bf16_round((base + spread * rng.standard_normal(q.shape)).astype(np.float32))
    return base


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [16, 20, 28, 60, 100])
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_attention_large_values_of_a_token_that_others_do_not_see(device, dim, r, room, power, kind):
    # new token 3's values are 2^power times the others'; rows that may not see it are as exact as without it
    counts = [8, 8]
    case = _case(31, [500, 40], counts, 16, 1, r, dim, room=room)
    vs, table, lengths = case[3], case[4], case[5]
    for b, n in enumerate(lengths):
        vs[table[b, (n + 3) // 16], (n + 3) % 16] *= np.float32(2.0**power)
    sees = None if kind == "chain" else [s - {3} if i % 8 != 3 else s for i, s in
                                         enumerate(_sees(np.random.default_rng(5), counts, 0))]
    _hold(_attn(device, case, sees), _exact(case, sees))


@DIMS
@FEW_AND_MANY
def test_attention_values_that_hardly_count(device, dim, r, room):
    # cached tokens of large values whose probability is some 2^-150, met first, last and in the middle
    case = _case(32, [700], [8], 64, 1, r, dim, room=room)
    base = _near(np.random.default_rng(6), case)
    k, ks, v, vs, table = case[:5]
    for t, power in ((0, 24), (350, 30), (690, 34)):
        at = table[0, t // 64], t % 64
        k[at] = np.where(base > 0, -127, 127)
        ks[at] *= 3
        vs[at] *= np.float32(2.0**power)
    _hold(_attn(device, case, None), _exact(case, None))


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("what", ["zero", "small", "unmapped"])
def test_attention_first_token_without_values(device, dim, r, room, what):
    # a first token (or page) that takes nearly all of the probability and has no value, or a small one: what
    # is left of the others, 2^-20 and less, is the output
    case = _case(33, [400], [8], 16, 1, r, dim, room=room)
    base = _near(np.random.default_rng(7), case)
    k, ks, v, vs, table = case[:5]
    if what == "unmapped":  # its keys are zero; all others' scores are near -16 log2(e)
        k[:] = np.clip(np.rint(k * 0.1 - base * (16 * dim**0.5 / (base @ base) / ks.mean())), -127, 127)
        table[0, 0] = -1
    else:
        at = table[0, 0], 0
        k[at] = np.clip(np.rint(base * (22 * dim**0.5 / (base @ base)) / ks[at][0]), -127, 127)
        vs[at] = 0 if what == "zero" else vs[at] * np.float32(2.0**-30)
    _hold(_attn(device, case, None), _exact(case, None))


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [-0.2, -0.03, 0.03, 0.2])
def test_attention_values_that_grow_or_fade(device, dim, r, room, power):
    # value scales that go up or down by 2^180 in all
    case = _case(34, [880, 300], [8, 5], 16, 1, r, dim, qscale=0.5, room=room)
    vs, table, lengths = case[3], case[4], case[5]
    for b, n in enumerate(lengths):
        t = np.arange(n + 8)
        vs[table[b, t // 16], t % 16] *= np.exp2(power * (t - t.mean()))[:, None].astype(np.float32)
    _hold(_attn(device, case, None), _exact(case, None))


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [9, 13, 16, 20, 28, 60, 100])
def test_attention_equal_keys_of_large_scores(device, dim, r, room, power):
    # scores of some 2^(power + 4) and more; four equal keys of different tiles lie 2^(power + 3) above all others, so
    # that a row is the mean of their values
    case = _case(39, [300, 295], [8, 6], 16, 1, r, dim, room=room)
    base = _near(np.random.default_rng(8), case)
    k, ks, v, vs, table, _, starts = case[:7]
    places = 5, 100, 200, 290
    for t in places:
        for b in range(2):
            at = table[b, t // 16], t % 16
            k[at], ks[at] = np.clip(np.rint(base * 30), -127, 127), 0.02
    case[9][:] *= np.float32(2.0**power)
    got = _attn(device, case, None)
    for b in range(2):
        at = table[b, np.array(places) // 16], np.array(places) % 16
        want = (v[at].astype(np.float64) * vs[at].astype(np.float64)[..., None]).mean((0, 1))
        _hold(got[starts[b]:starts[b + 1]], np.broadcast_to(want, got[starts[b]:starts[b + 1]].shape))


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [17, 28, 32, 40, 90, 126])
@pytest.mark.parametrize("what", ["row", "head"])
def test_attention_query_beside_a_larger_one(device, dim, r, room, power, what):
    # one token's queries, or one head's, are 2^power times the others': these keep their scores
    case = _case(35, [300, 77], [8, 6], 16, 1, r, dim, room=room)
    q = case[9]
    large = q[5] if what == "row" else q[2, 1]
    large *= np.float32(2.0**power if power < 126 else 2.0**126 / np.abs(large).max())
    bad = 5 if what == "row" else 2
    got, want = _attn(device, case, None), _exact(case, None)
    _hold(got, want, [i for i in range(len(q)) if i != bad])
    if power < 126:  # at 2^126 its scores leave the range of FP32
        _hold(got, want)
    else:
        others = [g for g in range(q.shape[1]) if g != 1]
        if what == "head":
            _hold(got[:, others], want[:, others])


@DIMS
@FEW_AND_MANY
@pytest.mark.parametrize("power", [60, 92, 100, 110])
def test_attention_small_queries_of_large_keys(device, dim, r, room, power):
    # key scales of 2^power, queries of 2^-power: ordinary scores
    case = _case(37, [200, 31], [8, 5], 16, 1, r, dim, room=room)
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = case
    small = bf16_round(q * np.float32(2.0**-power))
    ks = (ks * np.float32(2.0**power)).astype(np.float32)
    case = (k, ks, v, vs, table, lengths, starts, page, kvh, small, most)
    _hold(_attn(device, case, None), _exact(case, None))


@FEW_AND_MANY
@pytest.mark.parametrize("dim,scales", [(64, torch.float32), (128, torch.bfloat16), (256, torch.float32)])
@pytest.mark.parametrize("batch", [5, 70])
def test_attention_odd_scales_masks_and_empty_rows(device, dim, scales, batch, r, room):
    # value scales of 0, and some 2^+-30 times the others, in a part of the sequences; any masks, rows that see
    # nothing, unmapped pages; NaN and infinite scales where nobody looks and a NaN that one row sees
    rng = np.random.default_rng(batch + dim)
    lengths = np.where(rng.random(batch) < 0.3, 0, rng.integers(0, 300, batch))
    counts = rng.integers(0, 9, batch)
    lengths, counts = [40, *lengths[1:].tolist()], [8, *counts[1:].tolist()]
    case = _case(40, lengths, counts, 16, 2, r, dim, room=room)
    k, ks, v, vs, table, _, starts = case[:7]
    sees = [s - {2} if rng.random() < 0.8 else set() for s in _sees(rng, counts, 0, 0.4)]
    sees[1] |= {2}  # sequence 0's row 1 alone sees its token 2
    held = np.zeros(ks.shape[:2], bool)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        used = set().union(*sees[starts[b]:starts[b + 1]]) if c else set()
        t = np.array(list(range(n)) + [n + j for j in used], int)
        held[table[b, t // 16], t % 16] = True
        if b % 2 and len(t):
            at = t[rng.random(len(t)) < 0.2]
            vs[table[b, at // 16], at % 16] *= np.float32(2.0) ** rng.choice([-np.inf, -30, 30], (len(at), 1))
        if b % 5 == 3 and n > 32:
            table[b, 1] = -1 if b % 2 else k.shape[0] + 7
    ks[~held], vs[~held] = np.nan, np.inf
    case = (k, bf16_round(ks), v, bf16_round(vs), *case[4:]) if scales == torch.bfloat16 else case
    at = table[0, 42 // 16], 42 % 16
    case[3][at] = np.nan
    got = _attn(device, case, sees, scales_dtype=scales)
    assert np.isnan(got[1]).all()
    # what nobody sees is 0 to the oracle, whose products with weights of 0 are not NaN then
    clean = tuple(np.where(np.isfinite(x), x, 0).astype(np.float32) for x in (case[1], case[3]))
    want = _exact((case[0], clean[0], case[2], clean[1], *case[4:]), sees)
    none = np.array([not s and not lengths[b] for b in range(batch) for s in sees[starts[b]:starts[b + 1]]])
    assert (got[:len(none)][none] == 0).all()
    _hold(got, want, [i for i in range(len(got)) if i != 1])


@FEW_AND_MANY
def test_attention_replayed_with_odd_scales(device, r, room):
    # one graph, whose value scales become odd and ordinary again between the replays
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = _case(41, [900, 70, 333], [8, 5, 8], 64, 2, r, 128,
                                                                    room=room)
    pools = [_dev(k.reshape(*k.shape[:2], -1), device), _dev(ks, device), _dev(v.reshape(*v.shape[:2], -1), device),
             _dev(vs, device)]
    state = [_dev(np.asarray(t, np.int32), device) for t in (table, lengths, starts)]
    x, out = _dev(q, device, torch.bfloat16), torch.zeros(q.shape, dtype=torch.bfloat16, device=device)
    work = torch.empty(1 << 27, dtype=torch.uint8, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_tree_attention(x, *pools, *state, page_size=page, kv_heads=kvh, max_count=most, out=out, workspace=work)
    for odd in (False, True, False, True):
        changed = vs.copy()
        if odd:
            changed[table[0, :10:3], 7] *= np.float32(2.0**40)
            changed[table[2, 1], 30:40] = 0
        pools[3].copy_(_dev(changed, device))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        case = (k, ks, v, changed, table, lengths, starts, page, kvh, q, most)
        _hold(out.float().cpu().numpy(), _exact(case, None))
