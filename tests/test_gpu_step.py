"""GPU tests of a step with several new tokens per sequence, against the oracle in 64 bits.

Whole numbers, codes and scales must be equal. With A = sum p |v| / sum p an attention output may be off by
  2^-8 |want|     its rounding to BF16 (half a step),
  2^-11 A         the rounding of each probability to FP16,
  2 d A           the scores: d bounds their error, (2^-15 + D 2^-24) max|q| sum|k| / sqrt(D). The first
                  term is half a step of q held in 16 bits, the second a chain of D roundings in FP32,
  2^-16 A         the hardware exponential (1 ulp) of FP32 arguments,
  n 2^-21 max vs  probabilities near 0: p vs f is held in FP16, whose step below 2^-14 is 2^-24, with a factor
                  f of at least 2^3 / max vs (the kernel brings the largest value scale to 2^3 or more), so
                  that p vs is off by at most 2^-25 2^-3 max vs; times a code of at most 127, over n keys; the
                  sum of p that divides it is at least 1. (Found with a row whose largest key has code 0 and
                  all others p < 1e-9: 9.5e-11 over the bound without this term, at values of size 1.)
  n 2^-25 A       the sums over n keys: chains of n / 16 roundings, of codes up to 255 (the INT8 codes + 128)
                  where sum p |v| has their mean size, a seventh.
"""

import numpy as np
import pytest
import torch

from oracle import step as oracle
from oracle.packed_q6 import bf16_round
from q6moe import (keep_accepted, paged_decode_attention, paged_tree_attention, plan_pages, release_pages,
                   write_paged, write_tokens)

pytestmark = pytest.mark.gpu


def _dev(a, device, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(device)
    return t if dtype is None else t.to(dtype)


# ---------------------------------------------------------------------------
# Pages and slots
# ---------------------------------------------------------------------------
def _plan_case(seed, batch, pps, page, most, tree, extra, short=0):
    """A table whose cached tokens and a few of the new ones are mapped, and a free stack, ``short`` pages too small."""
    rng = np.random.default_rng(seed)
    cap = pps * page
    lengths = rng.integers(0, cap + 1, batch).astype(np.int32)
    counts = rng.integers(0, most + 1, batch).astype(np.int32)
    rows = int(counts.sum()) + extra or 1
    pages = rng.permutation(batch * pps + 20).astype(np.int32)
    table = pages[:batch * pps].reshape(batch, pps).copy()
    held = -(-lengths // page)
    table[np.arange(pps) >= held[:, None]] = -1
    ahead = (np.arange(pps) == held[:, None]) & (rng.random((batch, 1)) < 0.3)
    table[ahead] = 2000 + rng.permutation(batch * pps + 1000)[:ahead.sum()]
    need = sum(int((table[b, lengths[b] // page:-(-(lengths[b] + counts[b]) // page)] < 0).sum()) if counts[b] else 0
               for b in range(batch))
    count = max(0, need - short) if short else need + 5
    free = np.concatenate([5000 + rng.permutation(count), [-7] * 3]).astype(np.int32)
    parents = rng.integers(-1, most + 1, rows).astype(np.int32) if tree else None
    return table, lengths, counts, free, count, rows, parents


@pytest.mark.parametrize("seed,batch,pps,page,most,tree,extra,short", [
    (1, 1, 1, 1, 1, False, 0, 0), (2, 5, 7, 16, 40, False, 3, 0), (3, 300, 9, 64, 200, False, 100, 0),
    (4, 3, 600, 4, 2100, False, 0, 0), (5, 40, 8, 16, 30, False, 0, 11), (6, 1, 4, 8, 1, True, 2, 0),
    (7, 9, 12, 16, 64, True, 0, 0), (8, 33, 40, 7, 65, True, 17, 0), (9, 6, 64, 64, 256, True, 5, 4),
    (10, 700, 3, 5, 4, True, 1, 50), (11, 9, 700, 8, 3000, False, 7, 0), (12, 70, 80, 16, 150, True, 300, 20),
    (13, 1024, 5, 64, 3, False, 0, 0), (14, 1025, 4, 64, 3, False, 9, 0), (15, 3, 40, 4, 126, False, 0, 0),
])
def test_plan_and_release(device, seed, batch, pps, page, most, tree, extra, short):
    table, lengths, counts, free, count, rows, parents = _plan_case(seed, batch, pps, page, most, tree, extra, short)
    want = oracle.plan(table, lengths, counts, free, count, page, rows, parents, most if tree else None)
    t, f, n = _dev(table, device), _dev(free, device), _dev(np.array([count], np.int32), device)
    args = t, _dev(lengths, device), _dev(counts, device), f, n
    kw = dict(page_size=page, rows=rows, parents=None if parents is None else _dev(parents, device),
              max_count=most if tree else None)
    plan = plan_pages(*args, **kw)

    def check(plan):
        for got, w in ((plan.starts, want[0]), (plan.slots, want[1]), (plan.positions, want[2]), (t, want[5])):
            np.testing.assert_array_equal(got.cpu().numpy(), w)
        assert plan.missing.item() == want[4] and n.item() == want[6]
        if tree:
            np.testing.assert_array_equal(plan.masks.cpu().numpy(), oracle.masks_of(want[3], -(-most // 64)))
        else:
            assert plan.masks is None

    check(plan)
    if not short:  # nothing left to take
        check(plan_pages(*args, **kw, out=plan))
    back = oracle.release(want[5], lengths, free, want[6], page)
    release_pages(t, args[1], f, n, page_size=page)
    np.testing.assert_array_equal(t.cpu().numpy(), back[0])
    np.testing.assert_array_equal(f.cpu().numpy(), back[1])
    assert n.item() == back[2]


def test_plan_drops_what_does_not_fit(device):
    # rows for 5 of 3 + 4 tokens; negative lengths and counts; a stack that says more than it holds
    table = np.full((3, 4), -1, np.int32)
    lengths, counts, free = np.array([-4, 2, 3]), np.array([3, -2, 4]), np.array([4, 3], np.int32)
    want = oracle.plan(table, lengths, counts, free, 9, 2, 5)
    t, n = _dev(table, device), _dev(np.array([9], np.int32), device)
    plan = plan_pages(t, _dev(lengths, device), _dev(counts, device), _dev(free, device), n, page_size=2, rows=5)
    assert plan.starts.tolist() == want[0].tolist() == [0, 3, 3, 5]
    assert plan.slots.tolist() == want[1].tolist() and plan.missing.item() == want[4]
    assert t.cpu().tolist() == want[5].tolist() and n.item() == want[6] == 0


def test_release_without_room_leaves_pages_mapped(device):
    table, free = np.array([[1, 2, 3], [4, 5, 6]], np.int32), np.array([9, 9, 9, 9], np.int32)
    want = oracle.release(table, [4, 0], free, 2, 4)
    t, f, n = _dev(table, device), _dev(free, device), _dev(np.array([2], np.int32), device)
    release_pages(t, _dev(np.array([4, 0], np.int32), device), f, n, page_size=4)
    assert t.cpu().tolist() == want[0].tolist() and f.tolist() == want[1].tolist() and n.item() == want[2] == 4


# ---------------------------------------------------------------------------
# Ragged write
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,pages,page,kvh,dim,group,values,scales", [
    (1, 1, 1, 1, 64, 64, "f32", "f32"), (7, 5, 16, 4, 128, 128, "bf16", "f32"),
    (300, 40, 16, 2, 128, 32, "bf16", "bf16"), (33, 9, 5, 3, 24, 24, "f32", "bf16"),
    (65, 3, 64, 8, 256, 256, "bf16", "f32"), (50, 7, 10, 1, 7, 7, "f32", "f32"),
])
def test_write_tokens(device, rows, pages, page, kvh, dim, group, values, scales):
    rng = np.random.default_rng(rows)
    types = dict(f32=torch.float32, bf16=torch.bfloat16)
    n = pages * page
    slots = np.full(rows, -1, np.int64)
    live = rng.random(rows) < 0.8
    slots[live] = rng.permutation(n + 2 * rows)[:live.sum()]  # some past the pool
    fused = rng.standard_normal((rows, 3, kvh, dim)).astype(np.float32) * 10.0 ** rng.integers(-3, 3, (rows, 3, kvh, 1))
    fused[rows // 2, 1] = 0  # a row of zeros: scale 0
    x = _dev(fused, device, types[values])
    xv = x.float().cpu().numpy()
    pools = rng.integers(-127, 128, (2, pages, page, kvh * dim)).astype(np.int8)
    sc = torch.rand(2, pages, page, kvh * dim // group, device=device).to(types[scales])
    want = [oracle.write(pools[i].reshape(n, -1), sc[i].float().cpu().numpy().reshape(n, -1),
                         xv[:, 1 + i].reshape(rows, -1), slots, group, scales) for i in range(2)]
    p = _dev(pools, device)
    for stride in ("apart", "together"):
        key, value = (x[:, 1 + i] if stride == "apart" else x[:, 1 + i].reshape(rows, -1).contiguous()
                      for i in range(2))
        got, gs = p.clone(), sc.clone()
        write_tokens(got[0], gs[0], got[1], gs[1], key, value, _dev(slots, device), kv_heads=kvh, head_dim=dim,
                     group=group)
        for i in range(2):
            np.testing.assert_array_equal(got[i].cpu().numpy().reshape(n, -1), want[i][0])
            np.testing.assert_array_equal(gs[i].float().cpu().numpy().reshape(n, -1), want[i][1])


def test_write_tokens_is_write_paged_bit_for_bit(device):
    # every exponent, infinities, NaN and quotients next to half a step
    rows, kvh, dim, page = 2048, 2, 128, 16
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(rows, kvh * dim, generator=gen, device=device)
    x *= torch.exp2(torch.randint(-140, 120, (rows, 1), generator=gen, device=device).float())
    half = torch.randint(-127, 127, (rows // 2, kvh * dim), generator=gen, device=device) + 0.5
    half[:, ::dim] = 127
    x[::2] = half * torch.exp2(torch.randint(-130, 100, (rows // 2, 1), generator=gen, device=device).float())
    x[5, 3], x[6, 4], x[7, 5] = float("inf"), float("-inf"), float("nan")
    table = torch.randperm(rows // page, generator=gen, device=device).int().view(1, -1)
    t = torch.arange(rows, device=device)
    slots = table[0, t // page].long() * page + t % page
    for dtype in (torch.float32, torch.bfloat16):
        for st in (torch.float32, torch.bfloat16):
            pool = torch.zeros(3, rows // page, page, kvh * dim, dtype=torch.int8, device=device)
            sc = torch.zeros(3, rows // page, page, kvh, dtype=st, device=device)
            xx = x.to(dtype)
            write_paged(pool[0], sc[0], table.expand(rows, -1), xx, t.int(), page_size=page, kv_heads=kvh, head_dim=dim)
            write_tokens(pool[1], sc[1], pool[2], sc[2], xx, xx, slots, kv_heads=kvh, head_dim=dim)
            for i in (1, 2):
                assert torch.equal(pool[0], pool[i])
                assert torch.equal(sc[0].view(torch.uint8), sc[i].view(torch.uint8))


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _cache(rng, pages, page, kvh, dim):
    g = rng.standard_normal((pages, page, kvh, dim)).astype(np.float32)
    sc = (np.abs(g).max(-1) / np.float32(127)).astype(np.float32)
    return np.clip(np.rint(g / sc[..., None]), -127, 127).astype(np.int8), sc


def _attn(device, case, sees, *, q=None, scales_dtype=torch.float32, masks=None, words=None, fill=None, **kw):
    k, ks, v, vs, table, lengths, starts, page, kvh, qv, most = case
    rows = qv.shape[0]
    if sees is not None:
        words = words or -(-most // 64)
        masks = _dev(oracle.masks_of(sees, words), device)
    out = None if fill is None else torch.full(qv.shape, fill, dtype=torch.bfloat16, device=device)
    got = paged_tree_attention(
        _dev(qv, device, torch.bfloat16) if q is None else q, _dev(k.reshape(*k.shape[:2], -1), device),
        _dev(ks, device, scales_dtype), _dev(v.reshape(*v.shape[:2], -1), device), _dev(vs, device, scales_dtype),
        _dev(table, device), _dev(np.asarray(lengths, np.int32), device), _dev(np.asarray(starts, np.int32), device),
        masks, page_size=page, kv_heads=kvh, max_count=most, out=out, **kw)
    return got.float().cpu().numpy()


def _case(seed, lengths, counts, page, kvh, r, dim, extra=0, spare_pages=3, width=None, qscale=2.0, room=False):
    """``room``: tables wide enough that calls of many rows are taken for large ones."""
    rng = np.random.default_rng(seed)
    batch, most = len(lengths), max(1, *counts)
    pps = width or max(-(-(n + c) // page) for n, c in zip(lengths, counts)) + 1
    pages = batch * pps + spare_pages
    k, ks = _cache(rng, pages, page, kvh, dim)
    v, vs = _cache(rng, pages, page, kvh, dim)
    table = rng.permutation(pages)[:batch * pps].reshape(batch, pps).astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(counts)])
    q = bf16_round((rng.standard_normal((max(1, int(starts[-1]) + extra), kvh * r, dim)) * qscale).astype(np.float32))
    if room:
        wide = 2**36 // (4 * q.size * page) + 1
        table = np.concatenate([table, np.full((batch, wide), -1, np.int32)], 1)
    return k, ks, v, vs, table, lengths, starts, page, kvh, q, most


def _sees(rng, counts, extra, chance=None):
    """Random ancestors for each row: a tree, or any set of tokens (with ``chance``; empty ones too)."""
    out = []
    for c in counts:
        seen = []
        for j in range(c):
            if chance is not None:
                seen.append({jj for jj in range(c) if rng.random() < chance})
            else:
                p = int(rng.integers(-1, j)) if j else -1
                seen.append({j} | (seen[p] if p >= 0 else set()))
        out += seen
    return out + [set()] * extra


def _check(got, case, sees, rows=None, scales=None):
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = case
    if scales == torch.bfloat16:
        ks, vs = bf16_round(ks), bf16_round(vs)
    want, spread, slope = oracle.attention(q, k, ks, v, vs, table, lengths, starts, sees, page, most)
    live = ~np.isnan(want)
    top = np.abs(q).max(-1)
    d = (2.0**-15 + q.shape[2] * 2.0**-24) * top * slope
    n = min(max(lengths) + most, table.shape[1] * page)
    tol = 2.0**-8 * np.abs(want) + (2.0**-11 + 2 * d[..., None] + 2.0**-16 + n * 2.0**-25) * spread
    tol += n * 2.0**-21 * np.nanmax(np.where(np.isfinite(vs), vs, 0))
    over = (np.abs(got - want) - tol)[live]
    assert np.isfinite(got[live]).all() and (over <= 0).all(), over.max()
    return live


@pytest.mark.parametrize("page,kvh,r,dim,lengths,counts,extra", [
    (16, 1, 1, 64, [0], [1], 0),                                   # one token, no cache
    (64, 4, 8, 128, [63, 64, 65, 1], [1, 1, 1, 1], 0),             # single tokens, tile edges
    (16, 2, 7, 64, [100, 0, 31, 400], [5, 3, 0, 9], 4),            # page ends inside tiles, an idle sequence, padding
    (128, 1, 16, 256, [200, 511], [16, 11], 0),                    # wide heads
    (5, 3, 3, 128, [129, 64, 7], [4, 17, 33], 1),                  # pages of 5 tokens
    (256, 2, 6, 128, [700, 0], [64, 64], 0),                       # more rows than one tile
    (64, 1, 8, 64, [33], [70], 2),                                 # two words
    (1, 2, 1, 64, [70, 3], [2, 5], 0),                             # pages of one token
    (32, 1, 5, 128, [1000], [256], 0),                             # the largest tree
    (64, 1, 4, 128, [2500, 5000, 17], [7, 2, 3], 0),               # split over keys
])
@pytest.mark.parametrize("kind", ["tree", "any", "chain"])
@pytest.mark.parametrize("room", [False, True], ids=["small", "large"])
def test_attention(device, page, kvh, r, dim, lengths, counts, extra, kind, room):
    case = _case(len(lengths) * page + dim, lengths, counts, page, kvh, r, dim, extra, room=room)
    rng = np.random.default_rng(7)
    sees = None if kind == "chain" else _sees(rng, counts, extra, 0.3 if kind == "any" else None)
    scales = torch.bfloat16 if kind == "any" else torch.float32
    got = _attn(device, case, sees, scales_dtype=scales, fill=7.0)
    live = _check(got, case, sees, scales=scales)
    assert (got[~live] == 7.0).all()  # rows behind the last sequence
    again = _attn(device, case, sees, scales_dtype=scales, fill=7.0)
    np.testing.assert_array_equal(got, again)


@pytest.mark.parametrize("batch,kvh,r,dim,count,most_len,spare_count", [
    (300, 2, 2, 64, 1, 400, 0),    # few rows, more tiles than half the places: chunks run in turns
    (520, 4, 1, 128, 1, 30, 0),    # so many that none is split
    (70, 4, 9, 64, 12, 300, 5),    # many rows, in turns; max_count above any count
    (390, 8, 25, 64, 4, 20, 0),    # many rows, none split
    (64, 2, 3, 128, 3, 700, 0),    # the most that a wave looks through by itself
    (65, 2, 3, 128, 3, 700, 1),    # and more
    (1030, 1, 2, 64, 2, 60, 0),    # more than one workgroup has threads
    (2100, 2, 4, 256, 1, 15, 0),
    (80, 1, 4, 128, 2, 9000, 0),   # split into many chunks
])
def test_attention_of_many_sequences(device, batch, kvh, r, dim, count, most_len, spare_count):
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, most_len + 1, batch)
    counts = rng.integers(0, count + 1, batch)
    k, ks, v, vs, table, _, starts, page, kvh, q, _ = _case(batch, lengths, counts, 16, kvh, r, dim, 2)
    got = _attn(device, (k, ks, v, vs, table, lengths, starts, page, kvh, q, count + spare_count), None, fill=9.0)
    assert (got[starts[-1]:] == 9.0).all()
    for b in rng.permutation(batch)[:12]:  # each by itself
        a, e = starts[b], starts[b + 1]
        if e > a:
            one = (k, ks, v, vs, table[b:b + 1], lengths[b:b + 1], np.array([0, e - a]), page, kvh, q[a:e], count)
            _check(got[a:e], one, None)


@pytest.mark.parametrize("batch,kvh,r,dim,count", [(600, 4, 1, 64, 1), (300, 8, 2, 128, 2), (60, 2, 3, 128, 2)])
def test_attention_of_long_sequences_among_many(device, batch, kvh, r, dim, count):
    # two long ones among short ones are split, whatever fills the chip; pages are shared
    rng = np.random.default_rng(batch)
    k, ks = _cache(rng, 64, 64, kvh, dim)
    v, vs = _cache(rng, 64, 64, kvh, dim)
    lengths = rng.integers(0, 60, batch)
    lengths[[7, batch - 2]] = 20000, 9001
    counts = rng.integers(0, count + 1, batch)
    counts[[7, batch - 2]] = count
    starts = np.concatenate([[0], np.cumsum(counts)])
    table = rng.integers(0, 64, (batch, 320)).astype(np.int32)
    q = bf16_round((rng.standard_normal((int(starts[-1]), kvh * r, dim)) * 2).astype(np.float32))
    got = _attn(device, (k, ks, v, vs, table, lengths, starts, 64, kvh, q, count), None)
    for b in [7, batch - 2, *rng.permutation(batch)[:10]]:
        a, e = starts[b], starts[b + 1]
        if e > a:
            one = (k, ks, v, vs, table[b:b + 1], lengths[b:b + 1], np.array([0, e - a]), 64, kvh, q[a:e], count)
            _check(got[a:e], one, None)


@pytest.mark.parametrize("batch", [9, 70])
def test_attention_replayed_with_other_lengths(device, batch):
    # the same graph over other lengths and counts: how the work is cut is found anew each time
    rng = np.random.default_rng(batch)
    k, ks, v, vs, table, lengths, starts, page, kvh, q, most = _case(
        batch, [2500] * batch, [3] * batch, 64, 2, 4, 128)
    pools = [_dev(k.reshape(*k.shape[:2], -1), device), _dev(ks, device), _dev(v.reshape(*v.shape[:2], -1), device),
             _dev(vs, device)]
    state = [_dev(np.asarray(t, np.int32), device) for t in (table, lengths, starts)]
    x, out = _dev(q, device, torch.bfloat16), torch.empty(q.shape, dtype=torch.bfloat16, device=device)
    work = torch.empty(1 << 28, dtype=torch.uint8, device=device)

    def attend(to, workspace):
        return paged_tree_attention(x, *pools, *state, page_size=page, kv_heads=kvh, max_count=most, out=to,
                                    workspace=workspace)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(out, work)
    for turn in range(4):
        state[1].copy_(_dev(rng.integers(0, (2500, 40, 2500, 700)[turn], batch).astype(np.int32), device))
        counts = rng.integers(0, 4, batch)
        state[2].copy_(_dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device))
        out.fill_(5.0)
        graph.replay()
        want = attend(torch.full_like(out, 5.0), None)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("room", [False, True], ids=["small", "large"])
def test_attention_chain_of_a_prompt(device, dim, room):
    case = _case(3, [0, 300], [333, 130], 64, 2, 3, dim, room=room)
    _check(_attn(device, case, None), case, None)


# query heads per KV head: few rows, and many; of these as small calls and as large ones
FEW_AND_MANY = pytest.mark.parametrize("r,room", [(4, False), (20, False), (20, True)])


@FEW_AND_MANY
def test_attention_rows_that_see_nothing(device, r, room):
    # no cached tokens, empty masks: 0; a mask that names tokens past the sequence's own names nothing
    case = _case(11, [0, 0, 9], [3, 2, 9], 16, 2, r, 128, room=room)
    sees = [set(), {2}, {0, 5, 63}, set(), {0}, set(), {1, 2, 40}, {8}, {0}, {3, 4}, set(), {7}, {6, 5}, {8, 2}]
    got = _attn(device, case, sees)
    _check(got, case, sees)
    assert (got[0] == 0).all() and (got[3] == 0).all()
    assert got[1].any(-1).all()  # row 1 is one key's value, some of whose codes are 0


@FEW_AND_MANY
def test_attention_garbage_where_nothing_looks(device, r, room):
    # scales of every place that no row sees are NaN or infinite, codes are -128
    lengths, counts = [70, 5], [6, 4]
    case = _case(12, lengths, counts, 16, 2, r, 128, room=room)
    k, ks, v, vs, table = case[:5]
    sees = [s - {3} for s in _sees(np.random.default_rng(1), counts, 0)]
    held = np.zeros(ks.shape[:2], bool)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        for t in range(n + c):
            if t != n + 3:
                held[table[b, t // 16], t % 16] = True
    want = _attn(device, case, sees)
    for x, bad in ((ks, np.nan), (vs, np.inf)):
        x[~held] = bad
    k[~held], v[~held] = -128, -128
    got = _attn(device, case, sees)
    np.testing.assert_array_equal(got, want)
    for bad in ((np.nan, -np.inf), (3e38, 3e38), (-3e38, 1e-38)):
        vs[~held], ks[~held] = bad
        np.testing.assert_array_equal(_attn(device, case, sees), want)


@FEW_AND_MANY
def test_attention_scales_far_apart(device, r, room):
    # values whose scales span 2^40, some of them 0, in an order that grows; scores far from 0
    case = _case(13, [900], [8], 64, 1, r, 128, qscale=6.0, room=room)
    k, ks, v, vs, table = case[:5]
    rng = np.random.default_rng(2)
    vs *= 2.0 ** rng.integers(-20, 21, vs.shape).astype(np.float32)
    vs[rng.random(vs.shape) < 0.1] = 0
    ks[rng.random(ks.shape) < 0.1] = 0
    _check(_attn(device, case, None), case, None)
    for scale in (2.0**-60, 2.0**60):  # all of them small, or large
        vs2 = (vs * np.float32(scale)).astype(np.float32)
        _check(_attn(device, (k, ks, v, vs2, *case[4:]), None), (k, ks, v, vs2, *case[4:]), None)


@FEW_AND_MANY
def test_attention_queries_far_apart(device, r, room):
    # rows of queries from 2^-100 to 2^100 (with keys to match), one of zeros
    case = _case(14, [130], [6], 64, 1, r, 128, room=room)
    q = case[9]
    for i, e in enumerate((0, -100, -20, 3)):
        q[i] *= np.float32(2.0**e)
    q[4] = 0
    _check(_attn(device, case, None), case, None)
    big = bf16_round(case[9] * np.float32(2.0**100))
    big[4] = 0
    case = (case[0], case[1] * np.float32(2.0**-100), *case[2:9], big, case[10])
    _check(_attn(device, case, None), case, None)


@FEW_AND_MANY
def test_attention_unmapped_pages_and_short_tables(device, r, room):
    # unmapped pages read as zero; tokens past the table's width are not seen
    case = _case(15, [60, 40], [8, 8], 16, 2, r, 64, width=4, room=room)
    k, ks, v, vs, table = case[:5]
    table[0, 1], table[1, 2] = -1, k.shape[0] + 4
    sees = _sees(np.random.default_rng(3), [8, 8], 0)
    _check(_attn(device, case, sees), case, sees)
    _check(_attn(device, case, None), case, None)


def test_attention_short_tables_of_many_sequences(device):
    # enough of them that 6 tokens of 20 heads are many rows; tokens 32 and on are not seen
    lengths = [20 + b % 13 for b in range(60)]
    case = _case(19, lengths, [6] * 60, 16, 2, 20, 64, width=2)
    _check(_attn(device, case, None), case, None)
    sees = _sees(np.random.default_rng(4), [6] * 60, 0)
    _check(_attn(device, case, sees), case, sees)


def test_attention_counts_past_max_count_and_strided_queries(device):
    case = _case(16, [50, 3], [6, 5], 16, 2, 4, 128)
    rows, hq, dim = case[9].shape
    small = (*case[:10], 4)
    got = _attn(device, small, None, fill=3.0)
    live = _check(got, small, None)
    assert (got[~live] == 3.0).all() and not live[4].any()
    wide = torch.randn(rows, hq + 4, dim, device=device).to(torch.bfloat16)
    wide[:, 2:2 + hq] = _dev(case[9], device, torch.bfloat16)
    np.testing.assert_array_equal(_attn(device, case, None, q=wide[:, 2:2 + hq]), _attn(device, case, None))


def test_attention_of_single_tokens_is_decode_attention(device):
    # the same step through paged_decode_attention, whose keys, values, scores and
    # probabilities are rounded to BF16 on the way: five half steps of 2^-8
    lengths = [511, 64, 1, 300]
    case = _case(17, lengths, [1] * 4, 64, 4, 8, 128)
    k, ks, v, vs, table, _, _, page, kvh, q, _ = case
    got = _attn(device, case, None)
    want = paged_decode_attention(
        _dev(q, device, torch.bfloat16), _dev(k.reshape(*k.shape[:2], -1), device), _dev(ks, device),
        _dev(v.reshape(*v.shape[:2], -1), device), _dev(vs, device), _dev(table, device),
        _dev(np.array(lengths, np.int32) + 1, device), page_size=page, kv_heads=kvh).float().cpu().numpy()
    _, spread, slope = oracle.attention(q, k, ks, v, vs, table, lengths, case[6], None, page, 1)
    # a score s of size up to max|q| slope is rounded twice and its key once
    score = np.abs(q).max(-1) * slope
    tol = 2.0**-8 * (np.abs(want) * 2 + (2 + 6 * score[..., None]) * spread)
    assert (np.abs(got - want) <= tol).all()


def test_attention_long_sequence_of_shared_pages(device):
    # 65536 tokens of a pool of 64 pages; every sequence names them again and again
    rng = np.random.default_rng(18)
    k, ks = _cache(rng, 64, 64, 1, 64)
    v, vs = _cache(rng, 64, 64, 1, 64)
    table = rng.integers(0, 64, (2, 1024)).astype(np.int32)
    lengths, starts = [65533, 40000], np.array([0, 3, 5])
    q = bf16_round(rng.standard_normal((5, 2, 64)).astype(np.float32) * 2)
    case = (k, ks, v, vs, table, lengths, starts, 64, 1, q, 3)
    _check(_attn(device, case, None), case, None)


def test_attention_offsets_past_32_bits(device):
    # a pool of 2^32 + code bytes and more: the pages in use are its first and last
    pages, page, kvh, dim = 33000, 256, 4, 128  # 4.3 GB a pool
    k = torch.zeros(pages, page, kvh * dim, dtype=torch.int8, device=device)
    v = torch.zeros_like(k)
    ks = torch.zeros(pages, page, kvh, device=device)
    vs = torch.zeros_like(ks)
    case = _case(19, [600], [4], page, kvh, 4, dim, width=3, spare_pages=0)
    sk, sks, sv, svs = case[:4]
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    for i, pg in enumerate(case[4][0]):
        for big, small in ((k, sk.reshape(3, page, -1)), (ks, sks), (v, sv.reshape(3, page, -1)), (vs, svs)):
            big[table[0, i]] = _dev(small[pg], device)
    want = _attn(device, case, None)
    got = paged_tree_attention(_dev(case[9], device, torch.bfloat16), k, ks, v, vs, _dev(table, device),
                               _dev(np.array([600], np.int32), device), _dev(np.array([0, 4], np.int32), device),
                               page_size=page, kv_heads=kvh, max_count=4).float().cpu().numpy()
    np.testing.assert_array_equal(got, want)
    # and a write and a move in the last page
    slots = torch.tensor([pages * page - 1, -1, 3], device=device)
    x = torch.randn(3, kvh * dim, device=device)
    write_tokens(k, ks, v, vs, x, x, slots, kv_heads=kvh, head_dim=dim)
    assert torch.equal(k[-1, -1], v[-1, -1]) and k[-1, -1].abs().max() == 127 and k[0, 3].abs().max() == 127
    kept = k[-1, 7].clone()
    keep_accepted([(k, ks), (v, vs)], torch.tensor([[pages - 1]], device=device), torch.tensor([5], device=device),
                  torch.tensor([[2]], device=device), torch.tensor([1], device=device), page_size=page)
    assert torch.equal(k[-1, 5], kept)


# ---------------------------------------------------------------------------
# Accepted paths
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("batch,page,pps,chans,groups,dtype,layers,most", [
    (1, 16, 2, 64, 1, torch.float32, 1, 1), (5, 7, 9, 512, 4, torch.float32, 3, 12),
    (3, 64, 5, 36, 3, torch.bfloat16, 2, 5), (2, 16, 40, 130, 1, torch.bfloat16, 70, 256),
    (9, 64, 3, 1024, 32, torch.float32, 1, 40),
])
def test_keep_accepted(device, batch, page, pps, chans, groups, dtype, layers, most):
    rng = np.random.default_rng(batch * page)
    pages, cap = batch * pps + 2, pps * page
    codes = rng.integers(-128, 128, (layers, 2, pages, page, chans)).astype(np.int8)
    scales = torch.rand(layers, 2, pages, page, groups, device=device).to(dtype)
    bits = scales.view(torch.uint8).view(layers, 2, pages, page, -1).cpu().numpy()
    table = rng.permutation(pages)[:batch * pps].reshape(batch, pps).astype(np.int32)
    table[rng.random(table.shape) < 0.05] = -1
    lengths = rng.integers(0, max(1, cap - most // 2), batch).astype(np.int32)
    lengths[-1] -= 2 * lengths[-1] * (batch > 3)  # below 0: as 0
    path = np.sort(rng.integers(-1, most + 10, (batch, most)), 1).astype(np.int32)
    path[0] = rng.permutation(most)  # any order: the places are read before they are written
    accepted = rng.integers(0, most + 3, batch).astype(np.int32)
    accepted[0] = most
    got = _dev(codes, device)
    keep_accepted([(got[0], scales[0])] + ([(got[1:], scales[1:])] if layers > 1 else []), _dev(table, device),
                  _dev(lengths, device), _dev(path, device), _dev(accepted, device), page_size=page)
    after = scales.view(torch.uint8).view(layers, 2, pages, page, -1).cpu().numpy()
    for n in range(layers):
        for i in range(2):
            np.testing.assert_array_equal(got[n, i].cpu().numpy(),
                                          oracle.keep(codes[n, i], table, lengths, path, accepted, page))
            np.testing.assert_array_equal(after[n, i], oracle.keep(bits[n, i], table, lengths, path, accepted, page))


# ---------------------------------------------------------------------------
# Refusals and a whole step
# ---------------------------------------------------------------------------
def test_refusals(device):
    i32 = dict(dtype=torch.int32, device=device)
    table, one = torch.zeros(2, 3, **i32), torch.zeros(1, **i32)
    two, free = torch.zeros(2, **i32), torch.zeros(4, **i32)
    ok = dict(page_size=4, rows=2)
    for args, kw, text in (
            ((table.long(), two, two, free, one), ok, "page_table must be a contiguous torch.int32"),
            ((table[:, :2], two, two, free, one), ok, "page_table must be a contiguous"),
            ((table, one, two, free, one), ok, "lengths must be"), ((table, two, one, free, one), ok, "counts must be"),
            ((table, two, two, free.float(), one), ok, "free_pages must be"),
            ((table, two, two, free, two), ok, "free_count must be"),
            ((table, two, two, free, one), dict(ok, rows=0), "rows must be a positive integer"),
            ((table, two, two, free, one), dict(ok, page_size=0), "page_size must be"),
            ((table, two, two, free, one), dict(ok, parents=two), "a tree needs max_count"),
            ((table, two, two, free, one), dict(ok, parents=two, max_count=257), "a tree needs max_count"),
            ((table, two, two, free, one), dict(ok, parents=one, max_count=4), "parents must be"),
    ):
        with pytest.raises(ValueError, match=text):
            plan_pages(*args, **kw)
    plan = plan_pages(table, two, two, free, one, **ok)
    with pytest.raises(ValueError, match="out.slots must be"):
        plan_pages(table, two, two, free, one, page_size=4, rows=3, out=plan)
    with pytest.raises(ValueError, match="out.masks must be"):
        plan_pages(table, two, two, free, one, page_size=4, rows=2, parents=two, max_count=2, out=plan)
    pool = torch.zeros(3, 4, 128, dtype=torch.int8, device=device)
    scales, other = torch.ones(3, 4, 1, device=device), torch.zeros(3, 4, 128, dtype=torch.int8, device=device)
    x, slots = torch.zeros(2, 128, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    good = dict(kv_heads=1, head_dim=128)
    for args, kw, text in (
            ((pool, scales, other, scales + 1, x, x[:1], slots), good, "value must be"),
            ((pool, scales, other, scales + 1, x, x.half(), slots), good, "same type"),
            ((pool, scales, other, scales + 1, x.half(), x.half(), slots), good, "dtype must be"),
            ((pool, scales, other, scales + 1, x, x, slots[None]), good, "slots must be"),
            ((pool, scales, pool, scales, x, x, slots), good, "same memory"),
            ((pool, scales, other[:2], scales[:2], x, x, slots), good, "same size"),
            ((pool, scales, other, scales.bfloat16(), x, x, slots), good, "scale type"),
            ((pool.float(), scales, other, scales, x, x, slots), good, "k pool must be"),
            ((pool, scales, other, scales, x, x, slots), dict(good, group=48), "group must divide"),
    ):
        with pytest.raises(ValueError, match=text):
            write_tokens(*args, **kw)
    q, starts = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=device), torch.tensor([0, 1, 2], **i32)
    base = dict(q=q, k_pool=pool, k_scales=scales, v_pool=other, v_scales=scales, page_table=table, lengths=two,
                starts=starts, page_size=4, kv_heads=1, max_count=1)
    masks = torch.zeros(2, 1, dtype=torch.int64, device=device)
    for change, text in (
            (dict(q=q.float()), "q must be BF16"), (dict(q=q[..., :96]), "head_dim 64, 128 or 256"),
            (dict(kv_heads=3), "multiple of kv_heads"), (dict(max_count=0), "max_count must be"),
            (dict(page_size=2), "page_size"), (dict(v_pool=other[:2], v_scales=scales[:2]), "same size"),
            (dict(starts=two), "starts"), (dict(lengths=one), "lengths"), (dict(masks=masks[:1]), "masks must be"),
            (dict(masks=masks.int()), "masks must be"), (dict(masks=masks, max_count=65), "bit for each"),
            (dict(out=q[:1]), "out must be"),
            (dict(workspace=torch.zeros(8, dtype=torch.uint8, device=device)), "workspace"),
            (dict(k_scales=scales.half()), "k scales must be"),
    ):
        with pytest.raises(ValueError, match=text):
            paged_tree_attention(**{**base, **change})
    path = torch.zeros(2, 2, **i32)
    for caches, args, text in (
            ([(pool, scales)], (table, two, path[:1], two), "path must be"),
            ([(pool, scales)], (table, one, path, two), "lengths and accepted"),
            ([(pool, scales), (pool, scales)], (table, two, path, two), "only once"),
            ([(pool, scales), (other[:2], scales[:2])], (table, two, path, two), "same pages"),
            ([(pool[:, :2].contiguous(), scales)], (table, two, path, two), "codes must be"),
            ([(pool, scales[:2])], (table, two, path, two), "scales must be"),
    ):
        with pytest.raises(ValueError, match=text):
            keep_accepted(caches, *args, page_size=4)


def _step_state(device, batch, pps, page, kvh, dim, layers):
    pages = batch * pps
    return dict(
        table=torch.full((batch, pps), -1, dtype=torch.int32, device=device),
        free=torch.arange(pages, dtype=torch.int32, device=device),
        count=torch.tensor([pages], dtype=torch.int32, device=device),
        lengths=torch.zeros(batch, dtype=torch.int32, device=device),
        codes=torch.zeros(layers, 2, pages, page, kvh * dim, dtype=torch.int8, device=device),
        scales=torch.zeros(layers, 2, pages, page, kvh, device=device))


def test_whole_steps_together(device):
    """Prompts in chunks, then drafted trees of which a path is kept, on a stream of the test's own: every layer's
    attention equals the oracle's on what the cache holds, and at the end all pages are free again."""
    batch, pps, page, kvh, r, dim, layers = 3, 12, 16, 2, 4, 128, 2
    s = _step_state(device, batch, pps, page, kvh, dim, layers)
    rng = np.random.default_rng(21)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    # (new tokens, tree?, accepted): two chunks, then trees
    steps = [([40, 17, 0], False, None), ([33, 1, 50], False, None), ([9, 12, 7], True, [3, 0, 5]),
             ([1, 1, 1], False, None), ([12, 0, 12], True, [4, 0, 1])]
    with torch.cuda.stream(stream):
        for counts, tree, accepted in steps:
            rows, most = sum(counts) + 2, max(counts)
            parents = np.concatenate([rng.integers(-1, np.maximum(np.arange(c), 1)) if c else [] for c in counts]
                                     + [[-1, -1]]).astype(np.int32)
            plan = plan_pages(s["table"], s["lengths"], _dev(np.array(counts, np.int32), device), s["free"], s["count"],
                              page_size=page, rows=rows, parents=_dev(parents, device) if tree else None,
                              max_count=most if tree else None)
            assert plan.missing.item() == 0
            q = bf16_round(rng.standard_normal((rows, kvh * r, dim)).astype(np.float32))
            table, lengths = s["table"].cpu().numpy(), s["lengths"].cpu().numpy()
            starts = plan.starts.cpu().numpy()
            sees = None
            if tree:
                sees = oracle.plan(table, lengths, counts, [0], 0, page, rows, parents, most)[3]
            for n in range(layers):
                x = torch.randn(2, rows, kvh * dim, device=device).to(torch.bfloat16)
                (k, v), (ks, vs) = s["codes"][n], s["scales"][n]
                write_tokens(k, ks, v, vs, x[0], x[1], plan.slots, kv_heads=kvh, head_dim=dim)
                out = paged_tree_attention(_dev(q, device, torch.bfloat16), k, ks, v, vs, s["table"], s["lengths"],
                                           plan.starts, plan.masks, page_size=page, kv_heads=kvh, max_count=most)
                kk, vv = (t.view(-1, page, kvh, dim).cpu().numpy() for t in (k, v))
                case = (kk, ks.cpu().numpy(), vv, vs.cpu().numpy(), table, lengths, starts, page, kvh, q, most)
                _check(out.float().cpu().numpy(), case, sees)
            if accepted is None:
                s["lengths"] += _dev(np.array(counts, np.int32), device)
            else:
                path = np.zeros((batch, 6), np.int32)
                for b, a in enumerate(accepted):
                    path[b, :a] = np.sort(rng.permutation(counts[b])[:a]) if a else 0
                want = [oracle.keep(c, table, lengths, path, accepted, page)
                        for c in s["codes"].flatten(0, 1).cpu().numpy()]
                taken = _dev(np.array(accepted, np.int32), device)
                keep_accepted([(s["codes"], s["scales"])], s["table"], s["lengths"], _dev(path, device), taken,
                              page_size=page)
                np.testing.assert_array_equal(s["codes"].flatten(0, 1).cpu().numpy(), np.stack(want))
                s["lengths"] += taken
            release_pages(s["table"], s["lengths"], s["free"], s["count"], page_size=page)
            held = -(-s["lengths"].cpu().numpy() // page)
            assert ((s["table"].cpu().numpy() >= 0).sum(1) == held).all()
            assert s["count"].item() == batch * pps - held.sum()
        s["lengths"].zero_()
        release_pages(s["table"], s["lengths"], s["free"], s["count"], page_size=page)
    stream.synchronize()
    assert s["count"].item() == batch * pps and sorted(s["free"].tolist()) == list(range(batch * pps))


def test_captured_step_replays(device):
    """A padded step captured once and replayed with other lengths, counts and trees in the same buffers, eager work
    in between; the replays share their workspace with another captured step."""
    batch, pps, page, kvh, r, dim = 4, 8, 64, 2, 4, 128
    rows, most = 40, 16
    s = _step_state(device, batch, pps, page, kvh, dim, 1)
    rng = np.random.default_rng(22)
    counts = torch.zeros(batch, dtype=torch.int32, device=device)
    parents = torch.full((rows,), -1, dtype=torch.int32, device=device)
    x = torch.zeros(2, rows, kvh * dim, dtype=torch.bfloat16, device=device)
    q = torch.zeros(rows, kvh * r, dim, dtype=torch.bfloat16, device=device)
    path = torch.zeros(batch, 4, dtype=torch.int32, device=device)
    taken = torch.zeros(batch, dtype=torch.int32, device=device)
    (k, v), (ks, vs) = s["codes"][0], s["scales"][0]
    args = dict(page_size=page, rows=rows, parents=parents, max_count=most)
    plan = plan_pages(s["table"], s["lengths"], counts, s["free"], s["count"], **args)
    outs = [torch.zeros_like(q) for _ in range(2)]
    size = 1 << 26
    workspace = torch.empty(size, dtype=torch.uint8, device=device)

    def step(out):
        plan_pages(s["table"], s["lengths"], counts, s["free"], s["count"], **args, out=plan)
        write_tokens(k, ks, v, vs, x[0], x[1], plan.slots, kv_heads=kvh, head_dim=dim)
        paged_tree_attention(q, k, ks, v, vs, s["table"], s["lengths"], plan.starts, plan.masks, page_size=page,
                             kv_heads=kvh, max_count=most, out=out, workspace=workspace)

    def finish():
        keep_accepted([(s["codes"], s["scales"])], s["table"], s["lengths"], path, taken, page_size=page)
        s["lengths"].add_(taken)
        release_pages(s["table"], s["lengths"], s["free"], s["count"], page_size=page)

    step(outs[0])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(3)]
    for g, work in zip(graphs, (lambda: step(outs[0]), lambda: step(outs[1]), finish)):
        with torch.cuda.graph(g):
            work()
    for turn in range(5):
        c = rng.integers(0, 11, batch).astype(np.int32)
        counts.copy_(_dev(c, device))
        parents.copy_(_dev(rng.integers(-1, 6, rows).astype(np.int32), device))
        x.normal_()
        qv = bf16_round(rng.standard_normal((rows, kvh * r, dim)).astype(np.float32))
        q.copy_(_dev(qv, device))
        for o in outs:
            o.fill_(5)
        a = np.minimum(c, rng.integers(0, 5, batch)).astype(np.int32)
        taken.copy_(_dev(a, device))
        path.copy_(_dev(np.stack([np.sort(rng.permutation(max(4, n))[:4]) for n in c]).astype(np.int32), device))
        lengths = s["lengths"].cpu().numpy()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        table, starts = s["table"].cpu().numpy(), plan.starts.cpu().numpy()
        assert starts[-1] == c.sum()
        sees = oracle.plan(table, lengths, c, [0], 0, page, rows, parents.cpu().numpy(), most)[3]
        case = (k.view(-1, page, kvh, dim).cpu().numpy(), ks.cpu().numpy(), v.view(-1, page, kvh, dim).cpu().numpy(),
                vs.cpu().numpy(), table, lengths, starts, page, kvh, qv, most)
        got = outs[0].float().cpu().numpy()
        live = _check(got, case, sees)
        assert (got[~live] == 5).all()
        assert torch.equal(outs[0], outs[1])
        want = oracle.keep(k.cpu().numpy(), table, lengths, path.cpu().numpy(), a, page)
        graphs[2].replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(k.cpu().numpy(), want)
        np.testing.assert_array_equal(s["lengths"].cpu().numpy(), lengths + a)
