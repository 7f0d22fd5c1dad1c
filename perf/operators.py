"""The operators of a step that takes several new tokens per sequence, and the calls they are measured on.

A serving step over the paged INT8 cache takes a ragged batch of new tokens: a
chunk of each prompt, or a tree of drafted tokens of each sequence that the
model verifies in one pass. Four kinds of call:

* ``plan``   pages and slots for the new tokens, on the GPU (``plan_pages``),
             and the pages given back when all of them were rejected
             (``release_pages``);
* ``write``  the new tokens' keys and values, quantised into their slots
             (``write_tokens``), and the sequences' values read back;
* ``attn``   attention of the new tokens over the cache and over each other
             (``paged_tree_attention``);
* ``keep``   the accepted tokens of each tree moved to the front of its new
             places, in the caches of all layers (``keep_accepted``).

Sequence b has ``lengths[b]`` tokens in the cache and ``counts[b]`` new ones;
new token j lies at position ``lengths[b] + j``. A tree is ``parents``: the
index of the token that a new token follows, -1 for the last cached one. A new
token sees the cached tokens, its ancestors and itself.

``run`` is the plain form, in elementary torch operations, unless ``own`` is set.
"""

import math
import sys
from pathlib import Path

import torch

own = False

MOST_TREE = 256  # new tokens of a sequence that masks tell apart


def listed():
    return [
        # pages and slots of a decode step: 8 sequences, drafted trees of up to 16 tokens
        dict(name="plan_step", kind="plan", batch=8, tokens=16, context=4096, page=64, tree=True, spare=5),
        # a scheduler's step over many prompts at once
        dict(name="plan_prompts", kind="plan", batch=256, tokens=4096, context=0, page=64, tree=False, spare=77),
        # the keys and values of 8 sequences' drafted trees
        dict(name="write_step", kind="write", batch=8, tokens=8, context=100, page=64, kv_heads=4, dim=128,
             values="bf16", scales="f32"),
        # those of long prompts, odd lengths
        dict(name="write_prompts", kind="write", batch=6, tokens=4093, context=200, page=256, kv_heads=8, dim=128,
             values="bf16", scales="f32"),
        # one sequence, one token, a short context: latency
        dict(name="attn_one", kind="attn", batch=1, tokens=1, context=1000, page=64, kv_heads=4, heads_per_kv=8,
             dim=128, tree=False, scales="f32", spare=0),
        # one token of each of 8 sequences with ragged contexts of up to 32 K tokens
        dict(name="attn_tokens", kind="attn", batch=8, tokens=1, context=32768, page=256, kv_heads=4, heads_per_kv=8,
             dim=128, tree=False, scales="f32", spare=0),
        # small heads, small pages that end inside every tile, a padded batch, BF16 scales
        dict(name="attn_small_heads", kind="attn", batch=24, tokens=5, context=3000, page=16, kv_heads=2,
             heads_per_kv=7, dim=64, tree=True, scales="bf16", spare=9),
        # drafted trees of up to 16 tokens over long contexts
        dict(name="attn_tree", kind="attn", batch=8, tokens=16, context=32768, page=256, kv_heads=4, heads_per_kv=8,
             dim=128, tree=True, scales="f32", spare=0),
        # the widest trees in use
        dict(name="attn_wide_tree", kind="attn", batch=8, tokens=64, context=32768, page=64, kv_heads=4,
             heads_per_kv=8, dim=128, tree=True, scales="f32", spare=3),
        # a chunk of two prompts over what is cached of them, wide heads
        dict(name="attn_chunk", kind="attn", batch=2, tokens=1024, context=8192, page=128, kv_heads=2,
             heads_per_kv=6, dim=256, tree=False, scales="f32", spare=0),
        # one layer's cache after a small step
        dict(name="keep_step", kind="keep", batch=8, tokens=16, accepted=4, context=512, page=64, layers=1,
             kv_heads=4, dim=128),
        # the caches of many layers after a step of many sequences
        dict(name="keep_layers", kind="keep", batch=48, tokens=64, accepted=12, context=256, page=64, layers=24,
             kv_heads=4, dim=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(("plan", "write", "attn", "keep"), (2, 2, 6, 2))[0]
    page = rng.choice((16, 64, 128, 256))
    if kind == "plan":
        tree = rng.random() < 0.5
        batch = _log(rng, 1, 256)
        return dict(kind=kind, batch=batch, tokens=_log(rng, 1, MOST_TREE if tree else 4096),
                    context=_log(rng, 1, 8192), page=page, tree=tree, spare=rng.choice((0, rng.randint(1, 100))))
    kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, 256))
    if kind == "write":
        rows = _log(rng, 1, 16384 * 1024 // (kv_heads * dim))
        batch = _log(rng, 1, min(64, rows))
        return dict(kind=kind, batch=batch, tokens=max(1, rows // batch), context=_log(rng, 1, 256), page=page,
                    kv_heads=kv_heads, dim=dim, values=rng.choice(("bf16", "bf16", "f32")),
                    scales=rng.choice(("f32", "bf16")))
    if kind == "keep":
        batch, layers = _log(rng, 1, 48), _log(rng, 1, 24)
        return dict(kind=kind, batch=batch, tokens=64, accepted=_log(rng, 1, 12), context=_log(rng, 1, 256),
                    page=rng.choice((16, 64)), layers=layers, kv_heads=rng.choice((1, 2, 4)), dim=rng.choice((64, 128)))
    heads_per_kv = rng.choice((1, 4, 6, 7, 8, 16))
    context = _log(rng, 16, 32768)
    tree = rng.random() < 0.6
    tokens = _log(rng, 1, 128 if tree else 1024)
    batch = _log(rng, 1, 32)
    # no more cached tokens and no more products than the largest listed cases
    while batch > 1 and batch * context * kv_heads * dim > 8 * 32768 * 512:
        batch //= 2
    while batch * context * kv_heads * dim > 8 * 32768 * 512:
        context //= 2
    while batch * tokens * (context + tokens) * kv_heads * heads_per_kv * dim > 8 * 64 * 32768 * 4096:
        tokens = max(1, tokens // 2)
    return dict(kind=kind, batch=batch, tokens=tokens, context=context, page=page, kv_heads=kv_heads,
                heads_per_kv=heads_per_kv, dim=dim, tree=tree, scales=rng.choice(("f32", "f32", "bf16")),
                spare=rng.choice((0, 0, rng.randint(1, 40))))


# ---------------------------------------------------------------------------
# Inputs. Lengths and counts go by the case, so that its work is known; all
# values, page orders and trees go by the seed.
# ---------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of each sequence: a quarter to all of ``context``."""
    return [math.ceil(case["context"] * (0.25 + 0.75 * (0.618034 * (b + 1) % 1.0))) for b in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence: ``tokens``, every fourth with fewer (a sequence that waits has none)."""
    n = case["tokens"]
    if n == 1:
        return [1] * case["batch"]
    return [int(n * (0.754878 * (b + 1) % 1.0)) if b % 4 == 3 else n for b in range(case["batch"])]


def _starts(counts):
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    return starts


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _table(gen, case, lengths, counts):
    """A random page table that holds every sequence's cached and new tokens, and the pages of the pool."""
    batch, page = case["batch"], case["page"]
    per_seq = -(-(case["context"] + case["tokens"]) // page)
    pages = batch * per_seq
    return torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(batch, per_seq), pages


def _cache(gen, lead, kv_heads, dim, scales):
    """Codes and scales of N(0, 1) keys or values, one scale per token and head."""
    codes = (_randn(gen, *lead, kv_heads * dim) * 45).round_().clamp_(-127, 127).to(torch.int8)
    sc = torch.rand(*lead, kv_heads, generator=gen, device="cuda") * 0.008 + 0.018
    return codes, sc.to(_dtype(scales))


def _parents(gen, starts, rows):
    """A random tree for each sequence: token j follows one of the tokens -1 .. j-1."""
    _, j, live = _places(_ints(starts), rows)
    follow = (torch.rand(rows, generator=gen, device="cuda") * (j + 1)).floor().to(torch.int32) - 1
    return torch.where(live, torch.minimum(follow, (j - 1).int()), -1).int()


def prepare(case, seed):
    gen = _generator(seed)
    lengths, counts = _lengths(case), _counts(case)
    starts = _starts(counts)
    rows = max(1, starts[-1] + case.get("spare", 0))
    state = dict(kind=case["kind"], page=case["page"], rows=rows, most=case["tokens"],
                 lengths=_ints(lengths), counts=_ints(counts), starts=_ints(starts))
    table, pages = _table(gen, case, lengths, counts)
    if case["kind"] == "plan":
        # pages of the cached tokens are mapped; the others lie on the free stack
        held = (state["lengths"] + case["page"] - 1) // case["page"]
        index = torch.arange(table.shape[1], device="cuda")
        mapped = index < held[:, None]
        free = torch.cat((table[~mapped], torch.full((7,), -5, dtype=torch.int32, device="cuda")))
        state.update(table=torch.where(mapped, table, -1).contiguous(), free=free,
                     free_count=_ints([int((~mapped).sum())]),
                     parents=_parents(gen, starts, rows) if case["tree"] else None)
        return state
    kvh, dim = case["kv_heads"], case["dim"]
    state.update(table=table, kv_heads=kvh, dim=dim)
    if case["kind"] == "write":
        state["codes"], state["scales"] = _cache(gen, (2, pages, case["page"]), kvh, dim, case["scales"])
        # the key and value columns of a fused projection's output
        fused = _randn(gen, rows, 3, kvh, dim).to(_dtype(case["values"]))
        state["key"], state["value"] = fused[:, 1], fused[:, 2]
        b, j, live = _places(state["starts"], rows)
        where = torch.where(live, state["lengths"][b] + j, 0)
        slots = table[b, where // case["page"]].long() * case["page"] + where % case["page"]
        state["slots"] = torch.where(live, slots, -1)
        return state
    if case["kind"] == "keep":
        layers, most = case["layers"], case["accepted"]
        state["codes"], state["scales"] = _cache(gen, (layers, 2, pages, case["page"]), kvh, dim, "f32")
        # an accepted path: some of the tree's first tokens as they lie, the rest from deeper levels
        kept = torch.randint(0, most + 1, (case["batch"], 1), generator=gen, device="cuda")
        deep = torch.rand(case["batch"], case["tokens"], generator=gen, device="cuda")
        deep[:, :most] = 2.0  # the first places themselves are left out
        deep = deep.argsort(1)[:, :most].sort(1).values
        i = torch.arange(most, device="cuda")
        state["path"] = torch.where(i < kept, i, deep).int()
        state["accepted"] = torch.randint(0, most + 1, (case["batch"],), generator=gen, device="cuda").int()
        return state
    for name in ("k", "v"):
        state[name], state[name + "_scales"] = _cache(gen, (pages, case["page"]), kvh, dim, case["scales"])
    state["q"] = (_randn(gen, rows, kvh * case["heads_per_kv"], dim) * 2).to(torch.bfloat16)
    state["out"] = torch.zeros_like(state["q"])
    state["masks"] = None
    if case["tree"]:
        words = -(-min(case["tokens"], MOST_TREE) // 64)
        b, j, live = _places(state["starts"], rows)
        state["masks"], _ = _tree(_parents(gen, starts, rows), state["starts"], b, j, live, words)
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _places(starts, rows):
    """Sequence and place in it of each row, and whether it belongs to one."""
    r = torch.arange(rows, device=starts.device)
    b = torch.searchsorted(starts[1:].contiguous(), r.int(), right=True).clamp_(max=starts.numel() - 2)
    return b, r - starts[b], r < starts[-1]


def _tree(parents, starts, b, j, live, words):
    """(masks, depths): bit jj of row i's words says that new token jj is an ancestor of row i's token or itself."""
    rows = parents.numel()
    at = torch.arange(64 * words, device=parents.device)
    sees = (at == j[:, None]) & live[:, None]
    has = (parents >= 0) & (parents < j) & live
    up = torch.where(has, starts[b] + parents, rows).long()
    for _ in range(max(1, (64 * words - 1).bit_length())):  # the ancestors within 1, 2, 4, ... levels
        more = torch.cat((sees, torch.zeros_like(sees[:1])))
        sees = sees | more[up]
        up = torch.cat((up, up.new_full((1,), rows)))[up]
    bits = sees.view(rows, words, 64).long() << torch.arange(64, device=parents.device)
    return bits.sum(-1), (sees.sum(-1) - 1).clamp_(min=0)


def _plan(s):
    page, table, lengths = s["page"], s["table"], s["lengths"].long()
    counts = s["counts"].long()
    starts = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    index = torch.arange(table.shape[1], device=table.device)
    first, end = lengths // page, (lengths + counts + page - 1) // page
    need = (index >= first[:, None]) & (index < end[:, None]) & (table < 0)
    rank = need.flatten().cumsum(0).view_as(need) - 1
    have = s["free_count"].long()
    got = need & (rank < have)
    table.copy_(torch.where(got, s["free"][(have - 1 - rank).clamp_(0, s["free"].numel() - 1)], table))
    s["free_count"].sub_(got.sum().int())
    b, j, live = _places(starts, s["rows"])
    where = lengths[b] + j
    live_at = live & (where < table.shape[1] * page)
    entry = table[b, (where // page).clamp_(max=table.shape[1] - 1)].long()
    slots = torch.where(live_at & (entry >= 0), entry * page + where % page, -1)
    missing = (live & (slots < 0)).sum().int().view(1)
    masks, depth = None, j
    if s["parents"] is not None:
        masks, depth = _tree(s["parents"], starts, b, j, live, -(-s["most"] // 64))
    positions = torch.where(live, lengths[b] + depth, 0).int()
    return starts.int(), slots, positions, masks, missing


def _release(s):
    page, table = s["page"], s["table"]
    index = torch.arange(table.shape[1], device=table.device)
    back = (index >= ((s["lengths"] + page - 1) // page)[:, None]) & (table >= 0)
    total = back.sum()
    rank = back.flatten().cumsum(0).view_as(back)
    have = s["free_count"].long()
    # a place past the end for the entries that stay
    to = torch.where(back, have + total - rank, s["free"].numel())
    stack = torch.cat((s["free"], s["free"].new_zeros(1)))
    s["free"].copy_(stack.scatter(0, to.flatten(), table.flatten())[:-1])
    table.masked_fill_(back, -1)
    s["free_count"].add_(total.int())


def _quantized(x, scale_dtype):
    """Codes and scales of [..., D] values, one scale each: the stored scale divides."""
    x = x.float()
    scale = (x.abs().amax(-1, keepdim=True) / 127).to(scale_dtype)
    divisor = torch.where(scale == 0, 1.0, scale.float())
    return (x / divisor).round().clamp(-127, 127).to(torch.int8), scale.squeeze(-1)


def _write(s):
    slots = s["slots"]
    # rows without a slot go to a place that is cut off again
    codes, scales = s["codes"].flatten(1, 2), s["scales"].flatten(1, 2)
    new, sc = _quantized(torch.stack((s["key"], s["value"])), scales.dtype)
    to = torch.where((slots >= 0) & (slots < codes.shape[1]), slots, codes.shape[1])
    codes.copy_(torch.cat((codes, codes[:, :1]), 1).index_copy(1, to, new.flatten(2))[:, :-1])
    scales.copy_(torch.cat((scales, scales[:, :1]), 1).index_copy(1, to, sc)[:, :-1])


def _values(s):
    """The values that the sequences' codes stand for, [2, batch, tokens, heads, D]."""
    pages = s["table"].long()
    codes = s["codes"][:, pages].flatten(2, 3).unflatten(-1, (s["kv_heads"], s["dim"]))
    return (codes * s["scales"][:, pages].flatten(2, 3).float().unsqueeze(-1)).to(torch.bfloat16).unbind(0)


def _attend(s):
    starts, most, page, kvh, dim = s["starts"].long(), s["most"], s["page"], s["kv_heads"], s["dim"]
    table, lengths, rows = s["table"].long(), s["lengths"].long(), s["rows"]
    batch, size = table.shape[0], table.shape[1] * page
    row = starts[:-1, None] + torch.arange(most, device=table.device)
    live = row < starts[1:, None]
    pick = torch.where(live, row, 0)
    q = s["q"][pick].float().view(batch, most, kvh, -1, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    token = torch.arange(size, device=table.device)
    slot = table[:, token // page] * page + token % page

    def cached(name):
        codes = s[name].view(-1, kvh, dim)[slot]
        scales = s[name + "_scales"].view(-1, kvh)[slot].float()
        return (codes.float() * scales.unsqueeze(-1)).transpose(1, 2).contiguous()

    scores = torch.matmul(q, cached("k").transpose(2, 3).contiguous()) / math.sqrt(dim)
    new = token - lengths[:, None]  # [batch, size]: which new token, below zero for the cached ones
    if s["masks"] is None:
        sees = new[:, None] <= torch.arange(most, device=table.device)[:, None]
    else:
        words = s["masks"].shape[1]
        bits = s["masks"][pick]
        at = new.clamp(0, 64 * words - 1)[:, None].expand(batch, most, size)
        sees = (bits.gather(2, at // 64) >> (at % 64)) & 1
        sees = (sees > 0) | (new[:, None] < 0)
    sees = sees & (new[:, None] < (starts[1:] - starts[:-1])[:, None, None])
    sees = sees[:, None, :, None].expand(-1, 1, -1, q.shape[2] // most, -1).flatten(2, 3)
    scores = scores.masked_fill_(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    prob = torch.exp(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = prob.sum(-1, keepdim=True)
    out = torch.matmul(prob, cached("v")) / torch.where(total == 0, 1.0, total)
    out = out.unflatten(2, (most, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s["out"][row[live]] = out[live].to(torch.bfloat16)
    return s["out"]


def _keep(s):
    table, page = s["table"].long(), s["page"]
    most = s["path"].shape[1]
    i = torch.arange(most, device=table.device)
    on = i < s["accepted"][:, None]
    source = s["lengths"][:, None].long() + s["path"]
    target = s["lengths"][:, None].long() + i

    def slot(t):
        return torch.gather(table, 1, t // page) * page + t % page

    source, target = slot(source)[on], slot(target)[on]
    for held in (s["codes"], s["scales"]):
        flat = held.flatten(2, 3)
        flat.index_copy_(2, target, flat.index_select(2, source))


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "plan":
        plan = _plan(s)
        _release(s)
        return dict(plan=plan, table=s["table"], free=s["free"], free_count=s["free_count"])
    if s["kind"] == "write":
        _write(s)
        return _values(s)
    if s["kind"] == "attn":
        return _attend(s)
    _keep(s)
    return dict(codes=s["codes"], scales=s["scales"])  # moved, not computed


def _run_own(s):
    package = str(Path(__file__).resolve().parents[1] / "data-synth-tpu_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import q6moe

    if s["kind"] == "plan":
        plan = q6moe.plan_pages(s["table"], s["lengths"], s["counts"], s["free"], s["free_count"],
                                page_size=s["page"], rows=s["rows"], parents=s["parents"],
                                max_count=s["most"])
        q6moe.release_pages(s["table"], s["lengths"], s["free"], s["free_count"], page_size=s["page"])
        return dict(plan=tuple(plan), table=s["table"], free=s["free"], free_count=s["free_count"])
    if s["kind"] == "write":
        (k, v), (ks, vs) = s["codes"], s["scales"]
        q6moe.write_tokens(k, ks, v, vs, s["key"], s["value"], s["slots"], kv_heads=s["kv_heads"],
                           head_dim=s["dim"])
        return [q6moe.read_paged(pool, scales, s["table"], page_size=s["page"], kv_heads=s["kv_heads"],
                                 head_dim=s["dim"]) for pool, scales in ((k, ks), (v, vs))]
    if s["kind"] == "attn":
        return q6moe.paged_tree_attention(s["q"], s["k"], s["k_scales"], s["v"], s["v_scales"], s["table"],
                                          s["lengths"], s["starts"], s["masks"], page_size=s["page"],
                                          kv_heads=s["kv_heads"], max_count=s["most"], out=s["out"])
    q6moe.keep_accepted([(s["codes"], s["scales"])], s["table"], s["lengths"], s["path"], s["accepted"], page_size=s["page"])
    return dict(codes=s["codes"], scales=s["scales"])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    lengths, counts, page = _lengths(case), _counts(case), case["page"]
    batch, rows = case["batch"], sum(counts)
    pages = sum(-(-(n + c) // page) - n // page for n, c in zip(lengths, counts))
    if case["kind"] == "plan":
        words = -(-case["tokens"] // 64) if case["tree"] else 0
        out = (rows + case["spare"]) * (8 + 4 + 8 * words) + 4 * (batch + 1)
        # lengths, counts and parents; each page leaves the stack for the table and goes back
        return dict(bytes=8 * batch + (4 * rows if case["tree"] else 0) + 16 * pages + out, flops=0)
    width = case["kv_heads"] * case["dim"]
    scale = 4 * case["kv_heads"] if case.get("scales", "f32") == "f32" else 2 * case["kv_heads"]
    if case["kind"] == "write":
        size = 2 if case["values"] == "bf16" else 4
        held = batch * -(-(case["context"] + case["tokens"]) // page) * page
        # the new tokens read and written, then the codes read and their values written
        return dict(bytes=2 * rows * (width * (size + 1) + scale) + 8 * rows + 2 * held * (3 * width + scale), flops=0)
    if case["kind"] == "keep":
        # on average half of the longest path is accepted, and half of that lies where it belongs already
        moved = batch * case["accepted"] / 4 * case["layers"] * 2
        return dict(bytes=2 * moved * (width + scale) + batch * (4 * case["accepted"] + 8), flops=0)
    heads = case["kv_heads"] * case["heads_per_kv"]
    cached = sum(n + c for n, c in zip(lengths, counts) if c)
    # every (row, key) pair that is seen: a tree's depth is about the logarithm of its size
    pairs = sum(c * n + (c * (c + 1) // 2 if not case["tree"] else c * max(1, round(math.log(c + 1))))
                for n, c in zip(lengths, counts) if c)
    return dict(bytes=2 * cached * (width + scale) + 4 * rows * heads * case["dim"] + 4 * (cached // page + batch),
                flops=4 * pairs * heads * case["dim"])


# ---------------------------------------------------------------------------
# The definitions, in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------
def _exact_plan(s):
    page, rows = s["page"], s["rows"]
    table, free = s["table"].tolist(), s["free"].tolist()
    lengths, counts, have = s["lengths"].tolist(), s["counts"].tolist(), int(s["free_count"])
    parents = None if s["parents"] is None else s["parents"].tolist()
    words = -(-s["most"] // 64)
    starts, slots, positions, masks, missing = [0], [], [], [], 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        for e in range(n // page, min(len(table[b]), -(-(n + c) // page))):
            if table[b][e] < 0 and have > 0:
                have -= 1
                table[b][e] = free[have]
        first, seen, depth = starts[-1], [], []
        for j in range(c):
            e = (n + j) // page
            ok = e < len(table[b]) and table[b][e] >= 0
            slots.append(table[b][e] * page + (n + j) % page if ok else -1)
            missing += not ok
            if parents is None:
                positions.append(n + j)
                continue
            p = parents[first + j]
            seen.append((1 << j) | (seen[p] if 0 <= p < j else 0))
            depth.append(depth[p] + 1 if 0 <= p < j else 0)
            positions.append(n + depth[j])
            masks.append([(seen[j] >> (64 * w)) & (2**64 - 1) for w in range(words)])
        starts.append(first + c)
    behind = rows - len(slots)
    slots += [-1] * behind
    positions += [0] * behind
    masks += [[0] * words] * behind
    signed = [[m - 2**64 if m >= 2**63 else m for m in r] for r in masks]
    plan = (torch.tensor(starts, dtype=torch.int32), torch.tensor(slots, dtype=torch.int64),
            torch.tensor(positions, dtype=torch.int32),
            None if parents is None else torch.tensor(signed, dtype=torch.int64),
            torch.tensor([missing], dtype=torch.int32))
    # everything that the plan took goes back to where it was
    return dict(plan=plan, table=s["table"], free=s["free"], free_count=s["free_count"])


def _exact_pool(s):
    codes, scales = s["codes"].double(), s["scales"].double()
    return (codes.unflatten(-1, (s["kv_heads"], s["dim"])) * scales[..., None])


def _exact_write(s):
    values = _exact_pool(s)
    out, stored = values.flatten(1, 2), s["scales"].dtype
    live = s["slots"] >= 0
    for n, x in enumerate((s["key"], s["value"])):
        x = x.double()[live]
        # scale and quotient are FP32 numbers by definition: rounded from 64 bits
        scale = (x.abs().amax(-1, keepdim=True) / 127).float().to(stored).double()
        ratio = (x / torch.where(scale == 0, torch.ones_like(scale), scale)).float().double()
        out[n, s["slots"][live]] = torch.clamp(torch.round(ratio), -127, 127) * scale
    return [v[s["table"].long()].flatten(1, 2) for v in out.view(values.shape)]


def _exact_attn(s):
    kvh, dim, page = s["kv_heads"], s["dim"], s["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lengths):
        first, end = starts[b], starts[b + 1]
        if first == end:
            continue
        total = n + end - first
        pages = s["table"][b, : -(-total // page)].long()
        allowed = torch.ones(end - first, total, dtype=torch.bool, device=out.device)
        if s["masks"] is None:
            allowed[:, n:] = torch.ones(end - first, end - first, dtype=torch.bool, device=out.device).tril()
        else:
            for jj in range(end - first):
                allowed[:, n + jj] = (s["masks"][first:end, jj // 64] >> (jj % 64)) & 1 == 1
        for h in range(kvh):
            k, v = (s[name][pages].reshape(-1, kvh, dim)[:total, h].double()
                    * s[name + "_scales"][pages].reshape(-1, kvh)[:total, h, None].double() for name in ("k", "v"))
            per = s["q"].shape[1] // kvh
            for g in range(h * per, (h + 1) * per):
                score = s["q"][first:end, g].double() @ k.T / dim**0.5
                prob = torch.softmax(score.masked_fill(~allowed, -math.inf), -1)
                out[first:end, g] = torch.where(allowed.any(-1, keepdim=True), prob @ v, 0.0)
    return out


def _exact_keep(s):
    lengths, page, table = s["lengths"].tolist(), s["page"], s["table"].tolist()
    path, accepted = s["path"].tolist(), s["accepted"].tolist()
    after = {}
    for name in ("codes", "scales"):
        after[name] = s[name].clone()
        old, new = s[name].flatten(2, 3), after[name].flatten(2, 3)
        for b, n in enumerate(lengths):
            for i in range(accepted[b]):
                to, at = (table[b][t // page] * page + t % page for t in (n + i, n + path[b][i]))
                new[:, :, to] = old[:, :, at]
    return after


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attn" and work(case)["flops"] > 4e11:
        return None
    return {"plan": _exact_plan, "write": _exact_write, "attn": _exact_attn, "keep": _exact_keep}[case["kind"]](s)
