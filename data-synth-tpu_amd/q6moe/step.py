"""A step with several new tokens per sequence over the paged INT8 cache: chunks
of prompts, or trees of drafted tokens that the model verifies in one pass.

The reference's steps take one token per sequence (kaggle/qwen38_tpu/
attention_cache.py:128-172), so these operators have no counterpart there; they
stand beside ``write_paged``, ``read_paged`` and ``paged_decode_attention`` and
work on the same pools, scales and page tables. A step is

    plan = plan_pages(page_table, lengths, counts, free_pages, free_count, ...)
    for each layer:
        write_tokens(k_pool, k_scales, v_pool, v_scales, key, value, plan.slots, ...)
        out = paged_tree_attention(q, k_pool, k_scales, v_pool, v_scales, page_table,
                                   lengths, plan.starts, plan.masks, ...)
    keep_accepted(caches, page_table, lengths, path, accepted, ...)
    lengths += accepted
    release_pages(page_table, lengths, free_pages, free_count, ...)

Sequence b has ``lengths[b]`` cached tokens; its new ones are rows ``starts[b]``
to ``starts[b + 1] - 1`` of the ragged batch and lie at positions ``lengths[b] +
j``. All state stays on the GPU: no call waits for it, and every call can be
captured into a graph (pass the buffers of ``out`` and ``workspace``).
"""

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _launch, _lib
from .attention_cache import _dtype_code, _int32

MAX_TREE = 256  # new tokens of a sequence that masks tell apart


class PagePlan(NamedTuple):
    """What ``plan_pages`` found for a batch: see there."""

    starts: torch.Tensor            # int32 [batch + 1]
    slots: torch.Tensor             # int64 [rows]
    positions: torch.Tensor         # int32 [rows]
    masks: Optional[torch.Tensor]   # int64 [rows, words] with parents
    missing: torch.Tensor           # int32 [1]


def _on(device, name, t, dtype, shape=None):
    """``t`` where it is a contiguous tensor of this type (and shape) on ``device``."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or not t.is_contiguous()
            or (shape is not None and tuple(t.shape) != shape)):
        want = "" if shape is None else f" {list(shape)}"
        raise ValueError(f"{name} must be a contiguous {dtype}{want} tensor on {device}")
    return t


def _gpu(name, t):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor")
    return t.device


def _state(page_table, lengths, free_pages, free_count):
    device = _gpu("page_table", page_table)
    if page_table.ndim != 2 or not page_table.shape[0] or not page_table.shape[1]:
        raise ValueError("page_table must be [batch, pages_per_seq]")
    _on(device, "page_table", page_table, torch.int32)
    _on(device, "free_count", free_count, torch.int32, (1,))
    _on(device, "free_pages", free_pages, torch.int32)
    if free_pages.ndim != 1 or not free_pages.shape[0]:
        raise ValueError("free_pages must be [capacity]")
    lens = _int32(lengths, device)
    if lens.shape != (page_table.shape[0],):
        raise ValueError("lengths must be [batch]")
    return device, lens


def _positive(**named):
    for name, v in named.items():
        if type(v) is not int or v < 1:
            raise ValueError(f"{name} must be a positive integer")


def plan_pages(page_table, lengths, counts, free_pages, free_count, *, page_size, rows, parents=None, max_count=None,
               out=None):
    """Pages and slots for ``counts[b]`` new tokens of each sequence.

    ``page_table`` int32 [batch, pages_per_seq] (entries below 0 are unmapped)
    and ``free_count`` int32 [1] are updated in place: every unmapped entry under
    the new tokens takes the last page of the stack ``free_pages[:free_count]``
    (int32), in the order of sequence and page. A second call with the same
    arguments changes nothing.

    ``rows`` is the size of the ragged batch (tokens past it are dropped; rows
    behind the last sequence are padding). ``parents`` int32 [rows] makes each
    sequence's tokens a tree: the index, within the sequence, of the token that a
    row's token follows; -1 (and anything that is no earlier token) for the last
    cached one. ``max_count``, at most 256, then bounds a sequence's tokens.

    Returns ``PagePlan``: ``starts`` (running sum of the counts), ``slots`` (pool
    row of each new token, page * page_size + place; -1 for padding and for
    tokens without a page), ``positions`` (lengths[b] + j, for a tree lengths[b] +
    depth: what rotary embeddings take; 0 for padding), ``masks`` (with parents:
    int64 [rows, ceil(max_count / 64)], bit jj of a row's words set where new
    token jj is an ancestor or the token itself) and ``missing`` (how many new
    tokens got no slot, of those past ``max_count`` and ``rows`` at most (2**31 -
    1 - rows) // batch per sequence: check it before the step's results are used).
    ``out``: a plan whose buffers are written again.
    """
    device, lens = _state(page_table, lengths, free_pages, free_count)
    _positive(page_size=page_size, rows=rows)
    batch, pps = page_table.shape
    want = _int32(counts, device)
    if want.shape != (batch,):
        raise ValueError("counts must be [batch]")
    words = 0
    if parents is not None:
        if type(max_count) is not int or not 1 <= max_count <= MAX_TREE:
            raise ValueError(f"a tree needs max_count, from 1 to {MAX_TREE}")
        parents = _int32(parents, device)
        if parents.shape != (rows,):
            raise ValueError("parents must be [rows]")
        words = -(-max_count // 64)
    elif max_count is not None:
        _positive(max_count=max_count)
    if out is None:
        # one buffer for all of int32: an allocation takes 1.2 us, the split of one into four 1.6
        starts, positions, missing, work = torch.empty(
            2 * (batch + 1) + rows + 1, dtype=torch.int32, device=device).split_with_sizes(
                [batch + 1, rows, 1, batch + 1])
        out = PagePlan(starts, torch.empty(rows, dtype=torch.int64, device=device), positions,
                       torch.empty((rows, words), dtype=torch.int64, device=device) if words else None, missing)
    else:
        work = torch.empty(batch + 1, dtype=torch.int32, device=device)
        _on(device, "out.starts", out.starts, torch.int32, (batch + 1,))
        _on(device, "out.slots", out.slots, torch.int64, (rows,))
        _on(device, "out.positions", out.positions, torch.int32, (rows,))
        _on(device, "out.missing", out.missing, torch.int32, (1,))
        if words:
            _on(device, "out.masks", out.masks, torch.int64, (rows, words))
        elif out.masks is not None:
            raise ValueError("out.masks must be None without parents")
    # positionally, in the order of q6moe_kv_plan_args: a field assigned by name costs as much as a check
    a = _lib.PlanArgs(
        page_table.data_ptr(), lens.data_ptr(), want.data_ptr(), free_pages.data_ptr(), free_pages.shape[0],
        free_count.data_ptr(), parents.data_ptr() if words else None, batch, pps, page_size, rows,
        rows if max_count is None else max_count, out.starts.data_ptr(), out.slots.data_ptr(),
        out.positions.data_ptr(), out.masks.data_ptr() if words else None, out.missing.data_ptr(), work.data_ptr(),
        4 * (batch + 1))
    _launch.run("kv_plan", _lib.load().q6moe_kv_plan, device, ctypes.byref(a))
    return out


def release_pages(page_table, lengths, free_pages, free_count, *, page_size):
    """Unmaps every page past the cached tokens (page index ceil(lengths[b] /
    page_size) on; 0 for a sequence that has ended) and pushes it on the free
    stack, in the order that undoes ``plan_pages``. ``page_table``, ``free_pages``
    and ``free_count`` are updated in place. Pages that the stack has no room for
    stay mapped. Pages that several entries name are pushed once for each: keep
    shared pages out of what is released.
    """
    device, lens = _state(page_table, lengths, free_pages, free_count)
    _positive(page_size=page_size)
    batch, pps = page_table.shape
    work = torch.empty(batch + 1, dtype=torch.int32, device=device)
    _launch.run("kv_release", _lib.load().q6moe_kv_release, device, page_table.data_ptr(), lens.data_ptr(),
                free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), batch, pps, page_size,
                work.data_ptr(), 4 * (batch + 1))


def _rows_of(x, rows, kv_heads, head_dim, device, name):
    """x [rows, kv_heads * head_dim] or [rows, kv_heads, head_dim] with contiguous rows, and the stride between them."""
    if not isinstance(x, torch.Tensor) or x.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if tuple(x.shape) not in ((rows, kv_heads * head_dim), (rows, kv_heads, head_dim)):
        raise ValueError(f"{name} must be [rows, kv_heads * head_dim] or [rows, kv_heads, head_dim]")
    if x.stride(-1) != 1 or (x.ndim == 3 and x.stride(1) != head_dim):
        x = x.contiguous()
    return x, x.stride(0)


def _pool_rows(pool, scales, chans, groups, device, name):
    shape = pool.shape
    n = shape[0] * shape[1] if len(shape) > 2 else 0
    if pool.dtype is not torch.int8 or not n or pool.device != device or not pool.is_contiguous() or \
            pool.numel() != n * chans:
        raise ValueError(f"{name} pool must be contiguous int8 [pages, page_size, kv_heads * head_dim] on {device}")
    if scales.dtype not in (torch.bfloat16, torch.float32) or scales.device != device or \
            not scales.is_contiguous() or scales.numel() != n * groups:
        raise ValueError(f"{name} scales must be contiguous BF16 or FP32 [pages, page_size, {groups}] on {device}")
    return n


def write_tokens(k_pool, k_scales, v_pool, v_scales, key, value, slots, *, kv_heads, head_dim, group=None):
    """Keys and values of a ragged batch, quantised into their slots in one launch.

    ``key`` and ``value`` BF16 or FP32 [rows, kv_heads * head_dim] or [rows,
    kv_heads, head_dim]; their rows may lie apart (columns of a fused projection).
    ``slots`` int64 [rows] as ``plan_pages`` gives them; rows outside the pool (-1)
    are skipped, the others must be distinct. Pools int8 [pages, page_size, ...],
    scales [pages, page_size, kv_heads * head_dim / group] (group: head_dim by
    default; ``paged_tree_attention`` reads caches of one scale per head); K's and
    V's must not overlap. Codes and scales are those of ``write_paged`` bit for bit.
    """
    _positive(kv_heads=kv_heads, head_dim=head_dim)
    group = head_dim if group is None else group
    chans = kv_heads * head_dim
    if type(group) is not int or group < 1 or chans % group:
        raise ValueError("group must divide kv_heads * head_dim")
    device = _gpu("k_pool", k_pool)
    if not isinstance(slots, torch.Tensor) or slots.ndim != 1 or slots.device != device:
        raise ValueError(f"slots must be [rows] on {device}")
    if slots.dtype is not torch.int64:
        slots = slots.to(torch.int64)
    slots = slots.contiguous()
    rows = slots.shape[0]
    n = _pool_rows(k_pool, k_scales, chans, chans // group, device, "k")
    if _pool_rows(v_pool, v_scales, chans, chans // group, device, "v") != n or k_scales.dtype != v_scales.dtype:
        raise ValueError("the k and v pools must have the same size and scale type")
    if (abs(k_pool.data_ptr() - v_pool.data_ptr()) < n * chans
            or abs(k_scales.data_ptr() - v_scales.data_ptr()) < n * (chans // group) * k_scales.element_size()):
        raise ValueError("the k and v pools must not be the same memory, nor overlap")
    key, key_stride = _rows_of(key, rows, kv_heads, head_dim, device, "key")
    value, value_stride = _rows_of(value, rows, kv_heads, head_dim, device, "value")
    if key.dtype != value.dtype:
        raise ValueError("key and value must have the same type")
    if rows == 0:
        return
    a = _lib.KvWriteRowsArgs(
        key.data_ptr(), value.data_ptr(), key_stride, value_stride, _dtype_code(key.dtype), k_pool.data_ptr(),
        v_pool.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), _dtype_code(k_scales.dtype), slots.data_ptr(),
        rows, n, kv_heads, head_dim, group)
    _launch.run("kv_write_rows", _lib.load().q6moe_kv_write_rows, device, ctypes.byref(a))


@lru_cache(maxsize=256, typed=True)
def _tree_workspace_bytes(batch, rows, max_count, hq, kv_heads, head_dim, pps, page_size):
    return int(_lib.load().q6moe_tree_attn_workspace_size(batch, rows, max_count, hq, kv_heads, head_dim, pps,
                                                          page_size))


def paged_tree_attention(q, k_pool, k_scales, v_pool, v_scales, page_table, lengths, starts, masks=None, *, page_size,
                         kv_heads, max_count, workspace=None, out=None):
    """Attention of the new tokens over the cached ones and over each other.

    ``q`` BF16 [rows, Hq, D] with D 64, 128 or 256 (rows may lie apart); pools
    int8 [pages, page_size, kv_heads * D] and scales BF16 or FP32 [pages,
    page_size, kv_heads], which hold the new tokens' keys and values already
    (``write_tokens``); ``lengths`` the cached tokens WITHOUT the new ones;
    ``starts`` int32 [batch + 1]. Row j of a sequence sees every cached token and
    new token jj where bit jj of its row of ``masks`` (int64 [rows, words], as
    ``plan_pages`` gives them) is set; with ``masks=None``, jj <= j. ``max_count``
    bounds the new tokens of any one sequence (rows from it on are skipped; with
    masks at most 64 * words).

    Returns BF16 [rows, Hq, D]: softmax(q . k / sqrt(D)) . v with k and v the
    unrounded code * scale, rounded once. Scores and sums are FP32 (a row with a
    score past its range is NaN); a probability times its value scale has 11 bits
    where it is 2^-9 of the row's largest or more, else it is off by up to 2^-20
    of that. A page table far wider than the contexts can cost a fifth to a half
    more time (128 K tokens over 500 to 8000): kernels are chosen by its width.
    A row that sees nothing gives 0. Rows
    behind the last sequence, and of a sequence those from ``max_count`` on, are
    left as they were in ``out``; without ``out`` they are 0 (one launch more, for
    the fill). Unmapped pages read as zero keys and values.
    """
    device = _gpu("q", q)
    if q.dtype is not torch.bfloat16 or q.ndim != 3 or q.shape[2] not in (64, 128, 256):
        raise ValueError("q must be BF16 [rows, query_heads, head_dim] with head_dim 64, 128 or 256")
    _positive(page_size=page_size, kv_heads=kv_heads, max_count=max_count)
    rows, hq, dim = q.shape
    if not hq or hq % kv_heads:
        raise ValueError("query_heads must be a multiple of kv_heads")
    n = _pool_rows(k_pool, k_scales, kv_heads * dim, kv_heads, device, "k")
    if k_pool.shape[1] != page_size or v_pool.shape[:2] != k_pool.shape[:2] or \
            _pool_rows(v_pool, v_scales, kv_heads * dim, kv_heads, device, "v") != n or \
            k_scales.dtype != v_scales.dtype:
        raise ValueError("the pools must be [pages, page_size, kv_heads * head_dim], of the same size and scale type")
    table, lens, first = _int32(page_table, device), _int32(lengths, device), _int32(starts, device)
    shape = table.shape
    if len(shape) != 2 or 0 in shape or lens.shape != shape[:1] or first.shape != (shape[0] + 1,):
        raise ValueError("page_table must be [batch, pages_per_seq], lengths [batch] and starts [batch + 1]")
    batch, pps = shape
    words = 0
    if masks is not None:
        if not isinstance(masks, torch.Tensor) or masks.ndim != 2 or masks.shape[0] != rows or \
                not 1 <= masks.shape[1] <= MAX_TREE // 64:
            raise ValueError("masks must be [rows, words] with 1 to 4 words")
        masks = _on(device, "masks", masks, torch.int64)
        words = masks.shape[1]
        if max_count > 64 * words:
            raise ValueError("masks must have a bit for each of max_count tokens")
    if q.stride(2) != 1 or q.stride(1) != dim or q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.zeros((rows, hq, dim), dtype=torch.bfloat16, device=device)
    else:
        _on(device, "out", out, torch.bfloat16, (rows, hq, dim))
    if rows == 0:
        return out
    need = _tree_workspace_bytes(batch, rows, max_count, hq, kv_heads, dim, pps, page_size)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif (not isinstance(workspace, torch.Tensor) or workspace.dtype is not torch.uint8 or workspace.device != device
          or not workspace.is_contiguous() or workspace.numel() < need):
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on {device}")
    a = _lib.TreeAttnArgs(
        q.data_ptr(), q.stride(0), k_pool.data_ptr(), v_pool.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
        _dtype_code(k_scales.dtype), table.data_ptr(), lens.data_ptr(), first.data_ptr(),
        masks.data_ptr() if words else None, words, batch, rows, max_count, hq, kv_heads, dim, k_pool.shape[0], pps,
        page_size, out.data_ptr(), workspace.data_ptr(), workspace.numel())
    _launch.run("kv_tree_attention", _lib.load().q6moe_kv_tree_attention, device, ctypes.byref(a))
    return out


def keep_accepted(caches, page_table, lengths, path, accepted, *, page_size):
    """The accepted tokens of each tree, moved to the front of its places in every cache.

    For i < ``accepted[b]`` the cached token at position ``lengths[b] + path[b, i]``
    goes to position ``lengths[b] + i``, codes and scales; ``path`` int32 [batch,
    most] (most up to 256) holds the accepted path's indices within the tree, in
    any order: all are read before any is written. ``caches`` lists (codes, scales)
    pairs that share the page table: int8 [..., pages, page_size, channels] and
    [..., pages, page_size, groups], where leading dimensions stack the caches of
    several layers; up to 128 of them are updated in one launch. Then ``lengths +
    accepted`` are the cached tokens.
    """
    caches = list(caches)
    if not caches:
        raise ValueError("caches must hold at least one (codes, scales) pair")
    device = _gpu("codes", caches[0][0])
    _positive(page_size=page_size)
    table, lens = _int32(page_table, device), _int32(lengths, device)
    path, taken = _int32(path, device), _int32(accepted, device)
    if table.ndim != 2 or not table.shape[0] or not table.shape[1] or lens.shape != (table.shape[0],) or \
            taken.shape != lens.shape:
        raise ValueError("page_table must be [batch, pages_per_seq], lengths and accepted [batch]")
    if path.ndim != 2 or path.shape[0] != table.shape[0] or not 1 <= path.shape[1] <= MAX_TREE:
        raise ValueError(f"path must be [batch, most] with at most {MAX_TREE} tokens")
    pointers, stacked, spans, row = [], [], [], None
    for codes, scales in caches:
        if codes.dtype is not torch.int8 or codes.ndim < 3 or codes.device != device or not codes.is_contiguous() or \
                codes.shape[-2] != page_size:
            raise ValueError(f"codes must be contiguous int8 [..., pages, page_size, channels] on {device}")
        if scales.dtype not in (torch.bfloat16, torch.float32) or scales.shape[:-1] != codes.shape[:-1] or \
                scales.device != device or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous BF16 or FP32 [..., pages, page_size, groups] on {device}")
        sizes = codes.shape[-3], codes.shape[-1], scales.shape[-1] * scales.element_size()
        if row is None:
            row = sizes
        if sizes != row or not all(sizes):
            raise ValueError("all caches must have the same pages, channels and groups")
        held = codes.numel()
        if held:
            start, scale_start = codes.data_ptr(), scales.data_ptr()
            pointers += (start, scale_start)
            stacked.append(held // (sizes[0] * page_size * sizes[1]))
            spans += ((start, start + held), (scale_start, scale_start + held // sizes[1] * sizes[2]))
    spans.sort()
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
        raise ValueError("a cache may be listed only once")
    if not pointers:
        return
    a = _lib.KvKeepArgs(
        (ctypes.c_void_p * len(pointers))(*pointers), (ctypes.c_int64 * len(stacked))(*stacked), len(stacked), row[1],
        row[2], table.data_ptr(), lens.data_ptr(), path.data_ptr(), taken.data_ptr(), path.shape[0], path.shape[1],
        row[0], table.shape[1], page_size)
    _launch.run("kv_keep", _lib.load().q6moe_kv_keep, device, ctypes.byref(a))
