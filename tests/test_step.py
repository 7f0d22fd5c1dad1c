"""The step operators without a GPU: refusals of the C ABI and of the Python
layer, and the oracle against worked examples."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import step as oracle
from q6moe import _lib, keep_accepted, paged_tree_attention, plan_pages, release_pages, write_tokens

FAKE = 1 << 20  # an aligned address that no call here reaches


def _filled(cls, **over):
    a = cls()
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, FAKE)
        elif kind in (ctypes.c_int64, ctypes.c_int, ctypes.c_size_t):
            setattr(a, name, 1)
    for name, v in over.items():
        setattr(a, name, v)
    return a


def _refused(fn, a, text):
    assert fn(ctypes.byref(a), None) == -1
    assert text in _lib.load().q6moe_last_error().decode()


def _plan(**over):
    return _filled(_lib.PlanArgs, **{**dict(parents=None, masks=None, workspace_bytes=1 << 20), **over})


@pytest.mark.parametrize("over,text", [
    (dict(page_table=None), "null pointer"), (dict(missing=None), "null pointer"), (dict(batch=0), "positive"),
    (dict(batch=65536), "65535"), (dict(rows=0), "positive"), (dict(rows=1 << 31), "2^31"),
    (dict(page_size=0), "positive"), (dict(pages_per_seq=1 << 20, page_size=1 << 20), "below 2^31"),
    (dict(free_capacity=0), "positive"), (dict(max_count=0), "positive"), (dict(parents=FAKE), "masks"),
    (dict(parents=FAKE, masks=FAKE, max_count=257), "256"), (dict(masks=FAKE), "masks need parents"),
    (dict(workspace_bytes=7), "workspace too small (need 8 bytes)"),
])
def test_plan_refusals(over, text):
    _refused(_lib.load().q6moe_kv_plan, _plan(**over), text)


def test_null_args():
    lib = _lib.load()
    for fn in (lib.q6moe_kv_plan, lib.q6moe_kv_write_rows, lib.q6moe_kv_tree_attention, lib.q6moe_kv_keep):
        assert fn(None, None) == -1 and b"null args" in lib.q6moe_last_error()
    assert lib.q6moe_kv_plan_workspace_size(0) == 0 and lib.q6moe_kv_plan_workspace_size(3) == 16


def test_release_refusals():
    lib = _lib.load()
    good = [FAKE, FAKE, FAKE, 8, FAKE, 2, 4, 16, FAKE, 12]
    for at, v, text in ((0, None, b"null"), (3, 0, b"positive"), (5, 0, b"positive"), (5, 65536, b"65535"),
                        (6, 1 << 31, b"2^31"), (7, 0, b"positive"), (9, 11, b"need 12 bytes")):
        args = list(good)
        args[at] = v
        assert lib.q6moe_kv_release(*args, None) == -1 and text in lib.q6moe_last_error()


@pytest.mark.parametrize("over,text", [
    (dict(slots=None), "null pointer"), (dict(rows=0), "positive"), (dict(pool_rows=0), "positive"),
    (dict(head_dim=0), "positive"), (dict(head_dim=64, group=48), "group must divide"),
    (dict(key_stride=-1), "negative"), (dict(x_dtype=7), "x dtype"), (dict(scale_dtype=7), "scale dtype"),
])
def test_write_refusals(over, text):
    _refused(_lib.load().q6moe_kv_write_rows, _filled(_lib.KvWriteRowsArgs, **over), text)


@pytest.mark.parametrize("k,v,ks,vs", [(0, 0, 0, 4096), (0, 639, 0, 4096), (639, 0, 0, 4096), (0, 4096, 0, 36),
                                       (0, 4096, 36, 0)])
def test_write_refuses_pools_that_overlap(k, v, ks, vs):
    # 10 rows of 64 codes and an FP32 scale
    a = _filled(_lib.KvWriteRowsArgs, pool_rows=10, head_dim=64, group=64, scale_dtype=_lib.F32, k_codes=FAKE + k,
                v_codes=FAKE + v, k_scales=FAKE + ks, v_scales=FAKE + vs)
    _refused(_lib.load().q6moe_kv_write_rows, a, "must not overlap")


@pytest.mark.parametrize("over,text", [
    (dict(q=None), "null pointer"), (dict(starts=None), "null pointer"), (dict(head_dim=96), "64, 128 or 256"),
    (dict(query_heads=3, kv_heads=2), "multiple of kv_heads"), (dict(batch=0), "at most 65535"),
    (dict(rows=0), "rows"), (dict(max_count=0), "max_count"), (dict(rows=1 << 24), "2^24"),
    (dict(page_size=0), "page_size"), (dict(pages_per_seq=1 << 20, page_size=1 << 20), "2^30"),
    (dict(scale_dtype=7), "scale dtype"), (dict(mask_words=5), "4 words"), (dict(max_count=65), "max_count bits"),
    (dict(q_stride=12), "multiple of 8"), (dict(q=FAKE + 8), "alignment"), (dict(workspace=FAKE + 16), "alignment"),
    (dict(workspace_bytes=0), "workspace too small"),
])
def test_attention_refusals(over, text):
    a = _filled(_lib.TreeAttnArgs, **{**dict(head_dim=128, q_stride=128), **over})
    _refused(_lib.load().q6moe_kv_tree_attention, a, text)


@pytest.mark.parametrize("over,text", [
    (dict(rows=1 << 24), "2^24"), (dict(pages_per_seq=1 << 20, page_size=1 << 20), "2^30"),
    (dict(batch=65536), "65535"), (dict(query_heads=65536), "65535"), (dict(mask_words=5), "4 words"),
    (dict(rows=(1 << 24) - 1, query_heads=65), "below 2^30"), (dict(), "null pointer (workspace)"),
])
def test_attention_names_the_limit_before_the_workspace(over, text):
    # a caller beyond a limit has a workspace of 0 bytes, whose pointer may be null
    sizes = {**dict.fromkeys(("batch", "rows", "max_count", "query_heads", "kv_heads", "pages_per_seq", "page_size"), 1),
             **over, "head_dim": 128}
    if text != "null pointer (workspace)" and "mask_words" not in over:
        assert _lib.load().q6moe_tree_attn_workspace_size(*(sizes[n] for n in (
            "batch", "rows", "max_count", "query_heads", "kv_heads", "head_dim", "pages_per_seq", "page_size"))) == 0
    a = _filled(_lib.TreeAttnArgs, **{**dict(head_dim=128, q_stride=128, workspace=None, workspace_bytes=0), **over})
    _refused(_lib.load().q6moe_kv_tree_attention, a, text)


@pytest.mark.parametrize("over,text", [
    (dict(path=None), "null pointer"), (dict(count=0), "positive"), (dict(code_bytes=0), "row sizes"),
    (dict(path_len=257), "1 to 256"), (dict(path_len=0), "1 to 256"), (dict(pool_pages=0), "positive"),
    (dict(pools=(ctypes.c_void_p * 2)(FAKE, None)), "null pool"),
    (dict(stacked=(ctypes.c_int64 * 1)(0)), "stacks 1 to"), (dict(pages_per_seq=1 << 16, page_size=1 << 16), "2^31"),
])
def test_keep_refusals(over, text):
    a = _filled(_lib.KvKeepArgs, **{**dict(pools=(ctypes.c_void_p * 2)(FAKE, FAKE)), **over})
    _refused(_lib.load().q6moe_kv_keep, a, text)


def test_python_layer_refuses_host_tensors():
    i = torch.zeros(1, dtype=torch.int32)
    pool, scales = torch.zeros(1, 4, 64, dtype=torch.int8), torch.ones(1, 4, 1)
    with pytest.raises(ValueError, match="page_table must be a GPU tensor"):
        plan_pages(i.view(1, 1), i, i, i, i, page_size=4, rows=1)
    with pytest.raises(ValueError, match="page_table must be a GPU tensor"):
        release_pages(i.view(1, 1), i, i, i, page_size=4)
    with pytest.raises(ValueError, match="k_pool must be a GPU tensor"):
        write_tokens(pool, scales, pool, scales, scales, scales, i, kv_heads=1, head_dim=64)
    with pytest.raises(ValueError, match="q must be a GPU tensor"):
        paged_tree_attention(torch.zeros(1, 1, 64, dtype=torch.bfloat16), pool, scales, pool, scales, i.view(1, 1), i,
                             torch.zeros(2, dtype=torch.int32), page_size=4, kv_heads=1, max_count=1)
    with pytest.raises(ValueError, match="codes must be a GPU tensor"):
        keep_accepted([(pool, scales)], i.view(1, 1), i, i.view(1, 1), i, page_size=4)
    with pytest.raises(ValueError, match="at least one"):
        keep_accepted([], i.view(1, 1), i, i.view(1, 1), i, page_size=4)


def test_oracle_plan_by_hand():
    # pages of 4; sequence 0 holds 3 tokens (page 9) and takes 3 more: one place in
    # page 9 and a new page; sequence 1 is new, takes 5 and finds one page only
    starts, slots, positions, sees, missing, table, have = oracle.plan(
        [[9, -1], [-1, -1]], [3, 0], [3, 5], [7, 5, 99], 2, 4, 10, parents=[-1, 0, 0, -1, 0, 1, 0, 9, 0, 0])
    assert starts.tolist() == [0, 3, 8] and table.tolist() == [[9, 5], [7, -1]] and have == 0
    assert slots.tolist() == [39, 20, 21, 28, 29, 30, 31, -1, -1, -1] and missing == 1
    assert positions.tolist() == [3, 4, 4, 0, 1, 2, 1, 0, 0, 0]
    assert sees[:8] == [{0}, {0, 1}, {0, 2}, {0}, {0, 1}, {0, 1, 2}, {0, 3}, {4}]
    assert oracle.masks_of([{0, 63, 64}], 2).tolist() == [[1 - 2**63, 1]]
    table, free, have = oracle.release(table, [3, 0], [7, 5, 99], 0, 4)
    assert table.tolist() == [[9, -1], [-1, -1]] and free.tolist() == [7, 5, 99] and have == 2


def test_oracle_keep_and_attention_by_hand():
    pool = np.arange(8).reshape(2, 4, 1)
    after = oracle.keep(pool, np.array([[1, 0]]), [2], np.array([[1, 3, 0]]), [3], 4)
    # positions 2.. hold 6 7 0 1: tokens 1, 3, 0 of the tree move to its front
    assert after[..., 0].tolist() == [[6, 1, 2, 3], [4, 5, 7, 1]]
    codes = np.array([1, 2, 3, 4], np.int8).reshape(1, 4, 1, 1).repeat(2, -1)
    out, spread, slope = oracle.attention(np.zeros((3, 1, 2)), codes, np.ones((1, 4, 1)), codes, np.ones((1, 4, 1)),
                                          np.array([[0]]), [1], [0, 2], [{0}, {1}, {0}], 4, 2)
    assert out[0, 0].tolist() == [1.5, 1.5] and out[1, 0].tolist() == [2.0, 2.0] and np.isnan(out[2]).all()
    assert spread[0, 0, 0] == 1.5 and slope[1, 0] == 6 / np.sqrt(2)
