"""GPU tests of the step operators at the ends of their ranges."""

import numpy as np
import pytest
import torch

from q6moe import plan_pages, write_tokens

from .test_gpu_step import _attn, _case, _dev

pytestmark = pytest.mark.gpu


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
