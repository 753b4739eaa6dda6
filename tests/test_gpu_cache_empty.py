"""GPU: page operations on a pool without pages and on tables without columns."""
import pytest
import torch

import ops_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,width", [(0, 3), (0, 0), (5, 0)])
def test_nothing_to_hold(pages, width):
    i32 = dict(dtype=torch.int32, device="cuda")
    refs, table, lens = torch.zeros(pages, **i32), torch.full((2, width), -1, **i32), torch.zeros(2, **i32)
    pools = [torch.zeros(pages, 4, 3, device="cuda") for _ in range(2)]
    two, none = torch.tensor([0, 2], **i32), torch.zeros(2, **i32)
    assert ops_b200.paged_cache_reserve(refs, table, lens, two, 4).tolist() == [1, 0]
    ops_b200.paged_cache_trim(refs, table, lens, none, 4)
    assert ops_b200.paged_cache_fork(refs, table, lens, none, two - 1, pools).tolist() == [0, 1]
    assert ops_b200.paged_cache_accept(pools, table, lens, torch.full((2, 2), -1, **i32), none).tolist() == [0, 0]
    assert ops_b200.paged_cache_accept(pools, table, lens, torch.full((2, 2), -1, **i32), none, refcounts=refs).tolist() == [0, 0]
    assert ops_b200.paged_cache_compact(refs, table, pools).tolist() == [0]
    assert ops_b200.paged_cache_copy(pools, none, none + pages).tolist() == [0, 0]
    assert lens.tolist() == [0, 0] and (table == -1).all() and (refs == 0).all()
