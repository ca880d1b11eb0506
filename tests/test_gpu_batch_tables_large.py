"""batch_tables at the ends of its sizes: as many rows as there may be, and many thousands of requests."""
import pytest
import torch

from tests.gpu_util import note
from tests.test_gpu_batch_tables import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 1023, 2 ** 31 - 1024])
def test_as_many_rows_as_there_may_be(pkg, gpu, rows):
    """26 GB of positions and slots: a first request's few tokens, one that takes nearly all, rows of padding."""
    note(f"tables of {rows} rows")
    page, few, pad = 65536, 5, 1000
    new, context = [few, 0, rows - few - pad], [page - 2, 7, 10]
    width = -(-(rows + 10) // page)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    table = torch.full((3, width), -1, dtype=torch.int32, device=gpu)
    table[:, 0] = i32([3, 5, 7])
    free = torch.randperm(width + 8, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(gpu) + 11
    cu, cu_k, lens, pos, slots, end = pkg.batch_tables(i32(context), i32(new), free, table, page, rows)
    both = [a + b for a, b in zip(context, new)]
    assert cu.tolist() == [0, few, few, rows - pad]
    assert lens.tolist() == both and cu_k.tolist() == [0, both[0], both[0] + 7, min(sum(both), 2 ** 31 - 1)]
    want = [-(-b // page) - 1 for b in both]               # pages taken; each has one
    assert int(end) == sum(want)
    assert torch.equal(table[0, 1:2], free[:1]) and torch.equal(table[2, 1:1 + want[2]], free[1:1 + want[2]])
    assert pos[:few].tolist() == list(range(page - 2, page + 3))
    f = int(free[0]) * page
    assert slots[:few].tolist() == [4 * page - 2, 4 * page - 1, f, f + 1, f + 2]
    assert bool((pos[rows - pad:] == -1).all()) and bool((slots[rows - pad:] == -1).all())
    for a in range(few, rows - pad, 1 << 27):
        b = min(rows - pad, a + (1 << 27))
        at = torch.arange(a - few + 10, b - few + 10, device=gpu)
        assert torch.equal(pos[a:b].long(), at)
        assert torch.equal(slots[a:b], table[2, at // page].long() * page + at % page)


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_thousands_of_requests(pkg, gpu, idx):
    """More than one pass over the requests in each of several workgroups."""
    B = 30000
    context, new = [(i * 7) % 90 for i in range(B)], [(1, 1, 0, 3, 1, 20)[i % 6] for i in range(B)]
    note(f"tables of {B} requests {idx}")
    check(pkg, gpu, context, new, 16, sum(new) + 40, idx)
    check(pkg, gpu, context, new, 16, sum(new) - 999, idx)
