"""batch_tables on the GPU against a loop over the requests (tests/prompt_ref.py)."""
import random

import pytest
import torch

from tests import prompt_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

NAMES = ("cu_seqlens", "cu_seqlens_k", "kv_lens", "positions", "slots", "free_end")


def make(seed, context, new, page, spare_width=1, spare_pages=3, width=None):
    rng = random.Random(seed)
    have = [-(-max(0, c) // page) for c in context]
    need = [-(-(max(0, c) + max(0, n)) // page) for c, n in zip(context, new)]
    width = max(need + [0]) + spare_width if width is None else width
    order = rng.sample(range(sum(need) + spare_pages), sum(need) + spare_pages)
    table = torch.full((len(context), width), -7, dtype=torch.int32)
    at = 0
    for b, h in enumerate(have):
        h = min(h, width)
        table[b, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
        at += h
    return table, torch.tensor(order[at:], dtype=torch.int32)


def check(pkg, gpu, context, new, page, rows, idx=torch.int32, start=None, made=None, seed=1):
    table, free = make(seed, context, new, page) if made is None else made
    c, n = torch.tensor(context, dtype=idx), torch.tensor(new, dtype=idx)
    want = ref.tables(context, new, free, table, page, rows, 0 if start is None else start)
    t = table.to(gpu)
    s = None if start is None else torch.tensor([start], dtype=torch.int32, device=gpu)
    for _ in range(2):                                     # again: the same results
        got = pkg.batch_tables(c.to(gpu), n.to(gpu), free.to(gpu), t, page, rows, free_start=s)
        for name, g, w in zip(NAMES, got, want):
            assert g.dtype == w.dtype and torch.equal(g.cpu(), w), name
        assert torch.equal(t.cpu(), want[-1])


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("context,new,page,spare", [
    ([], [], 16, 0), ([], [], 16, 5), ([0], [1], 16, 0), ([16], [1], 16, 0), ([15], [1], 16, 3), ([15], [2], 16, 0),
    ([0, 5, 0], [0, 0, 0], 32, 4), ([100, 3, 0, 17], [1, 1, 1, 1], 16, 0), ([0, 40, 7], [33, 100, 0], 64, 9),
    ([-3, 10], [5, -9], 16, 0), ([1000] * 70, [3] * 70, 128, 1), ([5000, 0], [0, 6000], 16, 100),
    ([7] * 1024, [1] * 1024, 16, 0), ([7] * 1500, [2] * 1500, 16, 5), ([0] * 2100, [1, 0, 3] * 700, 16, 0),
])
def test_tables(pkg, gpu, context, new, page, spare, idx):
    note(f"tables {len(context)} {context[:3]} {new[:3]} page {page} spare {spare} {idx}")
    check(pkg, gpu, context, new, page, sum(max(0, n) for n in new) + spare, idx)


@pytest.mark.parametrize("seed", range(8))
def test_random(pkg, gpu, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 7, 64, 300])
    context = [rng.choice([0, rng.randint(0, 50), rng.randint(0, 3000)]) for _ in range(B)]
    new = [rng.choice([0, 1, rng.randint(0, 200)]) for _ in range(B)]
    page, start = rng.choice([16, 64, 256]), rng.choice([None, 0, 2])
    note(f"tables seed {seed}")
    check(pkg, gpu, context, new, page, sum(new) + rng.choice([0, 50]), start=start,
          made=make(seed, context, new, page))


def test_more_tokens_than_rows(pkg, gpu):
    note("more tokens than rows")
    for rows in (0, 1, 30, 55):
        check(pkg, gpu, [10, 0, 5], [20, 30, 6], 16, rows)


def test_free_pages_run_out(pkg, gpu):
    table, free = make(2, [3, 0, 20], [40, 50, 60], 16)
    note("free pages run out")
    for count in (0, 1, 4, 9):
        check(pkg, gpu, [3, 0, 20], [40, 50, 60], 16, 150, made=(table, free[:count]))
    check(pkg, gpu, [3, 0, 20], [40, 50, 60], 16, 150, made=(table, free), start=2 ** 31 - 2)
    check(pkg, gpu, [3, 0, 20], [40, 50, 60], 16, 150, made=(table, free), start=-2 ** 31)


def test_tokens_past_the_table(pkg, gpu):
    note("tokens past the table")
    for width in (0, 1, 3):
        check(pkg, gpu, [3, 0, 200], [40, 50, 60], 16, 150, made=make(3, [3, 0, 200], [40, 50, 60], 16, width=width))


def test_lengths_of_any_value(pkg, gpu):
    low, high = torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max
    note("lengths of any value")
    context, new = [low, high, 2 ** 31 - 3, 2 ** 31 - 1, 2 ** 40], [3, 2, 6, 2, low]
    made = (torch.zeros(5, 2, dtype=torch.int32), torch.arange(4, dtype=torch.int32))
    check(pkg, gpu, context, new, 65536, 15, torch.int64, made=made)
    check(pkg, gpu, [0, 4, 1], [high, high, 3], 16, 40, torch.int64,
          made=(torch.zeros(3, 4, dtype=torch.int32), torch.arange(9, dtype=torch.int32)))


def test_steps_chain_without_the_host(pkg, gpu):
    """free_end of a step is free_start of the next: no page is given out twice."""
    page, B = 16, 5
    free = torch.randperm(200, dtype=torch.int32, generator=torch.Generator().manual_seed(4)).to(gpu)
    table = torch.full((B, 30), -1, dtype=torch.int32, device=gpu)
    lens, start = torch.zeros(B, dtype=torch.int32, device=gpu), None
    seen = []
    note("steps in a chain")
    for step in range(6):
        new = torch.tensor([17, 1, 0, 40, 5] if step == 0 else [1, 1, 9, 1, 16], dtype=torch.int32, device=gpu)
        _, _, lens, _, slots, start = pkg.batch_tables(lens, new, free, table, page, 64, free_start=start)
        seen.append(slots[slots >= 0])
    slots = torch.cat(seen)
    assert len(slots.unique()) == len(slots) == int(lens.sum())
    assert int(start) == sum(-(-n // page) for n in lens.tolist())


def test_refusals(pkg, gpu):
    i = dict(dtype=torch.int32, device=gpu)
    ok = dict(context_lens=torch.zeros(3, **i), new_lens=torch.ones(3, **i), free_pages=torch.arange(5, **i),
              page_table=torch.zeros(3, 4, **i), page_size=16, num_tokens=3)
    pkg.batch_tables(**ok)
    for bad in (dict(context_lens=torch.zeros(2, **i)), dict(new_lens=torch.zeros(4, **i)),
                dict(new_lens=torch.zeros(3, device=gpu, dtype=torch.int64)), dict(new_lens=torch.zeros(3, dtype=torch.int32)),
                dict(free_pages=torch.zeros(5, device=gpu)), dict(free_pages=torch.zeros(5, 1, **i)),
                dict(free_pages=torch.zeros(10, **i)[::2]), dict(page_table=torch.zeros(3, 8, **i)[:, ::2]),
                dict(page_table=torch.zeros(3, 4, device=gpu, dtype=torch.int64)), dict(page_table=torch.zeros(3, 4, dtype=torch.int32)),
                dict(page_size=8), dict(page_size=24), dict(page_size=131072), dict(num_tokens=-1),
                dict(free_start=torch.zeros(2, **i)), dict(free_start=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            pkg.batch_tables(**{**ok, **bad})
    with pytest.raises(TypeError):
        pkg.batch_tables(**{**ok, "context_lens": torch.zeros(3, device=gpu)})
    with pytest.raises(pkg.FagqError) as e:
        pkg.batch_tables(**{**ok, "page_table": torch.zeros(3, 4, **i), "free_pages": ok["context_lens"],
                            "num_tokens": 2 ** 31})
    assert e.value.status == 7
    table = torch.zeros(3, 4, **i)
    with pytest.raises(pkg.FagqError) as e:
        pkg.batch_tables(**{**ok, "page_table": table, "free_pages": table.view(-1)})
    assert e.value.status == 9
