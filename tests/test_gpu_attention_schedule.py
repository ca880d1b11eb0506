"""paged_attention's ways to cut its work, each against the softmax in 64 bits: few rounds (chunks),
many (shares of equal rounds, worked out on the device), and so many that the codes are read past
the caches.  The host knows only a bound on the lengths, so a wide, mostly empty page table takes
short sequences down every way."""
import random

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_paged_attention import BF16, F16, FP8, INT8, check, make, run

pytestmark = pytest.mark.gpu

SLOTS = 2 * 256


def widened(made, tokens, page):
    """The same call with room for `tokens` tokens of each sequence in its page table."""
    q, caches, table, lens, pp = made
    wide = torch.full((table.shape[0], -(-tokens // page)), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table[:, :wide.shape[1]]
    return q, caches, wide, lens, pp


def bound_for(rounds, B, H):
    """Tokens of each of B sequences with H heads that make so many rounds of 128."""
    return -(-rounds // (B * H)) * 128


CASES = [
    # lens, S, Hq, H, D, page, prefix
    ([1], 1, 1, 1, 64, 16, 0), ([0, 0, 0], 1, 4, 2, 128, 16, 0), ([127, 128, 129, 256, 0], 1, 8, 2, 128, 16, 0),
    ([3000, 5, 700], 1, 16, 2, 64, 64, 0), ([1500, 1, 0, 900], 1, 8, 4, 256, 32, 0), ([2600], 1, 12, 1, 128, 128, 0),
    ([400, 0, 77], 3, 12, 2, 128, 16, 0), ([300, 17], 8, 6, 2, 64, 32, 0), ([90, 1100], 4, 8, 1, 128, 16, 0),
    ([1000, 3], 16, 4, 1, 64, 64, 0),
    ([200, 0, 31], 1, 8, 2, 128, 16, 300), ([700, 20, 5] * 6, 1, 16, 2, 64, 16, 130), ([40, 333], 2, 16, 2, 256, 32, 100),
    ([260, 9] * 5, 4, 8, 1, 128, 64, 1000), ([130] * 20, 1, 20, 4, 64, 16, 77),
]


@pytest.mark.parametrize("rounds", [8 * SLOTS - 100, 8 * SLOTS + 600, 64 * SLOTS])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_every_way(pkg, gpu, case, rounds):
    lens, S, Hq, H, D, page, prefix = case
    note(f"schedule {case} rounds {rounds}")
    qdt, ue8m0, dtype = random.Random(D + S + rounds).choice([(FP8, False, BF16), (INT8, True, F16), (FP8, True, F16)])
    made = make(len(lens) + rounds, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype)
    made = widened(made, max(bound_for(rounds, len(lens), H), max(lens)), page)
    check(pkg, gpu, made, prefix)


@pytest.mark.parametrize("B,idx", [(64, torch.int32), (65, torch.int64), (257, torch.int32), (700, torch.int64)])
def test_many_sequences(pkg, gpu, B, idx):
    """One lane for each of up to 64 sequences, the workgroup's threads for more."""
    rng = random.Random(B)
    lens = [rng.choice([0, 1, rng.randint(1, 300)]) for _ in range(B)]
    lens[B // 2] = 1700
    note(f"schedule {B} sequences")
    q, caches, table, n, pp = make(B, lens, 1, 4, 2, 64, 16)
    check(pkg, gpu, widened((q, caches, table, n.to(idx), pp), bound_for(9 * SLOTS, B, 2) + 1800, 16))


def test_full_shares(pkg, gpu):
    """More rounds than workgroups: shares that span units and units that span shares."""
    rng = random.Random(9)
    lens = [rng.randint(1, 1500) for _ in range(40)]
    note("schedule, full shares")
    made = make(3, lens, 1, 32, 16, 64, 64)
    assert sum(-(-n // 128) for n in lens) * 16 > 5 * SLOTS
    check(pkg, gpu, widened(made, 2048, 64))


def test_ways_agree_and_repeat(pkg, gpu):
    """Every way lies within the bounds of the same 64-bit result, and gives the same bits again."""
    lens = [1000, 0, 77, 2300, 128]
    made = make(4, lens, 1, 16, 2, 128, 16)
    for tokens in (2400, 128 * 500, 128 * 4000):
        wide = widened(made, tokens, 16)
        a, b = run(pkg, gpu, wide), run(pkg, gpu, wide)
        assert torch.equal(a, b)
        check(pkg, gpu, wide)


@pytest.mark.parametrize("prefix", [0, 90])
def test_missing_pages_in_shares(pkg, gpu, prefix):
    made = make(6, [1000, 640, 33], 1, 8, 2, 128, 16, prefix)
    table = made[2]
    table[0, 2], table[0, 40], table[1, 8:24], table[2, 0] = -1, 2 ** 31 - 1, -5, -1
    note(f"schedule, missing pages, prefix {prefix}")
    check(pkg, gpu, widened(made, 128 * 1000, 16), prefix)


@pytest.mark.parametrize("tokens", [128 * 300, 128 * 3000])
@pytest.mark.parametrize("prefix", [0, 200])
def test_workspace_of_shares(pkg, gpu, tokens, prefix):
    from fagq_mi355x import kv_cache
    note(f"schedule workspace {tokens} prefix {prefix}")
    made = widened(make(9, [700, 20, 0, 1300], 1, 16, 2, 128, 16, prefix), tokens, 16)
    need = kv_cache.attention_workspace_bytes(4, 1, 16, 2, 128, prefix, tokens)
    want = run(pkg, gpu, made, prefix)
    for fill in (0, 0xFF):
        buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
        buf[:need] = fill
        got = run(pkg, gpu, made, prefix, workspace=buf[:need])
        assert torch.equal(got, want) and bool((buf[need:] == 0xA5).all())


@pytest.mark.parametrize("B,idx,D", [(64, torch.int32, 64), (65, torch.int64, 128), (257, torch.int32, 64), (700, torch.int64, 256)])
def test_many_sequences_in_shares(pkg, gpu, B, idx, D):
    """As above, with room for sequences so long that they are cut into shares."""
    rng = random.Random(B)
    lens = [rng.choice([0, 1, rng.randint(1, 300)]) for _ in range(B)]
    lens[B // 2], lens[-1] = 1700, 900
    note(f"schedule {B} sequences in shares, D {D}")
    q, caches, table, n, pp = make(B, lens, 1, 4, 2, D, 16)
    check(pkg, gpu, widened((q, caches, table, n.to(idx), pp), 128 * 48, 16))


def test_full_shares_of_long_sequences(pkg, gpu):
    rng = random.Random(10)
    lens = [rng.randint(1, 1500) for _ in range(40)]
    note("schedule, full shares of long sequences")
    check(pkg, gpu, widened(make(5, lens, 1, 32, 16, 64, 64), 128 * 48, 64))
    check(pkg, gpu, widened(make(6, lens, 1, 32, 16, 128, 64, 70), 128 * 48, 64), 70)
