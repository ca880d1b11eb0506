"""paged_attention's tall units (64 or 128 query rows that see the same keys, for heads of 256 and
128): long chunks of new tokens and prefixes of large batches, against the softmax in 64 bits, at
row counts about the borders of units and lengths that end anywhere.  They are taken where the bound
on the keys is large; what is really there may be little."""
import random

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_attention_schedule import widened
from tests.test_gpu_paged_attention import BF16, F16, FP8, INT8, check, clean, make, run

pytestmark = pytest.mark.gpu

FORMATS = [(FP8, False, BF16), (FP8, True, F16), (INT8, False, F16), (INT8, True, BF16)]
KEYS = 1 << 25                     # of all units' lists together: so many that units are tall

CASES = [
    # lens, S, Hq, H, D, page
    ([300, 5, 64], 64, 4, 2, 128, 16), ([43, 42], 43, 2, 1, 128, 16), ([128, 1], 128, 1, 1, 128, 64),
    ([129, 257, 31], 129, 2, 2, 128, 32), ([400], 300, 4, 1, 128, 16), ([33, 700], 86, 1, 1, 128, 128),
    ([70, 20, 130], 22, 4, 2, 256, 16), ([100], 65, 1, 1, 256, 64), ([64, 65, 63], 64, 2, 2, 256, 32),
    ([0, 0], 128, 1, 1, 128, 16), ([2900, 1100], 96, 1, 1, 128, 64), ([1, 4100], 64, 1, 1, 256, 64),
    ([300, 90, 5], 40, 2, 1, 256, 16), ([2100], 50, 4, 2, 64, 16),
]


def spread(made, prefix, tokens):
    """(the same call with the prefix's pages among missing ones, in a list of about so many tokens,
    which ends where the last page does; that list's length)."""
    q, caches, table, lens, pp = made
    page = caches[0][0].shape[2]
    n = -(-tokens // page)
    at = sorted(random.Random(n).sample(range(n - 1), pp.numel() - 1)) + [n - 1]
    wide = torch.full((n,), -1, dtype=torch.int32)
    wide[1::2] = 2 ** 31 - 1
    wide[at] = pp
    return (q, caches, table, lens, wide), (n - 1) * page + (prefix - 1) % page + 1


def check_spread(pkg, gpu, made, prefix, tokens):
    q, _, table, lens, pp = made
    o = run(pkg, gpu, *spread(made, prefix, tokens))
    (kc, ks), (vc, vs) = clean(made)
    r, bound = ref.attention(q, kc, vc, ks, vs, table, lens, q.shape[-1] ** -0.5, pp, prefix)
    assert ref.outside(o, r, bound, q.dtype) == 0


@pytest.mark.parametrize("fmt", range(4))
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_own_keys(pkg, gpu, case, fmt):
    lens, S, Hq, H, D, page = case
    qdt, ue8m0, dtype = FORMATS[fmt]
    note(f"tall {case} {qdt} {ue8m0} {dtype}")
    made = make(len(lens) * 31 + D + S, lens, S, Hq, H, D, page, 0, qdt, ue8m0, dtype)
    check(pkg, gpu, widened(made, KEYS // len(lens) // H + 1, page))


PREFIXES = [
    # lens, S, Hq, H, D, page, prefix
    ([0] * 90, 1, 2, 2, 128, 16, 31), ([3, 0, 40] * 29, 1, 1, 1, 128, 16, 32), ([20] * 16, 1, 16, 2, 128, 32, 65),
    ([50, 2] * 3, 4, 4, 1, 256, 64, 97), ([33, 80], 64, 4, 2, 128, 16, 50), ([300, 90, 5], 40, 2, 1, 256, 16, 160),
    ([7] * 6, 1, 20, 1, 128, 16, 1500), ([9, 300] * 8, 2, 12, 1, 64, 16, 200), ([17] * 130, 1, 2, 1, 64, 16, 33),
]


@pytest.mark.parametrize("fmt", range(4))
@pytest.mark.parametrize("case", PREFIXES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_prefix(pkg, gpu, case, fmt):
    lens, S, Hq, H, D, page, prefix = case
    qdt, ue8m0, dtype = FORMATS[fmt]
    note(f"tall prefix {case} {qdt} {ue8m0} {dtype}")
    made = make(len(lens) * 31 + D + S, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype)
    check_spread(pkg, gpu, made, prefix, KEYS // H + 1)
    check_spread(pkg, gpu, widened(made, KEYS // len(lens) // H + 1, page), prefix, KEYS // H + 1)


@pytest.mark.parametrize("rows", [85, 86, 127, 128, 129, 170, 171, 172, 255, 256, 257])
def test_border_of_row_counts(pkg, gpu, rows):
    note(f"tall rows {rows}")
    check(pkg, gpu, widened(make(rows, [rows + 40], rows, 1, 1, 128, 16), KEYS, 16))
    check_spread(pkg, gpu, make(rows, [2] * rows, 1, 1, 1, 128, 16, 70), 70, KEYS)


@pytest.mark.parametrize("keys", [KEYS >> i for i in range(12)])
def test_number_of_keys(pkg, gpu, keys):
    """Few keys leave short units, many take tall ones."""
    note(f"tall keys {keys}")
    check(pkg, gpu, widened(make(5, [200, 90], 96, 1, 1, 128, 16), keys // 2, 16))
    check_spread(pkg, gpu, make(6, [2] * 100, 1, 1, 1, 128, 16, 70), 70, keys)


def test_missing_pages(pkg, gpu):
    note("tall missing pages")
    made = make(6, [260, 200, 133], 100, 2, 1, 128, 16)
    table = made[2]
    table[0, 2], table[0, 9:12], table[1, :4], table[2, 0] = -1, 2 ** 31 - 1, -5, -1
    check(pkg, gpu, widened(made, KEYS // 3 + 1, 16))


@pytest.mark.parametrize("tokens", [128 * 40, 128 * 400])
def test_prefix_beside_shares(pkg, gpu, tokens):
    """A tall prefix in the launch of own keys that are cut into shares on the device."""
    note(f"tall prefix beside shares, {tokens}")
    lens = [900, 3, 0, 260] * 30
    made = make(2, lens, 1, 4, 2, 128, 16, 300)
    check_spread(pkg, gpu, widened(made, tokens, 16), 300, KEYS)


def test_short_prefix_beside_many_rows(pkg, gpu):
    """Many rows of their own keys, whose units are short where the prefix's are."""
    note("short prefix beside many rows")
    made = make(8, [300, 90], 100, 1, 1, 128, 16, 75)
    check(pkg, gpu, widened(made, KEYS, 16), 75)
