"""paged_attention where value scales lie far apart: a token with a huge value scale and next to no
weight must not cost the others their precision, one with all the weight and a scale of zero gives
zeros, and the order of both does not matter.

The kernel rounds probability x value scale to fp16 relative to the largest of a row's own: half a step
of each (2^-11), and at most 2^-24 of the largest for those that fp16 holds as subnormals."""
import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_attention_schedule import widened
from tests.test_gpu_paged_attention import BF16, F16, FP8, INT8, clean, make, run

pytestmark = pytest.mark.gpu


def expected(made, prefix, sm):
    """(out, bound) in 64 bits."""
    q, _, table, lens, pp = made
    (kc, ks), (vc, vs) = clean(made)
    B, S, Hq, D = q.shape
    P, H, g = kc.shape[0], kc.shape[1], Hq // kc.shape[1]
    code = lambda c: c.float().double()
    wide = lambda s: ref.scale_value(s).double()[:, :, 0, :, None]
    kd, vcode, vw = code(kc) * wide(ks), code(vc), wide(vs).expand(vc.shape)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    for b in range(B):
        rows = [torch.cat([ref.token_rows(t, pp.tolist() if prefix else [], prefix, P)[0],
                           ref.token_rows(t, table[b].tolist(), int(lens[b]), P)[0]]) for t in (kd, vcode, vw)]
        for s in range(S):
            n = prefix + max(0, int(lens[b]) - S + s + 1)
            if n == 0:
                continue
            k, c, w = (r[:n] for r in rows)
            for h in range(H):
                qq = q[b, s, h * g:(h + 1) * g].double()
                x = qq @ k[:, h].T * sm
                mx = (qq.abs() @ k[:, h].abs().T * sm).amax(-1, keepdim=True)
                p = torch.softmax(x, -1) * w[:, h, 0]
                out[b, s, h * g:(h + 1) * g] = p @ c[:, h]
                off[b, s, h * g:(h + 1) * g] = (p @ c[:, h].abs() * (2.0 ** -11 + 4 * mx * (D + 4) * ref.U + (n + 40) * ref.U)
                                                + 2.0 ** -24 * p.amax(-1, keepdim=True) * c[:, h].abs().sum(0))
    return out, off


def place(made, prefix, token, b):
    """(page, offset) of a token of the prefix or, behind it, of sequence b."""
    caches, table, pp = made[1], made[2], made[4]
    page = caches[0][0].shape[2]
    pages, t = (pp, token) if token < prefix else (table[b], token - prefix)
    return int(pages[t // page]), t % page


def put(made, prefix, token, b, score, factor):
    """Gives a token the score of every query (all of q's elements are 1) and a factor to its values."""
    (kc, ks), (vc, vs) = made[1]
    D = kc.shape[3]
    page, at = place(made, prefix, token, b)
    level = 64.0
    kc[page, :, at] = torch.full((kc.shape[1], D), level if score > 0 else -level).to(kc.dtype)
    ks[page, :, 0, at] = abs(score) / level / D / D ** -0.5
    vs[page, :, 0, at] *= factor


FORMS = [
    # lens, S, Hq, H, D, prefix, tokens that the table has room for
    ([200, 33], 1, 8, 2, 128, 0, None), ([300], 1, 8, 1, 64, 0, 1 << 20), ([260, 90], 1, 2, 2, 256, 0, None),
    ([140, 150], 20, 4, 2, 64, 0, None), ([150, 120], 24, 4, 1, 128, 0, None), ([260, 190], 100, 2, 1, 128, 0, 1 << 24),
    ([190], 64, 2, 1, 256, 0, 1 << 24), ([40, 90, 0], 1, 8, 2, 64, 150, None), ([70] * 9, 2, 4, 1, 128, 150, None),
]


@pytest.mark.parametrize("qdt,dtype", [(FP8, BF16), (INT8, F16)])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{len(f[0])}x{max(f[0])}_{'_'.join(map(str, f[1:]))}")
@pytest.mark.parametrize("factor,score", [(2.0 ** 22, -25.0), (2.0 ** 40, -60.0), (2.0 ** 60, -80.0), (0.0, 30.0)])
def test_scales_far_apart(pkg, gpu, form, qdt, dtype, factor, score):
    lens, S, Hq, H, D, prefix, most = form
    note(f"scales far apart {form} {qdt} {dtype} {factor} {score}")
    for where in (0, 37, 100):             # of the sequence's tokens, the prefix ahead of them
        made = make(D + where, lens, S, Hq, H, D, 16, prefix, qdt, False, dtype)
        made = (torch.ones_like(made[0]), *made[1:])
        for b, n in enumerate(lens):
            if where < prefix and b == 0 or prefix <= where < n:
                put(made, prefix, where, b, score, factor)
        r, bound = expected(made, prefix, D ** -0.5)
        o = run(pkg, gpu, made if most is None else widened(made, most, 16), prefix)
        assert ref.outside(o, r, bound, dtype) == 0
