"""prompt_attention where one key takes nearly all of a row's weight and thousands of others make its output,
and where scores climb from tile to tile, against its formula in 64 bits."""
import pytest
import torch

from tests import attention_ref, prompt_ref as ref
from tests.gpu_util import note
from tests.test_gpu_prompt_range import ONCE, excess

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16



@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,m,Hq,H,D", [(3, 65536, 2, 1, 128), (4096, 32768, 16, 1, 64), (2, 65536, 4, 4, 64),
                                        (512, 40000, 8, 2, 256), (2048, 20000, 64, 1, 128)])
def test_many_small_weights(pkg, gpu, n, m, Hq, H, D, dtype):
    """A first key that takes nearly all of the weight and has no value, and thousands that share the
    rest, each 2^-26 of it: they alone make the output."""
    note(f"small weights {n} {m} {Hq} {H} {D} {dtype}")
    g = torch.Generator().manual_seed(m + D)
    q, k, v = (torch.randn(x, h, D, generator=g) for x, h in ((n, Hq), (m, H), (m, H)))
    q, k, v = q * 0.5, k * 0.5, v + 1.0
    q[..., 0], k[..., 0], k[0], v[0] = 8.0, 0.0, 0.0, 0.0
    k[0, :, 0] = 18.0 * 8.0 / 8.0                           # 18 = ln 2^26 at a scale of 1 / 8
    q, k, v = (t.to(dtype).to(gpu) for t in (q, k, v))
    cu, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=gpu) for x in (n, m))
    out, lse = pkg.prompt_attention(q, k, v, cu, 0.125, cu_seqlens_k=cu_k, return_lse=True)
    last = min(n, 128)
    hide = torch.ones(last, m, dtype=torch.bool, device=gpu).triu(m - last + 1)
    for h in {0, Hq // 2, Hq - 1}:
        kk, vv = k[:, h * H // Hq].double(), v[:, h * H // Hq].double()
        x = (q[n - last:, h].double() @ kk.T * 0.125).masked_fill(hide, float("-inf"))
        s = torch.logsumexp(x, 1)
        e = excess(out[n - last:, h], torch.exp(x - s[:, None]) @ vv)
        print(f"   head {h} {e:.3f}", flush=True)
        assert e <= ONCE, (h, e)
        # The score of 18 errs by 2 (D + 4) 2^-24 of itself; the sum of m terms, taken in steps of 32 and
        # more, by (m / 32 + 40) 2^-24, and so its logarithm.
        most = (36 * (D + 4) + m / 32 + 40) * 2.0 ** -24
        assert float((lse[h, n - last:].double() - s).abs().max()) <= most


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_climb_a_little(pkg, gpu, dtype):
    """Each tile's largest score a little above the last one's: weights up to the largest that the
    running maximum lets pass, and the type has to hold."""
    note(f"climbing scores {dtype}")
    for step in (0.5, 1.4, 2.0, 5.4, 9.0):                 # a tile of 64 keys, in units of ln
        m, D = 1024, 64
        g = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(x, 1, D, generator=g) for x in (200, m, m))
        q[..., 0], k[..., 0] = 1.0, (torch.arange(m) // 64 * step)[:, None]
        q[..., 1:] *= 0.2
        q, k, v = (t.to(dtype).to(gpu) for t in (q, k, v))
        cu, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=gpu) for x in (200, m))
        out, lse = pkg.prompt_attention(q, k, v, cu, 1.0, cu_seqlens_k=cu_k, return_lse=True)
        o, off, s, s_off = ref.forward(q.cpu(), k.cpu(), v.cpu(), cu.cpu(), 1.0, cu_k.cpu())
        assert attention_ref.outside(out, o, off, dtype) == 0
        assert bool(((lse.double().cpu() - s).abs() <= s_off).all())
