"""prompt_attention and its gradients at the ends of their sizes, on the GPU: more tiles of keys than one
launch holds, empty sequences by the hundred thousand."""
import pytest
import torch

from tests import attention_ref, prompt_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_more_tiles_of_keys_than_a_launch_holds(pkg, gpu):
    """2100 sequences of one or two tokens, 4096 heads: 8.6 million tiles, in three launches."""
    B, H, D = 2100, 4096, 64
    note(f"{B} sequences, {H} heads")
    lens = [2 if b % 11 == 3 else 1 for b in range(B)]
    T = sum(lens)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    g = torch.Generator(device=gpu).manual_seed(1)
    q, k, v, do = (torch.randn(T, H, D, generator=g, device=gpu, dtype=BF16) for _ in range(4))
    out, lse = pkg.prompt_attention(q, k, v, cu.to(gpu), 0.125, return_lse=True)
    grads = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu.to(gpu), 0.125)
    one = torch.tensor([int(cu[b]) for b in range(B) if lens[b] == 1], device=gpu)
    # A token that sees itself alone: its value, no gradients for its query and key but what fp32 leaves
    # of dP - delta, two sums of D products each.
    assert torch.equal(out[one], v[one]) and torch.equal(grads[2][one], do[one])
    left = 0.125 * 2 * (D + 8) * 2.0 ** -24 * (do[one].float() * v[one].float()).abs().sum(-1, keepdim=True)
    for x, y in zip(grads[:2], (k, q)):
        assert bool((x[one].float().abs() <= left * y[one].float().abs() * 1.01).all())
    for h in (0, 1, 2047, 4095):
        own = [t[:, h:h + 1].cpu() for t in (do, q, k, v, out)]
        o, off, _, _ = ref.forward(*own[1:4], cu, 0.125)
        assert attention_ref.outside(own[4], o, off, BF16) == 0
        want = ref.backward(*own, lse[h:h + 1].cpu(), cu, 0.125)
        for x, (r, off) in zip(grads, want):
            assert attention_ref.outside(x[:, h:h + 1], r, off, BF16) == 0


@pytest.mark.parametrize("T,Tk", [(0, 900), (300, 300), (300, 900), (40, 0)])
def test_hundreds_of_thousands_of_empty_sequences(pkg, gpu, T, Tk):
    """All rows in the last sequence but one, or in none."""
    note(f"empty sequences, {T} {Tk}")
    B, D = 300000, 64
    g = torch.Generator().manual_seed(2)
    q, do = (torch.randn(T, 1, D, generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(Tk, 1, D, generator=g).to(BF16) for _ in range(2))
    cu, cu_k = (torch.cat((torch.zeros(B - 1), torch.full((2,), float(n)))).to(torch.int32) for n in (T, Tk))
    up = [t.to(gpu) for t in (q, k, v, cu, cu_k, do)]
    out, lse = pkg.prompt_attention(*up[:4], 0.125, cu_seqlens_k=up[4], return_lse=True)
    grads = pkg.prompt_attention_bwd(up[5], *up[:3], out, lse, up[3], 0.125, cu_seqlens_k=up[4])
    two = lambda n: torch.tensor([0, n])
    o, off, _, _ = ref.forward(q, k, v, two(T), 0.125, two(Tk))
    assert attention_ref.outside(out, o, off, BF16) == 0
    for x, (r, off) in zip(grads, ref.backward(do, q, k, v, out.cpu(), lse.cpu(), two(T), 0.125, two(Tk))):
        assert attention_ref.outside(x, r, off, BF16) == 0


@pytest.mark.parametrize("B,H", [(1000, 2), (5000, 1)])
def test_gradients_of_many_sequences(pkg, gpu, B, H):
    """One workgroup for each sequence and more, empty ones and some of several tiles among them."""
    note(f"gradients of {B} sequences")
    lens = [[1, 0, 5, 17, 2, 40, 0][(b * 3 + b // 11) % 7] + (300 if b % 997 == 5 else 0) for b in range(B)]
    T, D = sum(lens), 64
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    g = torch.Generator().manual_seed(3)
    q, do = (torch.randn(T, 2 * H, D, generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(T, H, D, generator=g).to(BF16) for _ in range(2))
    up = [t.to(gpu) for t in (q, k, v, cu)]
    out, lse = pkg.prompt_attention(*up, 0.125, return_lse=True)
    grads = pkg.prompt_attention_bwd(do.to(gpu), *up[:3], out, lse, up[3], 0.125)
    for x, (r, off) in zip(grads, ref.backward(do, q, k, v, out.cpu(), lse.cpu(), cu, 0.125)):
        assert attention_ref.outside(x, r, off, BF16) == 0
