"""The torch.autograd.Function that users are shown for prompt_attention, with keys of a context before the
queries: gradients of the context's keys and values too."""
import pytest
import torch

from tests import attention_ref
from tests import prompt_ref as ref
from tests.gpu_util import note
from tests.test_gpu_prompt_autograd import shown

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_a_context(pkg, gpu, dtype):
    note(f"a context through autograd {dtype}")
    Hq, H, D, lens, lens_k = 6, 2, 64, [70, 1, 33], [100, 40, 33]
    g = torch.Generator().manual_seed(9)
    q, do = (torch.randn(sum(lens), Hq, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(sum(lens_k), H, D, generator=g).to(dtype) for _ in range(2))
    cu, cu_k = (torch.tensor([0] + x).cumsum(0).int() for x in (lens, lens_k))
    leaves = [t.to(gpu).requires_grad_() for t in (q, k, v)]
    out = shown(pkg).apply(*leaves, cu.to(gpu), 0.125, cu_k.to(gpu))
    o, off, lse, _ = ref.forward(q, k, v, cu, 0.125, cu_k)
    assert attention_ref.outside(out.detach(), o, off, dtype) == 0
    got = torch.autograd.grad(out, leaves, do.to(gpu))
    _, lse = pkg.prompt_attention(*[t.detach() for t in leaves], cu.to(gpu), 0.125, cu_k.to(gpu), return_lse=True)
    want = ref.backward(do, q, k, v, out.detach().cpu(), lse.cpu(), cu, 0.125, cu_k)
    for t, (r, off) in zip(got, want):
        assert attention_ref.outside(t, r, off, dtype) == 0
