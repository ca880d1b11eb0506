"""The torch.autograd.Function that users are shown for prompt_attention: its gradients are those
of prompt_attention_bwd, and of the formulas in 64 bits."""
import re
from pathlib import Path

import pytest
import torch

from tests import attention_ref
from tests import prompt_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu


def shown(pkg):
    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    block, = [b for b in re.findall(r"```python\n(.*?)```", text, flags=re.S) if "class PromptAttention" in b]
    ns = {"torch": torch, "fagq": pkg}
    exec(compile(block, "example", "exec"), ns)
    return ns["PromptAttention"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_through_autograd(pkg, gpu, dtype):
    note(f"prompts through autograd {dtype}")
    Hq, H, D, lens = 6, 2, 64, [70, 1, 33]
    T = sum(lens)
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(T, Hq + 2 * H, D, generator=g).to(dtype)
    do = torch.randn(T, Hq, D, generator=g).to(dtype)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    x = qkv.to(gpu).requires_grad_()
    out = shown(pkg).apply(x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:], cu.to(gpu), 0.125)
    got, = torch.autograd.grad(out, [x], [do.to(gpu)])
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    _, lse = pkg.prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), cu.to(gpu), 0.125, return_lse=True)
    own = pkg.prompt_attention_bwd(do.to(gpu), q.to(gpu), k.to(gpu), v.to(gpu), out.detach(), lse, cu.to(gpu),
                                   0.125)
    assert torch.equal(got, torch.cat(own, 1))
    want = ref.backward(do, q, k, v, out.detach().cpu(), lse.cpu(), cu, 0.125, None)
    for t, (r, off) in zip(got.split((Hq, H, H), 1), want):
        assert attention_ref.outside(t, r, off, dtype) == 0
