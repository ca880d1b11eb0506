"""The torch.autograd.Function that INTEGRATION.md shows for qk_norm_rope: its gradients are those of
qk_norm_rope_bwd, bit for bit, and the formula's; the operator alone records nothing."""
import re
from pathlib import Path

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu


def shown(pkg):
    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    block, = [b for b in re.findall(r"```python\n(.*?)```", text, flags=re.S) if "autograd.Function" in b]
    ns = {"torch": torch, "fagq": pkg}
    exec(compile(block, "INTEGRATION.md", "exec"), ns)
    return ns["QkNormRope"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_through_autograd(pkg, gpu, dtype):
    note(f"rope through autograd {dtype}")
    T, Hq, Hk, D, R = 37, 6, 2, 64, 32
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(T, Hq + Hk, D, generator=g).to(dtype)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]
    dy = torch.randn(T, Hq + Hk, D, generator=g).to(dtype)
    cos, sin = ref.tables(64, R)
    pos = torch.randint(0, 64, (T,), generator=g)
    x = qkv.to(gpu).requires_grad_()
    ws = [t.to(gpu).requires_grad_() for t in w]
    rest = cos.to(gpu), sin.to(gpu), pos.to(gpu)
    assert not any(t.requires_grad for t in pkg.qk_norm_rope(x[:, :Hq], x[:, Hq:], *ws, *rest))
    y = shown(pkg).apply(x[:, :Hq], x[:, Hq:], *ws, *rest, 1e-6)
    d = dy.to(gpu)
    got = torch.autograd.grad(y, [x, *ws], [d[:, :Hq], d[:, Hq:]])
    own = pkg.qk_norm_rope_bwd(d[:, :Hq].contiguous(), d[:, Hq:].contiguous(), x.detach()[:, :Hq],
                               x.detach()[:, Hq:], *[t.detach() for t in ws], *rest, 1e-6)
    assert torch.equal(got[0], torch.cat(own[:2], 1))
    assert torch.equal(got[1], own[2].to(dtype)) and torch.equal(got[2], own[3].to(dtype))
    for i, cut in enumerate((slice(0, Hq), slice(Hq, None))):
        dx, bx, dw, bw = ref.rope_bwd(dy[:, cut], qkv[:, cut], w[i], cos, sin, pos, 1e-6, False)
        assert ref.outside(got[0][:, cut], dx, bx, dtype) == 0
        assert ref.outside(got[1 + i], dw, bw, dtype) == 0
