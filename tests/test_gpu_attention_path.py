"""The attention side run as a decoder layer runs it: the quantizer's codes through the fp8 GEMM to
q, k and v, norm and rotation, the cache's write, attention over it step by step, and its read; in
captured graphs, on streams of their own and from two threads."""
import threading

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


class Layer:
    """One layer's attention with H cache heads, G query heads each, in pages of 16."""

    def __init__(self, pkg, dev, B, H=2, G=4, D=64, width=8, prefix=0, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.pkg, self.dev, self.B, self.H, self.Hq, self.D, self.prefix = pkg, dev, B, H, H * G, D, prefix
        self.hidden = 256
        n = (self.Hq + 2 * H) * D
        w = 0.1 * torch.randn(n, self.hidden, generator=g)
        self.w, self.ws = w.to(FP8).to(dev), torch.full((-(-n // 128), 2), 1.0, device=dev)
        self.norm = torch.ones(self.hidden, dtype=BF16, device=dev)
        self.qw, self.kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(BF16).to(dev) for _ in range(2))
        self.cos, self.sin = (t.to(dev) for t in ref.tables(512, D))
        pages = B * width + 8
        order = torch.randperm(pages, generator=g).int()
        self.table = order[:B * width].view(B, width).contiguous().to(dev)
        self.prefix_pages = order[B * width:].contiguous().to(dev) if prefix else None
        self.kc, self.ks = pkg.empty_kv_cache(pages, H, 16, D, device=dev)
        self.vc, self.vs = pkg.empty_kv_cache(pages, H, 16, D, device=dev)
        for c, s in ((self.kc, self.ks), (self.vc, self.vs)):
            c.view(torch.uint8).fill_(0x7F)               # NaN until written
            s.fill_(float("nan"))
        if prefix:
            x = torch.randn(prefix, 2 * H, D, generator=g).to(BF16).to(dev)
            at = torch.arange(prefix, device=dev)
            slots = self.prefix_pages.long()[at // 16] * 16 + at % 16
            pkg.kv_cache_write(x[:, :H], x[:, H:], slots, self.kc, self.vc, self.ks, self.vs)

    def step(self, x, residual, lens):
        """x, residual [B, hidden], the newest token of each sequence; lens: tokens so far with it."""
        p, B = self.pkg, self.B
        residual, q8, scale = p.fused_add_rmsnorm_group_quant_fn(x, residual, self.norm, 1e-6, 128, FP8,
                                                                 scale_col_major=True)
        qkv = p.fp8_block_scaled_gemm(q8, scale, self.w, self.ws).view(B, -1, self.D)
        q, k, v = qkv.split((self.Hq, self.H, self.H), 1)
        at = (lens - 1).long()
        q, k = p.qk_norm_rope(q, k, self.qw, self.kw, self.cos, self.sin, at + self.prefix)
        slots = self.table.gather(1, (at // 16)[:, None])[:, 0].long() * 16 + at % 16
        p.kv_cache_write(k, v, slots, self.kc, self.vc, self.ks, self.vs)
        out = p.paged_attention(q[:, None], self.kc, self.vc, self.ks, self.vs, self.table, lens,
                                self.D ** -0.5, prefix_pages=self.prefix_pages, prefix_len=self.prefix)
        return out[:, 0], q, k, v, slots

    def want(self, q, lens):
        """The attention in 64 bits over what the cache holds."""
        kc, ks, vc, vs = (t.cpu().clone() for t in (self.kc, self.ks, self.vc, self.vs))
        for c, s in ((kc, ks), (vc, vs)):
            bad = torch.isnan(s[:, :, 0])
            c.view(torch.uint8)[bad] = 0
            s[:, :, 0][bad] = 0.0
        return ref.attention(q[:, None].cpu(), kc, vc, ks, vs, self.table.cpu(), lens.cpu(), self.D ** -0.5,
                             None if self.prefix_pages is None else self.prefix_pages.cpu(), self.prefix)


@pytest.mark.parametrize("prefix", [0, 37])
def test_decode_steps(pkg, gpu, prefix):
    B, steps = 3, 20
    note(f"attention path prefix {prefix}")
    layer = Layer(pkg, gpu, B, prefix=prefix)
    g = torch.Generator().manual_seed(2)
    residual = torch.zeros(B, layer.hidden, dtype=BF16, device=gpu)
    start = torch.tensor([0, 5, 30], dtype=torch.int32, device=gpu)
    # What the sequences hold before: written as one ragged chunk.
    n = int(start.sum())
    old = torch.randn(n, 2 * layer.H, layer.D, generator=g).to(BF16).to(gpu)
    own = torch.cat([torch.arange(int(c)) for c in start.tolist()]).to(gpu)
    seq = torch.repeat_interleave(torch.arange(B), start.cpu().long()).to(gpu)
    slots = layer.table[seq, own // 16].long() * 16 + own % 16
    pkg.kv_cache_write(old[:, :layer.H], old[:, layer.H:], slots, layer.kc, layer.vc, layer.ks, layer.vs)
    kept = []
    for i in range(steps):
        x = torch.randn(B, layer.hidden, generator=g).to(BF16).to(gpu)
        lens = start + i + 1
        out, q, k, v, at = layer.step(x, residual, lens)
        kept.append((at, k.clone(), v.clone()))
        r, bound = layer.want(q, lens)
        assert ref.outside(out[:, None], r, bound, BF16) == 0, i
    # What was written reads back as its codes and scales say.
    lens = start + steps
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=gpu), lens.cumsum(0, dtype=torch.int32)])
    ko, vo = (torch.empty(int(cu[-1]), layer.H, layer.D, dtype=torch.float32, device=gpu) for _ in range(2))
    pkg.kv_cache_read(layer.kc, layer.vc, layer.ks, layer.vs, layer.table, cu, ko, vo)
    for i, (at, k, v) in enumerate(kept):
        for got, x in ((ko, k), (vo, v)):
            codes, scales = ref.quantize(x.cpu(), layer.D, FP8, False)
            want = codes.float() * scales
            rows = (cu[:B] + start + i).cpu().long()
            assert torch.equal(got.cpu()[rows], want)


def test_captured_steps(pkg, gpu):
    """One step of the layer in a graph: every replay, with eager steps between, equals an eager step
    of a second layer with the same weights."""
    B = 4
    note("attention path captured")
    a, b = (Layer(pkg, gpu, B, prefix=20, seed=3) for _ in range(2))
    g = torch.Generator().manual_seed(5)
    x = torch.zeros(B, a.hidden, dtype=BF16, device=gpu)
    residual = torch.zeros_like(x)
    lens = torch.ones(B, dtype=torch.int32, device=gpu)
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        a.step(x, residual, lens)
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = a.step(x, residual, lens)[0]
    for i in range(6):
        x.copy_(torch.randn(B, a.hidden, generator=g).to(BF16))
        lens.fill_(i + 1)
        torch.cuda.synchronize(gpu)
        graph.replay()
        torch.cuda.synchronize(gpu)
        want = b.step(x, residual, lens)[0]
        torch.cuda.synchronize(gpu)
        assert torch.equal(out, want), i
        for s, t in ((a.kc, b.kc), (a.vc, b.vc), (a.ks, b.ks), (a.vs, b.vs)):
            # slots not written yet hold NaN in both
            assert torch.equal(s.view(torch.uint8) if s.dtype == FP8 else s.view(torch.int32),
                               t.view(torch.uint8) if t.dtype == FP8 else t.view(torch.int32))


def test_captured_backward_and_shares(pkg, gpu):
    """The gradients, and attention in shares worked out on the device, replayed with other inputs."""
    note("backward and shares captured")
    from tests.test_gpu_paged_attention import make
    from tests.test_gpu_attention_schedule import widened
    g = torch.Generator().manual_seed(6)
    T, Hq, Hk, D = 300, 8, 2, 128
    dy = torch.randn(T, Hq + Hk, D, generator=g).to(BF16).to(gpu)
    x = torch.randn(T, Hq + Hk, D, generator=g).to(BF16).to(gpu)
    w = torch.ones(D, dtype=BF16, device=gpu)
    cos, sin = (t.to(gpu) for t in ref.tables(512, D))
    pos = torch.arange(T, device=gpu)
    q, caches, table, lens, _ = widened(make(2, [900, 40, 333], 1, 8, 2, 128, 16), 128 * 900, 16)
    (kc, ks), (vc, vs) = [(c.to(gpu), s.to(gpu)) for c, s in caches]
    q, table, lens = q.to(gpu), table.to(gpu), lens.to(gpu)

    def call():
        return (*pkg.qk_norm_rope_bwd(dy[:, :Hq], dy[:, Hq:], x[:, :Hq], x[:, Hq:], w, w, cos, sin, pos),
                pkg.paged_attention(q, kc, vc, ks, vs, table, lens, D ** -0.5))

    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for new in ([900, 40, 333], [1, 0, 2], [128, 40, 300], [900, 40, 0]):
        dy.copy_(torch.randn(dy.shape, generator=g).to(BF16))
        q.copy_(torch.randn(q.shape, generator=g).to(BF16))
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize(gpu)
        graph.replay()
        torch.cuda.synchronize(gpu)
        for a, b in zip(got, call()):
            assert torch.equal(a, b), new


def test_two_threads_on_streams_of_their_own(pkg, gpu):
    note("attention path, two threads")
    wants = []
    for seed in (1, 2):
        layer = Layer(pkg, gpu, 5, seed=seed)
        g = torch.Generator().manual_seed(seed)
        xs = [torch.randn(5, layer.hidden, generator=g).to(BF16).to(gpu) for _ in range(15)]
        res = torch.zeros_like(xs[0])
        wants.append((seed, xs, [layer.step(x, res, torch.full((5,), i + 1, dtype=torch.int32, device=gpu))[0]
                                 for i, x in enumerate(xs)]))
    torch.cuda.synchronize(gpu)
    got, errors = {}, []

    def work(seed, xs):
        try:
            torch.cuda.set_device(gpu)
            with torch.cuda.stream(torch.cuda.Stream(device=gpu)):
                layer = Layer(pkg, gpu, 5, seed=seed)
                res = torch.zeros_like(xs[0])
                outs = [layer.step(x, res, torch.full((5,), i + 1, dtype=torch.int32, device=gpu))[0]
                        for i, x in enumerate(xs)]
                torch.cuda.current_stream(gpu).synchronize()
            got[seed] = outs
        except Exception as e:                             # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s, xs)) for s, xs, _ in wants]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for seed, _, want in wants:
        assert all(torch.equal(a, b) for a, b in zip(got[seed], want))
