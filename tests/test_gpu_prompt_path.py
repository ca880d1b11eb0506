"""The attention of prompts, its gradients, draft trees and step tables run together, as a program
uses them: a request from its prompt to its drafts, a training step, graphs, streams, threads, large
tensors."""
import threading

import pytest
import torch

from tests import attention_ref, prompt_ref as ref
from tests.gpu_util import note
from tests.test_gpu_prompt_attention import cumulative, make

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn


class Cache:
    """One layer's cache, its page table and the steps that go through it."""

    def __init__(self, pkg, gpu, B, Hq, H, D, page=16, pages=64, width=14):
        self.pkg, self.gpu, self.page, self.dims = pkg, gpu, page, (Hq, H, D)
        self.k, self.ks = pkg.empty_kv_cache(pages, H, page, D, device=gpu)
        self.v, self.vs = pkg.empty_kv_cache(pages, H, page, D, device=gpu)
        for t in (self.k, self.ks, self.v, self.vs):
            t.view(torch.uint8).fill_(0x7F)                # NaN, and a scale that spoils what it touches
        g = torch.Generator().manual_seed(3)
        self.free = torch.randperm(pages, generator=g, dtype=torch.int32).to(gpu)
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=gpu)
        self.lens = torch.zeros(B, dtype=torch.int32, device=gpu)
        self.used = None
        self.w = torch.ones(D, dtype=BF16, device=gpu)
        self.cos, self.sin = (t.to(gpu) for t in attention_ref.tables(512, D))

    def step(self, qkv, new, ahead=None):
        """Positions, slots and lengths of `new` tokens of each sequence; q and k rotated, k and v written.
        ahead: positions in place of the tables', past each sequence's context."""
        Hq, H, D = self.dims
        cu, cu_k, self.lens, pos, slots, self.used = self.pkg.batch_tables(
            self.lens, new, self.free, self.table, self.page, qkv.shape[0], free_start=self.used)
        pos = pos if ahead is None else ahead
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        q, k = self.pkg.qk_norm_rope(q, k, self.w, self.w, self.cos, self.sin, pos)
        self.pkg.kv_cache_write(k, v, slots, self.k, self.v, self.ks, self.vs)
        return q, k, v, cu, cu_k

    def read(self, cu_k, rows):
        Hq, H, D = self.dims
        out = [torch.full((rows, H, D), 9.0, dtype=BF16, device=self.gpu) for _ in range(2)]
        return self.pkg.kv_cache_read(self.k, self.v, self.ks, self.vs, self.table, cu_k, *out)


def tokens(gpu, seed, T, Hq, H, D):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, Hq + 2 * H, D, generator=g).to(BF16).to(gpu)


def close(out, q, k, v, cu, cu_k, scale):
    o, off, _, _ = ref.forward(q.cpu(), k.cpu(), v.cpu(), cu.cpu(), scale, None if cu_k is None else cu_k.cpu())
    assert attention_ref.outside(out, o, off, q.dtype) == 0


def test_a_request_from_prompt_to_drafts(pkg, gpu):
    B, Hq, H, D, scale = 3, 4, 2, 64, 0.125
    c = Cache(pkg, gpu, B, Hq, H, D)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    note("prompts")
    T = 40 + 7 + 100
    q, k, v, cu, _ = c.step(tokens(gpu, 1, T, Hq, H, D), i32(40, 7, 100))
    assert cu.tolist() == [0, 40, 47, 147] and c.lens.tolist() == [40, 7, 100]
    close(pkg.prompt_attention(q, k, v, cu, scale), q, k, v, cu, None, scale)
    codes, stored = attention_ref.quantize(k.cpu(), D, FP8, False)
    first = (codes.float() * stored[..., :, None].flatten(-2)).to(BF16)

    note("a second chunk over the gathered context, with rows of padding")
    q, k, v, cu, cu_k = c.step(tokens(gpu, 2, 20, Hq, H, D), i32(5, 0, 9))
    kk, vv = c.read(cu_k, int(cu_k[-1]) + 3)
    assert torch.equal(kk[:40].cpu(), first[:40]) and torch.equal(kk[52:152].cpu(), first[47:])
    out = pkg.prompt_attention(q, kk, vv, cu, scale, cu_seqlens_k=cu_k)
    assert bool((out[14:] == 0).all()) and bool((kk[int(cu_k[-1]):] == 9.0).all())
    close(out[:14], q[:14], kk[:int(cu_k[-1])], vv[:int(cu_k[-1])], cu, cu_k, scale)

    note("drafts")
    S = 6
    parents = [-1, 0, 0, 1, 2, -1]
    mask, depth = torch.zeros(S, S, dtype=torch.bool), []
    for s, p in enumerate(parents):
        if p >= 0:
            mask[s] = mask[p]
        mask[s, s] = True
        depth.append(0 if p < 0 else depth[p] + 1)
    ahead = (c.lens[:, None] + i32(*depth)).flatten()
    q, k, v, cu, _ = c.step(tokens(gpu, 3, B * S, Hq, H, D), i32(S, S, S), ahead)
    out = pkg.paged_tree_attention(q.view(B, S, Hq, D), c.k, c.v, c.ks, c.vs, c.table, c.lens,
                                   mask.to(gpu), scale)
    live = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool)
    for b in range(B):
        for i in range(int(c.lens[b])):
            live[int(c.table[b, i // c.page]), i % c.page] = True
    kc, ks, vc, vs = (t.cpu().clone() for t in (c.k, c.ks, c.v, c.vs))
    for codes, s in ((kc, ks), (vc, vs)):
        dead = ~live[:, None, :].expand(codes.shape[:3])
        codes.view(torch.uint8)[dead] = 0
        s[:, :, 0][dead] = 0
    r, bound = ref.tree(q.view(B, S, Hq, D).cpu(), kc, vc, ks, vs, c.table.cpu(), c.lens.cpu(), mask, scale)
    assert attention_ref.outside(out, r, bound, BF16) == 0
    assert int(c.used) == sum(-(-n // c.page) for n in c.lens.tolist())


class PromptAttention(torch.autograd.Function):
    """What a training program makes of the two directions."""

    @staticmethod
    def forward(ctx, pkg, q, k, v, cu, scale):
        out, lse = pkg.prompt_attention(q, k, v, cu, scale, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, cu)
        ctx.pkg, ctx.scale = pkg, scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, cu = ctx.saved_tensors
        return None, *ctx.pkg.prompt_attention_bwd(dout.contiguous(), q, k, v, out, lse, cu, ctx.scale), None, None


def test_a_training_step_with_autograd(pkg, gpu):
    note("autograd")
    q, k, v, do, cu, _ = make(4, [90, 30, 0, 200], None, 4, 2, 64)
    leaves = [t.to(gpu).requires_grad_() for t in (q, k, v)]
    out = PromptAttention.apply(pkg, *leaves, cu.to(gpu), 0.125)
    for _ in range(2):                                     # the graph of one forward, used twice
        grads = torch.autograd.grad(out, leaves, do.to(gpu), retain_graph=True)
    _, lse = pkg.prompt_attention(*[t.detach() for t in leaves], cu.to(gpu), 0.125, return_lse=True)
    want = ref.backward(do, q, k, v, out.detach().cpu(), lse.cpu(), cu, 0.125)
    for g, (r, off) in zip(grads, want):
        assert attention_ref.outside(g, r, off, BF16) == 0
    # The mean's gradient is one number for all rows: an expanded tensor.
    loss = PromptAttention.apply(pkg, *leaves, cu.to(gpu), 0.125).float().sum()
    loss.backward()
    ones = torch.ones_like(do)
    for t, (r, off) in zip(leaves, ref.backward(ones, q, k, v, out.detach().cpu(), lse.cpu(), cu, 0.125)):
        assert attention_ref.outside(t.grad, r, off, BF16) == 0


def test_captured_steps_replay(pkg, gpu):
    """A whole step of fixed room captured once, replayed with other lengths and tokens."""
    note("captured steps")
    B, Hq, H, D, rows, S = 4, 4, 2, 128, 300, 8
    g = torch.Generator().manual_seed(5)
    make_cache = lambda: Cache(pkg, gpu, B, Hq, H, D, pages=200, width=40)
    new = torch.zeros(B, dtype=torch.int32, device=gpu)
    context = torch.zeros(B, dtype=torch.int32, device=gpu)
    qkv = tokens(gpu, 6, rows, Hq, H, D)
    drafts = tokens(gpu, 7, B * S, Hq, H, D)[:, :Hq].contiguous().view(B, S, Hq, D)
    mask = torch.ones(B, S, S, dtype=torch.bool, device=gpu).tril()

    def call(c):
        c.lens, c.used = context, None
        q, k, v, cu, cu_k = c.step(qkv, new)
        out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
        grads = pkg.prompt_attention_bwd(q, q, k, v, out, lse, cu, 0.1)
        kk, vv = c.read(cu_k, 900)
        late = pkg.prompt_attention(q, kk, vv, cu, 0.1, cu_seqlens_k=cu_k)
        tree = pkg.paged_tree_attention(drafts, c.k, c.v, c.ks, c.vs, c.table, c.lens, mask, 0.1)
        return [out, lse, *grads, kk, vv, late, tree, cu, cu_k, c.lens, c.used, c.table]

    a, b = make_cache(), make_cache()
    side = torch.cuda.Stream(device=gpu)
    new.copy_(torch.tensor([100, 3, 50, 20], dtype=torch.int32))
    torch.cuda.synchronize(gpu)
    with torch.cuda.stream(side):
        call(a)
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call(a)
    for n, ctx in (([100, 3, 50, 20], [0] * 4), ([1, 1, 1, 1], [100, 3, 50, 20]), ([0, 130, 0, 9], [0, 5, 16, 31]),
                   ([75] * 4, [64, 0, 7, 100]), ([0] * 4, [0] * 4)):
        for c in (a, b):
            c.table.fill_(-1)
            pages = torch.arange(100, 200, dtype=torch.int32, device=gpu).view(4, 25)
            for i, t in enumerate(ctx):
                c.table[i, :-(-t // 16)] = pages[i, :-(-t // 16)]
            for t in (c.k, c.v):
                t.view(torch.uint8).fill_(0x30)
            for t in (c.ks, c.vs):
                t.fill_(0.5)
        new.copy_(torch.tensor(n, dtype=torch.int32))
        context.copy_(torch.tensor(ctx, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        torch.cuda.synchronize(gpu)
        graph.replay()
        torch.cuda.synchronize(gpu)
        want = call(b)
        for i, (x, y) in enumerate(zip(got, want)):
            assert torch.equal(x, y), (n, i)


@pytest.mark.parametrize("lens,H", [([700, 40, 333], 2), ([60, 9], 2), ([4000], 1)])
def test_captured_gradients_replay(pkg, gpu, lens, H):
    """Workspaces of parts and of both passes are the graph's own."""
    note(f"captured gradients {lens}")
    g = torch.Generator().manual_seed(8)
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in make(8, lens, None, 4 * H, H, 128)]
    side = torch.cuda.Stream(device=gpu)

    def call():
        out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
        return [out, lse, *pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1)]

    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for _ in range(4):
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        torch.cuda.synchronize(gpu)
        graph.replay()
        torch.cuda.synchronize(gpu)
        assert all(torch.equal(a, b) for a, b in zip(got, call()))


def test_streams_and_threads(pkg, gpu):
    """Calls at once from two threads, each on a stream of its own."""
    note("two threads")
    cases = [make(s, [300, 70, 0, 129], None, 8, 2, 128) for s in (1, 2)]
    cases = [[None if t is None else t.to(gpu) for t in c] for c in cases]

    def call(c):
        q, k, v, do, cu, _ = c
        out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
        lens = torch.tensor([3, 40], dtype=torch.int64, device=gpu)
        table = torch.full((2, 5), -1, dtype=torch.int32, device=gpu)
        tables = pkg.batch_tables(lens, lens, torch.arange(20, dtype=torch.int32, device=gpu), table, 16, 50)
        return [out, lse, *pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1), *tables, table]

    wants = [call(c) for c in cases]
    torch.cuda.synchronize(gpu)
    got, errors = {}, []

    def work(i):
        try:
            torch.cuda.set_device(gpu)
            with torch.cuda.stream(torch.cuda.Stream(device=gpu)):
                got[i] = [call(cases[i]) for _ in range(10)]
                torch.cuda.current_stream(gpu).synchronize()
        except Exception as e:                             # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i, want in enumerate(wants):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def far_view(x, width, start):
    buf = torch.empty(x.shape[0], width, dtype=x.dtype, device=x.device)
    v = buf[:, start:start + x.shape[1] * x.shape[2]].view(x.shape)
    v.copy_(x)
    return v


@pytest.mark.parametrize("T,width", [(20000, 131072), (140, (1 << 24) - 8)])
def test_views_of_more_than_4_gib(pkg, gpu, T, width):
    """Token strides up to the largest: the same rows in small tensors give the same bits."""
    note(f"views of {T} rows of {width}")
    if torch.cuda.mem_get_info(gpu)[0] < 60 << 30:
        pytest.skip("needs 60 GiB")
    lens = [T - 37, 30]
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in make(9, lens, None, 2, 1, 64, spare=7)]
    out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
    want = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1)
    fk, fv, fq, fdo = (far_view(t, width, width - 128) for t in (k, v, q, do))
    assert (T - 1) * fk.stride(0) > 1 << 31
    o, s = pkg.prompt_attention(fq, fk, fv, cu, 0.1, return_lse=True)
    assert torch.equal(o[:T - 7], out[:T - 7]) and torch.equal(s, lse)
    del fv, o
    fdk, fdq = far_view(torch.zeros_like(k), width, 64), far_view(torch.zeros_like(q), width, 0)
    pkg.prompt_attention_bwd(fdo, fq, fk, v, out, lse, cu, 0.1, dq=fdq, dk=fdk)
    assert torch.equal(fdq[:T - 7], want[0][:T - 7]) and torch.equal(fdk[:T - 7], want[1][:T - 7])
    del fk, fq, fdo, fdk, fdq
    torch.cuda.empty_cache()


def test_many_sequences(pkg, gpu):
    """More sequences than lanes, and a slot table of thousands: every row is somebody's."""
    note("many sequences")
    for B in (65, 1000, 5000):
        lens = [(i * 7) % 5 for i in range(B)]
        made = make(B, lens, None, 2, 1, 64, spare=3)
        q, k, v, do, cu, _ = made
        out, lse = pkg.prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), cu.to(gpu), 0.1, return_lse=True)
        T = sum(lens)
        if B < 1000:
            close(out[:T], q[:T], k[:T], v[:T], cu, None, 0.1)
        # One by one, the same.
        some = [i for i in range(0, B, max(1, B // 40)) if lens[i]]
        for i in some:
            r = slice(int(cu[i]), int(cu[i + 1]))
            one = pkg.prompt_attention(q[r].to(gpu), k[r].to(gpu), v[r].to(gpu), cumulative([lens[i]]).to(gpu), 0.1)
            assert torch.equal(one, out[r]), i
        grads = pkg.prompt_attention_bwd(do.to(gpu), q.to(gpu), k.to(gpu), v.to(gpu), out, lse, cu.to(gpu), 0.1)
        assert all(bool(torch.isfinite(t).all()) for t in grads)
