"""A layer's operators in a run, as a decoder over quantized weights uses them: a prompt, then token by token,
eagerly and as a replayed graph, each stage against float64 of what the stage before left."""
import pytest
import torch

import layer_refs as R
from layer_refs import F64, U, tensor

pytestmark = pytest.mark.gpu
E, NH, KV, D, BT, S, PER = 256, 4, 2, 64, 16, 3, 6
EPS = 1e-5


class Layer:
    """norm, q/k/v product, rotation, cache write, attention, output product, next norm with the residual."""

    def __init__(self, mi, ctx, T):
        self.mi, self.ctx, self.T = mi, ctx, T
        g = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        self.w1, self.w2 = 1 + 0.2 * r(E), 1 + 0.2 * r(E)
        self.qkv_w = self.weight(r((NH + 2 * KV) * D, E, std=0.06))
        self.out_w = self.weight(r(E, NH * D, std=0.06))
        M = S * T
        self.x = torch.zeros((M, E), device="cuda")
        self.h8 = torch.zeros((M, E // 32 * 34), dtype=torch.uint8, device="cuda")
        self.qkv = torch.zeros((S, T, NH + 2 * KV, D), device="cuda")
        self.a = torch.zeros((S, T, NH, D), device="cuda")
        self.o, self.y = torch.zeros((M, E), device="cuda"), torch.zeros((M, E), device="cuda")
        self.pos = torch.zeros((3, S, T), dtype=torch.int32, device="cuda")
        self.n_new = torch.zeros(S, dtype=torch.int32, device="cuda")

    def weight(self, w):
        rows = torch.zeros((w.shape[0], w.shape[1] // 32 * 34), dtype=torch.uint8, device="cuda")
        self.ctx.quantize_weights(self.mi.Q8_0, tensor(self.mi, w), rows.data_ptr())
        self.ctx.synchronize()
        return self.mi.from_torch(rows, self.mi.Q8_0, [w.shape[1], w.shape[0]])

    def step(self, d):
        mi, ctx, M = self.mi, self.ctx, S * self.T
        h8 = mi.from_torch(self.h8, mi.Q8_0, [E, M])
        ctx.rms_norm(tensor(mi, self.x), h8, EPS, w=self.w1.data_ptr())
        ctx.mul_mat(self.qkv_w, h8, tensor(mi, self.qkv.reshape(M, -1)))
        qk = self.qkv[:, :, :NH + KV]
        ctx.rope_multi(tensor(mi, qk), self.pos.data_ptr(), mi.rope_params(D, [8, 12, 12], pairs=mi.ROPE_HALVES), tensor(mi, qk))
        k, v = self.qkv[:, :, NH:NH + KV].transpose(1, 2), self.qkv[:, :, NH + KV:].transpose(1, 2)
        ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, k), tensor(mi, v), n_new=self.n_new.data_ptr())
        ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, self.qkv[:, :, :NH].transpose(1, 2)), tensor(mi, self.a), D ** -0.5,
                          n_q=self.n_new.data_ptr())
        ctx.mul_mat(self.out_w, tensor(mi, self.a.reshape(M, -1)), tensor(mi, self.o))
        ctx.rms_norm(tensor(mi, self.x), tensor(mi, self.y), EPS, add=tensor(mi, self.o), w=self.w2.data_ptr(), sum=tensor(mi, self.x))


def state(layer, d):
    return [t.clone() for t in (layer.x, layer.h8, layer.qkv, layer.a, layer.o, layer.y, d["k"], d["v"], d["ks"], d["vs"])]


def set_step(layer, d, n_kv, new, x):
    layer.x.copy_(x)
    layer.n_new.copy_(torch.tensor(new, dtype=torch.int32))
    d["n_kv"].copy_(torch.tensor(n_kv, dtype=torch.int32))
    at = torch.tensor(n_kv)[:, None] - torch.tensor(new)[:, None] + torch.arange(layer.T)
    layer.pos.copy_(torch.stack([at, at // 7, at % 7]).to(torch.int32))


def test_layer_against_float64(mi, ctx):
    """Every stage within its own operator's tolerance of the definition on what the stage before it left."""
    c = R.Cache(S, PER, KV, BT, D, seed=2)
    c.table[2, 5] = -1
    d = c.on_gpu(mi)
    n_kv = [0] * S
    for T, new in ((37, [37, 20, 5]), (1, [1, 1, 1]), (1, [1, 1, 1]), (5, [5, 1, 3]), (1, [1, 0, 1])):
        layer = Layer(mi, ctx, T)
        n_kv = [a + b for a, b in zip(n_kv, new)]
        x = torch.randn((S * T, E), generator=torch.Generator().manual_seed(sum(n_kv))).cuda()
        set_step(layer, d, n_kv, new, x)
        layer.step(d)
        ctx.synchronize()
        valid = torch.arange(T)[None] < torch.tensor(new)[:, None]
        # the cache holds what the rotated keys and the values of the product give
        got = layer.qkv.cpu()
        c.n_kv = torch.tensor(n_kv, dtype=torch.int32)
        c.write(got[:, :, NH:NH + KV].transpose(1, 2), got[:, :, NH + KV:].transpose(1, 2), new)
        assert torch.equal(d["k"].cpu(), c.k) and torch.equal(d["v"].cpu(), c.v)
        want, tol = c.attn(got[:, :, :NH], new, D ** -0.5, True, 0, True, True)
        assert ((layer.a.cpu().to(F64) - want).abs() <= tol)[valid].all()
        # the queries, from the F32 product of the norm's own 8-bit rows
        plain = torch.empty_like(layer.qkv)
        y = torch.empty((S * T, E), device="cuda")
        ctx.rms_norm(tensor(mi, x), tensor(mi, y), EPS, w=layer.w1.data_ptr())
        ctx.mul_mat(layer.qkv_w, tensor(mi, y), tensor(mi, plain.reshape(S * T, -1)))
        ctx.synchronize()
        turned = R.rope(plain[:, :, :NH + KV], R.angles(layer.pos, [8, 12, 12], D, 10000.0), True)
        both = plain[:, :, :NH + KV].abs().to(F64)
        both = both + both.roll(D // 2, -1)
        assert ((layer.qkv[:, :, :NH + KV].to(F64) - turned).abs() <= 6 * U * both).all()
        assert torch.equal(layer.qkv[:, :, NH + KV:], plain[:, :, NH + KV:])
        h = x + layer.o
        assert torch.equal(layer.x, h)
        ref = h.to(F64) / torch.sqrt(h.to(F64).square().mean(-1, keepdim=True) + EPS) * layer.w2.to(F64)
        assert ((layer.y.to(F64) - ref).abs() <= 8 * U * ref.abs()).all()


def test_layer_prompt_and_tokens_agree(mi, ctx):
    """A prompt at once and the same tokens one by one attend to nearly the same cache: blocks that grow token by token are
    rounded once more for each time their scale grew, half a step of the final scale at most each."""
    T = 2 * BT + 3
    k, v = (torch.randn((1, KV, T, D), generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2))
    caches = [R.Cache(1, PER, KV, BT, D, seed=4).on_gpu(mi) for _ in range(2)]
    caches[0]["n_kv"].fill_(T)
    ctx.kv_cache_write(caches[0]["cache"], caches[0]["seqs"], tensor(mi, k), tensor(mi, v))
    for t in range(T):
        caches[1]["n_kv"].fill_(t + 1)
        ctx.kv_cache_write(caches[1]["cache"], caches[1]["seqs"], tensor(mi, k[:, :, t:t + 1]), tensor(mi, v[:, :, t:t + 1]))
    ctx.synchronize()
    ids = caches[0]["table"][0, :3].long()
    assert torch.equal(caches[0]["ks"][ids], caches[1]["ks"][ids]) and torch.equal(caches[0]["vs"][ids], caches[1]["vs"][ids])
    a, b = (torch.empty((1, KV, T, D), device="cuda") for _ in range(2))
    ctx.kv_cache_read(caches[0]["cache"], caches[0]["seqs"], tensor(mi, a), None)
    ctx.kv_cache_read(caches[1]["cache"], caches[1]["seqs"], tensor(mi, b), None)
    ctx.synchronize()
    top = caches[0]["ks"][ids].T[:, torch.arange(T) // BT][None, :, :, None]
    assert ((a - k).abs() <= 0.5 * top * (1 + 4 * U) + 128 * U * top).all()
    assert ((b - k).abs() <= 0.5 * BT * top).all() and ((b - k).abs().mean() < 1.0 * top.mean())


def test_layer_as_a_graph(mi):
    """A token's step captured once and replayed, with eager work of the same context between (a larger product and a longer
    attention, which grow its workspace): every replay has the bits of the eager step."""
    stream = torch.cuda.Stream()
    ctx = mi.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            layer = Layer(mi, ctx, 1)
            base = R.Cache(S, 400, KV, BT, D, seed=5).fill([6000, 37, 900])
            d, start = base.on_gpu(mi), base.on_gpu(mi)
            x = torch.randn((S, E), generator=torch.Generator().manual_seed(3)).cuda()

            def reset():
                for n in ("k", "v", "ks", "vs"):
                    d[n].copy_(start[n])
                set_step(layer, d, [6001, 38, 901], [1, 1, 1], x)

            q = tensor(mi, layer.qkv[:, :, :NH].transpose(1, 2))
            ctx.reserve_workspace(max(ctx.kv_cache_attn_workspace_size(d["cache"], d["seqs"], q), 8 << 20))
            reset()
            layer.step(d)
            eager = state(layer, d)
            stream.synchronize()
            reset()
            graph = torch.cuda.CUDAGraph()
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                layer.step(d)
            big = R.Cache(64, 40, 2, 64, 64, seed=6).fill([2500] * 64).on_gpu(mi)
            bq, bo = torch.randn((64, 16, 64, 64), device="cuda"), torch.empty((64, 64, 16, 64), device="cuda")
            rows, y = torch.zeros((4096, 34 * 32), dtype=torch.uint8, device="cuda"), torch.randn((3000, 1024), device="cuda")
            r = torch.empty((3000, 4096), device="cuda")
            for i in range(5):
                reset()
                for t in (layer.h8, layer.qkv, layer.a, layer.o, layer.y):
                    t.fill_(1)
                graph.replay()
                stream.synchronize()
                for got, want in zip(state(layer, d), eager):
                    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)), i
                if i:
                    ctx.mul_mat(mi.from_torch(rows, mi.Q8_0, [1024, 4096]), mi.from_torch(y, mi.F32, [1024, 700 * i]),
                                mi.from_torch(r, mi.F32, [4096, 700 * i]))
                    ctx.kv_cache_attn(big["cache"], big["seqs"], tensor(mi, bq[:, :8 * i, :4 * i]), tensor(mi, bo[:, :4 * i, :8 * i]), 0.125)
                    stream.synchronize()
    finally:
        ctx.close()


def test_capture_needs_its_workspace(mi):
    """A captured call whose ranges need workspace that the context lacks is refused, with the way out, and the capture goes
    on; after mi355_reserve_workspace it is taken, and replays survive the workspace's replacement."""
    stream = torch.cuda.Stream()
    ctx = mi.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            d = R.Cache(1, 200, 1, 64, 64, seed=8).fill([12800]).on_gpu(mi)
            q, out, mark = torch.randn((1, 4, 1, 64), device="cuda"), torch.zeros((1, 1, 4, 64), device="cuda"), torch.zeros(8, device="cuda")
            need = ctx.kv_cache_attn_workspace_size(d["cache"], d["seqs"], tensor(mi, q))
            assert need > 0
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                mark.add_(1)
                with pytest.raises(mi.Mi355Error, match="mi355_reserve_workspace"):
                    ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, out), 0.125)
            graph.replay()
            stream.synchronize()
            assert (mark == 1).all() and not out.any()
            ctx.reserve_workspace(need)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, out), 0.125)
            eager = torch.zeros_like(out)
            ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, eager), 0.125)
            for i in range(4):
                out.zero_()
                graph.replay()
                stream.synchronize()
                assert eager.any() and torch.equal(out, eager), i
                ctx.reserve_workspace(need + (i << 22))
    finally:
        ctx.close()


def test_graph_on_another_stream(mi):
    """A graph captured behind work that is still on its context's stream, and replayed at once on another one: what the
    reservation made is there."""
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    ctx, plain = mi.Context(0, stream.cuda_stream), mi.Context(0)
    try:
        d = R.Cache(1, 200, 1, 64, 64, seed=8).fill([12800]).on_gpu(mi)
        q, out, eager = torch.randn((1, 4, 1, 64), device="cuda"), torch.zeros((1, 1, 4, 64), device="cuda"), torch.zeros((1, 1, 4, 64), device="cuda")
        busy = torch.randn((4096, 4096), device="cuda")
        plain.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, eager), 0.125)
        plain.synchronize()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            work = busy @ busy  # (warms the product up)
            stream.synchronize()
            for _ in range(20):
                work = busy @ work
            ctx.reserve_workspace(ctx.kv_cache_attn_workspace_size(d["cache"], d["seqs"], tensor(mi, q)))
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, out), 0.125)
            graph.capture_end()
        with torch.cuda.stream(other):
            for i in range(4):
                graph.replay()
                other.synchronize()
                assert eager.any() and torch.equal(out, eager), i
                out.zero_()
                other.synchronize()
        stream.synchronize()
    finally:
        ctx.close()
        plain.close()


def test_two_contexts_at_once(mi):
    """Two streams with a context each, launched together."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [mi.Context(0, s.cuda_stream) for s in streams]
    try:
        c = R.Cache(4, 100, 2, 32, 128, seed=7).fill([3200, 3000, 500, 1])
        d = c.on_gpu(mi)
        q = torch.randn((2, 4, 8, 1, 128), device="cuda").half()
        out = torch.zeros((2, 5, 4, 1, 8, 128), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        for i in range(5):
            for j in (0, 1):
                ctxs[j].kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q[j]), tensor(mi, out[j, i]), 0.09)
        for x in ctxs:
            x.synchronize()
        for j in (0, 1):
            want, tol = c.attn(q[j].transpose(1, 2).cpu(), [1] * 4, 0.09, True, 0, False, False)
            for i in range(5):
                assert ((out[j, i].cpu().to(F64) - want).abs() <= tol).all()
                assert torch.equal(out[j, i], out[j, 0])
    finally:
        for x in ctxs:
            x.close()
