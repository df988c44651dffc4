"""The operators of a layer with a 4-bit cache in a run, as a decoder or a video's memory uses them: a prompt, then token by
token, then back to its budget, eagerly and as replayed graphs, each stage against float64 of what the stage before left."""
import math

import pytest
import torch

import layer_refs as R
import layer4_refs as R4
from layer_refs import F64, U, tensor
from test_gpu_layer4_ops import qk_close, same_bits, same_cache

pytestmark = pytest.mark.gpu
F16, F32, I32 = torch.float16, torch.float32, torch.int32
E, NH, KV, D, BT, S, PER = 256, 4, 2, 64, 16, 3, 6
EPS, KEEP, FIRST, RECENT = 1e-5, 40, 2, 8
SECTIONS = [8, 12, 12]


class Layer:
    """norm, q/k/v product, norms and rotation of q and k, cache write, attention, its weights' sums; and the eviction."""

    def __init__(self, mi, ctx, T):
        self.mi, self.ctx, self.T = mi, ctx, T
        g = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        self.w, self.q_w, self.k_w = 1 + 0.2 * r(E), 1.5 + 0.2 * r(D), 1.5 + 0.2 * r(D)
        rows = torch.zeros(((NH + 2 * KV) * D, E // 32 * 34), dtype=torch.uint8, device="cuda")
        ctx.quantize_weights(mi.Q8_0, tensor(mi, r((NH + 2 * KV) * D, E, std=0.06)), rows.data_ptr())
        self.qkv_w = mi.from_torch(rows, mi.Q8_0, [E, (NH + 2 * KV) * D])
        z = lambda *s, dtype=F32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        self.x, self.h8, self.qkv = z(S * T, E), z(S * T, E // 32 * 34, dtype=torch.uint8), z(S, T, NH + 2 * KV, D)
        self.q, self.k, self.v = z(S, T, NH, D, dtype=F16), z(S, T, KV, D, dtype=F16), z(S, T, KV, D, dtype=F16)
        self.a, self.lse = z(S, T, NH, D), z(S, T, NH)
        self.sums, self.sums_out = z(S, KV, PER * BT), z(S, KV, PER * BT)
        self.kept, self.n_out = z(S, KV, KEEP, dtype=I32), z(S, dtype=I32)
        self.pos, self.n_new = z(3, S, T, dtype=I32), z(S, dtype=I32)
        ctx.synchronize()

    def step(self, d):
        mi, ctx, M = self.mi, self.ctx, S * self.T
        t = lambda x: tensor(mi, x)  # noqa: E731
        h8 = mi.from_torch(self.h8, mi.Q8_0, [E, M])
        ctx.rms_norm(t(self.x), h8, EPS, w=self.w.data_ptr())
        ctx.mul_mat(self.qkv_w, h8, t(self.qkv.reshape(M, -1)))
        ctx.qk_norm_rope(t(self.qkv[:, :, :NH]), t(self.qkv[:, :, NH:NH + KV]), EPS, self.pos.data_ptr(),
                         mi.rope_params(D, SECTIONS, pairs=mi.ROPE_HALVES), t(self.q), t(self.k), q_w=self.q_w.data_ptr(), k_w=self.k_w.data_ptr())
        self.v.copy_(self.qkv[:, :, NH + KV:])
        ctx.kv_cache4_write(d["cache"], d["seqs"], t(self.k.transpose(1, 2)), t(self.v.transpose(1, 2)), n_new=self.n_new.data_ptr())
        q = t(self.q.transpose(1, 2))
        ctx.kv_cache4_attn(d["cache"], d["seqs"], q, t(self.a), D ** -0.5, n_q=self.n_new.data_ptr(), lse=self.lse.data_ptr())
        ctx.kv_cache4_weights(d["cache"], d["seqs"], q, self.lse.data_ptr(), self.sums.data_ptr(), D ** -0.5, n_q=self.n_new.data_ptr())

    def evict(self, d):
        self.ctx.kv_cache4_evict(d["cache"], d["seqs"], self.sums.data_ptr(), self.sums_out.data_ptr(), KEEP, self.kept.data_ptr(),
                                 self.n_out.data_ptr(), first=FIRST, recent=RECENT)


def at_step(layer, d, n_kv, seen, new, x):
    """seen: tokens that each sequence has seen in all, the new ones included: their positions go on behind an eviction."""
    layer.x.copy_(x)
    layer.n_new.copy_(torch.tensor(new, dtype=I32))
    d["n_kv"].copy_(torch.tensor(n_kv, dtype=I32))
    at = torch.tensor(seen)[:, None] - torch.tensor(new)[:, None] + torch.arange(layer.T)
    layer.pos.copy_(torch.stack([at, at // 7, at % 7]).to(I32))


def test_layer_against_float64(mi, ctx):
    c = R4.Cache4(S, PER, KV, BT, D, seed=2)
    c.table[2, 5] = -1
    d = c.on_gpu(mi)
    n_kv, seen = [0] * S, [0] * S
    sums = torch.zeros((S, KV, PER * BT))
    evicted = 0
    for T, new in ((45, [45, 20, 5]), (1, [1, 1, 1]), (5, [5, 1, 3]), (30, [3, 30, 30]), (1, [1, 0, 1]), (1, [1, 1, 1])):
        layer = Layer(mi, ctx, T)
        layer.sums.copy_(sums)
        n_kv, seen = [a + b for a, b in zip(n_kv, new)], [a + b for a, b in zip(seen, new)]
        x = torch.randn((S * T, E), generator=torch.Generator().manual_seed(sum(seen))).cuda()
        at_step(layer, d, n_kv, seen, new, x)
        layer.step(d)
        ctx.synchronize()
        valid = torch.arange(T)[None] < torch.tensor(new)[:, None]
        # the norms and turns of the product's rows, the rows themselves as the plain product gives them
        y, plain = torch.empty((S * T, E), device="cuda"), torch.empty_like(layer.qkv)
        ctx.rms_norm(tensor(mi, x), tensor(mi, y), EPS, w=layer.w.data_ptr())
        ctx.mul_mat(layer.qkv_w, tensor(mi, y), tensor(mi, plain.reshape(S * T, -1)))
        ctx.synchronize()
        assert torch.equal(plain, layer.qkv)
        ang = R.angles(layer.pos.cpu(), SECTIONS, D, 10000.0)
        qk_close(layer.q, plain[:, :, :NH].cpu(), layer.q_w.cpu(), EPS, ang, True)
        qk_close(layer.k, plain[:, :, NH:NH + KV].cpu(), layer.k_w.cpu(), EPS, ang, True)
        # the cache of these keys and values
        c.n_kv = torch.tensor(n_kv, dtype=I32)
        c.write(layer.k.cpu().transpose(1, 2).float(), layer.v.cpu().transpose(1, 2).float(), new)
        same_cache(c, d)
        # the attention and its weights
        q = layer.q.cpu()
        want, tol, lse, ltol = c.attn(q, new, D ** -0.5, True, 0, False, True)
        got, l = layer.a.cpu().to(F64), layer.lse.cpu()
        assert ((got - want).abs() <= tol)[valid].all() and ((l.to(F64) - lse).abs() <= ltol)[valid].all()
        add, wtol = c.weights(q, new, l, D ** -0.5, True, 0, False)
        now = layer.sums.cpu()
        assert ((now.to(F64) - (sums.to(F64) + add)).abs() <= wtol + U * (sums.to(F64) + add)).all()
        sums = now
        if max(n_kv) > KEEP:
            evicted += 1
            layer.evict(d)
            ctx.synchronize()
            out, kept = torch.zeros_like(sums), torch.zeros((S, KV, KEEP), dtype=I32)
            n_kv = c.evict(sums, [KEEP] * S, FIRST, RECENT, out, kept)
            assert layer.n_out.tolist() == n_kv and torch.equal(layer.sums_out.cpu(), out)
            for s in range(S):
                assert torch.equal(layer.kept.cpu()[s, :, :n_kv[s]], kept[s, :, :n_kv[s]])
            same_cache(c, d)
            sums = out
    assert evicted >= 4


def test_layer_as_graphs(mi):
    """A token's step and the eviction behind it, a graph each, replayed in turn with eager work of the same context between:
    every replay has the bits of the eager run."""
    stream = torch.cuda.Stream()
    ctx = mi.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            layer = Layer(mi, ctx, 1)
            base = R4.Cache4(S, PER, KV, BT, D, seed=5).fill([90, 37, 60])
            d, start = base.on_gpu(mi), base.on_gpu(mi)
            x = torch.randn((S, E), generator=torch.Generator().manual_seed(3)).cuda()
            sums = torch.rand((S, KV, PER * BT), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
            state = lambda: [t.clone() for t in (layer.q, layer.k, layer.a, layer.lse, layer.sums, layer.sums_out, layer.kept, layer.n_out,  # noqa: E731
                                                 d["k"], d["v"], d["ks"], d["vs"])]

            def reset():
                for n in ("k", "v", "ks", "vs"):
                    d[n].copy_(start[n])
                for t in (layer.q, layer.k, layer.a, layer.lse, layer.sums_out):
                    t.fill_(1)
                layer.kept.fill_(-1)
                layer.sums.copy_(sums)
                at_step(layer, d, [91, 38, 61], [91, 138, 61], [1, 1, 1], x)

            q = tensor(mi, layer.q.transpose(1, 2))
            ctx.reserve_workspace(max(ctx.kv_cache4_attn_workspace_size(d["cache"], d["seqs"], q),
                                      ctx.kv_cache4_weights_workspace_size(d["cache"], d["seqs"], q), 8 << 20))
            reset()
            layer.step(d)
            layer.evict(d)
            stream.synchronize()
            eager = state()
            graphs = []
            for f in (layer.step, layer.evict):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    f(d)
                graphs.append(g)
            big = R4.Cache4(2, 40, 2, 64, 64, seed=6).fill([2500, 900]).on_gpu(mi)
            bq, bo = torch.randn((2, 16, 300, 64), device="cuda"), torch.empty((2, 300, 16, 64), device="cuda")
            bl, bs = torch.empty((2, 300, 16), device="cuda"), torch.zeros((2, 2, 2560), device="cuda")
            for i in range(5):
                reset()
                graphs[0].replay()
                graphs[1].replay()
                stream.synchronize()
                for got, want in zip(state(), eager):
                    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)), i
                if i:  # (larger than the graphs' workspace)
                    ctx.kv_cache4_attn(big["cache"], big["seqs"], tensor(mi, bq), tensor(mi, bo), 0.125, causal=False, lse=bl.data_ptr())
                    ctx.kv_cache4_weights(big["cache"], big["seqs"], tensor(mi, bq), bl.data_ptr(), bs.data_ptr(), 0.125, causal=False)
                    stream.synchronize()
                    assert abs(float(bs.sum()) - i * 2 * 16 * 300) < 1.0
    finally:
        ctx.close()


def test_capture_needs_its_workspace(mi):
    """A captured call whose ranges or halves need workspace that the context lacks is refused, with the way out; after
    mi355_reserve_workspace it is taken, and replays survive the workspace's replacement."""
    stream = torch.cuda.Stream()
    ctx = mi.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            d = R4.Cache4(1, 100, 1, 64, 64, seed=8).fill([6400]).on_gpu(mi)
            for nq, heads in ((1, 4), (2000, 8)):
                q, out = torch.randn((1, heads, nq, 64), device="cuda"), torch.zeros((1, nq, heads, 64), device="cuda")
                lse, sums = torch.zeros((1, nq, heads), device="cuda"), torch.zeros((1, 1, 6400), device="cuda")
                need = max(ctx.kv_cache4_attn_workspace_size(d["cache"], d["seqs"], tensor(mi, q)),
                           ctx.kv_cache4_weights_workspace_size(d["cache"], d["seqs"], tensor(mi, q)))
                assert need > 0

                def both():
                    ctx.kv_cache4_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, out), 0.125, lse=lse.data_ptr())
                    ctx.kv_cache4_weights(d["cache"], d["seqs"], tensor(mi, q), lse.data_ptr(), sums.data_ptr(), 0.125)

                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    out.add_(1)
                    with pytest.raises(mi.Mi355Error, match="mi355_reserve_workspace"):
                        both()
                graph.replay()
                stream.synchronize()
                assert (out == 1).all()
                ctx.reserve_workspace(need)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    both()
                sums.zero_()
                both()
                stream.synchronize()
                want = [t.clone() for t in (out, lse, sums)]
                for i in range(4):
                    for t in (out, lse, sums):
                        t.zero_()
                    graph.replay()
                    stream.synchronize()
                    for got, w in zip((out, lse, sums), want):
                        assert torch.equal(got, w), (nq, i)
                    ctx.reserve_workspace(need + (i << 22))
                    stream.synchronize()
    finally:
        ctx.close()


def test_two_contexts_at_once(mi):
    """Two streams with a context each over one cache, launched together."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [mi.Context(0, s.cuda_stream) for s in streams]
    try:
        c = R4.Cache4(4, 40, 2, 32, 128, seed=7).fill([1200, 1000, 500, 1])
        d = c.on_gpu(mi)
        q = torch.randn((2, 4, 8, 1, 128), device="cuda").half()
        out = torch.zeros((2, 5, 4, 1, 8, 128), dtype=F16, device="cuda")
        torch.cuda.synchronize()
        for i in range(5):
            for j in (0, 1):
                ctxs[j].kv_cache4_attn(d["cache"], d["seqs"], tensor(mi, q[j]), tensor(mi, out[j, i]), 0.09)
        for x in ctxs:
            x.synchronize()
        for j in (0, 1):
            want, tol, _, _ = c.attn(q[j].transpose(1, 2).cpu(), [1] * 4, 0.09, True, 0, False, False)
            for i in range(5):
                assert ((out[j, i].cpu().to(F64) - want).abs() <= tol).all()
                assert torch.equal(out[j, i], out[j, 0])
    finally:
        for x in ctxs:
            x.close()


@pytest.mark.parametrize("D_", [64, 96, 128])
def test_nan_token_under_prompts(mi, ctx, D_):
    """Where the halves are made by a launch of their own a NaN token spoils the queries that see it and no others, whatever
    stands in the places behind the sequence's end."""
    n, nq, heads = 2000, 1900, 24
    c = R4.Cache4(2, 32, 4, 64, D_, seed=D_).fill([n, 1555])
    good = c.on_gpu(mi)
    bad = torch.ones((1, 4, D_))
    bad[0, 2, 5] = math.nan
    c.set(0, 1500, torch.ones((1, 4, D_)), bad)
    d = c.on_gpu(mi)
    q = torch.randn((2, heads, nq, D_), device="cuda").half()
    a, b = (torch.full((2, nq, heads, D_), 7.0, device="cuda") for _ in range(2))
    ctx.profile(True)
    ctx.kv_cache4_attn(good["cache"], good["seqs"], tensor(mi, q), tensor(mi, a), D_ ** -0.5)
    ctx.kv_cache4_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, b), D_ ** -0.5)
    ctx.synchronize()
    assert "kv_cache4_attn_128_halves" in ctx.profile_collect()
    ctx.profile(False)
    first = 1500 - (n - nq)  # the first query of sequence 0 that sees the token
    assert torch.isfinite(a).all()
    assert b[0, first:, 12:18].isnan().all() and torch.isfinite(b[1]).all()
    assert torch.isfinite(b[0, :first]).all() and torch.isfinite(b[0, :, :12]).all() and torch.isfinite(b[0, :, 18:]).all()
    # what does not see it: the same numbers, but for the references that rows of a wavefront move together, which change the
    # fp32 sums of n terms, (n + 8) U each, and the probabilities' halves, 2^-22, of the largest value (the weights are one in all)
    tol = 2 * ((n + 8) * U + 2.0 ** -22) * float(c.values(0, "v")[0].nan_to_num(0.0).abs().max())
    assert ((a - b).abs()[0, :first] <= tol).all() and ((a - b).abs()[1] <= tol).all()
