"""What the entry points of a layer with a 4-bit cache refuse, on the host, and the cache's format on the CPU."""
import ctypes as C

import pytest
import torch

import layer4_refs as R4
from layer_refs import F64
from test_layer_refusals import BAD_CACHES, BAD_SEQS, F16, F32, INVALID, Q8_0, UNSUPPORTED, refused, seqs, t


def test_format():
    """Pack and unpack are each other's inverse; a group's values stand for it to half a step, or the last one's reach."""
    q = torch.randint(0, 16, (5, 7, 96), dtype=torch.uint8)
    assert torch.equal(R4.unpack(R4.pack(q)), q)
    assert R4.pack(torch.tensor([[1, 2, 3, 4, 5, 6, 7, 8]], dtype=torch.uint8)).tolist() == [[0x31, 0x75, 0x42, 0x86]]
    x = torch.randn((400, 32))
    d = R4.group_scale(x)
    assert torch.equal(d.half().to(F64), d) and torch.equal(d.bfloat16().to(F64), d)
    y = (R4.nibbles(x, d).to(F64) - 8) * d[:, None]
    assert torch.equal(y.half().to(F64), y)  # every value is an fp16 number
    top = x.abs().amax(-1, keepdim=True).to(F64)
    # Half a step where the nibbles reach.  On the other side they end at 7 d, and d = top / 8 (1 - r) with r up to half a step
    # of eight significant bits, 2^-8: top - 7 d = top / 8 (1 + 7 r).
    assert ((x - y).abs() <= top / 8 * (1 + 7 * 2.0 ** -8)).all()
    assert ((x - y).abs().mean() < 0.5 * (top / 8).mean())


def qk(mi, q, k, p, qd, kd, pos=0x10000, eps=1e-6, q_w=None, k_w=None):
    return mi.lib().mi355_qk_norm_rope(None, q, k, q_w, k_w, eps, pos, p, qd, kd)


def test_qk_norm_rope(mi):
    L = mi.lib()
    q, k = t(mi, F32, [64, 8, 5, 2]), t(mi, F32, [64, 2, 5, 2])
    p = mi.rope_params(64, [32])
    for sq in (F32, F16):
        for d in (F32, F16):
            a, b, c, e = t(mi, sq, [64, 8, 5, 2]), t(mi, sq, [64, 2, 5, 2]), t(mi, d, [64, 8, 5, 2]), t(mi, d, [64, 2, 5, 2])
            assert L.mi355_supports_qk_norm_rope(a, b, p, c, e) == 1
            refused(mi, qk(mi, a, b, p, c, e), INVALID, "null context")
            refused(mi, qk(mi, a, None, p, c, None), INVALID, "null context")
            refused(mi, qk(mi, None, b, p, None, e), INVALID, "null context")
    refused(mi, qk(mi, None, None, p, None, None), INVALID, "null argument")
    refused(mi, qk(mi, q, k, p, q, None), INVALID, "without its output")
    refused(mi, qk(mi, q, None, p, q, k), INVALID, "without its output")
    refused(mi, qk(mi, q, k, None, q, k), INVALID, "null argument")
    refused(mi, qk(mi, t(mi, F32, [64, 8, 5, 2], ptr=None), k, p, q, k), INVALID, "null argument")
    refused(mi, qk(mi, q, k, mi.rope_params(64, [31]), q, k), INVALID, "out of range")
    refused(mi, qk(mi, q, k, mi.rope_params(128, [64]), q, k), INVALID, "beyond ne0")
    refused(mi, qk(mi, q, t(mi, F16, [64, 2, 5, 2]), p, q, k), UNSUPPORTED, "same types")
    refused(mi, qk(mi, q, k, p, q, t(mi, F16, [64, 2, 5, 2])), UNSUPPORTED, "same types")
    refused(mi, qk(mi, t(mi, Q8_0, [64, 8, 5, 2]), k, p, q, k), UNSUPPORTED, "F32 or F16")
    refused(mi, qk(mi, q, k, p, t(mi, F32, [64, 8, 5, 3]), k), INVALID, "shape")
    refused(mi, qk(mi, q, t(mi, F32, [64, 2, 6, 2]), p, q, t(mi, F32, [64, 2, 6, 2])), INVALID, "same head size")
    big = t(mi, F32, [264, 8, 5, 2])
    refused(mi, qk(mi, big, None, p, big, None), UNSUPPORTED, "more than")
    refused(mi, qk(mi, t(mi, F32, [64, 8, 5, 2], nb=[8, 512, 4096, 20480]), k, p, q, k), UNSUPPORTED, "contiguous")
    refused(mi, qk(mi, q, k, p, q, k, pos=None), INVALID, "pos")
    refused(mi, qk(mi, q, k, p, q, k, pos=0x10002), INVALID, "pos")
    refused(mi, qk(mi, q, k, p, q, k, eps=-1.0), INVALID, "eps")
    refused(mi, qk(mi, q, k, p, q, k, eps=float("nan")), INVALID, "eps")
    refused(mi, qk(mi, q, k, p, q, k, k_w=0x10002), INVALID, "weights")
    long = t(mi, F32, [8, 1 << 20, 1 << 12])
    refused(mi, qk(mi, long, None, mi.rope_params(8, [4]), long, None), UNSUPPORTED, "launch limits")


def cache4(mi, **kw):
    c = mi.KvCache4(0x10000, 0x20000, 0x30000, 0x40000, 4, 2, 32, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def call(mi, op, c, s, q=None, dst=None, **kw):
    L = mi.lib()
    n = s.n_seq if s else 3
    kv = t(mi, F16, [64, 5, 2, n])
    a = dict(n_q=None, scale=0.1, causal=1, window=0, lse=0x70000, sums=0x80000, out=0x90000, n_keep=None, max_keep=10, first=1, recent=2,
             kept=0xa0000, n_out=0xb0000)
    a.update(kw)
    q = t(mi, F16, [64, 5, 4, n]) if q is None else q
    if op == "write":
        return L.mi355_kv_cache4_write(None, c, s, kv, kv, None)
    if op == "read":
        return L.mi355_kv_cache4_read(None, c, s, None, kv, kv)
    if op == "attn":
        dst = t(mi, F16, [64, 4, 5, n]) if dst is None else dst
        return L.mi355_kv_cache4_attn(None, c, s, q, a["n_q"], a["scale"], a["causal"], a["window"], dst, a["lse"])
    if op == "weights":
        return L.mi355_kv_cache4_weights(None, c, s, q, a["n_q"], a["lse"], a["scale"], a["causal"], a["window"], a["sums"])
    return L.mi355_kv_cache4_evict(None, c, s, a["sums"], a["n_keep"], a["max_keep"], a["first"], a["recent"], a["out"], a["kept"], a["n_out"])


@pytest.mark.parametrize("op", ["write", "read", "attn", "weights", "evict"])
def test_description(mi, op):
    refused(mi, call(mi, op, cache4(mi), seqs(mi)), INVALID, "null context")
    for kw, st, text in BAD_CACHES[:-1] + [(dict(k_scale=0x30004), INVALID, "8-byte"), (dict(v_scale=0x40002), INVALID, "8-byte")]:
        refused(mi, call(mi, op, cache4(mi, **kw), seqs(mi)), st, text)
    for kw, st, text in BAD_SEQS:
        s = seqs(mi, **kw)
        refused(mi, call(mi, op, cache4(mi), s), st, text)
    refused(mi, call(mi, op, None, seqs(mi)), INVALID, "null argument")
    refused(mi, call(mi, op, cache4(mi), None), INVALID, "null argument")


@pytest.mark.parametrize("op", ["attn", "weights"])
def test_queries(mi, op):
    c, s = cache4(mi), seqs(mi)
    for kw in (dict(scale=float("inf")), dict(scale=float("nan")), dict(window=-1), dict(causal=2)):
        refused(mi, call(mi, op, c, s, **kw), INVALID, "scale must be")
    refused(mi, call(mi, op, c, s, n_q=0x50002), INVALID, "n_q and lse")
    refused(mi, call(mi, op, c, s, lse=0x50002), INVALID, "n_q and lse")
    for ne in ([128, 5, 4, 3], [64, 5, 3, 3], [64, 5, 4, 2], [64, 5, 0, 3]):
        refused(mi, call(mi, op, c, s, q=t(mi, F16, ne)), INVALID, "n_head a multiple")
    refused(mi, call(mi, op, c, s, q=t(mi, Q8_0, [64, 5, 4, 3])), UNSUPPORTED, "F32 or F16")
    refused(mi, call(mi, op, c, s, q=t(mi, F16, [64, 5, 4, 3], ptr=None)), INVALID, "null argument")
    refused(mi, call(mi, op, c, s, q=t(mi, F16, [64, 5, 4, 3], nb=[4, 256, 1280, 5120])), UNSUPPORTED, "contiguous")
    if op == "attn":
        for ne in ([64, 5, 4, 3], [64, 4, 5, 2], [32, 4, 5, 3]):
            refused(mi, call(mi, op, c, s, dst=t(mi, F16, ne)), INVALID, "dst must be")
        refused(mi, call(mi, op, c, s, dst=t(mi, Q8_0, [64, 4, 5, 3])), UNSUPPORTED, "F32 or F16")
        refused(mi, call(mi, op, c, s, dst=t(mi, F16, [64, 4, 5, 3], ptr=None)), INVALID, "null argument")
        assert mi.lib().mi355_supports_kv_cache4_attn(c, s, t(mi, F32, [64, 5, 4, 3]), t(mi, F16, [64, 4, 5, 3])) == 1
        assert mi.lib().mi355_supports_kv_cache4_attn(c, s, t(mi, F32, [64, 5, 4, 3]), t(mi, F16, [64, 5, 4, 3])) == 0


def test_evict(mi):
    c, s = cache4(mi), seqs(mi)
    for kw in (dict(max_keep=-1), dict(first=-1), dict(recent=-1)):
        refused(mi, call(mi, "evict", c, s, **kw), INVALID, "must not be negative")
    for kw in (dict(sums=None), dict(out=None), dict(kept=None), dict(n_out=None)):
        refused(mi, call(mi, "evict", c, s, **kw), INVALID, "null argument")
    for kw in (dict(sums=0x80002), dict(out=0x90001), dict(kept=0xa0002), dict(n_out=0xb0002), dict(n_keep=0x50002)):
        refused(mi, call(mi, "evict", c, s, **kw), INVALID, "4-byte")
    for kw in (dict(out=0x80000), dict(n_out=0x60000), dict(n_keep=0xb0000)):
        refused(mi, call(mi, "evict", c, s, **kw), INVALID, "must not be the inputs")
    assert C.sizeof(mi.KvCache4) == C.sizeof(mi.KvCache)


def test_python_descriptions(mi):
    z = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    c = mi.kv_cache4(z(3, 2, 16, 32), z(3, 2, 16, 32), h(3, 2, 16, 2), h(3, 2, 2, 16))
    assert (c.n_blocks, c.n_head_kv, c.block_tokens, c.head_dim) == (3, 2, 16, 64)
    for bad in ((z(3, 2, 16, 32), z(3, 2, 16, 48), h(3, 2, 16, 2), h(3, 2, 2, 16)), (z(3, 2, 16, 32), z(3, 2, 16, 32), h(3, 2, 2, 16), h(3, 2, 2, 16)),
                (z(3, 2, 16, 32), z(3, 2, 16, 32), h(3, 2, 16, 2), h(3, 2, 2, 16).float()),
                (z(3, 2, 16, 32), z(3, 16, 2, 32).transpose(1, 2), h(3, 2, 16, 2), h(3, 2, 2, 16))):
        with pytest.raises(ValueError):
            mi.kv_cache4(*bad)


def test_sizes_beyond_a_launch(mi):
    c, n = cache4(mi, n_head_kv=1), (1 << 27) + 1
    wide = t(mi, F16, [64, n, 1, 3])
    refused(mi, mi.lib().mi355_kv_cache4_write(None, c, seqs(mi), wide, wide, None), UNSUPPORTED, "launch limits")
    refused(mi, mi.lib().mi355_kv_cache4_read(None, c, seqs(mi), None, wide, None), UNSUPPORTED, "launch limits")
    refused(mi, call(mi, "evict", cache4(mi, n_head_kv=300), seqs(mi, n_seq=2001)), UNSUPPORTED, "launch limits")
    for ne0, tokens in ((64, 1 << 28), (128, 1 << 27), (256, 1 << 26)):
        q, fits = t(mi, F16, [ne0, 4, tokens, 1]), t(mi, F16, [ne0, 4, tokens - 64, 1])
        p = mi.rope_params(ne0, [ne0 // 2])
        refused(mi, qk(mi, q, None, p, q, None), UNSUPPORTED, "launch limits")
        refused(mi, qk(mi, fits, None, p, fits, None), INVALID, "null context")


def test_workspace_of_what_has_no_plan(mi):
    ctx = C.create_string_buffer(1 << 16)  # (no field is read of a call that has no plan)
    q = t(mi, F16, [64, 5, 4, 3])
    for size in (mi.lib().mi355_kv_cache4_attn_workspace_size, mi.lib().mi355_kv_cache4_weights_workspace_size):
        assert size(None, cache4(mi), seqs(mi), q, 0) == 0
        for c, s, x in ((None, seqs(mi), q), (cache4(mi), None, q), (cache4(mi), seqs(mi), None), (cache4(mi, n_head_kv=0), seqs(mi), q),
                        (cache4(mi, n_head_kv=8), seqs(mi), q), (cache4(mi, block_tokens=0), seqs(mi), q), (cache4(mi), seqs(mi, max_blocks=-1), q),
                        (cache4(mi), seqs(mi, n_seq=2), q), (cache4(mi), seqs(mi), t(mi, F16, [64, -5, 4, 3])),
                        (cache4(mi), seqs(mi), t(mi, F16, [64, 5, 0, 3])), (cache4(mi), seqs(mi), t(mi, F16, [32, 5, 4, 3]))):
            assert size(ctx, c, s, x, 0) == 0
