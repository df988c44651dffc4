"""What the entry points around a layer's products refuse, on the host: bad shapes, types, strides and
parameters come back as a status with a text, without a context and without a GPU."""
import ctypes as C

import pytest

INVALID, UNSUPPORTED = -4, -3
F32, F16, Q4_0, Q4_1, Q8_0, Q8_1 = 0, 1, 2, 3, 8, 9


def t(mi, ty, ne, ptr=0x10000, nb=None):
    return mi.make_tensor(ptr, ty, ne, nb)


def refused(mi, st, want, text):
    assert st == want, (st, mi.lib().mi355_last_error(None))
    assert text.encode() in mi.lib().mi355_last_error(None), mi.lib().mi355_last_error(None)


def rms(mi, x, dst, add=None, total=None, w=None, eps=1e-5):
    return mi.lib().mi355_rms_norm(None, x, add, w, eps, total, dst)


def test_rms_norm(mi):
    L = mi.lib()
    x, q = t(mi, F32, [64, 3]), t(mi, Q8_0, [64, 3])
    for ty in (F32, F16):
        for out in (F32, F16, Q8_0, Q8_1):
            a, d = t(mi, ty, [64, 3]), t(mi, out, [64, 3])
            assert L.mi355_supports_rms_norm(a, a, a, d) == 1
            refused(mi, rms(mi, a, d), INVALID, "null context")
    refused(mi, rms(mi, x, None), INVALID, "null argument")
    refused(mi, rms(mi, t(mi, F32, [64, 3], ptr=None), q), INVALID, "null argument")
    refused(mi, rms(mi, q, q), UNSUPPORTED, "x must be")
    refused(mi, rms(mi, x, t(mi, Q4_0, [64, 3])), UNSUPPORTED, "dst type")
    refused(mi, rms(mi, x, q, add=t(mi, F16, [64, 3])), UNSUPPORTED, "x's type")
    refused(mi, rms(mi, x, q, total=t(mi, F16, [64, 3])), UNSUPPORTED, "x's type")
    refused(mi, rms(mi, x, t(mi, F32, [64, 4])), INVALID, "shape")
    refused(mi, rms(mi, x, q, add=t(mi, F32, [32, 6])), INVALID, "shape")
    refused(mi, rms(mi, t(mi, F32, [40, 3]), t(mi, Q8_0, [40, 3])), INVALID, "block size")
    refused(mi, rms(mi, t(mi, F32, [64, 3], nb=[8, 512, 1536, 1536]), q), UNSUPPORTED, "contiguous")
    refused(mi, rms(mi, t(mi, F32, [64, 3], ptr=0x10002), q), UNSUPPORTED, "aligned")
    refused(mi, rms(mi, x, t(mi, Q8_0, [64, 3], ptr=0x10001)), UNSUPPORTED, "aligned")
    refused(mi, rms(mi, x, t(mi, Q8_1, [64, 3], ptr=0x10002)), UNSUPPORTED, "aligned")
    refused(mi, rms(mi, t(mi, F32, [32800, 1]), t(mi, F32, [32800, 1])), UNSUPPORTED, "longer")
    refused(mi, rms(mi, t(mi, F32, [1, 1 << 20, 1 << 12]), t(mi, F32, [1, 1 << 20, 1 << 12])), UNSUPPORTED, "too many")
    refused(mi, rms(mi, x, q, w=0x10002), INVALID, "w must be")
    refused(mi, rms(mi, x, q, eps=-1.0), INVALID, "eps")
    refused(mi, rms(mi, x, q, eps=float("nan")), INVALID, "eps")
    bad = t(mi, F32, [64, 3])
    bad.layout = mi.LAYOUT_INT8
    refused(mi, rms(mi, bad, q), INVALID, "layout")


def test_dequantize_rows(mi):
    f = lambda ty, d, src=0x10000: mi.lib().mi355_dequantize_rows(None, ty, src, d)  # noqa: E731
    for ty in (Q8_0, Q8_1, Q4_0, Q4_1):
        refused(mi, f(ty, t(mi, F16, [64, 3])), INVALID, "null context")
    refused(mi, f(Q8_0, None), INVALID, "null argument")
    refused(mi, f(Q8_0, t(mi, F16, [64, 3]), None), INVALID, "null argument")
    refused(mi, f(F16, t(mi, F32, [64, 3])), UNSUPPORTED, "type")
    refused(mi, f(Q8_0, t(mi, Q8_0, [64, 3])), UNSUPPORTED, "F32 or F16")
    refused(mi, f(Q8_0, t(mi, F32, [48, 3])), INVALID, "block size")
    refused(mi, f(Q8_0, t(mi, F32, [64, 3]), 0x10001), INVALID, "aligned")
    refused(mi, f(Q8_1, t(mi, F32, [64, 3]), 0x10002), INVALID, "aligned")
    refused(mi, f(Q8_0, t(mi, F32, [64, 3], nb=[8, 512, 1536, 1536])), UNSUPPORTED, "contiguous")


def rope(mi, src, p, dst, pos=0x10000):
    return mi.lib().mi355_rope_multi(None, src, pos, p, dst)


def test_rope_multi(mi):
    L = mi.lib()
    x = t(mi, F32, [64, 4, 5, 2])
    good = dict(n_dims=64, sections=[32])
    for kw in (good, dict(n_dims=64, sections=[8, 12, 12]), dict(n_dims=64, sections=[16, 16], restart=True),
               dict(n_dims=64, sections=[8, 8, 8, 8], pairs=1), dict(n_dims=32, sections=[0, 16], inverse=True),
               dict(n_dims=64, sections=[12, 10, 10], order=1)):
        p = mi.rope_params(**kw)
        assert L.mi355_supports_rope_multi(x, p, x) == 1, kw
        refused(mi, rope(mi, x, p, x), INVALID, "null context")
    bad = [dict(n_dims=64, sections=[31]), dict(n_dims=64, sections=[33, -1]), dict(n_dims=63, sections=[31]), dict(n_dims=0, sections=[0]),
           dict(n_dims=258, sections=[129]), dict(n_dims=64, sections=[32], pairs=2), dict(n_dims=64, sections=[32], order=2),
           dict(n_dims=64, sections=[32], freq_base=0.0), dict(n_dims=64, sections=[32], freq_base=float("nan")),
           dict(n_dims=64, sections=[32], freq_scale=float("inf")),
           dict(n_dims=64, sections=[8, 8, 8, 8], order=1),     # interleaved: three axes
           dict(n_dims=64, sections=[2, 15, 15], order=1)]      # not enough places of axis 1 and 2
    for kw in bad:
        refused(mi, rope(mi, x, mi.rope_params(**kw), x), INVALID, "out of range")
    p = mi.rope_params(**good)
    p.restart = 2
    refused(mi, rope(mi, x, p, x), INVALID, "out of range")
    p = mi.rope_params(**good)
    refused(mi, rope(mi, x, None, x), INVALID, "null argument")
    refused(mi, rope(mi, x, p, None), INVALID, "null argument")
    refused(mi, rope(mi, x, p, x, pos=None), INVALID, "pos")
    refused(mi, rope(mi, x, p, x, pos=0x10002), INVALID, "pos")
    refused(mi, rope(mi, x, p, t(mi, F16, [64, 4, 5, 2])), UNSUPPORTED, "both")
    refused(mi, rope(mi, t(mi, Q8_0, [64, 4, 5, 2]), p, t(mi, Q8_0, [64, 4, 5, 2])), UNSUPPORTED, "both")
    refused(mi, rope(mi, x, p, t(mi, F32, [64, 4, 5, 3])), INVALID, "shape")
    refused(mi, rope(mi, t(mi, F32, [32, 4, 5, 2]), p, t(mi, F32, [32, 4, 5, 2])), INVALID, "beyond ne0")
    refused(mi, rope(mi, t(mi, F32, [64, 4], nb=[8, 512, 2048, 2048]), p, t(mi, F32, [64, 4])), UNSUPPORTED, "contiguous")


def cache(mi, **kw):
    c = mi.KvCache(0x10000, 0x20000, 0x30000, 0x40000, 4, 2, 32, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def seqs(mi, **kw):
    s = mi.KvSeqs(0x50000, 0x60000, 3, 2)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


BAD_CACHES = [(dict(k=None), INVALID, "null"), (dict(v_scale=None), INVALID, "null"), (dict(n_blocks=-1), INVALID, "negative"),
              (dict(n_head_kv=0), INVALID, "no heads"), (dict(block_tokens=8), UNSUPPORTED, "block_tokens"),
              (dict(block_tokens=48), UNSUPPORTED, "block_tokens"), (dict(head_dim=80), UNSUPPORTED, "head size"),
              (dict(v=0x20008), INVALID, "16-byte"), (dict(k_scale=0x30002), INVALID, "4-byte")]
BAD_SEQS = [(dict(table=None), INVALID, "null"), (dict(n_kv=None), INVALID, "null"), (dict(n_seq=-1), INVALID, "negative"),
            (dict(max_blocks=-1), INVALID, "negative"), (dict(table=0x50002), INVALID, "4-byte"),
            (dict(max_blocks=1 << 26), UNSUPPORTED, "launch limits"), (dict(n_seq=70000), UNSUPPORTED, "launch limits")]


@pytest.mark.parametrize("op", ["write", "read", "attn"])
def test_kv_cache_description(mi, op):
    L = mi.lib()

    def call(c, s):
        n = s.n_seq if s else 3
        kv = t(mi, F16, [64, 5, 2, n])
        if op == "write":
            return L.mi355_kv_cache_write(None, c, s, kv, kv, None)
        if op == "read":
            return L.mi355_kv_cache_read(None, c, s, None, kv, kv)
        return L.mi355_kv_cache_attn(None, c, s, t(mi, F16, [64, 5, 4, n]), None, 0.1, 1, 0, t(mi, F16, [64, 4, 5, n]))

    refused(mi, call(cache(mi), seqs(mi)), INVALID, "null context")
    refused(mi, call(None, seqs(mi)), INVALID, "null argument")
    refused(mi, call(cache(mi), None), INVALID, "null argument")
    for kw, st, text in BAD_CACHES:
        refused(mi, call(cache(mi, **kw), seqs(mi)), st, text)
    for kw, st, text in BAD_SEQS:
        refused(mi, call(cache(mi), seqs(mi, **kw)), st, text)


def test_kv_cache_of_no_blocks(mi):
    """A cache without blocks needs no memory, whatever the table says."""
    L = mi.lib()
    c, s = cache(mi, n_blocks=0, k=None, v=None, k_scale=None, v_scale=None), seqs(mi)
    assert L.mi355_supports_kv_cache_attn(c, s, t(mi, F16, [64, 5, 4, 3]), t(mi, F16, [64, 4, 5, 3]))
    refused(mi, L.mi355_kv_cache_write(None, c, s, t(mi, F16, [64, 5, 2, 3]), t(mi, F16, [64, 5, 2, 3]), None), INVALID, "null context")


def test_kv_cache_rows(mi):
    L, c, s = mi.lib(), cache(mi), seqs(mi)
    kv = t(mi, F16, [64, 5, 2, 3])
    w = lambda k, v, n=None: L.mi355_kv_cache_write(None, c, s, k, v, n)  # noqa: E731
    r = lambda k, v, p=None: L.mi355_kv_cache_read(None, c, s, p, k, v)  # noqa: E731
    refused(mi, w(kv, None), INVALID, "null argument")
    refused(mi, r(None, None), INVALID, "neither")
    refused(mi, r(kv, None), INVALID, "null context")  # one of them alone is allowed
    refused(mi, r(None, kv), INVALID, "null context")
    for f in (w, r):
        refused(mi, f(kv, t(mi, F32, [64, 5, 2, 3])), UNSUPPORTED, "both")
        refused(mi, f(t(mi, Q8_0, [64, 5, 2, 3]), t(mi, Q8_0, [64, 5, 2, 3])), UNSUPPORTED, "both")
        refused(mi, f(kv, t(mi, F16, [64, 6, 2, 3])), INVALID, "must be [")
        for ne in ([96, 5, 2, 3], [64, 5, 1, 3], [64, 5, 2, 2]):
            refused(mi, f(t(mi, F16, ne), t(mi, F16, ne)), INVALID, "must be [")
        refused(mi, f(t(mi, F16, [64, 5, 2, 3], ptr=0x10001), kv), UNSUPPORTED, "aligned")
        refused(mi, f(t(mi, F16, [64, 5, 2, 3], nb=[4, 256, 1280, 2560]), kv), UNSUPPORTED, "contiguous")
        refused(mi, f(kv, kv, 0x10002), INVALID, "4-byte")
        refused(mi, f(kv, t(mi, F16, [64, 5, 2, 3], ptr=None)), INVALID, "null data")


def test_kv_cache_attn(mi):
    L, c, s = mi.lib(), cache(mi), seqs(mi)

    def f(q=None, d=None, n_q=None, scale=0.1, causal=1, window=0):
        return L.mi355_kv_cache_attn(None, c, s, q or t(mi, F16, [64, 5, 4, 3]), n_q, scale, causal, window, d or t(mi, F16, [64, 4, 5, 3]))

    for a in (F16, F32):
        for b in (F16, F32):
            assert L.mi355_supports_kv_cache_attn(c, s, t(mi, a, [64, 5, 4, 3]), t(mi, b, [64, 4, 5, 3])) == 1
    refused(mi, f(), INVALID, "null context")
    refused(mi, f(q=t(mi, F16, [64, 5, 3, 3]), d=t(mi, F16, [64, 3, 5, 3])), INVALID, "multiple of n_head_kv")
    refused(mi, f(q=t(mi, F16, [96, 5, 4, 3])), INVALID, "q must be")
    refused(mi, f(q=t(mi, F16, [64, 5, 4, 2])), INVALID, "q must be")
    refused(mi, f(d=t(mi, F16, [64, 5, 4, 3])), INVALID, "dst must be")
    refused(mi, f(q=t(mi, Q8_0, [64, 5, 4, 3])), UNSUPPORTED, "F32 or F16")
    refused(mi, f(d=t(mi, F32, [64, 4, 5, 3], ptr=0x10002)), UNSUPPORTED, "aligned")
    refused(mi, f(n_q=0x10002), INVALID, "n_q")
    refused(mi, f(scale=float("nan")), INVALID, "scale")
    refused(mi, f(window=-1), INVALID, "window")
    refused(mi, f(causal=2), INVALID, "causal")
    # (an unsupported head size is no node for this backend)
    assert L.mi355_supports_kv_cache_attn(cache(mi, head_dim=80), s, t(mi, F16, [80, 5, 4, 3]), t(mi, F16, [80, 4, 5, 3])) == 0


@pytest.mark.parametrize("t0,t1,want", [(Q8_0, Q8_0, 1), (Q4_0, Q8_0, 1), (Q4_1, Q8_1, 1), (Q8_0, Q8_1, 0), (Q4_1, Q8_0, 0), (F16, Q8_0, 0),
                                        (F32, Q8_0, 0)])
def test_mul_mat_of_quantized_rows(mi, t0, t1, want):
    L = mi.lib()
    w, x, d = t(mi, t0, [64, 16]), t(mi, t1, [64, 8]), t(mi, F32, [16, 8])
    assert L.mi355_supports_mul_mat(C.byref(w), C.byref(x), C.byref(d)) == want
    if want:
        x3, d3 = t(mi, t1, [64, 8, 2]), t(mi, F32, [16, 8, 2])
        assert L.mi355_supports_mul_mat(C.byref(w), C.byref(x3), C.byref(d3)) == 0
        odd = t(mi, t1, [64, 8], ptr=0x10001)
        assert L.mi355_supports_mul_mat(C.byref(w), C.byref(odd), C.byref(d)) == 0
        short = t(mi, t1, [64, 8])
        short.nb[1] = 36
        assert L.mi355_supports_mul_mat(C.byref(w), C.byref(short), C.byref(d)) == 0


def test_python_descriptors(mi):
    import torch
    k = torch.zeros((3, 2, 16, 64), dtype=torch.uint8)
    sc = torch.zeros((3, 2))
    c = mi.kv_cache(k, k.clone(), sc, sc.clone())
    assert (c.n_blocks, c.n_head_kv, c.block_tokens, c.head_dim) == (3, 2, 16, 64)
    with pytest.raises(ValueError):
        mi.kv_cache(k, k[:2], sc, sc)
    with pytest.raises(ValueError):
        mi.kv_cache(k, k, sc, sc.double())
    with pytest.raises(ValueError):
        mi.kv_cache(k.transpose(0, 1), k.transpose(0, 1), sc, sc)
    s = mi.kv_seqs(torch.zeros((4, 7), dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    assert (s.n_seq, s.max_blocks) == (4, 7)
    with pytest.raises(ValueError):
        mi.kv_seqs(torch.zeros((4, 7), dtype=torch.int64), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        mi.kv_seqs(torch.zeros((4, 7), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_empty_tensors_need_no_other_operand(mi):
    """No rows and no tokens: neither source nor positions are asked for, whatever the tensor's own pointer is."""
    for ptr in (None, 0x10000):
        for ne in ([64, 0], [64, 3, 0, 2], [0, 3]):
            refused(mi, mi.lib().mi355_dequantize_rows(None, Q8_0, None, t(mi, F32, ne, ptr=ptr)), INVALID, "null context")
        for ne in ([64, 0, 5, 1], [64, 2, 0, 1], [64, 2, 5, 0]):
            x = t(mi, F16, ne, ptr=ptr)
            refused(mi, rope(mi, x, mi.rope_params(64, [32]), x, pos=None), INVALID, "null context")
    refused(mi, rope(mi, t(mi, F16, [64, 2, 5, 1]), mi.rope_params(64, [32]), t(mi, F16, [64, 2, 5, 1]), pos=None), INVALID, "pos null")
