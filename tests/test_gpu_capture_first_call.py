"""A context whose first call is a captured one, in a capture that allows allocations (relaxed): the call makes its
workspace then, and replays have the eager bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _rnd(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("op", ["mul_mat_q8_0", "mul_mat_f16", "flash_attn_ext"])
def test_first_call_captured(mi, op):
    stream = torch.cuda.Stream()
    eager, first = mi.Context(0), mi.Context(0, stream.cuda_stream)
    try:
        if op == "flash_attn_ext":  # few queries over many keys: key ranges, whose parts are in the workspace
            q, k, v = _rnd(1, 2, 40, 64).half(), _rnd(2, 2, 4000, 64).half(), _rnd(3, 2, 4000, 64).half()
            ts = [mi.from_torch(x, mi.F16, [64, x.shape[1], 2, 1]) for x in (q, k, v)]
            out, want = (torch.zeros((40, 2, 64), device="cuda") for _ in range(2))
            run = lambda c, o: c.flash_attn_ext(*ts, mi.from_torch(o, mi.F32, [64, 2, 40, 1]), 0.125)  # noqa: E731
        else:
            M, N, K = 300, 512, 1024
            w, x = _rnd(4, N, K) * 0.05, _rnd(5, M, K)
            if op == "mul_mat_f16":
                keep = w.half()
                wt = mi.from_torch(keep, mi.F16, [K, N])
            else:
                keep = torch.zeros((N, K // 32 * 34), dtype=torch.uint8, device="cuda")
                eager.quantize_weights(mi.Q8_0, mi.from_torch(w, mi.F32, [K, N]), keep.data_ptr())
                wt = mi.from_torch(keep, mi.Q8_0, [K, N])
            out, want = (torch.zeros((M, N), device="cuda") for _ in range(2))
            run = lambda c, o: c.mul_mat(wt, mi.from_torch(x, mi.F32, [K, M]), mi.from_torch(o, mi.F32, [N, M]))  # noqa: E731
        run(eager, want)
        eager.synchronize()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            graph.capture_begin(capture_error_mode="relaxed")
            try:
                run(first, out)
            finally:
                graph.capture_end()
        for i in range(4):
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert want.any() and torch.equal(out, want), i
            first.reserve_workspace(32 << (20 + i))  # (a larger one takes its place)
            run(first, want)
            first.synchronize()
    finally:
        first.close()
        eager.close()
