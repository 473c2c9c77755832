"""A program that holds its data in torch tensors and records the library's calls with torch's graphs; run by
test_float8_torch_gpu in a process of its own, because torch has to be imported before the device library is loaded."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ocean-tensor-package_amd"))
import ocean_hip as oh  # noqa: E402

BF16, E4M3, FLOAT = oh.BFLOAT16, oh.FLOAT8_E4M3, oh.FLOAT


def main():
    check, lib = oh.check, oh.lib
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    t, n, m = 300, 1024, 256                                    # tokens, features, outputs
    x, r = (torch.randn(t, n, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(m, n, generator=g, device="cuda") / 32
    dz = torch.randn(t, m, generator=g, device="cuda").bfloat16()
    gain = 1 + 0.1 * torch.randn(n, generator=g, device="cuda")
    byte, flt = dict(dtype=torch.uint8, device="cuda"), dict(dtype=torch.float32, device="cuda")
    tb = -(-t // 128)
    wq, ws, yq, ys, rstd = torch.empty(m, n, **byte), torch.empty(m // 128, n // 128, **flt), torch.empty(t, n, **byte), torch.empty(t, n // 128, **flt), torch.empty(t, **flt)
    h, z, dx, dy = torch.empty_like(x), torch.empty_like(dz), torch.empty_like(x), torch.empty_like(x)
    xt, xts, dzt, dzts = torch.empty(t, n, **byte), torch.empty(tb, n, **flt), torch.empty(t, m, **byte), torch.empty(tb, m, **flt)
    dgain, dw = torch.empty(n, **flt), torch.zeros(m, n, **flt)

    def step():
        s = torch.cuda.current_stream().cuda_stream
        p = lambda a: a.data_ptr()      # noqa: E731
        check(lib.och_quantize_blocks(FLOAT, E4M3, n, m, p(w), n, 128, 128, p(wq), n, p(ws), n // 128, s))
        check(lib.och_rms_norm(BF16, n, t, p(x), n, p(r), n, p(h), n, FLOAT, p(gain), 1e-5, E4M3, p(yq), n, p(ys), n // 128, p(rstd), s))
        check(lib.och_gemm_scaled(E4M3, E4M3, BF16, b"T", b"N", m, t, n, 1.0, p(wq), n, p(ws), n // 128, 128, p(yq), n, p(ys), n // 128, 1, 0.0, p(z), m, s))
        check(lib.och_quantize_blocks(BF16, E4M3, n, t, p(h), n, 1, 128, p(xt), n, p(xts), n, s))
        check(lib.och_quantize_blocks(BF16, E4M3, m, t, p(dz), m, 1, 128, p(dzt), m, p(dzts), m, s))
        check(lib.och_gemm_scaled(E4M3, E4M3, FLOAT, b"N", b"T", n, m, t, 1.0, p(xt), n, p(xts), n, 1, p(dzt), m, p(dzts), m, 1, 1.0, p(dw), n, s))
        dy.copy_(x)
        check(lib.och_rms_norm_grad(BF16, n, t, p(dy), n, p(h), n, p(rstd), FLOAT, p(gain), None, 0, p(dx), n, p(dgain), s))

    out = (wq, ws, yq, ys, rstd, h, z, xt, xts, dx, dgain, dw)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = None
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            step()
        except oh.OceanHipError as e:
            refused = str(e)
        graph.capture_end()
    assert refused and "och_stream_reserve_workspace" in refused, refused
    del graph
    check(lib.och_stream_reserve_workspace(stream.cuda_stream))
    torch.cuda.synchronize()
    dw.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    got = []
    for _ in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        got.append([o.clone() for o in out])
    dw.zero_()
    for k in range(3):
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        for a, b in zip(out, got[k]):
            assert torch.equal(a, b), k
    assert torch.isfinite(dw).all() and dw.abs().max() > 0 and not torch.equal(got[0][-1], got[1][-1])
    print("replays equal the eager calls")


if __name__ == "__main__":
    main()
