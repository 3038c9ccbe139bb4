"""A mixture-of-experts layer from the package's operators: bf16 forward, one training step,
and the same routing over NVFP4 experts.

    python gpu-kernels_b200/examples/moe_layer.py [--tokens 4096] [--experts 8] [--top-k 2]
        [--hidden 4096] [--ffn 14336] [--steps 3]

    y = x + sum_j weight_j  W2_e ( silu(W1_e x) * (W3_e x) )      over the token's experts e

W1 and W3 are one weight with their rows interleaved in blocks of 16 (swiglu_interleave).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import nvfp4_b200 as nv  # noqa: E402

ops = torch.ops.nvfp4_b200


def forward(x, router, w13, w2, top_k):
    """Inference: six kernels, nothing of the routing passes through the host."""
    r = nv.moe_route(nv.linear(x, router), top_k)
    h = nv.linear_grouped(nv.moe_dispatch(x, r), w13, r.m_offsets, activation="swiglu")
    return nv.moe_combine(nv.linear_grouped(h, w2, r.m_offsets), r, residual=x), r, h


def train_forward(x, router, w13, w2, top_k):
    """The same through the differentiable operators."""
    r = ops.moe_route(ops.linear_preact(x, router)[0], top_k)
    h, _ = ops.linear_preact(ops.moe_dispatch(x, *r), w13, r[3], None, "swiglu")
    return ops.moe_combine(ops.linear_preact(h, w2, r[3])[0], *r, x)


def quantize_weight(w, experts):
    """Per-expert NVFP4 weight: (codes, scales, global scales)."""
    rows = w.shape[0] // experts
    parts = [nv.quantize_dynamic(w[e * rows:(e + 1) * rows].contiguous()) for e in range(experts)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), torch.cat([p[2] for p in parts])


def forward_nvfp4(x, r, q13, q2, hidden_scale):
    """The experts in NVFP4 on the same routing; the hidden state never leaves NVFP4.
    hidden_scale: calibrated on the bf16 run."""
    xs = nv.moe_dispatch(x, r)
    _, gx = nv.global_scale(xs)
    xq, xsf = nv.quantize_grouped(xs, gx, r.m_offsets)
    hq, hsf = nv.gemm_grouped_epilogue(xq, xsf, q13[0], q13[1], gx * q13[2], r.m_offsets, activation="swiglu",
                                       out_global_scale=hidden_scale)
    ys = nv.gemm_grouped(hq, hsf, q2[0], q2[1], hidden_scale * q2[2], r.m_offsets)
    return nv.moe_combine(ys, r, residual=x)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--top-k", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--ffn", type=int, default=14336)
    ap.add_argument("--steps", type=int, default=3)
    a = ap.parse_args()
    E, K, F = a.experts, a.hidden, a.ffn
    g = torch.Generator(device="cuda").manual_seed(0)

    def weight(rows, cols):
        return torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16).normal_(std=cols ** -0.5, generator=g)

    x = torch.randn(a.tokens, K, device="cuda", generator=g).bfloat16()
    router, w2 = weight(E, K), weight(E * K, F)
    w13 = torch.cat([nv.swiglu_interleave(weight(F, K), weight(F, K)) for _ in range(E)])

    def timed(fn):
        for _ in range(2):
            out = fn()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(a.steps):
            out = fn()
        t1.record()
        torch.cuda.synchronize()
        nv.device_status()
        return out, t0.elapsed_time(t1) / a.steps

    (y, r, h), ms = timed(lambda: forward(x, router, w13, w2, a.top_k))
    print(f"bf16 forward          {ms:8.3f} ms   rows by expert {torch.diff(r.m_offsets).tolist()}")

    _, gh = nv.global_scale(h)
    q13, q2 = quantize_weight(w13, E), quantize_weight(w2, E)
    y4, ms = timed(lambda: forward_nvfp4(x, r, q13, q2, gh))
    err = ((y4 - y).float().norm() / (y - x).float().norm()).item()
    print(f"NVFP4 experts         {ms:8.3f} ms   relative difference of the experts' part {err:.3f}")

    params = [t.requires_grad_() for t in (x, router, w13, w2)]
    dy = torch.randn(x.shape, device="cuda", generator=g).bfloat16()
    grads, ms = timed(lambda: torch.autograd.grad(train_forward(*params, a.top_k), params, dy))
    print(f"bf16 forward+backward {ms:8.3f} ms   gradient norms "
          + " ".join(f"{t.float().norm().item():.1f}" for t in grads))


if __name__ == "__main__":
    main()
