"""The feed-forward half of two transformer blocks, one dense and one routed to experts, on the operators of the package:

    s, y   = BlockNorm(attention output, residual)          residual sum and the norm in front of the block
    h      = Linear gated (y)                               act(gate) * up
    f      = Linear (h)                                     back to the model's width
    s, y   = BlockNorm(f, s)                                the seam between the blocks, norms on both sides
    logits = Linear (y), fp32                               the router's scores
    ids, w = Route(logits)
    m      = Experts(y, ids, w)
    s, out = BlockNorm(m, s)

    python examples/feed_forward.py [--rows 512] [--channels 1024] [--dtype bf16|f16] [--graph]

Random weights and inputs; the result is compared with the same chain in 64 bits (choices of experts taken from the run, since a
score that lies at the edge of a choice may fall either way).  Prints the largest error and the time of a pass.
"""
import argparse
import importlib
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
E = importlib.import_module("deep-learning-math-kernel-research_b200")


def check(rc):
    if rc != E.ELB_OK:
        raise RuntimeError(f"rc={rc}: {E.last_error()}")


class FeedForward:
    """Plans, weights and buffers for up to ``max_rows`` tokens."""

    def __init__(self, channels, mid, experts, top_k, expert_mid, max_rows, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        td = {E.bf16: torch.bfloat16, E.f16: torch.float16}[dtype]

        def weights(*shape):
            return (torch.randn(*shape, generator=g, device="cuda") * (1.4 / math.sqrt(shape[-1]))).to(td)

        def vector():
            return 1.0 + 0.1 * torch.randn(channels, generator=g, device="cuda")

        self.w = dict(norm1=vector(), post2=vector(), pre2=vector(), post3=vector(), pre3=vector(), up=weights(2 * mid, channels),
                      down=weights(channels, mid), down_bias=0.1 * torch.randn(channels, generator=g, device="cuda"), router=weights(experts, channels),
                      balance=0.02 * torch.randn(experts, generator=g, device="cuda"), w_in=weights(experts, 2 * expert_mid, channels),
                      w_out=weights(experts, channels, expert_mid))
        w = self.w
        self.norm1 = E.BlockNorm(channels, dtype=dtype, residual_dtype=E.f32, pre=E.NORM_RMS)
        check(self.norm1.prepare(pre_weight=w["norm1"]))
        self.up = E.Linear(channels, mid, dtype=dtype, activation=E.ACT_SILU, gated=True)
        check(self.up.prepare(w["up"]))
        self.down = E.Linear(mid, channels, dtype=dtype, with_bias=True)
        check(self.down.prepare(w["down"], w["down_bias"]))
        self.norm2 = E.BlockNorm(channels, dtype=dtype, residual_dtype=E.f32, post=E.NORM_RMS, pre=E.NORM_RMS, scale=0.5)
        check(self.norm2.prepare(post_weight=w["post2"], pre_weight=w["pre2"]))
        self.router = E.Linear(channels, experts, dtype=dtype, out_dtype=E.f32)
        check(self.router.prepare(w["router"]))
        self.route = E.Route(experts, top_k, score=E.SCORE_SIGMOID, with_bias=True, groups=4, top_groups=2, group_best=2)
        check(self.route.prepare(w["balance"]))
        self.experts = E.Experts(experts, top_k, channels, expert_mid, max_rows=max_rows, dtype=dtype)
        check(self.experts.prepare(w["w_in"], w["w_out"]))
        self.norm3 = E.BlockNorm(channels, dtype=dtype, residual_dtype=E.f32, post=E.NORM_RMS, pre=E.NORM_RMS)
        check(self.norm3.prepare(post_weight=w["post3"], pre_weight=w["pre3"]))
        self.top_k = top_k
        new = lambda n, t=td: torch.empty(max_rows, n, dtype=t, device="cuda")      # noqa: E731
        self.y, self.h, self.f, self.m, self.out = new(channels), new(mid), new(channels), new(channels), new(channels)
        self.logits, self.ids, self.share = new(experts, torch.float32), new(top_k, torch.int32), new(top_k, torch.float32)

    def __call__(self, x, s, stream=None):
        """x: what the attention before the block gave; s: the residual stream in fp32, updated in place.  Returns the last norm's output."""
        n, q = x.shape[0], stream
        check(self.norm1.enqueue(self.y, s, x, s, rows=n, stream=q))
        check(self.up.enqueue(self.h, self.y, rows=n, stream=q))
        check(self.down.enqueue(self.f, self.h, rows=n, stream=q))
        check(self.norm2.enqueue(self.y, s, self.f, s, rows=n, stream=q))
        check(self.router.enqueue(self.logits, self.y, rows=n, stream=q))
        check(self.route.enqueue(self.ids, self.share, self.logits, rows=n, stream=q))
        check(self.experts.enqueue(self.m, self.y, self.ids, self.share, rows=n, stream=q))
        check(self.norm3.enqueue(self.out, s, self.m, s, rows=n, stream=q))
        return self.out[:n]

    def plans(self):
        return [self.norm1, self.up, self.down, self.norm2, self.router, self.route, self.experts, self.norm3]

    def in_64_bits(self, x, s, ids):
        """The same chain in 64 bits, with the experts that the run has chosen."""
        w = {k: v.double() for k, v in self.w.items()}

        def rms(v, weight):
            return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * weight

        def gated(z):
            a, b = z.chunk(2, dim=-1)
            return a * torch.sigmoid(a) * b

        s = s.double() + x.double()
        f = gated(rms(s, w["norm1"]) @ w["up"].T) @ w["down"].T + w["down_bias"]
        s = s + 0.5 * rms(f, w["post2"])
        y = rms(s, w["pre2"])
        score = torch.sigmoid(y @ w["router"].T).gather(1, ids.long())
        share = score / score.sum(1, keepdim=True)
        m = torch.zeros_like(y)
        for e in range(w["w_in"].shape[0]):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            m.index_add_(0, t, gated(y[t] @ w["w_in"][e].T) @ w["w_out"][e].T * share[t, j][:, None])
        s = s + rms(m, w["post3"])
        return rms(s, w["pre3"]), s


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=512)
    ap.add_argument("--channels", type=int, default=1024)
    ap.add_argument("--dtype", choices=("bf16", "f16"), default="bf16")
    ap.add_argument("--graph", action="store_true", help="capture a pass in a CUDA graph and time its replay")
    a = ap.parse_args()
    dtype = {"bf16": E.bf16, "f16": E.f16}[a.dtype]
    ff = FeedForward(a.channels, 4 * a.channels, 32, 4, a.channels // 2, a.rows, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(a.rows, a.channels, generator=g, device="cuda").to(ff.y.dtype)
    s0 = 2.0 * torch.randn(a.rows, a.channels, generator=g, device="cuda")
    s = s0.clone()
    torch.cuda.synchronize()
    out = ff(x, s)
    torch.cuda.synchronize()
    bad = [p.device_status() for p in ff.plans()]
    assert not any(bad), bad
    want, want_s = ff.in_64_bits(x, s0, ff.ids[:a.rows])
    rel = lambda v, t: float((v.double() - t).norm() / t.norm())                    # noqa: E731
    print(f"{a.rows} rows of {a.channels}, {a.dtype}: relative error of the output {rel(out, want):.2e}, of the residual stream {rel(s, want_s):.2e}")
    run = lambda: ff(x, s)                                                          # noqa: E731
    if a.graph:
        graph, q = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=q):
            ff(x, s, stream=q.cuda_stream)
        run = graph.replay
    for _ in range(5):
        run()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(50):
        run()
    end.record()
    torch.cuda.synchronize()
    print(f"{begin.elapsed_time(end) / 50 * 1e3:.1f} us a pass")


if __name__ == "__main__":
    main()
