"""The attention half of transformer blocks on the operators of the package: an encoder layer over padded inputs, and a decoder layer that takes prompts of uneven
length and then answers token by token from a cache of pages.

    encoder   y = BlockNorm(x); q, k, v = Linear(y); q, k = Rotary(q, k); a = Attention(q, k, v) over each input's own length; x = x + Linear(a)
              k, v of the states for the decoder = Linear(x), once
    decoder   y = BlockNorm(x); q, k, v = Linear(y); CacheAppend: q turned, k turned and v into the cache; a = Attention(q, cache); x = x + Linear(a)
              y = BlockNorm(x); q = Linear(y); a = Attention(q, the encoder's k and v); x = x + Linear(a)

    python examples/encoder_decoder.py [--seqs 6] [--heads 8] [--kv-heads 2] [--dim 64] [--steps 20] [--dtype bf16|f16] [--graph]

q, k and v are parts of one product's rows.  Random weights and inputs; everything that comes out is compared with the same layers in 64 bits.  Prints the
errors and the time of a token step.
"""
import argparse
import importlib
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
E = importlib.import_module("deep-learning-math-kernel-research_b200")
PAGE = 16


def check(rc):
    if rc != E.ELB_OK:
        raise RuntimeError(f"rc={rc}: {E.last_error()}")


class Layers:
    """Plans, weights, buffers and the cache for ``seqs`` sequences of up to ``most`` tokens beside inputs of up to ``src`` states."""

    def __init__(self, seqs, src, most, heads, kv_heads, dim, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        td = {E.bf16: torch.bfloat16, E.f16: torch.float16}[dtype]
        c, wide = heads * dim, (heads + 2 * kv_heads) * dim
        self.seqs, self.src, self.most, self.heads, self.kv_heads, self.dim, self.td, self.wide, self.c = seqs, src, most, heads, kv_heads, dim, td, wide, c
        draw = lambda *shape: (torch.randn(*shape, generator=g, device="cuda") * (1.2 / math.sqrt(shape[-1]))).to(td)     # noqa: E731
        self.w = dict(enc_qkv=draw(wide, c), enc_out=draw(c, c), memory=draw(2 * kv_heads * dim, c), qkv=draw(wide, c), out=draw(c, c), cross_q=draw(c, c), cross_out=draw(c, c))

        def linear(name, ic, oc, **kw):
            plan = E.Linear(ic, oc, dtype=dtype, **kw)
            check(plan.prepare(self.w[name]))
            return plan
        self.norm = E.BlockNorm(c, dtype=dtype, pre=E.NORM_RMS, with_residual=False)
        check(self.norm.prepare())
        self.enc_qkv, self.qkv = linear("enc_qkv", c, wide), linear("qkv", c, wide)
        self.enc_out, self.out, self.cross_out = (linear(n, c, c, with_residual=True) for n in ("enc_out", "out", "cross_out"))
        self.memory, self.cross_q = linear("memory", c, 2 * kv_heads * dim), linear("cross_q", c, c)
        self.rotary = E.Rotary(heads, kv_heads, dim, dtype=dtype, ld_q=wide, ld_k=wide, ld_q_out=wide, ld_k_out=wide)
        check(self.rotary.prepare())
        self.enc_attention = E.Attention(heads, kv_heads, dim, dtype=dtype, causal=False, ld_input=wide, ld_token=wide)
        self.append = E.CacheAppend(heads, kv_heads, dim, PAGE, dtype=dtype, ld_q=wide, ld_k=wide, ld_v=wide, scaling=E.SCALE_LINEAR, factor=2.0)
        check(self.append.prepare())
        self.attention = E.Attention(heads, kv_heads, dim, dtype=dtype, page_size=PAGE)
        self.cross = E.Attention(heads, kv_heads, dim, dtype=dtype, causal=False, ld_token=2 * kv_heads * dim)
        new = lambda rows, n: torch.empty(rows, n, dtype=td, device="cuda")                                              # noqa: E731
        rows = max(seqs * src, seqs * most)
        self.y, self.h, self.q, self.a = new(rows, c), new(rows, wide), new(rows, c), new(rows, c)
        self.states, self.kv, self.positions = new(seqs * src, c), new(seqs * src, 2 * kv_heads * dim), torch.arange(src, dtype=torch.int32, device="cuda").repeat(seqs)
        pages, width = seqs * -(-most // PAGE) + 1, -(-most // PAGE)
        self.k_cache, self.v_cache = (torch.empty(pages, kv_heads, PAGE, dim, dtype=td, device="cuda") for _ in range(2))
        self.table = torch.randperm(pages, generator=g, device="cuda")[:seqs * width].to(torch.int32).reshape(seqs, width).contiguous()
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def parts(self, h):
        """q, k and v in the rows of a product"""
        q = self.heads * self.dim
        return h[:, :q], h[:, q:q + self.kv_heads * self.dim], h[:, q + self.kv_heads * self.dim:]

    def encode(self, x, lengths, stream=None):
        """x: [seqs * src, c], of which each input has the first ``lengths``"""
        n, s = x.shape[0], stream
        check(self.norm.enqueue(self.y, None, x, rows=n, stream=s))
        check(self.enc_qkv.enqueue(self.h, self.y, rows=n, stream=s))
        q, k, v = self.parts(self.h[:n])
        check(self.rotary.enqueue(q, k, q, k, self.positions, rows=n, stream=s))
        keys = [t.unflatten(0, (self.seqs, self.src)).unflatten(2, (self.kv_heads, self.dim)) for t in (k, v)]
        check(self.enc_attention.enqueue(self.a, q, *keys, lengths=lengths, rows=n, seqs=self.seqs, stream=s))
        check(self.enc_out.enqueue(self.states, self.a, x, rows=n, stream=s))
        check(self.memory.enqueue(self.kv, self.states, rows=n, stream=s))
        self.src_lengths = lengths
        return self.states

    def decode(self, x, starts=None, stream=None):
        """x: new tokens [rows, c], one of each sequence, or as ``starts`` says; ``self.lengths`` counts them already.  x is replaced by what comes out."""
        n, s = x.shape[0], stream
        check(self.norm.enqueue(self.y, None, x, rows=n, stream=s))
        check(self.qkv.enqueue(self.h, self.y, rows=n, stream=s))
        q, k, v = self.parts(self.h[:n])
        check(self.append.enqueue(self.q, self.k_cache, self.v_cache, q, k, v, self.table, self.lengths, starts, rows=n, seqs=self.seqs, stream=s))
        check(self.attention.enqueue(self.a, self.q, self.k_cache, self.v_cache, self.table, self.lengths, starts, rows=n, seqs=self.seqs, stream=s))
        check(self.out.enqueue(x, self.a, x, rows=n, stream=s))
        check(self.norm.enqueue(self.y, None, x, rows=n, stream=s))
        check(self.cross_q.enqueue(self.q, self.y, rows=n, stream=s))
        kv = self.kv.view(self.seqs, self.src, 2, self.kv_heads, self.dim)
        check(self.cross.enqueue(self.a, self.q, kv[:, :, 0], kv[:, :, 1], lengths=self.src_lengths, starts=starts, rows=n, seqs=self.seqs, stream=s))
        check(self.cross_out.enqueue(x, self.a, x, rows=n, stream=s))
        return x

    def plans(self):
        return [self.norm, self.enc_qkv, self.rotary, self.enc_attention, self.enc_out, self.memory, self.qkv, self.append, self.attention, self.out, self.cross_q, self.cross,
                self.cross_out]

    # ---- the same layers in 64 bits, a sequence at a time
    def _attend64(self, q, k, v, causal):
        group = self.heads // self.kv_heads
        s = torch.einsum("nhd,mhd->hnm", q, k.repeat_interleave(group, 1)) / math.sqrt(self.dim)
        if causal:
            s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -math.inf)
        return torch.einsum("hnm,mhd->nhd", torch.softmax(s, -1), v.repeat_interleave(group, 1)).flatten(1)

    def _turn64(self, x, factor):
        f = 10000.0 ** (-torch.arange(0, self.dim, 2, dtype=torch.float64, device="cuda") / self.dim) / factor
        t = torch.arange(x.shape[0], dtype=torch.float64, device="cuda")[:, None, None] * f
        a, b = x.chunk(2, -1)
        return torch.cat((a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()), -1)

    def in_64_bits(self, source, tokens):
        """What encode and decode give for one input (its own length) and one sequence's tokens."""
        w = {k: v.double() for k, v in self.w.items()}
        norm = lambda v: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)                                            # noqa: E731
        heads = lambda v: v.unflatten(1, (-1, self.dim))                                                                 # noqa: E731
        split = (self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim)
        x = source.double()
        q, k, v = map(heads, (norm(x) @ w["enc_qkv"].T).split(split, 1))
        states = x + self._attend64(self._turn64(q, 1.0), self._turn64(k, 1.0), v, False) @ w["enc_out"].T
        mk, mv = map(heads, (states @ w["memory"].T).chunk(2, 1))
        x = tokens.double()
        q, k, v = map(heads, (norm(x) @ w["qkv"].T).split(split, 1))
        x = x + self._attend64(self._turn64(q, 2.0), self._turn64(k, 2.0), v, True) @ w["out"].T
        x = x + self._attend64(heads(norm(x) @ w["cross_q"].T), mk, mv, False) @ w["cross_out"].T
        return states, x


def run(seqs=6, heads=8, kv_heads=2, dim=64, steps=20, dtype=None, graph=False, src=200, longest=150, seed=0):
    """(relative errors of the encoder's states, the prompts' and the answers' rows; seconds of a token step; the layers)"""
    dtype = E.bf16 if dtype is None else dtype
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    new = [1 + (longest * (3 * i + 1) // (3 * seqs)) for i in range(seqs)]                  # prompts of uneven length
    own = [src - 7 * i % src for i in range(seqs)]                                          # inputs too
    layers = Layers(seqs, src, longest + steps + 1, heads, kv_heads, dim, dtype, seed)
    draw = lambda rows: torch.randn(rows, layers.c, generator=g, device="cuda").to(layers.td)                          # noqa: E731
    source, prompts, answers = draw(seqs * src), draw(sum(new)), [draw(seqs) for _ in range(steps)]
    starts = torch.tensor([sum(new[:i]) for i in range(seqs + 1)], dtype=torch.int32, device="cuda")
    lengths = torch.tensor(own, dtype=torch.int32, device="cuda")
    x, steps_out, slot, s = prompts.clone(), [], torch.empty_like(answers[0]) if steps else None, torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        states = layers.encode(source, lengths, s.cuda_stream)
        layers.lengths += starts.diff()
        layers.decode(x, starts, s.cuda_stream)
        step = lambda: (layers.lengths.add_(1), layers.decode(slot, stream=s.cuda_stream))                              # noqa: E731
        if graph and steps:
            slot.copy_(answers[0])
            step()                                          # (a call of as many rows before a capture; its token is written again)
            layers.lengths -= 1
            s.synchronize()
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=s):
                step()
            step = captured.replay
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for i, a in enumerate(answers):
            if i == 1:
                begin.record()
            slot.copy_(a)
            step()
            steps_out.append(slot.clone())
        end.record()
    torch.cuda.synchronize()
    bad = [p.device_status() for p in layers.plans()]
    assert not any(bad), bad
    off = [[], [], []]
    for i in range(seqs):
        r = slice(sum(new[:i]), sum(new[:i + 1]))
        tokens = torch.cat([prompts[r]] + [a[i:i + 1] for a in answers])
        want_states, want = layers.in_64_bits(source[i * src:i * src + own[i]], tokens)
        got = torch.cat([x[r]] + [a[i:i + 1] for a in steps_out])
        off[0].append((states[i * src:i * src + own[i]], want_states))
        off[1].append((got[:new[i]], want[:new[i]]))
        off[2].append((got[new[i]:], want[new[i]:]))
    rel = [math.sqrt(sum(float((a.double() - b).pow(2).sum()) for a, b in o) / max(1e-300, sum(float(b.pow(2).sum()) for _, b in o))) for o in off]
    return rel, begin.elapsed_time(end) * 1e-3 / (steps - 1) if steps > 1 else 0.0, layers


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("seqs", 6), ("heads", 8), ("kv-heads", 2), ("dim", 64), ("steps", 20)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--dtype", choices=("bf16", "f16"), default="bf16")
    ap.add_argument("--graph", action="store_true", help="capture a token step in a CUDA graph and replay it")
    a = ap.parse_args()
    rel, seconds, _ = run(a.seqs, a.heads, a.kv_heads, a.dim, a.steps, {"bf16": E.bf16, "f16": E.f16}[a.dtype], a.graph)
    print(f"{a.seqs} sequences, {a.heads} heads of {a.dim} over {a.kv_heads}, {a.dtype}: relative error of the encoder's states {rel[0]:.2e}, of the prompts' rows {rel[1]:.2e}, "
          f"of the answers' {rel[2]:.2e}; {seconds * 1e6:.1f} us a token step")


if __name__ == "__main__":
    main()
