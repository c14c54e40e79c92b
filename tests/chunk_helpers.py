"""Steps of ragged chunks over a paged pool for the tests: their inputs, and the
operators' definitions in 64 bits on the CPU."""
import math

import torch

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# A rounding to the type is off by at most half its step, relative to the value.
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Step:
    """new[i] tokens of sequence i after cached[i] keys; pages drawn from a
    shuffled pool with some to spare, the tables' unused entries -1."""

    def __init__(self, seed, dtype, heads, new, cached, window=0, sinks=0, mbps=None, gap=0,
                 max_tokens=None, scale=None):
        self.dtype, (self.hq, self.hkv, self.d) = dtype, heads
        self.new, self.cached = list(new), list(cached)
        self.lens = [a + b for a, b in zip(new, cached)]
        self.window, self.sinks, self.n = window, sinks, len(self.new)
        self.scale = scale or 1.0 / math.sqrt(self.d)
        pages = [(x + 15) // 16 for x in self.lens]
        self.mbps = mbps or max(max(pages), 1)
        self.nb = sum(pages) + 5
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(self.nb, generator=g).tolist()
        self.tables = torch.full((self.n, self.mbps), -1, dtype=torch.int32)
        for i, k in enumerate(pages):
            self.tables[i, :k] = torch.tensor(perm[:k], dtype=torch.int32)
            perm = perm[k:]
        self.cu = [0]
        for t in self.new:
            self.cu.append(self.cu[-1] + t)
        self.total = max(self.cu[-1] + gap, 1)
        self.most = max_tokens or max(max(self.new), 1)
        rnd = lambda *s: torch.randn(s, generator=g).to(TORCH[dtype])  # noqa: E731
        self.q = rnd(self.total, self.hq, self.d)
        self.k = rnd(self.nb, self.hkv, 16, self.d)
        self.v = rnd(self.nb, self.hkv, 16, self.d)

    def visible(self, b):
        """[new tokens][keys] of sequence b."""
        q = torch.arange(self.cached[b], self.lens[b])[:, None]
        k = torch.arange(self.lens[b])[None, :]
        see = k <= q
        if self.window:
            see &= (q - k < self.window) | (k < self.sinks)
        page = self.tables[b, torch.arange(self.lens[b]) // 16]
        return see & ((page >= 0) & (page < self.nb))[None, :]

    def keys(self, pool, b, h):
        """Sequence b's rows of KV head h, zeros for pages out of range."""
        pos = torch.arange(self.lens[b])
        page = self.tables[b, pos // 16].long()
        ok = (page >= 0) & (page < self.nb)
        rows = pool[page.clamp(0, self.nb - 1), h, pos % 16].double()
        return torch.where(ok[:, None], rows, torch.zeros_like(rows))

    # -- definitions ---------------------------------------------------------
    def attention(self):
        """(out, lse, bound on out's error, bound on lse's error) in 64 bits.

        The bounds add up what the kernels' arithmetic can be off by. u is the
        type's rounding, e = 2^-24 a 32-bit one. A score is a 32-bit sum of d
        products: at most (d + 2) e sum|q k| scale off, and 4 e |s| more for
        the scale in log2 units (constant, product, difference from the max,
        whose own size is at most |s| more), so its weight is off by that
        relative amount, plus 4 e for the exponential. Sums of n weights and
        the joining of partial ones: (n + 64) e. A weight is rounded to the
        type once for the product with V (u), the result once (u |out|)."""
        e, u = 2.0 ** -24, (0.0 if self.dtype == "f32" else ROUND[self.dtype])
        out = torch.zeros(self.total, self.hq, self.d, dtype=torch.float64)
        lse = torch.full((self.total, self.hq), -math.inf, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        g = self.hq // self.hkv
        for b in range(self.n):
            if not self.new[b]:
                continue
            rows = slice(self.cu[b], self.cu[b + 1])
            see = self.visible(b)
            for h in range(self.hkv):
                k, v = self.keys(self.k, b, h), self.keys(self.v, b, h)
                for j in range(h * g, (h + 1) * g):
                    q = self.q[rows, j].double()
                    s = (q @ k.T * self.scale).masked_fill(~see, -math.inf)
                    off = (q.abs() @ k.abs().T * self.scale * (self.d + 2) * e +
                           8 * e * s.abs()).masked_fill(~see, 0).amax(-1, keepdim=True)
                    top = s.amax(-1, keepdim=True)
                    p = (s - top.masked_fill(top == -math.inf, 0)).exp()
                    total = p.sum(-1, keepdim=True)
                    some = total > 0
                    vv = v.masked_fill(~see.any(0)[:, None], 0)
                    o = torch.where(some, p @ vv / total, torch.zeros_like(p @ vv))
                    size = torch.where(some, p @ vv.abs() / total, torch.zeros_like(o))
                    rel = 2 * off + (2 * len(k) + 80) * e
                    out[rows, j], lse[rows, j] = o, (top + total.log()).squeeze(-1)
                    tol[rows, j] = (rel + u) * size + (u + 4 * e) * o.abs() + 1e-30
                    ltol[rows, j] = (rel + 4 * e * (1 + lse[rows, j].abs().nan_to_num(
                        posinf=0)[:, None])).squeeze(-1)
        return out, lse, tol, ltol

    # -- calls ---------------------------------------------------------------
    def upload(self):
        self.dev = {n: getattr(self, n).to(DEV) for n in ("q", "k", "v", "tables")}
        self.dev["cu"] = torch.tensor(self.cu, dtype=torch.int32, device=DEV)
        self.dev["lens"] = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        return self

    def plan(self, kv, stream=None):
        size = kv.chunk_plan_size(self.n, self.total, self.hq, self.hkv)
        self.dev["plan"] = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
        self.build(kv, stream)
        return self

    def build(self, kv, stream=None):
        kv.chunk_plan(self.dev["cu"], self.dev["lens"], self.n, self.total, self.most, self.hq,
                      self.hkv, self.mbps, self.window, self.sinks, self.dev["plan"],
                      self.dev["plan"].numel(), stream)

    def shape(self):
        return (self.n, self.total, self.most, self.hq, self.hkv, self.d, self.mbps, self.nb,
                self.window, self.sinks, self.scale, self.dtype)

    def workspace(self, kv):
        size = kv.chunk_workspace_size(self.n, self.total, self.most, self.hq, self.hkv, self.d)
        return torch.zeros(size, dtype=torch.uint8, device=DEV)

    def run(self, kv, ws=None, out=None, lse=None, stream=None):
        d = self.dev
        ws = self.workspace(kv) if ws is None else ws
        out = torch.full_like(d["q"], 7.0) if out is None else out
        if lse is None:
            lse = torch.full((self.total, self.hq), 7.0, device=DEV)
        kv.chunk_attn(d["q"], d["k"], d["v"], d["tables"], d["plan"], out, lse, *self.shape(), ws,
                      ws.numel(), stream)
        return out, lse


def assert_within(got, want, tol, what):
    """|got - want| <= tol everywhere; NaN and infinities in the same places."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    hard = ~fin & ~torch.isnan(want)
    assert torch.equal(got[hard], want[hard]), f"{what}: infinities differ"
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or over.max() <= 0, (
        f"{what}: {int((over > 0).sum())} of {over.numel()} beyond their bound, by up to "
        f"{float(over.max()):.3e}")




def step_scores(step, lse, prev=None):
    """(weights [n][hkv][slots], bound on their error) in 64 bits, from the
    32-bit lse given. A weight is off by what its score is (as in
    Step.attention) and 4 e |lse| for the subtraction in log2 units; the sum of
    r weights by (r + 8) e of it."""
    e = 2.0 ** -24
    slots, g = step.mbps * 16, step.hq // step.hkv
    w = torch.zeros(step.n, step.hkv, slots, dtype=torch.float64)
    tol = torch.zeros_like(w)
    for b in range(step.n):
        if not step.new[b]:
            continue
        rows, n = slice(step.cu[b], step.cu[b + 1]), step.lens[b]
        see = step.visible(b)
        for h in range(step.hkv):
            k = step.keys(step.k, b, h)
            for j in range(h * g, (h + 1) * g):
                q = step.q[rows, j].double()
                s = (q @ k.T * step.scale).masked_fill(~see, -math.inf)
                l = lse[rows, j].double()[:, None]
                p = torch.where(see & (l > -math.inf), (s - l).exp(), torch.zeros_like(s))
                off = q.abs() @ k.abs().T * step.scale * (step.d + 2) * e + 16 * e * (
                    s.abs().nan_to_num(posinf=0) + l.abs().nan_to_num(posinf=0) + 1)
                w[b, h, :n] += p.sum(0)
                tol[b, h, :n] += (p * (2 * off + (step.new[b] * g + 8) * e)).sum(0)
        if prev is not None:
            w[b, :, :step.cached[b]] += prev[b, :, :step.cached[b]].double()
            tol[b, :, :n] += 2 * e * w[b, :, :n].abs()
    return w, tol + 1e-30


def evict_reference(scores, lens, budget, sinks, recent):
    """Kept slots [layers][n][hkv] as lists, from the definition."""
    layers, n, hkv, _ = scores.shape
    kept = [[[None] * hkv for _ in range(n)] for _ in range(layers)]
    for l in range(layers):
        for b in range(n):
            for h in range(hkv):
                size = lens[b]
                if size <= budget:
                    kept[l][b][h] = list(range(size))
                    continue
                w = scores[l, b, h, :size].tolist()
                middle = range(sinks, size - recent)
                order = sorted(middle, key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0,
                                                      i))
                best = sorted(order[:budget - sinks - recent])
                kept[l][b][h] = list(range(sinks)) + best + list(range(size - recent, size))
    return kept
