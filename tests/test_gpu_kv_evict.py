"""Eviction by accumulated weight (rlse_kv_evict) against its definition: exact,
to the bit, in what stays, in which order, and what is left alone."""
import math

import pytest
import torch

from chunk_helpers import DEV, TORCH, evict_reference

pytestmark = pytest.mark.gpu


class Cache:
    def __init__(self, seed, dtype, layers, hkv, d, lens, budget, sinks, recent, mbps=None,
                 weights="spread", spare=2):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.layers, self.hkv, self.d = dtype, layers, hkv, d
        self.lens, self.budget, self.sinks, self.recent = lens, budget, sinks, recent
        self.n = len(lens)
        pages = [max(0, x + 15) // 16 for x in lens]
        self.mbps = max(mbps or max(pages), (budget + 15) // 16)
        self.nbps = (budget + 15) // 16 + spare
        fresh = [(min(max(x, 0), budget) + 15) // 16 for x in lens]
        self.nb = sum(pages) + sum(fresh) + 3
        perm = torch.randperm(self.nb, generator=g).tolist()
        self.tables = torch.full((self.n, self.mbps), -1, dtype=torch.int32)
        self.new_tables = torch.full((self.n, self.nbps), -1, dtype=torch.int32)
        for i, (a, b) in enumerate(zip(pages, fresh)):
            a = min(a, self.mbps)
            self.tables[i, :a] = torch.tensor(perm[:a], dtype=torch.int32)
            self.new_tables[i, :b] = torch.tensor(perm[a:a + b], dtype=torch.int32)
            perm = perm[a + b:]
        shape = (layers, 2, self.nb, hkv, 16, d)  # K and V of a layer together, as the pool's
        self.pool = torch.randn(shape, generator=g).to(TORCH[dtype])
        w = torch.randn(layers, self.n, hkv, self.mbps * 16, generator=g).mul(2).exp()
        if weights == "ties":
            w = torch.randint(0, 3, w.shape, generator=g).float()
        elif weights == "equal":
            w = torch.ones_like(w)
        elif weights == "odd":
            some = torch.rand(w.shape, generator=g)
            w[some < 0.1] = math.nan
            w[(some > 0.2) & (some < 0.3)] = math.inf
            w[(some > 0.3) & (some < 0.4)] = -math.inf
            w[(some > 0.4) & (some < 0.5)] = 0.0
            w[(some > 0.5) & (some < 0.6)] = -0.0
            w[(some > 0.6) & (some < 0.7)] *= -1
            w[(some > 0.7) & (some < 0.75)] = 1e-42
        elif weights == "close":
            w = 1 + torch.randint(0, 4, w.shape, generator=g).float() * 2.0 ** -23
        self.scores = w

    def upload(self):
        self.dev = {n: getattr(self, n).to(DEV) for n in ("pool", "scores", "tables", "new_tables")}
        self.dev["lens"] = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.dev["new_lens"] = torch.full((self.n,), 9, dtype=torch.int32, device=DEV)
        self.dev["new_scores"] = torch.full_like(self.dev["scores"], -5.0)
        self.dev["keep"] = torch.full((self.layers, self.n, self.hkv, self.budget), 9,
                                      dtype=torch.int32, device=DEV)
        return self

    def run(self, kv, stream=None):
        d = self.dev
        kv.kv_evict(d["pool"][0, 0], d["pool"][0, 1], d["pool"][0].numel(), self.layers,
                    d["tables"], d["lens"], d["scores"], d["scores"][0].numel(), d["new_tables"],
                    d["new_lens"], d["new_scores"], d["keep"], self.n, self.hkv, self.d,
                    self.mbps, self.nbps, self.nb, self.budget, self.sinks, self.recent,
                    self.dtype, stream)

    def check(self, kept=None):
        lens = [x if 0 <= x <= self.mbps * 16 else 0 for x in self.lens]
        kept = kept or evict_reference(self.scores, lens, self.budget, self.sinks, self.recent)
        pool, scores = self.pool.clone(), torch.full_like(self.scores, -5.0)
        keep = torch.full((self.layers, self.n, self.hkv, self.budget), -1, dtype=torch.int32)
        for l in range(self.layers):
            for b in range(self.n):
                for h in range(self.hkv):
                    src = torch.tensor(kept[l][b][h], dtype=torch.long)
                    if not len(src):
                        continue
                    to = torch.arange(len(src))
                    keep[l, b, h, :len(src)] = src.int()
                    scores[l, b, h, :len(src)] = self.scores[l, b, h, src]
                    old = self.tables[b, src // 16].long()
                    new = self.new_tables[b, to // 16].long()
                    ok = (old >= 0) & (old < self.nb) & (new >= 0) & (new < self.nb)
                    pool[l, :, new[ok], h, to[ok] % 16] = self.pool[l, :, old[ok], h, src[ok] % 16]
        torch.cuda.synchronize()
        assert self.dev["new_lens"].tolist() == [min(x, self.budget) for x in lens]
        assert torch.equal(self.dev["keep"].cpu(), keep)
        bits = lambda t: t.contiguous().view(torch.int32 if t.element_size() == 4  # noqa: E731
                                             else torch.int16)
        assert torch.equal(bits(self.dev["new_scores"].cpu()), bits(scores))
        assert torch.equal(bits(self.dev["pool"].cpu()), bits(pool))
        assert torch.equal(bits(self.dev["scores"].cpu()), bits(self.scores))


@pytest.mark.parametrize("weights", ["spread", "ties", "equal", "odd", "close"])
@pytest.mark.parametrize("dtype,layers,hkv,d,lens,budget,sinks,recent", [
    ("bf16", 2, 8, 128, [100, 33, 32, 5, 0], 32, 4, 8),
    ("f32", 1, 2, 64, [700], 129, 0, 0),
    ("f32", 2, 2, 128, [300, 17], 200, 1, 50),
    ("f16", 3, 2, 64, [500, 1200, 64], 63, 16, 40),
    ("bf16", 1, 4, 128, [90, 91], 90, 0, 90),
    ("f16", 1, 1, 128, [50, 49, 1], 1, 0, 0),
    ("bf16", 1, 3, 64, [2000, 1999], 1998, 3, 5),
])
def test_what_stays(kv, dtype, layers, hkv, d, lens, budget, sinks, recent, weights):
    c = Cache(41, dtype, layers, hkv, d, lens, budget, sinks, recent, weights=weights).upload()
    c.run(kv)
    c.check()


@pytest.mark.parametrize("weights", ["spread", "ties", "odd"])
def test_long_cache(kv, weights):
    """More keys than the selection holds on chip."""
    c = Cache(42, "bf16", 1, 2, 64, [20011, 8193 + 17, 9000], 1234, 4, 100, weights=weights)
    c.upload().run(kv)
    c.check()


def test_lengths_and_pages_out_of_range(kv):
    """A length that does not fit counts as 0; rows of pages out of range are
    not copied, the rest are."""
    c = Cache(43, "bf16", 2, 2, 64, [200, 120, 90], 50, 2, 10)
    c.tables[1, 0] = c.nb
    c.tables[1, 5] = -1
    c.new_tables[2, 1] = c.nb + 3
    c.lens[0] = c.mbps * 16 + 1
    c.upload().run(kv)
    c.check()
    c.lens[0] = -1
    c.upload().run(kv)
    c.check()


def test_short_sequences_may_keep_their_pages(kv):
    c = Cache(44, "f16", 2, 4, 128, [40, 300, 48], 48, 0, 4)
    for b in (0, 2):
        c.new_tables[b, :3] = c.tables[b, :3]
    c.upload().run(kv)
    c.check()


def test_shared_pages_are_only_read(kv):
    """Two sequences forked from one prefix, each with its own weights."""
    c = Cache(45, "bf16", 1, 2, 128, [150, 170], 40, 4, 4)
    c.tables[1, :8] = c.tables[0, :8]
    c.upload().run(kv)
    c.check()


def test_again_captured_and_on_another_stream(kv):
    c = Cache(46, "bf16", 2, 4, 64, [400, 77, 1000], 100, 4, 20)
    kept = evict_reference(c.scores, c.lens, c.budget, c.sinks, c.recent)
    c.upload()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c.run(kv, st)
    st.synchronize()
    c.check(kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        c.run(kv, st)
    for _ in range(3):
        for name, fill in (("keep", 9), ("new_lens", 9), ("new_scores", -5.0)):
            c.dev[name].fill_(fill)
        c.dev["pool"].copy_(c.pool)
        graph.replay()
        torch.cuda.synchronize()
        c.check(kept)


def test_pool_offsets_past_32_bits(kv):
    c = Cache(47, "f32", 1, 2, 128, [100], 30, 2, 3)
    kept = evict_reference(c.scores, c.lens, c.budget, c.sinks, c.recent)
    blocks = 2 ** 31 // (2 * 16 * 128) + c.nb
    c.upload()
    small, first = c.dev["pool"], blocks - c.nb
    big = torch.empty((1, 2, blocks, 2, 16, 128), device=DEV)
    big[:, :, first:] = small
    c.dev["pool"] = big
    for name in ("tables", "new_tables"):
        c.dev[name] = torch.where(c.dev[name] >= 0, c.dev[name] + first, -1)
    nb, c.nb = c.nb, blocks
    c.run(kv)
    c.nb = nb
    torch.cuda.synchronize()
    c.dev["pool"] = big[:, :, first:].clone()
    c.check(kept)


def test_weights_between_each_other(kv):
    """Old and new weights in one buffer, layer by layer."""
    c = Cache(48, "bf16", 3, 2, 64, [200, 90], 50, 2, 10).upload()
    both = torch.full((3, 2) + tuple(c.scores.shape[1:]), -5.0, device=DEV)
    both[:, 0] = c.dev["scores"]
    d = c.dev
    kv.kv_evict(d["pool"][0, 0], d["pool"][0, 1], d["pool"][0].numel(), 3, d["tables"], d["lens"],
                both[0, 0], both[0].numel(), d["new_tables"], d["new_lens"], both[0, 1],
                d["keep"], c.n, c.hkv, c.d, c.mbps, c.nbps, c.nb, c.budget, c.sinks, c.recent,
                c.dtype)
    d["scores"], d["new_scores"] = both[:, 0].contiguous(), both[:, 1].contiguous()
    c.check()
