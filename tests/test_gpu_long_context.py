"""A long chat served from a cache of bounded size, as an engine would: prompt
chunks and decode steps of several sequences in ragged steps, the keys' weights
added up, the cache cut to a budget into fresh pages when it grows past a limit,
and on. Every step is compared with the same run in 64 bits."""
import math

import pytest
import torch

from chunk_helpers import DEV, ROUND, TORCH

pytestmark = pytest.mark.gpu

HQ, HKV, D, LAYERS = 8, 2, 64, 2
BUDGET, SINKS, RECENT, LIMIT = 48, 4, 16, 96


class Chat:
    """One sequence: its 64-bit keys, values and weights of every layer and KV
    head, and how many tokens it has seen (their true positions)."""

    def __init__(self, name):
        self.name, self.seen, self.pages = name, 0, []
        self.k = [[torch.zeros(0, D, dtype=torch.float64) for _ in range(HKV)]
                  for _ in range(LAYERS)]
        self.v = [[torch.zeros(0, D, dtype=torch.float64) for _ in range(HKV)]
                  for _ in range(LAYERS)]
        self.w = [[torch.zeros(0, dtype=torch.float64) for _ in range(HKV)]
                  for _ in range(LAYERS)]

    @property
    def length(self):
        return len(self.w[0][0])


def rope64(x, positions, cos, sin):
    """NeoX rotation of rows x [n][heads][D] by the tables' own (rounded) values."""
    c, s = cos[positions].double()[:, None], sin[positions].double()[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 40])
def test_bounded_cache(kv, dtype, window):
    t = TORCH[dtype]
    g = torch.Generator().manual_seed(7)
    nb, mbps, max_batch = 80, 8, 3
    bm = kv.BlockManager(nb)
    pool = kv.KVPool(LAYERS, nb, HKV, D, dtype)
    cos_b, sin_b = kv.rope_tables(1e6, D, 4096, dtype)
    cos, sin = (torch.frombuffer(bytearray(b), dtype=t).view(4096, D // 2) for b in (cos_b, sin_b))
    cos_d, sin_d = cos.to(DEV), sin.to(DEV)
    layers = [pool.layer(l) for l in range(LAYERS)]
    slots = mbps * 16
    scores = torch.zeros(LAYERS, max_batch, HKV, slots, device=DEV)
    spare = torch.zeros_like(scores)
    ws = torch.zeros(kv.chunk_workspace_size(max_batch, 80, 80, HQ, HKV, D), dtype=torch.uint8,
                     device=DEV)
    chats = [Chat("a"), Chat("b"), Chat("c")]
    scale, evictions = 1.0 / math.sqrt(D), 0
    # a's prompt in two chunks while b answers, c idle at first; then all decode
    plan_of_steps = [[40, 5, 0], [37, 1, 0], [1, 1, 70]] + [[1, 1, 1]] * 24 + [[1, 30, 1], [1, 1, 1]]
    # then more of a's and c's prompts, which cuts the caches a second time
    plan_of_steps += [[30, 1, 1], [1, 1, 45], [1, 1, 1]]
    for new in plan_of_steps:
        # cut the caches that would outgrow the limit, all layers at once
        cut = [c.length + n > LIMIT for c, n in zip(chats, new)]
        if any(cut):
            evictions += 1
            lens = torch.tensor([c.length for c in chats], dtype=torch.int32, device=DEV)
            tables = torch.zeros(max_batch, mbps, dtype=torch.int32)
            fresh = torch.zeros(max_batch, (BUDGET + 15) // 16, dtype=torch.int32)
            old = [c.pages for c in chats]
            for i, c in enumerate(chats):
                tables[i, :len(c.pages)] = torch.tensor(c.pages, dtype=torch.int32)
                if c.length:
                    c.name += "+"
                    c.pages = bm.allocate(c.name, min(c.length, BUDGET))
                    fresh[i, :len(c.pages)] = torch.tensor(c.pages, dtype=torch.int32)
            new_lens = torch.zeros(max_batch, dtype=torch.int32, device=DEV)
            keep = torch.zeros(LAYERS, max_batch, HKV, BUDGET, dtype=torch.int32, device=DEV)
            kv.kv_evict(layers[0][0], layers[0][1], pool.layer_stride_elems, LAYERS,
                        tables.to(DEV), lens, scores, scores[0].numel(), fresh.to(DEV), new_lens,
                        spare, keep, max_batch, HKV, D, mbps, fresh.shape[1], nb, BUDGET, SINKS,
                        RECENT, dtype)
            torch.cuda.synchronize()
            scores, spare = spare, scores
            keep = keep.cpu()
            for i, c in enumerate(chats):
                if old[i]:
                    bm.release(c.name[:-1])
                count = min(c.length, BUDGET)
                assert int(new_lens[i]) == count
                for l in range(LAYERS):
                    for h in range(HKV):
                        at = keep[l, i, h, :count].long()
                        # the heaviest by the device's own (32-bit) weights: every
                        # one kept is at least as heavy as every one dropped, to
                        # the weights' error
                        w = c.w[l][h]
                        if c.length > BUDGET:
                            mid = torch.arange(SINKS, c.length - RECENT)
                            stays = torch.isin(mid, at)
                            assert w[mid[stays]].min() >= w[mid[~stays]].max() - 1e-2
                            assert (at[:SINKS] == torch.arange(SINKS)).all()
                        c.k[l][h], c.v[l][h], c.w[l][h] = c.k[l][h][at], c.v[l][h][at], w[at]
        # grow the pages
        for c, n in zip(chats, new):
            while len(c.pages) * 16 < c.length + n:
                c.pages = (c.pages + [bm.allocate_block(c.name)] if c.pages else
                           bm.allocate(c.name, c.length + n))
        batch, total = max_batch, sum(new)
        tables = torch.zeros(batch, mbps, dtype=torch.int32)
        for i, c in enumerate(chats):
            tables[i, :len(c.pages)] = torch.tensor(c.pages, dtype=torch.int32)
        tables = tables.to(DEV)
        cu = [sum(new[:i]) for i in range(batch + 1)]
        lens = [c.length + n for c, n in zip(chats, new)]
        seq = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], dtype=torch.int32)
        slot = torch.tensor([c.length + j for c, n in zip(chats, new) for j in range(n)],
                            dtype=torch.int32)
        true = torch.tensor([c.seen + j for c, n in zip(chats, new) for j in range(n)],
                            dtype=torch.int32)
        plan = torch.zeros(kv.chunk_plan_size(batch, total, HQ, HKV), dtype=torch.uint8, device=DEV)
        most = max(new)
        kv.chunk_plan(torch.tensor(cu, dtype=torch.int32, device=DEV),
                      torch.tensor(lens, dtype=torch.int32, device=DEV), batch, total, most, HQ,
                      HKV, mbps, window, SINKS if window else 0, plan, plan.numel())
        shape = (batch, total, most, HQ, HKV, D, mbps, nb, window, SINKS if window else 0, scale,
                 dtype)
        for l, (kp, vp) in enumerate(layers):
            q, k, v = (torch.randn(total, n, D, generator=g).to(t) for n in (HQ, HKV, HKV))
            qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
            # rotated at their true positions, appended at the cache's slots
            kv.rope(qd, kd, cos_d, sin_d, true.to(DEV), total, HQ, HKV, D, 4096, dtype)
            kv.kv_append(kd, vd, kp, vp, tables, batch, seq.to(DEV), slot.to(DEV), total, HKV, D,
                         mbps, nb, dtype)
            out = torch.zeros_like(qd)
            lse = torch.zeros(total, HQ, device=DEV)
            kv.chunk_attn(qd, kp, vp, tables, plan, out, lse, *shape, ws, ws.numel())
            kv.kv_scores(qd, kp, tables, plan, lse, scores[l], scores[l], *shape)
            torch.cuda.synchronize()
            # the rotation itself, to the type's rounding (three of them)
            u = ROUND[dtype]
            for x, xd in ((q, qd), (k, kd)):
                r = rope64(x.double(), true.long(), cos, sin)
                size = x.double().abs().amax() * 2
                assert (xd.cpu().double() - r).abs().max() <= 4 * u * size
            qd, kd = qd.cpu().double(), kd.cpu().double()
            for i, (c, n) in enumerate(zip(chats, new)):
                rows = slice(cu[i], cu[i + 1])
                if not n:
                    continue
                for h in range(HKV):
                    c.k[l][h] = torch.cat([c.k[l][h], kd[rows, h]])
                    c.v[l][h] = torch.cat([c.v[l][h], v[rows, h].double()])
                    here = torch.arange(lens[i])
                    at = here[lens[i] - n:, None]
                    see = here[None] <= at
                    if window:
                        see &= (at - here[None] < window) | (here[None] < SINKS)
                    gained = torch.zeros(lens[i], dtype=torch.float64)
                    for j in range(h * HQ // HKV, (h + 1) * HQ // HKV):
                        s = (qd[rows, j] @ c.k[l][h].T * scale).masked_fill(~see, -math.inf)
                        p = s.softmax(-1)
                        want = p @ c.v[l][h]
                        size = p @ c.v[l][h].abs()
                        # p rounded once, the result once; 32-bit sums beside them
                        tol = ((0 if dtype == "f32" else u) + 2e-4) * size + u * want.abs()
                        assert ((out[rows, j].cpu().double() - want).abs() <= tol).all()
                        assert torch.allclose(lse[rows, j].cpu().double(), s.logsumexp(-1),
                                              atol=2e-4)
                        gained += p.sum(0)
                    old = torch.cat([c.w[l][h], torch.zeros(n, dtype=torch.float64)])
                    c.w[l][h] = old + gained
                    got = scores[l, i, h, :lens[i]].cpu().double()
                    assert torch.allclose(got, c.w[l][h], rtol=1e-3, atol=1e-3)
        for c, n in zip(chats, new):
            c.seen += n
        kv.workspace_check(plan)
    assert evictions >= 2 and all(c.length <= LIMIT for c in chats)
    assert bm.free_count() == nb - sum(len(c.pages) for c in chats)
    pool.close()
