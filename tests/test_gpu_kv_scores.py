"""The weights cached keys receive (rlse_kv_scores) against their definition in
64 bits."""
import math

import pytest
import torch

from chunk_helpers import DEV, Step, assert_within, step_scores
from test_gpu_chunk import HEADS, STEPS, WINDOWS

pytestmark = pytest.mark.gpu


def scores(kv, step, lse, prev=None, out=None, stream=None):
    d = step.dev
    if out is None:
        out = torch.full((step.n, step.hkv, step.mbps * 16), 7.0, device=DEV)
    kv.kv_scores(d["q"], d["k"], d["tables"], d["plan"], lse, prev, out, *step.shape(), stream)
    return out


def check(kv, step, what, prev=None, seen=None):
    want_lse = (seen or step.attention())[1].float()
    step.upload().plan(kv)
    got = scores(kv, step, want_lse.to(DEV), None if prev is None else prev.to(DEV))
    want, tol = step_scores(step, want_lse, prev)
    torch.cuda.synchronize()
    kv.workspace_check(step.dev["plan"])
    for b in range(step.n):
        n = step.lens[b] if step.new[b] else 0
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"{what} sequence {b}")
        assert (got[b, :, n:] == 7).all(), f"{what}: slots after sequence {b}"
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_causal(kv, heads, name, dtype):
    step = Step(31, dtype, heads, *STEPS[name], gap=3)
    check(kv, step, name)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", WINDOWS, ids=lambda w: f"w{w[0]}s{w[1]}")
@pytest.mark.parametrize("name", list(STEPS))
def test_window_added_to_what_was_there(kv, name, window, dtype):
    heads = (16, 8, 128) if dtype != "f16" else (14, 2, 64)
    step = Step(32, dtype, heads, *STEPS[name], *window)
    prev = torch.rand(step.n, step.hkv, step.mbps * 16,
                      generator=torch.Generator().manual_seed(5)) * 3
    check(kv, step, f"{name} {window}", prev)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 80]])
def test_in_place_over_steps(kv, new):
    """prev is scores itself: two steps' weights add up, and every query gives
    one in all."""
    step = Step(33, "bf16", (16, 8, 128), new, [40, 200, 7], mbps=20)
    want_lse = step.attention()[1].float()
    first, tol = step_scores(step, want_lse)
    step.upload().plan(kv)
    lse = want_lse.to(DEV)
    acc = scores(kv, step, lse, None)
    acc = scores(kv, step, lse, acc, acc)
    for b in range(3):
        c, n = step.cached[b], step.lens[b]
        assert_within(acc[b, :, :c], 2 * first[b, :, :c], 4 * tol[b, :, :c], "older keys")
        assert_within(acc[b, :, c:n], first[b, :, c:n], tol[b, :, c:n], "new keys")
    got = scores(kv, step, lse, None)
    for b in range(3):
        total = got[b, :, :step.lens[b]].double().sum(-1).cpu()
        assert torch.allclose(total, torch.full_like(total, 2.0 * new[b]), rtol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_masked_places_hold_anything(kv, new, dtype):
    """Pages no token sees are not read; NaN in stale slots and hidden keys
    changes nothing; rows that saw nothing give nothing."""
    step = Step(34, dtype, (8, 4, 64), [new, new, new], [177, 850, 20], window=35, sinks=3)
    seen = step.attention()
    want, tol = step_scores(step, seen[1].float())
    for b in range(2):
        see = step.visible(b).any(0)
        for pg in range((step.lens[b] + 15) // 16):
            mine = slice(pg * 16, min(pg * 16 + 16, step.lens[b]))
            if not see[mine].any():
                step.tables[b, pg] = -7
                continue
            for pos in range(pg * 16, pg * 16 + 16):
                if pos >= step.lens[b] or not see[pos]:
                    step.k[step.tables[b, pg], :, pos % 16] = math.nan
    step.tables[2] = step.nb + 1  # the third sequence sees nothing
    lse = seen[1].float()
    lse[step.cu[2]:step.cu[3]] = -math.inf
    want[2], tol[2] = 0, 1e-30
    step.upload().plan(kv)
    got = scores(kv, step, lse.to(DEV))
    for b in range(3):
        n = step.lens[b]
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"sequence {b}")


def test_follows_the_attention(kv):
    """The lse of rlse_chunk_attn, the same plan."""
    step = Step(35, "bf16", (28, 4, 128), [1, 9, 200], [500, 60, 100]).upload().plan(kv)
    _, lse = step.run(kv)
    got = scores(kv, step, lse)
    want, tol = step_scores(step, lse.cpu())
    for b in range(3):
        n = step.lens[b]
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"sequence {b}")


def test_same_bits_captured_and_on_another_stream(kv):
    step = Step(36, "f16", (16, 8, 128), [1, 3, 260, 1], [3000, 60, 100, 40]).upload().plan(kv)
    _, lse = step.run(kv)
    torch.cuda.synchronize()
    want = scores(kv, step, lse)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        other = scores(kv, step, lse, stream=st)
    st.synchronize()
    assert torch.equal(other, want)
    out = torch.full_like(want, 7.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        scores(kv, step, lse, out=out, stream=st)
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        scores(kv, step, lse)


def test_plan_of_another_step(kv):
    step = Step(37, "bf16", (16, 8, 128), [1, 50], [20, 40]).upload().plan(kv)
    _, lse = step.run(kv)
    step.sinks = 1
    assert (scores(kv, step, lse) == 7).all()
    with pytest.raises(kv.RlseError, match="other arguments"):
        kv.workspace_check(step.dev["plan"])


def test_pool_offsets_past_32_bits(kv):
    step = Step(38, "bf16", (16, 8, 128), [1, 40], [90, 33])
    lse = step.attention()[1].float()
    want, tol = step_scores(step, lse)
    step.upload()
    blocks = 2 ** 31 // (8 * 16 * 128) + step.nb
    big = torch.empty((blocks, 8, 16, 128), dtype=torch.bfloat16, device=DEV)
    big[-step.nb:] = step.dev["k"]
    step.dev["k"] = big
    step.dev["tables"] = torch.where(step.dev["tables"] >= 0,
                                     step.dev["tables"] + (blocks - step.nb), -1)
    step.nb = blocks
    step.plan(kv)
    got = scores(kv, step, lse.to(DEV))
    for b in range(2):
        n = step.lens[b]
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"sequence {b}")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_key_of_score_minus_infinity(kv, new, dtype):
    """A visible key whose score is -inf in every row has no weight, and the
    others theirs."""
    step = Step(39, dtype, (6, 2, 64), [new, new], [200, 75])
    step.q[..., 7] = 1.0
    for b, at in ((0, 3), (0, 37), (1, 70)):
        step.k[step.tables[b, at // 16], :, at % 16, 7] = -math.inf
    want_lse = torch.zeros(step.total, 6)
    for b in range(2):
        rows = slice(step.cu[b], step.cu[b + 1])
        for j in range(6):
            s = step.q[rows, j].double() @ step.keys(step.k, b, j // 3).T * step.scale
            want_lse[rows, j] = s.masked_fill(~step.visible(b), -math.inf).logsumexp(-1).float()
    step.upload().plan(kv)
    got = scores(kv, step, want_lse.to(DEV)).cpu()
    for b, at in ((0, 3), (0, 37), (1, 70)):
        assert (got[b, :, at] == 0).all()
        step.k[step.tables[b, at // 16], :, at % 16, 7] = -1e4 if dtype != "f32" else -1e5
    want, tol = step_scores(step, want_lse)
    for b in range(2):
        n = step.lens[b]
        keys = torch.isfinite(step.keys(step.k, b, 0)).all(-1)
        assert keys.all()
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"sequence {b}")


def test_flag_for_shared_pages(kv):
    step = Step(40, "bf16", (16, 8, 128), [1, 2, 40], [300, 310, 320])
    step.tables[1:, :18] = step.tables[0, :18]
    step.upload().plan(kv)
    _, lse = step.run(kv)
    got, d = scores(kv, step, lse), step.dev
    other = torch.full_like(got, 7.0)
    kv.kv_scores(d["q"], d["k"], d["tables"], d["plan"], lse, None, other, *step.shape(),
                 shared_pages=True)
    assert torch.equal(got, other)
    want, tol = step_scores(step, lse.cpu())
    for b in range(3):
        n = step.lens[b]
        assert_within(got[b, :, :n], want[b, :, :n], tol[b, :, :n], f"sequence {b}")


def test_many_sequences(kv):
    """More sequences than workgroups."""
    step = Step(41, "bf16", (4, 2, 64), [i % 3 for i in range(700)],
                [(i * 37) % 90 for i in range(700)])
    check(kv, step, "many")


@pytest.mark.parametrize("window", [(0, 0), (40, 3)])
def test_many_chunks(kv, window):
    """More key blocks than are sorted by the rows they meet."""
    step = Step(42, "bf16", (16, 8, 64), [17 + i % 20 for i in range(330)],
                [(i * 37) % 200 for i in range(330)], *window)
    check(kv, step, "many chunks")
