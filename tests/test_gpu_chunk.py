"""Attention of ragged steps (rlse_chunk_plan, rlse_chunk_attn) against its
definition in 64 bits: decode steps, drafts and prompt chunks, windows and
sinks, and what masked places, pages and rows may hold."""
import copy
import math

import pytest
import torch

from chunk_helpers import DEV, Step, assert_within

pytestmark = pytest.mark.gpu

HEADS = [(16, 8, 128), (14, 2, 64), (28, 4, 128), (4, 4, 64), (20, 1, 128), (40, 1, 64)]
# new tokens and cached keys of every sequence
STEPS = {
    "one": ([1], [0]),
    "one_long": ([1], [2999]),
    "step": ([1, 1, 1, 1, 1], [0, 15, 16, 130, 1023]),
    "draft": ([2, 5, 1, 4], [3, 200, 31, 64]),
    "prompt": ([77], [0]),
    "chunks": ([33, 1, 100, 0, 17, 260], [0, 47, 201, 9, 16, 5]),
    "long_chunk": ([300, 70], [700, 1000]),
}
WINDOWS = [(0, 0), (1, 0), (16, 4), (40, 0), (100, 33), (5000, 4)]


def check(step, kv, what):
    out, lse = step.run(kv)
    want, wlse, tol, ltol = step.attention()
    torch.cuda.synchronize()
    kv.workspace_check(step.dev["plan"])
    covered = torch.zeros(step.total, dtype=torch.bool)
    covered[:step.cu[-1]] = True
    assert_within(out[covered.to(DEV)], want[covered], tol[covered], what + " out")
    assert_within(lse[covered.to(DEV)], wlse[covered], ltol[covered], what + " lse")
    assert (out[step.cu[-1]:] == 7).all() and (lse[step.cu[-1]:] == 7).all(), "rows after the last"
    return out, lse


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_causal(kv, heads, name, dtype):
    step = Step(1, dtype, heads, *STEPS[name], gap=3).upload().plan(kv)
    check(step, kv, name)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", WINDOWS, ids=lambda w: f"w{w[0]}s{w[1]}")
@pytest.mark.parametrize("name", list(STEPS))
def test_window(kv, name, window, dtype):
    heads = (16, 8, 128) if dtype != "f16" else (14, 2, 64)
    step = Step(2, dtype, heads, *STEPS[name], *window).upload().plan(kv)
    check(step, kv, f"{name} {window}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_pages_no_token_sees_are_not_read(kv, new, dtype):
    """Under a window the entries between the sinks' pages and the window's may
    be anything; the pages they named hold NaN here."""
    step = Step(3, dtype, (8, 2, 64), [new, new], [900, 333], window=50, sinks=20)
    want = step.attention()
    for b in range(2):
        first = step.cached[b] - 50 + 1
        for pg in range(2, first // 16):
            step.k[step.tables[b, pg]] = math.nan
            step.v[step.tables[b, pg]] = math.nan
            step.tables[b, pg] = [-1, 2 ** 31 - 1, -2 ** 31][pg % 3]
    step.upload().plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want[0], want[2], "out")
    assert_within(lse, want[1], want[3], "lse")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new", [1, 6, 70])
def test_masked_places_hold_anything(kv, new, dtype, bad):
    """Stale slots behind the last key, and keys outside a window that share a
    page with visible ones, hold NaN or infinities in K and V."""
    step = Step(4, dtype, (8, 4, 128), [new, new], [77, 150], window=35, sinks=3)
    want = step.attention()
    for b in range(2):
        see = step.visible(b).any(0)
        hidden = [int(i) for i in torch.nonzero(~see).flatten()]
        hidden += range(step.lens[b], (step.lens[b] + 15) // 16 * 16)
        for pos in hidden:
            pg = int(step.tables[b, pos // 16])
            step.k[pg, :, pos % 16] = bad
            step.v[pg, :, pos % 16] = bad
    step.upload().plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want[0], want[2], "out")
    assert_within(lse, want[1], want[3], "lse")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new", [6, 70, 300])
def test_values_reach_only_rows_that_see_them(kv, new, dtype, bad):
    """A new token whose V is not finite spoils its own row and later ones, in
    its dimensions; the rows before it are as if it were not there."""
    step = Step(5, dtype, (8, 4, 64), [new], [40])
    want, wlse, tol, ltol = step.attention()
    at = step.cached[0] + new // 2
    step.v[step.tables[0, at // 16], 1, at % 16, 5] = bad
    heads = slice(2, 4)
    want[new // 2:, heads, 5] = bad
    step.upload().plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want, tol, "out")
    assert_within(lse, wlse, ltol, "lse")


def test_both_infinities_give_nan(kv):
    step = Step(6, "bf16", (4, 2, 64), [40], [0])
    want, _, tol, _ = step.attention()
    for pos, bad in ((10, math.inf), (20, -math.inf)):
        step.v[step.tables[0, pos // 16], 0, pos % 16, 3] = bad
    want[10:20, :2, 3] = math.inf
    want[20:, :2, 3] = math.nan
    step.upload().plan(kv)
    assert_within(step.run(kv)[0], want, tol, "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 60])
def test_nan_query_and_key(kv, new, dtype):
    """A NaN query spoils its row, a NaN key the rows that see it."""
    step = Step(7, dtype, (4, 2, 64), [new, new], [30, 30])
    want, wlse, tol, ltol = step.attention()
    step.q[0, 3] = math.nan
    at = step.cached[1] + new // 2
    step.k[step.tables[1, at // 16], 0, at % 16, 0] = math.nan
    rows = slice(new + new // 2, 2 * new)
    want[0, 3], wlse[0, 3] = math.nan, math.nan
    want[rows, :2], wlse[rows, :2] = math.nan, math.nan
    step.upload().plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want, tol, "out")
    assert_within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new", [1, 50])
def test_pages_out_of_range_give_nothing(kv, new, dtype):
    """Rows all of whose pages are out of range are zeros with lse -inf."""
    step = Step(8, dtype, (8, 2, 128), [new, new, new], [100, 100, 3])
    step.tables[0, :] = step.nb
    step.tables[1, 2] = -5
    step.tables[1, 4] = step.nb + 7
    step.upload().plan(kv)
    out, lse = check(step, kv, "invalid pages")
    assert (out[:new] == 0).all() and (lse[:new] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_and_small_scores(kv, dtype):
    """Scores that grow along the keys by far more than a lazy max allows."""
    step = Step(9, dtype, (4, 2, 64), [1, 40], [200, 100], scale=1.0)
    for pos in range(200):
        step.k[step.tables[0, pos // 16], :, pos % 16] *= pos / 20
    check(step.upload().plan(kv), kv, "growing scores")


@pytest.mark.parametrize("dtype,heads,new,cached", [
    ("bf16", (16, 8, 128), [1], [40000]),
    ("f32", (14, 2, 64), [2], [20000]),
    ("f16", (32, 8, 128), [40], [9000]),
    ("bf16", (14, 2, 64), [600, 1], [3000, 8000]),
    ("f32", (4, 1, 64), [100], [5000]),
])
def test_tiles_cut_between_workgroups(kv, dtype, heads, new, cached):
    """Few rows over long contexts: their keys are spread over the chip and
    the pieces joined, twice to the same bits in one workspace."""
    step = Step(10, dtype, heads, new, cached).upload().plan(kv)
    check(step, kv, "pieces")
    ws = step.workspace(kv)
    a, la = step.run(kv, ws)
    for _ in range(3):
        b, lb = step.run(kv, ws)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_lse_may_be_left_out(kv):
    step = Step(11, "bf16", (16, 8, 128), [1, 30], [100, 0]).upload().plan(kv)
    d, ws = step.dev, step.workspace(kv)
    with_lse, _ = step.run(kv, ws)
    out = torch.zeros_like(d["q"])
    kv.chunk_attn(d["q"], d["k"], d["v"], d["tables"], d["plan"], out, None, *step.shape(), ws,
                  ws.numel())
    assert torch.equal(out[:step.cu[-1]], with_lse[:step.cu[-1]])


def test_bound_on_new_tokens(kv):
    """max_tokens may be more than any sequence has."""
    for n in (1, 3, 40):
        step = Step(12, "bf16", (16, 8, 128), [n], [50], gap=200, max_tokens=150)
        check(step.upload().plan(kv), kv, f"{n} of at most 150")


@pytest.mark.parametrize("change", ["long", "short", "negative", "descends", "past", "more"])
def test_lengths_that_do_not_fit(kv, change):
    """A sequence whose lengths do not fit is left out and flagged; the others
    are attended."""
    step = Step(13, "bf16", (16, 8, 128), [1, 3, 2], [20, 40, 60])
    want, _, tol, _ = step.attention()
    step.upload()
    lens, cu = list(step.lens), list(step.cu)
    if change == "long":
        lens[1] = step.mbps * 16 + 1
    elif change == "short":
        lens[1] = 2
    elif change == "negative":
        lens[1] = -4
    elif change == "descends":
        cu = [0, 4, 1, 3]
        step.dev["lens"] = None
    elif change == "past":
        cu = [0, 1, 4, 900]
    else:
        step.most = 2
    step.dev["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    step.dev["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    step.plan(kv)
    out, _ = step.run(kv)
    torch.cuda.synchronize()
    with pytest.raises(kv.TokenLimitExceeded):
        kv.workspace_check(step.dev["plan"])
    kv.workspace_check(step.dev["plan"])  # cleared
    if change == "descends":
        return
    left_out = slice(4, 6) if change == "past" else slice(1, 4)
    keep = torch.ones(6, dtype=torch.bool)
    keep[left_out] = False
    assert (out[left_out] == 7).all()
    assert_within(out[keep.to(DEV)], want[keep], tol[keep], "the others")


def test_plan_of_another_step(kv):
    step = Step(14, "bf16", (16, 8, 128), [1, 3], [20, 40]).upload().plan(kv)
    step.window = 5
    out, lse = step.run(kv)
    torch.cuda.synchronize()
    assert (out == 7).all() and (lse == 7).all()
    with pytest.raises(kv.RlseError, match="other arguments"):
        kv.workspace_check(step.dev["plan"])


def test_other_stream_and_two_steps_at_once(kv):
    """Two steps on two streams, each with its own plan and workspace."""
    a = Step(15, "bf16", (16, 8, 128), [1] * 9, list(range(100, 1000, 100)))
    b = Step(16, "f16", (14, 2, 64), [90, 1], [200, 3000])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in (a, b):
        s.upload()
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                s.plan(kv, st)
                got.append(s.run(kv, stream=st))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        want, wlse, tol, ltol = (a, b)[i % 2].attention()
        assert_within(out, want, tol, "out")
        assert_within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("new", [[1] * 6, [40, 1, 1, 200, 1, 3]])
def test_captured_and_replayed(kv, new):
    """Plan and attention in a graph: the replays follow the lengths."""
    step = Step(17, "bf16", (16, 8, 128), new, [30, 700, 1500, 64, 2, 999]).upload().plan(kv)
    ws = step.workspace(kv)
    out, lse = step.run(kv, ws)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step.build(kv, st)
        step.run(kv, ws, out, lse, st)
    lens = step.dev["lens"].clone()
    for shorter in (0, 7, 20, 0):
        step.cached = [max(0, n - shorter) for n in [30, 700, 1500, 64, 2, 999]]
        step.lens = [a + b for a, b in zip(step.new, step.cached)]
        step.dev["lens"].copy_(torch.tensor(step.lens, dtype=torch.int32))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        again = step.run(kv, ws)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
        want, wlse, tol, ltol = step.attention()
        assert_within(got[0], want, tol, f"shorter by {shorter}")
        assert_within(got[1], wlse, ltol, f"shorter by {shorter}")
    step.dev["lens"].copy_(lens)


def test_pool_offsets_past_32_bits(kv):
    """Pages whose elements lie past 2^31 (and bytes past 2^32)."""
    step = Step(18, "bf16", (16, 8, 128), [1, 40], [90, 33])
    want, wlse, tol, ltol = step.attention()
    step.upload()
    blocks = 2 ** 31 // (8 * 16 * 128) + step.nb
    for name in ("k", "v"):
        big = torch.empty((blocks, 8, 16, 128), dtype=torch.bfloat16, device=DEV)
        big[-step.nb:] = step.dev[name]
        step.dev[name] = big
    step.dev["tables"] = torch.where(step.dev["tables"] >= 0,
                                     step.dev["tables"] + (blocks - step.nb), -1)
    step.nb = blocks
    step.plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want, tol, "out")
    assert_within(lse, wlse, ltol, "lse")


def test_agrees_with_prefill_and_decode(kv):
    """The calls for one sequence's chunk and for a decode step, within the
    bounds of both."""
    step = Step(19, "bf16", (16, 8, 128), [120], [500]).upload().plan(kv)
    out, _ = step.run(kv)
    _, _, tol, _ = step.attention()
    d = step.dev
    other = torch.empty_like(d["q"])
    kv.prefill_attn(d["q"], d["k"], d["v"], d["tables"], 620, 120, other, 16, 8, 128, step.mbps,
                    step.nb, step.scale, "bf16")
    assert_within(out, other.cpu().double(), 2 * tol, "prefill")
    step = Step(20, "bf16", (16, 8, 128), [1] * 5, [3, 17, 200, 900, 31]).upload().plan(kv)
    out, _ = step.run(kv)
    _, _, tol, _ = step.attention()
    d = step.dev
    other = torch.empty_like(d["q"])
    kv.paged_gqa_decode(d["q"], d["k"], d["v"], d["tables"], d["lens"], other, 5, 16, 8, 128,
                        step.mbps, step.nb, step.scale, "bf16")
    assert_within(out, other.cpu().double(), 2 * tol, "decode")


def test_refuses_a_small_workspace(kv):
    step = Step(21, "bf16", (16, 8, 128), [1, 30], [100, 0]).upload().plan(kv)
    ws = step.workspace(kv)
    with pytest.raises(kv.RlseError, match="workspace"):
        step.run(kv, ws[:-16])
    small = step.dev["plan"][:-16]
    with pytest.raises(kv.RlseError, match="plan"):
        kv.chunk_plan(step.dev["cu"], step.dev["lens"], step.n, step.total, step.most, step.hq,
                      step.hkv, step.mbps, 0, 0, small, small.numel())


def test_flag_for_shared_pages(kv):
    """Sequences forked from one prefix; the flag changes no bit."""
    step = Step(22, "bf16", (16, 8, 128), [1, 1, 4, 50], [200, 210, 220, 230])
    step.tables[1:, :12] = step.tables[0, :12]
    step.upload().plan(kv)
    check(step, kv, "forks")
    d, ws = step.dev, step.workspace(kv)
    out, lse = step.run(kv, ws)
    other, olse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    kv.chunk_attn(d["q"], d["k"], d["v"], d["tables"], d["plan"], other, olse, *step.shape(), ws,
                  ws.numel(), shared_pages=True)
    assert torch.equal(out, other) and torch.equal(lse, olse)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_workspace_and_the_same_bits_again(kv, dtype):
    """Steps of many kinds through one workspace, over and over: a tile's pieces
    give the same bits whichever workgroup joins them."""
    steps = [Step(23 + i, dtype, (14, 2, 64), *args).upload().plan(kv) for i, args in enumerate([
        ([90, 200, 37, 150, 61], [40, 300, 0, 77, 1200]),
        ([1] * 7, [30, 9000, 100, 2000, 7, 64, 511]),
        ([300], [0]),
        ([41] * 9, [333] * 9, 200, 4),
    ])]
    ws = max((s.workspace(kv) for s in steps), key=lambda w: w.numel())
    first = [s.run(kv, ws) for s in steps]
    for s, (out, lse) in zip(steps, first):
        want, wlse, tol, ltol = s.attention()
        assert_within(out, want, tol, "out")
        assert_within(lse, wlse, ltol, "lse")
    for _ in range(30):
        for s, (out, lse) in zip(steps, first):
            again, alse = s.run(kv, ws)
            assert torch.equal(out, again) and torch.equal(lse, alse)


@pytest.mark.parametrize("heads", [(6, 6, 64), (33, 3, 128), (256, 1, 64)],
                         ids=lambda h: "x".join(map(str, h)))
def test_odd_groups(kv, heads):
    step = Step(27, "bf16", heads, [1, 3, 20], [50, 0, 70], 30, 2).upload().plan(kv)
    check(step, kv, "odd groups")


def test_many_sequences(kv):
    """More sequences than workgroups: several tiles each, some empty."""
    new = [i % 3 for i in range(700)]
    cached = [(i * 37) % 90 for i in range(700)]
    step = Step(28, "f16", (4, 2, 64), new, cached).upload().plan(kv)
    check(step, kv, "many")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new", [2, 70])
def test_a_value_of_little_weight_still_reaches_its_rows(kv, new, dtype):
    """The last token's V is infinite and its weight below the type's smallest:
    its own row has the infinity, those before it do not."""
    step = Step(29, dtype, (4, 2, 64), [new], [24])
    step.q[..., 0] = 30.0
    step.k[..., 0] = 4.0
    at = step.lens[0] - 1
    step.k[step.tables[0, at // 16], :, at % 16, 0] = -2.0
    want, wlse, tol, ltol = step.attention()
    step.v[step.tables[0, at // 16], :, at % 16, 9] = math.inf
    want[new - 1, :, 9] = math.inf
    step.upload().plan(kv)
    out, lse = step.run(kv)
    assert_within(out, want, tol, "out")
    assert_within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("window", [(0, 0), (300, 5)])
def test_more_tiles_than_the_plan_holds_on_chip(kv, window):
    """5000 tokens of 256 heads that share one KV head: a tile a token. Four of
    the heads are compared."""
    step = Step(30, "bf16", (256, 1, 64), [4300, 700], [0, 40], *window).upload().plan(kv)
    out, lse = step.run(kv)
    torch.cuda.synchronize()
    kv.workspace_check(step.dev["plan"])
    some = [0, 1, 100, 255]
    part = copy.copy(step)
    part.hq, part.q = len(some), step.q[:, some]
    want, wlse, tol, ltol = part.attention()
    assert_within(out[:, some], want, tol, "out")
    assert_within(lse[:, some], wlse, ltol, "lse")
    weights = torch.zeros(2, 1, step.mbps * 16, device=DEV)
    d = step.dev
    kv.kv_scores(d["q"], d["k"], d["tables"], d["plan"], lse, None, weights, *step.shape())
    # every query gives one in all
    for b in range(2):
        given = float(weights[b].double().sum())
        assert abs(given - 256 * step.new[b]) <= 1e-4 * 256 * step.new[b]


def test_two_calls_at_once(kv):
    """One plan, two layers' calls on two streams, each with a workspace."""
    step = Step(31, "bf16", (28, 4, 128), [150, 1, 90, 1, 260], [100, 2500, 0, 4000, 700])
    step.upload().plan(kv)
    want = [t.clone() for t in step.run(kv)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    spaces = [step.workspace(kv) for _ in streams]
    outs = [(torch.full_like(want[0], 7.0), torch.full_like(want[1], 7.0)) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, ws, (out, lse) in zip(streams, spaces, outs):
            with torch.cuda.stream(st):
                step.run(kv, ws, out, lse, st)
    torch.cuda.synchronize()
    for out, lse in outs:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_captured_step_follows_its_lengths(kv):
    """Plan, attention and key weights captured once; every replay attends what
    the lengths say then, from no new token to all of them."""
    step = Step(32, "f16", (16, 8, 128), [3, 1, 40], [300, 50, 200], 64, 4).upload().plan(kv)
    d, ws = step.dev, step.workspace(kv)
    out, lse = torch.empty_like(d["q"]), torch.empty(step.total, step.hq, device=DEV)
    acc = torch.empty(step.n, step.hkv, step.mbps * 16, device=DEV)
    st = torch.cuda.Stream()

    def all_of_it(stream=None):
        step.build(kv, stream)
        step.run(kv, ws, out, lse, stream)
        kv.kv_scores(d["q"], d["k"], d["tables"], d["plan"], lse, None, acc, *step.shape(),
                     stream)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        all_of_it(st)
    for new, cached in [([3, 1, 40], [300, 50, 200]), ([0, 0, 40], [300, 51, 10]),
                        ([3, 0, 0], [0, 9, 5]), ([0, 0, 0], [1, 1, 1]), ([1, 1, 1], [299, 50, 239])]:
        cu = [0, new[0], new[0] + new[1], sum(new)]
        d["cu"].copy_(torch.tensor(cu, dtype=torch.int32))
        d["lens"].copy_(torch.tensor([a + b for a, b in zip(new, cached)], dtype=torch.int32))
        results = []
        for call in (graph.replay, all_of_it):
            for t in (out, lse, acc):
                t.fill_(7)
            call()
            torch.cuda.synchronize()
            kv.workspace_check(d["plan"])
            results.append([t.clone() for t in (out, lse, acc)])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert (results[0][0][sum(new):] == 7).all()
        now = copy.copy(step)
        now.new, now.cached, now.cu = new, cached, cu
        now.lens = [a + b for a, b in zip(new, cached)]
        want, wlse, tol, ltol = now.attention()
        rows = slice(0, sum(new))
        assert_within(results[0][0][rows], want[rows], tol[rows], f"{new} out")
        assert_within(results[0][1][rows], wlse[rows], ltol[rows], f"{new} lse")
