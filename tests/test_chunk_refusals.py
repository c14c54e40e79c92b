"""The ragged step's calls reject bad arguments before they touch a device."""
import pytest

GOOD = dict(n=2, total=10, most=8, hq=16, hkv=8, d=128, mbps=4, nb=64, window=0, sinks=0,
            scale=0.1, dtype=1)


def _plan(kv, **a):
    return kv.load().rlse_chunk_plan(16, 16, a["n"], a["total"], a["most"], a["hq"], a["hkv"],
                                     a["mbps"], a["window"], a["sinks"], 16, 1 << 40, None)


def _attn(kv, ptr=16, **a):
    return kv.load().rlse_chunk_attn(ptr, 16, 16, 16, 16, 16, None, a["n"], a["total"], a["most"],
                                     a["hq"], a["hkv"], a["d"], a["mbps"], a["nb"], a["window"],
                                     a["sinks"], a["scale"], a["dtype"], 16, 1 << 40,
                                     a.get("flags", 0), None)


SHAPES = [dict(n=0), dict(n=4097), dict(total=0), dict(most=0), dict(most=11), dict(hq=12),
          dict(hq=0), dict(hkv=0), dict(mbps=0), dict(mbps=1 << 25), dict(mbps=(1 << 17) + 1),
          dict(window=-1), dict(sinks=-1), dict(total=1 << 24, hq=64), dict(hq=514, hkv=2)]


@pytest.mark.parametrize("change", SHAPES, ids=str)
def test_shapes(kv, change):
    assert _plan(kv, **{**GOOD, **change}) == kv.ERR_INVALID_VALUE
    assert "chunk_plan" in kv.last_error()
    assert _attn(kv, **{**GOOD, **change}) == kv.ERR_INVALID_VALUE
    assert "chunk_attn" in kv.last_error()


@pytest.mark.parametrize("change", [dict(d=96), dict(dtype=7), dict(nb=0), dict(scale=0.0),
                                    dict(scale=float("nan")), dict(scale=float("inf")),
                                    dict(flags=2)], ids=str)
def test_attention_arguments(kv, change):
    assert _attn(kv, **{**GOOD, **change}) == kv.ERR_INVALID_VALUE
    assert "chunk_attn" in kv.last_error()


def test_pointers(kv):
    lib = kv.load()
    assert _attn(kv, ptr=None, **GOOD) == kv.ERR_INVALID_VALUE
    assert "null" in kv.last_error()
    assert _attn(kv, ptr=24, **GOOD) == kv.ERR_INVALID_VALUE
    assert "aligned" in kv.last_error()
    assert lib.rlse_chunk_plan(None, 16, 1, 1, 1, 8, 8, 1, 0, 0, 16, 1 << 30,
                               None) == kv.ERR_INVALID_VALUE
    assert lib.rlse_chunk_plan(16, 16, 1, 1, 1, 8, 8, 1, 0, 0, 8, 1 << 30,
                               None) == kv.ERR_INVALID_VALUE
    assert lib.rlse_chunk_plan_size(1, 1, 8, 8, None) == kv.ERR_INVALID_VALUE
    assert lib.rlse_chunk_workspace_size(1, 1, 1, 8, 8, 128, None) == kv.ERR_INVALID_VALUE


def _scores(kv, ptr=16, **a):
    return kv.load().rlse_kv_scores(ptr, 16, 16, 16, 16, a.get("prev"), 4096, a["n"], a["total"], a["most"],
                                    a["hq"], a["hkv"], a["d"], a["mbps"], a["nb"], a["window"],
                                    a["sinks"], a["scale"], a["dtype"],
                                    a.get("flags", 0), None)


@pytest.mark.parametrize("change", SHAPES + [dict(d=96), dict(dtype=7), dict(nb=0),
                                             dict(scale=0.0), dict(flags=4)], ids=str)
def test_score_arguments(kv, change):
    assert _scores(kv, **{**GOOD, **change}) == kv.ERR_INVALID_VALUE
    assert "kv_scores" in kv.last_error()


def test_score_pointers(kv):
    assert _scores(kv, ptr=None, **GOOD) == kv.ERR_INVALID_VALUE
    assert "null" in kv.last_error()
    assert _scores(kv, ptr=24, **GOOD) == kv.ERR_INVALID_VALUE
    assert "aligned" in kv.last_error()


EVICT = dict(k=16, stride=64 * 8 * 16 * 128, layers=2, scores=16, sstride=2 * 8 * 128,
             new=1 << 20, lens=16, nlens=24,
             n=2, hkv=8, d=128, mbps=8, nbps=2, nb=64, budget=20, sinks=2, recent=3, dtype=1)


def _evict(kv, **a):
    return kv.load().rlse_kv_evict(a["k"], 16, a["stride"], a["layers"], 16, a["lens"],
                                   a["scores"], a["sstride"], 16, a["nlens"], a["new"], 16, a["n"], a["hkv"], a["d"],
                                   a["mbps"], a["nbps"], a["nb"], a["budget"], a["sinks"],
                                   a["recent"], a["dtype"], None)


@pytest.mark.parametrize("change", [
    dict(layers=0), dict(n=0), dict(hkv=0), dict(d=96), dict(mbps=0), dict(nbps=0), dict(nb=0),
    dict(budget=0), dict(budget=33), dict(budget=129, nbps=20), dict(sinks=-1), dict(recent=-1),
    dict(sinks=18), dict(dtype=5), dict(sstride=2047), dict(stride=64 * 8 * 16 * 128 - 1),
    dict(stride=64 * 8 * 16 * 128 + 1), dict(k=None), dict(k=24), dict(new=16),
    dict(new=16 + 2 * 2 * 8 * 128 * 4 - 4), dict(scores=(1 << 20) + 64), dict(nlens=16),
    dict(nlens=20), dict(lens=28),
    dict(layers=1 << 20, n=4096, sstride=1 << 40)], ids=str)
def test_evict_arguments(kv, change):
    assert _evict(kv, **{**EVICT, **change}) == kv.ERR_INVALID_VALUE
    assert "kv_evict" in kv.last_error()


def test_overlaps_name_their_reason(kv):
    for change in (dict(new=16), dict(new=16 + 2 * 2 * 8 * 128 * 4 - 4),
                   dict(scores=(1 << 20) + 64)):
        _evict(kv, **{**EVICT, **change})
        assert "new_scores overlaps" in kv.last_error()
    for change in (dict(nlens=16), dict(nlens=20), dict(lens=28)):
        _evict(kv, **{**EVICT, **change})
        assert "new_lens overlaps" in kv.last_error()
    for prev in (4092, 4100, 4096 + 4 * GOOD["n"] * GOOD["hkv"] * GOOD["mbps"] * 16 - 4):
        assert _scores(kv, **{**GOOD, "prev": prev}) == kv.ERR_INVALID_VALUE
        assert "prev overlaps" in kv.last_error()


def test_layers_of_weights_that_meet(kv):
    """Two layers of 2048 floats 5000 apart: refused where one of the new ones
    meets one of the old ones."""
    row, stride = 4 * 2 * 8 * 128, 4 * 5000
    base = 1 << 20
    for at in (0, row - 4, stride, stride - row + 4, stride + row - 4, -stride, -4, 4 - row):
        _evict(kv, **{**EVICT, "scores": base, "sstride": 5000, "new": base + at})
        assert "new_scores overlaps" in kv.last_error(), at
    for at in (row, stride - row, -row, 2 * stride, -2 * stride):
        _evict(kv, **{**EVICT, "scores": base, "sstride": 5000, "new": base + at, "lens": 16,
                      "nlens": 16})
        assert "new_lens overlaps" in kv.last_error(), at
