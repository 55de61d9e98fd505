"""plh_rope_* and plh_kv8_* without a device: sizes, frequencies, refusals (every
argument is checked before the device is looked for), and the reference the
GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import picolm_amd as P
from kv8_ref import Ref, from_tiles, starts, to_tiles


def refused(rc, word):
    assert rc == -1
    assert word in P._native.last_error(), P._native.last_error()


FAKE = 4096  # a pointer that no refused call follows


def cache(**kw):
    d = dict(n_layers=2, n_kv_heads=2, head_dim=64, n_pages=8, page_tokens=64, codes=FAKE,
             scales=FAKE)
    d.update(kw)
    return P._native.PlhKv8Cache(**d)


def seqs(**kw):
    d = dict(n_seqs=3, max_pages=4, table=FAKE, len=FAKE, refs=FAKE)
    d.update(kw)
    return P._native.PlhKv8Seqs(**d)


def test_bytes():
    for D, tiles in ((2, 1), (32, 1), (34, 2), (80, 3), (128, 4), (256, 8)):
        c = cache(head_dim=D)
        blocks = 8 * 2 * 2 * 2
        assert P.lib.plh_kv8_code_bytes(C.byref(c)) == blocks * 2 * tiles * 1024
        assert P.lib.plh_kv8_scale_bytes(C.byref(c)) == blocks * 2 * 4
    big = cache(n_layers=80, n_kv_heads=8, head_dim=128, n_pages=100000, page_tokens=64)
    assert P.lib.plh_kv8_code_bytes(C.byref(big)) == 100000 * 80 * 8 * 64 * 128 * 2


BAD_CACHES = [dict(head_dim=0), dict(head_dim=63), dict(head_dim=258), dict(n_layers=0),
              dict(n_kv_heads=0), dict(n_pages=0), dict(page_tokens=0), dict(page_tokens=48),
              dict(page_tokens=-32), dict(page_tokens=1 << 30, n_layers=1000)]


@pytest.mark.parametrize("kw", BAD_CACHES, ids=str)
def test_caches_outside_the_limits(kw):
    c, s = cache(**kw), seqs()
    assert P.lib.plh_kv8_code_bytes(C.byref(c)) == 0
    assert P.lib.plh_kv8_scale_bytes(C.byref(c)) == 0
    refused(P.lib.plh_kv8_trim(C.byref(c), C.byref(s), FAKE), "not built")
    refused(P.lib.plh_kv8_fork(C.byref(c), C.byref(s), FAKE), "not built")
    refused(P.lib.plh_kv8_extend(C.byref(c), C.byref(s), FAKE, FAKE), "not built")
    refused(P.lib.plh_kv8_compact(C.byref(c), C.byref(s), FAKE), "not built")
    refused(P.lib.plh_kv8_attn(C.byref(c), C.byref(s), 0, 2, 1, FAKE, FAKE, 128, FAKE, 128),
            "not built")
    refused(P.lib.plh_kv8_fetch(C.byref(c), C.byref(s), 0, 1, FAKE, FAKE, 128, FAKE, 128),
            "not built")
    refused(P.lib.plh_kv8_append(C.byref(c), C.byref(s), 0, 1, FAKE, None, None, 0, 0, None, 0,
                                 FAKE, 128, FAKE, 128), "not built")


@pytest.mark.parametrize("c,s,word", [
    (dict(codes=None), {}, "codes"), (dict(scales=None), {}, "codes"),
    (dict(codes=FAKE + 8), {}, "codes"), (dict(scales=FAKE + 2), {}, "codes"),
    ({}, dict(n_seqs=0), "sequences"), ({}, dict(n_seqs=1025), "sequences"),
    ({}, dict(max_pages=0), "sequences"), ({}, dict(max_pages=1 << 24), "sequences"),
    ({}, dict(table=None), "table"), ({}, dict(len=None), "table"), ({}, dict(refs=None), "table")])
def test_descriptors(c, s, word):
    c, s = C.byref(cache(**c)), C.byref(seqs(**s))
    refused(P.lib.plh_kv8_extend(c, s, FAKE, FAKE), word)
    refused(P.lib.plh_kv8_attn(c, s, 0, 2, 1, FAKE, FAKE, 128, FAKE, 128), word)


def test_null_descriptors_and_vectors():
    c, s = C.byref(cache()), C.byref(seqs())
    for a, b in ((None, s), (c, None), (None, None)):
        refused(P.lib.plh_kv8_trim(a, b, FAKE), "no cache")
        refused(P.lib.plh_kv8_fork(a, b, FAKE), "no cache")
        refused(P.lib.plh_kv8_extend(a, b, FAKE, FAKE), "no cache")
        refused(P.lib.plh_kv8_compact(a, b, FAKE), "no cache")
        refused(P.lib.plh_kv8_attn(a, b, 0, 2, 1, FAKE, FAKE, 128, FAKE, 128), "no cache")
    refused(P.lib.plh_kv8_trim(c, s, None), "null")
    refused(P.lib.plh_kv8_fork(c, s, None), "null")
    refused(P.lib.plh_kv8_extend(c, s, None, FAKE), "null")
    refused(P.lib.plh_kv8_extend(c, s, FAKE, None), "null")
    refused(P.lib.plh_kv8_compact(c, s, None), "null")
    assert P.lib.plh_kv8_code_bytes(None) == 0 and P.lib.plh_kv8_scale_bytes(None) == 0


def attn(**kw):
    d = dict(layer=0, n_heads=4, n_rows=1, row_start=FAKE, q=FAKE, q_stride=256, out=FAKE,
             out_stride=256)
    d.update(kw)
    return P.lib.plh_kv8_attn(C.byref(cache()), C.byref(seqs()), *d.values())


@pytest.mark.parametrize("kw,word", [
    (dict(layer=-1), "layer"), (dict(layer=2), "layer"), (dict(n_rows=-1), "rows"),
    (dict(row_start=None), "rows"), (dict(n_heads=0), "heads"), (dict(n_heads=3), "heads"),
    (dict(q=None), "q or out"), (dict(out=None), "q or out"), (dict(q=FAKE + 2), "q or out"),
    (dict(q_stride=255), "q or out"), (dict(out_stride=0), "q or out"),
    (dict(n_rows=1 << 29), "too many")])
def test_attention_refuses(kw, word):
    refused(attn(**kw), word)


def append(rope=None, **kw):
    d = dict(layer=0, n_rows=1, row_start=FAKE, rope=rope, q=None, n_heads=0, q_stride=0,
             q_out=None, q_out_stride=0, k=FAKE, k_stride=128, v=FAKE, v_stride=128)
    d.update(kw)
    return P.lib.plh_kv8_append(C.byref(cache()), C.byref(seqs()), *d.values())


def tables(**kw):
    d = dict(rope_type=0, rot_dim=64, n_pos=16, cos_tab=FAKE, sin_tab=FAKE)
    d.update(kw)
    return C.byref(P._native.PlhRope(**d))


@pytest.mark.parametrize("kw,word", [
    (dict(layer=5), "layer"), (dict(n_rows=-2), "rows"), (dict(row_start=None), "rows"),
    (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(k=FAKE + 1), "k is null"),
    (dict(k_stride=127), "k rows"), (dict(v_stride=-1), "v rows"),
    (dict(n_heads=2, q=FAKE, q_out=FAKE, q_stride=128, q_out_stride=128), "tables"),
    (dict(rope=tables(), n_heads=-1), "q heads"),
    (dict(rope=tables(), n_heads=2, q=None, q_out=FAKE, q_stride=128, q_out_stride=128),
     "q is null"),
    (dict(rope=tables(), n_heads=2, q=FAKE, q_out=None, q_stride=128, q_out_stride=128),
     "q_out is null"),
    (dict(rope=tables(), n_heads=2, q=FAKE, q_out=FAKE, q_stride=100, q_out_stride=128), "q rows"),
    (dict(rope=tables(rope_type=2)), "rope_type"), (dict(rope=tables(rot_dim=66)), "rot_dim"),
    (dict(rope=tables(rot_dim=31)), "rot_dim"), (dict(rope=tables(rot_dim=0)), "rot_dim"),
    (dict(rope=tables(n_pos=0)), "tables"), (dict(rope=tables(cos_tab=None)), "tables"),
    (dict(n_rows=2**31 - 1, k_stride=128), "too many")])
def test_append_refuses(kw, word):
    refused(append(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(layer=2), "layer"), (dict(n_rows=-1), "rows"), (dict(k=None), "k is null"),
    (dict(v_stride=100), "v rows"), (dict(n_rows=2**31 - 1), "too many")])
def test_fetch_refuses(kw, word):
    d = dict(layer=0, n_rows=1, row_start=FAKE, k=FAKE, k_stride=128, v=FAKE, v_stride=128)
    d.update(kw)
    refused(P.lib.plh_kv8_fetch(C.byref(cache()), C.byref(seqs()), *d.values()), word)


def rows(tab=None, **kw):
    d = dict(n_rows=1, pos=FAKE, head_dim=64, q=FAKE, n_heads=2, q_stride=128, q_out=FAKE,
             q_out_stride=128, k=FAKE, n_kv_heads=1, k_stride=64, k_out=FAKE, k_out_stride=64)
    d.update(kw)
    return P.lib.plh_rope_rows(tables() if tab is None else tab, *d.values())


@pytest.mark.parametrize("kw,word", [
    (dict(head_dim=63), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=258), "head_dim"),
    (dict(head_dim=32), "rot_dim"), (dict(n_rows=-1), "rows"), (dict(n_heads=-1), "heads"),
    (dict(q_stride=127), "stride"), (dict(k_out_stride=63), "stride"), (dict(pos=None), "null"),
    (dict(q=None), "null"), (dict(k_out=None), "null"),
    (dict(n_rows=2**31 - 1), "too many")])
def test_rope_rows_refuses(kw, word):
    refused(rows(**kw), word)


def test_rope_rows_refuses_tables():
    refused(P.lib.plh_rope_rows(None, 1, FAKE, 64, FAKE, 2, 128, FAKE, 128, None, 0, 0, None, 0),
            "no tables")
    refused(rows(tables(rope_type=-1)), "rope_type")
    refused(rows(tables(sin_tab=None)), "tables")


def spec(**kw):
    d = dict(rot_dim=64, freq_base=1e4)
    d.update(kw)
    return P.rope.Spec(**d)


BANDS = dict(scaling="bands", factor=8.0, trained_len=4096, low=1.0, high=4.0)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(freq_base=1.0),
    dict(freq_base=float("inf")), dict(freq_base=float("nan")), dict(scaling="linear", factor=0.5),
    dict(scaling="ntk", factor=2.0, rot_dim=2), dict(magnitude=-1.0),
    dict(scaling="linear", factor=float("nan")), dict(BANDS, trained_len=0), dict(BANDS, low=0.0),
    dict(BANDS, high=1.0), dict(BANDS, high=float("inf")), dict(BANDS, scaling="ramp", low=-1.0)])
def test_specifications_refused(kw):
    with pytest.raises(P.PicolmHipError):
        spec(**kw).frequencies()
    refused(P.lib.plh_rope_tables(C.byref(spec(**kw).desc), 0, 4, FAKE, FAKE), "rope")


def test_table_ranges_refused():
    d = C.byref(spec().desc)
    for first, n in ((-1, 4), (0, -1), (2**31 - 1, 1), (2**31 - 10, 20)):
        refused(P.lib.plh_rope_tables(d, first, n, FAKE, FAKE), "positions")
    refused(P.lib.plh_rope_tables(d, 0, 2**27, FAKE, FAKE), "too many")
    refused(P.lib.plh_rope_tables(d, 0, 4, None, FAKE), "null")
    with pytest.raises(ValueError):
        P.rope.Spec(64, 1e4, "other")


@pytest.mark.parametrize("rot", [2, 48, 64, 128, 256])
def test_frequencies(rot):
    """Against the formulas, in another form (logarithms): 1e-14 relative leaves room
    for the errors of exp and log of values up to 2^6."""
    i = np.arange(rot // 2)
    base = np.exp(-2 * i / rot * np.log(1e4))
    close = dict(rtol=2e-14, atol=0)
    f, m = spec(rot_dim=rot).frequencies()
    assert np.allclose(f, base, **close) and m == 1
    f, m = spec(rot_dim=rot, scaling="linear", factor=4.0, magnitude=0.5).frequencies()
    assert np.allclose(f, base / 4, **close) and m == 0.5
    if rot > 2:
        f, _ = spec(rot_dim=rot, scaling="ntk", factor=8.0).frequencies()
        assert np.allclose(f, np.exp(-2 * i / rot * (np.log(1e4) + rot / (rot - 2) * np.log(8.0))),
                           **close)
    f, m = spec(rot_dim=rot, **BANDS).frequencies()
    wave = 2 * np.pi / base
    for x, y, w in zip(f, base, wave):
        if w < 4096 / 4.0:
            assert abs(x - y) <= 2e-14 * y
        elif w > 4096 / 1.0:
            assert abs(x - y / 8) <= 2e-14 * y
        else:
            s = (4096 / w - 1) / 3
            assert abs(x - ((1 - s) * y / 8 + s * y)) <= 1e-13 * y
    f, m = spec(rot_dim=rot, scaling="ramp", factor=16.0, trained_len=4096, low=1.0,
                high=32.0).frequencies()
    assert abs(m - (1 + 0.1 * np.log(16.0))) < 1e-15

    def number(turns):
        return rot * np.log(4096 / (turns * 2 * np.pi)) / (2 * np.log(1e4))
    lo, hi = max(0, np.floor(number(32.0))), min(rot - 1, np.ceil(number(1.0)))
    keep = 1 - np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    assert np.allclose(f, base / 16 * (1 - keep) + base * keep, **close)


def test_not_initialised():
    if P.lib.plh_device_count() > 0:
        pytest.skip("a device is visible")
    refused(attn(), "not initialised")
    refused(append(), "not initialised")
    refused(append(rope=tables()), "not initialised")  # no q rows to rotate
    refused(append(n_rows=0, k=None, v=None), "not initialised")
    refused(rows(), "not initialised")
    refused(P.lib.plh_rope_tables(C.byref(spec().desc), 0, 4, FAKE, FAKE), "not initialised")
    refused(P.lib.plh_kv8_extend(C.byref(cache()), C.byref(seqs()), FAKE, FAKE), "not initialised")


def test_python_descriptors():
    with pytest.raises(ValueError):
        P.kv8.Cache(1, 1, 63, 1, 32, codes=FAKE, scales=FAKE)
    with pytest.raises(ValueError):
        P.kv8.Sequences(1, 1)
    with pytest.raises(ValueError):
        P.kv8.Sequences(1, 1, table=FAKE)


# ---- the reference itself -------------------------------------------------------


def test_tiles_round_trip():
    rng = np.random.default_rng(0)
    for D in (2, 32, 50, 128):
        x = rng.integers(-127, 128, (3, 32, 2, D)).astype(np.int8)
        t = to_tiles(x)
        assert t.shape == (3, 2, (D + 31) // 32, 1024)
        assert np.array_equal(from_tiles(t, D), x)
    # one element of each kind, by hand: token 21, element 45
    x = np.zeros((32, 2, 64), np.int8)
    x[21, :, 45] = 1
    t = to_tiles(x)
    assert t[0, 1, 256 * 1 + 16 * 5 + 8 * 1 + 5] == 1 and t[0].sum() == 1
    assert t[1, 1, 256 * 1 + 16 * 13 + 8 * 0 + 5] == 1 and t[1].sum() == 1


def test_reference_append_and_attention():
    """Half a step per element, a block whose scale grows, and attention over the
    values it holds."""
    rng = np.random.default_rng(1)
    ref = Ref(1, 1, 16, 4, 32, 1, 3)
    assert ref.extend([40]) == (0, 0)
    x = rng.normal(size=(2, 40, 1, 16)).astype(np.float32)
    ref.append(0, starts([40]), x[0], x[1])
    v = ref.values(0, 0)
    for kind in (0, 1):
        assert np.abs(v[kind][0] - x[kind][:, 0]).max() <= np.abs(x).max() / 127 * 0.5001
    assert ref.extend([1]) == (0, 0)
    big = 10 * np.ones((1, 1, 16), np.float32)
    ref.append(0, starts([1]), big, big)
    v2 = ref.values(0, 0)
    assert np.array_equal(v2[:, :, :32], v[:, :, :32])
    assert np.abs(v2[:, :, 32:40] - v[:, :, 32:]).max() <= 10 / 127 * 0.5001
    q = rng.normal(size=(2, 2, 16)).astype(np.float32)
    out = ref.attention(0, starts([2]), q)
    k, vv = v2[0][0], v2[1][0]
    w = np.exp(k[:40] @ q[0, 1].astype(np.float64) / 4)
    assert np.allclose(out[0, 1], w @ vv[:40] / w.sum(), rtol=1e-12)
