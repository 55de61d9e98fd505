"""plh_rope_tables and plh_rope_rows against 64-bit numpy.

Tables: the angle in 64 bits, cos and sin rounded once to fp32: off by at most
half an ulp (2^-24 of values up to the magnitude) and the 64-bit errors of a
position times a frequency, position * theta * 2^-52 for the two sides' roundings
of theta and the product.  Rotated rows are the 64-bit result rounded once; the
kernel's fused form may differ from numpy's in the last 64-bit place, which
reaches fp32 only beside a rounding border: at most one ulp, of few elements."""
import numpy as np
import pytest

from kv8_ref import rope_ref

pytestmark = pytest.mark.gpu

SPECS = [dict(rot_dim=64, freq_base=1e4),
         dict(rot_dim=128, freq_base=1e6, scaling="linear", factor=4.0),
         dict(rot_dim=80, freq_base=1e4, scaling="ntk", factor=8.0),
         dict(rot_dim=64, freq_base=5e5, scaling="bands", factor=32.0, trained_len=8192, low=1.0,
              high=4.0),
         dict(rot_dim=96, freq_base=1e4, scaling="ramp", factor=16.0, trained_len=4096, low=1.0,
              high=32.0),
         dict(rot_dim=2, freq_base=1e4, magnitude=1.5), dict(rot_dim=256, freq_base=1e4)]


@pytest.mark.parametrize("kw", SPECS, ids=lambda k: f"{k.get('scaling', 'none')}{k['rot_dim']}")
@pytest.mark.parametrize("first,n", [(0, 1), (0, 777), (131070, 65), (10**6, 300),
                                     (2**31 - 70, 69)])
def test_tables(gpu, kw, first, n):
    P = gpu
    spec = P.rope.Spec(**kw)
    theta, mag = spec.frequencies()
    half = kw["rot_dim"] // 2
    guard = np.full(n * half + 8, 7.0, np.float32)
    cos, sin = P.DeviceBuffer.from_numpy(guard), P.DeviceBuffer.from_numpy(guard)
    print(f"[case] tables {kw} {first}+{n}", flush=True)
    P.rope.make_tables(spec, first, n, cos.ptr, sin.ptr)
    P.synchronize()
    angle = (first + np.arange(n, dtype=np.float64))[:, None] * theta
    tol = mag * (2.0**-24 + 1e-13 + np.abs(angle) * 2.0**-52)
    for buf, want in ((cos, np.cos(angle) * mag), (sin, np.sin(angle) * mag)):
        got = buf.download(np.float32, guard.shape)
        assert (got[n * half:] == 7.0).all()
        assert (np.abs(got[:n * half].reshape(n, half) - want) <= tol).all()


def test_tables_match_the_reference_tables_to_rounding(gpu):
    """Unscaled, near positions: the host tables (fp32 angles, model.c:545-556) within
    what their fp32 angle loses."""
    P = gpu
    cos, sin = P.DeviceBuffer(512 * 32 * 4), P.DeviceBuffer(512 * 32 * 4)
    P.rope.make_tables(P.rope.Spec(64, 1e4), 0, 512, cos.ptr, sin.ptr)
    P.synchronize()
    want = P.rope_tables(512, 64, 1e4)
    for buf, w in zip((cos, sin), want):
        # angle up to 511, relative fp32 errors of theta (powf and a division) and of the product
        assert np.abs(buf.download(np.float32, (512, 32)) - w).max() <= 512 * 4 * 2.0**-24


def ulps(a, b):
    return np.abs(a.view(np.int32).astype(np.int64) - b.view(np.int32).astype(np.int64))


CASES = [  # rows, Hq, Hkv, D, rot, type, extra stride, offset in floats
    (1, 32, 8, 64, 64, 0, 0, 0), (7, 16, 8, 128, 128, 1, 0, 0), (300, 4, 4, 80, 80, 0, 4, 0),
    (33, 5, 1, 128, 64, 1, 8, 4), (9, 3, 3, 96, 32, 0, 0, 0), (20, 2, 1, 50, 50, 1, 2, 0),
    (20, 2, 1, 100, 50, 1, 0, 2), (5, 3, 2, 66, 34, 0, 1, 1), (4, 1, 1, 2, 2, 0, 0, 0),
    (4, 1, 1, 2, 2, 1, 3, 1), (64, 7, 1, 256, 256, 1, 0, 0), (11, 0, 3, 64, 64, 0, 0, 0),
    (11, 3, 0, 64, 16, 1, 0, 0)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rows(gpu, case, in_place):
    P = gpu
    n, Hq, Hkv, D, rot, kind, extra, off = case
    rng = np.random.default_rng(n + D)
    n_pos = 500
    angle = rng.uniform(-4, 4, (n_pos, rot // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    pos = rng.integers(0, n_pos, n).astype(np.int32)
    pos[:min(n, 2)] = [n_pos - 1, 0][:min(n, 2)]
    stride = [max(H * D, 1) + extra for H in (Hq, Hkv)]
    x = [rng.normal(size=off + n * s + 8).astype(np.float32) for s in stride]
    src = [P.DeviceBuffer.from_numpy(v) for v in x]
    guard = [np.full_like(v, 9.0) for v in x]
    dst = src if in_place else [P.DeviceBuffer.from_numpy(v) for v in guard]
    bufs = [P.DeviceBuffer.from_numpy(v) for v in (cos, sin, pos)]
    print(f"[case] rope rows {case} in_place {in_place}", flush=True)
    tab = P.rope.Tables(kind, rot, n_pos, bufs[0].ptr, bufs[1].ptr)
    P.rope.rotate(tab, n, bufs[2].ptr, D, src[0].ptr + 4 * off, Hq, stride[0],
                  dst[0].ptr + 4 * off, stride[0], src[1].ptr + 4 * off, Hkv, stride[1],
                  dst[1].ptr + 4 * off, stride[1])
    P.synchronize()
    for H, s, v, buf, g in zip((Hq, Hkv), stride, x, dst, guard):
        got = buf.download(np.float32, v.shape)
        want = (v if in_place else g).copy()
        rows = v[off:off + n * s].reshape(n, s)
        if H:
            want[off:off + n * s].reshape(n, s)[:, :H * D] = rope_ref(
                rows[:, :H * D].reshape(n, H, D), cos[pos], sin[pos], kind, rot).reshape(n, -1)
        far = ulps(got, want)
        assert far.max() <= 1 and (far > 0).mean() < 1e-3


def test_positions_outside_the_tables_give_nan(gpu):
    P = gpu
    cos = P.DeviceBuffer.from_numpy(np.ones((4, 8), np.float32))
    sin = P.DeviceBuffer.from_numpy(np.zeros((4, 8), np.float32))
    pos = P.DeviceBuffer.from_numpy(np.array([3, 4, -1, 2**31 - 1], np.int32))
    x = np.arange(4 * 24, dtype=np.float32).reshape(4, 24) + 1
    for kind in (0, 1):
        buf = P.DeviceBuffer.from_numpy(x)
        tab = P.rope.Tables(kind, 16, 4, cos.ptr, sin.ptr)
        P.rope.rotate(tab, 4, pos.ptr, 24, buf.ptr, 1, 24, buf.ptr, 24)
        P.synchronize()
        got = buf.download(np.float32, x.shape)
        assert np.array_equal(got[0], x[0])
        assert np.isnan(got[1:, :16]).all() and np.array_equal(got[1:, 16:], x[1:, 16:])


def test_tables_feed_the_existing_attention(gpu, oracle_mod):
    """Tables made on the device, scaled, in plh_attn_decode: the oracle with the
    same table values."""
    O, P = oracle_mod, gpu
    from attn_check import assert_attn_close, filled_cache, normal_f32
    cfg = P.AttnConfig(1, 8, 2, 64, 96, 1e4, 0)
    rng = np.random.default_rng(3)
    kc, vc = filled_cache(O, cfg, 70, rng)
    q, k, v = (normal_f32(rng, (1, d)) for d in (cfg.q_dim, cfg.kv_dim, cfg.kv_dim))
    cache = P.KVCache(cfg)
    cache.load(kc, vc)
    spec = P.rope.Spec(64, 1e4, "bands", 8.0, 32, 1.0, 4.0)
    P.rope.make_tables(spec, 0, 96, cache.cos.ptr, cache.sin.ptr)
    d = [P.DeviceBuffer.from_numpy(x) for x in (q, k, v)]
    out = P.DeviceBuffer(cfg.q_dim * 4)
    P.decode(cache, 0, 70, d[0].ptr, d[1].ptr, d[2].ptr, out.ptr)
    P.synchronize()
    cos, sin = (b.download(np.float32, (96, 32)) for b in (cache.cos, cache.sin))
    assert np.abs(cos[70] - cache.cos_host[70]).max() > 0.1
    shp = O.Shape(1, 8, 2, 64, 96, 1e4, 0)
    want = O.attn_decode(shp, 0, 70, q[0].copy(), k[0].copy(), v[0], kc, vc, cos, sin)
    assert_attn_close(out.download(np.float32, (cfg.q_dim,)), want, 64, 1e-3, "scaled tables")
    cache.free()
