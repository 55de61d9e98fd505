"""The paged 8-bit cache (plh_kv8_*) against tests/kv8_ref.py: codes, scales,
tables and counts exactly, attention against 64 bits.

Attention's tolerance.  A score is a sum of D products of codes and q parts: q keeps
22 bits (2^-22 of each element), and the fp32 sum of a column takes fewer than 96
roundings of at most 2^-24 of sum |q k|, which Cauchy bounds by |q| |k|; the exponent's
own roundings are below 2^-20 in all for scores below 2^6.  A weight is then off by a
factor 1 +- d, d = (2^-21 + 96 2^-24) |q| |k| / sqrt(D) + 2^-20, both in the numerator and
in the sum, the weights' fp16 parts and the sums of the second product by another 2^-20;
so an output is off by at most (2 d + 2^-19) max |v|."""
import numpy as np
import pytest

from kv8_ref import Dev, Ref, rope_ref, starts

pytestmark = pytest.mark.gpu


def attention_tol(ref, layer, q):
    most_k = most_v = 0.0
    for s in range(ref.S):
        if ref.len[s] and (ref.table[s, :ref.pages(ref.len[s])] >= 0).all():
            k, v = ref.values(s, layer)
            k, v = np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0)
            most_k = max(most_k, np.sqrt((k**2).sum(-1)).max())
            most_v = max(most_v, np.abs(v).max())
    nq = np.where(np.isfinite(q), q, 0).astype(np.float64)
    s = np.sqrt((nq**2).sum(-1)).max() * most_k / np.sqrt(ref.D)
    d = (2.0**-21 + 96 * 2.0**-24) * s + 2.0**-20
    return (2 * d + 2.0**-19) * most_v


def attend(P, dev, layer, Hq, row_start, q, n_rows=None, extra=0, q_off=0, out_off=0):
    """out [n_rows][Hq][D] of q [n_rows][Hq][D]; rows nobody writes hold 5."""
    n, D = q.shape[0], dev.ref.D
    width = Hq * D + extra
    qb = np.zeros(q_off + n * width + 4, np.float32)
    qb[q_off:q_off + n * width].reshape(n, width)[:, :Hq * D] = q.reshape(n, -1)
    dq = P.DeviceBuffer.from_numpy(qb)
    do = P.DeviceBuffer.from_numpy(np.full(out_off + n * width + 4, 5.0, np.float32))
    rs = P.DeviceBuffer.from_numpy(np.asarray(row_start, np.int32))
    P.kv8.attend(dev.cache, dev.seqs, layer, Hq, n if n_rows is None else n_rows, rs.ptr,
                 dq.ptr + 4 * q_off, do.ptr + 4 * out_off, width, width)
    P.synchronize()
    raw = do.download(np.float32, (out_off + n * width + 4,))
    body = raw[out_off:out_off + n * width].reshape(n, width)
    assert (raw[:out_off] == 5).all() and (raw[out_off + n * width:] == 5).all()
    assert (body[:, Hq * D:] == 5).all()
    return body[:, :Hq * D].reshape(n, Hq, D)


def check_attention(P, ref, Hq, rows, seed, layer=0, dev=None, q=None, **kw):
    rng = np.random.default_rng(seed)
    own = dev is None
    dev = dev or Dev(P, ref)
    rs = starts(rows)
    if q is None:
        q = rng.normal(size=(int(rs[-1]), Hq, ref.D)).astype(np.float32)
    out = attend(P, dev, layer, Hq, rs, q, **kw)
    want = ref.attention(layer, rs, q)
    assert np.array_equal(np.isnan(out), np.isnan(want))
    err = np.abs(out - want)[~np.isnan(want)].max(initial=0)
    assert err <= attention_tol(ref, layer, q), err
    if own:
        dev.free()
    return out


def pool_for(lens, page, spare=2):
    return sum(-(-n // page) for n in lens) + spare


def make(L, H, D, page, lens, seed, spare=2, **kw):
    rng = np.random.default_rng(seed)
    P = pool_for(lens, page, spare)
    width = max(-(-max(max(lens), 1) // page), 1) + 1
    return Ref(L, H, D, P, page, len(lens), width).fill(lens, rng, **kw)


# ---- attention ------------------------------------------------------------------


@pytest.mark.parametrize("D", [2, 6, 16, 32, 34, 48, 50, 64, 80, 96, 100, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("G", [1, 4])
def test_tokens_of_every_head_size(gpu, D, G):
    lens = [1, 31, 32, 33, 100, 257]
    ref = make(2, 2, D, 64, lens, D + G)
    print(f"[case] tokens D {D} G {G}", flush=True)
    check_attention(gpu, ref, 2 * G, [1] * len(lens), D, layer=1)


@pytest.mark.parametrize("D", [2, 18, 32, 48, 64, 80, 96, 128, 144, 180, 208, 256])
@pytest.mark.parametrize("G", [1, 3])
def test_prompts_of_every_head_size(gpu, D, G):
    lens, rows = [150, 5, 64], [130, 5, 20]
    ref = make(1, 2, D, 32, lens, D + G)
    print(f"[case] prompts D {D} G {G}", flush=True)
    check_attention(gpu, ref, 2 * G, rows, D)


@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (7, 1), (14, 2), (16, 1), (17, 1), (40, 1),
                                   (72, 1), (160, 1), (64, 8)])
@pytest.mark.parametrize("rows", [1, 2, 9])
def test_groups(gpu, heads, rows):
    """Column tiles that are partly filled, full, and several; units whose waves
    split the keys four, two and one way."""
    Hq, Hkv = heads
    lens = [300, 40, 77]
    ref = make(1, Hkv, 64, 96, lens, Hq)
    print(f"[case] groups {heads} rows {rows}", flush=True)
    check_attention(gpu, ref, Hq, [rows, 0, rows], Hq + rows)


@pytest.mark.parametrize("n", [1, 16, 511, 512, 513, 1024, 1025, 2049, 5000, 40000])
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts(gpu, n, D):
    """One token whose keys are split over workgroups from some length on."""
    ref = make(1, 2, D, 128, [n], n + D)
    print(f"[case] long {n} D {D}", flush=True)
    check_attention(gpu, ref, 8, [1], n)


@pytest.mark.parametrize("rows", [40, 200])
def test_prompt_chunk_over_a_long_context(gpu, rows):
    ref = make(1, 1, 64, 64, [9000], rows)
    print(f"[case] chunk {rows}", flush=True)
    check_attention(gpu, ref, 4, [rows], rows)


@pytest.mark.parametrize("page", [32, 64, 96, 224, 1024])
def test_mixed_batch(gpu, page):
    """Prompts, single tokens, idle and empty sequences in one call, rows behind
    the last sequence, strides and offsets that leave no 16-byte alignment."""
    lens = [700, 1, 0, 90, 333, 64, 0, 1500]
    rows = [300, 1, 0, 2, 0, 64, 0, 1]
    ref = make(1, 4, 80, page, lens, page)
    P = gpu
    dev = Dev(P, ref)
    rs = starts(rows)
    n = int(rs[-1])
    rng = np.random.default_rng(page)
    q = rng.normal(size=(n + 5, 8, 80)).astype(np.float32)
    print(f"[case] mixed page {page}", flush=True)
    outs = [attend(P, dev, 0, 8, rs, q, **kw)
            for kw in (dict(), dict(extra=4), dict(extra=3), dict(q_off=1, out_off=1))]
    want = ref.attention(0, rs, q[:n])
    for o in outs:
        assert (o[n:] == 5).all()
        assert np.abs(o[:n] - want).max() <= attention_tol(ref, 0, q)
        assert np.array_equal(o, outs[0])
    dev.free()


@pytest.mark.parametrize("n_seqs", [63, 65, 257, 1024])
def test_many_sequences(gpu, n_seqs):
    rng = np.random.default_rng(n_seqs)
    lens = [int(x) for x in rng.integers(0, 200, n_seqs)]
    rows = [min(n, 1) for n in lens]
    ref = make(1, 1, 32, 32, lens, n_seqs)
    print(f"[case] sequences {n_seqs}", flush=True)
    check_attention(gpu, ref, 3, rows, n_seqs)
    some = [int(x) if n >= x else 0 for n, x in zip(lens, rng.integers(0, 30, n_seqs))]
    check_attention(gpu, ref, 3, some, n_seqs + 1)


# Launches of many units (from two for every CU on) give a wave two tiles of columns:
# kv heads enough for that at any number of CUs up to 256.


@pytest.mark.parametrize("D", [2, 32, 50, 64, 80, 96, 128, 144, 192, 208, 256])
def test_wide_units_of_every_head_size(gpu, D):
    lens, rows = [230, 90, 40, 33, 7], [200, 70, 33, 2, 1]
    ref = make(1, 128, D, 32, lens, D)
    print(f"[case] wide units D {D}", flush=True)
    check_attention(gpu, ref, 128, rows, D)


@pytest.mark.parametrize("case", [(64, 64, 3, [1900, 2500, 31]), (128, 96, 2, [1100, 2100, 1]),
                                  (80, 128, 1, [1300, 700, 400])])
def test_wide_units_over_long_contexts(gpu, case):
    """Their chunks' partial results joined."""
    D, H, G, lens = case
    rows = [150, 65, 1]
    ref = make(1, H, D, 64, lens, D)
    # two units for each of 256 CUs
    assert sum(rows) * H * G // 128 + 3 * H >= 2 * 256
    print(f"[case] wide units {case}", flush=True)
    out = check_attention(gpu, ref, H * G, rows, D)
    assert np.array_equal(out, check_attention(gpu, ref, H * G, rows, D))


@pytest.mark.parametrize("n_seqs", [64, 65, 300])
def test_wide_units_of_many_sequences(gpu, n_seqs):
    rng = np.random.default_rng(n_seqs)
    lens = [int(x) for x in rng.integers(0, 200, n_seqs)]
    lens[5] = 1500
    ref = make(1, 8, 32, 32, lens, n_seqs)
    rows = [int(x) if n >= x else 0 for n, x in zip(lens, rng.integers(0, 60, n_seqs))]
    rows[5] = 300
    print(f"[case] wide units, sequences {n_seqs}", flush=True)
    check_attention(gpu, ref, 16, rows, n_seqs)


def test_rows_before_position_zero(gpu):
    """More rows than tokens: the first ones see nothing and give zeros."""
    for rows, lens in (([5, 3, 200], [2, 0, 150]), ([1, 1, 1], [0, 0, 1])):
        ref = make(1, 2, 64, 64, lens, 3)
        out = check_attention(gpu, ref, 4, rows, 9)
        rs = starts(rows)
        for s in range(3):
            assert (out[rs[s]:rs[s] + max(rows[s] - lens[s], 0)] == 0).all()


@pytest.mark.parametrize("case", ["jumps", "outlier", "tiny", "huge", "zero", "subnormal"])
def test_v_scales_far_apart(gpu, case):
    """The unit in which the weighted sum is kept has to follow v scales that jump
    by any power of two from block to block, up and down."""
    rng = np.random.default_rng(5)
    lens = [1000, 300, 64]
    ref = make(1, 2, 64, 64, lens, 11)
    sv = ref.scales[..., 1]
    if case == "jumps":
        sv[:] = 2.0 ** rng.integers(-60, 60, sv.shape)
    elif case == "outlier":
        sv[rng.random(sv.shape) < 0.1] = 1e20
    elif case == "tiny":
        sv[:] = 1e-30
    elif case == "huge":
        sv[:] = 1e30
    elif case == "zero":
        sv[rng.random(sv.shape) < 0.5] = 0
    else:
        sv[:] = 1e-40
    for rows in ([1, 1, 1], [40, 7, 64]):
        rs = starts(rows)
        q = rng.normal(size=(int(rs[-1]), 8, 64)).astype(np.float32)
        if case == "outlier":
            q *= 20  # softmax concentrates: the outlier's weight is far below the top's
        dev = Dev(gpu, ref)
        out = attend(gpu, dev, 0, 8, rs, q)
        want = ref.attention(0, rs, q)
        # relative to the largest weighted value of each row, not of the whole cache
        top = np.zeros(out.shape[:2])
        for s in range(3):
            k, v = ref.values(s, 0)
            for r in range(rs[s], rs[s + 1]):
                n = lens[s] - (rs[s + 1] - r) + 1
                for h in range(8):
                    w = k[h // 4, :n] @ q[r, h].astype(np.float64) / 8
                    w = np.exp(w - w.max())
                    top[r, h] = (w[:, None] * np.abs(v[h // 4, :n])).sum(0).max() / w.sum()
        s = np.sqrt((q.astype(np.float64)**2).sum(-1)).max() * 40 / 8
        d = (2.0**-21 + 96 * 2.0**-24) * s + 2.0**-20
        floor = 2.0**-149 if case == "subnormal" else 0.0  # the output's own type
        assert (np.abs(out - want) <= (2 * d + 2.0**-15) * top[..., None] + floor).all(), case
        dev.free()


def test_q_of_any_size(gpu):
    ref = make(1, 1, 64, 64, [200], 4)
    rng = np.random.default_rng(8)
    k = ref.values(0, 0)[0]
    for size in (1e-30, 1e-6, 1.0, 3e4, 1e30):
        q = rng.normal(size=(1, 4, 64)).astype(np.float32) * np.float32(size)
        if size > 1e4:  # scores too far apart for the tolerance's exponents: one key wins
            out = attend(gpu, Dev(gpu, ref), 0, 4, [0, 1], q)
            best = (q[0].astype(np.float64) @ k[0].T).argmax(1)
            gap = np.sort(q[0].astype(np.float64) @ k[0].T / 8, 1)
            sure = gap[:, -1] - gap[:, -2] > 100
            # one weight of 1 and its sum: its two fp16 parts (2^-21), its exponent's
            # logarithm and sum (2^-22 each), two exponentials and the quotient
            # (2^-22 each): below 2^-19 of each value
            assert np.allclose(out[0][sure], ref.values(0, 0)[1][0][best[sure]], rtol=2.0**-19)
            assert np.isfinite(out).all()
        else:
            check_attention(gpu, ref, 4, [1], 0, q=q)


def test_nan_and_inf_stay_where_they_are(gpu):
    """A block whose scale is NaN reaches the rows that see it and no others; a q
    head with NaN or inf its own column only."""
    ref = make(1, 2, 64, 64, [500, 100], 6)
    dev = Dev(gpu, ref)
    rs = starts([300, 1])
    rng = np.random.default_rng(1)
    q = rng.normal(size=(301, 4, 64)).astype(np.float32)
    clean = attend(gpu, dev, 0, 4, rs, q)
    page = ref.table[0, 400 // 64]
    for kind in (0, 1):
        old = ref.scales[page, 0, 1, 400 % 64 // 32, kind]
        ref.scales[page, 0, 1, 400 % 64 // 32, kind] = np.nan
        dev.put()
        out = attend(gpu, dev, 0, 4, rs, q)
        block = 400 // 32 * 32 - 200  # the first row that sees the block
        assert np.array_equal(out[:, :2], clean[:, :2])
        assert np.array_equal(out[300], clean[300])
        assert np.array_equal(out[:block, 2:], clean[:block, 2:])
        assert np.isnan(out[block:300, 2:]).all()
        ref.scales[page, 0, 1, 400 % 64 // 32, kind] = old
    dev.put()
    for bad in (np.nan, np.inf, -np.inf):
        q2 = q.copy()
        q2[7, 1, 5] = bad
        out = attend(gpu, dev, 0, 4, rs, q2)
        assert np.isnan(out[7, 1]).all()
        out[7, 1] = clean[7, 1]
        assert np.array_equal(out, clean)
    dev.free()


def test_bad_pages(gpu):
    """Page numbers outside the cache: rows that would read them give NaN, the
    others are as before; lengths past the table row are cut to it."""
    ref = make(1, 2, 64, 64, [200, 90], 12)
    dev = Dev(gpu, ref)
    rs = starts([150, 1])
    q = np.random.default_rng(2).normal(size=(151, 4, 64)).astype(np.float32)
    clean = attend(gpu, dev, 0, 4, rs, q)
    for bad in (-1, ref.P, 2**31 - 1, -2**31):
        table = ref.table.copy()
        table[0, 2] = bad
        dev.table.upload(table)
        out = attend(gpu, dev, 0, 4, rs, q)
        assert np.array_equal(out[:128 - 50], clean[:128 - 50])
        assert np.isnan(out[128 - 50:150]).all()
        assert np.array_equal(out[150], clean[150])
    dev.table.upload(ref.table)
    for long in (ref.max_pages * 64 + 1, 2**31 - 1):
        lens = ref.len.copy()
        lens[1] = long
        dev.len.upload(lens)
        out = attend(gpu, dev, 0, 4, rs, q)
        assert np.array_equal(out[:150], clean[:150]) and np.isnan(out[150]).all()
    lens[1] = -7
    dev.len.upload(lens)
    assert (attend(gpu, dev, 0, 4, rs, q)[150] == 0).all()
    dev.free()


def test_wrong_row_starts_stay_inside(gpu):
    """row_start that does not rise or leaves the batch: unspecified rows, nothing
    outside them, and the next call is right."""
    ref = make(1, 2, 64, 64, [1000, 1000, 1000], 13)
    dev = Dev(gpu, ref)
    q = np.random.default_rng(2).normal(size=(20, 4, 64)).astype(np.float32)
    good = starts([10, 3, 7])
    clean = attend(gpu, dev, 0, 4, good, q)
    for bad in ([0, 30, 5, 9], [-4, 3, 2**31 - 1, 20], [20, 10, 5, 0], [0, 20, 0, 20]):
        attend(gpu, dev, 0, 4, bad, q)
        assert np.array_equal(attend(gpu, dev, 0, 4, good, q), clean)
    dev.free()


# ---- append and fetch -------------------------------------------------------------


def run_append(P, dev, layer, rows, k, v, rope=None, q=None, k_extra=0, k_off=0):
    """k, v [n][H][D], q [n][Hq][D] or None; returns q_out."""
    ref, n = dev.ref, k.shape[0]
    width = ref.H * ref.D + k_extra
    bufs = []
    for x in (k, v):
        a = np.full(k_off + n * width, np.nan, np.float32)
        a[k_off:].reshape(n, width)[:, :ref.H * ref.D] = x.reshape(n, -1)
        bufs.append(P.DeviceBuffer.from_numpy(a))
    rs = P.DeviceBuffer.from_numpy(starts(rows))
    kw = {}
    if q is not None:
        dq = P.DeviceBuffer.from_numpy(q)
        do = P.DeviceBuffer.from_numpy(np.full(q.shape, 5.0, np.float32))
        kw = dict(q=dq.ptr, n_heads=q.shape[1], q_out=do.ptr)
    P.kv8.append(dev.cache, dev.seqs, layer, n, rs.ptr, bufs[0].ptr + 4 * k_off,
                 bufs[1].ptr + 4 * k_off, width, width, rope=rope, **kw)
    P.synchronize()
    return do.download(np.float32, q.shape) if q is not None else None


def run_fetch(P, dev, layer, rows, extra=0):
    ref, n = dev.ref, int(sum(rows))
    width = ref.H * ref.D + extra
    bufs = [P.DeviceBuffer.from_numpy(np.full((n + 1, width), 5.0, np.float32)) for _ in range(2)]
    rs = P.DeviceBuffer.from_numpy(starts(rows))
    P.kv8.fetch(dev.cache, dev.seqs, layer, n, rs.ptr, bufs[0].ptr, bufs[1].ptr, width, width)
    P.synchronize()
    got = [b.download(np.float32, (n + 1, width)) for b in bufs]
    for g in got:
        assert (g[n] == 5).all() and (g[:, ref.H * ref.D:] == 5).all()
    return [g[:n, :ref.H * ref.D].reshape(n, ref.H, ref.D) for g in got]


def check_fetch(P, dev, layer, rows, **kw):
    got = run_fetch(P, dev, layer, rows, **kw)
    ref, rs = dev.ref, starts(rows)
    for s in range(ref.S):
        n, m = int(ref.len[s]), rows[s]
        x = ref.values(s, layer).astype(np.float32)
        for kind in (0, 1):
            part = got[kind][rs[s]:rs[s + 1]]
            assert (part[:max(m - n, 0)] == 0).all()
            assert np.array_equal(part[max(m - n, 0):],
                                  x[kind].transpose(1, 0, 2)[max(n - m, 0):]), (s, kind)


@pytest.mark.parametrize("D", [2, 16, 32, 50, 64, 80, 100, 128, 162, 192, 222, 256])
@pytest.mark.parametrize("page", [32, 96])
def test_append_chunks(gpu, D, page):
    """Blocks begun, continued with and without growth, ended inside a call; each
    call twice, which stores the same."""
    rng = np.random.default_rng(D)
    ref = make(2, 3, D, page, [200, 170, 33], D)
    dev = Dev(gpu, ref)
    for step, (lens, rows) in enumerate([([70, 1, 32], [70, 1, 32]), ([71, 33, 32], [1, 32, 0]),
                                         ([72, 34, 33], [1, 1, 1]), ([200, 170, 33], [128, 136, 0])]):
        ref.len[:] = lens
        dev.len.upload(ref.len)
        n = sum(rows)
        size = np.exp(rng.normal(0, 1, (n, 1, 1)))
        k, v = ((rng.normal(size=(n, 3, D)) * size).astype(np.float32) for _ in range(2))
        if step == 1:
            k[:, 1] = 0
        ref.append(1, starts(rows), k, v)
        print(f"[case] append D {D} page {page} step {step}", flush=True)
        for extra, off in ((0, 0), (3, 1)):
            run_append(gpu, dev, 1, rows, k, v, k_extra=extra, k_off=off)
            dev.same_contents((D, page, step, extra))
        check_fetch(gpu, dev, 1, [min(r + 31, n) for r, n in zip(rows, lens)], extra=step % 3)
    dev.free()


@pytest.mark.parametrize("case", [(64, 64, 0), (64, 64, 1), (128, 64, 1), (128, 128, 1), (80, 80, 0),
                                  (96, 24, 0), (50, 50, 1), (50, 26, 0), (100, 36, 1), (256, 256, 1),
                                  (256, 128, 0), (34, 34, 1)])
@pytest.mark.parametrize("misaligned", [False, True])
def test_append_rotates(gpu, case, misaligned):
    D, rot, kind = case
    P = gpu
    rng = np.random.default_rng(D + rot)
    lens, rows = [130, 60, 9], [129, 1, 0]
    ref = make(1, 2, D, 64, lens, D)
    dev = Dev(P, ref)
    n, n_pos = sum(rows), 131
    angle = rng.uniform(-4, 4, (n_pos, rot // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    pad = 1 if misaligned else 0
    tabs = [P.DeviceBuffer.from_numpy(np.concatenate([np.zeros(pad, np.float32), t.ravel()]))
            for t in (cos, sin)]
    rope = P.rope.Tables(kind, rot, n_pos, tabs[0].ptr + 4 * pad, tabs[1].ptr + 4 * pad)
    k, v = (rng.normal(size=(n, 2, D)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(n, 6, D)).astype(np.float32)
    pos = np.concatenate([np.arange(1, 130), [59]])
    print(f"[case] append rope {case} misaligned {misaligned}", flush=True)
    # the rows as plh_rope_rows turns them (checked against 64 bits elsewhere), so
    # that codes can be compared exactly
    turned = []
    dpos = P.DeviceBuffer.from_numpy(pos.astype(np.int32))
    for x in (k, q):
        b = P.DeviceBuffer.from_numpy(x)
        w = x.shape[1] * D
        P.rope.rotate(rope, n, dpos.ptr, D, b.ptr, x.shape[1], w, b.ptr, w)
        P.synchronize()
        turned.append(b.download(np.float32, x.shape))
        assert np.abs(turned[-1] - rope_ref(x, cos[pos], sin[pos], kind, rot)).max() <= 2.0**-21
    ref.append(0, starts(rows), turned[0], v)
    q_out = run_append(P, dev, 0, rows, k, v, rope=rope, q=q, k_extra=pad, k_off=pad)
    dev.same_contents(case)
    assert np.array_equal(q_out, turned[1])
    run_append(P, dev, 0, rows, k, v, rope=rope)  # k alone: the same again
    dev.same_contents(case)
    dev.free()


def test_append_values_of_any_size(gpu):
    """Zero blocks, subnormals, the largest numbers; quotients that are ties (a
    scale of exactly 1: a row's largest is 127)."""
    rng = np.random.default_rng(0)
    D = 64
    for size in (0.0, 1e-45, 1e-40, 1e-38, 1e-20, 1e20, 2e38):
        ref = make(1, 1, D, 32, [40], 1)
        dev = Dev(gpu, ref)
        k, v = (np.clip(rng.normal(size=(40, 1, D)), -1.6, 1.6).astype(np.float32)
                * np.float32(size) for _ in range(2))
        ref.append(0, [0, 40], k, v)
        run_append(gpu, dev, 0, [40], k, v)
        dev.same_contents(size)
        dev.free()
    ref = make(1, 1, D, 32, [32], 1)
    dev = Dev(gpu, ref)
    k = (rng.integers(-252, 253, (32, 1, D)) / 2).astype(np.float32)
    k[:, :, 0] = 127.0
    near = np.nextafter(k, np.float32(0))
    near[:, :, 0] = 127.0
    ref.append(0, [0, 32], k, near)
    run_append(gpu, dev, 0, [32], k, near)
    dev.same_contents("ties")
    # growth by exactly two: every odd code is a tie
    ref.len[:] = 16
    dev.len.upload(ref.len)
    ref.append(0, [0, 16], k[:16], k[:16])
    run_append(gpu, dev, 0, [16], k[:16], k[:16])
    ref.len[:] = 17
    dev.len.upload(ref.len)
    ref.append(0, [0, 1], 2 * k[:1], 2 * k[:1])
    run_append(gpu, dev, 0, [1], 2 * k[:1], 2 * k[:1])
    dev.same_contents("growth")
    assert (ref.scales[ref.table[0, 0]] == 2).all()
    dev.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_rows_that_are_not_finite(gpu, bad):
    ref = make(1, 2, 64, 64, [70], 2)
    dev = Dev(gpu, ref)
    rng = np.random.default_rng(0)
    k, v = (rng.normal(size=(10, 2, 64)).astype(np.float32) for _ in range(2))
    k[5, 1, 3] = bad  # position 65: block 2 (rows 4..9) of head 1
    ref.append(0, [0, 10], k, v)
    run_append(gpu, dev, 0, [10], k, v)
    dev.same_contents(bad)
    assert np.isnan(ref.scales[ref.table[0, 1], 0, 1, 0, 0])
    assert np.isnan(ref.scales).sum() == 1
    # more rows do not heal the block, a call that begins it does
    ref.len[:] = 71
    dev.len.upload(ref.len)
    ref.append(0, [0, 1], v[:1], v[:1])
    run_append(gpu, dev, 0, [1], v[:1], v[:1])
    dev.same_contents(bad)
    assert np.isnan(ref.scales).sum() == 1
    ref.append(0, [0, 7], v[:7], v[:7])
    run_append(gpu, dev, 0, [7], v[:7], v[:7])
    dev.same_contents(bad)
    assert np.isnan(ref.scales).sum() == 0
    dev.free()


def test_append_drops_rows_without_a_page_of_their_own(gpu):
    """Missing, shared and impossible pages, and rows before position 0."""
    ref = make(1, 2, 64, 32, [100, 64, 3], 2)
    ref.refs[ref.table[0, 1]] = 2
    ref.table[0, 2] = -1
    ref.table[1, 0] = ref.P
    dev = Dev(gpu, ref)
    rows = [90, 64, 9]
    n = sum(rows)
    k, v = (np.random.default_rng(s).normal(size=(n, 2, 64)).astype(np.float32) for s in (0, 1))
    ref.append(0, starts(rows), k, v)
    run_append(gpu, dev, 0, rows, k, v)
    dev.same_contents()
    got = run_fetch(gpu, dev, 0, rows)
    assert np.isnan(got[0][64 - 10:96 - 10]).all() and np.isnan(got[1][90:90 + 32]).all()
    assert (got[0][154:160] == 0).all() and np.isfinite(got[0][160:]).all()
    dev.free()


def test_q_rows_behind_the_tables_and_sequences(gpu):
    P = gpu
    ref = make(1, 1, 32, 32, [40, 20], 3)
    dev = Dev(P, ref)
    cos = P.DeviceBuffer.from_numpy(np.ones((39, 16), np.float32))
    sin = P.DeviceBuffer.from_numpy(np.zeros((39, 16), np.float32))
    rope = P.rope.Tables(1, 32, 39, cos.ptr, sin.ptr)
    x = np.ones((6, 1, 32), np.float32)
    rs = P.DeviceBuffer.from_numpy(np.array([1, 3, 4], np.int32))
    b = [P.DeviceBuffer.from_numpy(x) for _ in range(3)]
    out = P.DeviceBuffer.from_numpy(np.full(x.shape, 5.0, np.float32))
    P.kv8.append(dev.cache, dev.seqs, 0, 6, rs.ptr, b[0].ptr, b[1].ptr, rope=rope, q=b[2].ptr,
                 n_heads=1, q_out=out.ptr)
    P.synchronize()
    got = out.download(np.float32, (6, 32))
    assert (got[[0, 4, 5]] == 5).all()
    assert (got[[1, 3]] == 1).all() and np.isnan(got[2]).all()
    dev.free()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("case", [(3, 1400), (70, 60), (65, 1), (300, 2), (1024, 5)])
def test_append_many_rows_and_sequences(gpu, case, kind):
    """Few and many sequences, rows enough that a workgroup takes several q rows; q
    is rotated in place, and everything is read back."""
    n_seqs, rows = case
    P, D = gpu, 32
    rng = np.random.default_rng(n_seqs + kind)
    rows = [int(x) for x in rng.integers(max(rows - 8, 0), rows + 1, n_seqs)]
    lens = [m + int(x) for m, x in zip(rows, rng.integers(0, 40, n_seqs))]
    n = sum(rows)
    ref = make(1, 2, D, 64, lens, n_seqs)
    dev = Dev(P, ref)
    n_pos = max(lens)
    angle = rng.uniform(-4, 4, (n_pos, 12))
    tabs = [P.DeviceBuffer.from_numpy(f(angle).astype(np.float32)) for f in (np.cos, np.sin)]
    rope = P.rope.Tables(kind, 24, n_pos, tabs[0].ptr, tabs[1].ptr)
    k, v = (rng.normal(size=(n, 2, D)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(n, 3, D)).astype(np.float32)
    pos = np.concatenate([np.arange(a - m, a) for a, m in zip(lens, rows)]).astype(np.int32)
    print(f"[case] append {case} kind {kind}", flush=True)
    dpos, drs = P.DeviceBuffer.from_numpy(pos), P.DeviceBuffer.from_numpy(starts(rows))
    turned = []
    for x in (k, q):
        b = P.DeviceBuffer.from_numpy(x)
        w = x.shape[1] * D
        P.rope.rotate(rope, n, dpos.ptr, D, b.ptr, x.shape[1], w, b.ptr, w)
        P.synchronize()
        turned.append(b.download(np.float32, x.shape))
    ref.append(0, starts(rows), turned[0], v)
    dk, dv, dq = (P.DeviceBuffer.from_numpy(x) for x in (k, v, q))
    P.kv8.append(dev.cache, dev.seqs, 0, n, drs.ptr, dk.ptr, dv.ptr, rope=rope, q=dq.ptr,
                 n_heads=3, q_out=dq.ptr)
    P.synchronize()
    assert np.array_equal(dq.download(np.float32, q.shape), turned[1])
    dev.same_contents(case)
    check_fetch(P, dev, 0, rows)
    dev.free()


# ---- pages ----------------------------------------------------------------------


def vec(P, x):
    return P.DeviceBuffer.from_numpy(np.asarray(x, np.int32))


def status(P, buf):
    P.synchronize()
    return tuple(int(x) for x in buf.download(np.int32, (2,)))


@pytest.mark.parametrize("seed", range(8))
def test_page_operations_in_any_order(gpu, seed):
    """Random operations on a small pool that runs out now and then: tables, lengths,
    counts, statuses and contents as the sequence-by-sequence form has them."""
    P = gpu
    rng = np.random.default_rng(seed)
    page = int(rng.choice([32, 64, 160]))
    ref = Ref(2, 2, int(rng.choice([32, 80])), int(rng.integers(6, 40)), page,
              int(rng.integers(1, 12)), int(rng.integers(2, 9)))
    ref.codes[:] = rng.integers(-127, 128, ref.codes.shape)
    ref.scales[:] = rng.random(ref.scales.shape)
    dev = Dev(P, ref)
    st = vec(P, [-1, -1])
    done = {}
    for step in range(40):
        op = rng.choice(["extend", "extend", "extend", "trim", "fork", "compact"])
        if op == "extend":
            x = rng.integers(-2, page * 2, ref.S) * (rng.random(ref.S) < 0.5)
            want = ref.extend(x)
            P.kv8.extend(dev.cache, dev.seqs, vec(P, x).ptr, st.ptr)
            assert status(P, st) == want, (seed, step, x)
            op += "" if want == (0, 0) else " refused"
        elif op == "trim":
            x = np.where(rng.random(ref.S) < 0.4, rng.integers(0, page * 4, ref.S), -1)
            ref.trim(x)
            P.kv8.trim(dev.cache, dev.seqs, vec(P, x).ptr)
        elif op == "fork":
            x = np.where(rng.random(ref.S) < 0.5, rng.integers(-1, ref.S + 1, ref.S), -1)
            ref.fork(x)
            P.kv8.fork(dev.cache, dev.seqs, vec(P, x).ptr)
        else:
            want = ref.compact()
            P.kv8.compact(dev.cache, dev.seqs, st.ptr)
            assert status(P, st) == want, (seed, step)
        P.synchronize()
        dev.same_state((seed, step, op))
        dev.same_contents((seed, step, op))
        done[op] = done.get(op, 0) + 1
    assert len(done) >= 4, done
    dev.free()


def test_fork_permutes(gpu):
    P = gpu
    ref = make(1, 1, 32, 32, [100, 33, 0, 64], 1)
    dev = Dev(P, ref)
    for x in ([1, 2, 3, 0], [3, 3, 0, 0], [0, 1, 2, 3], [2, 2, 2, 2]):
        ref.fork(x)
        P.kv8.fork(dev.cache, dev.seqs, vec(P, x).ptr)
        dev.same_state(x)
    dev.free()


@pytest.mark.parametrize("shape", [(200, 50), (1024, 12), (3, 4000)])
def test_pages_of_large_tables(gpu, shape):
    """Forks beyond one workgroup's table, branches of one parent that all grow, ends
    and compaction."""
    P = gpu
    S, width = shape
    rng = np.random.default_rng(S)
    n_pages = 4 * S + 3 * width
    ref = Ref(1, 1, 32, n_pages, 32, S, width)
    ref.codes[:] = rng.integers(-127, 128, ref.codes.shape)
    dev = Dev(P, ref)
    st = vec(P, [-1, -1])
    add = np.zeros(S, np.int64)
    add[:3] = [32 * (width - 2) + 5, 40, 7]
    x = np.full(S, -1)
    x[3:] = rng.integers(0, 3, S - 3)
    shift = np.where(rng.random(S) < 0.5, rng.integers(0, S, S), -1)
    print(f"[case] large tables {shape}", flush=True)
    for step, (op, arg) in enumerate([("extend", add), ("fork", x), ("extend", np.ones(S, int)),
                                      ("fork", shift), ("extend", rng.integers(0, 9, S)),
                                      ("trim", np.where(rng.random(S) < 0.6, 0, -1)),
                                      ("compact", None)]):
        if op in ("extend", "compact"):
            want = ref.extend(arg) if op == "extend" else ref.compact()
            getattr(P.kv8, op)(dev.cache, dev.seqs, *([] if arg is None else [vec(P, arg).ptr]),
                               st.ptr)
            assert status(P, st) == want, step
        else:
            getattr(ref, op)(arg)
            getattr(P.kv8, op)(dev.cache, dev.seqs, vec(P, arg).ptr)
        P.synchronize()
        dev.same_state((step, op))
        dev.same_contents((step, op))
    dev.free()


@pytest.mark.parametrize("n_pages", [1, 4095, 4096, 4097, 20000])
def test_allocation_over_many_pages(gpu, n_pages):
    """The free pages are the last ones, or every third; a request for all of them,
    for one more, and of one long sequence."""
    P = gpu
    rng = np.random.default_rng(n_pages)
    S = 3
    ref = Ref(1, 1, 2, n_pages, 32, S, n_pages + 2)
    for free in (np.arange(n_pages) >= n_pages - 1, np.arange(n_pages) % 3 == 0):
        used = np.flatnonzero(~free)
        ref.table[:] = -1
        ref.table[0, :len(used)] = rng.permutation(used)
        ref.len[:] = [32 * len(used), 0, 0]
        ref.refs[:] = ~free
        n = int(free.sum())
        for add in ([0, 32 * n + 1, 0], [0, 32 * (n - n // 2), 32 * (n // 2)]):
            dev = Dev(P, ref)
            st = vec(P, [-1, -1])
            want = ref.extend(add)
            P.kv8.extend(dev.cache, dev.seqs, vec(P, add).ptr, st.ptr)
            assert status(P, st) == want == ((1, 0) if add[1] > 32 * n else (0, 0))
            dev.same_state((n_pages, add))
            ref.trim([-1, 0, 0])
            P.kv8.trim(dev.cache, dev.seqs, vec(P, [-1, 0, 0]).ptr)
            dev.same_state((n_pages, add, "trim"))
            # and what is left moves down
            keep = [32 * (len(used) // 2), -1, -1]
            saved = [x.copy() for x in (ref.table, ref.len, ref.refs, ref.codes, ref.scales)]
            ref.trim(keep)
            P.kv8.trim(dev.cache, dev.seqs, vec(P, keep).ptr)
            want = ref.compact()
            P.kv8.compact(dev.cache, dev.seqs, st.ptr)
            assert status(P, st) == want
            dev.same_state((n_pages, "compact"))
            ref.table, ref.len, ref.refs, ref.codes, ref.scales = saved
            dev.free()


def test_extend_to_the_end_of_the_table(gpu):
    P = gpu
    ref = make(1, 1, 32, 32, [64, 10], 1, spare=10)  # 3 entries a row
    dev = Dev(P, ref)
    st = vec(P, [-1, -1])
    for add, want in (([32, 0], (0, 0)), ([1, 5], (0, 1)), ([0, 2**31 - 1], (0, 2)),
                      ([2**31 - 1, 2**31 - 1], (0, 1)), ([-5, -2**31], (0, 0))):
        assert ref.extend(add) == want
        P.kv8.extend(dev.cache, dev.seqs, vec(P, add).ptr, st.ptr)
        assert status(P, st) == want
        dev.same_state(add)
    dev.free()


# ---- together ---------------------------------------------------------------------


def test_serving_steps(gpu):
    """Prompts, branches, growth, an ended sequence and compaction, with rotation:
    every layer's attention against the reference after every step, and unchanged
    bit for bit by the pages' moves."""
    P = gpu
    rng = np.random.default_rng(42)
    L, Hkv, Hq, D, page = 2, 2, 6, 64, 64
    ref = Ref(L, Hkv, D, 40, page, 4, 8)
    dev = Dev(P, ref)
    n_pos = 512
    spec = P.rope.Spec(32, 1e4, "linear", 2.0)
    cos, sin = P.DeviceBuffer(n_pos * 64), P.DeviceBuffer(n_pos * 64)
    P.rope.make_tables(spec, 0, n_pos, cos.ptr, sin.ptr)
    rope = P.rope.Tables(1, 32, n_pos, cos.ptr, sin.ptr)
    P.synchronize()
    c, s = (b.download(np.float32, (n_pos, 16)) for b in (cos, sin))
    st = vec(P, [-1, -1])

    def step(rows):
        assert ref.extend(rows) == (0, 0)
        P.kv8.extend(dev.cache, dev.seqs, vec(P, rows).ptr, st.ptr)
        assert status(P, st) == (0, 0)
        dev.same_state(rows)
        rs = starts(rows)
        n = int(rs[-1])
        pos = np.concatenate([int(ref.len[i]) - r + np.arange(r) for i, r in enumerate(rows)])
        outs = []
        for layer in range(L):
            k, v = (rng.normal(size=(n, Hkv, D)).astype(np.float32) for _ in range(2))
            q = rng.normal(size=(n, Hq, D)).astype(np.float32)
            turned = [rope_ref(x, c[pos], s[pos], 1, 32) for x in (k, q)]
            ref.append(layer, rs, turned[0], v)
            q_out = run_append(P, dev, layer, rows, k, v, rope=rope, q=q)
            assert np.abs(q_out - turned[1]).max() <= 2.0**-21
            # the device's own codes from here on (a rotation's last place may
            # turn a code that lies on a border)
            codes, scales = dev.contents()
            assert (codes != ref.codes).mean() < 1e-4 and np.allclose(scales, ref.scales, rtol=1e-6)
            ref.codes, ref.scales = codes, scales
            outs.append((q_out, check_attention(P, ref, Hq, rows, 0, layer, dev, q=q_out)))
        return outs

    step([100, 37, 0, 0])
    step([1, 1, 0, 0])
    ref.fork([-1, -1, 0, 0])
    P.kv8.fork(dev.cache, dev.seqs, vec(P, [-1, -1, 0, 0]).ptr)
    dev.same_state("fork")
    step([1, 1, 1, 30])
    step([0, 200, 1, 1])
    ref.trim([0, -1, 101, -1])
    P.kv8.trim(dev.cache, dev.seqs, vec(P, [0, -1, 101, -1]).ptr)
    dev.same_state("trim")
    rows = [0, 1, 1, 5]
    outs = step(rows)
    want = ref.compact()
    P.kv8.compact(dev.cache, dev.seqs, st.ptr)
    assert status(P, st) == want and want[1] > 0
    dev.same_state("compact")
    for layer, (q, out) in enumerate(outs):
        assert np.array_equal(attend(P, dev, layer, Hq, starts(rows), q), out)
    step([0, 1, 1, 1])
    dev.free()


def test_captured_steps(gpu):
    """A decode step (extend, append, attention) captured once and replayed: lengths
    and pages follow on the device.  Two graphs that share the workspace and eager
    calls take turns; every replay equals the eager steps of a second cache."""
    P = gpu
    rng = np.random.default_rng(9)
    Hkv, Hq, D, page, S = 2, 8, 64, 32, 3
    lens = [600, 1500, 31]
    refs = [make(1, Hkv, D, page, lens, 77, spare=30) for _ in range(2)]
    for r in refs:
        r.max_pages += 8
        r.table = np.pad(r.table, ((0, 0), (0, 8)), constant_values=-1)
    devs = [Dev(P, r) for r in refs]
    one, many = [1, 1, 1], [2, 40, 0]
    bufs = []
    for rows in (one, many):
        n = sum(rows)
        bufs.append([P.DeviceBuffer(n * h * D * 4) for h in (Hkv, Hkv, Hq, Hq)]
                    + [vec(P, rows), vec(P, starts(rows)), vec(P, [-1, -1])])

    def step(dev, which):
        k, v, q, out, add, rs, st = (b.ptr for b in bufs[which])
        n = sum((one, many)[which])
        P.kv8.extend(dev.cache, dev.seqs, add, st)
        P.kv8.append(dev.cache, dev.seqs, 0, n, rs, k, v)
        P.kv8.attend(dev.cache, dev.seqs, 0, Hq, n, rs, q, out)

    def inputs(which, seed):
        r = np.random.default_rng(seed)
        for b in bufs[which][:3]:
            b.upload(r.normal(size=b.nbytes // 4).astype(np.float32))

    # sizes the workspace once, on a state that is put back
    for which in (0, 1):
        inputs(which, which)
        step(devs[0], which)
    P.synchronize()
    devs[0].put()
    graphs = []
    for which in (0, 1):
        with P.Graph() as g:
            step(devs[0], which)
        graphs.append(g)
    for turn in range(6):
        which = turn % 2 if turn < 4 else 0
        got = []
        inputs(which, 100 + turn)
        for dev in devs:
            bufs[which][3].zero()
            if dev is devs[0]:
                graphs[which].launch()
            else:
                step(dev, which)
            assert status(P, bufs[which][6]) == (0, 0)
            n = sum((one, many)[which])
            got.append((bufs[which][3].download(np.float32, (n, Hq * D)), dev.state(),
                        dev.contents()))
        for a, b in zip(got[0][1], got[1][1]):
            assert np.array_equal(a, b), turn
        assert np.array_equal(got[0][0], got[1][0]), turn
        for a, b in zip(got[0][2], got[1][2]):
            assert np.array_equal(a, b), turn
    for d in devs:
        d.free()


def test_same_results_every_time(gpu):
    """Cut units are joined in the order of their chunks."""
    ref = make(1, 2, 128, 64, [20000, 3000, 77], 1)
    dev = Dev(gpu, ref)
    q = np.random.default_rng(0).normal(size=(3, 16, 128)).astype(np.float32)
    outs = [attend(gpu, dev, 0, 16, [0, 1, 2, 3], q) for _ in range(8)]
    assert all(np.array_equal(o, outs[0]) for o in outs)
    dev.free()


def test_offsets_past_32_bits(gpu):
    """Pages that lie past 4 GiB of codes."""
    P = gpu
    rng = np.random.default_rng(0)
    H, L, page = 8, 32, 1024  # 32 MiB a page of codes
    n_pages = 140
    big = P.kv8.Cache(L, H, 64, n_pages, page)
    keep = [vec(P, [n_pages - 1]), vec(P, [100]), vec(P, np.ones(n_pages))]
    seqs = P.kv8.Sequences(1, 1, table=keep[0].ptr, lens=keep[1].ptr, refs=keep[2].ptr)
    rs = vec(P, [0, 100])
    k, v = (rng.normal(size=(100, H * 64)).astype(np.float32) for _ in range(2))
    b = [P.DeviceBuffer.from_numpy(x) for x in (k, v, k, v)]
    P.kv8.append(big, seqs, L - 1, 100, rs.ptr, b[0].ptr, b[1].ptr)
    P.kv8.fetch(big, seqs, L - 1, 100, rs.ptr, b[2].ptr, b[3].ptr)
    P.synchronize()
    for x, y in ((k, b[2]), (v, b[3])):
        # half a step of a block's scale
        assert np.abs(y.download(np.float32, x.shape) - x).max() <= np.abs(x).max() / 127 * 0.5001
    out = P.DeviceBuffer(H * 64 * 4)
    one = vec(P, [0, 1])
    P.kv8.attend(big, seqs, L - 1, H, 1, one.ptr, b[0].ptr, out.ptr)
    P.synchronize()
    got = out.download(np.float32, (H, 64))
    kk, vv = (y.download(np.float32, (100, H, 64)).astype(np.float64) for y in (b[2], b[3]))
    for h in range(H):
        w = kk[:, h] @ k[0, h * 64:h * 64 + 64].astype(np.float64) / 8
        w = np.exp(w - w.max())
        assert np.abs(got[h] - w @ vv[:, h] / w.sum()).max() <= 1e-4
    big.free()
