"""The paged 8-bit cache in plain numpy, 64 bits, for the tests: natural order
[page][layer][head][token][k, v][element], the tiles' byte order, the append's
quantisation, attention, and the page operations one sequence at a time."""
import numpy as np

BLOCK = 32


def byte_of(kind, token, d):
    """Tile and byte of a block's (token, element), as picolm_hip.h states it."""
    t, e = np.broadcast_arrays(token, d)
    if kind == 0:  # token 16 h + i, element 8 g + j
        return e // 32, 256 * (e % 32 // 8) + 16 * (t % 16) + 8 * (t // 16) + e % 8
    # token 16 (j/4) + 4 g + j%4, element 16 h + i
    return e // 32, (256 * (t % 16 // 4) + 16 * (e % 16) + 8 * (e % 32 // 16) + 4 * (t // 16)
                     + t % 4)


def to_tiles(codes):
    """[..., 32 tokens, 2, D] int8 -> [..., 2, Dp/32, 1024]; elements from D on are 77."""
    lead, D = codes.shape[:-3], codes.shape[-1]
    out = np.full(lead + (2, (D + 31) // 32, 1024), 77, np.int8)
    t, d = np.arange(32)[:, None], np.arange(D)[None]
    for kind in (0, 1):
        tile, byte = byte_of(kind, t, d)
        out[..., kind, tile, byte] = codes[..., kind, :]
    return out


def from_tiles(tiles, D):
    t, d = np.arange(32)[:, None], np.arange(D)[None]
    out = np.empty(tiles.shape[:-3] + (32, 2, D), np.int8)
    for kind in (0, 1):
        tile, byte = byte_of(kind, t, d)
        out[..., kind, :] = tiles[..., kind, tile, byte]
    return out


class Ref:
    """A cache and its sequences; codes [P][L][H][B][32][2][D], scales [P][L][H][B][2]."""

    def __init__(self, L, H, D, P, page, S, max_pages):
        self.L, self.H, self.D, self.P, self.page, self.S = L, H, D, P, page, S
        self.max_pages = max_pages
        self.codes = np.zeros((P, L, H, page // BLOCK, BLOCK, 2, D), np.int8)
        self.scales = np.zeros((P, L, H, page // BLOCK, 2), np.float32)
        self.table = np.full((S, max_pages), -1, np.int32)
        self.len = np.zeros(S, np.int32)
        self.refs = np.zeros(P, np.int32)

    def fill(self, lens, rng, shuffle=True, spread=0.2):
        """Random contents, sequences of these lengths on pages anywhere."""
        self.codes[:] = np.clip(np.rint(rng.normal(0, 36, self.codes.shape)), -127, 127)
        self.scales[:] = 0.028 * np.exp(rng.normal(0, spread, self.scales.shape))
        ids = rng.permutation(self.P) if shuffle else np.arange(self.P)
        at = 0
        for s, n in enumerate(lens):
            k = -(-n // self.page)
            self.table[s, :k] = ids[at:at + k]
            self.refs[ids[at:at + k]] = 1
            self.len[s] = n
            at += k
        return self

    def pages(self, n):
        return -(-int(n) // self.page)

    def values(self, s, layer):
        """[2][H][len][D] float64 of sequence s."""
        p = self.table[s, :self.pages(self.len[s])]
        x = (self.codes[p, layer].astype(np.float64)
             * self.scales[p, layer].astype(np.float64)[:, :, :, None, :, None])
        x = x.transpose(4, 1, 0, 2, 3, 5).reshape(2, self.H, -1, self.D)
        return x[:, :, :self.len[s]]

    # ---- rows ---------------------------------------------------------------
    def append(self, layer, row_start, k, v):
        """k, v [rows][H][D] float32, already rotated."""
        for s in range(self.S):
            a, z = row_start[s], row_start[s + 1]
            start = int(self.len[s]) - (z - a)
            for pos0 in range(max(start, 0) // BLOCK * BLOCK, int(self.len[s]), BLOCK):
                lo, hi = max(pos0, start, 0), min(pos0 + BLOCK, int(self.len[s]))
                if hi <= lo:
                    continue
                page = self.table[s, pos0 // self.page]
                if not 0 <= page < self.P or self.refs[page] != 1:
                    continue
                b, u = pos0 % self.page // BLOCK, lo - pos0
                for h in range(self.H):
                    for kind, x in ((0, k), (1, v)):
                        new = x[a + lo - start:a + hi - start, h]
                        codes = self.codes[page, layer, h, b, :, kind]
                        was = self.scales[page, layer, h, b, kind]
                        amax = np.abs(new).max()
                        if u == 0:
                            codes[:] = 0
                            was = np.float32(0)
                        if not np.isfinite(amax) or not np.isfinite(was):
                            self.scales[page, layer, h, b, kind] = np.nan
                            codes[u:u + hi - lo] = 0
                            continue
                        now = max(was, np.float32(amax) / np.float32(127))
                        if u and now > was:
                            codes[:] = np.rint(codes.astype(np.float64) * np.float64(was)
                                               / np.float64(now))
                        q = np.zeros(new.shape) if now == 0 else np.clip(
                            np.rint(new.astype(np.float64) / np.float64(now)), -127, 127)
                        codes[u:u + hi - lo] = q
                        self.scales[page, layer, h, b, kind] = now

    def attention(self, layer, row_start, q):
        """q [rows][Hq][D] -> float64 [rows][Hq][D]; rows without tokens: zeros."""
        n, Hq, D = q.shape
        G = Hq // self.H
        out = np.zeros((n, Hq, D))
        for s in range(self.S):
            a, z = row_start[s], row_start[s + 1]
            if z == a:
                continue
            k, v = self.values(s, layer)
            pos = int(self.len[s]) - (z - a) + np.arange(z - a)
            hide = np.arange(int(self.len[s]))[None] > pos[:, None]
            for h in range(Hq):
                with np.errstate(invalid="ignore"):
                    w = q[a:z, h].astype(np.float64) @ k[h // G].T / np.sqrt(D)
                w[hide] = -np.inf
                top = w.max(1, initial=-np.inf, keepdims=True)
                w = np.exp(w - np.where(np.isneginf(top), 0, top))
                den = w.sum(1, keepdims=True)
                vv = v[h // G]
                for r in range(z - a):  # a hidden token's NaN stays hidden
                    if pos[r] >= 0:
                        out[a + r, h] = w[r, :pos[r] + 1] @ vv[:pos[r] + 1] / den[r]
        return out

    # ---- pages ----------------------------------------------------------------
    def drop(self, s, first):
        for e in range(first, self.pages(self.len[s])):
            self.refs[self.table[s, e]] -= 1
            self.table[s, e] = -1

    def trim(self, keep):
        for s, k in enumerate(keep):
            if 0 <= k < self.len[s]:
                self.drop(s, self.pages(k))
                self.len[s] = k

    def fork(self, parent):
        table, length = self.table.copy(), self.len.copy()
        for s, p in enumerate(parent):
            if not 0 <= p < self.S or p == s:
                continue
            self.drop(s, 0)
            n = self.pages(length[p])
            self.table[s, :n] = table[p, :n]
            self.len[s] = length[p]
        for s, p in enumerate(parent):
            if 0 <= p < self.S and p != s:
                for x in self.table[s, :self.pages(self.len[s])]:
                    self.refs[x] += 1

    def extend(self, add):
        """Sequence by sequence; the status."""
        before = [x.copy() for x in (self.table, self.len, self.refs, self.codes, self.scales)]
        over = [s for s, a in enumerate(add)
                if a > 0 and self.pages(int(self.len[s]) + int(a)) > self.max_pages]
        if over:
            return 0, over[0] + 1
        # pages that were shared by a sequence that leaves them now do not become
        # free for the later ones of the same call
        free = [int(x) for x in np.flatnonzero(self.refs == 0)]
        short = 0
        for s, a in enumerate(add):
            if a <= 0:
                continue
            have, want = self.pages(self.len[s]), self.pages(int(self.len[s]) + int(a))
            last = self.table[s, self.len[s] // self.page] if self.len[s] % self.page else -1
            copy = last >= 0 and self.refs[last] > 1
            for e in ([int(self.len[s]) // self.page] if copy else []) + list(range(have, want)):
                if e < have:
                    self.refs[last] -= 1
                if not free:
                    short += 1
                    continue
                p = free.pop(0)
                if e < have:
                    self.codes[p], self.scales[p] = self.codes[last], self.scales[last]
                self.table[s, e] = p
                self.refs[p] = 1
            self.len[s] += a
        if short:
            self.table, self.len, self.refs, self.codes, self.scales = before
        return short, 0

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        moves = [p for p in range(live, self.P) if self.refs[p] > 0]
        for to, p in zip(holes, moves):
            self.codes[to], self.scales[to] = self.codes[p], self.scales[p]
            self.refs[to], self.refs[p] = self.refs[p], 0
            self.table[self.table == p] = to
        return live, len(moves)


class Dev:
    """A Ref's contents on the device."""

    def __init__(self, P, ref):
        self.P, self.ref = P, ref
        self.cache = P.kv8.Cache(ref.L, ref.H, ref.D, ref.P, ref.page)
        self.seqs = P.kv8.Sequences(ref.S, ref.max_pages, ref.P)
        self.codes, self.scales = self.cache._own
        self.table, self.len, self.refs = self.seqs._own
        self.put()

    def put(self):
        r = self.ref
        self.codes.upload(to_tiles(r.codes))
        self.scales.upload(r.scales)
        self.table.upload(r.table)
        self.len.upload(r.len)
        self.refs.upload(r.refs)

    def state(self):
        r = self.ref
        return (self.table.download(np.int32, r.table.shape),
                self.len.download(np.int32, r.len.shape),
                self.refs.download(np.int32, r.refs.shape))

    def contents(self):
        r = self.ref
        C = (r.D + 31) // 32
        tiles = self.codes.download(np.int8, (r.P, r.L, r.H, r.page // BLOCK, 2, C, 1024))
        return from_tiles(tiles, r.D), self.scales.download(np.float32, r.scales.shape)

    def same_state(self, what=""):
        for name, got, want in zip(("table", "len", "refs"), self.state(),
                                   (self.ref.table, self.ref.len, self.ref.refs)):
            assert np.array_equal(got, want), (what, name, got, want)

    def same_contents(self, what=""):
        codes, scales = self.contents()
        assert np.array_equal(scales.view(np.uint32)[~np.isnan(self.ref.scales)],
                              self.ref.scales.view(np.uint32)[~np.isnan(self.ref.scales)]), what
        assert np.array_equal(np.isnan(scales), np.isnan(self.ref.scales)), what
        assert np.array_equal(codes, self.ref.codes), (what, np.argwhere(codes != self.ref.codes))

    def free(self):
        self.cache.free()
        self.seqs.free()


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def rope_ref(x, cos, sin, rope_type, rot):
    """x [rows][H][D] float32 by cos, sin [rows][rot/2] float32; rounded once."""
    y = x.astype(np.float64)
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    i0 = np.arange(0, rot, 2) if rope_type == 0 else np.arange(rot // 2)
    i1 = i0 + 1 if rope_type == 0 else i0 + rot // 2
    a, b = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    return y.astype(np.float32)


def attn_error(out, want):
    """Largest difference of a head row relative to the largest value of the row."""
    top = np.abs(want).max(-1)
    return float((np.abs(out - want).max(-1) / np.where(top > 0, top, 1)).max())
