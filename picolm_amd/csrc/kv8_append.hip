// kv8_append.hip -- rows into the paged 8-bit cache and back as values
// (include/picolm_hip.h, plh_kv8_append and plh_kv8_fetch).
#include <limits.h>
#include <math.h>

#include "attn_common.h"
#include "kv8.h"

namespace plh {

int kv_check(const plh_kv8_cache* c, const plh_kv8_seqs* s, const char* what) {
  if (!c || !s) {
    set_error("%s: no cache or no sequences", what);
    return -1;
  }
  if (plh_kv8_code_bytes(c) == 0) {
    set_error("%s: a cache of %d layers, %d kv heads of %d, %d pages of %d tokens is not built",
              what, c->n_layers, c->n_kv_heads, c->head_dim, c->n_pages, c->page_tokens);
    return -1;
  }
  if (!c->codes || !c->scales || ((uintptr_t)c->codes & 15) || ((uintptr_t)c->scales & 3)) {
    set_error("%s: codes (16-byte aligned) or scales are missing", what);
    return -1;
  }
  if (s->n_seqs < 1 || s->n_seqs > kKvMaxSeqs || s->max_pages < 1 ||
      (int64_t)s->max_pages * c->page_tokens >= (1 << 30)) {
    set_error("%s: %d sequences (1..%d) of %d pages of %d tokens (below 2^30 in all)", what,
              s->n_seqs, kKvMaxSeqs, s->max_pages, c->page_tokens);
    return -1;
  }
  if (!s->table || !s->len || !s->refs) {
    set_error("%s: table, len or refs is null", what);
    return -1;
  }
  return 0;
}

int kv_ready(const char* what) {
  if (ctx().stream) return 0;
  set_error("%s: library not initialised", what);
  return -1;
}

int kv_view(const plh_kv8_cache* c, const plh_kv8_seqs* s, int layer, int n_rows,
            const int32_t* row_start, const char* what, KvView& v) {
  if (kv_check(c, s, what)) return -1;
  if (layer < 0 || layer >= c->n_layers) {
    set_error("%s: layer %d of %d", what, layer, c->n_layers);
    return -1;
  }
  if (n_rows < 0 || (n_rows && !row_start)) {
    set_error("%s: %d rows, row_start %p", what, n_rows, (const void*)row_start);
    return -1;
  }
  const int64_t head = (int64_t)(c->page_tokens / kKvBlock) * 2 * kv_tiles(c->head_dim) * kKvTile;
  const int64_t head_scales = (int64_t)(c->page_tokens / kKvBlock) * 2;
  v = KvView{};
  v.codes = c->codes + layer * c->n_kv_heads * head;
  v.scales = c->scales + layer * c->n_kv_heads * head_scales;
  v.page_codes = c->n_layers * c->n_kv_heads * head;
  v.page_scales = c->n_layers * c->n_kv_heads * head_scales;
  v.n_kv_heads = c->n_kv_heads, v.D = c->head_dim, v.blocks = c->page_tokens / kKvBlock;
  v.n_pages = c->n_pages, v.n_seqs = s->n_seqs, v.max_pages = s->max_pages;
  v.table = s->table, v.len = s->len, v.refs = s->refs;
  v.row_start = row_start, v.n_rows = n_rows;
  v.fd_blocks = make_fastdiv((uint32_t)v.blocks);
  return 0;
}

namespace {

struct AppendArgs {
  KvView v;
  const float *k, *vv;
  int k_stride, v_stride;
  int groups;      // workgroups of a slot: Share::kJobs jobs (a head's k or v) each
  FastDiv fd_groups;
  int block_wgs;   // workgroups of the slots; those behind them rotate q rows
  int q_rows;      // rows of such a workgroup (1..kQRows)
  int rope;        // rotate
  int k_vec;       // float4 reads of k rows and tables
  RopeRows r;      // the tables, and q
};

constexpr int kQRows = 4;
enum { PLAIN, LLAMA, QWEN };  // how a kernel rotates

// x / s rounded to the nearest integer, ties to even, as the 64-bit quotient
// rounds: x times the fp32 reciprocal is within 3e-5 of the quotient (|quotient|
// below 128), which decides all but the values within 1e-4 of a tie; those
// (and reciprocals that overflow) take the 64-bit division.
__device__ __forceinline__ int quant(float x, float s, float inv) {
  const float y = x * inv;
  float r = __builtin_rintf(y);
  if (!(__builtin_fabsf(y - r) < 0.4999f)) r = (float)__builtin_rint((double)x / (double)s);
  return min(max((int)r, -127), 127);
}
// c * was / now likewise (was <= now: no clamp is needed).
__device__ __forceinline__ int requant(int c, float was, float now, float ratio) {
  const float y = (float)c * ratio;
  float r = __builtin_rintf(y);
  if (!(__builtin_fabsf(y - r) < 0.4999f))
    r = (float)__builtin_rint((double)c * (double)was / (double)now);
  return (int)r;
}

__device__ __forceinline__ float wave_amax(float x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = vmax(x, __shfl_xor(x, o, 64));
  return x;
}

// Loads stay where they are written: all of a row's before the first use (the
// compiler otherwise puts each into a branch of its own, one latency after the
// other).
template <int N>
__device__ __forceinline__ void here(float (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[n]));
}

// N elements of a row from d on, inside it (D elements) whatever d is.
template <int N, bool VEC>
__device__ __forceinline__ void load_n(const float* row, int d, int D, float (&x)[N]) {
  if (VEC) {
#pragma unroll
    for (int n = 0; n < N; n += 4) {
      const float4 a = *(const float4*)(row + min(d + n, D - 4));
      x[n] = a.x, x[n + 1] = a.y, x[n + 2] = a.z, x[n + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = row[min(d + n, D - 1)];
  }
}

// What turns a k row's elements 32 (c0 + t) + e .. + 3: the tables' entries and, in
// half-split pairs, the elements' partners.  VEC: half of the rotated part is a
// multiple of 4, so that all four lie on one side of it.  (Without branches: the
// compiler otherwise waits for one element's loads before it asks for the next's.)
template <int N, int MODE, bool VEC>
struct Turn {
  float y[N][4], c[N][4], s[N][4];
  bool known;

  __device__ __forceinline__ void load(const AppendArgs& a, const float* row, int c0, int e,
                                       int pos) {
    const int rot = a.r.rot, half = rot / 2;
    known = pos < a.r.n_pos;
    const int64_t tab = (int64_t)(known ? pos : 0) * half;
    const float* cos_t = a.r.cos_t + tab;
    const float* sin_t = a.r.sin_t + tab;
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int d = 32 * (c0 + t) + e;
      if (MODE == LLAMA && VEC) {
        const int k = min(d / 2, half - 2);
        const float2 c2 = *(const float2*)(cos_t + k), s2 = *(const float2*)(sin_t + k);
        c[t][0] = c2.x, c[t][1] = c2.y, s[t][0] = s2.x, s[t][1] = s2.y;
      } else if (MODE == LLAMA) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = min(d / 2 + j, half - 1);
          c[t][j] = cos_t[k], s[t][j] = sin_t[k];
        }
      } else if (VEC) {
        const int k = min(d, rot - 4);
        const bool lo = k < half;
        load_n<4, true>(row, lo ? k + half : k - half, a.v.D, y[t]);
        load_n<4, true>(cos_t, lo ? k : k - half, half, c[t]);
        load_n<4, true>(sin_t, lo ? k : k - half, half, s[t]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int f = min(d + j, rot - 1), k = f < half ? f : f - half;
          y[t][j] = row[f < half ? f + half : f - half];
          c[t][j] = cos_t[k], s[t][j] = sin_t[k];
        }
      }
    }
  }
  __device__ __forceinline__ void stay() {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int j = 0; j < (MODE == LLAMA ? 2 : 4); ++j) {
        if (MODE == QWEN) asm volatile("" : "+v"(y[t][j]));
        asm volatile("" : "+v"(c[t][j]), "+v"(s[t][j]));
      }
  }

  __device__ __forceinline__ void apply(const AppendArgs& a, int c0, int e, float (&x)[N][4]) {
    const int rot = a.r.rot, half = rot / 2;
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int d = 32 * (c0 + t) + e;
      if (MODE == LLAMA) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x0 = x[t][2 * j], x1 = x[t][2 * j + 1];
          rotate_pair(x0, x1, known ? c[t][j] : nan, known ? s[t][j] : nan);
          const bool in = d + 2 * j < rot;
          x[t][2 * j] = in ? x0 : x[t][2 * j], x[t][2 * j + 1] = in ? x1 : x[t][2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // (the pair's output that this element is: rotate_pair's bits, as products
          // of two fp32 values are exact)
          const int f = d + j;
          const double sn = known ? (f < half ? -s[t][j] : s[t][j]) : nan;
          const double cs = known ? c[t][j] : nan;
          const float r = (float)__builtin_fma((double)x[t][j], cs, (double)y[t][j] * sn);
          x[t][j] = f >= rot ? x[t][j] : r;
        }
      }
    }
  }
};

// A block's place and its new rows.
struct Place {
  int row0, start;  // first row of the sequence's, and its position
  int t0, lo, len;  // the block's first token; new rows are positions lo..len-1
  int head, is_v;
};

// The block's scale, given the largest magnitude of its new rows.
struct Scale {
  float was, now, ratio, inv;
  bool grown, zero;
  __device__ __forceinline__ Scale(float amax, float was_, bool older) : was(was_) {
    const float need = amax / 127.0f;
    now = older ? fmaxf(was, need) : need;
    const bool bad = !(amax < INFINITY) || !(was < INFINITY);
    if (bad) now = __builtin_nanf("");
    grown = older && now > was;  // false where bad
    ratio = grown ? was / now : 1.0f;
    zero = bad || now == 0.0f;
    inv = zero ? 0.0f : 1.0f / now;
  }
  __device__ __forceinline__ int code(float x) const { return zero ? 0 : quant(x, now, inv); }
};

// Sixteen values of a lane as codes.  x times the reciprocal plus 1.5 * 2^23 rounds
// to the nearest integer, ties to even, and has it in its low byte; the
// reciprocal's rounding moves a quotient below 128 by less than 1e-5, so only
// where a wave has a value that near a tie (one wave in fifty) are all of them
// taken from 64-bit quotients.
__device__ __forceinline__ void codes16(const float (&x)[16], const Scale& s, uint32_t (&w)[4]) {
  constexpr float kMagic = 12582912.0f;
  float worst = 0.0f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = x[4 * q + e], n = __builtin_fmaf(y, s.inv, kMagic);
      worst = vmax(worst, __builtin_fabsf(__builtin_fmaf(y, s.inv, -(n - kMagic))));
      t[e] = __float_as_uint(n);
    }
    const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(t[3], t[2], 0x0C0C0400u);
    w[q] = lo | hi << 16;
  }
  if (s.zero) {
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = 0;
  } else if (__any(!(worst < 0.49998f))) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      w[q] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[q] |= (uint32_t)(s.code(x[4 * q + e]) & 0xFF) << (8 * e);
    }
  }
}

// Sixteen codes of a lane rounded again.
__device__ __forceinline__ uint4 requant16(uint4 old, const Scale& s) {
  uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t out = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out |= (uint32_t)(requant((int)(int8_t)(w[q] >> (8 * e)), s.was, s.now, s.ratio) & 0xFF)
             << (8 * e);
    w[q] = out;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One new row in a block (a single token): two elements a lane at a time, the pairs
// that rotate together, and single bytes stored.  The block's tiles are only
// touched where its scale grows, or cleared where the row begins it.
template <int DT, int MODE>
__device__ __forceinline__ void append_row(const AppendArgs& a, const Place& p, uint4* tiles,
                                           float* scale, bool may_store) {
  constexpr int kPairs = (16 * DT + 63) / 64;  // of a lane
  const int lane = threadIdx.x & 63, D = a.v.D;
  const int pos = max(p.t0, p.lo), t = pos - p.t0;
  const bool older = p.lo > p.t0;
  const float* row = (p.is_v ? a.vv + (int64_t)(p.row0 + pos - p.start) * a.v_stride
                             : a.k + (int64_t)(p.row0 + pos - p.start) * a.k_stride) +
                     p.head * D;
  const float was = older ? *scale : 0.0f;
  const bool turn = !p.is_v && MODE != PLAIN;
  const int rot = turn ? a.r.rot : 0, half = rot / 2;
  const bool known = pos < a.r.n_pos;
  const int64_t tab = (int64_t)(known ? pos : 0) * half;
  float x[kPairs][2];
  int d[kPairs][2];
  float amax = 0.0f;
#pragma unroll
  for (int n = 0; n < kPairs; ++n) {
    const int i = lane + 64 * n;
    const bool in = i < D / 2, rotates = i < half;
    d[n][0] = rotates && MODE == QWEN ? i : 2 * i;
    d[n][1] = rotates && MODE == QWEN ? i + half : 2 * i + 1;
    x[n][0] = in ? row[d[n][0]] : 0.0f;
    x[n][1] = in ? row[d[n][1]] : 0.0f;
    if (rotates) {
      const float nan = __builtin_nanf("");
      const float c = a.r.cos_t[tab + i], s = a.r.sin_t[tab + i];
      rotate_pair(x[n][0], x[n][1], known ? c : nan, known ? s : nan);
    }
    amax = vmax(amax, vmax(__builtin_fabsf(x[n][0]), __builtin_fabsf(x[n][1])));
  }
  const Scale s(wave_amax(amax), was, older);
  if (!may_store) return;
  if (s.grown || !older) {
#pragma unroll 1
    for (int c = 0; c < DT; ++c)
      tiles[c * 64 + lane] =
          older ? requant16(tiles[c * 64 + lane], s) : make_uint4(0u, 0u, 0u, 0u);
    // the bytes below lie in other lanes' sixteen
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
  }
  int8_t* bytes = (int8_t*)tiles;
#pragma unroll
  for (int n = 0; n < kPairs; ++n)
    if (lane + 64 * n < D / 2)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = d[n][e], in = k & 31;
        const int at = p.is_v
                           ? 256 * ((t & 15) >> 2) + 16 * (in & 15) + 8 * (in >> 4) +
                                 4 * (t >> 4) + (t & 3)
                           : 256 * (in >> 3) + 16 * (t & 15) + 8 * (t >> 4) + (in & 7);
        bytes[(k >> 5) * kKvTile + at] = (int8_t)s.code(x[n][e]);
      }
  // elements behind D of the last tile
  for (int k = D + lane; k < 32 * DT; k += 64) {
    const int in = k & 31;
    const int at = p.is_v ? 256 * ((t & 15) >> 2) + 16 * (in & 15) + 8 * (in >> 4) + 4 * (t >> 4) +
                                (t & 3)
                          : 256 * (in >> 3) + 16 * (t & 15) + 8 * (t >> 4) + (in & 7);
    bytes[(k >> 5) * kKvTile + at] = 0;
  }
  if (lane == 0) *scale = s.now;
}

// How the four waves of a workgroup share its jobs (a block of a kv head's k or v):
// a wave a tile, two tiles of wide heads.
template <int DT>
struct Share {
  static constexpr int kWaves = DT < 4 ? (DT == 3 ? 4 : DT) : 4;  // of a job
  static constexpr int kTiles = (DT + 3) / 4;                     // of a wave
  static constexpr int kJobs = 4 / kWaves;                        // of a workgroup
};

// Elements e + j of tokens 8 n + u of a k block's tiles c0.., rotated, as x[t][4 n + j].
// ask: what else is asked for meanwhile.
template <int T, int MODE, bool VEC, class Ask>
__device__ __forceinline__ void k_values(const AppendArgs& a, const Place& p, int c0, int e, int u,
                                         Ask ask, float (&x)[T][16]) {
  float y[4][T][4];
  Turn<T, MODE, VEC> turn[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int at = min(max(p.t0 + 8 * n + u, p.lo), p.len - 1);
    const float* row = a.k + (int64_t)(p.row0 + at - p.start) * a.k_stride + p.head * a.v.D;
#pragma unroll
    for (int t = 0; t < T; ++t) load_n<4, VEC>(row, 32 * (c0 + t) + e, a.v.D, y[n][t]);
    if (MODE != PLAIN) turn[n].load(a, row, c0, e, at);
  }
  ask();
#pragma unroll
  for (int n = 0; n < 4; ++n) {
#pragma unroll
    for (int t = 0; t < T; ++t) here(y[n][t]);
    if (MODE != PLAIN) turn[n].stay();
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (MODE != PLAIN) turn[n].apply(a, c0, e, y[n]);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[t][4 * n + j] = y[n][t][j];
  }
}

// Several new rows: a wave's tiles of them in registers in the order of the codes (so
// each lane ends with 16 adjacent bytes of every tile); the waves of a job
// exchange their largest magnitudes.  Blocks with older rows read their tiles and
// put them back whole.
template <int DT, int MODE>
__device__ __forceinline__ void append_rows(const AppendArgs& a, const Place& p, bool active,
                                            const int32_t* entry, int b, float* red,
                                            uint32_t (*turned)[256]) {
  constexpr int T = Share<DT>::kTiles;
  const KvView& v = a.v;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int c0 = wave % Share<DT>::kWaves * T;
  const bool older = p.lo > p.t0;
  active = active && c0 < DT;
  const int page = *entry;
  // The page's count, the scale and old tiles are asked for as soon as its number
  // is there, while the rows are on their way.
  const bool in_cache = page >= 0 && page < v.n_pages;
  uint4 old[T];
  float was = 0.0f;
  int sharers = 0;
  uint4* tiles = nullptr;
  float* scale = nullptr;
  auto ask = [&]() {
    const int at = in_cache ? page : 0, unit = (p.head * v.blocks + b) * 2 + p.is_v;
    tiles = (uint4*)(v.codes + at * v.page_codes + (int64_t)unit * DT * kKvTile);
    scale = v.scales + at * v.page_scales + unit;
    sharers = v.refs[at];
#pragma unroll
    for (int t = 0; t < T; ++t) old[t] = make_uint4(0u, 0u, 0u, 0u);
    if (older && active) {
      was = *scale;
#pragma unroll
      for (int t = 0; t < T; ++t)
        if (c0 + t < DT) old[t] = tiles[(c0 + t) * 64 + lane];
    }
  };
  // v: x[t][8 h + j] is the element whose code is byte 8 h + j of this lane's sixteen of
  // tile c0 + t.  k: x[t][4 n + j] is element e + j of token 8 n + u, so that eight lanes
  // read 128 bytes of a row and of the tables, and the codes change lanes through LDS.
  // (In the codes' order neighbouring lanes have different rows: 64 cache accesses a
  // load, which bound it: 5000 rows of 8 heads of 128, half-split pairs, took 55 us
  // and take 14.)
  // Rows that are not new: a new one's, not used.
  float x[T][16];
  float amax = 0.0f;
  const int e = 4 * (lane & 7), u = lane >> 3;
  if (!active) {
  } else if (!p.is_v) {
    if (a.k_vec)
      k_values<T, MODE, true>(a, p, c0, e, u, ask, x);
    else
      k_values<T, MODE, false>(a, p, c0, e, u, ask, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int pos = min(max(p.t0 + 16 * (j >> 2) + 4 * g + (j & 3), p.lo), p.len - 1);
      const float* row = a.vv + (int64_t)(p.row0 + pos - p.start) * a.v_stride + p.head * v.D;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[t][8 * h + j] = row[min(32 * (c0 + t) + 16 * h + i, v.D - 1)];
    }
    ask();
#pragma unroll
    for (int t = 0; t < T; ++t) here(x[t]);
  }
  if (active) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int c = 32 * (c0 + t);
      if (c + 32 > v.D) {  // elements behind D
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int d = c + (p.is_v ? 16 * (n >> 3) + i : e + (n & 3));
          x[t][n] = d < v.D ? x[t][n] : 0.0f;
        }
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) amax = vmax(amax, __builtin_fabsf(x[t][n]));
    }
  }
  amax = wave_amax(amax);
  if (Share<DT>::kWaves > 1) {
    if (lane == 0) red[wave] = amax;
    __syncthreads();
    const int w0 = wave / Share<DT>::kWaves * Share<DT>::kWaves;
#pragma unroll
    for (int w = 0; w < Share<DT>::kWaves; ++w) amax = vmax(amax, red[w0 + w]);
  }
  if (!active || !in_cache || sharers != 1) return;
  const Scale s(amax, was, older);
  // which bytes are new rows': k's lane has tokens i and 16 + i, v's 4 g + (0..3) and
  // 16 + those
  uint32_t mask[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mask[h] = 0;
#pragma unroll
    for (int b8 = 0; b8 < 4; ++b8) {
      const int pos = p.t0 + 16 * h + (p.is_v ? 4 * g + b8 : i);
      mask[h] |= pos >= p.lo && pos < p.len ? 0xFFu << (8 * b8) : 0u;
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    if (c0 + t >= DT) continue;
    const uint4 kept = s.grown ? requant16(old[t], s) : old[t];
    const uint32_t k4[4] = {kept.x, kept.y, kept.z, kept.w};
    uint32_t w[4];
    codes16(x[t], s, w);
    if (!p.is_v) {
      // w[n] is bytes e & 7 .. of token 8 n + u (the wave's own 1024 bytes)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        turned[wave][64 * (e >> 3) + 4 * ((8 * n + u) & 15) + 2 * (n >> 1) + ((e & 7) >> 2)] = w[n];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = turned[wave][4 * lane + q];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t m = p.is_v ? mask[q & 1] : mask[q >> 1];
      w[q] = (w[q] & m) | (k4[q] & ~m);
    }
    tiles[(c0 + t) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane == 0 && c0 == 0) *scale = s.now;
}

// The waves of a workgroup share a touched block's jobs (a kv head's k or v: its
// rows' largest magnitude, the scale, the codes); workgroups behind the blocks'
// rotate q rows.
//
// HBM bounds prompts (4 bytes read and 1 written an element); single tokens are
// three memory latencies: row_start with len, the row with the page number, the
// page's count and scale.  4870 prompt rows with 32 q heads and 8 kv heads of 64
// take 24 us (100 MB, 4.2 TB/s; 9.4 without q); 64 single tokens with 16 and 8 heads
// of 128 take 6 us; 872 rows of 32 and 32 heads of 80 take 14 us, two or three rounds
// of these latencies (40 MB, 9 us at a large copy's rate).
//
// A wave a tile, so that a job's loads are few and together: with whole jobs a wave
// the last of these took 1.4 times as long.
template <int DT, int MODE>
__global__ __launch_bounds__(kKvThreads, DT > 4 ? 2 : MODE == QWEN ? 5 : 6) void
kv8_append_kernel(AppendArgs a) {
  __shared__ float red[4];
  __shared__ __align__(16) uint32_t turned[4][256];
  const KvView& v = a.v;
  if (MODE != PLAIN && (int)blockIdx.x >= a.block_wgs) {
    const int wg = (int)blockIdx.x - a.block_wgs;
    const int group = (int)fdiv((uint32_t)wg, a.r.fd_chunk);
    const int item = (wg - group * a.r.chunks) * kRopeThreads + (int)threadIdx.x;
    const KvLanes lanes = kv_lanes(v);
    const int first = v.row_start[0];
    RopeItem it[kQRows];
#pragma unroll
    for (int n = 0; n < kQRows; ++n) {
      const int64_t row = (int64_t)group * a.q_rows + n;
      if (n < a.q_rows && row < v.n_rows && item < a.r.per_row)
        it[n] = rope_load<MODE == QWEN>(a.r, row, item);
    }
#pragma unroll
    for (int n = 0; n < kQRows; ++n) {
      const int64_t row = (int64_t)group * a.q_rows + n;
      if (n >= a.q_rows || row >= v.n_rows) continue;
      const int s = kv_find(v, lanes, [&](int, int next) { return next <= row; });
      if (s >= v.n_seqs || row < first) continue;
      const KvSeq q = kv_seq(v, lanes, s);
      const int pos = q.len - q.count + (int)row - q.row0;
      if (pos >= 0 && item < a.r.per_row) rope_store<MODE == QWEN>(a.r, it[n], pos);
    }
    return;
  }
  // everything but the job is the same for the workgroup
  const int slot = (int)fdiv(blockIdx.x, a.fd_groups);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int job = ((int)blockIdx.x - slot * a.groups) * Share<DT>::kJobs +
                  wave / Share<DT>::kWaves;
  const KvLanes lanes = kv_lanes(v);
  const KvBlock k = kv_block_of(v, lanes, slot);
  if (k.s < 0) return;
  Place p;
  p.row0 = k.q.row0, p.len = k.q.len;
  p.start = k.q.len - k.q.count;  // negative: rows before position 0 are dropped
  p.lo = max(p.start, 0);
  p.t0 = k.block * kKvBlock;
  const bool active = job < 2 * v.n_kv_heads;
  p.head = active ? job >> 1 : 0, p.is_v = job & 1;
  const int e = (int)fdiv((uint32_t)k.block, v.fd_blocks), b = k.block - e * v.blocks;
  const int32_t* entry = v.table + (size_t)k.s * v.max_pages + e;
  if (min(p.len, p.t0 + kKvBlock) - max(p.lo, p.t0) > 1) {
    append_rows<DT, MODE>(a, p, active, entry, b, red, turned);
    return;
  }
  if (!active || wave % Share<DT>::kWaves) return;
  const int page = *entry;
  const bool ok = page >= 0 && page < v.n_pages;
  const int at = ok ? page : 0, unit = (p.head * v.blocks + b) * 2 + p.is_v;
  append_row<DT, MODE>(a, p, (uint4*)(v.codes + at * v.page_codes + (int64_t)unit * DT * kKvTile),
                 v.scales + at * v.page_scales + unit, ok && v.refs[at] == 1);
}

struct FetchArgs {
  KvView v;
  float *k, *vv;
  int k_stride, v_stride, k_vec, v_vec;
  int groups;
  FastDiv fd_groups;
};

__device__ __forceinline__ float code_of(uint32_t w, int byte) {
  return (float)(int)(int8_t)(w >> (8 * byte));
}
// four elements of a row from d on, inside it
__device__ __forceinline__ void store_four(float* row, int d, int D, int vec, float4 y) {
  if (vec) {
    if (d < D) *(float4*)(row + d) = y;
  } else {
    if (d < D) row[d] = y.x;
    if (d + 1 < D) row[d + 1] = y.y;
    if (d + 2 < D) row[d + 2] = y.z;
    if (d + 3 < D) row[d + 3] = y.w;
  }
}

// A wave per block, kv head, k or v and tile; a lane's four words are chosen so that
// rows are written 128 bytes at a time by eight neighbouring lanes.  HBM (the 4-byte
// values written) bounds it, or for few rows the latencies of lengths, page, codes and
// stores: 2 K rows of 8 heads of 128 (17 MB written) take 8 us; with a whole head a
// wave it was 9.3.
template <int DT>
__global__ __launch_bounds__(kKvThreads) void kv8_fetch_kernel(FetchArgs a) {
  const KvView& v = a.v;
  const int slot = (int)fdiv(blockIdx.x, a.fd_groups);
  const int job = ((int)blockIdx.x - slot * a.groups) * 4 +
                  __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const KvLanes lanes = kv_lanes(v);
  const KvBlock kb = kv_block_of(v, lanes, slot, true);
  const int part = job / DT, c = job - part * DT;
  if (kb.s < 0 || part >= 2 * v.n_kv_heads) return;
  const int row0 = kb.q.row0, count = kb.q.count, len = kb.q.len;
  const int start = len - count, lo = max(start, 0);
  const int head = part >> 1, is_v = part & 1;
  const int lane = threadIdx.x & 63, D = v.D;
  float* dst = (is_v ? a.vv : a.k) + head * D;
  const int stride = is_v ? a.v_stride : a.k_stride, vec = is_v ? a.v_vec : a.k_vec;
  if (start < 0 && kb.first && c == 0) {  // rows before position 0
    for (int r = 0; r < min(-start, count); ++r)
      for (int d = lane; d < D; d += 64) dst[(int64_t)(row0 + r) * stride + d] = 0.0f;
  }
  const int blk = kb.block;
  if (blk * kKvBlock >= len) return;
  const int page = kv_page(v, kb.s, blk), src = page < 0 ? 0 : page;
  const int b = blk - (int)fdiv((uint32_t)blk, v.fd_blocks) * v.blocks;
  const int unit = (head * v.blocks + b) * 2 + is_v;
  const int8_t* tile = v.codes + src * v.page_codes + ((int64_t)unit * DT + c) * kKvTile;
  const float* sc = v.scales + src * v.page_scales + unit;
  const int t0 = blk * kKvBlock;
  // A lane's four words: of k elements d .. d + 3 of tokens t, t + 8, .., of v elements
  // d .. d + 3, each of tokens t .. t + 3.
  const int e = lane & 7, q = lane >> 3, d = 32 * c + 4 * e;
  uint32_t w[4];
  if (!is_v) {
    const int8_t* x = tile + 256 * (e >> 1) + 4 * (e & 1) + 16 * q;
#pragma unroll
    for (int n = 0; n < 4; ++n) w[n] = *(const uint32_t*)(x + 128 * (n & 1) + 8 * (n >> 1));
  } else {
    const int8_t* x = tile + 256 * (q & 3) + 16 * (4 * e & 15) + 8 * (e >> 2) + 4 * (q >> 2);
#pragma unroll
    for (int n = 0; n < 4; ++n) w[n] = *(const uint32_t*)(x + 16 * n);
  }
  const float s = page < 0 ? __builtin_nanf("") : *sc;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int t = t0 + (is_v ? 16 * (q >> 2) + 4 * (q & 3) + n : 8 * n + q);
    if (t < lo || t >= len) continue;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (is_v ? code_of(w[j], n) : code_of(w[n], j)) * s;
    store_four(dst + (int64_t)(row0 + t - start) * stride, d, D, vec,
               make_float4(y[0], y[1], y[2], y[3]));
  }
}

// Pointer and row stride of rows of n heads; strides cover the rows.
int check_rows(const char* what, const char* name, const void* p, int n_heads, int D, int stride) {
  if (!p || ((uintptr_t)p & 3)) {
    set_error("%s: %s is null or not aligned", what, name);
    return -1;
  }
  if ((int64_t)n_heads * D > stride) {
    set_error("%s: %s rows of %d heads of %d are %d floats apart", what, name, n_heads, D, stride);
    return -1;
  }
  return 0;
}

bool quads(const void* p, int stride, int D) {
  return (((uintptr_t)p | (uintptr_t)stride * 4 | (uintptr_t)D * 4) & 15) == 0;
}

template <int DT>
void launch_append(const AppendArgs& a, unsigned wgs) {
  const dim3 grid(wgs), block(kKvThreads);
  if (!a.rope)
    hipLaunchKernelGGL((kv8_append_kernel<DT, PLAIN>), grid, block, 0, ctx().stream, a);
  else if (a.r.qwen)
    hipLaunchKernelGGL((kv8_append_kernel<DT, QWEN>), grid, block, 0, ctx().stream, a);
  else
    hipLaunchKernelGGL((kv8_append_kernel<DT, LLAMA>), grid, block, 0, ctx().stream, a);
}
template <int DT>
void launch_fetch(const FetchArgs& a, unsigned wgs) {
  hipLaunchKernelGGL(kv8_fetch_kernel<DT>, dim3(wgs), dim3(kKvThreads), 0, ctx().stream, a);
}

}  // namespace
}  // namespace plh

using namespace plh;

#define PLH_KV_TILES(dt, fn, ...)                    \
  switch (dt) {                                      \
    case 1: fn<1>(__VA_ARGS__); break;               \
    case 2: fn<2>(__VA_ARGS__); break;               \
    case 3: fn<3>(__VA_ARGS__); break;               \
    case 4: fn<4>(__VA_ARGS__); break;               \
    case 5: fn<5>(__VA_ARGS__); break;               \
    case 6: fn<6>(__VA_ARGS__); break;               \
    case 7: fn<7>(__VA_ARGS__); break;               \
    default: fn<8>(__VA_ARGS__); break;              \
  }

extern "C" {

size_t plh_kv8_code_bytes(const plh_kv8_cache* c) {
  if (!c || c->n_layers < 1 || c->n_kv_heads < 1 || c->head_dim < 2 || c->head_dim > 256 ||
      (c->head_dim & 1) || c->n_pages < 1 || c->page_tokens < kKvBlock ||
      c->page_tokens % kKvBlock)
    return 0;
  const int64_t tiles = (int64_t)(c->page_tokens / kKvBlock) * 2 * kv_tiles(c->head_dim);
  const int64_t heads = (int64_t)c->n_layers * c->n_kv_heads;
  if (heads > INT_MAX || tiles > INT_MAX / kKvTile || heads * tiles > INT_MAX / kKvTile) return 0;
  return (size_t)(heads * tiles) * kKvTile * (size_t)c->n_pages;
}

size_t plh_kv8_scale_bytes(const plh_kv8_cache* c) {
  const size_t codes = plh_kv8_code_bytes(c);
  return codes ? codes / ((size_t)kv_tiles(c->head_dim) * kKvTile) * sizeof(float) : 0;
}

int plh_kv8_append(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, int layer, int n_rows,
                   const int32_t* row_start, const plh_rope* rope, const float* q, int n_heads,
                   int q_stride, float* q_out, int q_out_stride, const float* k, int k_stride,
                   const float* v, int v_stride) {
  const char* what = "plh_kv8_append";
  AppendArgs a{};
  if (kv_view(cache, seqs, layer, n_rows, row_start, what, a.v)) return -1;
  const int D = cache->head_dim, H = cache->n_kv_heads;
  if (n_heads < 0 || (n_heads && !rope)) {
    set_error("%s: %d q heads are rotated by tables only", what, n_heads);
    return -1;
  }
  if (rope && check_rope(rope, D, what)) return -1;
  if (n_rows && (check_rows(what, "k", k, H, D, k_stride) ||
                 check_rows(what, "v", v, H, D, v_stride) ||
                 (n_heads && (check_rows(what, "q", q, n_heads, D, q_stride) ||
                              check_rows(what, "q_out", q_out, n_heads, D, q_out_stride)))))
    return -1;
  if ((int64_t)n_heads * D > INT_MAX / 2) {
    set_error("%s: %d q heads are too many", what, n_heads);
    return -1;
  }
  a.k = k, a.vv = v, a.k_stride = k_stride, a.v_stride = v_stride;
  // (as Share<tiles>::kJobs)
  const int jobs = kv_tiles(D) == 1 ? 4 : kv_tiles(D) == 2 ? 2 : 1;
  a.groups = (2 * H + jobs - 1) / jobs;
  a.fd_groups = make_fastdiv((uint32_t)a.groups);
  a.k_vec = quads(k, k_stride, D);
  a.rope = rope != nullptr;
  int64_t wgs = kv_slots(n_rows, seqs->n_seqs) * a.groups;
  if (rope) {
    a.r = rope_rows_args(rope, D, q, n_heads, q_stride, q_out, q_out_stride, nullptr, 0, 0,
                         nullptr, 0);
    const bool tab16 = (((uintptr_t)rope->cos_tab | (uintptr_t)rope->sin_tab) & 15) == 0;
    a.k_vec = a.k_vec && tab16 && rope->rot_dim % 8 == 0;
  }
  a.block_wgs = (int)(wgs < INT_MAX ? wgs : INT_MAX);
  // Prompts: several rows' loads in flight a workgroup; while there are few rows,
  // each has its own.
  a.q_rows = n_rows >= 16 * ctx().num_cus ? kQRows : 1;
  if (n_heads) wgs += (int64_t)((n_rows + a.q_rows - 1) / a.q_rows) * a.r.chunks;
  if (wgs > kMaxWorkgroups) {
    set_error("%s: %d rows of %d sequences are too many for one call", what, n_rows, seqs->n_seqs);
    return -1;
  }
  if (kv_ready(what)) return -1;
  if (n_rows == 0) return 0;
  PLH_KV_TILES(kv_tiles(D), launch_append, a, (unsigned)wgs);
  return check_hip(hipGetLastError(), "kv8_append_kernel");
}

int plh_kv8_fetch(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, int layer, int n_rows,
                  const int32_t* row_start, float* k, int k_stride, float* v, int v_stride) {
  const char* what = "plh_kv8_fetch";
  FetchArgs a{};
  if (kv_view(cache, seqs, layer, n_rows, row_start, what, a.v)) return -1;
  const int D = cache->head_dim, H = cache->n_kv_heads;
  if (n_rows && (check_rows(what, "k", k, H, D, k_stride) ||
                 check_rows(what, "v", v, H, D, v_stride)))
    return -1;
  a.k = k, a.vv = v, a.k_stride = k_stride, a.v_stride = v_stride;
  a.k_vec = quads(k, k_stride, D), a.v_vec = quads(v, v_stride, D);
  a.groups = (2 * H * kv_tiles(D) + 3) / 4;
  a.fd_groups = make_fastdiv((uint32_t)a.groups);
  const int64_t wgs = kv_slots(n_rows, seqs->n_seqs) * a.groups;
  if (wgs > kMaxWorkgroups) {
    set_error("%s: %d rows of %d sequences are too many for one call", what, n_rows, seqs->n_seqs);
    return -1;
  }
  if (kv_ready(what)) return -1;
  if (n_rows == 0) return 0;
  PLH_KV_TILES(kv_tiles(D), launch_fetch, a, (unsigned)wgs);
  return check_hip(hipGetLastError(), "kv8_fetch_kernel");
}

}  // extern "C"
