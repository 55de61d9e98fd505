// kv8_attn.hip -- causal grouped-query attention over the paged 8-bit cache, for
// any mixture of single tokens and prompts in one launch (include/picolm_hip.h,
// plh_kv8_attn).
//
// Mathematics.  For a column (a row's q head) and the tokens t up to its
// position, with the block scales k_b, v_b of t's block and codes k_t, v_t:
//   s_t = k_b (q . k_t) / sqrt(D),   out = sum_t e^{s_t} v_b v_t / sum_t e^{s_t}
// in one pass over the blocks with the running maximum m (log2 units) and sum
// l of every column.  A block is one contraction step of both matrix products:
//   S^T[t][col] = k_t . q           codes times q (two fp16 parts)
//   O^T[d][col] += v_t[d] P[t][col] codes times weights (two fp16 parts)
// Codes are integers up to 127, exact in fp16, so the products are exact and
// sums are fp32.  k_b multiplies S with the score scale in the exponent's
// fused multiply-add.  v_b belongs into the weights but may be any fp32 number,
// so O has a unit of its own, 2^(m + dO) with a whole number dO per column, and a
// weight enters the second product times v_b 2^-dO (exact but for one rounding).
// Where that factor leaves [2^-4, 2^4), the unit moves to the largest
// s_t + log2 v_b so far: what is small beside the largest contribution is
// rounded, nothing else, whatever powers of two the v scales jump by.
//
// Layout.  A tile's bytes are in operand order (include/picolm_hip.h): lane
// 16 g + i of a wave loads 16 adjacent bytes, a tile of k serves two row blocks
// of S (tokens i and 16 + i), a tile of v two row blocks of O; the S
// accumulators of lane (g, col) are tokens 4 g + r and 16 + 4 g + r, which are the
// lane's contraction slots of the second product: no LDS, no transposition and
// no exchange between lanes but the maximum's.
//
// Work.  A unit is some columns of one (sequence, kv head).  Sequences of up to 32
// columns (single tokens) have units of 16, whose keys the four waves split; longer
// ones are cut into units of 64 CT columns, a wave taking 16 CT of them and all keys.
// Every workgroup finds its unit from row_start and len, so nothing
// is planned on the host and a captured graph follows the lengths.  Units are cut
// into chunks of blocks where there are few of them; the last workgroup of a unit
// to finish joins the chunks' partial results in their order.
// Three kernels, as their registers allow different numbers of waves: tokens only (SPLIT
// units), and mixtures whose waves take one or two tiles of columns.  Two tiles read
// the keys from LDS half as often (8 prompts of 1023 rows on 3000 tokens, 32 heads
// of 64 on 8: 551 us, one tile 607), one tile makes twice as many units (512 rows on
// 1000: 32 us, two tiles 40).  An exactly equal share of the work for every workgroup,
// units cut wherever that falls, was tried and lost: most units then have partial
// results (the 512 rows 57 us, the eight prompts 590).
//
// Measured: 64 tokens of 1000..8191 keys, 16 heads of 128 on 8: 86 us, 397 MB at
// 4.6 TB/s, a large copy's rate.  One token on 130001 keys, 32 heads of 64 on 8: 40
// us, of which 30 are the keys' bytes; the rest is the chain length, page, first
// keys, and at the end partial results, counter, join.  Three prompts of 1000..2047
// rows on 2000..4001 keys, 32 heads of 64 on 8: 174 us, 354 TFLOP/s counting a
// product once; each runs as two fp16 parts, and a large fp16 product reaches 1215.
#include <limits.h>
#include <math.h>

#include "attn_common.h"
#include "kv8.h"

namespace plh {
namespace {

constexpr int kDevScope = 16;      // buffer cache policy sc1: past the XCD's L2
constexpr float kPlainMax = 65536.0f;  // log2 units: larger running maxima take exact steps
// Weights (up to 2^8) times a v scale in units of 2^dO: exponents that leave both
// fp16 parts their bits.
constexpr int kUnitLo = -4, kUnitHi = 3;
constexpr int kMinChunk = 16;      // blocks (a SHARE unit: for each of a wave's tiles, as its
                                   // partial results grow with them)
constexpr int kMaxTarget = 2048;   // most chunks asked for of the units that are cut

// Arrival counters of cut units, zero between launches.
__device__ unsigned g_kv8_ctr[3 * kMaxTarget];

struct AttnArgs {
  KvView v;
  const float* q;
  float* out;
  int q_stride, out_stride;
  int G;               // q heads of a kv head
  int target;          // chunks aimed at
  float per_target;    // 1 / target, rounded up
  float score_scale;   // log2(e) / sqrt(D)
  float* part;         // [slot][part_cols][Dp + 2]
  int part_cols;
  int q_vec, out_vec;
  FastDiv fd_g, fd_kvh;
};

// 32 codes of four lanes' words: bytes -> fp16.  A byte c + 128 in the low
// bits of 0x6400 is the fp16 number 1024 + 128 + c, and subtracting 1152 is exact.
__device__ __forceinline__ half8_t codes_to_half(uint32_t w0, uint32_t w1) {
  const uint32_t a = w0 ^ 0x80808080u, b = w1 ^ 0x80808080u;
  const uint32_t k = 0x64646464u;
  const half2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const half2_t p0 = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(k, a, 0x04010400u)) + off;
  const half2_t p1 = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(k, a, 0x04030402u)) + off;
  const half2_t p2 = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(k, b, 0x04010400u)) + off;
  const half2_t p3 = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(k, b, 0x04030402u)) + off;
  return half8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// Weights as fp16 hi (rounded toward zero) and lo = x - hi (exact, then rounded).
__device__ __forceinline__ void split8(const float (&p)[8], half8_t& ph, half8_t& pl) {
#pragma unroll
  for (int r = 0; r < 8; r += 2) {
    const uint32_t h =
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p[r], p[r + 1]));
    // x - hi by a mixed-precision FMA into a whole register.  (Its 16-bit forms
    // would save one instruction, but write half a register, and a matrix
    // instruction that follows too closely reads the other value; the compiler
    // does not count wait states of asm.)
    float d0, d1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d0) : "v"(h), "v"(p[r]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(d1)
        : "v"(h), "v"(p[r + 1]));
    const half2_t hi = __builtin_bit_cast(half2_t, h);
    const half2_t lo = {(_Float16)d0, (_Float16)d1};
    ph[r] = hi[0], ph[r + 1] = hi[1];
    pl[r] = lo[0], pl[r + 1] = lo[1];
  }
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a workgroup works on.
struct Unit {
  int s;             // sequence, or -1
  int row0, rows;    // its rows
  int len, form;
  int kvh, col0;     // first column (token * G + head of the group)
  int chunk, chunks;
  int slot;          // of the unit's first chunk among the cut units' partials
};

struct PlanLds {
  int64_t part[kKvThreads / 64];
  float work[kKvThreads / 64];
  int found[6];
};

__device__ __forceinline__ float wave_sums(float x) {
  auto f = [](int i) { return __uint_as_float((uint32_t)i); };
  x += f(kv_dpp<0x111, 0xF>((int)__float_as_uint(x)));
  x += f(kv_dpp<0x112, 0xF>((int)__float_as_uint(x)));
  x += f(kv_dpp<0x114, 0xF>((int)__float_as_uint(x)));
  x += f(kv_dpp<0x118, 0xF>((int)__float_as_uint(x)));
  x += f(kv_dpp<0x142, 0xA>((int)__float_as_uint(x)));
  x += f(kv_dpp<0x143, 0xC>((int)__float_as_uint(x)));
  return x;
}

// Sum over the earlier threads of the workgroup and over all of them.
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t sum = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(sum, o, 64);
    if (lane >= o) sum += y;
  }
  __syncthreads();
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kKvThreads / 64; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + sum - x;
}

// How a sequence's columns are cut: for waves that split the keys of one tile of 16
// columns, or for waves that share them.  A launch of short sequences has no
// other form than SPLIT.
enum { SPLIT = 1, SHARE = 4 };
template <bool MIXED>
__device__ __forceinline__ int form_of(int64_t cols) {
  return !MIXED || cols <= 32 ? SPLIT : SHARE;
}
template <int CT>
__device__ __forceinline__ int unit_cols(int form) {
  return form == SPLIT ? 16 : 64 * CT;
}
__device__ __forceinline__ int blocks_of(int len) { return (len + kKvBlock - 1) / kKvBlock; }

// A unit's work in wave-blocks: a block of a SHARE unit is work for all four waves.
__device__ __forceinline__ float work_of(int units, int len, int form) {
  return (float)units * (float)(blocks_of(len) * (form == SHARE ? 4 : 1));
}
// Work of a chunk: all units' over the target (rounded up, the sum's roundings
// included), so that no more than target chunks come of it.
__device__ __forceinline__ int quota_of(const AttnArgs& a, float work) {
  const float q = work * (float)a.v.n_kv_heads * a.per_target * 1.0001f + 1.0f;
  return (int)fminf(q, 1e9f);
}
// Chunks of a sequence's units: a quota of work each, at least kMinChunk blocks.
template <int CT>
__device__ __forceinline__ int chunks_of(int len, int form, int quota) {
  const int c = form == SHARE ? max(kMinChunk * CT, quota / 4) : max(kMinChunk, quota);
  const int n = blocks_of(len);
  return c >= n ? 1 : (int)(((uint32_t)n + (uint32_t)c - 1) / (uint32_t)c);
}

// The local-th of a sequence's workgroups: units (those of the longest contexts
// first), kv heads, chunks.
template <int CT>
__device__ __forceinline__ void place_unit(const AttnArgs& a, Unit& u, int local, int slot) {
  const int unit_kvh = u.chunks == 1 ? local : (int)((uint32_t)local / (uint32_t)u.chunks);
  u.chunk = local - unit_kvh * u.chunks;
  const int unit = (int)fdiv((uint32_t)unit_kvh, a.fd_kvh);
  u.kvh = unit_kvh - unit * a.v.n_kv_heads;
  const int64_t cols = (int64_t)u.rows * a.G;
  const int uc = unit_cols<CT>(u.form), units = (int)((cols + uc - 1) / uc);
  u.col0 = (units - 1 - unit) * uc;
  u.slot = slot + unit_kvh * u.chunks;
}

// Workgroup `wg`'s unit.  The quota is all units' work over the target, so at most
// target + units workgroups have work.  A unit that is cut has more blocks than a
// chunk and so fewer than twice as many chunks as quotas of work; rounding a SHARE
// unit's quota down to blocks (16 and more) adds a sixteenth: cut units' chunks are
// below 3 target.
template <int CT, bool MIXED>
__device__ __forceinline__ Unit find_unit(const AttnArgs& a, int wg, PlanLds& lds) {
  const KvView& v = a.v;
  Unit u{};
  u.s = -1;
  if (v.n_seqs == 1) {
    kv_rows(v, 0, u.row0, u.rows);
    u.len = kv_len(v, 0);
    const int64_t cols = (int64_t)u.rows * a.G;
    u.form = form_of<MIXED>(cols);
    const int uc = unit_cols<CT>(u.form), units = (int)((cols + uc - 1) / uc);
    u.chunks = uniform(chunks_of<CT>(u.len, u.form, quota_of(a, work_of(units, u.len, u.form))));
    if (wg >= (int64_t)units * u.chunks * v.n_kv_heads) return u;
    u.s = 0;
    place_unit<CT>(a, u, wg, 0);
    return u;
  }
  if (v.n_seqs <= 64) {  // a lane a sequence, every wave for itself
    const int lane = (int)threadIdx.x & 63;
    int row0 = 0, rows = 0, len = 0;
    if (lane < v.n_seqs) {
      kv_rows(v, lane, row0, rows);
      len = kv_len(v, lane);
    }
    const int64_t cols = (int64_t)rows * a.G;
    const int form = form_of<MIXED>(cols), uc = unit_cols<CT>(form);
    const int units = (int)((cols + uc - 1) / uc);
    const float work = wave_sums(work_of(units, len, form));
    const int quota = quota_of(a, __uint_as_float((uint32_t)__builtin_amdgcn_readlane(
                                      (int)__float_as_uint(work), 63)));
    const int n_chunks = chunks_of<CT>(len, form, quota);
    // (more than the grid: as good as one more, and 64 of them no overflow)
    const int64_t all = (int64_t)units * n_chunks * v.n_kv_heads;
    const int n_wgs = all > kMaxWorkgroups ? kMaxWorkgroups + 1 : (int)all;
    const int end = wave_sums(n_wgs), at = end - n_wgs;
    const int cut = n_chunks > 1 ? n_wgs : 0, slot = wave_sums(cut) - cut;
    // row_start that does not rise: more units than rows; no chunk may be left out
    // of a cut unit
    if (__builtin_amdgcn_readlane(end, 63) > (int)gridDim.x) return u;
    const uint64_t hit = __ballot(wg >= at && wg < end);
    if (hit == 0) return u;
    const int l = __ffsll((unsigned long long)hit) - 1;
    u.s = l;
    u.chunks = __builtin_amdgcn_readlane(n_chunks, l);
    u.row0 = __builtin_amdgcn_readlane(row0, l);
    u.rows = __builtin_amdgcn_readlane(rows, l);
    u.len = __builtin_amdgcn_readlane(len, l);
    u.form = __builtin_amdgcn_readlane(form, l);
    place_unit<CT>(a, u, wg - __builtin_amdgcn_readlane(at, l),
                   __builtin_amdgcn_readlane(slot, l));
    return u;
  }
  // four sequences a thread at most
  const int per = (v.n_seqs + kKvThreads - 1) / kKvThreads;
  const int s0 = (int)threadIdx.x * per;
  int row0[4], rows[4], len[4], form[4], units[4];
  float work = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    row0[k] = rows[k] = len[k] = 0;
    if (k < per && s0 + k < v.n_seqs) {
      kv_rows(v, s0 + k, row0[k], rows[k]);
      len[k] = kv_len(v, s0 + k);
    }
    const int64_t cols = (int64_t)rows[k] * a.G;
    form[k] = form_of<MIXED>(cols);
    const int uc = unit_cols<CT>(form[k]);
    units[k] = (int)((cols + uc - 1) / uc);
    work += work_of(units[k], len[k], form[k]);
  }
  work = wave_sums(work);
  if ((threadIdx.x & 63) == 63) lds.work[threadIdx.x >> 6] = work;
  __syncthreads();
  const int quota = quota_of(a, (lds.work[0] + lds.work[1]) + (lds.work[2] + lds.work[3]));
  // workgroups and cut chunks (below 2^16) of each thread's sequences
  int64_t wgs = 0, cut = 0;
  int n_wgs[4], n_chunks[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    n_chunks[k] = chunks_of<CT>(len[k], form[k], quota);
    n_wgs[k] = units[k] * n_chunks[k] * v.n_kv_heads;
    wgs += n_wgs[k];
    cut += n_chunks[k] > 1 ? n_wgs[k] : 0;
  }
  int64_t total;
  const int64_t before = plan_scan(cut << 48 | wgs, lds.part, total);
  constexpr int64_t kLow = (1ll << 48) - 1;
  if ((total & kLow) > (int64_t)gridDim.x) return u;
  int at = (int)(before & kLow), slot = (int)(before >> 48);
  if (threadIdx.x == 0) lds.found[0] = -1;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (wg >= at && wg < at + n_wgs[k]) {
      lds.found[0] = s0 + k, lds.found[1] = wg - at, lds.found[2] = n_chunks[k];
      lds.found[3] = slot, lds.found[4] = row0[k], lds.found[5] = rows[k];
    }
    at += n_wgs[k];
    slot += n_chunks[k] > 1 ? n_wgs[k] : 0;
  }
  __syncthreads();
  if (lds.found[0] < 0) return u;
  u.s = uniform(lds.found[0]);
  u.chunks = uniform(lds.found[2]);
  u.row0 = uniform(lds.found[4]), u.rows = uniform(lds.found[5]);
  u.len = uniform(kv_len(v, u.s));
  u.form = form_of<MIXED>((int64_t)u.rows * a.G);
  place_unit<CT>(a, u, uniform(lds.found[1]), uniform(lds.found[3]));
  return u;
}

// A wave's columns: 16 CT of them, lane (g, i) holding its share of columns 16 ct + i.
template <int DT, int CT>
struct Columns {
  half8_t qh[CT][DT], ql[CT][DT];  // q in two parts, B operand order
  float4_t o[CT][2 * DT];          // O^T: elements 16 j + 4 g + r
  float f0[CT];                    // score scale (q's power of two in it)
  float m[CT], l[CT];
  int dO[CT];     // O is in units of 2^(m + dO)
  float thr[CT];  // a lane's scores up to here need no step but the plain one
  int lim[CT];    // position (no column: sees all, is not stored)
  bool far;       // some column's scores or unit need the careful weights
  int d_lo, d_hi; // smallest and largest dO
  int top, low;   // last and first position

  // c0: the first column's number in the unit
  __device__ __forceinline__ void load(const AttnArgs& a, const Unit& u, int c0, int live) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int G = a.G, D = a.v.D, base = u.len - u.rows;
    top = -1, low = INT_MAX;
    far = true, d_lo = d_hi = 0;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = c0 + ct * 16 + i;
      const bool on = c < live;
      const int col = u.col0 + (on ? c : 0);
      const int t = (int)fdiv((uint32_t)col, a.fd_g);
      const int head = u.kvh * G + col - t * G;
      const float* qr = a.q + (int64_t)(u.row0 + t) * a.q_stride + (int64_t)head * D;
      lim[ct] = on ? base + t : INT_MAX;
      float x[DT][8];
      float amax = 0.0f;
#pragma unroll
      for (int c8 = 0; c8 < DT; ++c8) {
        const int d = 32 * c8 + 8 * g;
        if (a.q_vec) {
          const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
          const float4 lo = on && d < D ? *(const float4*)(qr + d) : z;
          const float4 hi = on && d + 4 < D ? *(const float4*)(qr + d + 4) : z;
          x[c8][0] = lo.x, x[c8][1] = lo.y, x[c8][2] = lo.z, x[c8][3] = lo.w;
          x[c8][4] = hi.x, x[c8][5] = hi.y, x[c8][6] = hi.z, x[c8][7] = hi.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[c8][j] = on && d + j < D ? qr[d + j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = vmax(amax, __builtin_fabsf(x[c8][j]));
      }
      amax = max_xor32(max_xor16(amax));
      // q times 2^-e with the largest element in [2^10, 2^11): its two fp16 parts
      // keep 22 bits of elements down to 2^-13 of it, and 2^-35 of it below
      int e = (int)((__float_as_uint(amax) >> 23) & 0xFFu) - 127 - 10;
      e = min(max(e, -126), 117);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      f0[ct] = a.score_scale * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int c8 = 0; c8 < DT; ++c8)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          _Float16 h, lo;
          split_hi_lo(x[c8][j] * down, h, lo);
          qh[ct][c8][j] = h, ql[ct][c8][j] = lo;
        }
      top = max(top, on ? lim[ct] : -1);
      low = min(low, lim[ct]);
      m[ct] = kNegBig, l[ct] = 0.0f, dO[ct] = 0, thr[ct] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2 * DT; ++j) o[ct][j] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int o_ = 1; o_ < 16; o_ <<= 1) {
      top = max(top, __shfl_xor(top, o_, 64));
      low = min(low, __shfl_xor(low, o_, 64));
    }
    top = uniform(top), low = uniform(low);
  }

  // One block: tokens t0.., scales ks and vs; k(c, h) and v(c, h) are the fp16
  // operands of row half h of tile c.
  template <class K, class V>
  __device__ __forceinline__ void step(int t0, float ks, float vs, K k, V v) {
    const int g = (threadIdx.x & 63) >> 4;
    float4_t s0[CT], s1[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) s0[ct] = s1[ct] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      const half8_t k0 = k(c, 0), k1 = k(c, 1);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        s0[ct] = mfma16x16x32(k0, ql[ct][c], s0[ct]);
        s1[ct] = mfma16x16x32(k1, ql[ct][c], s1[ct]);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        s0[ct] = mfma16x16x32(k0, qh[ct][c], s0[ct]);
        s1[ct] = mfma16x16x32(k1, qh[ct][c], s1[ct]);
      }
    }
    // exponent of the v scale (of 0: any; NaN, inf: past all units)
    const float up = vs < 0x1p-100f ? vs * 0x1p64f : vs;
    const int ve = uniform((int)(__float_as_uint(up) >> 23) -
                           (vs < 0x1p-100f ? 127 + 64 : 127));
    const bool seen_whole = t0 + kKvBlock - 1 <= low;
    // The plain step: the v scale fits every column's unit and no lane has a score
    // above its column's threshold (which a column's lanes need not exchange).  One
    // vote for all columns.
    float f[CT];
    float above = -INFINITY;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f[ct] = f0[ct] * ks;
      const float top8 = vmax(vmax(vmax(s0[ct][0], s0[ct][1]), vmax(s0[ct][2], s0[ct][3])),
                              vmax(vmax(s1[ct][0], s1[ct][1]), vmax(s1[ct][2], s1[ct][3])));
      above = vmax(above, __builtin_fmaf(top8, f[ct], -thr[ct]));
    }
    const bool unit_fits = (ve - d_hi >= kUnitLo && ve - d_lo <= kUnitHi) ||
                           __builtin_amdgcn_readfirstlane(vs == 0.0f);
    if (!seen_whole || !unit_fits || !__all(above <= 0.0f)) {
      far = false, d_lo = INT_MAX, d_hi = INT_MIN;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) adapt(ct, s0[ct], s1[ct], f[ct], t0, ve, vs);
#pragma unroll
      for (int o_ = 1; o_ < 16; o_ <<= 1) {  // the lanes of a column agree
        d_lo = min(d_lo, __shfl_xor(d_lo, o_, 64));
        d_hi = max(d_hi, __shfl_xor(d_hi, o_, 64));
      }
      d_lo = uniform(d_lo), d_hi = uniform(d_hi);
    }
    half8_t ph[CT], pl[CT];
    if (seen_whole && !far) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float p[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = fast_exp2(__builtin_fmaf(s0[ct][r], f[ct], -m[ct]));
          p[4 + r] = fast_exp2(__builtin_fmaf(s1[ct][r], f[ct], -m[ct]));
        }
        l[ct] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        const float ratio = __builtin_ldexpf(vs, -dO[ct]);
#pragma unroll
        for (int r = 0; r < 8; ++r) p[r] *= ratio;
        split8(p, ph[ct], pl[ct]);
      }
    } else {
      const float lv = __builtin_amdgcn_logf(up) - (vs < 0x1p-100f ? 64.0f : 0.0f);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        // Scores so large that their rounding tells: the rounded product, which m is
        // the largest of.  v scales far from the unit: one exponential for both.
        const bool large = !(__builtin_fabsf(m[ct]) <= kPlainMax);
        const bool apart = vs > 0.0f && !(abs(ve - dO[ct]) <= 60);
        const float ratio = __builtin_ldexpf(vs, -dO[ct]);
        const int seen = lim[ct] - t0 - 4 * g;  // tokens r and 16 + r up to here
        float p[8], w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float s = r < 4 ? s0[ct][r & 3] : s1[ct][r & 3];
          const float t = large ? s * f[ct] - m[ct] : __builtin_fmaf(s, f[ct], -m[ct]);
          const bool see = (r & 3) + (r >> 2) * 16 <= seen;
          w[r] = see ? fast_exp2(t) : 0.0f;
          p[r] = see ? (apart ? fast_exp2(t + (lv - (float)dO[ct])) : w[r] * ratio) : 0.0f;
        }
        l[ct] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        split8(p, ph[ct], pl[ct]);
      }
    }
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      const half8_t v0 = v(c, 0), v1 = v(c, 1);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][2 * c] = mfma16x16x32(v0, pl[ct], o[ct][2 * c]);
        o[ct][2 * c + 1] = mfma16x16x32(v1, pl[ct], o[ct][2 * c + 1]);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][2 * c] = mfma16x16x32(v0, ph[ct], o[ct][2 * c]);
        o[ct][2 * c + 1] = mfma16x16x32(v1, ph[ct], o[ct][2 * c + 1]);
      }
    }
  }

  // m, l and O follow a block's scores and v scale, each column by itself, so that
  // no other column's values reach its result, not even its last bits: m where the
  // largest score is more than 2^8 above it; O's unit where the v scale does not fit
  // it, to the largest score + log2(v scale) so far.
  __device__ __forceinline__ void adapt(int ct, float4_t s0, float4_t s1, float f, int t0, int ve,
                                        float vs) {
    const int seen = lim[ct] - t0 - 4 * (int)((threadIdx.x & 63) >> 4);
    float mt = kNegBig;  // NaN scores go into the weights, not the maximum
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r <= seen) mt = fmaxf(mt, s0[r] * f);
      if (16 + r <= seen) mt = fmaxf(mt, s1[r] * f);
    }
    mt = max_xor32(max_xor16(mt));
    const float to = mt > m[ct] + 8.0f ? mt : m[ct];
    int dn = dO[ct];
    if (!(m[ct] > kNegBig)) {
      // nothing seen yet: the block's own unit
      if (vs > 0.0f && vs < INFINITY) dn = ve + 1;
    } else if ((ve - dn < kUnitLo || ve - dn > kUnitHi) && vs > 0.0f && vs < INFINITY &&
               mt > kNegBig) {
      // relative to m first: where neither changes the unit stays, not one up by a
      // rounding
      const float most = fmaxf((float)dn + (m[ct] - to), (float)(ve + 1) + (mt - to));
      dn = (int)__builtin_ceilf(fmaxf(most, -400.0f));
    }
    const float shrink = fast_exp2(m[ct] - to);
    const float turn = fast_exp2((m[ct] - to) + (float)(dO[ct] - dn));
    l[ct] *= shrink;
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j) o[ct][j] = o[ct][j] * turn;
    m[ct] = to, dO[ct] = dn;
    d_lo = min(d_lo, dn), d_hi = max(d_hi, dn);
    const bool large = !(__builtin_fabsf(to) <= kPlainMax);
    thr[ct] = large ? -INFINITY : to + 8.0f;
    far = far || __any(large || (vs > 0.0f && !(abs(ve - dn) <= 60)));
  }

  // l over the lanes of a column, O in values
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      l[ct] = add_xor32(add_xor16(l[ct]));
#pragma unroll
      for (int j = 0; j < 2 * DT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[ct][j][r] = __builtin_ldexpf(o[ct][j][r], dO[ct]);
    }
  }
};

// Where a unit's chunk and its blocks lie.
struct Walk {
  int live;          // columns
  int b_lo, b_hi;    // blocks of the chunk
  const int32_t* row;
  int64_t head_off;  // tile pairs before the kv head's in a page

  template <int CT>
  __device__ __forceinline__ void start(const AttnArgs& a, const Unit& u) {
    const KvView& v = a.v;
    live = min(unit_cols<CT>(u.form), u.rows * a.G - u.col0);
    const int top = u.len - u.rows + (int)fdiv((uint32_t)(u.col0 + live - 1), a.fd_g);
    const int nb = top < 0 ? 0 : top / kKvBlock + 1;
    const int per = u.chunks == 1 ? nb : (int)(((uint32_t)nb + (uint32_t)u.chunks - 1) /
                                               (uint32_t)u.chunks);
    b_lo = min(nb, per * u.chunk);
    b_hi = min(nb, b_lo + per);
    row = v.table + (size_t)u.s * v.max_pages;
    head_off = (int64_t)u.kvh * v.blocks * 2;
  }
};

// A block's tiles (k's, then v's) and scales.  A page outside the cache stands for
// page 0 with NaN scales.
struct Block {
  const uint4* tiles;
  float sc[2];
  bool ok;
  __device__ __forceinline__ float scale(int i) const {
    return ok ? sc[i] : __builtin_nanf("");
  }
};
__device__ __forceinline__ int page_entry(const KvView& v, const Walk& w, int b) {
  return w.row[fdiv((uint32_t)b, v.fd_blocks)];
}
template <int DT>
__device__ __forceinline__ Block locate(const KvView& v, const Walk& w, int b, int page) {
  Block at;
  int p = uniform(page);
  at.ok = p >= 0 && p < v.n_pages;
  p = at.ok ? p : 0;
  const int in = b - (int)fdiv((uint32_t)b, v.fd_blocks) * v.blocks;
  const int64_t unit = w.head_off + in * 2;
  at.tiles = (const uint4*)(v.codes + p * v.page_codes + unit * DT * kKvTile);
  const float* s = v.scales + p * v.page_scales + unit;
  at.sc[0] = s[0], at.sc[1] = s[1];
  return at;
}

template <int DT>
struct Sizes {
  static constexpr int DP = 32 * DT;
  static constexpr int kRow = DP + 2;       // floats of a partial column
  static constexpr int kMergeRow = DP + 4;  // LDS pitch of a column's O, m, l
};

// Results of a unit's columns: to out, or as a chunk's partial ones.
template <int DT>
struct Results {
  using Sz = Sizes<DT>;
  const AttnArgs& a;
  const Unit& u;
  int live;  // columns of the unit

  __device__ __forceinline__ float* out_row(int c) const {
    const int col = u.col0 + c, t = (int)fdiv((uint32_t)col, a.fd_g);
    return a.out + (int64_t)(u.row0 + t) * a.out_stride +
           (int64_t)(u.kvh * a.G + col - t * a.G) * a.v.D;
  }
  __device__ __forceinline__ void store4(float* y, int d, float4_t x) const {
    if (a.out_vec) {
      if (d < a.v.D) *(float4_t*)(y + d) = x;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.v.D) y[d + e] = x[e];
    }
  }
  __device__ __forceinline__ float* unit_part() const {
    return a.part + (int64_t)u.slot * a.part_cols * Sz::kRow;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_part(int n) const {
    return __builtin_amdgcn_make_buffer_rsrc(unit_part() + (int64_t)n * a.part_cols * Sz::kRow, 0,
                                             a.part_cols * Sz::kRow * 4, 0x00020000);
  }
  __device__ __forceinline__ int ml_at(int c) const {
    return (a.part_cols * Sz::DP + 2 * c) * 4;
  }
  __device__ __forceinline__ float load_ml(__amdgpu_buffer_rsrc_t prs, int c, int which) const {
    return __uint_as_float(
        __builtin_amdgcn_raw_buffer_load_b32(prs, ml_at(c) + 4 * which, 0, kDevScope));
  }

  // columns c0 + 16 ct + i of one wave.  Partials (O, m and l) are written past
  // the L2, so that the workgroup that joins them may run on another XCD.
  template <int CT>
  __device__ __forceinline__ void put(const Columns<DT, CT>& w, int c0) const {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const __amdgpu_buffer_rsrc_t prs = chunk_part(u.chunk);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = c0 + ct * 16 + i;
      if (c >= live) continue;
      if (u.chunks == 1) {
        float* y = out_row(c);
        const float inv = w.l[ct] == 0.0f ? 0.0f : 1.0f / w.l[ct];
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) store4(y, 16 * j + 4 * g, w.o[ct][j] * inv);
      } else {
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j)
          __builtin_amdgcn_raw_buffer_store_b128(w.o[ct][j], prs,
                                                 (c * Sz::DP + 16 * j + 4 * g) * 4, 0, kDevScope);
        if (g == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w.m[ct]), prs, ml_at(c), 0,
                                                kDevScope);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w.l[ct]), prs, ml_at(c) + 4, 0,
                                                kDevScope);
        }
      }
    }
  }

  // After every wave's put of a cut unit: its last chunk to finish joins them.
  // lds: 6 kKvThreads floats.
  __device__ __forceinline__ void join(float* merge, int& s_last) const {
    __builtin_amdgcn_s_waitcnt(0);  // the partials have arrived before the count goes up
    __syncthreads();
    unsigned* ctr = g_kv8_ctr + u.slot;
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               (unsigned)(u.chunks - 1);
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int items = live * (Sz::DP / 4);  // four elements of a column each
    if (items > 2 * kKvThreads)
      join_wide(merge, items);
    else
      join_long(merge, items);
  }

  // Few elements, many chunks: each thread every ng-th chunk of its elements where
  // there are fewer elements than threads, eight loads ahead; the shares are
  // joined through LDS.
  __device__ __forceinline__ void join_long(float* merge, int items) const {
    const int ng = items <= 64 ? 4 : items <= 128 ? 2 : 1, span = kKvThreads / ng;
    const int share = (int)threadIdx.x / span;
    for (int idx = (int)threadIdx.x - share * span; idx < items; idx += span) {
      const int c = idx / (Sz::DP / 4), d = 4 * (idx - c * (Sz::DP / 4));
      float M = kNegBig, L = 0.0f;
      float4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int n0 = share; n0 < u.chunks; n0 += 8 * ng) {
        float4_t on[8];
        float mn[8], ln[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int n = min(n0 + k * ng, u.chunks - 1);  // past the last: again, not used
          const __amdgpu_buffer_rsrc_t prs = chunk_part(n);
          on[k] = __builtin_amdgcn_raw_buffer_load_b128(prs, (c * Sz::DP + d) * 4, 0, kDevScope);
          mn[k] = load_ml(prs, c, 0);
          ln[k] = load_ml(prs, c, 1);
        }
        float Mn = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) Mn = fmaxf(Mn, mn[k]);
        const float r = fast_exp2(M - Mn);
        L *= r;
        O = O * r;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n0 + k * ng < u.chunks) {
            const float w = fast_exp2(mn[k] - Mn);
            L += ln[k] * w;
            O = O + on[k] * w;
          }
        M = Mn;
      }
      if (ng > 1) {  // one pass of the loop
        float* x = merge + (share * span + idx) * 6;
        *(float2*)x = make_float2(O[0], O[1]), *(float2*)(x + 2) = make_float2(O[2], O[3]);
        *(float2*)(x + 4) = make_float2(M, L);
      } else {
        store4(out_row(c), d, O * (L == 0.0f ? 0.0f : 1.0f / L));
      }
    }
    if (ng == 1) return;
    __syncthreads();
    const int idx = (int)threadIdx.x;
    if (idx >= items) return;
    float M = kNegBig, L = 0.0f;
    float4_t O = {0.f, 0.f, 0.f, 0.f};
    for (int n = 0; n < ng; ++n) M = fmaxf(M, merge[(n * span + idx) * 6 + 4]);
    for (int n = 0; n < ng; ++n) {
      const float* x = merge + (n * span + idx) * 6;
      const float w = fast_exp2(x[4] - M);
      L += x[5] * w;
      O = O + float4_t{x[0], x[1], x[2], x[3]} * w;
    }
    const int c = idx / (Sz::DP / 4), d = 4 * (idx - c * (Sz::DP / 4));
    store4(out_row(c), d, O * (L == 0.0f ? 0.0f : 1.0f / L));
  }

  // Many elements: a thread per column finds its maximum and sum, then each
  // thread adds four elements' chunks two at a time, eight loads ahead.
  __device__ __forceinline__ void join_wide(float* merge, int items) const {
    if ((int)threadIdx.x < live) {
      const int c = (int)threadIdx.x;
      float M = kNegBig, L = 0.0f;
#pragma unroll 4
      for (int n = 0; n < u.chunks; ++n) {
        const __amdgpu_buffer_rsrc_t prs = chunk_part(n);
        const float mn = load_ml(prs, c, 0), ln = load_ml(prs, c, 1), Mn = fmaxf(M, mn);
        L = L * fast_exp2(M - Mn) + ln * fast_exp2(mn - Mn);
        M = Mn;
      }
      merge[2 * c] = M, merge[2 * c + 1] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    __syncthreads();
    for (int i0 = (int)threadIdx.x; i0 < items; i0 += 4 * kKvThreads) {
      float4_t O[4];
      int c[4], d[4];
      float M[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int idx = min(i0 + k * kKvThreads, items - 1);  // past the last: not stored
        c[k] = idx / (Sz::DP / 4), d[k] = 4 * (idx - c[k] * (Sz::DP / 4));
        M[k] = merge[2 * c[k]];
        O[k] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll 2
      for (int n = 0; n < u.chunks; ++n) {
        const __amdgpu_buffer_rsrc_t prs = chunk_part(n);
        float4_t x[4];
        float m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = __builtin_amdgcn_raw_buffer_load_b128(prs, (c[k] * Sz::DP + d[k]) * 4, 0,
                                                       kDevScope);
          m[k] = load_ml(prs, c[k], 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) O[k] = O[k] + x[k] * fast_exp2(m[k] - M[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * kKvThreads < items) store4(out_row(c[k]), d[k], O[k] * merge[2 * c[k] + 1]);
    }
  }
};

// Four waves take every fourth block of a chunk each, for the same columns, and
// are merged through LDS.
//
// HBM bounds it (a block is read once): a block's loads are in flight while the one
// before is worked on, its page number one more block ahead.
template <int DT>
__device__ __forceinline__ void attend_split(const AttnArgs& a, const Unit& u, float* merge,
                                             int& s_last) {
  using Sz = Sizes<DT>;
  const KvView& v = a.v;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  Walk w;
  w.start<1>(a, u);
  const int b_end = w.b_hi;
  uint4 kt[DT], vt[DT];
  Block now{};
  int b = w.b_lo + wave, page = 0;
  if (b < b_end) {
    const int first = page_entry(v, w, b);
    page = page_entry(v, w, min(b + 4, b_end - 1));
    now = locate<DT>(v, w, b, first);
#pragma unroll
    for (int c = 0; c < DT; ++c) kt[c] = now.tiles[c * 64 + lane];
#pragma unroll
    for (int c = 0; c < DT; ++c) vt[c] = now.tiles[(DT + c) * 64 + lane];
  }
  Columns<DT, 1> cols;
  cols.load(a, u, 0, w.live);
#pragma unroll 1
  for (; b < b_end; b += 4) {
    uint4 kn[DT], vn[DT];
    Block next{};
    if (b + 4 < b_end) {
      const int after = page_entry(v, w, min(b + 8, b_end - 1));
      next = locate<DT>(v, w, b + 4, page);
#pragma unroll
      for (int c = 0; c < DT; ++c) kn[c] = next.tiles[c * 64 + lane];
#pragma unroll
      for (int c = 0; c < DT; ++c) vn[c] = next.tiles[(DT + c) * 64 + lane];
      page = after;
    }
    cols.step(
        b * kKvBlock, now.scale(0), now.scale(1),
        [&](int c, int h) { return codes_to_half(h ? kt[c].z : kt[c].x, h ? kt[c].w : kt[c].y); },
        [&](int c, int h) { return codes_to_half(h ? vt[c].z : vt[c].x, h ? vt[c].w : vt[c].y); });
#pragma unroll
    for (int c = 0; c < DT; ++c) kt[c] = kn[c], vt[c] = vn[c];
    now = next;
  }
  cols.finish();
  // waves 2, 3 hand over to 0, 1, then 1 to 0
#pragma unroll
  for (int h = 2; h >= 1; h >>= 1) {
    float* buf = merge + (h == 2 ? wave & 1 : 0) * 16 * Sz::kMergeRow;
    __syncthreads();
    if (wave >= h && wave < 2 * h) {
      float* c = buf + i * Sz::kMergeRow;
#pragma unroll
      for (int j = 0; j < 2 * DT; ++j) *(float4_t*)(c + 16 * j + 4 * g) = cols.o[0][j];
      if (g == 0) c[Sz::DP] = cols.m[0], c[Sz::DP + 1] = cols.l[0];
    }
    __syncthreads();
    if (wave < h) {
      const float* c = buf + i * Sz::kMergeRow;
      const float m1 = cols.m[0], m2 = c[Sz::DP], l2 = c[Sz::DP + 1];
      const float mn = fmaxf(m1, m2), r1 = fast_exp2(m1 - mn), r2 = fast_exp2(m2 - mn);
      cols.m[0] = mn;
      cols.l[0] = cols.l[0] * r1 + l2 * r2;
#pragma unroll
      for (int j = 0; j < 2 * DT; ++j)
        cols.o[0][j] = cols.o[0][j] * r1 + *(const float4_t*)(c + 16 * j + 4 * g) * r2;
    }
  }
  const Results<DT> res{a, u, w.live};
  if (wave == 0) res.put(cols, 0);
  if (u.chunks > 1) res.join(merge, s_last);
}

// Four waves go over the same blocks with 16 CT columns each.  A block's codes are
// turned into fp16 once, every wave a quarter of them, into one of two LDS
// buffers, from which all read their operands (16 bytes a lane, no bank twice).
//
// The VALU bounds it: per 16 columns and block 8 exponentials, the weights' two
// parts and the sums, about 70 instructions, against 8 DT matrix instructions of
// four times an instruction's length.  Where all CUs have work it reaches 450 TFLOP/s
// with heads of 64 and 525 with heads of 128 (8 prompts of 1024 rows on 8192 keys); the
// two parts leave 607 of what a large product reaches.
template <int DT, int CT>
__device__ __forceinline__ void attend_share(const AttnArgs& a, const Unit& u, half8_t* tiles,
                                             float* merge, int& s_last) {
  const KvView& v = a.v;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  constexpr int kMine = (2 * DT + 3) / 4;  // tiles of a wave
  float* scales = merge;                   // of the two buffers; free before the join
  Walk w;
  w.start<CT>(a, u);
  const int b_end = w.b_hi;
  uint4 raw[kMine];
  float sc[2];
  bool ok = false;
  auto fetch = [&](int b, int page) {
    const Block at = locate<DT>(v, w, b, page);
#pragma unroll
    for (int k = 0; k < kMine; ++k)
      if (wave + 4 * k < 2 * DT) raw[k] = at.tiles[(wave + 4 * k) * 64 + lane];
    sc[0] = at.sc[0], sc[1] = at.sc[1], ok = at.ok;
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int k = 0; k < kMine; ++k)
      if (wave + 4 * k < 2 * DT) {
        half8_t* y = tiles + ((buf * 2 * DT + wave + 4 * k) * 2) * 64 + lane;
        y[0] = codes_to_half(raw[k].x, raw[k].y);
        y[64] = codes_to_half(raw[k].z, raw[k].w);
      }
    if (threadIdx.x == 0) {
      scales[2 * buf] = ok ? sc[0] : __builtin_nanf("");
      scales[2 * buf + 1] = ok ? sc[1] : __builtin_nanf("");
    }
  };
  int b = w.b_lo, page = 0;
  if (b < b_end) {
    const int first = page_entry(v, w, b);
    page = page_entry(v, w, min(b + 1, b_end - 1));
    fetch(b, first);
  }
  Columns<DT, CT> cols;
  cols.load(a, u, wave * 16 * CT, w.live);
  if (b < b_end) {
    put(0);
    const int after = page_entry(v, w, min(b + 2, b_end - 1));
    fetch(min(b + 1, b_end - 1), page);
    page = after;
  }
#pragma unroll 1
  for (int buf = 0; b < b_end; ++b, buf ^= 1) {
    // this block's buffer is whole, and the other one is read no more
    __syncthreads();
    if (b + 1 < b_end) {
      put(buf ^ 1);
      const int after = page_entry(v, w, min(b + 3, b_end - 1));
      fetch(min(b + 2, b_end - 1), page);
      page = after;
    }
    if (b * kKvBlock <= cols.top) {
      const half8_t* x = tiles + buf * 2 * DT * 2 * 64 + lane;
      cols.step(
          b * kKvBlock, scales[2 * buf], scales[2 * buf + 1],
          [&](int c, int h) { return x[(2 * c + h) * 64]; },
          [&](int c, int h) { return x[(2 * (DT + c) + h) * 64]; });
    }
  }
  cols.finish();
  const Results<DT> res{a, u, w.live};
  res.put(cols, wave * 16 * CT);
  if (u.chunks > 1) res.join(merge, s_last);
}

// Waves a SIMD holds: what the registers of a wave's column tiles allow without
// spills (tiles 0: single tokens only).
constexpr int waves_per_simd(int DT, int tiles) {
  return tiles == 2 ? (DT <= 2 ? 3 : DT <= 4 ? 2 : 1) : DT <= 2 ? 4 : DT <= 3 ? 3 : DT <= 5 ? 2 : 1;
}

// Launches of sequences of up to 16 columns only, and any others.
template <int DT>
__global__ __launch_bounds__(kKvThreads, waves_per_simd(DT, 0))
void kv8_attn_tokens_kernel(AttnArgs a) {
  constexpr int kMerge = 2 * 16 * Sizes<DT>::kMergeRow, kJoin = 6 * kKvThreads;
  __shared__ PlanLds plan;
  __shared__ __align__(16) float merge[kMerge > kJoin ? kMerge : kJoin];
  __shared__ int s_last;
  const Unit u = find_unit<1, false>(a, (int)blockIdx.x, plan);
  if (u.s >= 0) attend_split<DT>(a, u, merge, s_last);
}
template <int DT, int CT>
__global__ __launch_bounds__(kKvThreads, waves_per_simd(DT, CT))
void kv8_attn_mixed_kernel(AttnArgs a) {
  constexpr int kMerge = 2 * 16 * Sizes<DT>::kMergeRow, kJoin = 6 * kKvThreads;
  constexpr int kTiles = 2 * 2 * DT * 2 * 64 * 4;  // floats of the two buffers
  __shared__ PlanLds plan;
  __shared__ __align__(16) float lds[kTiles + kJoin > kMerge ? kTiles + kJoin : kMerge];
  __shared__ int s_last;
  const Unit u = find_unit<CT, true>(a, (int)blockIdx.x, plan);
  if (u.s < 0) return;
  if (u.form == SPLIT)
    attend_split<DT>(a, u, lds, s_last);
  else
    attend_share<DT, CT>(a, u, (half8_t*)lds, lds + kTiles, s_last);
}

// tiles: 0 for the tokens kernel, else column tiles of a wave that shares its keys
template <int DT>
int launch_attn(AttnArgs& a, int n_heads, int tiles) {
  const KvView& v = a.v;
  const int uc = tiles ? 64 * tiles : 16;
  // As many chunks as run at once; twice as many of the larger units, which then end
  // more evenly.
  a.target = min((tiles == 2 ? 2 : 1) * waves_per_simd(DT, tiles) * ctx().num_cus, kMaxTarget);
  a.per_target = nextafterf(1.0f / (float)a.target, 1.0f);
  a.part_cols = uc;
  if (ensure_workspace((size_t)3 * a.target * uc * Sizes<DT>::kRow * sizeof(float))) return -1;
  a.part = (float*)ctx().ws;
  // The kernel's own plan has at most target + units workgroups with work, and no
  // unit more chunks than its table row can fill.  (A sequence's units are at most
  // its columns / uc and two more, also where it is cut in tiles of 16.)
  const int64_t units = (int64_t)v.n_kv_heads * ((int64_t)v.n_rows * a.G / uc +
                                                 2 * min(v.n_rows, v.n_seqs));
  const int64_t most_chunks = ((int64_t)v.max_pages * v.blocks + kMinChunk - 1) / kMinChunk;
  const int64_t wgs = min(units + a.target, units * most_chunks);
  if (wgs > kMaxWorkgroups) {
    set_error("plh_kv8_attn: %d rows of %d heads are too many for one call", v.n_rows, n_heads);
    return -1;
  }
  const dim3 grid((unsigned)wgs), block(kKvThreads);
  if (tiles == 0)
    hipLaunchKernelGGL(kv8_attn_tokens_kernel<DT>, grid, block, 0, ctx().stream, a);
  else if (tiles == 1)
    hipLaunchKernelGGL((kv8_attn_mixed_kernel<DT, 1>), grid, block, 0, ctx().stream, a);
  else
    hipLaunchKernelGGL((kv8_attn_mixed_kernel<DT, 2>), grid, block, 0, ctx().stream, a);
  return check_hip(hipGetLastError(), "kv8_attn_kernel");
}

}  // namespace
}  // namespace plh

using namespace plh;

extern "C" int plh_kv8_attn(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, int layer,
                            int n_heads, int n_rows, const int32_t* row_start, const float* q,
                            int q_stride, float* out, int out_stride) {
  const char* what = "plh_kv8_attn";
  AttnArgs a{};
  if (kv_view(cache, seqs, layer, n_rows, row_start, what, a.v)) return -1;
  const int D = cache->head_dim;
  if (n_heads < 1 || n_heads % cache->n_kv_heads) {
    set_error("%s: %d q heads over %d kv heads", what, n_heads, cache->n_kv_heads);
    return -1;
  }
  if (n_rows && (!q || !out || (((uintptr_t)q | (uintptr_t)out) & 3) ||
                 (int64_t)n_heads * D > q_stride || (int64_t)n_heads * D > out_stride)) {
    set_error("%s: q or out is null, not aligned, or has rows of %d and %d floats for %d heads",
              what, q_stride, out_stride, n_heads);
    return -1;
  }
  if ((int64_t)n_rows * n_heads > INT_MAX / 2) {
    set_error("%s: %d rows of %d heads are too many for one call", what, n_rows, n_heads);
    return -1;
  }
  if (kv_ready(what)) return -1;
  if (n_rows == 0) return 0;
  a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
  a.G = n_heads / cache->n_kv_heads;
  a.score_scale = kLog2e / sqrtf((float)D);
  a.q_vec = (((uintptr_t)q | (uintptr_t)q_stride * 4 | (uintptr_t)D * 4) & 15) == 0;
  a.out_vec = (((uintptr_t)out | (uintptr_t)out_stride * 4 | (uintptr_t)D * 4) & 15) == 0;
  a.fd_g = make_fastdiv((uint32_t)a.G);
  a.fd_kvh = make_fastdiv((uint32_t)cache->n_kv_heads);
  // Short sequences (on average) in a launch of their own registers.  Others' waves
  // take two tiles of columns, so that keys are read from LDS half as often, where
  // that leaves two units and more for every CU.
  const int64_t seqs_rows = min(n_rows, seqs->n_seqs);
  const bool tokens = (int64_t)n_rows * a.G <= 16 * seqs_rows;
  const bool few = (int64_t)n_rows * n_heads / 128 + seqs_rows * cache->n_kv_heads <
                   2ll * ctx().num_cus;
  const int tiles = tokens ? 0 : few ? 1 : 2;
  switch (kv_tiles(D)) {
    case 1: return launch_attn<1>(a, n_heads, tiles);
    case 2: return launch_attn<2>(a, n_heads, tiles);
    case 3: return launch_attn<3>(a, n_heads, tiles);
    case 4: return launch_attn<4>(a, n_heads, tiles);
    case 5: return launch_attn<5>(a, n_heads, tiles);
    case 6: return launch_attn<6>(a, n_heads, tiles);
    case 7: return launch_attn<7>(a, n_heads, tiles);
    default: return launch_attn<8>(a, n_heads, tiles);
  }
}
