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
// so O has a unit of its own: 2^(m + dO), dO a whole number per column.  While
// log2 v_b stays within [dO - 6, dO + 4] it goes into the weights' exponent for
// free, and l gets the weights times 2^-(that difference).  A block outside it
// (the first one; v scales that jump by powers of two; scores past 2^5) moves the
// unit to the largest s_t + log2 v_b so far and takes its own exponentials for l:
// what is small beside the largest contribution is rounded, nothing else.
//
// Layout.  A tile's bytes are in operand order (include/picolm_hip.h): lane
// 16 g + i of a wave loads 16 adjacent bytes, a tile of k serves two row blocks
// of S (tokens i and 16 + i), a tile of v two row blocks of O; the S
// accumulators of lane (g, col) are tokens 4 g + r and 16 + 4 g + r, which are the
// lane's contraction slots of the second product: no LDS, no transposition and
// no exchange between lanes but the maximum's.
//
// Work.  A unit is up to UC columns of one (sequence, kv head): 16 columns whose
// keys the four waves split (CT 1), or up to 128, each wave 32 of them (CT 2; a
// unit with at most 64 or 32 live columns splits its keys over two or four
// waves as well).  Every workgroup finds its unit from row_start and len, so
// nothing is planned on the host and a captured graph follows the lengths.  Units
// are cut into chunks of blocks where there are few of them; the last workgroup
// of a unit to finish joins the chunks' partial results in their order.
#include <limits.h>
#include <math.h>

#include "attn_common.h"
#include "kv8.h"

namespace plh {
namespace {

constexpr int kDevScope = 16;      // buffer cache policy sc1: past the XCD's L2
constexpr float kPlainMax = 32.0f;  // log2 units: larger running maxima take exact steps
constexpr int kMaxTarget = 2048;   // most chunks asked for of the units that are cut

// Arrival counters of cut units, zero between launches.
__device__ unsigned g_kv8_ctr[2 * kMaxTarget];

struct AttnArgs {
  KvView v;
  const float* q;
  float* out;
  int q_stride, out_stride;
  int G;               // q heads of a kv head
  int target;          // chunks aimed at
  int min_chunk;       // blocks
  float score_scale;   // log2(e) / sqrt(D)
  float* part;         // [slot][columns][Dp + 2]
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

// x0, x1 as fp16 hi (rounded toward zero) and lo = x - hi (exact, then rounded).
// Left to the compiler rather than written in asm: it knows how many wait states
// lie between the write of half a register and a matrix instruction that reads it.
__device__ __forceinline__ void split_pair(float x0, float x1, half2_t& hi, half2_t& lo) {
  hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
  lo[0] = (_Float16)__builtin_fmaf((float)hi[0], -1.0f, x0);
  lo[1] = (_Float16)__builtin_fmaf((float)hi[1], -1.0f, x1);
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a workgroup works on.
struct Unit {
  int s;             // sequence, or -1
  int row0, rows;    // its rows
  int len;
  int kvh, col0;     // first column (token * G + head of the group)
  int chunk, chunks;
  int slot;          // of the unit's first chunk among the cut units' partials
};

// Inclusive sum over the wave.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

struct PlanLds {
  int64_t part[kKvThreads / 64];
  int found[6];
};

// Sum over the workgroup of a value per thread, and over the threads before.
__device__ __forceinline__ int64_t group_scan(int64_t x, PlanLds& lds, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t sum = wave_scan(x);
  __syncthreads();
  if (lane == 63) lds.part[wave] = sum;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kKvThreads / 64; ++w) {
    before += w < wave ? lds.part[w] : 0;
    total += lds.part[w];
  }
  return before + sum - x;
}

// Workgroup `wg`'s unit.  Chunk length C = max(min_chunk, blocks of all units /
// target), so at most target + units workgroups have work and at most 2 target
// chunks belong to cut units (each has more than C blocks).
template <int UC>
__device__ __forceinline__ Unit find_unit(const AttnArgs& a, int wg, PlanLds& lds) {
  const KvView& v = a.v;
  Unit u{};
  u.s = -1;
  // four sequences a thread at most
  const int per = (v.n_seqs + kKvThreads - 1) / kKvThreads;
  const int s0 = (int)threadIdx.x * per;
  int row0[4], rows[4], len[4];
  int64_t blocks = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    row0[k] = rows[k] = len[k] = 0;
    if (k < per && s0 + k < v.n_seqs) {
      kv_rows(v, s0 + k, row0[k], rows[k]);
      len[k] = kv_len(v, s0 + k);
      const int units = (int)(((int64_t)rows[k] * a.G + UC - 1) / UC);
      blocks += (int64_t)units * ((len[k] + kKvBlock - 1) / kKvBlock);
    }
  }
  int64_t all;
  group_scan(blocks, lds, all);
  const int64_t chunk = max((int64_t)a.min_chunk, (all * v.n_kv_heads + a.target - 1) / a.target);
  // workgroups and cut chunks (at most 2 target: 16 bits) of each thread's sequences
  int64_t wgs = 0, cut = 0;
  int n_wgs[4], n_chunks[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int units = (int)(((int64_t)rows[k] * a.G + UC - 1) / UC);
    const int nb = (len[k] + kKvBlock - 1) / kKvBlock;
    n_chunks[k] = max(1, (int)((nb + chunk - 1) / chunk));
    n_wgs[k] = units * n_chunks[k] * v.n_kv_heads;
    wgs += n_wgs[k];
    cut += n_chunks[k] > 1 ? n_wgs[k] : 0;
  }
  int64_t total;
  const int64_t before = group_scan(cut << 48 | wgs, lds, total);
  constexpr int64_t kLow = (1ll << 48) - 1;
  // row_start that does not rise: more units than rows; no chunk may be left out
  // of a cut unit
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
  // a sequence's workgroups: units (those of the longest contexts first), kv
  // heads, chunks
  const int local = uniform(lds.found[1]);
  const int unit_kvh = local / u.chunks;
  u.chunk = local - unit_kvh * u.chunks;
  const int unit = (int)fdiv((uint32_t)unit_kvh, a.fd_kvh);
  u.kvh = unit_kvh - unit * v.n_kv_heads;
  const int units = (int)(((int64_t)u.rows * a.G + UC - 1) / UC);
  u.col0 = (units - 1 - unit) * UC;
  u.slot = uniform(lds.found[3]) + unit_kvh * u.chunks;
  return u;
}

template <int DT, int CT>
struct Shape {
  static constexpr int kGroups = CT == 1 ? 1 : 4;       // column groups of a unit
  static constexpr int kCols = 16 * CT;                 // columns of a group
  static constexpr int UC = kGroups * kCols;
  static constexpr int DP = 32 * DT;
  static constexpr int kRow = DP + 2;                   // floats of a partial column
  static constexpr int kMergeRow = DP + 4;              // LDS pitch of a column's O, m, l
};

template <int DT, int CT>
__global__ __launch_bounds__(kKvThreads, CT == 1 ? (DT <= 2 ? 4 : DT <= 3 ? 3 : DT <= 6 ? 2 : 1) : DT <= 3 ? 2 : 1)
void kv8_attn_kernel(AttnArgs a) {
  using Sh = Shape<DT, CT>;
  __shared__ PlanLds plan;
  __shared__ __align__(16) float merge[2 * Sh::kCols * Sh::kMergeRow];
  __shared__ int s_last;
  const KvView& v = a.v;
  const Unit u = find_unit<Sh::UC>(a, (int)blockIdx.x, plan);
  if (u.s < 0) return;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int G = a.G, D = v.D;
  const int cols = u.rows * G;                       // of the (sequence, kv head)
  const int live = min(Sh::UC, cols - u.col0);       // of the unit
  // the waves: column group, and which share of its keys
  const int groups = Sh::kGroups == 1 || live <= Sh::kCols ? 1 : live <= 2 * Sh::kCols ? 2 : 4;
  const int cg = wave % groups, part = wave / groups, parts = 4 / groups;
  const int base = u.len - u.rows;                   // position of the first row

  // ---- columns and q -----------------------------------------------------------
  int lim[CT];                  // the column's position (no column: sees all, is not stored)
  half8_t qh[CT][DT], ql[CT][DT];
  float f0[CT];                 // score scale of the column (q's power of two in it)
  int top = -1, low = INT_MAX;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = cg * Sh::kCols + ct * 16 + i;
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
        _Float16 h, l;
        split_hi_lo(x[c8][j] * down, h, l);
        qh[ct][c8][j] = h, ql[ct][c8][j] = l;
      }
    top = max(top, on ? lim[ct] : -1);
    low = min(low, lim[ct]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    top = max(top, __shfl_xor(top, o, 64));
    low = min(low, __shfl_xor(low, o, 64));
  }
  top = uniform(top), low = uniform(low);

  // ---- the blocks ----------------------------------------------------------------
  // of the unit (its last column's position) and of this chunk
  const int last_col = u.col0 + live - 1;
  const int unit_top = base + (int)fdiv((uint32_t)last_col, a.fd_g);
  const int nb = unit_top < 0 ? 0 : unit_top / kKvBlock + 1;
  const int b_lo = (int)((int64_t)nb * u.chunk / u.chunks);
  const int b_hi = (int)((int64_t)nb * (u.chunk + 1) / u.chunks);
  const int b_end = min(b_hi, top < 0 ? 0 : top / kKvBlock + 1);

  float4_t o[CT][2 * DT];
  float m[CT], l[CT], dO[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kNegBig, l[ct] = 0.0f, dO[ct] = kNegBig;
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j) o[ct][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* row = v.table + (size_t)u.s * v.max_pages;
  const int64_t head_off = (int64_t)u.kvh * v.blocks * 2;
  // Loads run ahead: a block's page number two blocks before it, its tiles and
  // scales one.  A page outside the cache reads page 0, with NaN scales.
  auto entry = [&](int b) { return row[fdiv((uint32_t)b, v.fd_blocks)]; };
  auto fetch = [&](int b, int page, uint4 (&kt)[DT], uint4 (&vt)[DT], float (&sc)[2], bool& ok) {
    int p = uniform(page);
    ok = p >= 0 && p < v.n_pages;
    p = ok ? p : 0;
    const int in = b - (int)fdiv((uint32_t)b, v.fd_blocks) * v.blocks;
    const int64_t unit = head_off + in * 2;
    const uint4* tiles = (const uint4*)(v.codes + p * v.page_codes + unit * DT * kKvTile) + lane;
#pragma unroll
    for (int c = 0; c < DT; ++c) kt[c] = tiles[c * 64];
#pragma unroll
    for (int c = 0; c < DT; ++c) vt[c] = tiles[(DT + c) * 64];
    const float* s = v.scales + p * v.page_scales + unit;
    sc[0] = s[0], sc[1] = s[1];
  };
  uint4 kt[DT], vt[DT];
  float sc[2] = {0.0f, 0.0f};
  bool ok = false;
  int b = b_lo + part, page = 0;
  if (b < b_end) {
    const int first = entry(b);
    page = entry(min(b + parts, b_end - 1));
    fetch(b, first, kt, vt, sc, ok);
  }
#pragma unroll 1
  for (; b < b_end; b += parts) {
    uint4 kn[DT], vn[DT];
    float scn[2] = {0.0f, 0.0f};
    bool okn = false;
    if (b + parts < b_end) {
      const int after = entry(min(b + 2 * parts, b_end - 1));
      fetch(b + parts, page, kn, vn, scn, okn);
      page = after;
    }
    const float nan = __builtin_nanf("");
    const float ks = ok ? sc[0] : nan, vs = ok ? sc[1] : nan;
    // S
    float4_t s0[CT], s1[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) s0[ct] = s1[ct] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      const half8_t k0 = codes_to_half(kt[c].x, kt[c].y), k1 = codes_to_half(kt[c].z, kt[c].w);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        s0[ct] = mfma16x16x32(k0, ql[ct][c], s0[ct]);
        s1[ct] = mfma16x16x32(k1, ql[ct][c], s1[ct]);
        s0[ct] = mfma16x16x32(k0, qh[ct][c], s0[ct]);
        s1[ct] = mfma16x16x32(k1, qh[ct][c], s1[ct]);
      }
    }
    // log2 of the v scale as exponent and remainder (0: -inf; NaN, inf: NaN)
    const float vn_ = vs < 1e-30f ? vs * 0x1p100f : vs;
    const int ve = (int)(__float_as_uint(vn_) >> 23) - 127;
    float lm = __builtin_amdgcn_logf(__uint_as_float((__float_as_uint(vn_) & 0x7FFFFFu) |
                                                     0x3F800000u));
    float ex = (float)(ve - (vs < 1e-30f ? 100 : 0));
    if (vs == 0.0f) ex = -INFINITY;
    if (!(vs < INFINITY)) lm = nan;
    const int t0 = b * kKvBlock;
    const bool masked = t0 + kKvBlock - 1 > low;
    half8_t ph[CT], pl[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float f = f0[ct] * ks;
      float p[8];
      float mt;
      if (masked) {
        mt = kNegBig;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (t0 + 4 * g + r <= lim[ct]) mt = fmaxf(mt, s0[ct][r] * f);
          if (t0 + 16 + 4 * g + r <= lim[ct]) mt = fmaxf(mt, s1[ct][r] * f);
        }
      } else {
        mt = vmax(vmax(vmax(s0[ct][0], s0[ct][1]), vmax(s0[ct][2], s0[ct][3])),
                  vmax(vmax(s1[ct][0], s1[ct][1]), vmax(s1[ct][2], s1[ct][3]))) * f;
        mt = fmaxf(kNegBig, mt);  // NaN scores go into the weights, not the maximum
      }
      mt = max_xor32(max_xor16(mt));
      // Every column decides for itself, so that no other column's values reach
      // its result, not even its last bits.
      float lr = lm - (dO[ct] - ex);
      const float mn = fmaxf(m[ct], mt);
      const bool apart = !(lr >= -6.0f && lr <= 4.0f && __builtin_fabsf(mn) <= kPlainMax);
      const bool any_apart = __any(apart);
      if (any_apart || __any(mt > m[ct] + 8.0f)) {
        // O and l follow the maximum only where it grew by more than 2^8: the
        // weights stay below 2^12, far inside fp16
        const float to = apart || mt > m[ct] + 8.0f ? mn : m[ct];
        const float at = fmaxf(m[ct] + dO[ct], mt + (lm + ex));
        const float dn = apart ? __builtin_ceilf(at - to) : dO[ct];
        const float r = fast_exp2((m[ct] - to) + (dO[ct] - dn));
        l[ct] *= fast_exp2(m[ct] - to);
        m[ct] = to, dO[ct] = dn;
        lr = lm - (dn - ex);
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) o[ct][j] = o[ct][j] * r;
      }
      // 2^(score - m + up), zero where the column does not see, and their sum.  As
      // one fused step the exponent is off by the roundings of m and up - m, at
      // most 2^-19 for |m| up to kPlainMax; larger scores take the rounded
      // product, which m is the largest of, and each sum by itself.
      auto hide = [&]() {
        if (masked) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (t0 + 4 * g + r > lim[ct]) p[r] = 0.0f;
            if (t0 + 16 + 4 * g + r > lim[ct]) p[4 + r] = 0.0f;
          }
        }
        return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      };
      const float off = lr - m[ct];
      if (any_apart) {
        auto exact = [&](float up) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[r] = fast_exp2(apart ? (s0[ct][r] * f - m[ct]) + up
                                   : __builtin_fmaf(s0[ct][r], f, off));
            p[4 + r] = fast_exp2(apart ? (s1[ct][r] * f - m[ct]) + up
                                       : __builtin_fmaf(s1[ct][r], f, off));
          }
          return hide();
        };
        const float plain = exact(0.0f), sum = exact(lr);
        l[ct] = apart ? l[ct] + plain : __builtin_fmaf(sum, fast_exp2(-lr), l[ct]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = fast_exp2(__builtin_fmaf(s0[ct][r], f, off));
          p[4 + r] = fast_exp2(__builtin_fmaf(s1[ct][r], f, off));
        }
        l[ct] = __builtin_fmaf(hide(), fast_exp2(-lr), l[ct]);
      }
#pragma unroll
      for (int r = 0; r < 8; r += 2) {
        half2_t h, lo;
        split_pair(p[r], p[r + 1], h, lo);
        ph[ct][r] = h[0], ph[ct][r + 1] = h[1];
        pl[ct][r] = lo[0], pl[ct][r + 1] = lo[1];
      }
    }
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      const half8_t v0 = codes_to_half(vt[c].x, vt[c].y), v1 = codes_to_half(vt[c].z, vt[c].w);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct][2 * c] = mfma16x16x32(v0, pl[ct], o[ct][2 * c]);
        o[ct][2 * c + 1] = mfma16x16x32(v1, pl[ct], o[ct][2 * c + 1]);
        o[ct][2 * c] = mfma16x16x32(v0, ph[ct], o[ct][2 * c]);
        o[ct][2 * c + 1] = mfma16x16x32(v1, ph[ct], o[ct][2 * c + 1]);
      }
    }
#pragma unroll
    for (int c = 0; c < DT; ++c) kt[c] = kn[c], vt[c] = vn[c];
    sc[0] = scn[0], sc[1] = scn[1], ok = okn;
  }

  // ---- l over the lanes of a column, O in values ---------------------------------
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] = add_xor32(add_xor16(l[ct]));
    const int e = (int)fmaxf(dO[ct], -400.0f);
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[ct][j][r] = __builtin_ldexpf(o[ct][j][r], e);
  }
  // ---- waves that share columns: the upper half hands over to the lower ---------
  for (int h = parts / 2; h >= 1; h >>= 1) {
    // parts 4: waves 2, 3 to 0, 1, then 1 to 0; parts 2 (two groups): 2, 3 to 0, 1
    const bool gives = part >= h && part < 2 * h, takes = part < h;
    float* buf = merge + (size_t)((groups == 2 ? cg : part % h) & 1) * Sh::kCols * Sh::kMergeRow;
    __syncthreads();
    if (gives) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float* c = buf + (ct * 16 + i) * Sh::kMergeRow;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) *(float4_t*)(c + 16 * j + 4 * g) = o[ct][j];
        if (g == 0) c[Sh::DP] = m[ct], c[Sh::DP + 1] = l[ct];
      }
    }
    __syncthreads();
    if (takes) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float* c = buf + (ct * 16 + i) * Sh::kMergeRow;
        const float m2 = c[Sh::DP], l2 = c[Sh::DP + 1];
        const float mn = fmaxf(m[ct], m2), r1 = fast_exp2(m[ct] - mn), r2 = fast_exp2(m2 - mn);
        m[ct] = mn;
        l[ct] = l[ct] * r1 + l2 * r2;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j)
          o[ct][j] = o[ct][j] * r1 + *(const float4_t*)(c + 16 * j + 4 * g) * r2;
      }
    }
  }
  // ---- results ----------------------------------------------------------------------
  auto out_row = [&](int c) {
    const int col = u.col0 + c, t = (int)fdiv((uint32_t)col, a.fd_g);
    return a.out + (int64_t)(u.row0 + t) * a.out_stride + (int64_t)(u.kvh * G + col - t * G) * D;
  };
  auto store4 = [&](float* y, int d, float4_t x) {
    if (a.out_vec) {
      if (d < D) *(float4_t*)(y + d) = x;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < D) y[d + e] = x[e];
    }
  };
  if (u.chunks == 1) {
    if (part == 0) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int c = cg * Sh::kCols + ct * 16 + i;
        if (c >= live) continue;
        float* y = out_row(c);
        const float inv = l[ct] == 0.0f ? 0.0f : 1.0f / l[ct];
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) store4(y, 16 * j + 4 * g, o[ct][j] * inv);
      }
    }
    return;
  }
  // a chunk's partial columns: O, m and l, written past the L2 so that the
  // workgroup that joins them may run on another XCD
  constexpr int kPartBytes = Sh::UC * Sh::kRow * 4;
  float* unit_part = a.part + (int64_t)u.slot * Sh::UC * Sh::kRow;
  if (part == 0) {
    const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(
        unit_part + (int64_t)u.chunk * Sh::UC * Sh::kRow, 0, kPartBytes, 0x00020000);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = cg * Sh::kCols + ct * 16 + i;
      if (c >= live) continue;
#pragma unroll
      for (int j = 0; j < 2 * DT; ++j)
        __builtin_amdgcn_raw_buffer_store_b128(o[ct][j], prs, (c * Sh::DP + 16 * j + 4 * g) * 4, 0,
                                               kDevScope);
      if (g == 0) {
        const int at = (Sh::UC * Sh::DP + 2 * c) * 4;
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(m[ct]), prs, at, 0, kDevScope);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l[ct]), prs, at + 4, 0, kDevScope);
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // the partials have arrived before the count goes up
  __syncthreads();
  unsigned* ctr = g_kv8_ctr + u.slot;
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             (unsigned)(u.chunks - 1);
  __syncthreads();
  if (!s_last) return;
  if (threadIdx.x == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int idx = threadIdx.x; idx < live * (Sh::DP / 4); idx += kKvThreads) {
    const int c = idx / (Sh::DP / 4), d = 4 * (idx - c * (Sh::DP / 4));
    float M = kNegBig, L = 0.0f;
    float4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int n0 = 0; n0 < u.chunks; n0 += 8) {
      float4_t on[8];
      float mn[8], ln[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int n = min(n0 + k, u.chunks - 1);  // past the last: again, not used
        const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(
            unit_part + (int64_t)n * Sh::UC * Sh::kRow, 0, kPartBytes, 0x00020000);
        on[k] = __builtin_amdgcn_raw_buffer_load_b128(prs, (c * Sh::DP + d) * 4, 0, kDevScope);
        const int at = (Sh::UC * Sh::DP + 2 * c) * 4;
        mn[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at, 0, kDevScope));
        ln[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at + 4, 0, kDevScope));
      }
      float Mn = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) Mn = fmaxf(Mn, mn[k]);
      const float r = fast_exp2(M - Mn);
      L *= r;
      O = O * r;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n0 + k < u.chunks) {
          const float w = fast_exp2(mn[k] - Mn);
          L += ln[k] * w;
          O = O + on[k] * w;
        }
      M = Mn;
    }
    store4(out_row(c), d, O * (L == 0.0f ? 0.0f : 1.0f / L));
  }
}

template <int DT, int CT>
int launch_attn(AttnArgs& a, int n_heads) {
  using Sh = Shape<DT, CT>;
  const KvView& v = a.v;
  const int cus = ctx().num_cus;
  a.target = min(CT == 1 ? 4 * cus : 2 * cus, kMaxTarget);
  a.min_chunk = 16;
  if (ensure_workspace((size_t)2 * a.target * Sh::UC * Sh::kRow * sizeof(float))) return -1;
  a.part = (float*)ctx().ws;
  // The kernel's own plan has at most target + units workgroups with work, and no
  // unit more chunks than its table row can fill.
  const int64_t units = (int64_t)v.n_kv_heads * ((int64_t)v.n_rows * a.G / Sh::UC +
                                                 min(v.n_rows, v.n_seqs));
  const int64_t most_chunks =
      ((int64_t)v.max_pages * v.blocks + a.min_chunk - 1) / a.min_chunk;
  const int64_t wgs = min(units + a.target, units * most_chunks);
  if (wgs > kMaxWorkgroups) {
    set_error("plh_kv8_attn: %d rows of %d heads are too many for one call", v.n_rows, n_heads);
    return -1;
  }
  hipLaunchKernelGGL((kv8_attn_kernel<DT, CT>), dim3((unsigned)wgs), dim3(kKvThreads), 0,
                     ctx().stream, a);
  return check_hip(hipGetLastError(), "kv8_attn_kernel");
}

template <int CT>
int launch_tiles(AttnArgs& a, int n_heads) {
  switch (kv_tiles(a.v.D)) {
    case 1: return launch_attn<1, CT>(a, n_heads);
    case 2: return launch_attn<2, CT>(a, n_heads);
    case 3: return launch_attn<3, CT>(a, n_heads);
    case 4: return launch_attn<4, CT>(a, n_heads);
    case 5: return launch_attn<5, CT>(a, n_heads);
    case 6: return launch_attn<6, CT>(a, n_heads);
    case 7: return launch_attn<7, CT>(a, n_heads);
    default: return launch_attn<8, CT>(a, n_heads);
  }
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
  // Sequences of up to 16 columns on average: 16-column units, their keys split
  // over the waves; more: units of 128.
  const bool narrow = (int64_t)n_rows * a.G <= 16ll * min(n_rows, seqs->n_seqs);
  return narrow ? launch_tiles<1>(a, n_heads) : launch_tiles<2>(a, n_heads);
}
