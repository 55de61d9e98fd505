// rope.hip -- rotary positions: tables with scaled frequencies, and the
// rotation of q and k rows by them (include/picolm_hip.h, plh_rope_*).
#include <limits.h>
#include <math.h>

#include "picolm_hip.h"
#include "plh_internal.h"
#include "rope_dev.h"

namespace plh {

int check_rope(const plh_rope* r, int head_dim, const char* what) {
  if (r->rope_type != PLH_ROPE_LLAMA && r->rope_type != PLH_ROPE_QWEN) {
    set_error("%s: rope_type %d", what, r->rope_type);
    return -1;
  }
  if (r->rot_dim < 2 || (r->rot_dim & 1) || r->rot_dim > head_dim) {
    set_error("%s: rot_dim %d of head_dim %d (even, 2..head_dim)", what, r->rot_dim, head_dim);
    return -1;
  }
  if (r->n_pos < 1 || !r->cos_tab || !r->sin_tab) {
    set_error("%s: no rotation tables", what);
    return -1;
  }
  return 0;
}

RopeRows rope_rows_args(const plh_rope* r, int head_dim, const float* q, int n_heads, int q_stride,
                        float* q_out, int q_out_stride, const float* k, int n_kv_heads,
                        int k_stride, float* k_out, int k_out_stride) {
  RopeRows a{};
  a.cos_t = r->cos_tab, a.sin_t = r->sin_tab;
  a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
  a.q_stride = q_stride, a.k_stride = k_stride;
  a.q_out_stride = q_out_stride, a.k_out_stride = k_out_stride;
  a.n_heads = n_heads, a.D = head_dim, a.rot = r->rot_dim, a.n_pos = r->n_pos;
  a.qwen = r->rope_type == PLH_ROPE_QWEN;
  // Four floats at a time where every address and every part of a head
  // allows it, else pair by pair.
  uintptr_t bits = (uintptr_t)(head_dim | (a.qwen ? a.rot / 2 : a.rot)) * 4;
  const bool hq = n_heads > 0, hk = n_kv_heads > 0;
  if (hq) bits |= (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)(q_stride | q_out_stride) * 4;
  if (hk) bits |= (uintptr_t)k | (uintptr_t)k_out | (uintptr_t)(k_stride | k_out_stride) * 4;
  const uintptr_t tab = (uintptr_t)r->cos_tab | (uintptr_t)r->sin_tab | (uintptr_t)(a.rot / 2) * 4;
  a.vec = (bits & 15) == 0 && (tab & (a.qwen ? 15 : 7)) == 0;
  const int v = a.vec ? 4 : 1;
  a.pairs = a.qwen ? a.rot / 2 / v : a.vec ? a.rot / 4 : a.rot / 2;
  a.per_head = a.pairs + (head_dim - a.rot) / v;
  a.per_row = (n_heads + n_kv_heads) * a.per_head;
  a.chunks = (a.per_row + kRopeThreads - 1) / kRopeThreads;
  if (a.chunks < 1) a.chunks = 1;  // no heads: nothing is launched for them
  a.fd_head = make_fastdiv((uint32_t)a.per_head);
  a.fd_chunk = make_fastdiv((uint32_t)a.chunks);
  return a;
}

}  // namespace plh

using namespace plh;

namespace {

constexpr int kMaxPairs = 128;

int rope_ready(const char* what) {
  if (ctx().stream) return 0;
  set_error("%s: library not initialised", what);
  return -1;
}

struct TableArgs {
  double freq[kMaxPairs];
  double magnitude;
  float* cos_t;
  float* sin_t;
  uint32_t n;  // n_pos * pairs
  int first, pairs;
  FastDiv fd_pairs;
};

// One table entry per thread: angle = position * theta in 64 bits, reduced to
// r in [-pi/4, pi/4] by the nearest multiple n of pi/2 (two parts of pi/2, each
// step a fused multiply-add, so the error stays below 2^-50 for every n of a
// 32-bit position), and the Taylor sums of sin and cos about 0 to r^13 and
// r^14 (the next terms are below 2.1e-14): 14 fused multiply-adds, where a
// general sincos has its large-argument path besides.
//
// HBM and 64-bit arithmetic bound it about equally: 8 bytes and some 30
// 64-bit operations an entry.  131072 positions of 32 pairs (33.6 MB) take 10.8
// us, 7.4 at a large copy's rate.
__global__ __launch_bounds__(256) void rope_tables_kernel(TableArgs a) {
  __shared__ double freq[kMaxPairs];
  if (threadIdx.x < (unsigned)a.pairs) freq[threadIdx.x] = a.freq[threadIdx.x];
  __syncthreads();
  const uint32_t stride = gridDim.x * 256u;
  for (uint64_t at = blockIdx.x * 256u + threadIdx.x; at < a.n; at += stride) {
    const uint32_t p = fdiv((uint32_t)at, a.fd_pairs), i = (uint32_t)at - p * a.pairs;
    const double angle = ((double)a.first + (double)p) * freq[i];
    const double n = __builtin_rint(angle * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489655800e+00, angle);
    r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double s = 1.0 / 6227020800.0;
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, r, r);
    double c = -1.0 / 87178291200.0;
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    // n mod 4 quarter turns
    const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    const double cn = (k & 1) ? s : c, sn = (k & 1) ? c : s;
    a.cos_t[at] = (float)((k == 1 || k == 2 ? -cn : cn) * a.magnitude);
    a.sin_t[at] = (float)((k >= 2 ? -sn : sn) * a.magnitude);
  }
}

// A thread per item; the row's position arrives while its elements do.  HBM
// bounds it: every element is read and written once.  203 MB (8191 rows of 24 heads
// of 128, half of each rotated) take 43 us, 4.7 TB/s; a single row 2.4 us, its latency.
template <bool QWEN>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeRows a, const int32_t* pos) {
  const int row = (int)fdiv(blockIdx.x, a.fd_chunk);
  const int item = ((int)blockIdx.x - row * a.chunks) * kRopeThreads + (int)threadIdx.x;
  if (item >= a.per_row) return;
  const int p = pos[row];
  rope_store<QWEN>(a, rope_load<QWEN>(a, row, item), p);
}

}  // namespace

extern "C" {

int plh_rope_frequencies_host(const plh_rope_spec* s, double* freq, double* magnitude) {
  if (!s || !freq || !magnitude) {
    set_error("plh_rope_frequencies_host: null argument");
    return -1;
  }
  const int R = s->rot_dim;
  if (R < 2 || (R & 1) || R > 2 * kMaxPairs) {
    set_error("rope: rot_dim %d (even, 2..%d)", R, 2 * kMaxPairs);
    return -1;
  }
  const bool scaled = s->scaling != PLH_ROPE_SCALE_NONE;
  const bool banded = s->scaling == PLH_ROPE_SCALE_BANDS || s->scaling == PLH_ROPE_SCALE_RAMP;
  if (s->scaling < PLH_ROPE_SCALE_NONE || s->scaling > PLH_ROPE_SCALE_RAMP ||
      (s->scaling == PLH_ROPE_SCALE_NTK && R == 2)) {
    set_error("rope: scaling %d with rot_dim %d", s->scaling, R);
    return -1;
  }
  if (!(s->freq_base > 1.0) || !isfinite(s->freq_base) ||
      (scaled && (!(s->factor >= 1.0) || !isfinite(s->factor))) || !(s->magnitude >= 0.0) ||
      !isfinite(s->magnitude)) {
    set_error("rope: freq_base above 1, factor from 1 and magnitude from 0 on are taken");
    return -1;
  }
  if (banded && (!(s->trained_len > 0.0) || !isfinite(s->trained_len) || !(s->low > 0.0) ||
                 !(s->high > s->low) || !isfinite(s->high))) {
    set_error("rope: trained_len above 0 and 0 < low < high are taken");
    return -1;
  }
  const double two_pi = 6.283185307179586476925;
  double base = s->freq_base;
  if (s->scaling == PLH_ROPE_SCALE_NTK) base *= pow(s->factor, (double)R / (R - 2));
  double lo = 0.0, hi = 0.0;
  if (s->scaling == PLH_ROPE_SCALE_RAMP) {
    const double den = 2.0 * log(base);
    lo = fmax(0.0, floor(R * log(s->trained_len / (two_pi * s->high)) / den));
    hi = fmin(R - 1.0, ceil(R * log(s->trained_len / (two_pi * s->low)) / den));
  }
  for (int i = 0; i < R / 2; ++i) {
    const double theta = pow(base, -2.0 * i / R);
    freq[i] = theta;
    if (s->scaling == PLH_ROPE_SCALE_LINEAR) {
      freq[i] = theta / s->factor;
    } else if (s->scaling == PLH_ROPE_SCALE_BANDS) {
      const double t = s->trained_len * theta / two_pi;
      const double k = fmin(1.0, fmax(0.0, (t - s->low) / (s->high - s->low)));
      freq[i] = (1.0 - k) * theta / s->factor + k * theta;
    } else if (s->scaling == PLH_ROPE_SCALE_RAMP) {
      const double g = fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 1e-3)));
      freq[i] = theta * (1.0 - g) + theta / s->factor * g;
    }
  }
  *magnitude = s->magnitude > 0.0 ? s->magnitude
               : s->scaling == PLH_ROPE_SCALE_RAMP ? 0.1 * log(s->factor) + 1.0
                                                   : 1.0;
  return 0;
}

int plh_rope_tables(const plh_rope_spec* spec, int first_pos, int n_pos, float* cos_tab,
                    float* sin_tab) {
  TableArgs a{};
  if (plh_rope_frequencies_host(spec, a.freq, &a.magnitude)) return -1;
  a.pairs = spec->rot_dim / 2;
  if (first_pos < 0 || n_pos < 0 || n_pos > INT_MAX - first_pos) {
    set_error("plh_rope_tables: %d positions from %d", n_pos, first_pos);
    return -1;
  }
  if ((int64_t)n_pos * a.pairs > INT_MAX) {
    set_error("plh_rope_tables: %d positions of %d pairs are too many for one call", n_pos,
              a.pairs);
    return -1;
  }
  if (n_pos && (!cos_tab || !sin_tab)) {
    set_error("plh_rope_tables: null table");
    return -1;
  }
  if (rope_ready("plh_rope_tables")) return -1;
  if (n_pos == 0) return 0;
  const Context& c = ctx();
  a.cos_t = cos_tab, a.sin_t = sin_tab;
  a.n = (uint32_t)n_pos * (uint32_t)a.pairs;
  a.first = first_pos;
  a.fd_pairs = make_fastdiv((uint32_t)a.pairs);
  const uint32_t need = (a.n + 255) / 256, most = (uint32_t)c.num_cus * 16;
  hipLaunchKernelGGL(rope_tables_kernel, dim3(need < most ? need : most), dim3(256), 0, c.stream,
                     a);
  return check_hip(hipGetLastError(), "rope_tables_kernel");
}

int plh_rope_rows(const plh_rope* rope, int n_rows, const int32_t* pos, int head_dim,
                  const float* q, int n_heads, int q_stride, float* q_out, int q_out_stride,
                  const float* k, int n_kv_heads, int k_stride, float* k_out, int k_out_stride) {
  if (!rope || head_dim < 2 || (head_dim & 1) || head_dim > 256) {
    set_error("plh_rope_rows: no tables, or head_dim %d (even, 2..256)", head_dim);
    return -1;
  }
  if (check_rope(rope, head_dim, "plh_rope_rows")) return -1;
  if (n_rows < 0 || n_heads < 0 || n_kv_heads < 0 ||
      (int64_t)n_heads * head_dim > (n_heads ? q_stride : 0) ||
      (int64_t)n_heads * head_dim > (n_heads ? q_out_stride : 0) ||
      (int64_t)n_kv_heads * head_dim > (n_kv_heads ? k_stride : 0) ||
      (int64_t)n_kv_heads * head_dim > (n_kv_heads ? k_out_stride : 0)) {
    set_error("plh_rope_rows: %d rows of %d and %d heads of %d: a stride is too small", n_rows,
              n_heads, n_kv_heads, head_dim);
    return -1;
  }
  const bool any = n_rows && (n_heads || n_kv_heads);
  if (any && (!pos || (n_heads && (!q || !q_out)) || (n_kv_heads && (!k || !k_out)))) {
    set_error("plh_rope_rows: null pointer");
    return -1;
  }
  if (((int64_t)n_heads + n_kv_heads) * head_dim > INT_MAX / 2) {
    set_error("plh_rope_rows: %d and %d heads are too many", n_heads, n_kv_heads);
    return -1;
  }
  const RopeRows a = rope_rows_args(rope, head_dim, q, n_heads, q_stride, q_out, q_out_stride, k,
                                    n_kv_heads, k_stride, k_out, k_out_stride);
  if ((int64_t)n_rows * a.chunks > kMaxWorkgroups) {
    set_error("plh_rope_rows: %d rows are too many for one call", n_rows);
    return -1;
  }
  if (rope_ready("plh_rope_rows")) return -1;
  if (!any) return 0;
  const dim3 grid((unsigned)n_rows * (unsigned)a.chunks), block(kRopeThreads);
  if (a.qwen)
    hipLaunchKernelGGL(rope_rows_kernel<true>, grid, block, 0, ctx().stream, a, pos);
  else
    hipLaunchKernelGGL(rope_rows_kernel<false>, grid, block, 0, ctx().stream, a, pos);
  return check_hip(hipGetLastError(), "rope_rows_kernel");
}

}  // extern "C"
