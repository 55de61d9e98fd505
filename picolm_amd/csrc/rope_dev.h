// rope_dev.h -- rotation of q and k rows by cos / sin tables, shared by
// plh_rope_rows and the cache append (which rotates q on the way).
//
// A pair (x0, x1) becomes (x0 c - x1 s, x0 s + x1 c).  The products of two
// fp32 values are exact in 64 bits, so each output is the exact rotation by
// the table's entries up to one 64-bit and one fp32 rounding: 4 multiply-adds
// and 4 conversions a pair, which the memory traffic (16 bytes a pair) hides.
#pragma once

#include "picolm_hip.h"
#include "plh_internal.h"

namespace plh {

constexpr int kRopeThreads = 256;
constexpr int kMaxWorkgroups = (1 << 24) - 1;  // of 256 threads: a launch is below 2^32 threads

struct RopeRows {
  const float *cos_t, *sin_t;
  const float *q, *k;
  float *q_out, *k_out;
  int q_stride, k_stride, q_out_stride, k_out_stride;
  int n_heads;          // q heads; kv heads follow them in a row's items
  int D, rot, n_pos, qwen;
  int vec;              // items of four floats (else of one pair, or one plain element)
  int pairs, per_head;  // items of a head: rotated ones, then plain ones
  int per_row, chunks;  // items and workgroups of a row
  FastDiv fd_head, fd_chunk;
};

// 0, or -1 with the message set.
int check_rope(const plh_rope* r, int head_dim, const char* what);
RopeRows rope_rows_args(const plh_rope* r, int head_dim, const float* q, int n_heads, int q_stride,
                        float* q_out, int q_out_stride, const float* k, int n_kv_heads,
                        int k_stride, float* k_out, int k_out_stride);

__device__ __forceinline__ void rotate_pair(float& x0, float& x1, float c, float s) {
  const double a = x0, b = x1, cd = c, sd = s;
  x0 = (float)__builtin_fma(a, cd, -(b * sd));
  x1 = (float)__builtin_fma(a, sd, b * cd);
}

// One item of a row: loaded before its position is known, then turned and
// stored.  Positions outside the tables rotate by NaN.
struct RopeItem {
  float* y;
  int i;       // number in its head
  float4 x0, x1;
};
template <bool QWEN>
__device__ __forceinline__ RopeItem rope_load(const RopeRows& a, int64_t row, int item) {
  RopeItem it;
  int head = (int)fdiv((uint32_t)item, a.fd_head);
  it.i = item - head * a.per_head;
  const bool is_q = head < a.n_heads;
  head -= is_q ? 0 : a.n_heads;
  const float* x = (is_q ? a.q + row * a.q_stride : a.k + row * a.k_stride) + (int64_t)head * a.D;
  it.y = (is_q ? a.q_out + row * a.q_out_stride : a.k_out + row * a.k_out_stride) +
         (int64_t)head * a.D;
  it.x0 = it.x1 = make_float4(0.f, 0.f, 0.f, 0.f);
  const int i = it.i;
  if (i >= a.pairs) {  // behind the rotated part
    const int d = a.rot + (i - a.pairs) * (a.vec ? 4 : 1);
    if (a.vec)
      it.x0 = *(const float4*)(x + d);
    else
      it.x0.x = x[d];
  } else if (!a.vec) {
    it.x0.x = x[QWEN ? i : 2 * i];
    it.x1.x = x[QWEN ? i + a.rot / 2 : 2 * i + 1];
  } else if (QWEN) {
    it.x0 = *(const float4*)(x + 4 * i), it.x1 = *(const float4*)(x + 4 * i + a.rot / 2);
  } else {
    it.x0 = *(const float4*)(x + 4 * i);
  }
  return it;
}
template <bool QWEN>
__device__ __forceinline__ void rope_store(const RopeRows& a, RopeItem it, int pos) {
  const int i = it.i;
  float* y = it.y;
  const bool known = pos >= 0 && pos < a.n_pos;
  const int64_t tab = (int64_t)(known ? pos : 0) * (a.rot / 2);
  const float nan = __builtin_nanf("");
  if (i >= a.pairs) {
    const int d = a.rot + (i - a.pairs) * (a.vec ? 4 : 1);
    if (a.vec)
      *(float4*)(y + d) = it.x0;
    else
      y[d] = it.x0.x;
  } else if (!a.vec) {
    rotate_pair(it.x0.x, it.x1.x, known ? a.cos_t[tab + i] : nan, known ? a.sin_t[tab + i] : nan);
    y[QWEN ? i : 2 * i] = it.x0.x;
    y[QWEN ? i + a.rot / 2 : 2 * i + 1] = it.x1.x;
  } else if (QWEN) {
    float4 c = *(const float4*)(a.cos_t + tab + 4 * i), s = *(const float4*)(a.sin_t + tab + 4 * i);
    if (!known) c = s = make_float4(nan, nan, nan, nan);
    rotate_pair(it.x0.x, it.x1.x, c.x, s.x);
    rotate_pair(it.x0.y, it.x1.y, c.y, s.y);
    rotate_pair(it.x0.z, it.x1.z, c.z, s.z);
    rotate_pair(it.x0.w, it.x1.w, c.w, s.w);
    *(float4*)(y + 4 * i) = it.x0, *(float4*)(y + 4 * i + a.rot / 2) = it.x1;
  } else {
    float2 c = *(const float2*)(a.cos_t + tab + 2 * i), s = *(const float2*)(a.sin_t + tab + 2 * i);
    if (!known) c = s = make_float2(nan, nan);
    rotate_pair(it.x0.x, it.x0.y, c.x, s.x);
    rotate_pair(it.x0.z, it.x0.w, c.y, s.y);
    *(float4*)(y + 4 * i) = it.x0;
  }
}

}  // namespace plh
