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

// Chunk `chunk` of row `row`'s items, one per thread.  Positions outside the
// tables rotate by NaN.
__device__ __forceinline__ void rope_row_items(const RopeRows& a, int row, int chunk, int pos) {
  const int item = chunk * kRopeThreads + (int)threadIdx.x;
  if (item >= a.per_row) return;
  int head = (int)fdiv((uint32_t)item, a.fd_head);
  const int i = item - head * a.per_head;
  const bool is_q = head < a.n_heads;
  head -= is_q ? 0 : a.n_heads;
  const float* x = (is_q ? a.q + (size_t)row * a.q_stride : a.k + (size_t)row * a.k_stride) +
                   (size_t)head * a.D;
  float* y = (is_q ? a.q_out + (size_t)row * a.q_out_stride
                   : a.k_out + (size_t)row * a.k_out_stride) +
             (size_t)head * a.D;
  const bool known = pos >= 0 && pos < a.n_pos;
  const size_t tab = (size_t)(known ? pos : 0) * (a.rot / 2);
  const float nan = __builtin_nanf("");
  if (i >= a.pairs) {  // behind the rotated part
    const int d = a.rot + (i - a.pairs) * (a.vec ? 4 : 1);
    if (a.vec)
      *(float4*)(y + d) = *(const float4*)(x + d);
    else
      y[d] = x[d];
  } else if (!a.vec) {
    const int d0 = a.qwen ? i : 2 * i, d1 = a.qwen ? i + a.rot / 2 : 2 * i + 1;
    float x0 = x[d0], x1 = x[d1];
    rotate_pair(x0, x1, known ? a.cos_t[tab + i] : nan, known ? a.sin_t[tab + i] : nan);
    y[d0] = x0, y[d1] = x1;
  } else if (a.qwen) {
    const int d0 = 4 * i, d1 = 4 * i + a.rot / 2;
    float4 x0 = *(const float4*)(x + d0), x1 = *(const float4*)(x + d1);
    float4 c = *(const float4*)(a.cos_t + tab + d0), s = *(const float4*)(a.sin_t + tab + d0);
    if (!known) c = s = make_float4(nan, nan, nan, nan);
    rotate_pair(x0.x, x1.x, c.x, s.x);
    rotate_pair(x0.y, x1.y, c.y, s.y);
    rotate_pair(x0.z, x1.z, c.z, s.z);
    rotate_pair(x0.w, x1.w, c.w, s.w);
    *(float4*)(y + d0) = x0, *(float4*)(y + d1) = x1;
  } else {
    float4 x0 = *(const float4*)(x + 4 * i);
    float2 c = *(const float2*)(a.cos_t + tab + 2 * i), s = *(const float2*)(a.sin_t + tab + 2 * i);
    if (!known) c = s = make_float2(nan, nan);
    rotate_pair(x0.x, x0.y, c.x, s.x);
    rotate_pair(x0.z, x0.w, c.y, s.y);
    *(float4*)(y + 4 * i) = x0;
  }
}

}  // namespace plh
