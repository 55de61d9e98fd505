// kv8.h -- the paged 8-bit cache as its kernels see it (layout and meaning:
// include/picolm_hip.h, plh_kv8_*).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "picolm_hip.h"
#include "plh_internal.h"
#include "rope_dev.h"

namespace plh {

constexpr int kKvBlock = 32;     // tokens of a block
constexpr int kKvTile = 1024;    // codes of a tile: 32 tokens x 32 elements
constexpr int kKvMaxSeqs = 1024;
constexpr int kKvThreads = 256;

// One layer of a cache and the rows of a batch.
struct KvView {
  int8_t* codes;     // of the layer, page 0
  float* scales;
  int64_t page_codes, page_scales;  // bytes, floats from page to page
  int n_kv_heads, D, blocks;        // blocks of a page
  int n_pages, n_seqs, max_pages;
  const int32_t *table, *len, *refs, *row_start;
  int n_rows;
  FastDiv fd_blocks;
};

inline int kv_tiles(int head_dim) { return (head_dim + 31) / 32; }

// The checks every call shares; 0 or -1 with the message set.
int kv_check(const plh_kv8_cache* c, const plh_kv8_seqs* s, const char* what);
int kv_ready(const char* what);  // the library is initialised; last of the checks
// ... and of a batch over a layer; -1, or 0 with the view filled.
int kv_view(const plh_kv8_cache* c, const plh_kv8_seqs* s, int layer, int n_rows,
            const int32_t* row_start, const char* what, KvView& v);

// Rows of sequence s: the first and how many (any row_start keeps them inside
// the batch).
__device__ __forceinline__ void kv_rows(const KvView& v, int s, int& first, int& count) {
  const int a = min(max(v.row_start[s], 0), v.n_rows);
  const int b = min(max(v.row_start[s + 1], a), v.n_rows);
  first = a, count = b - a;
}

// Tokens of sequence s, at most what its table row holds.
__device__ __forceinline__ int kv_len(const KvView& v, int s) {
  return min(max(v.len[s], 0), v.max_pages * v.blocks * kKvBlock);
}

// Page of a sequence's block, or -1 where the table has none in the cache.
__device__ __forceinline__ int kv_page(const KvView& v, int s, int block) {
  const int e = (int)fdiv((uint32_t)block, v.fd_blocks);
  const int p = v.table[(size_t)s * v.max_pages + e];
  return p >= 0 && p < v.n_pages ? p : -1;
}

// What a wave knows of the first 64 sequences, a lane each: loaded together, so
// that finding a row's or a slot's sequence costs one memory latency.
struct KvLanes {
  int start, next, len;  // row_start[lane], row_start[lane + 1], tokens
};
__device__ __forceinline__ KvLanes kv_lanes(const KvView& v) {
  const int lane = (int)threadIdx.x & 63;
  KvLanes l{0, 0, 0};
  if (lane < v.n_seqs) {
    l.start = v.row_start[lane];
    l.next = v.row_start[lane + 1];
    l.len = v.len[lane];
  }
  return l;
}
// The number of sequences i for which before(i, row_start[i + 1]) holds: with
// row_start rising, the first sequence for which it does not (n_seqs: none).  More
// than 64: the last of each 64th part first, then the part where it ends.
template <class F>
__device__ __forceinline__ int kv_find(const KvView& v, const KvLanes& l, F before) {
  const int lane = (int)threadIdx.x & 63, n = v.n_seqs;
  if (n <= 64) return __popcll(__ballot(lane < n && before(lane, l.next)));
  const int per = (n + 63) / 64;
  int i = min((lane + 1) * per, n) - 1;
  const int at = per * __popcll(__ballot(lane * per < n && before(i, v.row_start[i + 1])));
  i = min(at + lane, n - 1);
  const bool mine = lane < per && at + lane < n;
  return min(at + (int)__popcll(__ballot(mine && before(i, v.row_start[i + 1]))), n);
}
// Rows (as kv_rows) and tokens of sequence s, from the lanes where they hold it.
struct KvSeq {
  int row0, count, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvView& v, const KvLanes& l, int s) {
  int a, b, n;
  if (s < 64) {
    a = __builtin_amdgcn_readlane(l.start, s);
    b = __builtin_amdgcn_readlane(l.next, s);
    n = __builtin_amdgcn_readlane(l.len, s);
  } else {
    a = v.row_start[s], b = v.row_start[s + 1], n = v.len[s];
  }
  a = min(max(a, 0), v.n_rows);
  b = min(max(b, a), v.n_rows);
  return KvSeq{a, b - a, min(max(n, 0), v.max_pages * v.blocks * kKvBlock)};
}
// Sums over the lanes up to each one (DPP: within rows of 16, then rows).
template <int CTRL, int ROWS>
__device__ __forceinline__ int kv_dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_sums(int x) {
  x += kv_dpp<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x += kv_dpp<0x112, 0xF>(x);
  x += kv_dpp<0x114, 0xF>(x);
  x += kv_dpp<0x118, 0xF>(x);
  x += kv_dpp<0x142, 0xA>(x);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  x += kv_dpp<0x143, 0xC>(x);
  return x;
}

// Slots: the blocks that a batch's rows touch, one after the other.  Up to 64
// sequences are counted out exactly.  With more, sequence s has the slots from
// row_start[s]/32 + 2 s on, at least as many as its m rows can touch ((m + 30)/32 + 1
// rounded down), and the slots without a block do nothing.
inline int64_t kv_slots(int n_rows, int n_seqs) {
  if (n_seqs > 64) return n_rows / kKvBlock + 2ll * n_seqs;
  const int64_t most = n_rows / kKvBlock + 2ll * n_seqs;
  return most < n_rows ? most : n_rows;
}
struct KvBlock {
  int s, block;  // sequence (-1: none) and block of it
  bool first;    // its first slot
  KvSeq q;
};
// empties: sequences whose rows all lie before position 0 have one slot too.
__device__ __forceinline__ KvBlock kv_block_of(const KvView& v, const KvLanes& l, int slot,
                                               bool empties = false) {
  KvBlock k;
  k.s = -1;
  int local;
  if (v.n_seqs <= 64) {
    const int lane = (int)threadIdx.x & 63;
    const int a = min(max(l.start, 0), v.n_rows), b = min(max(l.next, a), v.n_rows);
    const int len = min(max(l.len, 0), v.max_pages * v.blocks * kKvBlock);
    const int lo = max(len - (b - a), 0);
    int n = b > a && len > lo ? (len - 1) / kKvBlock - lo / kKvBlock + 1 : 0;
    if (empties && b > a && n == 0) n = 1;
    if (lane >= v.n_seqs) n = 0;
    const int end = wave_sums(n);
    const uint64_t hit = __ballot(slot >= end - n && slot < end);
    if (hit == 0) return k;
    k.s = __ffsll((unsigned long long)hit) - 1;
    local = slot - __builtin_amdgcn_readlane(end - n, k.s);
    k.q = kv_seq(v, l, k.s);
  } else {
    auto key = [&](int i, int start) { return min(max(start, 0), v.n_rows) / kKvBlock + 2 * i; };
    const int s = kv_find(v, l, [&](int i, int next) { return key(i + 1, next) <= slot; });
    if (s >= v.n_seqs) return k;
    k.q = kv_seq(v, l, s);
    local = slot - key(s, k.q.row0);
    const int lo = max(k.q.len - k.q.count, 0);
    if (k.q.count == 0 || (lo / kKvBlock + local) * kKvBlock >= k.q.len) {
      if (!empties || k.q.count == 0 || local) return k;
    }
    k.s = s;
  }
  k.first = local == 0;
  k.block = max(k.q.len - k.q.count, 0) / kKvBlock + local;
  return k;
}

}  // namespace plh
