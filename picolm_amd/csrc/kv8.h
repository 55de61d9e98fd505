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

// Slots.  The blocks that a batch's rows touch are numbered without a scan:
// sequence s has the slots from row_start[s]/32 + 2 s on, at least as many as
// its m rows can touch ((m + 30)/32 + 1 rounded down), and slot i of them is its
// i-th touched block.  Slots without a block do nothing.
inline int64_t kv_slots(int n_rows, int n_seqs) { return n_rows / kKvBlock + 2ll * n_seqs; }

// Sequence of a slot (n_seqs: none); every thread of the workgroup calls it.
__device__ __forceinline__ int kv_seq_of_slot(const KvView& v, int slot) {
  int s = 0;
  for (int at = 0; at < v.n_seqs; at += kKvThreads) {
    const int i = at + (int)threadIdx.x;
    s += __syncthreads_count(
        i < v.n_seqs && min(max(v.row_start[i + 1], 0), v.n_rows) / kKvBlock + 2 * (i + 1) <= slot);
  }
  return s;
}
__device__ __forceinline__ int kv_first_slot(const KvView& v, int s) {
  return min(max(v.row_start[s], 0), v.n_rows) / kKvBlock + 2 * s;
}
// Sequence of a row, likewise.
__device__ __forceinline__ int kv_seq_of_row(const KvView& v, int row) {
  int s = 0;
  for (int at = 0; at < v.n_seqs; at += kKvThreads) {
    const int i = at + (int)threadIdx.x;
    s += __syncthreads_count(i < v.n_seqs && v.row_start[i + 1] <= row);
  }
  return s;
}

}  // namespace plh
