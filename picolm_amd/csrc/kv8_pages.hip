// kv8_pages.hip -- page operations of the paged 8-bit cache: freeing, sharing,
// allocating with copies on write, compacting (include/picolm_hip.h,
// plh_kv8_trim / _fork / _extend / _compact).
//
// The pages' bookkeeping stays on the device, so a decode loop needs no round
// trip to the host.  It is integers and small: what an operation costs is a
// launch or two, and where pages move, their copy (HBM; a page's codes and
// scales are one run of bytes each).
#include <limits.h>

#include "kv8.h"

namespace plh {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PageArgs {
  int8_t* codes;
  float* scales;
  int64_t page_codes, page_scales;  // bytes, floats
  int page_tokens, n_pages, n_seqs, max_pages;
  int32_t *table, *len, *refs;
  const int32_t* wish;  // keep, parent or add
  int32_t* status;
  // workspace
  int32_t* head;   // [0]: copies
  int32_t* src;    // copied pages
  int32_t* dst;
  int32_t* spare;  // free page numbers; compact: where a page goes; fork: the parents' rows
  int chunks;      // of a copied page
};

constexpr int kCopyChunk = 64 * 1024;  // bytes of codes a workgroup copies at a time

__device__ __forceinline__ int seq_len(const PageArgs& a, int s) {
  return min(max(a.len[s], 0), a.max_pages * a.page_tokens);
}
__device__ __forceinline__ int pages_of(const PageArgs& a, int n) {
  return (n + a.page_tokens - 1) / a.page_tokens;
}
__device__ __forceinline__ bool in_cache(const PageArgs& a, int page) {
  return page >= 0 && page < a.n_pages;
}

// A workgroup per sequence: pages behind the kept tokens are counted down.
__global__ __launch_bounds__(kKvThreads) void kv8_trim_kernel(PageArgs a) {
  const int s = blockIdx.x, keep = a.wish[s], len = seq_len(a, s);
  if (keep < 0 || keep >= len) return;
  int32_t* row = a.table + (size_t)s * a.max_pages;
  const int end = pages_of(a, len);
  for (int e = pages_of(a, keep) + (int)threadIdx.x; e < end; e += kKvThreads) {
    const int p = row[e];
    if (in_cache(a, p)) atomicSub(a.refs + p, 1);
    row[e] = -1;
  }
  __syncthreads();  // len is read before it changes
  if (threadIdx.x == 0) a.len[s] = keep;
}

__device__ __forceinline__ int parent_of(const PageArgs& a, int s) {
  const int p = a.wish[s];
  return p >= 0 && p < a.n_seqs && p != s ? p : -1;
}

// fork, first launch: what every sequence is to become goes to the workspace
// (a parent's own row may change in the second) and the pages are counted.
__global__ __launch_bounds__(kKvThreads) void kv8_fork_count_kernel(PageArgs a) {
  const int s = blockIdx.x, parent = parent_of(a, s);
  if (parent < 0) return;
  const int32_t *own = a.table + (size_t)s * a.max_pages,
                *row = a.table + (size_t)parent * a.max_pages;
  int32_t* kept = a.spare + (size_t)s * (a.max_pages + 1);
  const int len = seq_len(a, parent), n = pages_of(a, len), had = pages_of(a, seq_len(a, s));
  for (int e = (int)threadIdx.x; e < max(n, had); e += kKvThreads) {
    if (e < had && in_cache(a, own[e])) atomicSub(a.refs + own[e], 1);
    if (e < n) {
      const int p = row[e];
      if (in_cache(a, p)) atomicAdd(a.refs + p, 1);
      kept[1 + e] = p;
    }
  }
  if (threadIdx.x == 0) kept[0] = len;
}
__global__ __launch_bounds__(kKvThreads) void kv8_fork_write_kernel(PageArgs a) {
  const int s = blockIdx.x;
  if (parent_of(a, s) < 0) return;
  int32_t* own = a.table + (size_t)s * a.max_pages;
  const int32_t* kept = a.spare + (size_t)s * (a.max_pages + 1);
  const int len = kept[0], n = pages_of(a, len), had = pages_of(a, seq_len(a, s));
  for (int e = (int)threadIdx.x; e < max(n, had); e += kKvThreads)
    own[e] = e < n ? kept[1 + e] : -1;
  __syncthreads();
  if (threadIdx.x == 0) a.len[s] = len;
}

// Sum of the earlier threads' x (of a workgroup of kPlanThreads) and of all.
// part: kPlanWaves + 1 values of LDS, free again once every thread returned.
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
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + sum - x;
}

// extend: a thread per sequence finds what it needs, all of them walk refs
// for the free pages of the lowest numbers until there are enough, and if so
// hand them out.  One workgroup: the walk is 16 KB a step and ends early; a
// pool of 64 K pages with its free ones last takes 16 steps.
__global__ __launch_bounds__(kPlanThreads) void kv8_extend_kernel(PageArgs a) {
  __shared__ int32_t last[kKvMaxSeqs], at[kKvMaxSeqs], from[kKvMaxSeqs], to[kKvMaxSeqs];
  __shared__ int64_t part[kPlanWaves];
  __shared__ int over;
  const int s = (int)threadIdx.x, lane = s & 63, wave = s >> 6;
  const bool mine = s < a.n_seqs;
  const int add = mine ? max(a.wish[s], 0) : 0;
  const int len = mine ? seq_len(a, s) : 0;
  const int have = pages_of(a, len);
  const int64_t want64 = ((int64_t)len + add + a.page_tokens - 1) / a.page_tokens;
  const int32_t* row = a.table + (size_t)(mine ? s : 0) * a.max_pages;
  int tail = -1;
  if (add > 0 && len % a.page_tokens) {
    tail = row[len / a.page_tokens];
    if (!in_cache(a, tail)) tail = -1;
  }
  last[s] = tail;
  if (s == 0) over = INT_MAX;
  __syncthreads();
  if (want64 > a.max_pages && add > 0) atomicMin(&over, s);
  // the earlier sharers of this last page leave it to the later ones
  int before = 0;
  if (tail >= 0)
    for (int j = 0; j < s; ++j) before += last[j] == tail;
  const int copies = tail >= 0 && a.refs[tail] - before > 1;
  const int64_t count = (add > 0 ? want64 - have : 0) + copies;
  int64_t total, n_copies;
  const int64_t first = plan_scan(count, part, total);
  const int64_t copy_at = plan_scan(copies, part, n_copies);
  const int first_over = over;  // written before the scans' barriers
  int64_t found = 0;
  if (first_over == INT_MAX)
    for (int base = 0; base < a.n_pages && found < total; base += 4 * kPlanThreads) {
      const int p0 = base + 4 * s;
      int free4[4], n = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        free4[k] = p0 + k < a.n_pages && a.refs[p0 + k] == 0;
        n += free4[k];
      }
      int64_t all;
      int64_t rank = found + plan_scan(n, part, all);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (free4[k]) {
          if (rank < total) a.spare[rank] = p0 + k;
          ++rank;
        }
      found += all;
    }
  const bool ok = first_over == INT_MAX && found >= total;
  if (s == 0) {
    a.status[0] = first_over == INT_MAX && found < total
                      ? (int)(total - found < INT_MAX ? total - found : INT_MAX)
                      : 0;
    a.status[1] = first_over == INT_MAX ? 0 : first_over + 1;
    a.head[0] = ok ? (int)n_copies : 0;
  }
  if (!ok) return;  // the same for every thread
  const int want = (int)want64;
  at[s] = (int)(first + copies), from[s] = have, to[s] = add > 0 ? want : have;
  __syncthreads();  // spare and the LDS are whole (this workgroup wrote them)
  if (copies) {
    const int p = a.spare[first];
    a.table[(size_t)s * a.max_pages + len / a.page_tokens] = p;
    a.refs[p] = 1;
    atomicSub(a.refs + tail, 1);
    a.src[copy_at] = tail, a.dst[copy_at] = p;
  }
  if (add > 0) a.len[s] = len + add;
  for (int q = wave; q < a.n_seqs; q += kPlanWaves)
    for (int e = from[q] + lane; e < to[q]; e += 64) {
      const int p = a.spare[at[q] + e - from[q]];
      a.table[(size_t)q * a.max_pages + e] = p;
      a.refs[p] = 1;
    }
}

// compact: counts the live pages, lists the places below that count which are
// free and the pages from it on which are live, pairs them in order.
__global__ __launch_bounds__(kPlanThreads) void kv8_compact_kernel(PageArgs a) {
  __shared__ int64_t part[kPlanWaves];
  const int s = (int)threadIdx.x;
  int n = 0;
  for (int p = s; p < a.n_pages; p += kPlanThreads) n += a.refs[p] > 0;
  int64_t live, all;
  plan_scan(n, part, live);
  int64_t holes = 0, moves = 0;
  for (int base = 0; base < a.n_pages; base += 4 * kPlanThreads) {
    const int p0 = base + 4 * s;
    int used[4], nh = 0, nm = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = p0 + k < a.n_pages;
      used[k] = in && a.refs[p0 + k] > 0;
      nh += in && !used[k] && p0 + k < live;
      nm += used[k] && p0 + k >= live;
    }
    const int64_t ranks = plan_scan((int64_t)nh << 32 | nm, part, all);
    int64_t hole = holes + (ranks >> 32), move = moves + (ranks & 0xFFFFFFFF);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p0 + k >= a.n_pages) continue;
      if (p0 + k < live) {
        if (!used[k]) a.dst[hole++] = p0 + k;
      } else if (used[k]) {
        a.src[move++] = p0 + k;
      } else {
        a.spare[p0 + k] = -1;
      }
    }
    holes += all >> 32, moves += all & 0xFFFFFFFF;
  }
  __syncthreads();  // src and dst are whole (this workgroup wrote them)
  for (int i = s; i < moves; i += kPlanThreads) {
    const int p = a.src[i], q = a.dst[i];
    a.spare[p] = q;
    a.refs[q] = a.refs[p];
    a.refs[p] = 0;
  }
  if (s == 0) {
    a.head[0] = (int)moves, a.head[1] = (int)live;
    a.status[0] = (int)live, a.status[1] = (int)moves;
  }
}

// The listed pages' codes and scales, workgroups striding over (page, chunk);
// compact also follows the moves in the table.
__global__ __launch_bounds__(kKvThreads) void kv8_copy_kernel(PageArgs a, int remap) {
  const int n = a.head[0];
  const int64_t items = (int64_t)n * a.chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int c = (int)(item / a.chunks), chunk = (int)(item - (int64_t)c * a.chunks);
    const int64_t from = a.src[c], to = a.dst[c];
    const uint4* x = (const uint4*)(a.codes + from * a.page_codes);
    uint4* y = (uint4*)(a.codes + to * a.page_codes);
    const int end = min((chunk + 1) * (kCopyChunk / 16), (int)(a.page_codes / 16));
    int i = chunk * (kCopyChunk / 16) + (int)threadIdx.x;
    // eight loads in flight a thread
    for (; i + 7 * kKvThreads < end; i += 8 * kKvThreads) {
      uint4 r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = x[i + k * kKvThreads];
#pragma unroll
      for (int k = 0; k < 8; ++k) y[i + k * kKvThreads] = r[k];
    }
    for (; i < end; i += kKvThreads) y[i] = x[i];
    if (chunk == 0) {
      const float* sx = a.scales + from * a.page_scales;
      float* sy = a.scales + to * a.page_scales;
      for (int k = threadIdx.x; k < a.page_scales; k += kKvThreads) sy[k] = sx[k];
    }
  }
  if (!remap || n == 0) return;
  const int live = a.head[1];
  const int64_t entries = (int64_t)a.n_seqs * a.max_pages;
  for (int64_t e = (int64_t)blockIdx.x * kKvThreads + threadIdx.x; e < entries;
       e += (int64_t)gridDim.x * kKvThreads) {
    const int p = a.table[e];
    if (p >= live && p < a.n_pages && a.spare[p] >= 0) a.table[e] = a.spare[p];
  }
}

// Checks and the arguments; the workspace holds the copy list and `spare`
// values behind it.
int page_args(const plh_kv8_cache* c, const plh_kv8_seqs* s, const int32_t* wish, int32_t* status,
              bool has_wish, bool has_status, int copies, size_t spare, const char* what,
              PageArgs& a) {
  if (kv_check(c, s, what)) return -1;
  if ((has_wish && !wish) || (has_status && !status)) {
    set_error("%s: null pointer", what);
    return -1;
  }
  if (kv_ready(what)) return -1;
  a = PageArgs{};
  a.codes = c->codes, a.scales = c->scales;
  a.page_codes = (int64_t)(plh_kv8_code_bytes(c) / (size_t)c->n_pages);
  a.page_scales = (int64_t)(plh_kv8_scale_bytes(c) / (size_t)c->n_pages / sizeof(float));
  a.page_tokens = c->page_tokens, a.n_pages = c->n_pages;
  a.n_seqs = s->n_seqs, a.max_pages = s->max_pages;
  a.table = s->table, a.len = s->len, a.refs = s->refs;
  a.wish = wish, a.status = status;
  a.chunks = (int)((a.page_codes + kCopyChunk - 1) / kCopyChunk);
  const size_t words = 4 + 2 * (size_t)copies + spare;
  if (words > 4 && ensure_workspace(words * sizeof(int32_t))) return -1;
  a.head = (int32_t*)ctx().ws;
  a.src = a.head + 4, a.dst = a.src + copies, a.spare = a.dst + copies;
  return 0;
}

int launch_copies(const PageArgs& a, int64_t most, int remap) {
  // enough workgroups for every CU to have four, or one an item
  const int64_t items = most * a.chunks, full = 4ll * ctx().num_cus;
  hipLaunchKernelGGL(kv8_copy_kernel, dim3((unsigned)(items < full ? items : full)),
                     dim3(kKvThreads), 0, ctx().stream, a, remap);
  return check_hip(hipGetLastError(), "kv8_copy_kernel");
}

}  // namespace
}  // namespace plh

using namespace plh;

extern "C" {

int plh_kv8_trim(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, const int32_t* keep) {
  PageArgs a;
  if (page_args(cache, seqs, keep, nullptr, true, false, 0, 0, "plh_kv8_trim", a)) return -1;
  hipLaunchKernelGGL(kv8_trim_kernel, dim3((unsigned)a.n_seqs), dim3(kKvThreads), 0, ctx().stream,
                     a);
  return check_hip(hipGetLastError(), "kv8_trim_kernel");
}

int plh_kv8_fork(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, const int32_t* parent) {
  PageArgs a;
  const size_t rows = seqs ? (size_t)(seqs->n_seqs > 0 ? seqs->n_seqs : 0) *
                                 (size_t)(seqs->max_pages > 0 ? seqs->max_pages + 1ll : 0)
                           : 0;
  if (page_args(cache, seqs, parent, nullptr, true, false, 0, rows, "plh_kv8_fork", a)) return -1;
  hipLaunchKernelGGL(kv8_fork_count_kernel, dim3((unsigned)a.n_seqs), dim3(kKvThreads), 0,
                     ctx().stream, a);
  hipLaunchKernelGGL(kv8_fork_write_kernel, dim3((unsigned)a.n_seqs), dim3(kKvThreads), 0,
                     ctx().stream, a);
  return check_hip(hipGetLastError(), "kv8_fork_kernel");
}

int plh_kv8_extend(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, const int32_t* add,
                   int32_t* status) {
  PageArgs a;
  const size_t pages = cache && cache->n_pages > 0 ? (size_t)cache->n_pages : 0;
  if (page_args(cache, seqs, add, status, true, true, kKvMaxSeqs, pages, "plh_kv8_extend", a))
    return -1;
  hipLaunchKernelGGL(kv8_extend_kernel, dim3(1), dim3(kPlanThreads), 0, ctx().stream, a);
  if (check_hip(hipGetLastError(), "kv8_extend_kernel")) return -1;
  return launch_copies(a, a.n_seqs, 0);
}

int plh_kv8_compact(const plh_kv8_cache* cache, const plh_kv8_seqs* seqs, int32_t* status) {
  PageArgs a;
  const int pages = cache && cache->n_pages > 0 ? cache->n_pages : 0;
  if (page_args(cache, seqs, nullptr, status, false, true, pages, (size_t)pages,
                "plh_kv8_compact", a))
    return -1;
  hipLaunchKernelGGL(kv8_compact_kernel, dim3(1), dim3(kPlanThreads), 0, ctx().stream, a);
  if (check_hip(hipGetLastError(), "kv8_compact_kernel")) return -1;
  return launch_copies(a, a.n_pages, 1);
}

}  // extern "C"
