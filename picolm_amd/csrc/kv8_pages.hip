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
constexpr int kSmallTable = 8 * kPlanThreads;  // entries

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
  FastDiv fd_page; // page_tokens
};

// A workgroup copies kCopyChunk bytes of codes at a time, kCopyLoads loads in
// flight a thread.  Its stores pass L2 by: 16 copied pages of 704 KB take 12.5
// us with their plan (13.4 through L2), 231 MB of moves 51 us (56; 4.5 TB/s,
// what a large copy reaches).  One load a thread measures the same, eight 2%
// more.
constexpr int kCopyLoads = 4;
constexpr int kCopyChunk = kCopyLoads * 16 * kKvThreads;
typedef uint32_t Vec16 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int seq_len(const PageArgs& a, int s) {
  return min(max(a.len[s], 0), a.max_pages * a.page_tokens);
}
__device__ __forceinline__ int pages_of(const PageArgs& a, int n) {
  return (int)fdiv((uint32_t)(n + a.page_tokens - 1), a.fd_page);
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

// Both in one workgroup, for tables of few entries: one launch.
__global__ __launch_bounds__(kPlanThreads) void kv8_fork_small_kernel(PageArgs a) {
  const int entries = a.n_seqs * a.max_pages;
  for (int i = (int)threadIdx.x; i < entries; i += kPlanThreads) {
    const int s = i / a.max_pages, e = i - s * a.max_pages, parent = parent_of(a, s);
    if (parent < 0) continue;
    const int old = a.table[i], p = a.table[(size_t)parent * a.max_pages + e];
    const int len = seq_len(a, parent), n = pages_of(a, len), had = pages_of(a, seq_len(a, s));
    if (e < had && in_cache(a, old)) atomicSub(a.refs + old, 1);
    if (e < n && in_cache(a, p)) atomicAdd(a.refs + p, 1);
    a.spare[i] = e < n ? p : e < had ? -1 : old;
    if (e == 0) a.spare[entries + s] = len;
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < entries; i += kPlanThreads) {
    const int s = i / a.max_pages;
    if (parent_of(a, s) < 0) continue;
    a.table[i] = a.spare[i];
    if (i == s * a.max_pages) a.len[s] = a.spare[entries + s];
  }
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

constexpr int kListed = 4096;  // free pages kept in LDS; more go to the workspace

// extend: a thread per sequence finds what it needs, all of them walk refs
// for the free pages of the lowest numbers until there are enough, and if so
// hand them out (5.1 us for 18 sequences).  One workgroup: the walk is 16 KB a
// step and ends early; a pool of 64 K pages with its free ones last takes 16
// steps.  Few sequences on few pages (a decode step) are four memory latencies
// and two barriers: wish, len and the first 4096 counts together; last pages;
// their counts; stores.
__global__ __launch_bounds__(kPlanThreads) void kv8_extend_kernel(PageArgs a) {
  __shared__ int32_t last[kKvMaxSeqs], at[kKvMaxSeqs], from[kKvMaxSeqs], to[kKvMaxSeqs];
  __shared__ int32_t list[kListed];
  __shared__ int32_t sum_lo[kPlanWaves], sum_hi[kPlanWaves], sum_copy[kPlanWaves],
      sum_free[kPlanWaves];
  __shared__ int over;
  const int s = (int)threadIdx.x, lane = s & 63, wave = s >> 6;
  const bool mine = s < a.n_seqs;
  if (s == 0) over = INT_MAX;
  const int add = mine ? max(a.wish[s], 0) : 0;
  const int len = mine ? seq_len(a, s) : 0;
  int count4[4];  // counts of the step's pages 4 s .. 4 s + 3
#pragma unroll
  for (int k = 0; k < 4; ++k) count4[k] = 4 * s + k < a.n_pages ? a.refs[4 * s + k] : 1;
  const int full = (int)fdiv((uint32_t)len, a.fd_page), in_last = len - full * a.page_tokens;
  const int have = full + (in_last > 0);
  const int64_t want64 = ((int64_t)len + add + a.page_tokens - 1) / a.page_tokens;
  int tail = -1;
  if (add > 0 && in_last) {
    tail = a.table[(size_t)s * a.max_pages + full];
    if (!in_cache(a, tail)) tail = -1;
  }
  const int sharers = tail >= 0 ? a.refs[tail] : 0;
  last[s] = tail;
  __syncthreads();
  if (add > 0 && want64 > a.max_pages) atomicMin(&over, s);
  // the earlier sharers of this last page leave it to the later ones
  int before = 0;
  if (sharers > 1)
    for (int j = 0; j < s; ++j) before += last[j] == tail;
  const int copies = sharers - before > 1;
  const int64_t count = (add > 0 ? want64 - have : 0) + copies;
  // sums over the sequences in two halves of 16 and more bits (counts are below
  // 2^26), and over the first step's free pages
  int n_free = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) n_free += count4[k] == 0;
  const int c_lo = (int)(count & 0xFFFF), c_hi = (int)(min(count, (int64_t)1 << 36) >> 16);
  int lo = wave_sums(c_lo), hi = wave_sums(c_hi), cp = wave_sums(copies), fr = wave_sums(n_free);
  if (lane == 63) sum_lo[wave] = lo, sum_hi[wave] = hi, sum_copy[wave] = cp, sum_free[wave] = fr;
  __syncthreads();
  int64_t total = 0, first = 0;
  int n_copies = 0, copy_at = 0, rank = 0, found = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const int64_t x = ((int64_t)sum_hi[w] << 16) + sum_lo[w];
    first += w < wave ? x : 0, total += x;
    copy_at += w < wave ? sum_copy[w] : 0, n_copies += sum_copy[w];
    rank += w < wave ? sum_free[w] : 0, found += sum_free[w];
  }
  first += ((int64_t)(hi - c_hi) << 16) + (lo - c_lo);
  copy_at += cp - copies, rank += fr - n_free;
  const int first_over = over;
  auto keep = [&](int p0) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (count4[k] == 0) {
        if (rank < total) (rank < kListed ? list : a.spare)[rank] = p0 + k;
        ++rank;
      }
  };
  if (first_over == INT_MAX) {
    keep(4 * s);
    for (int base = 4 * kPlanThreads; base < a.n_pages && found < total;
         base += 4 * kPlanThreads) {
      const int p0 = base + 4 * s;
      n_free = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        count4[k] = p0 + k < a.n_pages ? a.refs[p0 + k] : 1;
        n_free += count4[k] == 0;
      }
      fr = wave_sums(n_free);
      __syncthreads();
      if (lane == 63) sum_free[wave] = fr;
      __syncthreads();
      rank = found + fr - n_free;
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        rank += w < wave ? sum_free[w] : 0;
        found += sum_free[w];
      }
      keep(p0);
    }
  }
  const bool ok = first_over == INT_MAX && found >= total;
  if (s == 0) {
    a.status[0] = first_over == INT_MAX && found < total
                      ? (int)min(total - found, (int64_t)INT_MAX)
                      : 0;
    a.status[1] = first_over == INT_MAX ? 0 : first_over + 1;
    a.head[0] = ok ? n_copies : 0;
  }
  if (!ok) return;  // the same for every thread
  at[s] = (int)(first + copies), from[s] = have, to[s] = add > 0 ? (int)want64 : have;
  __syncthreads();  // the lists are whole (this workgroup wrote them)
  auto listed = [&](int64_t n) { return n < kListed ? list[n] : a.spare[n]; };
  if (copies) {
    const int p = listed(first);
    a.table[(size_t)s * a.max_pages + full] = p;
    a.refs[p] = 1;
    atomicSub(a.refs + tail, 1);
    a.src[copy_at] = tail, a.dst[copy_at] = p;
  }
  if (add > 0) a.len[s] = len + add;
  for (int q = wave; q < a.n_seqs; q += kPlanWaves)
    for (int e = from[q] + lane; e < to[q]; e += 64) {
      const int p = listed(at[q] + (int64_t)(e - from[q]));
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
  // (page, chunk) advance by the grid's quotient and remainder
  const int step_c = (int)gridDim.x / a.chunks, step_k = (int)gridDim.x - step_c * a.chunks;
  int c = (int)blockIdx.x / a.chunks, chunk = (int)blockIdx.x - c * a.chunks;
  while (c < n) {
    const int64_t from = a.src[c], to = a.dst[c];
    const uint32_t at = (uint32_t)chunk * kCopyChunk + threadIdx.x * 16;
    const uint32_t end = (uint32_t)a.page_codes;
    const int8_t* x = a.codes + from * a.page_codes + at;
    int8_t* y = a.codes + to * a.page_codes + at;
    Vec16 r[kCopyLoads];
#pragma unroll
    for (int k = 0; k < kCopyLoads; ++k)
      if (at + k * 16 * kKvThreads < end) r[k] = *(const Vec16*)(x + k * 16 * kKvThreads);
#pragma unroll
    for (int k = 0; k < kCopyLoads; ++k)
      if (at + k * 16 * kKvThreads < end)
        __builtin_nontemporal_store(r[k], (Vec16*)(y + k * 16 * kKvThreads));
    if (chunk == 0) {
      const float* sx = a.scales + from * a.page_scales;
      float* sy = a.scales + to * a.page_scales;
      for (int k = threadIdx.x; k < a.page_scales; k += kKvThreads) sy[k] = sx[k];
    }
    c += step_c, chunk += step_k;
    if (chunk >= a.chunks) chunk -= a.chunks, ++c;
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
  a.fd_page = make_fastdiv((uint32_t)c->page_tokens);
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
  // enough workgroups for every CU to have eight, or one an item
  const int64_t items = most * a.chunks, full = 8ll * ctx().num_cus;
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
  if ((int64_t)a.n_seqs * a.max_pages <= kSmallTable) {
    hipLaunchKernelGGL(kv8_fork_small_kernel, dim3(1), dim3(kPlanThreads), 0, ctx().stream, a);
    return check_hip(hipGetLastError(), "kv8_fork_small_kernel");
  }
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
