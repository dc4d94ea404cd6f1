// Bookkeeping of a paged key/value cache on the device: allocation, release, forks, compaction and copies of pages.
//
// The counts and tables are small (a pool of 64 K pages has 256 KB of counts) and every decision is in order (lowest free page
// first, sequences one after the other), so one block of 1 024 threads makes them with prefix sums; what moves data or walks
// tables runs on the whole GPU in a kernel behind it. Nothing comes back to the host: a step that forks and grows its
// sequences can be captured into a graph. What counts is the number of launches, and for the copies HBM.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"

namespace sparge {

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 8;                    // pages that a thread of the plan looks at per round
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;                     // 16-byte words in flight per thread

struct PagePool {
  char* data;
  long long outer, outer_bytes, page_stride, page_bytes;
};
struct PageTable {
  int32_t *table, *lens, *refs;
  long long stride;
  int sequences, width, pages, page_size;
};

// Exclusive prefix sum over the block; every thread gets the total. s: 33 ints.
__device__ __forceinline__ int block_scan(int v, int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                               // the words of the call before are read
  if (lane == 31) s[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int t = s[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += y;
    }
    s[lane] = t;
  }
  __syncthreads();
  total = s[31];
  return x - v + (warp ? s[warp - 1] : 0);
}

__device__ __forceinline__ void load_counts(const int32_t* refs, int at, int pages, bool vec, int* c) {
  if (vec && at + kPerThread <= pages) {
#pragma unroll
    for (int i = 0; i < kPerThread; i += 4) *reinterpret_cast<int4*>(c + i) = *reinterpret_cast<const int4*>(refs + at + i);
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; i++) c[i] = at + i < pages ? refs[at + i] : -1;
  }
}

// Walks the pool in order; list gets the numbers of the pages that pick(number, count) takes, `most` of them at the most.
// Returns how many it found (a round may find more than are listed). The next round's counts travel while this one is summed.
template <typename Pick>
__device__ __forceinline__ int collect(const int32_t* refs, int pages, int most, int32_t* list, int* s, Pick pick) {
  const bool vec = reinterpret_cast<uintptr_t>(refs) % 16 == 0;
  int found = 0, c[kPerThread], n[kPerThread];
  load_counts(refs, threadIdx.x * kPerThread, pages, vec, c);
  for (int base = 0; base < pages && found < most; base += kPlanThreads * kPerThread) {
    const int at = base + threadIdx.x * kPerThread;
    if (pages - base > kPlanThreads * kPerThread) load_counts(refs, at + kPlanThreads * kPerThread, pages, vec, n);
    int mine = 0, total;
#pragma unroll
    for (int i = 0; i < kPerThread; i++) mine += at + i < pages && pick(at + i, c[i]);
    int to = found + block_scan(mine, s, total);
    if (list && mine) {
#pragma unroll
      for (int i = 0; i < kPerThread; i++)
        if (at + i < pages && pick(at + i, c[i])) {
          if (to < most) list[to] = at + i;
          to++;
        }
    }
    found += total;
#pragma unroll
    for (int i = 0; i < kPerThread; i++) c[i] = n[i];
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ int pages_of(long long tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }
__device__ __forceinline__ int held_tokens(const PageTable& t, int s) {
  return (int)max(0LL, min((long long)t.lens[s], (long long)t.width * t.page_size));
}
__device__ __forceinline__ void report_page(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// ---------------------------------------------------------------------------------------------------------- allocation
__global__ void __launch_bounds__(kPlanThreads) allocate_kernel(PageTable t, const int32_t* new_tokens, unsigned char* served,
                                                                int32_t* list, int32_t* offset, int32_t* need) {
  __shared__ int s_scan[33];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x;
  int total_need = 0;
  for (int base = 0; base < t.sequences; base += kPlanThreads) {
    const int i = base + tid;
    int want = 0;
    bool refused = false;
    if (i < t.sequences) {
      const int len = t.lens[i];
      const long long grown = (long long)len + new_tokens[i];
      refused = new_tokens[i] < 0 || len < 0 || grown > (long long)t.width * t.page_size;
      want = refused ? 0 : pages_of(grown, t.page_size) - pages_of(len, t.page_size);
    }
    int total;
    const int at = block_scan(want, s_scan, total);
    if (i < t.sequences) {
      offset[i] = min(total_need + at, 1 << 30);
      need[i] = refused ? -1 : want;
    }
    total_need = min(total_need + min(total, 1 << 29), 1 << 29);   // far above any pool: the order still decides
  }
  const int have = min(total_need, collect(t.refs, t.pages, min(total_need, t.pages), list, s_scan, [](int, int c) { return c == 0; }));
  for (int i = tid >> 5; i < t.sequences; i += kPlanThreads / 32) {
    const int want = need[i], at = offset[i], lane = tid & 31;
    const bool yes = want == 0 || (want > 0 && at + want <= have);
    if (yes) {
      const int first = pages_of(t.lens[i], t.page_size);
      for (int j = lane; j < want; j += 32) {
        const int page = list[at + j];
        t.table[i * t.stride + first + j] = page;
        t.refs[page] = 1;
      }
      __syncwarp();
      if (lane == 0) t.lens[i] += new_tokens[i];
    }
    if (lane == 0) served[i] = yes;
  }
}

// ------------------------------------------------------------------------------------------------------------- release
// Every entry is taken out by an exchange: two blocks with the same sequence release each page once.
__global__ void __launch_bounds__(256) free_kernel(PageTable t, const int32_t* which, int32_t* dev_status) {
  pdl_wait();
  pdl_trigger();
  const int s = which[blockIdx.x];
  if (s < 0 || s >= t.sequences) {
    if (s != -1 && threadIdx.x == 0) report_page(dev_status, SPARGE_DEV_BAD_PAGE);
    return;
  }
  for (int e = threadIdx.x; e < t.width; e += 256) {
    const int page = atomicExch(t.table + s * t.stride + e, -1);
    if (page >= 0 && page < t.pages) atomicSub(t.refs + page, 1);
  }
  if (threadIdx.x == 0) t.lens[s] = 0;
}

// ---------------------------------------------------------------------------------------------------------------- copies
// One warp copies 2 KB at a time; a block's warps, and the blocks, take neighbouring pieces.
template <typename PairOf>
__device__ __forceinline__ void copy_tasks(const PagePool& pool, int pairs, int block, int blocks, PairOf pair_of) {
  constexpr int kPiece = 32 * kCopyVecs * 16;
  const int lane = threadIdx.x & 31;
  const long long pieces = (pool.page_bytes + kPiece - 1) / kPiece, per_pair = pool.outer * pieces;
  const long long tasks = per_pair * pairs, step = (long long)blocks * (kCopyThreads / 32);
  for (long long task = (long long)block * (kCopyThreads / 32) + (threadIdx.x >> 5); task < tasks; task += step) {
    const int i = (int)(task / per_pair);
    const long long rest = task - i * per_pair, o = rest / pieces, piece = rest - o * pieces;
    int from, to;
    if (!pair_of(i, from, to)) continue;
    const char* src = pool.data + o * pool.outer_bytes + from * pool.page_stride + piece * kPiece;
    char* dst = pool.data + o * pool.outer_bytes + to * pool.page_stride + piece * kPiece;
    const int left = (int)min((long long)kPiece, pool.page_bytes - piece * kPiece);
    uint4 w[kCopyVecs];
#pragma unroll
    for (int j = 0; j < kCopyVecs; j++)
      if ((j * 32 + lane) * 16 < left) w[j] = reinterpret_cast<const uint4*>(src)[j * 32 + lane];
#pragma unroll
    for (int j = 0; j < kCopyVecs; j++)
      if ((j * 32 + lane) * 16 < left) reinterpret_cast<uint4*>(dst)[j * 32 + lane] = w[j];
  }
}

// A block per pair and slice of the pool, so that the search for its hazards is made once for all its copies. Pairs that copy
// nothing are nobody's hazard.
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(PagePool pool, const int32_t* src, const int32_t* dst, int n, int pages,
                                                                  int32_t* dev_status) {
  pdl_wait();
  const int i = blockIdx.x, from = src[i], to = dst[i];
  const auto inside = [=](int page) { return page >= 0 && page < pages; };
  if (!inside(from) || !inside(to)) {
    if (from != -1 && to != -1 && threadIdx.x == 0) report_page(dev_status, SPARGE_DEV_BAD_PAGE);
    return;
  }
  int clash = 0;
  for (int j = threadIdx.x; j < n; j += kCopyThreads) {
    const int a = src[j], b = dst[j];
    clash |= (j != i && b == to && inside(a)) || (a == to && b != to && inside(b));
  }
  if (__syncthreads_or(clash)) {
    if (threadIdx.x == 0) report_page(dev_status, SPARGE_DEV_PAGE_HAZARD);
    return;
  }
  if (from == to) return;
  copy_tasks(pool, 1, blockIdx.y, gridDim.y, [&](int, int& a, int& b) {
    a = from, b = to;
    return true;
  });
}

// ----------------------------------------------------------------------------------------------------------------- forks
// What becomes of pair i: 0 nothing (not served), 1 a new row, 2 a new row with a copied last page, 3 its own source.
struct ForkPlan {
  int32_t *state, *len, *at, *from, *to, *rows, *list;   // [n] each, rows [n][width], list [pages]
};

// Whether pair j (j > i) takes pair i's destination d from it: the later one has it, unless it is skipped.
__device__ __forceinline__ bool takes(const PageTable& t, const int32_t* src, const int32_t* dst, int j, int d) {
  return dst[j] == d && src[j] >= 0 && src[j] < t.sequences;
}

// Pair i by `threads` threads, of which this is number `tid`; later: whether a pair behind it has its destination.
__device__ __forceinline__ void gather_pair(const PageTable& t, int i, int s, int d, bool later, const ForkPlan& f, int tid, int threads, int32_t* dev_status) {
  const bool inside = s >= 0 && s < t.sequences && d >= 0 && d < t.sequences;
  int state = !inside || later ? 0 : s == d ? 3 : 1;
  if (!inside && s != -1 && d != -1 && tid == 0) report_page(dev_status, SPARGE_DEV_BAD_PAGE);
  if (state == 1) {
    const int len = held_tokens(t, s), used = pages_of(len, t.page_size);
    for (int e = tid; e < t.width; e += threads) f.rows[(long long)i * t.width + e] = e < used ? t.table[s * t.stride + e] : -1;
    if (len % t.page_size) {
      const int page = t.table[s * t.stride + used - 1];
      if (page >= 0 && page < t.pages) state = 2;
      if (tid == 0) f.from[i] = page, f.at[i] = used - 1;
    }
    if (tid == 0) f.len[i] = len;
  }
  if (tid == 0) f.state[i] = state;
}

__global__ void __launch_bounds__(256) fork_gather_kernel(PageTable t, const int32_t* src, const int32_t* dst, int n, ForkPlan f,
                                                          int32_t* dev_status) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x, d = dst[i];
  int later = 0;
  for (int j = i + 1 + threadIdx.x; j < n; j += 256) later |= takes(t, src, dst, j, d);
  gather_pair(t, i, src[i], d, __syncthreads_or(later) != 0, f, threadIdx.x, 256, dev_status);
}

// GATHER: does what fork_gather_kernel does first, a warp for each pair. Where the rows are few that takes less than a launch: a
// step of 16 forks, 32 pages wide, with what it releases and allocates 24 -> 17 us.
template <bool GATHER>
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(PageTable t, const int32_t* src, const int32_t* dst, int n, ForkPlan f,
                                                                 unsigned char* served, int32_t* dev_status) {
  __shared__ int s_scan[33];
  pdl_wait();
  pdl_trigger();
  if (GATHER) {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
      const int d = dst[i];
      int later = 0;
      for (int j = i + 1 + lane; j < n; j += 32) later |= takes(t, src, dst, j, d);
      gather_pair(t, i, src[i], d, __any_sync(0xffffffffu, later), f, lane, 32, dev_status);
    }
    __syncthreads();
  }
  int want = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    const int mine = i < n && f.state[i] == 2;
    int total;
    const int at = want + block_scan(mine, s_scan, total);
    if (mine) f.to[i] = at;                      // its place among the fresh pages, for now
    want += total;
  }
  const int have = collect(t.refs, t.pages, min(want, t.pages), f.list, s_scan, [](int, int c) { return c == 0; });
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    int state = f.state[i];
    if (state == 2) {
      if (f.to[i] < have) {
        const int page = f.list[f.to[i]];
        f.to[i] = page;
        f.rows[(long long)i * t.width + f.at[i]] = page;
      } else {
        f.state[i] = state = 0;
      }
    }
    served[i] = state != 0;
  }
}

// The first n blocks give the destinations their rows, the others copy pages.
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(PageTable t, const int32_t* dst, int n, ForkPlan f, PagePool pool) {
  pdl_wait();
  if ((int)blockIdx.x < n) {
    const int i = blockIdx.x, state = f.state[i];
    if (state != 1 && state != 2) return;
    const int d = dst[i];
    for (int e = threadIdx.x; e < t.width; e += kCopyThreads) {
      const int now = f.rows[(long long)i * t.width + e];
      int32_t* entry = t.table + d * t.stride + e;
      const int old = *entry;
      if (old >= 0 && old < t.pages) atomicSub(t.refs + old, 1);
      if (now >= 0 && now < t.pages) atomicAdd(t.refs + now, 1);
      *entry = now;
    }
    if (threadIdx.x == 0) t.lens[d] = f.len[i];
  } else {
    copy_tasks(pool, n, blockIdx.x - n, gridDim.x - n, [&](int i, int& a, int& b) {
      a = f.from[i], b = f.to[i];
      return f.state[i] == 2;
    });
  }
}

// ------------------------------------------------------------------------------------------------------------ compaction
// list: the holes below the count of live pages, then as many live pages above it; to: where a page from the count up goes.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(int32_t* refs, int pages, int32_t* live, int32_t* moves,
                                                                    int32_t* list, int32_t* to) {
  __shared__ int s_scan[33];
  pdl_wait();
  pdl_trigger();
  const int count = collect(refs, pages, pages, (int32_t*)nullptr, s_scan, [](int, int c) { return c > 0; });
  const int n = collect(refs, pages, pages, list, s_scan, [=](int p, int c) { return (p < count) != (c > 0); }) / 2;
  for (int p = count + threadIdx.x; p < pages; p += kPlanThreads) to[p] = p;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int a = list[n + i], b = list[i];
    to[a] = b;
    refs[b] = refs[a];
    refs[a] = 0;
  }
  if (threadIdx.x == 0) *live = count, *moves = n;
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(PagePool pool, int32_t* table, int sequences, int width, long long stride,
                                                                     int pages, const int32_t* live, const int32_t* moves, const int32_t* list,
                                                                     const int32_t* to) {
  pdl_wait();
  const int n = *moves, count = *live;
  if (n == 0) return;
  const long long entries = (long long)sequences * width;
  for (long long e = (long long)blockIdx.x * kCopyThreads + threadIdx.x; e < entries; e += (long long)gridDim.x * kCopyThreads) {
    const long long s = e / width;
    int32_t* entry = table + s * stride + (e - s * width);
    const int page = *entry;
    if (page >= count && page < pages) *entry = to[page];
  }
  copy_tasks(pool, n, blockIdx.x, gridDim.x, [&](int i, int& a, int& b) {
    a = list[n + i], b = list[i];
    return true;
  });
}

static bool pool_ok(const PagePool& p) {
  return p.outer >= 0 && p.page_bytes >= 0 && p.page_bytes % 16 == 0 && p.outer_bytes % 16 == 0 && p.page_stride % 16 == 0 &&
         reinterpret_cast<uintptr_t>(p.data) % 16 == 0;
}
static bool table_ok(const PageTable& t) {
  return t.sequences >= 0 && t.width >= 0 && t.pages >= 0 && t.page_size >= 1 && t.pages < (1 << 29) && t.width <= (1 << 20);
}
// Blocks for copies of up to `tasks` pieces of 2 KB: eight resident on each SM, fewer where there is less to do.
static int copy_blocks(const PagePool& p, long long pairs) {
  const long long pieces = (p.page_bytes + 32 * kCopyVecs * 16 - 1) / (32 * kCopyVecs * 16) * p.outer * pairs;
  return (int)std::max(1LL, std::min((pieces + kCopyThreads / 32 - 1) / (kCopyThreads / 32), 8LL * sm_count()));
}

}  // namespace sparge

extern "C" size_t sparge_pages_workspace_bytes(int n, int table_width, int num_pages) {
  if (n < 0 || table_width < 0 || num_pages < 0) return 0;
  return 4 * ((size_t)2 * num_pages + (size_t)n * (8 + (size_t)table_width) + 16);
}

extern "C" int sparge_allocate_pages(int32_t* page_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* new_tokens,
                                     unsigned char* served, void* workspace, int sequences, int table_width, long long table_stride,
                                     int num_pages, int page_size, sparge_stream_t stream) {
  using namespace sparge;
  const PageTable t{page_table, seq_lens, ref_counts, table_stride, sequences, table_width, num_pages, page_size};
  if (!table_ok(t)) return SPARGE_ERR_INVALID_ARG;
  if (sequences == 0) return SPARGE_OK;
  if ((table_width && !page_table) || !seq_lens || (num_pages && !ref_counts) || !new_tokens || !served || !workspace) return SPARGE_ERR_NULL;
  int32_t* w = (int32_t*)workspace;
  return launch(allocate_kernel, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, true, t, new_tokens, served, w, w + num_pages,
                w + num_pages + sequences) == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}

extern "C" int sparge_free_sequences(int32_t* page_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* which, int n,
                                     int sequences, int table_width, long long table_stride, int num_pages, int32_t* dev_status,
                                     sparge_stream_t stream) {
  using namespace sparge;
  const PageTable t{page_table, seq_lens, ref_counts, table_stride, sequences, table_width, num_pages, 1};
  if (!table_ok(t) || n < 0) return SPARGE_ERR_INVALID_ARG;
  if (n == 0) return SPARGE_OK;
  if ((sequences && ((table_width && !page_table) || !seq_lens)) || (num_pages && !ref_counts) || !which) return SPARGE_ERR_NULL;
  return launch(free_kernel, dim3(n), dim3(256), 0, (cudaStream_t)stream, true, t, which, dev_status) == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}

extern "C" int sparge_fork_sequences(void* pages, long long outer, long long outer_bytes, long long page_stride_bytes, long long page_bytes,
                                     int32_t* page_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* src, const int32_t* dst,
                                     unsigned char* served, void* workspace, int n, int sequences, int table_width,
                                     long long table_stride, int num_pages, int page_size, int32_t* dev_status, sparge_stream_t stream) {
  using namespace sparge;
  const PageTable t{page_table, seq_lens, ref_counts, table_stride, sequences, table_width, num_pages, page_size};
  const PagePool pool{(char*)pages, outer, outer_bytes, page_stride_bytes, page_bytes};
  if (!table_ok(t) || !pool_ok(pool) || n < 0) return SPARGE_ERR_INVALID_ARG;
  if (n > SPARGE_MAX_PAIRS) return SPARGE_ERR_TOO_LARGE;
  if (n == 0) return SPARGE_OK;
  if ((sequences && ((table_width && !page_table) || !seq_lens)) || (num_pages && (!ref_counts || !pages)) || !src || !dst || !served || !workspace)
    return SPARGE_ERR_NULL;
  int32_t* w = (int32_t*)workspace;
  const ForkPlan f{w, w + n, w + 2 * (size_t)n, w + 3 * (size_t)n, w + 4 * (size_t)n, w + 5 * (size_t)n + num_pages, w + 5 * (size_t)n};
  const cudaStream_t st = (cudaStream_t)stream;
  // one block reads and writes about 8 entries a cycle: up to 32 K of them cost it no more than the launch that they save
  if ((long long)n * (table_width + n / 32) <= 32768) {
    if (launch(fork_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, st, true, t, src, dst, n, f, served, dev_status) != cudaSuccess) return SPARGE_ERR_CUDA;
  } else {
    if (launch(fork_gather_kernel, dim3(n), dim3(256), 0, st, true, t, src, dst, n, f, dev_status) != cudaSuccess ||
        launch(fork_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, st, true, t, src, dst, n, f, served, dev_status) != cudaSuccess)
      return SPARGE_ERR_CUDA;
  }
  if (launch(fork_apply_kernel, dim3(n + copy_blocks(pool, n)), dim3(kCopyThreads), 0, st, true, t, dst, n, f, pool) != cudaSuccess)
    return SPARGE_ERR_CUDA;
  return SPARGE_OK;
}

extern "C" int sparge_compact_pages(void* pages, long long outer, long long outer_bytes, long long page_stride_bytes, long long page_bytes,
                                    int32_t* page_table, int32_t* ref_counts, int32_t* live, void* workspace, int sequences,
                                    int table_width, long long table_stride, int num_pages, sparge_stream_t stream) {
  using namespace sparge;
  const PageTable t{page_table, nullptr, ref_counts, table_stride, sequences, table_width, num_pages, 1};
  const PagePool pool{(char*)pages, outer, outer_bytes, page_stride_bytes, page_bytes};
  if (!table_ok(t) || !pool_ok(pool)) return SPARGE_ERR_INVALID_ARG;
  if (!live || !workspace || (num_pages && (!ref_counts || !pages)) || (sequences && table_width && !page_table)) return SPARGE_ERR_NULL;
  int32_t *list = (int32_t*)workspace, *to = list + num_pages, *moves = to + num_pages;
  const cudaStream_t st = (cudaStream_t)stream;
  if (launch(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, true, ref_counts, num_pages, live, moves, list, to) != cudaSuccess ||
      launch(compact_apply_kernel, dim3(copy_blocks(pool, num_pages / 2 + 1)), dim3(kCopyThreads), 0, st, true, pool, page_table, sequences, table_width,
             table_stride, num_pages, live, moves, list, to) != cudaSuccess)
    return SPARGE_ERR_CUDA;
  return SPARGE_OK;
}

extern "C" int sparge_copy_pages(void* pages, long long outer, long long outer_bytes, long long page_stride_bytes, long long page_bytes,
                                 const int32_t* src, const int32_t* dst, int n, int num_pages, int32_t* dev_status, sparge_stream_t stream) {
  using namespace sparge;
  const PagePool pool{(char*)pages, outer, outer_bytes, page_stride_bytes, page_bytes};
  if (!pool_ok(pool) || n < 0 || num_pages < 0) return SPARGE_ERR_INVALID_ARG;
  if (n > SPARGE_MAX_PAIRS) return SPARGE_ERR_TOO_LARGE;
  if (n == 0 || outer == 0 || page_bytes == 0) return SPARGE_OK;
  if ((num_pages && !pages) || !src || !dst) return SPARGE_ERR_NULL;
  // one pair at a time fills the GPU only where pages are large or the pool has many slices
  const int slices = std::min(copy_blocks(pool, 1), std::max(1, 8 * sm_count() / n));
  return launch(copy_pages_kernel, dim3(n, slices), dim3(kCopyThreads), 0, (cudaStream_t)stream, true, pool, src, dst, n, num_pages, dev_status) == cudaSuccess
             ? SPARGE_OK : SPARGE_ERR_CUDA;
}
