// What the kernels of attention over a paged cache share: their parameters, how a CTA finds its share of the work, and the warp
// that brings key and value tiles from the pages into shared memory.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "paged_schedule.cuh"
#include "sm100_ptx.cuh"

namespace sparge {

// A share's first tile, for the kernel that joins tiles which lie in several shares.
struct ShareStart {
  long long begin, first, last;   // the share's first unit; the tile's units [first, last)
  int token, row, rows, head;     // the sequence's first row of q; the tile's first row and their count; key head
};

struct PagedParams {
  const void* q;
  void* out;
  float* lse;
  long long q_token, q_head, out_token, out_head, table_stride;
  const int32_t *cu, *seq_lens, *table;
  int tokens, sequences, width, num_pages, page_size, kv_heads, group;
  bool causal, zero_rest;
  float scale_log2;
  ShareStart* starts;             // [shares + 1]: entry [shares] holds {units, shares, 0, ...}
  float* part_o;                  // [shares][2][rows][D]: the share's first tile, its last one
  float* part_ml;                 // [shares][2][rows][2]
  int max_shares;
  int32_t* dev_status;
};

// What the loading warp tells the others about one unit.
struct Unit {
  int flags;                      // kFirst, kLast: of the share's piece of a tile; kWhole: the piece is the tile; kHead: the share's first piece
  int token, row, rows, head;     // as in ShareStart
  int key;                        // the unit's first key
  int length;                     // keys of the sequence
  int visible0;                   // row r of the sequence sees min(length, visible0 + r / group + 1) keys
};
constexpr int kFirst = 1, kLast = 2, kWhole = 4, kHead = 8;

__device__ __forceinline__ void paged_report(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

__device__ __forceinline__ SeqWork load_seq(const PagedParams& p, int i, int rows, int& token) {
  long long lo = i, hi = i + 1;
  if (p.cu) {
    lo = max(0, min(p.cu[i], p.tokens));
    hi = max((int)lo, min(p.cu[i + 1], p.tokens));
  }
  const long long most = (long long)p.width * p.page_size, len = p.seq_lens[i];
  token = (int)lo;
  return SeqWork{hi - lo, max(0LL, min(len, most)), p.group, rows, p.causal};
}

// A place on the line of units.
struct Place {
  int seq, head, token;
  long long tile, block, first;   // first: the tile's first unit
  SeqWork w;
};

// Every thread of the CTA calls this. Returns the share's units [begin, end), and the place of its first one.
// s: kThreads + 8 long longs of shared memory.
template <int kThreads>
__device__ __forceinline__ void find_share(const PagedParams& p, int rows, long long* s, long long& begin, long long& end,
                                           long long& units, int& shares, Place& at) {
  const int tid = threadIdx.x;
  const int per = (p.sequences + kThreads - 1) / kThreads, lo = min(tid * per, p.sequences), hi = min(lo + per, p.sequences);
  long long mine = 0;
  for (int i = lo; i < hi; i++) {
    int token;
    const SeqWork w = load_seq(p, i, rows, token);
    mine += w.units() * p.kv_heads;
    if (p.seq_lens[i] != w.length) paged_report(p.dev_status, SPARGE_DEV_BAD_PAGE);
  }
  s[tid] = mine;
  __syncthreads();
  if (tid < 32) {   // prefix sums of the threads' sums
    constexpr int kEach = (kThreads + 31) / 32;
    long long part[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      part[i] = sum;
      if (tid * kEach + i < kThreads) sum += s[tid * kEach + i];
    }
    long long x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (tid >= o) x += y;
    }
#pragma unroll
    for (int i = 0; i < kEach; i++)
      if (tid * kEach + i < kThreads) s[tid * kEach + i] = x - sum + part[i];
    if (tid == 31) s[kThreads] = x;
  }
  __syncthreads();
  units = s[kThreads];
  shares = (int)min((long long)p.max_shares, units);
  const int c = blockIdx.x;
  begin = end = 0;
  if (c >= shares) return;
  begin = share_begin(c, units, shares), end = share_begin(c + 1, units, shares);
  const long long before = s[tid];
  if (before <= begin && begin < before + mine) {
    long long left = begin - before;
    for (int i = lo; i < hi; i++) {
      int token;
      const SeqWork w = load_seq(p, i, rows, token);
      const long long n = w.units() * p.kv_heads;
      if (left < n) {
        s[kThreads + 1] = i;
        s[kThreads + 2] = left;
        break;
      }
      left -= n;
    }
  }
  if (tid == 0) s[kThreads + 3] = 0;
  __syncthreads();
  at.seq = (int)s[kThreads + 1];
  long long left = s[kThreads + 2];
  at.w = load_seq(p, at.seq, rows, at.token);
  const long long per_head = at.w.units(), tiles = at.w.tiles();
  at.head = (int)(left / per_head);
  left -= at.head * per_head;
  // the last tile that begins at or before the place: all threads try one each, then the gap between two of them
  long long base = 0;
  for (long long step = (tiles + kThreads - 1) / kThreads;; step = (step + kThreads - 1) / kThreads) {
    const long long t = base + tid * step;
    if (tiles > 1 && t < tiles && at.w.blocks_before(t) <= left) atomicMax(reinterpret_cast<unsigned long long*>(s + kThreads + 3), (unsigned long long)t);
    __syncthreads();
    base = s[kThreads + 3];
    if (step <= 1) break;
    __syncthreads();
  }
  at.tile = base;
  at.block = left - at.w.blocks_before(base);
  at.first = begin - at.block;
}

// The place of the tile behind this one, at its first block.
__device__ __forceinline__ void next_tile(const PagedParams& p, int rows, Place& at) {
  at.first += at.w.blocks(at.tile);
  at.block = 0;
  if (++at.tile < at.w.tiles()) return;
  at.tile = 0;
  if (++at.head < p.kv_heads) return;
  at.head = 0;
  do {
    at.seq++;
    if (at.seq >= p.sequences) return;
    at.w = load_seq(p, at.seq, rows, at.token);
  } while (at.w.tokens == 0);
}

__device__ __forceinline__ ShareStart share_start(const PagedParams& p, int rows, long long begin, const Place& at) {
  return ShareStart{begin, at.first, at.first + at.w.blocks(at.tile), at.token, (int)(at.tile * rows),
                    (int)min((long long)rows, at.w.all_rows() - at.tile * rows), at.head};
}

// Rows of q that belong to no sequence become zeros.
template <typename T, int D>
__device__ __forceinline__ void zero_rest(const PagedParams& p, int thread, int threads) {
  if (!p.zero_rest || !p.cu) return;
  const int lo = max(0, min(p.cu[0], p.tokens)), hi = max(lo, min(p.cu[p.sequences], p.tokens)), heads = p.kv_heads * p.group;
  const long long rows = (long long)(p.tokens - (hi - lo)) * heads;
  constexpr int kWords = D * (int)sizeof(T) / 16;
  for (long long i = thread; i < rows * kWords; i += threads) {
    const long long r = i / kWords, t = r / heads, token = t < lo ? t : t - lo + hi;
    const int h = (int)(r - t * heads), word = (int)(i - r * kWords);
    reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + token * p.out_token + h * p.out_head)[word] = make_uint4(0, 0, 0, 0);
    if (word == 0 && p.lse) p.lse[token * heads + h] = -INFINITY;
  }
}

// Key or value tile of a unit: kBlockKeys rows of D channels, in column halves of 64 (128 bytes, 128-byte swizzle). A copy
// takes a page's rows of one half; keys that the sequence does not have, and pages that the pool does not have, are read
// at a page number behind the last one, where the copy engine fills in zeros. So every tile is complete, and nothing of what
// an earlier owner left behind in the tile's last pages is in it but the rest of the one page that the length ends in.
template <int D>
__device__ __forceinline__ void load_tile(const PagedParams& p, uint8_t* dst, const CUtensorMap* map, uint64_t* bar, const int32_t* table,
                                          int key0, int length, int head, int lane) {
  const int box = min(p.page_size, kBlockKeys), boxes = kBlockKeys / box;
  if (lane < boxes * (D / 64)) {
    const int half = lane / boxes, piece = lane - half * boxes, key = key0 + piece * box;
    int page = p.num_pages;
    if (key < length) {
      page = table[key / p.page_size];
      if (page < 0 || page >= p.num_pages) {
        paged_report(p.dev_status, SPARGE_DEV_BAD_PAGE);
        page = p.num_pages;
      }
    }
    tma_load_4d(dst + half * (kBlockKeys * 128) + piece * box * 128, map, bar, half * 64, key & (p.page_size - 1), head, page);
  }
}

int paged_decode_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st);
int paged_tile_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st);
constexpr int kDecodeRows = 16, kTileRows = 256;

}  // namespace sparge
