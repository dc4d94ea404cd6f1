// What the kernels of attention over a paged cache share: their parameters, how a CTA finds its share of the work, and the warp
// that brings key and value tiles from the pages into shared memory.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "paged_schedule.cuh"
#include "sm100_ptx.cuh"

namespace sparge {

// The border in front of a share that begins inside a tile, for the kernel that joins tiles which lie in several shares.
struct ShareJoin {
  int pieces;                     // of the tile; 0: the share begins with a tile
  int border;                     // which of the tile's pieces - 1 borders this one is
  int first;                      // the share of the first piece
  int slot;                       // of the first piece; piece i > 0 has 2 (first + i)
  int token, row, rows, head;     // the sequence's first row of q; the tile's first row and their count; key head
};

struct PagedParams {
  const void* q;
  void* out;
  float* lse;
  long long q_token, q_head, out_token, out_head, table_stride;
  const int32_t *cu, *seq_lens, *table;
  int tokens, sequences, width, num_pages, page_size, page_shift, kv_heads, group;
  bool causal, zero_out, zero_lse;
  float scale_log2;
  ShareJoin* joins;               // [max_shares]
  float* part_o;                  // [shares][2][rows][D]: the share's first tile, its last one
  float* part_ml;                 // [shares][2][rows][2]
  int max_shares;
  int32_t* dev_status;
};

// What the loading warp tells the others about one unit.
struct Unit {
  int flags;                      // kFirst, kLast: of the share's piece of a tile; kWhole: the piece is the tile; kHead: the share's first piece
  int token, row, rows, head;     // as in ShareJoin
  int key;                        // the unit's first key
  int length;                     // keys of the sequence
  int visible0;                   // row r of the sequence sees min(length, visible0 + r / group + 1) keys
};
constexpr int kFirst = 1, kLast = 2, kWhole = 4, kHead = 8;

__device__ __forceinline__ void paged_report(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

template <int ROWS>
__device__ __forceinline__ SeqWork<ROWS> load_seq(const PagedParams& p, int i, int& token) {
  int lo = i, hi = i + 1;
  if (p.cu) {
    lo = max(0, min(p.cu[i], p.tokens));
    hi = max(lo, min(p.cu[i + 1], p.tokens));
  }
  token = lo;
  return SeqWork<ROWS>{(unsigned)(hi - lo), (unsigned)max(0, min(p.seq_lens[i], p.width << p.page_shift)), (unsigned)p.group, p.causal};
}

// A place on the line of units.
template <int ROWS>
struct Place {
  int seq, head, token;
  unsigned tile, block;
  long long first;                // the tile's first unit
  SeqWork<ROWS> w;
};

// Every thread of the CTA calls this. Returns the share's units [begin, end), and the place of its first one. What a launch
// spends here it spends before anything is loaded, so there are two barriers, and most of the arithmetic is 32-bit (with 64-bit
// divisions and a barrier for every step: 6.5 us, of 18 that a call over one short sequence took).
struct ShareSearch {              // in shared memory
  long long warp[32], left;
  int seq, token;
  unsigned tokens, length;
  unsigned tile;
};
template <int kThreads, int ROWS>
__device__ __forceinline__ void find_share(const PagedParams& p, ShareSearch& s, long long& begin, long long& end, long long& units,
                                           int& shares, Place<ROWS>& at) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.sequences + kThreads - 1) / kThreads, lo = min(tid * per, p.sequences), hi = min(lo + per, p.sequences);
  long long mine = 0;
  SeqWork<ROWS> w = {};
  int token = 0;
  for (int i = lo; i < hi; i++) {
    w = load_seq<ROWS>(p, i, token);
    mine += w.units() * p.kv_heads;
    if (p.seq_lens[i] != (int)w.length) paged_report(p.dev_status, SPARGE_DEV_BAD_PAGE);
  }
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s.warp[warp] = x;
  if (tid == 0) s.tile = 0;
  __syncthreads();
  long long before = x - mine;
  units = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; i++) {
    const long long v = s.warp[i];
    if (i < warp) before += v;
    units += v;
  }
  shares = units < p.max_shares ? (int)units : p.max_shares;
  const int c = blockIdx.x;
  begin = end = 0;
  if (c >= shares) return;
  begin = share_begin(c, units, shares), end = share_begin(c + 1, units, shares);
  if (before <= begin && begin < before + mine) {
    long long left = begin - before;
    int i = hi - 1;               // w is the last one of the thread's, most often the only one
    if (per > 1) {
      for (i = lo; i < hi; i++) {
        w = load_seq<ROWS>(p, i, token);
        const long long n = w.units() * p.kv_heads;
        if (left < n) break;
        left -= n;
      }
    }
    s.seq = i, s.left = left, s.token = token, s.tokens = w.tokens, s.length = w.length;
  }
  __syncthreads();
  at.seq = s.seq, at.token = s.token;
  at.w = SeqWork<ROWS>{s.tokens, s.length, (unsigned)p.group, p.causal};
  long long left = s.left;
  const unsigned tiles = at.w.tiles();
  if (tiles == 1) {
    const unsigned blocks = at.w.blocks(0);
    at.head = (int)((unsigned)left / blocks);          // heads times blocks of one sequence: below 2^31
    at.tile = 0, at.block = (unsigned)left - at.head * blocks;
  } else {
    const long long per_head = at.w.units();
    at.head = (int)(left / per_head);
    left -= at.head * per_head;
    // the last tile that begins at or before the place: all threads try one each, then the gap between two of them
    unsigned base = 0;
    for (unsigned step = (tiles + kThreads - 1) / kThreads;; step = (step + kThreads - 1) / kThreads) {
      const unsigned t = base + tid * step;
      if (t < tiles && at.w.blocks_before(t) <= left) atomicMax(&s.tile, t);
      __syncthreads();
      base = s.tile;
      if (step <= 1) break;
      __syncthreads();
    }
    at.tile = base;
    at.block = (unsigned)(left - at.w.blocks_before(base));
  }
  at.first = begin - at.block;
}

// The place of the tile behind this one, at its first block.
template <int ROWS>
__device__ __forceinline__ void next_tile(const PagedParams& p, Place<ROWS>& at) {
  at.first += at.w.blocks(at.tile);
  at.block = 0;
  if (++at.tile < at.w.tiles()) return;
  at.tile = 0;
  if (++at.head < p.kv_heads) return;
  at.head = 0;
  do {
    at.seq++;
    if (at.seq >= p.sequences) return;
    at.w = load_seq<ROWS>(p, at.seq, at.token);
  } while (at.w.tokens == 0);
}

// What the joining kernel has to know of the border in front of this share. One thread of every CTA calls it.
template <int ROWS>
__device__ __forceinline__ void note_join(const PagedParams& p, long long begin, long long units, int shares, const Place<ROWS>& at) {
  ShareJoin j = {};
  const int c = blockIdx.x;
  if (c < shares && begin > at.first) {
    const int first = share_of(at.first, units, shares), last = share_of(at.first + at.w.blocks(at.tile) - 1, units, shares);
    j = ShareJoin{last - first + 1, c - first - 1, first, 2 * first + (share_begin(first, units, shares) < at.first), at.token, (int)(at.tile * ROWS),
                  (int)at.w.tile_rows(at.tile), at.head};
  }
  p.joins[c] = j;
}

// Rows of q that belong to no sequence become zeros, and minus infinity in lse.
template <typename T, int D>
__device__ __forceinline__ void zero_rest(const PagedParams& p, int thread, int threads) {
  if (!p.cu || !(p.zero_out || p.zero_lse)) return;
  const int lo = max(0, min(p.cu[0], p.tokens)), hi = max(lo, min(p.cu[p.sequences], p.tokens)), heads = p.kv_heads * p.group;
  const long long rows = (long long)(p.tokens - (hi - lo)) * heads;
  constexpr int kWords = D * (int)sizeof(T) / 16;
  for (long long i = thread; i < rows * kWords; i += threads) {
    const long long r = i / kWords, t = r / heads, token = t < lo ? t : t - lo + hi;
    const int h = (int)(r - t * heads), word = (int)(i - r * kWords);
    if (p.zero_out) reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + token * p.out_token + h * p.out_head)[word] = make_uint4(0, 0, 0, 0);
    if (word == 0 && p.zero_lse) p.lse[token * heads + h] = -INFINITY;
  }
}

// Keys and values reach shared memory by the copy engine, a page's rows of one head at a time, in column halves of 64 (128 bytes,
// 128-byte swizzle). Keys that the sequence does not have, and pages that the pool does not have, are read at a page number
// behind the last one, where the copy engine fills in zeros. So every tile is complete, and nothing of what an earlier owner left
// behind is in it but the rest of the one page that the length ends in.
// A lane's entry of the table for a unit (the pages of its pieces, lane by lane), read while the unit before it is under way (just
// before the copies: 216 us for 64 sequences of up to 8 191 keys in pages of 16, where this takes 200).
__device__ __forceinline__ int table_entry(const PagedParams& p, int seq, int key, int length) {
  return key < length ? p.table[seq * p.table_stride + (key >> p.page_shift)] : 0;
}
__device__ __forceinline__ int page_of(const PagedParams& p, int entry, int key, int length) {
  if (key >= length) return p.num_pages;
  if (entry >= 0 && entry < p.num_pages) return entry;
  paged_report(p.dev_status, SPARGE_DEV_BAD_PAGE);
  return p.num_pages;
}

int paged_decode_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st);
int paged_tile_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st);
constexpr int kDecodeRows = 16, kTileRows = 256;

}  // namespace sparge
