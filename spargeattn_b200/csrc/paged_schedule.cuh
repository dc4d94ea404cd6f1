// How the work of one call of attention over a paged cache is cut into equal shares. (No other header: the host compiler can
// read this one alone.)
//
// A sequence with n new tokens has n * group rows for each key head (row r: token r / group, query head r % group), in tiles of
// `rows` rows. A tile sees the keys up to the position of its last row, in blocks of kBlockKeys: its number of units. All
// units of a call, sequence by sequence, key head by key head, tile by tile, block by block, lie on one line, and every share
// is a contiguous run of it: a long context is cut where there are few rows, and no share is longer than another by more than
// one unit. A tile that lies in several shares is joined afterwards. The line depends on the lengths alone, which are on
// the device; each CTA finds its place on it by itself, so nothing is planned on the host and a captured call follows lengths
// that change between replays.
#pragma once
#if defined(__CUDACC__)
#define SPARGE_SCHED __host__ __device__ __forceinline__
#else
#define SPARGE_SCHED inline
#endif

namespace sparge {

constexpr int kBlockKeys = 128;

// sum over i in [0, n) of floor((a + b i) / m), for a, b >= 0, m > 0: the number of lattice points under a line, counted by
// exchanging the axes as in Euclid's algorithm.
SPARGE_SCHED long long floor_sum(long long n, long long a, long long b, long long m) {
  long long sum = 0;
  while (n > 0) {
    if (b >= m) {
      sum += n * (n - 1) / 2 * (b / m);
      b %= m;
    }
    if (a >= m) {
      sum += n * (a / m);
      a %= m;
    }
    const long long top = a + b * n;
    if (top < m) break;
    n = top / m;
    a = top % m;
    const long long t = b;
    b = m;
    m = t;
  }
  return sum;
}

// One sequence: its new tokens, its length with them, and the rows of a tile.
struct SeqWork {
  long long tokens, length;
  int group, rows;
  bool causal;

  SPARGE_SCHED long long all_rows() const { return tokens * group; }
  SPARGE_SCHED long long tiles() const { return (all_rows() + rows - 1) / rows; }
  // keys that row r sees; not above zero: none
  SPARGE_SCHED long long visible(long long r) const { return causal ? length - tokens + r / group + 1 : length; }
  SPARGE_SCHED long long last_row(long long tile) const {
    const long long end = (tile + 1) * rows, all = all_rows();
    return (end < all ? end : all) - 1;
  }
  // blocks of one tile; a tile that sees nothing has one all the same, which writes its zeros
  SPARGE_SCHED long long blocks(long long tile) const {
    const long long v = visible(last_row(tile));
    return v <= kBlockKeys ? 1 : (v + kBlockKeys - 1) / kBlockKeys;
  }
  // blocks of the tiles [0, t), t <= tiles()
  SPARGE_SCHED long long blocks_before(long long t) const {
    if (t <= 0) return 0;
    if (!causal) return t * blocks(0);
    const long long all = tiles();
    if (t == all) return blocks_before(t - 1) + blocks(t - 1);
    // blocks(i) = max(1, floor((a + b i) / m)) for every tile but the last: the floor of a floor is one floor
    const long long m = (long long)kBlockKeys * group, a = group * (length - tokens + kBlockKeys) + rows - 1, b = rows;
    long long first = 0;   // the tiles before it see one block or less
    if (a < m) {
      first = (m - a + b - 1) / b;
      if (first > t) first = t;
    }
    return first + floor_sum(t - first, a + b * first, b, m);
  }
  SPARGE_SCHED long long units() const { return blocks_before(tiles()); }   // of one key head
};

// Where share c of `shares` begins on a line of `units`.
SPARGE_SCHED long long share_begin(long long c, long long units, long long shares) { return c * units / shares; }

}  // namespace sparge
