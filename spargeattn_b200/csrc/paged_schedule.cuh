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

// sum over i in [0, n) of floor((a + b i) / m), for m > 0: the floor sum of an arithmetic progression, which counts the lattice points
// under a line. By its reciprocity law (Graham, Knuth, Patashnik, Concrete Mathematics, 3.5): whole parts of the slope and of the
// start are taken out, then the axes change places, as in Euclid's algorithm.
SPARGE_SCHED unsigned long long floor_sum(unsigned long long n, unsigned long long a, unsigned long long b, unsigned long long m) {
  unsigned long long sum = 0;
  while (n > 0) {
    if (b >= m) {
      sum += n * (n - 1) / 2 * (b / m);
      b %= m;
    }
    if (a >= m) {
      sum += n * (a / m);
      a %= m;
    }
    const unsigned long long top = a + b * n;
    if (top < m) break;
    n = top / m;
    a = top % m;
    const unsigned long long t = b;
    b = m;
    m = t;
  }
  return sum;
}

// One sequence: its new tokens, its length with them, and the query heads of a key head. tokens * group and length are below 2^31.
template <int ROWS>
struct SeqWork {
  unsigned tokens, length, group;
  bool causal;

  SPARGE_SCHED unsigned all_rows() const { return tokens * group; }
  SPARGE_SCHED unsigned tiles() const { return (all_rows() + ROWS - 1) / ROWS; }
  SPARGE_SCHED unsigned tile_rows(unsigned tile) const {
    const unsigned left = all_rows() - tile * ROWS;
    return left < ROWS ? left : ROWS;
  }
  // keys that row r sees; not above zero: none
  SPARGE_SCHED int visible(unsigned r) const {
    return causal ? (int)length - (int)tokens + (tokens == 1 ? 1 : (int)(r / group) + 1) : (int)length;
  }
  // blocks of one tile; a tile that sees nothing has one all the same, which writes its zeros
  SPARGE_SCHED unsigned blocks(unsigned tile) const {
    const int v = visible(tile * ROWS + tile_rows(tile) - 1);
    return v <= kBlockKeys ? 1u : ((unsigned)v + kBlockKeys - 1) / kBlockKeys;
  }
  // blocks of the tiles [0, t), t <= tiles()
  SPARGE_SCHED long long blocks_before(unsigned t) const {
    if (t == 0) return 0;
    if (!causal || tokens == 1) return (long long)t * blocks(0);
    const unsigned all = tiles();
    long long sum = 0;
    if (t == all) {   // the last one may have fewer rows
      sum = blocks(t - 1);
      t--;
    }
    // blocks(i) = max(1, floor((a + b i) / m)) of the others: the floor of a floor is one floor
    const long long m = (long long)kBlockKeys * group, b = ROWS;
    long long a = (long long)group * ((long long)length - tokens + kBlockKeys) + ROWS - 1, first = 0;   // first: the tiles before it see one block or less
    if (a < m) {
      first = (m - a + b - 1) / b;
      if (first > t) first = t;
      a += b * first;
    }
    return sum + first + (t > first ? (long long)floor_sum(t - first, a, b, m) : 0);
  }
  SPARGE_SCHED long long units() const { return blocks_before(tiles()); }   // of one key head
};

// Where share c of `shares` begins on a line of `units`.
SPARGE_SCHED long long share_begin(int c, long long units, int shares) {
  const unsigned long long x = (unsigned long long)c * units;
  return x >> 32 ? (long long)(x / (unsigned)shares) : (long long)((unsigned)x / (unsigned)shares);
}
// The share that a unit lies in: the last one that begins at or before it.
SPARGE_SCHED int share_of(long long unit, long long units, int shares) {
  const unsigned long long x = (unsigned long long)(unit + 1) * shares - 1;
  return x >> 32 ? (int)(x / (unsigned long long)units) : (int)((unsigned)x / (unsigned)units);
}

}  // namespace sparge
