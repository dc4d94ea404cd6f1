// Attention of chunks of new tokens over a paged cache: tiles of 256 rows on the 5th-generation tensor cores.
//
//   S = Q K^T   tcgen05.mma kind::f16, Q and K from 128B-swizzled shared memory, 128 rows by 128 keys, f32 in tensor memory
//   softmax     one thread per row: maximum, exponentials, sum in registers; P rounded to the 16-bit type and stored over S
//   O += P V    tcgen05.mma kind::f16 with P from tensor memory and V token-major (an MN-major operand), f32 in tensor memory
//
// A CTA has two tiles of 128 rows (the rows of one key head: tokens by query heads of its group, so grouped heads share every
// key that is fetched) and works on both in turn: while the softmax warps of one are busy, the tensor cores do P V and the next
// Q K^T of the other. Their S, P and O fill tensor memory: columns [0, 128) S and P of the first, [128, 256) of the second,
// [256, 384) and [384, 512) their outputs. 12 warps: 0-3 and 4-7 softmax and epilogue of a tile each, 8 the copies, 9 the
// products (10 and 11 complete a warpgroup, whose registers the softmax warps take over). One warp asks for the products of both
// tiles, in turn: with a warp for each they fall into step and want the exponential unit at the same time (1 273 us against 1 176).
// One CTA on each SM takes an equal run of the call's units (paged_schedule.cuh); the copies run ahead over the borders of tiles,
// heads and sequences, and a tile's queries are fetched while the last product of the tile before it is under way.
//
// The products of a step of 128 keys take 2 048 cycles for the two tiles at D = 128 and the exponentials as many (16 a cycle on
// an SM), so both would have to run all the time; measured: 3 330 cycles a step, tensor cores 62 % and the exponential unit 65 %
// busy, 1.10 PFLOP/s for 4 096 tokens over 20 477 keys, 32 heads to 8 (0.66 of the measured bf16 rate). What bounds it is the chain
// of one tile (stamps of a warp, medians): 650 cycles of waiting for S, 130 to read it, 430 for the maximum, 1 780 for the
// exponentials and the hand-over of P, then P V and the next Q K^T, which has to wait because P lies over S. At D = 64 the products are
// half of that, and a step inside a tile takes the same 3 400 cycles (510 of them waiting for S); over a launch of ragged chunks
// (nine of 172 to 700 tokens over up to 5 003 keys, 16 heads) it is 4 410: a share has two or three tiles, and at the end of each the
// products wait until the next one's queries, which are fetched after the last exponentials, have arrived.
// The running maximum moves only when a row's maximum grows by more than 2^8 (probabilities up to 256 round as exactly as ones up
// to 1), so that the output is hardly ever rescaled. The rounding of the probabilities to the 16-bit type is the products': it
// costs 2^-9 (2^-12) of each one's share, as much as the rounding of the output itself.
//
// Every wait is bounded; on expiry the kernel reports and unwinds.
#include <atomic>

#include "launch.cuh"
#include "paged.cuh"

namespace sparge {

constexpr int kTileThreads = 384, kLoadWarp = 8, kMmaWarpT = 9;
// Registers of a thread: the launch gives every one of the 384 the same 168; the softmax warps hold a row's 128 scores.
constexpr int kSoftmaxRegs = 208, kOtherRegs = 80;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kTileThreads * 168, "more than the launch has");
constexpr int kTileRing = 8;                     // tiles whose description may wait to be read
// P is handed to the products 32 keys at a time (at once: 1 138 us for 4 096 tokens over 20 477 keys, in two parts 1 105, in four
// 1 078).
constexpr int kPartKeys = 32, kParts = kBlockKeys / kPartKeys;
constexpr float kRescaleFrom = 8.f;              // in log2
template <int D>
struct TileShape {
  static constexpr int kQ = 128 * D * 2;                       // one tile's queries
  static constexpr int kTile = kBlockKeys * D * 2;             // K or V of a unit
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kSmemBytes = 1024 + 2 * kQ + kSlots * kTile;
};

// What a tile's roles have to know.
struct TileWork {
  int units;                      // of this share
  int key;                        // first key
  int token, row, rows, head, length, visible0, flags;
};

template <int N, bool MORE>
__device__ __forceinline__ void set_registers() {   // by whole warpgroups
  if (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// D[tmem] (+)= A[tmem] * B[smem], 16-bit inputs of one type, f32 accumulate, K = 16.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The largest of a row's scores of a step: three-input maxima in four chains.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float row_max(const float* s) {
  constexpr int kChain = kBlockKeys / 4;
  float top[4];
#pragma unroll
  for (int g = 0; g < 4; g++) {
    top[g] = max3(s[kChain * g], s[kChain * g + 1], s[kChain * g + 2]);
#pragma unroll
    for (int k = 3; k < kChain - 1; k += 2) top[g] = max3(top[g], s[kChain * g + k], s[kChain * g + k + 1]);
    top[g] = fmaxf(top[g], s[kChain * g + kChain - 1]);
  }
  return fmaxf(max3(top[0], top[1], top[2]), top[3]);
}

template <typename T>
__device__ __forceinline__ uint32_t pack_probs(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Key or value tile of a unit: [half][128 rows][128 bytes], as the products' descriptors want it.
template <int D>
__device__ __forceinline__ void load_tile(const PagedParams& p, uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int entry, int key0, int length, int head,
                                          int lane) {
  const int box = min(p.page_size, kBlockKeys), boxes = kBlockKeys / box;
  if (lane < boxes * (D / 64)) {
    const int half = lane / boxes, piece = lane - half * boxes, key = key0 + piece * box;
    tma_load_5d(dst + half * (kBlockKeys * 128) + piece * box * 128, map, bar, 0, key & (p.page_size - 1), half, head, page_of(p, entry, key, length));
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedParams p) {
  using Shape = TileShape<D>;
  constexpr int NS = Shape::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_ring = smem + 2 * Shape::kQ;
  __shared__ uint64_t bar_full[NS], bar_empty[NS], bar_tile[kTileRing], bar_q[2], bar_s[2], bar_p[2][kParts], bar_o[2], bar_end;
  __shared__ TileWork s_tile[kTileRing];
  __shared__ ShareSearch s_search;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (warp == kMmaWarpT) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < kTileRing; i++) mbar_init(&bar_tile[i], 1);
    mbar_init(&bar_end, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&bar_q[i], 4);
      mbar_init(&bar_s[i], 1);
      for (int k = 0; k < kParts; k++) mbar_init(&bar_p[i][k], 4);
      mbar_init(&bar_o[i], 1);
    }
    mbar_fence_init();
    s_fail = 0;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  pdl_wait();                                                // lengths, tables and queries come from the kernels before
  zero_rest<T, D>(p, blockIdx.x * kTileThreads + tid, gridDim.x * kTileThreads);
  long long begin, end, units;
  int shares;
  Place<kTileRows> at;
  find_share<kTileThreads>(p, s_search, begin, end, units, shares, at);
  if (tid == kTileThreads - 32) note_join(p, begin, units, shares, at);   // the warp that has nothing else to do
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = s_tmem;
  const int n = (int)(end - begin);

  if (warp >= kLoadWarp) {
    set_registers<kOtherRegs, false>();
    if (warp == kLoadWarp) {
      // ------------------------------------------------------------------ copies
      const int box = min(p.page_size, kBlockKeys), piece_key = (lane & (kBlockKeys / box - 1)) * box;   // of this lane's copies
      bool ok = true, first_piece = true;
      int issued = 0;                                          // tiles of K or V
      auto load = [&](int i, const CUtensorMap* map, int entry, int key, int length, int head) {
        const int slot = i % NS;
        if (i >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&bar_empty[slot], ((i / NS) - 1) & 1));
        ok = ok && !__any_sync(0xffffffffu, *(volatile int*)&s_fail);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&bar_full[slot], Shape::kTile);
        __syncwarp();
        load_tile<D>(p, s_ring + slot * Shape::kTile, map, &bar_full[slot], entry, key, length, head, lane);
        issued = i + 1;
      };
      auto entry_at = [&](int key) { return table_entry(p, at.seq, key + piece_key, (int)at.w.length); };
      int done = 0, entry = n > 0 ? entry_at((int)(at.block * kBlockKeys)) : 0;
      for (int t = 0; done < n && ok; t++) {
        const unsigned blocks = at.w.blocks(at.tile);
        const int here = (int)min(blocks - at.block, (unsigned)(n - done));
        const int key0 = (int)(at.block * kBlockKeys), length = (int)at.w.length, head = at.head;
        if (lane == 0) {
          TileWork w;
          const bool whole = at.block == 0 && here == (int)blocks;
          w.units = here, w.key = key0;
          w.token = at.token, w.row = (int)(at.tile * kTileRows), w.rows = (int)at.w.tile_rows(at.tile);
          w.head = at.head, w.length = length, w.visible0 = p.causal ? length - (int)at.w.tokens : length;
          w.flags = (whole ? kWhole : 0) | (first_piece ? kHead : 0);
          s_tile[t % kTileRing] = w;
          mbar_arrive(&bar_tile[t % kTileRing]);
        }
        for (int j = 0; j < here && ok; j++) {
          const int key = key0 + j * kBlockKeys, i = 2 * (done + j);
          // the next unit's place and pages are looked up while slots become free; behind the first unit's copies
          const int now = entry;
          auto advance = [&]() {
            if (j + 1 < here) {
              entry = entry_at(key + kBlockKeys);
            } else if (done + here < n) {
              next_tile(p, at);
              entry = entry_at(0);
            }
          };
          if (i > 0) advance();
          load(i, &map_k, now, key, length, head);
          if (ok) load(i + 1, &map_v, now, key, length, head);
          if (i == 0) advance();
        }
        done += here;
        first_piece = false;
      }
      if (!ok) {
        if (lane == 0) {
          paged_report(p.dev_status, SPARGE_DEV_TIMEOUT_PRODUCER);
          *(volatile int*)&s_fail = SPARGE_DEV_TIMEOUT_PRODUCER;
        }
        for (int i = max(0, issued - NS); i < issued; i++) mbar_wait(&bar_full[i % NS], (i / NS) & 1);   // our own copies land first
      }
    } else if (warp == kMmaWarpT) {
      // ------------------------------------------------------------------ products
      constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t idesc_qk = make_idesc(1, fmt, fmt, 0, 0, 128, kBlockKeys);
      constexpr uint32_t idesc_pv = make_idesc(1, fmt, fmt, 0, 1, 128, D);
      const uint64_t qd = make_smem_desc(smem_u32(smem), 16, 1024, kSwizzle128B);
      const uint64_t kd = make_smem_desc(smem_u32(s_ring), 16, 1024, kSwizzle128B);
      const uint64_t vd = make_smem_desc(smem_u32(s_ring), kBlockKeys * 128, 1024, kSwizzle128B);
      const bool leader = elect_one();
      // Waits record a failure and run on, on whatever is there: the loop ends with its tile. With votes on the outcome of every
      // wait this warp, through which every product goes, bounded the kernel: 3 750 cycles a step without any softmax, 3 100 like this.
      auto wait = [&](uint64_t* bar, uint32_t parity) { mbar_wait_or_flag(bar, parity, &s_fail, SPARGE_DEV_TIMEOUT_MMA); };
      auto issue_qk = [&](int x, uint64_t kslot) {
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; k++) {
            const uint64_t off = (k & 3) * 2 + (k >> 2) * (kBlockKeys * 128 >> 4);
            mma_f16_ss(tbase + x * 128, qd + x * (Shape::kQ >> 4) + off, kslot + off, idesc_qk, k > 0);
          }
          tc_commit(&bar_s[x]);
        }
      };
      int done = 0, steps[2] = {0, 0};                         // steps of each half so far
      for (int t = 0; done < n; t++) {
        wait(&bar_tile[t % kTileRing], (t / kTileRing) & 1);
        if (*(volatile int*)&s_fail) break;
        const int here = s_tile[t % kTileRing].units, rows = s_tile[t % kTileRing].rows, length = s_tile[t % kTileRing].length;
        const int key0 = s_tile[t % kTileRing].key;
        const bool both = rows > 128;
        int islot = 2 * done % NS;                             // of the tile of K or V in hand
        uint32_t iphase = (2 * done / NS) & 1;
        auto step_slot = [&]() {
          if (++islot == NS) islot = 0, iphase ^= 1;
        };
        wait(&bar_q[0], t & 1);
        wait(&bar_q[1], t & 1);
        wait(&bar_full[islot], iphase);
        tc_fence_after();
        const uint64_t first = kd + islot * (Shape::kTile >> 4);
        issue_qk(0, first);
        if (both) issue_qk(1, first);
        if (leader) tc_commit(&bar_empty[islot]);
        step_slot();
        for (int j = 0; j < here; j++) {
          const bool more = j + 1 < here;
          const int vslot = islot, behind = length - (key0 + j * kBlockKeys);
          wait(&bar_full[islot], iphase);
          step_slot();
          const int kslot = islot;
          if (more) {
            wait(&bar_full[islot], iphase);
            step_slot();
          }
          const uint64_t vt = vd + vslot * (Shape::kTile >> 4), kt = kd + kslot * (Shape::kTile >> 4);
          if (behind < kBlockKeys) {
            // What an earlier owner left behind the length in its last page may be anything, NaN too, and 0 x NaN is no 0.
            const int from = max(0, behind);
            for (int c = lane; c < (kBlockKeys - from) * 8; c += 32) {
#pragma unroll
              for (int h = 0; h < D / 64; h++)
                *reinterpret_cast<uint4*>(s_ring + vslot * Shape::kTile + h * (kBlockKeys * 128) + from * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          auto half_step = [&](auto which) {
            constexpr int x = decltype(which)::value;
#pragma unroll
            for (int part = 0; part < kParts; part++) {
              wait(&bar_p[x][part], steps[x] & 1);
              tc_fence_after();
              if (leader) {
#pragma unroll
                for (int k = part * (kPartKeys / 16); k < (part + 1) * (kPartKeys / 16); k++)
                  mma_f16_ts(tbase + 256 + x * 128, tbase + x * 128 + k * 8, vt + k * (2048 >> 4), idesc_pv, j > 0 || k > 0);
              }
            }
            steps[x]++;
            if (more) issue_qk(x, kt);
            else if (leader) tc_commit(&bar_o[x]);
          };
          half_step(std::integral_constant<int, 0>());
          if (both) half_step(std::integral_constant<int, 1>());
          if (leader) {
            tc_commit(&bar_empty[vslot]);
            if (more) tc_commit(&bar_empty[kslot]);
          }
        }
        if (!both && leader) tc_commit(&bar_o[1]);
        done += here;
      }
      // every product, and every word about one, has arrived before the shared memory and the tensor memory go away
      if (leader) tc_commit(&bar_end);
      const bool ended = __all_sync(0xffffffffu, mbar_wait(&bar_end, 0));
      if (lane == 0 && (!ended || *(volatile int*)&s_fail)) paged_report(p.dev_status, SPARGE_DEV_TIMEOUT_MMA);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax, epilogue
    set_registers<kSoftmaxRegs, true>();
    const int x = warp >> 2, local = (warp & 3) * 32 + lane;   // tile, row of it
    const uint32_t tlane = (uint32_t)((warp & 3) * 32) << 16, tS = tbase + x * 128 + tlane, tO = tbase + 256 + x * 128 + tlane;
    uint8_t* s_q = smem + x * Shape::kQ + local * 128;
    const bool negate = p.scale_log2 < 0.f;                    // the maximum of the products is that of the scores for a positive factor
    const float c = fmaxf(fabsf(p.scale_log2), 1e-30f);        // (0 times minus infinity would be no score)
    auto failed = [&]() { return *(volatile int*)&s_fail != 0; };

    // A row's queries, on their way while the tile before it ends.
    auto load_q = [&](const TileWork& w) {
      const int r = x * 128 + local, seq_row = w.row + r, tok = seq_row / p.group;
      const T* src = reinterpret_cast<const T*>(p.q) + (long long)(w.token + tok) * p.q_token + (long long)(w.head * p.group + seq_row - tok * p.group) * p.q_head;
      const uint32_t flip = negate ? 0x80008000u : 0u;
      uint4 v[D / 8];
#pragma unroll
      for (int k = 0; k < D / 8; k++) v[k] = r < w.rows ? reinterpret_cast<const uint4*>(src)[k] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < D / 8; k++)
        *reinterpret_cast<uint4*>(s_q + (k >> 3) * (128 * 128) + (((k & 7) ^ (local & 7)) << 4)) = make_uint4(v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q[x]);
    };

    // Both halves go through every tile, one that has no rows in it too: nobody is more than a tile ahead of another, so that a
    // barrier's parity names one phase.
    int done = 0, t = 0;
    uint32_t phase = 0;                                        // parity of the next S
    TileWork w;
    auto next_work = [&]() {
      if (done >= n) return false;
      mbar_wait_or_flag(&bar_tile[t % kTileRing], (t / kTileRing) & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
      if (failed()) return false;
      w = s_tile[t % kTileRing];
      t++;
      done += w.units;
      if (w.rows > x * 128) load_q(w);
      else if (lane == 0) mbar_arrive(&bar_q[x]);
      return true;
    };
    bool have = next_work();
    while (have) {
      if (w.rows <= x * 128) {
        mbar_wait_or_flag(&bar_o[x], (t - 1) & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
        if (failed()) break;
        have = next_work();
        continue;
      }
      const int tile = t - 1;
      const int r = x * 128 + local, seq_row = w.row + r, tok = seq_row / p.group;
      const bool mine = r < w.rows, idle = x * 128 + (warp & 3) * 32 >= w.rows;   // no row of this warp is in the tile
      const int limit = mine ? min(w.length, w.visible0 + (p.causal ? tok + 1 : 0)) : 0;
      // A score s weighs 2^((s - sub) c + off): off is -m c as it is rounded, the same for every key (what it is off by goes out in the
      // division), so that a weight takes one instruction and one rounding. Where off could be off by whole powers of two m is
      // subtracted first (sub; else 0).
      float m = -INFINITY, l = 0.f, sub = 0.f, off = 0.f;
      const int here = w.units, key0 = w.key;
      for (int j = 0; j < here; j++) {
        mbar_wait_or_flag(&bar_s[x], phase, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
        phase ^= 1;
        if (!idle) {
          tc_fence_after();
          uint32_t sr[kBlockKeys];
          tmem_ld32(tS, sr);
          tmem_ld32(tS + 32, sr + 32);
          tmem_ld32(tS + 64, sr + 64);
          tmem_ld32(tS + 96, sr + 96);
          tmem_wait_ld();
          float* s = reinterpret_cast<float*>(sr);
          const int see = limit - (key0 + j * kBlockKeys);
          const bool masked = __any_sync(0xffffffffu, see < kBlockKeys);
          if (masked) {
#pragma unroll
            for (int k = 0; k < kBlockKeys; k++) s[k] = k < see ? s[k] : -INFINITY;
          }
          const float mx = fmaxf(row_max(s), m);
          if (__any_sync(0xffffffffu, (mx - m) * c > kRescaleFrom)) {   // (from minus infinity: always; both: NaN, never)
            const float shift = mx == -INFINITY ? 0.f : -mx * c;
            const bool far = fabsf(shift) > 1048576.f;
            const float sub_to = far ? mx : 0.f, off_to = far ? 0.f : shift;
            // what the earlier weights have to be multiplied by, from the very numbers that they were formed with
            const float alpha = m == -INFINITY ? 0.f : ex2_approx(fmaf(sub - sub_to, c, off_to - off));
            m = mx, sub = sub_to, off = off_to;
            l *= alpha;
            if (j > 0) {   // the products up to the step before are in O: S of this step came behind them
#pragma unroll
              for (int d = 0; d < D; d += 16) {
                uint32_t ov[16];
                tmem_ld16(tO + d, ov);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e++) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                tmem_st16(tO + d, ov);
              }
            }
          }
          if (__any_sync(0xffffffffu, sub != 0.f)) {
#pragma unroll
            for (int k = 0; k < kBlockKeys; k++) s[k] -= sub;
          }
          const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
          float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
          for (int k0 = 0; k0 < kBlockKeys; k0 += kPartKeys) {
            uint32_t pk[kPartKeys / 2];
#pragma unroll
            for (int k = 0; k < kPartKeys; k += 4) {
              float2 a = __ffma2_rn(make_float2(s[k0 + k], s[k0 + k + 1]), c2, off2);
              float2 b = __ffma2_rn(make_float2(s[k0 + k + 2], s[k0 + k + 3]), c2, off2);
              a = make_float2(ex2_approx(a.x), ex2_approx(a.y));
              b = make_float2(ex2_approx(b.x), ex2_approx(b.y));
              sum0 = __fadd2_rn(sum0, a);                   // the sum is of the unrounded values
              sum1 = __fadd2_rn(sum1, b);
              pk[k / 2] = pack_probs<T>(a.x, a.y);
              pk[k / 2 + 1] = pack_probs<T>(b.x, b.y);
            }
            tmem_st16(tS + k0 / 2, pk);
            // The product with these keys runs under the exponentials of the next.
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_p[x][k0 / kPartKeys]);
          }
          sum0 = __fadd2_rn(sum0, sum1);
          l += sum0.x + sum0.y;
        } else if (lane < kParts) {
          mbar_arrive(&bar_p[x][lane]);
        }
        if (failed()) break;
      }
      if (failed()) break;
      const TileWork now = w;
      have = next_work();                                    // S of this tile's last step is read: its queries are not needed any more
      mbar_wait_or_flag(&bar_o[x], tile & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
      if (failed()) break;
      if (idle) continue;
      tc_fence_after();
      const bool whole = now.flags & kWhole;
      const float inv = 1.f / l;
      const int head = now.head * p.group + seq_row - tok * p.group;
      T* dst = reinterpret_cast<T*>(p.out) + (long long)(now.token + tok) * p.out_token + (long long)head * p.out_head;
      const long long part = ((long long)blockIdx.x * 2 + (now.flags & kHead ? 0 : 1)) * kTileRows + r;
#pragma unroll
      for (int d = 0; d < D; d += 32) {
        uint32_t ov[32];
        tmem_ld32(tO + d, ov);
        tmem_wait_ld();
        float* o = reinterpret_cast<float*>(ov);
        if (mine && whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(dst + d + e) =
                l != 0.f ? make_uint4(pack_probs<T>(o[e] * inv, o[e + 1] * inv), pack_probs<T>(o[e + 2] * inv, o[e + 3] * inv),
                                     pack_probs<T>(o[e + 4] * inv, o[e + 5] * inv), pack_probs<T>(o[e + 6] * inv, o[e + 7] * inv))
                        : make_uint4(0, 0, 0, 0);
        } else if (mine) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(p.part_o + part * D + d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      tc_fence_before();
      if (mine && whole && p.lse)
        p.lse[(long long)(now.token + tok) * (p.kv_heads * p.group) + head] = l != 0.f ? (m * c + log2f(l)) * 0.6931471805599453f : -INFINITY;
      if (mine && !whole) p.part_ml[part * 2] = m == -INFINITY ? m : m * c, p.part_ml[part * 2 + 1] = l;
    }
    if (lane == 0 && failed()) paged_report(p.dev_status, SPARGE_DEV_TIMEOUT_SOFTMAX);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarpT) tmem_dealloc(tbase, 512);
}

template <typename T, int D>
static int tile_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  auto kern = paged_tile_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  if (!kernel_attributes((const void*)kern, TileShape<D>::kSmemBytes, done)) return SPARGE_ERR_CUDA;
  return launch(kern, dim3(p.max_shares), dim3(kTileThreads), TileShape<D>::kSmemBytes, st, true, k, v, p) == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}

int paged_tile_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st) {
  if (dtype == SPARGE_BF16) return D == 64 ? tile_launch<__nv_bfloat16, 64>(p, k, v, st) : tile_launch<__nv_bfloat16, 128>(p, k, v, st);
  return D == 64 ? tile_launch<__half, 64>(p, k, v, st) : tile_launch<__half, 128>(p, k, v, st);
}

}  // namespace sparge
