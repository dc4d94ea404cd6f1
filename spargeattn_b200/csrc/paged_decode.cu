// Attention of a few rows over a paged cache: tiles of 16 rows (one token of up to 16 query heads to a key head, or a few tokens
// of fewer).
//
// Every key and value is read once for 16 rows, 4 multiply-adds a byte each way, so HBM bounds it by far: what the kernel has to
// do is keep enough bytes in flight (a GPU at 6.5 TB/s with a microsecond of latency wants 44 KB of them on each SM) and stay
// out of their way. One CTA on each SM takes an equal run of the call's units (paged_schedule.cuh), whatever sequences and heads it
// falls on, and a ring of three 64 KB stages (K and V of 128 keys; D = 64: six of 32 KB) keeps two loading while one is used.
// The loading warp runs ahead over the borders of tiles and sequences.
//
// Four warps take 32 keys of a unit each, with a running maximum, sum and output of their own, and are joined only where a
// tile ends: inside the loop they wait for nothing but the stage. The products are mma.sync m16n8k16, 32-bit accumulators:
// 16 rows are its M, where tcgen05 would compute 128. A 16-key step takes 32 of them, about 64 cycles of an SM for 8 KB that
// HBM takes 350 cycles to bring.
#include <atomic>

#include "launch.cuh"
#include "paged.cuh"

namespace sparge {

constexpr int kDecodeWarps = 4, kDecodeThreads = 32 * (kDecodeWarps + 1);
constexpr int kWarpKeys = kBlockKeys / kDecodeWarps;

template <int D>
struct DecodeShape {
  static constexpr int kTile = kBlockKeys * D * 2;
  static constexpr int kStage = 2 * kTile;                     // K, V
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kJoin = kDecodeWarps * kDecodeRows * D * 4;
  static constexpr int kSmemBytes = 1024 + kStages * kStage + kJoin;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Keys and values of a unit, a piece of up to 128 rows of one page after the other: [piece][half][rows][128 bytes]. A copy brings
// both halves: with a copy for each, 2 KB of a 16-token page at a time, the copy engine was what bounded the kernel (4 150 cycles a
// unit where HBM takes 2 850).
template <int D>
__device__ __forceinline__ void load_unit(const PagedParams& p, uint8_t* dst, const CUtensorMap* map_k, const CUtensorMap* map_v, uint64_t* bar,
                                          int entry, int key0, int length, int head, int lane) {
  const int box = min(p.page_size, kBlockKeys), boxes = kBlockKeys / box;
  if (lane < 2 * boxes) {
    const int of_v = lane >= boxes, piece = lane - of_v * boxes, key = key0 + piece * box;
    tma_load_5d(dst + of_v * (kBlockKeys * D * 2) + piece * box * D * 2, of_v ? map_v : map_k, bar, 0, key & (p.page_size - 1), 0, head,
                page_of(p, entry, key, length));
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kDecodeThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PagedParams p) {
  using Shape = DecodeShape<D>;
  constexpr int ST = Shape::kStages, R = kDecodeRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_o = reinterpret_cast<float*>(smem + ST * Shape::kStage);       // [warp][row][D]
  __shared__ uint64_t bar_full[ST], bar_empty[ST], bar_join[2];
  __shared__ Unit s_unit[ST];
  __shared__ float s_ml[kDecodeWarps][R][2];
  __shared__ ShareSearch s_search;
  __shared__ int s_fail;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < ST; i++) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], kDecodeWarps);
    }
    mbar_init(&bar_join[0], kDecodeWarps);
    mbar_init(&bar_join[1], kDecodeWarps);
    mbar_fence_init();
    s_fail = 0;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  pdl_wait();                                                             // lengths, tables and queries come from the kernels before
  zero_rest<T, D>(p, blockIdx.x * kDecodeThreads + tid, gridDim.x * kDecodeThreads);
  long long begin, end, units;
  int shares;
  Place<R> at;
  find_share<kDecodeThreads>(p, s_search, begin, end, units, shares, at);
  if (begin >= end) {
    if (tid == 0) note_join(p, begin, units, shares, at);
    return;
  }

  if (warp == kDecodeWarps) {
    // ------------------------------------------------------------------ loads
    const int n = (int)(end - begin);
    const int box = min(p.page_size, kBlockKeys), piece_key = (lane & (kBlockKeys / box - 1)) * box;   // of this lane's copy
    auto entry_at = [&]() { return table_entry(p, at.seq, (int)(at.block * kBlockKeys) + piece_key, (int)at.w.length); };
    bool ok = true, first_piece = true, fresh = true;
    int issued = 0, entry = entry_at();
    for (int i = 0; i < n; i++) {
      const int slot = i % ST;
      const unsigned blocks = at.w.blocks(at.tile);
      const bool last = at.block + 1 == blocks || i + 1 == n;
      const int key = (int)(at.block * kBlockKeys), length = (int)at.w.length, head = at.head;
      Unit u;
      const bool whole = at.first >= begin && at.first + blocks <= end;
      u.flags = (fresh ? kFirst : 0) | (last ? kLast : 0) | (whole ? kWhole : 0) | (first_piece ? kHead : 0);
      u.token = at.token, u.row = (int)(at.tile * R), u.rows = (int)at.w.tile_rows(at.tile), u.head = head;
      u.key = key, u.length = length;
      u.visible0 = p.causal ? length - (int)at.w.tokens : length;
      // The next unit's place and pages are looked up while a stage becomes free; in front of that, behind the copies.
      const int now = entry;
      auto advance = [&]() {
        fresh = last;
        if (last) first_piece = false;
        if (i + 1 < n) {
          if (!last) at.block++;
          else next_tile(p, at);
          entry = entry_at();
        }
      };
      if (i >= ST) {
        advance();
        ok = __all_sync(0xffffffffu, mbar_wait(&bar_empty[slot], ((i / ST) - 1) & 1));
      }
      if (!ok || __any_sync(0xffffffffu, *(volatile int*)&s_fail)) break;
      if (lane == 0) {
        s_unit[slot] = u;
        mbar_arrive_expect_tx(&bar_full[slot], Shape::kStage);
      }
      __syncwarp();
      load_unit<D>(p, smem + slot * Shape::kStage, &map_k, &map_v, &bar_full[slot], now, key, length, head, lane);
      issued = i + 1;
      if (i < ST) advance();
    }
    if (!ok && lane == 0) {
      paged_report(p.dev_status, SPARGE_DEV_TIMEOUT_PRODUCER);
      *(volatile int*)&s_fail = SPARGE_DEV_TIMEOUT_PRODUCER;
    }
    if (issued < n)   // our own copies land before the shared memory goes away
      for (int i = max(0, issued - ST); i < issued; i++) mbar_wait(&bar_full[i % ST], (i / ST) & 1);
    return;
  }

  // -------------------------------------------------------------------- products
  const int g = lane >> 2, q4 = lane & 3;            // fragment row (and row + 8), column pair
  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2], l[2];
  int limit[2];                                      // keys that the rows see
  int joins = 0;
  const int n = (int)(end - begin);
  // where the warp's keys lie in a tile: rows of a piece of a page are together
  const int box = min(p.page_size, kBlockKeys), half_bytes = box * 128;
  auto row_at = [&](int row) { return (row & ~(box - 1)) * (D * 2) + (row & (box - 1)) * 128; };
  uint32_t k_at[kWarpKeys / 8], v_at[kWarpKeys / 16];
#pragma unroll
  for (int t = 0; t < kWarpKeys / 8; t++) k_at[t] = row_at(warp * kWarpKeys + t * 8 + (lane & 7));
#pragma unroll
  for (int t = 0; t < kWarpKeys / 16; t++) v_at[t] = row_at(warp * kWarpKeys + t * 16 + (lane & 15));
  auto load_q = [&](int token, int row, int rows, int kv_head) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const int r = g + 8 * x, seq_row = row + r, tok = seq_row / p.group;
      const T* src = reinterpret_cast<const T*>(p.q) + (long long)(token + tok) * p.q_token + (long long)(kv_head * p.group + seq_row - tok * p.group) * p.q_head;
#pragma unroll
      for (int k = 0; k < D / 16; k++) {
        qf[k][x] = r < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 2 * q4) : 0u;
        qf[k][x + 2] = r < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 + 2 * q4) : 0u;
      }
    }
  };
  load_q(at.token, (int)(at.tile * R), (int)at.w.tile_rows(at.tile), at.head);
  if (tid == 0) note_join(p, begin, units, shares, at);     // (in front of the search's other work it cost a short call 0.7 us)
  for (int i = 0; i < n; i++) {
    const int slot = i % ST;
    mbar_wait_or_flag(&bar_full[slot], (i / ST) & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
    if (*(volatile int*)&s_fail) break;
    const Unit u = s_unit[slot];
    if (u.flags & kFirst) {
      if (i > 0) load_q(u.token, u.row, u.rows, u.head);               // (the first tile's are under way)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int r = g + 8 * x;
        limit[x] = r < u.rows ? min(u.length, u.visible0 + (p.causal ? (u.row + r) / p.group + 1 : 0)) : 0;
        m[x] = -INFINITY, l[x] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < D / 8; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    }
    const int key0 = u.key + warp * kWarpKeys;
    if (key0 < u.length) {
      const uint32_t sk = smem_u32(smem + slot * Shape::kStage), sv = sk + Shape::kTile;
      float s[kWarpKeys / 8][4];
#pragma unroll
      for (int t = 0; t < kWarpKeys / 8; t++) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
      // S = Q K^T: a load brings 8 keys by 32 channels, two steps of K = 16
#pragma unroll
      for (int k = 0; k < D / 32; k++) {
#pragma unroll
        for (int t = 0; t < kWarpKeys / 8; t++) {
          const int chunk = (k & 1) * 4 + (lane >> 3);
          uint32_t b[4];
          ldmatrix_x4<false>(b, sk + (k >> 1) * half_bytes + k_at[t] + ((chunk ^ (lane & 7)) << 4));
          mma_16816<T>(s[t], qf[2 * k], b[0], b[1]);
          mma_16816<T>(s[t], qf[2 * k + 1], b[2], b[3]);
        }
      }
      const bool masked = key0 + kWarpKeys > min(limit[0], limit[1]);   // some score of this thread is not seen
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int t = 0; t < kWarpKeys / 8; t++) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          s[t][c] *= p.scale_log2;
          if (masked && key0 + t * 8 + 2 * q4 + (c & 1) >= limit[c >> 1]) s[t][c] = -INFINITY;
          top[c >> 1] = fmaxf(top[c >> 1], s[t][c]);
        }
      }
      float alpha[2], base[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        top[x] = fmaxf(top[x], m[x]);
        base[x] = top[x] == -INFINITY ? 0.f : top[x];               // a row that has seen nothing yet
        alpha[x] = ex2_approx(m[x] - base[x]);
      }
      if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
        for (int d = 0; d < D / 8; d++) {
          o[d][0] *= alpha[0], o[d][1] *= alpha[0];
          o[d][2] *= alpha[1], o[d][3] *= alpha[1];
        }
        l[0] *= alpha[0], l[1] *= alpha[1];
        m[0] = top[0], m[1] = top[1];
      }
      uint32_t pf[kWarpKeys / 16][4];
#pragma unroll
      for (int t = 0; t < kWarpKeys / 8; t++) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float a = ex2_approx(s[t][2 * x] - base[x]), b = ex2_approx(s[t][2 * x + 1] - base[x]);
          l[x] += a + b;                                            // the sum is of the unrounded values
          pf[t / 2][(t & 1) * 2 + x] = pack_pair<T>(a, b);
        }
      }
      // What an earlier owner left behind the length in its last page may be anything, NaN too, and 0 x NaN is no 0. (V's
      // other rows behind the length are the copy engine's zeros.)
      if (key0 + kWarpKeys > u.length) {
        for (int r = u.length - key0; r < kWarpKeys; r++) {
#pragma unroll
          for (int h = 0; h < D / 64; h++)
            *reinterpret_cast<uint32_t*>(smem + slot * Shape::kStage + Shape::kTile + h * half_bytes + row_at(warp * kWarpKeys + r) + lane * 4) = 0u;
        }
        fence_proxy_async_smem();                                   // the copy engine writes here next
        __syncwarp();
      }
      // O += P V: a load brings 16 keys by 16 channels
#pragma unroll
      for (int t = 0; t < kWarpKeys / 16; t++) {
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
          const int chunk = (d & 3) * 2 + (lane >> 4);
          uint32_t b[4];
          ldmatrix_x4<true>(b, sv + (d >> 2) * half_bytes + v_at[t] + ((chunk ^ (lane & 7)) << 4));
          mma_16816<T>(o[2 * d], pf[t], b[0], b[1]);
          mma_16816<T>(o[2 * d + 1], pf[t], b[2], b[3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_empty[slot]);

    if (u.flags & kLast) {
      // ---------------------------------------------------------------- the four warps' parts become one
#pragma unroll
      for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (q4 == 0) s_ml[warp][g + 8 * x][0] = m[x], s_ml[warp][g + 8 * x][1] = l[x];
      }
      // groups of eight channels change places by row, so that the rows of a store fall on different banks
      float* mine = s_o + warp * R * D;
#pragma unroll
      for (int d = 0; d < D / 8; d++) {
        *reinterpret_cast<float2*>(mine + g * D + ((d ^ g) * 8) + 2 * q4) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(mine + (g + 8) * D + ((d ^ g) * 8) + 2 * q4) = make_float2(o[d][2], o[d][3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_join[0]);
      mbar_wait_or_flag(&bar_join[0], joins & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
      if (*(volatile int*)&s_fail) break;
      // eight threads a row, D / 8 channels each
      constexpr int C = D / 8;
      const int r = tid >> 3, part = tid & 7;
      float w[kDecodeWarps], top = -INFINITY, sum = 0.f, acc[C];
#pragma unroll
      for (int j = 0; j < kDecodeWarps; j++) top = fmaxf(top, s_ml[j][r][0]);
#pragma unroll
      for (int j = 0; j < kDecodeWarps; j++) {
        w[j] = top == -INFINITY ? 0.f : ex2_approx(s_ml[j][r][0] - top);
        sum += w[j] * s_ml[j][r][1];
      }
#pragma unroll
      for (int c = 0; c < C; c += 8) {
        const int group8 = (part * C + c) / 8;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float x = 0.f;
#pragma unroll
          for (int j = 0; j < kDecodeWarps; j++) x += w[j] * s_o[(j * R + r) * D + ((group8 ^ (r & 7)) * 8) + e];
          acc[c + e] = x;
        }
      }
      if (r < u.rows) {
        if (u.flags & kWhole) {
          const int seq_row = u.row + r, tok = seq_row / p.group, head = u.head * p.group + seq_row - tok * p.group;
          const float inv = sum != 0.f ? 1.f / sum : 0.f;
          T* dst = reinterpret_cast<T*>(p.out) + (long long)(u.token + tok) * p.out_token + (long long)head * p.out_head + part * C;
#pragma unroll
          for (int c = 0; c < C; c += 8) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; e++) pk[e] = pack_pair<T>(acc[c + 2 * e] * inv, acc[c + 2 * e + 1] * inv);
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
          if (p.lse && part == 0)
            p.lse[(long long)(u.token + tok) * (p.kv_heads * p.group) + head] = sum != 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        } else {
          const long long at_row = ((long long)blockIdx.x * 2 + (u.flags & kHead ? 0 : 1)) * R + r;
          float* dst = p.part_o + at_row * D + part * C;
#pragma unroll
          for (int c = 0; c < C; c += 4) *reinterpret_cast<float4*>(dst + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
          if (part == 0) p.part_ml[at_row * 2] = top, p.part_ml[at_row * 2 + 1] = sum;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_join[1]);          // the parts are read: the next tile's may overwrite them
      if (i + 1 < n) mbar_wait_or_flag(&bar_join[1], joins & 1, &s_fail, SPARGE_DEV_TIMEOUT_SOFTMAX);
      joins++;
    }
  }
  if (lane == 0 && *(volatile int*)&s_fail) paged_report(p.dev_status, SPARGE_DEV_TIMEOUT_SOFTMAX);
}

template <typename T, int D>
static int decode_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  auto kern = paged_decode_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  if (!kernel_attributes((const void*)kern, DecodeShape<D>::kSmemBytes, done)) return SPARGE_ERR_CUDA;
  return launch(kern, dim3(p.max_shares), dim3(kDecodeThreads), DecodeShape<D>::kSmemBytes, st, true, k, v, p) == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}

int paged_decode_launch(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, int D, int dtype, cudaStream_t st) {
  if (dtype == SPARGE_BF16) return D == 64 ? decode_launch<__nv_bfloat16, 64>(p, k, v, st) : decode_launch<__nv_bfloat16, 128>(p, k, v, st);
  return D == 64 ? decode_launch<__half, 64>(p, k, v, st) : decode_launch<__half, 128>(p, k, v, st);
}

}  // namespace sparge
