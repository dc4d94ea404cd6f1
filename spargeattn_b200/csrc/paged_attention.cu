// Attention of new tokens over a paged cache: the entry point, and the kernel that joins tiles which several CTAs worked on.
#include <algorithm>
#include <cmath>

#include "launch.cuh"
#include "paged.cuh"
#include "tensor_map.cuh"

namespace sparge {

// Tiles that lie in several shares. Every border between two shares has kJoinBlocks blocks; those of all borders inside a tile work on
// its rows together, so that one token over a long context (36 borders for 16 rows) and a chunk (one border for 256) find the
// warps that they need: up to eight for a row, which take its pieces in turn. Maxima and sums are read 32 pieces at a time, then
// the outputs, in an order that does not depend on who was first.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
constexpr int kJoinBlocks = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(PagedParams p, int rows) {
  __shared__ float s_part[kJoinWarps][D + 1];
  pdl_wait();
  const ShareJoin a = p.joins[blockIdx.x + 1];
  if (a.pieces == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = (a.pieces - 1) * kJoinBlocks;
  int per_row = 1;                                         // warps
  while (per_row < kJoinWarps && 2 * per_row * a.rows <= blocks * kJoinWarps) per_row *= 2;
  const int sub = warp & (per_row - 1), at_once = kJoinWarps / per_row, mine = warp / per_row;
  for (int r0 = (a.border * kJoinBlocks + blockIdx.y) * at_once; r0 < a.rows; r0 += blocks * at_once) {
    const int r = min(r0 + mine, a.rows - 1);              // (a row twice: the same values)
    const auto slot = [&](int i) { return (long long)(i == 0 ? a.slot : 2 * (a.first + i)) * rows + r; };
    float top = -INFINITY;
    for (int i = lane; i < a.pieces; i += 32) top = fmaxf(top, p.part_ml[slot(i) * 2]);
    top = warp_max(top);
    float sum = 0.f, acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; d++) acc[d] = 0.f;
    for (int i0 = sub; i0 < a.pieces; i0 += 32 * per_row) {
      const int own = i0 + lane * per_row;
      float w = 0.f;
      if (own < a.pieces) {
        w = top == -INFINITY ? 1.f : ex2_approx(p.part_ml[slot(own) * 2] - top);   // (no key seen: sums of 0, or of NaN)
        sum += w * p.part_ml[slot(own) * 2 + 1];
      }
      const int here = min(32, (a.pieces - i0 + per_row - 1) / per_row);
#pragma unroll 8
      for (int i = 0; i < here; i++) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const float* src = p.part_o + slot(i0 + i * per_row) * D + lane * (D / 32);
        if constexpr (D == 128) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          acc[0] += wi * x.x, acc[1] += wi * x.y, acc[2] += wi * x.z, acc[3] += wi * x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src);
          acc[0] += wi * x.x, acc[1] += wi * x.y;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (per_row > 1) {
#pragma unroll
      for (int d = 0; d < D / 32; d++) s_part[warp][lane * (D / 32) + d] = acc[d];
      if (lane == 0) s_part[warp][D] = sum;
      __syncthreads();
      if (sub == 0) {
        for (int j = 1; j < per_row; j++) {
#pragma unroll
          for (int d = 0; d < D / 32; d++) acc[d] += s_part[warp + j][lane * (D / 32) + d];
          sum += s_part[warp + j][D];
        }
      }
      __syncthreads();
    }
    if (sub == 0 && r0 + mine < a.rows) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      const int seq_row = a.row + r, tok = seq_row / p.group, head = a.head * p.group + seq_row - tok * p.group;
      T* dst = reinterpret_cast<T*>(p.out) + (long long)(a.token + tok) * p.out_token + (long long)head * p.out_head + lane * (D / 32);
#pragma unroll
      for (int d = 0; d < D / 32; d++) dst[d] = Elem<T>::from_float(acc[d] * inv);
      if (p.lse && lane == 0)
        p.lse[(long long)(a.token + tok) * (p.kv_heads * p.group) + head] = sum != 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
  }
}

template <typename T, int D>
static cudaError_t join_launch(const PagedParams& p, int rows, cudaStream_t st) {
  return launch(paged_join_kernel<T, D>, dim3(p.max_shares - 1, kJoinBlocks), dim3(kJoinThreads), 0, st, true, p, rows);
}

// 16-bit pages [pages, heads, page_size, D] by their strides; a copy takes up to kBlockKeys rows of one page, `halves` times 64
// channels.
static bool page_map(CUtensorMap* m, const void* ptr, const long long* st, const sparge_cache& c, int halves) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  cuuint64_t dims[5] = {64, (cuuint64_t)c.page_size, (cuuint64_t)c.D / 64, (cuuint64_t)c.kv_heads, (cuuint64_t)c.num_pages};
  cuuint64_t strides[4] = {2 * (cuuint64_t)st[2], 128, 2 * (cuuint64_t)st[1], 2 * (cuuint64_t)st[0]};
  cuuint32_t box[5] = {64, (cuuint32_t)std::min(c.page_size, kBlockKeys), (cuuint32_t)halves, 1, 1}, es[5] = {1, 1, 1, 1, 1};
  return enc(m, c.dtype == SPARGE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(ptr), dims,
             strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernel: tiles of 16 rows or of 256. The first reads K and V once for 16 rows and keeps up with HBM; the second's step takes
// the same time for 1 row and for 128. Measured, us, 16 rows / 256 rows, 32 heads to 4, 16 sequences of 8 000 keys: rows 16: 45 / 62
// at D = 64, 59 / 74 at D = 128; rows 32: 79 / 57 and 90 / 73; rows 64: 144 / 58 and 181 / 75. One sequence of 30 000 keys, rows 16:
// 18.6 / 24.4 and 20.8 / 27.9; rows 32: 26.9 / 23.2 and 29.9 / 27.9.
static int tile_rows(int group, int max_chunk) { return (long long)group * max_chunk <= kDecodeRows ? kDecodeRows : kTileRows; }

static size_t joins_bytes(int shares) { return (sizeof(ShareJoin) * shares + 255) / 256 * 256; }

}  // namespace sparge

extern "C" size_t sparge_paged_attention_workspace_bytes(int q_heads, int kv_heads, int D, int max_chunk) {
  using namespace sparge;
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || D <= 0) return 0;
  const size_t shares = sm_count(), rows = tile_rows(q_heads / kv_heads, max_chunk);
  return joins_bytes((int)shares) + shares * 2 * rows * (D + 2) * sizeof(float);
}

extern "C" int sparge_paged_attention(const sparge_paged_attention_args* a, sparge_stream_t stream) {
  using namespace sparge;
  if (!a) return SPARGE_ERR_NULL;
  const sparge_cache& c = a->cache;
  if (c.tokens < 0 || c.sequences < 0 || c.kv_heads <= 0 || a->q_heads <= 0 || a->q_heads % c.kv_heads || (c.D != 64 && c.D != 128) ||
      (c.dtype != SPARGE_F16 && c.dtype != SPARGE_BF16) || c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)) ||
      c.table_width < 0 || c.num_pages <= 0 || (!c.cu_seqlens && c.tokens != c.sequences) || a->max_chunk < 0 || !(a->scale > -INFINITY && a->scale < INFINITY))
    return SPARGE_ERR_INVALID_ARG;
  if ((long long)c.table_width * c.page_size > 0x7fffff00LL || (long long)c.tokens * (a->q_heads / c.kv_heads) > 0x7fffff00LL ||
      (long long)c.table_width * c.page_size / kBlockKeys * c.kv_heads > 0x7fffff00LL) return SPARGE_ERR_TOO_LARGE;
  if (c.tokens == 0) return SPARGE_OK;
  if (!a->q || !a->out || !c.k_pages || !c.v_pages || !a->workspace) return SPARGE_ERR_NULL;
  if (c.sequences && (!c.seq_lens || (c.table_width && !c.page_table))) return SPARGE_ERR_NULL;
  for (const void* x : {a->q, (const void*)a->out, (const void*)c.k_pages, (const void*)c.v_pages, (const void*)a->workspace})
    if (reinterpret_cast<uintptr_t>(x) % 16) return SPARGE_ERR_INVALID_ARG;
  for (long long st : {a->q_st[0], a->q_st[1], a->out_st[0], a->out_st[1], c.k_st[0], c.k_st[1], c.k_st[2], c.v_st[0], c.v_st[1], c.v_st[2]})
    if (st % 8 || st < 0) return SPARGE_ERR_INVALID_ARG;
  const int group = a->q_heads / c.kv_heads, rows = tile_rows(group, a->max_chunk);
  PagedParams p = {};
  p.max_shares = sm_count();
  if (a->workspace_bytes < sparge_paged_attention_workspace_bytes(a->q_heads, c.kv_heads, c.D, a->max_chunk)) return SPARGE_ERR_INVALID_ARG;
  CUtensorMap k, v;
  const int halves = rows == kDecodeRows ? c.D / 64 : 1;
  if (!page_map(&k, c.k_pages, c.k_st, c, halves) || !page_map(&v, c.v_pages, c.v_st, c, halves)) return SPARGE_ERR_CUDA;
  p.q = a->q, p.out = a->out, p.lse = a->lse;
  p.q_token = a->q_st[0], p.q_head = a->q_st[1], p.out_token = a->out_st[0], p.out_head = a->out_st[1], p.table_stride = c.table_stride;
  p.cu = c.cu_seqlens, p.seq_lens = c.seq_lens, p.table = c.page_table;
  p.tokens = c.tokens, p.sequences = c.sequences, p.width = c.table_width, p.num_pages = c.num_pages, p.page_size = c.page_size;
  while ((1 << p.page_shift) < c.page_size) p.page_shift++;
  p.kv_heads = c.kv_heads, p.group = group, p.causal = a->is_causal != 0, p.zero_out = a->zero_rest && a->zero_rest != 2, p.zero_lse = a->lse && a->zero_rest;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.joins = reinterpret_cast<ShareJoin*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + joins_bytes(p.max_shares));
  p.part_ml = p.part_o + (size_t)p.max_shares * 2 * rows * c.D;
  p.dev_status = a->dev_status;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rc = rows == kDecodeRows ? paged_decode_launch(p, k, v, c.D, c.dtype, st) : paged_tile_launch(p, k, v, c.D, c.dtype, st);
  if (rc != SPARGE_OK || p.max_shares < 2) return rc;
  const cudaError_t e = c.dtype == SPARGE_BF16 ? (c.D == 64 ? join_launch<__nv_bfloat16, 64>(p, rows, st) : join_launch<__nv_bfloat16, 128>(p, rows, st))
                                               : (c.D == 64 ? join_launch<__half, 64>(p, rows, st) : join_launch<__half, 128>(p, rows, st));
  return e == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}
