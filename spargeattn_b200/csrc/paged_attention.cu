// Attention of new tokens over a paged cache: the entry point, and the kernel that joins tiles which several CTAs worked on.
#include <algorithm>
#include <cmath>

#include "launch.cuh"
#include "paged.cuh"
#include "tensor_map.cuh"

namespace sparge {

// One warp per row of a tile that lies in several shares. The pieces' maxima and sums are read 32 at a time, then their outputs
// in the order of the shares, so that a result does not depend on who was first. A block for every share's border and eight
// rows; most find that they have nothing to do: that a border is the first one inside its tile is seen from the two starts.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedParams p, int rows) {
  pdl_wait();
  const ShareStart total = p.starts[p.max_shares];
  const long long units = total.begin;
  const int shares = (int)total.first, c = blockIdx.x + 1;
  if (c >= shares) return;
  const ShareStart a = p.starts[c];
  const long long before = share_begin(c - 1, units, shares);
  if (a.begin <= a.first || before > a.first) return;      // between two tiles, or not the first border inside this one
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  int pieces = 2;                                          // of the shares c - 1, c, ...
  while (c - 1 + pieces < shares && share_begin(c - 1 + pieces, units, shares) < a.last) pieces++;
  // a share's first piece has slot 0; the first share of the tile may have begun before it
  const auto slot = [&](int i) { return ((long long)(c - 1 + i) * 2 + (i == 0 && before < a.first)) * rows + r; };
  float top = -INFINITY;
  for (int i = lane; i < pieces; i += 32) top = fmaxf(top, p.part_ml[slot(i) * 2]);
  top = warp_max(top);
  float sum = 0.f, acc[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; d++) acc[d] = 0.f;
  for (int i0 = 0; i0 < pieces; i0 += 32) {
    float w = 0.f;
    if (i0 + lane < pieces) {
      w = top == -INFINITY ? 1.f : ex2_approx(p.part_ml[slot(i0 + lane) * 2] - top);   // (no key seen: sums of 0, or of NaN)
      sum += w * p.part_ml[slot(i0 + lane) * 2 + 1];
    }
    const int here = min(32, pieces - i0);
#pragma unroll 8
    for (int i = 0; i < here; i++) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const float* src = p.part_o + slot(i0 + i) * D + lane * (D / 32);
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
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int seq_row = a.row + r, tok = seq_row / p.group, head = a.head * p.group + seq_row - tok * p.group;
  T* dst = reinterpret_cast<T*>(p.out) + (long long)(a.token + tok) * p.out_token + (long long)head * p.out_head + lane * (D / 32);
#pragma unroll
  for (int d = 0; d < D / 32; d++) dst[d] = Elem<T>::from_float(acc[d] * inv);
  if (p.lse && lane == 0)
    p.lse[(long long)(a.token + tok) * (p.kv_heads * p.group) + head] = sum != 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

// 16-bit pages [pages, heads, page_size, D] by their strides; a copy takes up to kBlockKeys rows of 64 channels of one page.
static bool page_map(CUtensorMap* m, const void* ptr, const long long* st, const sparge_cache& c) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads, (cuuint64_t)c.num_pages};
  cuuint64_t strides[3] = {2 * (cuuint64_t)st[2], 2 * (cuuint64_t)st[1], 2 * (cuuint64_t)st[0]};
  cuuint32_t box[4] = {64, (cuuint32_t)std::min(c.page_size, kBlockKeys), 1, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, c.dtype == SPARGE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims,
             strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernel: tiles of 16 rows or of 256.
static int tile_rows(int group, int max_chunk) { return (long long)group * max_chunk <= kDecodeRows ? kDecodeRows : kTileRows; }

static size_t starts_bytes(int shares) { return (sizeof(ShareStart) * (shares + 1) + 255) / 256 * 256; }

}  // namespace sparge

extern "C" size_t sparge_paged_attention_workspace_bytes(int q_heads, int kv_heads, int D, int max_chunk) {
  using namespace sparge;
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || D <= 0) return 0;
  const size_t shares = sm_count(), rows = tile_rows(q_heads / kv_heads, max_chunk);
  return starts_bytes((int)shares) + shares * 2 * rows * (D + 2) * sizeof(float);
}

extern "C" int sparge_paged_attention(const sparge_paged_attention_args* a, sparge_stream_t stream) {
  using namespace sparge;
  if (!a) return SPARGE_ERR_NULL;
  const sparge_cache& c = a->cache;
  if (c.tokens < 0 || c.sequences < 0 || c.kv_heads <= 0 || a->q_heads <= 0 || a->q_heads % c.kv_heads || (c.D != 64 && c.D != 128) ||
      (c.dtype != SPARGE_F16 && c.dtype != SPARGE_BF16) || c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)) ||
      c.table_width < 0 || c.num_pages <= 0 || (!c.cu_seqlens && c.tokens != c.sequences) || a->max_chunk < 0 || !(a->scale > -INFINITY && a->scale < INFINITY))
    return SPARGE_ERR_INVALID_ARG;
  if ((long long)c.table_width * c.page_size > 0x7fffff00LL || (long long)c.tokens * (a->q_heads / c.kv_heads) > 0x7fffff00LL) return SPARGE_ERR_TOO_LARGE;
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
  if (!page_map(&k, c.k_pages, c.k_st, c) || !page_map(&v, c.v_pages, c.v_st, c)) return SPARGE_ERR_CUDA;
  p.q = a->q, p.out = a->out, p.lse = a->lse;
  p.q_token = a->q_st[0], p.q_head = a->q_st[1], p.out_token = a->out_st[0], p.out_head = a->out_st[1], p.table_stride = c.table_stride;
  p.cu = c.cu_seqlens, p.seq_lens = c.seq_lens, p.table = c.page_table;
  p.tokens = c.tokens, p.sequences = c.sequences, p.width = c.table_width, p.num_pages = c.num_pages, p.page_size = c.page_size;
  p.kv_heads = c.kv_heads, p.group = group, p.causal = a->is_causal != 0, p.zero_rest = a->zero_rest != 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.starts = reinterpret_cast<ShareStart*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(a->workspace) + starts_bytes(p.max_shares));
  p.part_ml = p.part_o + (size_t)p.max_shares * 2 * rows * c.D;
  p.dev_status = a->dev_status;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rc = rows == kDecodeRows ? paged_decode_launch(p, k, v, c.D, c.dtype, st) : paged_tile_launch(p, k, v, c.D, c.dtype, st);
  if (rc != SPARGE_OK || p.max_shares < 2) return rc;
  const dim3 grid(p.max_shares - 1, (rows + 7) / 8);
#define SPARGE_JOIN(T, D) launch(paged_join_kernel<T, D>, grid, dim3(256), 0, st, true, p, rows)
  const cudaError_t e = c.dtype == SPARGE_BF16 ? (c.D == 64 ? SPARGE_JOIN(__nv_bfloat16, 64) : SPARGE_JOIN(__nv_bfloat16, 128))
                                               : (c.D == 64 ? SPARGE_JOIN(__half, 64) : SPARGE_JOIN(__half, 128));
#undef SPARGE_JOIN
  return e == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}
