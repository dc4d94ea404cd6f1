// Rotary positions, and the write of new tokens into a paged key/value cache, which turns keys and queries on its way.
//
//   (a, b) -> magnitude (a cos t - b sin t, a sin t + b cos t),  t = position * frequency
//
// The phase is formed in 64 bits and reduced to half a turn before it becomes a float: at position 10^6 a phase of 32 bits is
// off by 0.06 radians. The products are 32-bit and rounded once to the tensor's type.
//
// Every element is read and written once, so HBM bounds it; what the kernel must not do is spend its time on the angles. A
// phase and its sine cost about 60 instructions, and a token's pairs are the same for all its heads: a block computes those of
// its tokens once into shared memory, and a thread keeps the ones of its channels in registers while it walks the heads.
#include "common.cuh"
#include "launch.cuh"

namespace sparge {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 8;      // most tokens of a block: a power of two

// What keeps HBM busy is blocks on an SM, and heads loaded together; both take registers. Forward and backward pass of
// [1,12,32760,128] bf16 queries and keys, neighbouring pairs: six blocks of two heads 144 us (20 bytes of a thread spilled), five 151,
// seven 160, four of four heads 153, eight of one 164. A unit of two halves needs more: partial rotation of fp16 [4097, 16 + 4, 128] with
// four blocks 10.0 us (11.0 in later runs), five 14.1, six 25.7. Without a rotation there is nothing else to hold: four heads (17.0 us for
// 9 450 tokens' keys and values, two 19.1). Tokens of a block: eight 144 us, four 176, sixteen 150. fp32 takes the same shapes and spills
// more (76 bytes of neighbouring pairs, 114 of half-apart ones); it was not timed apart.
template <bool INTER, bool ROT>
struct RotShape {
  static constexpr int kAhead = ROT ? 2 : 4, kBlocks = ROT && INTER ? 6 : 4;
};

struct RotSlot {                   // q, k or v
  const void* x;
  void* y;                         // paged: the pages
  long long xb, xh, xn;            // strides of the source: batch, head, token
  long long yb, yh, yn;            // of the destination; paged: page, head, row
  int heads;
  bool rotate, paged;
};

struct RotParams {
  RotSlot slot[3];
  int slots, B, N, D, pairs, axes, sections[4];
  const void* positions;
  bool pos64, inverse;
  long long pos_st[3];
  const double* freq;
  float magnitude;
  int tokens_per_block, tok_shift;   // a power of two
  // append
  const int32_t *table, *seq_lens, *cu;
  const unsigned char* served;
  long long table_stride;
  int sequences, width, num_pages, page_size;
  int32_t* dev_status;
};

// V consecutive elements as they lie in memory.
template <typename T, int V>
struct Raw {
  T v[V];
};
template <typename T, int V, bool VEC>
__device__ __forceinline__ Raw<T, V> raw_load(const T* p) {
  Raw<T, V> r;
  if constexpr (VEC) {
    constexpr int kWords = V * (int)sizeof(T) / 16;
    uint4 w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
    memcpy(&r, w, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = p[i];
  }
  return r;
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void raw_store(T* p, const Raw<T, V>& r) {
  if constexpr (VEC) {
    constexpr int kWords = V * (int)sizeof(T) / 16;
    uint4 w[kWords];
    memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < kWords; i++) reinterpret_cast<uint4*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = r.v[i];
  }
}

// The batch that a token lies in. A division of 64 bits is as many instructions as turning two heads.
__device__ __forceinline__ int batch_of(const RotParams& p, long long t) {
  if (p.B == 1) return 0;
  return t >> 32 ? (int)(t / p.N) : (int)((unsigned)t / (unsigned)p.N);
}

// Two neighbours rounded by one instruction where there is one.
__device__ __forceinline__ void round_two(float& x, float& y, float u, float w) { x = u, y = w; }
__device__ __forceinline__ void round_two(__half& x, __half& y, float u, float w) {
  const __half2 h = __floats2half2_rn(u, w);
  x = h.x, y = h.y;
}
__device__ __forceinline__ void round_two(__nv_bfloat16& x, __nv_bfloat16& y, float u, float w) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(u, w);
  x = h.x, y = h.y;
}

template <>
struct Elem<float> {
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};

// A unit of channels of kAhead heads, a stride of dx (dy) elements apart, `left` of them there: loaded together, so that a thread
// does not wait for one head after the other, then turned and stored. turn: else the unit lies behind the rotated channels and
// is copied. The pointers walk: with an offset computed for every access the kernel was bound by its instructions.
template <typename T, int V, bool VEC, bool INTER, bool ROT>
struct HeadBatch {
  static constexpr int kAhead = RotShape<INTER, ROT>::kAhead, kPairs = INTER ? V / 2 : V;
  Raw<T, V> a[kAhead], b[kAhead];

  __device__ __forceinline__ void load(const T* x, long long dx, int left, int pairs, bool turn, bool zero) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (j < left && !zero) {
        a[j] = raw_load<T, V, VEC>(x);
        if (ROT && !INTER && turn) b[j] = raw_load<T, V, VEC>(x + pairs);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) a[j].v[i] = b[j].v[i] = Elem<T>::from_float(0.f);
      }
      x += dx;
    }
  }

  __device__ __forceinline__ void store(T* y, long long dy, int left, int pairs, bool turn, const float2* c) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (j >= left) break;
      if (ROT && turn) {
        float u[kPairs], w[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
          const float x = Elem<T>::to_float(INTER ? a[j].v[2 * i] : a[j].v[i]), z = Elem<T>::to_float(INTER ? a[j].v[2 * i + 1] : b[j].v[i]);
          u[i] = x * c[i].x - z * c[i].y;
          w[i] = x * c[i].y + z * c[i].x;
        }
        if constexpr (INTER) {
#pragma unroll
          for (int i = 0; i < kPairs; i++) round_two(a[j].v[2 * i], a[j].v[2 * i + 1], u[i], w[i]);
        } else if constexpr (kPairs % 2 == 0) {
#pragma unroll
          for (int i = 0; i < kPairs; i += 2) {
            round_two(a[j].v[i], a[j].v[i + 1], u[i], u[i + 1]);
            round_two(b[j].v[i], b[j].v[i + 1], w[i], w[i + 1]);
          }
        } else {
          a[j].v[0] = Elem<T>::from_float(u[0]), b[j].v[0] = Elem<T>::from_float(w[0]);
        }
        if (!INTER) raw_store<T, V, VEC>(y + pairs, b[j]);
      }
      raw_store<T, V, VEC>(y, a[j]);
      y += dy;
    }
  }
};

// How a block's threads share a slot: `per` threads for a token's head, groups of them side by side over tokens, then heads.
struct RotShare {
  int pairs, rot_units, units, per, group, unit, step;
  bool in;
  __device__ __forceinline__ int channel(int u, int v) const { return u < rot_units ? u * v : 2 * pairs + (u - rot_units) * v; }
};
template <int V, bool INTER, bool ROT>
__device__ __forceinline__ RotShare rot_share(const RotParams& p, const RotSlot& sl, int tid) {
  RotShare s;
  s.pairs = ROT && sl.rotate ? p.pairs : 0;
  s.rot_units = INTER ? 2 * s.pairs / V : s.pairs / V;
  s.units = s.rot_units + (p.D - 2 * s.pairs) / V;
  s.per = min(s.units, kRotThreads);
  const int groups = kRotThreads / s.per;
  s.group = tid / s.per, s.unit = tid - s.group * s.per;
  s.step = max(1, groups >> p.tok_shift);
  s.in = s.group < groups;
  return s;
}

// V elements make a unit of the copied channels and half a unit of (i, i + pairs); VEC: 16-byte accesses.
template <typename T, int V, bool VEC, bool INTER, bool PAGED, bool ROT>
__global__ void __launch_bounds__(kRotThreads, (RotShape<INTER, ROT>::kBlocks)) rotary_kernel(const __grid_constant__ RotParams p) {
  extern __shared__ float2 s_cs[];                  // [tokens_per_block][pairs]
  __shared__ int s_page[kRotTokens], s_row[kRotTokens], s_pos[kRotTokens];   // paged: -1 no page; row -1 of no sequence, or of one not served
  __shared__ int s_seq;
  const int tid = threadIdx.x, TOK = p.tokens_per_block;
  const long long tokens = (long long)p.B * p.N, t0 = (long long)blockIdx.x * TOK;
  pdl_wait();
  pdl_trigger();

  if (PAGED) {
    // the sequence of the block's first token: how many of them end at or before it
    int seq = 0;
    if (p.cu) {
      if (tid == 0) s_seq = 0;
      __syncthreads();
      int ended = 0;
      for (int i = tid; i < p.sequences; i += kRotThreads) ended += p.cu[i + 1] <= t0;
      if (ended) atomicAdd(&s_seq, ended);
      __syncthreads();
      seq = s_seq;
    }
    if (tid < TOK) {
      const long long t = t0 + tid;
      int page = -1, row = -1, pos = 0;
      if (t < tokens) {
        long long end = t + 1;
        if (p.cu) {
          while (seq < p.sequences && p.cu[seq + 1] <= t) seq++;
          if (seq < p.sequences && t < p.cu[seq]) seq = p.sequences;   // in front of the first
          if (seq < p.sequences) end = p.cu[seq + 1];
        } else {
          seq = (int)t;
        }
        if (seq < p.sequences && (!p.served || p.served[seq])) {
          const long long at = (long long)p.seq_lens[seq] - (end - t);
          row = 0;
          if (at >= 0 && at < (long long)p.width * p.page_size) {
            pos = (int)at;
            row = pos & (p.page_size - 1);
            page = p.table[seq * p.table_stride + pos / p.page_size];
            if (page < 0 || page >= p.num_pages) page = -1;
          }
          if (page < 0 && p.dev_status) atomicCAS(p.dev_status, 0, SPARGE_DEV_BAD_PAGE);
        }
      }
      s_page[tid] = page, s_row[tid] = row, s_pos[tid] = pos;
    }
    __syncthreads();
  }

  // The first heads travel while the angles are computed.
  HeadBatch<T, V, VEC, INTER, ROT> batch;
  bool ahead = false;
  if (!PAGED) {
    const RotSlot& sl = p.slot[0];
    const RotShare s = rot_share<V, INTER, ROT>(p, sl, tid);
    const int tok = s.group & (TOK - 1), h0 = s.group >> p.tok_shift;
    const long long t = t0 + tok;
    if (s.in && s.group < TOK * s.step && t < tokens && h0 < sl.heads) {
      const int b = batch_of(p, t);
      const bool turn = s.unit < s.rot_units;
      batch.load(reinterpret_cast<const T*>(sl.x) + b * sl.xb + (t - (long long)b * p.N) * sl.xn + h0 * sl.xh + s.channel(s.unit, V), s.step * sl.xh,
                 (sl.heads - h0 + s.step - 1) / s.step, s.pairs, turn, false);
      ahead = true;
    }
  }

  for (int i = tid; ROT && i < TOK * p.pairs; i += kRotThreads) {
    const int tok = i / p.pairs, pair = i - tok * p.pairs;
    const long long t = t0 + tok;
    if (t >= tokens) break;
    double pos;
    if (PAGED) {
      pos = s_pos[tok];
    } else {
      int axis = 0;
      for (int first = 0; axis + 1 < p.axes && pair >= first + p.sections[axis]; axis++) first += p.sections[axis];
      const int b = batch_of(p, t);
      const long long at = axis * p.pos_st[0] + b * p.pos_st[1] + (t - (long long)b * p.N) * p.pos_st[2];
      pos = p.pos64 ? (double)reinterpret_cast<const long long*>(p.positions)[at]
                    : (double)reinterpret_cast<const int32_t*>(p.positions)[at];
    }
    double turn = pos * p.freq[pair] * 0.15915494309189533577;   // in turns
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    s_cs[i] = make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
  }
  if (ROT) __syncthreads();

  for (int j = 0; j < p.slots; j++) {
    const RotSlot& sl = p.slot[j];
    const RotShare s = rot_share<V, INTER, ROT>(p, sl, tid);
    const int groups = kRotThreads / s.per;
    for (int g = s.group; g < TOK * s.step && s.in; g += groups) {
      const int tok = g & (TOK - 1), h0 = g >> p.tok_shift;
      const long long t = t0 + tok;
      if (t >= tokens) continue;
      const int b = PAGED ? 0 : batch_of(p, t);
      const T* x = reinterpret_cast<const T*>(sl.x) + b * sl.xb + (t - (long long)b * p.N) * sl.xn;
      T* y = reinterpret_cast<T*>(sl.y);
      bool zero = false;
      if (PAGED && sl.paged) {
        if (s_page[tok] < 0) continue;
        y += s_page[tok] * sl.yb + s_row[tok] * sl.yn;
      } else {
        zero = PAGED && s_row[tok] < 0;
        y += b * sl.yb + (t - (long long)b * p.N) * sl.yn;
      }
      const long long dx = s.step * sl.xh, dy = s.step * sl.yh;
      for (int u = s.unit; u < s.units; u += s.per) {
        const bool turn = u < s.rot_units;
        float2 c[batch.kPairs];
        if (ROT && turn) {
#pragma unroll
          for (int i = 0; i < batch.kPairs; i++) c[i] = s_cs[tok * p.pairs + u * batch.kPairs + i];
        }
        const T* px = x + h0 * sl.xh + s.channel(u, V);
        T* py = y + h0 * sl.yh + s.channel(u, V);
        for (int left = (sl.heads - h0 + s.step - 1) / s.step; left > 0; left -= batch.kAhead) {
          if (!ahead) batch.load(px, dx, left, s.pairs, turn, zero);
          ahead = false;
          batch.store(py, dy, left, s.pairs, turn, c);
          px += batch.kAhead * dx, py += batch.kAhead * dy;
        }
      }
    }
  }
}

template <typename T, bool INTER, bool PAGED, bool ROT>
static int rotary_launch(RotParams& p, bool vec, cudaStream_t st) {
  const long long tokens = (long long)p.B * p.N;
  // Few tokens: a block each, so that a step's heads spread over the GPU; many: eight, whose angles share one pass.
  p.tok_shift = tokens >= 8 * 148 ? 3 : tokens >= 2 * 148 ? 1 : 0;
  p.tokens_per_block = 1 << p.tok_shift;
  const size_t smem = sizeof(float2) * p.tokens_per_block * p.pairs;
  const long long blocks = (tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  if (blocks > 0x7fffffffLL) return SPARGE_ERR_TOO_LARGE;
  const auto kern = vec ? rotary_kernel<T, 8, true, INTER, PAGED, ROT> : rotary_kernel<T, INTER ? 2 : 1, false, INTER, PAGED, ROT>;
  return launch(kern, dim3((unsigned)blocks), dim3(kRotThreads), smem, st, true, p) == cudaSuccess ? SPARGE_OK : SPARGE_ERR_CUDA;
}

// 16-byte accesses of 8 elements: the base, every stride and the channels' borders have to be multiples of them.
static bool vec_ok(const RotParams& p, bool inter, int elem) {
  if (p.D % 8 || (p.pairs && (inter ? p.pairs % 4 : p.pairs % 8))) return false;
  for (int j = 0; j < p.slots; j++) {
    const RotSlot& s = p.slot[j];
    if (reinterpret_cast<uintptr_t>(s.x) % 16 || reinterpret_cast<uintptr_t>(s.y) % 16) return false;
    for (long long st : {s.xb, s.xh, s.xn, s.yb, s.yh, s.yn})
      if (st * elem % 16) return false;
  }
  return true;
}

template <bool PAGED>
static int rotary_dispatch(RotParams& p, bool inter, int dtype, cudaStream_t st) {
  const bool vec = vec_ok(p, inter, dtype == SPARGE_F32 ? 4 : 2);
#define SPARGE_ROT(T) \
  (PAGED && p.pairs == 0 ? rotary_launch<T, false, PAGED, !PAGED>(p, vec, st) \
                         : inter ? rotary_launch<T, true, PAGED, true>(p, vec, st) : rotary_launch<T, false, PAGED, true>(p, vec, st))
  if (dtype == SPARGE_BF16) return SPARGE_ROT(__nv_bfloat16);
  if (dtype == SPARGE_F16) return SPARGE_ROT(__half);
  if constexpr (!PAGED) return SPARGE_ROT(float);
  return SPARGE_ERR_INVALID_ARG;
#undef SPARGE_ROT
}

static RotSlot rot_slot(const void* x, void* y, const long long* xs, const long long* ys, int heads) {
  return RotSlot{x, y, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2], heads, true, false};
}

}  // namespace sparge

extern "C" int sparge_rotary(const sparge_rotary_args* a, sparge_stream_t stream) {
  using namespace sparge;
  if (!a) return SPARGE_ERR_NULL;
  if (a->B < 0 || a->N < 0 || a->q_heads < 0 || a->k_heads < 0 || a->D <= 0 || a->D % 2 || a->D > 1024 || a->pairs <= 0 || 2 * a->pairs > a->D ||
      a->dtype < 0 || a->dtype > SPARGE_F32 || a->axes < 1 || a->axes > 4)
    return SPARGE_ERR_INVALID_ARG;
  if (a->axes > 1) {
    int sum = 0;
    for (int i = 0; i < a->axes; i++) {
      if (a->sections[i] < 0) return SPARGE_ERR_INVALID_ARG;
      sum += a->sections[i];
    }
    if (sum != a->pairs) return SPARGE_ERR_INVALID_ARG;
  }
  if ((long long)a->B * a->N == 0 || a->q_heads + a->k_heads == 0) return SPARGE_OK;
  if ((a->q_heads && (!a->q || !a->q_out)) || (a->k_heads && (!a->k || !a->k_out)) || !a->positions || !a->frequencies) return SPARGE_ERR_NULL;
  RotParams p = {};
  if (a->q_heads) p.slot[p.slots++] = rot_slot(a->q, a->q_out, a->q_st, a->q_out_st, a->q_heads);
  if (a->k_heads) p.slot[p.slots++] = rot_slot(a->k, a->k_out, a->k_st, a->k_out_st, a->k_heads);
  p.B = a->B, p.N = a->N, p.D = a->D, p.pairs = a->pairs, p.axes = a->axes;
  for (int i = 0; i < 4; i++) p.sections[i] = a->sections[i];
  p.positions = a->positions, p.pos64 = a->positions_64 != 0, p.inverse = a->inverse != 0;
  for (int i = 0; i < 3; i++) p.pos_st[i] = a->positions_st[i];
  p.freq = a->frequencies, p.magnitude = a->magnitude;
  return rotary_dispatch<false>(p, a->interleaved != 0, a->dtype, (cudaStream_t)stream);
}

extern "C" int sparge_append_kv(const sparge_append_args* a, sparge_stream_t stream) {
  using namespace sparge;
  if (!a) return SPARGE_ERR_NULL;
  const sparge_cache& c = a->cache;
  if (c.tokens < 0 || c.sequences < 0 || c.kv_heads <= 0 || c.D <= 0 || c.D % 8 || c.D > 1024 || (c.dtype != SPARGE_F16 && c.dtype != SPARGE_BF16) ||
      c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)) || c.table_width < 0 || c.num_pages < 0 ||
      (!c.cu_seqlens && c.tokens != c.sequences) || (a->q && a->q_heads <= 0))
    return SPARGE_ERR_INVALID_ARG;
  if (a->frequencies && (a->pairs <= 0 || 2 * a->pairs > c.D)) return SPARGE_ERR_INVALID_ARG;
  if (a->q && !a->frequencies) return SPARGE_ERR_INVALID_ARG;
  if ((long long)c.table_width * c.page_size > 0x7fffffffLL) return SPARGE_ERR_TOO_LARGE;
  if (c.tokens == 0) return SPARGE_OK;
  if (!a->k || !a->v || (c.num_pages && (!c.k_pages || !c.v_pages)) || (a->q && !a->q_out)) return SPARGE_ERR_NULL;
  if (c.sequences && (!c.seq_lens || (c.table_width && !c.page_table))) return SPARGE_ERR_NULL;
  RotParams p = {};
  const auto paged = [&](const void* x, const long long* xs, void* pages, const long long* ps, bool rotate) {
    p.slot[p.slots++] = RotSlot{x, pages, 0, xs[1], xs[0], ps[0], ps[1], ps[2], c.kv_heads, rotate, true};
  };
  if (a->q) p.slot[p.slots++] = RotSlot{a->q, a->q_out, 0, a->q_st[1], a->q_st[0], 0, a->q_out_st[1], a->q_out_st[0], a->q_heads, true, false};
  paged(a->k, a->k_st, c.k_pages, c.k_st, a->frequencies != nullptr);
  paged(a->v, a->v_st, c.v_pages, c.v_st, false);
  p.B = 1, p.N = c.tokens, p.D = c.D, p.pairs = a->frequencies ? a->pairs : 0, p.axes = 1, p.freq = a->frequencies, p.magnitude = a->magnitude;
  p.table = c.page_table, p.seq_lens = c.seq_lens, p.cu = c.cu_seqlens, p.served = a->served, p.table_stride = c.table_stride;
  p.sequences = c.sequences, p.width = c.table_width, p.num_pages = c.num_pages, p.page_size = c.page_size, p.dev_status = a->dev_status;
  return rotary_dispatch<true>(p, a->interleaved != 0, c.dtype, (cudaStream_t)stream);
}
