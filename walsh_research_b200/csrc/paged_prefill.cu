// Attention of several new tokens per sequence (prompts, later parts of
// prompts) over a paged key/value cache, with a sliding window and sinks.
//
// Sequence b has the queries q_offsets[b] .. q_offsets[b+1]-1 (rows of q);
// they are its last tokens, already appended, so query t of T sits at
// position kv_len - T + t.  It sees key j when j <= position and, under a
// window, j > position - window or j < sinks.
//
// Rows of a tile are (token, head of the group) pairs, token-major, so shared
// key/value heads are read once for their whole group.
#include <math_constants.h>

#include "mma.cuh"
#include "paged.cuh"

namespace walsh {

template <typename T>
struct PrefillArgs {
  Pages<T> pg;
  const T* q;
  int64_t q_ts, q_hs;  // token and head strides, elements
  int64_t q_rows;      // rows of q and o
  const int* q_off;    // [B + 1]
  T* o;                // [rows, Hq, hd]
  int kv_heads;
  FastDiv group;
  float scale_log2;
};

// The span of q of sequence b; offsets outside the rows are reported and the sequence is empty.
template <typename T>
__device__ __forceinline__ int query_span(const PrefillArgs<T>& a, int b, int64_t* first) {
  const int64_t q0 = a.q_off[b], q1 = a.q_off[b + 1];
  *first = q0;
  if (q0 < 0 || q1 < q0 || q1 > a.q_rows) {
    if (a.pg.err) atomicExch(a.pg.err, (int)WALSH_ERR_INDEX);
    return 0;
  }
  return (int)(q1 - q0);
}

// CUDA-core form: 64 rows x 32 keys a step, 256 threads; a half warp owns four
// rows (scores, softmax and accumulator), so only K and V tiles need barriers.
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_prefill_vec_kernel(const PrefillArgs<T> a) {
  constexpr int QT = 64, KT = 32, LD = HD + 4, VEC = 16 / (int)sizeof(T), CH = HD / VEC;
  extern __shared__ __align__(16) float sm[];
  float* Qs = sm;             // [QT][LD]
  float* Ks = Qs + QT * LD;   // [KT][LD]
  float* Vs = Ks + KT * LD;   // [KT][LD]
  float* Ps = Vs + KT * LD;   // [QT][KT + 1]
  __shared__ int okk[KT];
  const int b = blockIdx.z, hk = blockIdx.y, tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  int64_t first;
  const int T_ = query_span(a, b, &first);
  const int G = (int)a.group.d;
  const int64_t nrows = (int64_t)T_ * G;
  const int len = seq_len(a.pg, b), pos0 = len - T_;
  const int* trow = a.pg.table + (int64_t)b * a.pg.table_stride;
  const int64_t hoff = (int64_t)hk * a.pg.head_stride;
  // the grid covers max_q tokens; tiles of a longer span follow in further turns
  for (int64_t r0 = (int64_t)blockIdx.x * QT; r0 < nrows; r0 += (int64_t)gridDim.x * QT) {
  const int nr = (int)min64(QT, nrows - r0);
  __syncthreads();
  for (int i = tid; i < QT * CH; i += 256) {
    const int r = i / CH, c = i - r * CH;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (r < nr) {
      const uint32_t t = fdiv((uint32_t)(r0 + r), a.group), g = (uint32_t)(r0 + r) - t * G;
      raw = *reinterpret_cast<const uint4*>(a.q + (first + t) * a.q_ts + (int64_t)(hk * G + g) * a.q_hs + c * VEC);
    }
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) Qs[r * LD + c * VEC + j] = to_f(e[j]) * a.scale_log2;
  }
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = min(ty * 4 + i, nr - 1);
    pos[i] = pos0 + (int)fdiv((uint32_t)(r0 + r), a.group);
  }
  // keys some row of this tile sees: sinks, then lo .. hi
  const int pos_first = pos0 + (int)fdiv((uint32_t)r0, a.group);
  const int pos_last = pos0 + (int)fdiv((uint32_t)(r0 + nr - 1), a.group);
  const int lo = a.pg.window > 0 ? max(0, pos_first + 1 - a.pg.window) : 0;
  const int nsink = min(a.pg.sinks, lo), n = nsink + max(0, pos_last + 1 - lo);
  float m[4], l[4], acc[4][HD / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -CUDART_INF_F;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) acc[i][d] = 0.f;
  }
  for (int k0 = 0; k0 < n; k0 += KT) {
    __syncthreads();
    for (int i = tid; i < KT * CH; i += 256) {
      const int r = i / CH, c = i - r * CH, x = k0 + r;
      const int key = x < nsink ? x : lo + (x - nsink);
      int64_t off = -1;
      if (x < n) off = key_offset(a.pg, trow, key);
      uint4 kr = make_uint4(0u, 0u, 0u, 0u), vr = kr;
      if (off >= 0) {
        kr = __ldg(reinterpret_cast<const uint4*>(a.pg.k + hoff + off + c * VEC));
        vr = __ldg(reinterpret_cast<const uint4*>(a.pg.v + hoff + off + c * VEC));
      }
      if (c == 0) okk[r] = off >= 0 ? key : -1;
      const T *ke = reinterpret_cast<const T*>(&kr), *ve = reinterpret_cast<const T*>(&vr);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        Ks[r * LD + c * VEC + j] = to_f(ke[j]);
        Vs[r * LD + c * VEC + j] = to_f(ve[j]);
      }
    }
    __syncthreads();
    float s[4][2] = {};
    for (int d = 0; d < HD; d += 4) {
      float4 q4[4], k4[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(&Qs[(ty * 4 + i) * LD + d]);
#pragma unroll
      for (int j = 0; j < 2; ++j) k4[j] = *reinterpret_cast<const float4*>(&Ks[(tx + 16 * j) * LD + d]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          s[i][j] = fmaf(q4[i].x, k4[j].x, fmaf(q4[i].y, k4[j].y, fmaf(q4[i].z, k4[j].z, fmaf(q4[i].w, k4[j].w, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool see[2];
      float mt = -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = okk[tx + 16 * j];
        see[j] = key >= 0 && key <= pos[i] &&
                 (a.pg.window == 0 || key > pos[i] - a.pg.window || key < a.pg.sinks);
        if (!see[j]) s[i][j] = -CUDART_INF_F;
        mt = fmaxf(mt, s[i][j]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float mn = fmaxf(m[i], mt), sub_m = mn == -CUDART_INF_F ? 0.f : mn;
      const float corr = ex2_f32(m[i] - sub_m);
      m[i] = mn;
      l[i] *= corr;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) acc[i][d] *= corr;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p = see[j] ? ex2_f32(s[i][j] - sub_m) : 0.f;
        l[i] += p;
        Ps[(ty * 4 + i) * (KT + 1) + tx + 16 * j] = p;
      }
    }
    __syncwarp();
    for (int j = 0; j < KT; ++j) {
      float v[HD / 16];
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) v[d] = Vs[j * LD + tx + 16 * d];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = Ps[(ty * 4 + i) * (KT + 1) + j];
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) acc[i][d] = fmaf(p, v[d], acc[i][d]);
      }
    }
    __syncwarp();
  }
  const int64_t Hq = (int64_t)a.kv_heads * G;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float L = l[i];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const int r = ty * 4 + i;
    if (r < nr) {
      const uint32_t t = fdiv((uint32_t)(r0 + r), a.group), g = (uint32_t)(r0 + r) - t * G;
      T* op = a.o + ((first + t) * Hq + (int64_t)hk * G + g) * HD;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) op[tx + 16 * d] = round_f<T>(L == 0.f ? 0.f : acc[i][d] / L);
    }
  }
  }
}

template <typename T, int HD>
static int launch_prefill(const PrefillArgs<T>& a, int B, int max_q, cudaStream_t s) {
  constexpr int QT = 64, KT = 32, LD = HD + 4;
  const int smem = ((QT + 2 * KT) * LD + QT * (KT + 1)) * 4;
  auto* kern = paged_prefill_vec_kernel<T, HD>;
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status();
  const int64_t tiles = ((int64_t)max_q * a.group.d + QT - 1) / QT;
  kern<<<dim3((unsigned)tiles, a.kv_heads, B), 256, smem, s>>>(a);
  return launch_status();
}

}  // namespace walsh

using namespace walsh;

extern "C" walsh_status walsh_paged_prefill_fwd(const walsh_paged_kv* kv, const void* q, int64_t q_ts, int64_t q_hs,
                                                int64_t q_rows, const int32_t* q_offsets, int B, int q_heads,
                                                int max_q, void* o, void* stream) {
  if (int e = injected("paged_prefill_fwd")) return e;
  if (int e = check_pages(kv, true)) return e;
  WALSH_CHECK_ARG(q && q_offsets && o);
  WALSH_CHECK_SHAPE(B >= 0 && B <= 65535 && q_heads > 0 && q_heads <= 65535 && q_heads % kv->kv_heads == 0);
  WALSH_CHECK_SHAPE(q_rows >= 0 && q_rows < (1ll << 31) && max_q >= 0 && (int64_t)max_q * q_heads < (1ll << 31) &&
                    q_rows * (q_heads / kv->kv_heads) < (1ll << 31));
  const int64_t vec = kv->dtype == WALSH_F32 ? 4 : 8;
  WALSH_CHECK_SHAPE(q_ts >= 0 && q_hs >= 0);
  if (((((uintptr_t)q) | ((uintptr_t)o)) & 15u) != 0 || q_ts % vec || q_hs % vec) return WALSH_ERR_ALIGN;
  if (B == 0 || max_q == 0 || q_rows == 0) return WALSH_OK;
  return WALSH_DISPATCH_DTYPE(kv->dtype, ET, [&]() -> int {
    PrefillArgs<ET> a;
    a.pg = make_pages<ET>(kv);
    a.q = (const ET*)q, a.q_ts = q_ts, a.q_hs = q_hs, a.q_rows = q_rows, a.q_off = q_offsets, a.o = (ET*)o;
    a.kv_heads = kv->kv_heads;
    a.group = make_fastdiv((uint32_t)(q_heads / kv->kv_heads));
    a.scale_log2 = kv->scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    switch (kv->head_dim) {
      case 16: return launch_prefill<ET, 16>(a, B, max_q, s);
      case 32: return launch_prefill<ET, 32>(a, B, max_q, s);
      case 64: return launch_prefill<ET, 64>(a, B, max_q, s);
      default: return launch_prefill<ET, 128>(a, B, max_q, s);
    }
  }());
}
