// Attention of one new token per sequence over a paged key/value cache
// (batched decode), split over the cache's length and joined.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2 e
//
// over the keys j the token sees: the last `window` of its sequence's keys
// and the first `sinks` (all of them without a window).  Each cache byte is
// used for 2 multiply-adds per query head of its group, so HBM bounds it.
//
// The visible keys of a (sequence, key/value head) are numbered 0..n-1 and
// cut into nsplit ranges of `chunk`; a CTA of W warps takes one range, each
// warp a slice of it with its own running maximum, sum and accumulator
// (float32), joined through shared memory.  With more than one non-empty
// range the CTA leaves (m, l, o) in the workspace and paged_join_kernel
// combines them in order of the ranges, so results do not depend on timing.
#include <math_constants.h>

#include "mma.cuh"
#include "paged.cuh"

namespace walsh {

template <typename T>
struct DecodeArgs {
  Pages<T> pg;
  const T* q;
  int64_t q_bs, q_hs;  // batch and head strides, elements
  T* o;                // [B, Hq, hd]
  float* part_o;       // [B, Hq, nsplit, hd]
  float* part_ml;      // [B, Hq, nsplit, 2]
  int B, kv_heads, group;
  int gtiles;          // head tiles of a group
  int nsplit, chunk;
  float scale_log2;
};

// Range c of n visible keys: the last range takes whatever is left.
__device__ __forceinline__ void split_range(int n, int chunk, int nsplit, int c, int* beg, int* end) {
  *beg = min((int64_t)n, (int64_t)c * chunk);
  *end = c == nsplit - 1 ? n : (int)min((int64_t)n, (int64_t)(c + 1) * chunk);
}

// ---------------------------------------------------------------------------
// CUDA-core form, any type.  LPK lanes share one key, 16 bytes of it each; a
// warp step covers 32 / LPK keys and KPT steps are in flight.
// ---------------------------------------------------------------------------
template <typename T, int HD, int GH, int W>
__global__ void __launch_bounds__(W * 32) paged_decode_vec_kernel(const DecodeArgs<T> a) {
  constexpr int VEC = 16 / (int)sizeof(T), LPK = HD / VEC, KS = 32 / LPK, KPT = 4;
  __shared__ float red[W][GH][LPK][VEC + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LPK, slot = lane / LPK;
  int unit = blockIdx.x;
  const int c = unit % a.nsplit;
  unit /= a.nsplit;
  const int gt = unit % a.gtiles;
  unit /= a.gtiles;
  const int hk = unit % a.kv_heads, b = unit / a.kv_heads;
  const int len = seq_len(a.pg, b);
  const Visible vis = visible_keys(len - 1, a.pg.window, a.pg.sinks);
  int beg, end;
  split_range(vis.n, a.chunk, a.nsplit, c, &beg, &end);
  if (beg >= end && c > 0) return;
  const int gh0 = gt * GH, ng = min(GH, a.group - gh0);
  const int h0 = hk * a.group + gh0;
  const int per = ((end - beg + W - 1) / W + KS - 1) / KS * KS;
  const int wbeg = min(end, beg + warp * per), wend = min(end, wbeg + per);
  float qv[GH][VEC], acc[GH][VEC], m[GH], l[GH];
#pragma unroll
  for (int g = 0; g < GH; ++g) {
    m[g] = -CUDART_INF_F;
    l[g] = 0.f;
    const T* qp = a.q + (int64_t)b * a.q_bs + (int64_t)(h0 + min(g, ng - 1)) * a.q_hs + sub * VEC;
    const uint4 raw = *reinterpret_cast<const uint4*>(qp);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      qv[g][j] = to_f(e[j]) * a.scale_log2;
      acc[g][j] = 0.f;
    }
  }
  const int* trow = a.pg.table + (int64_t)b * a.pg.table_stride;
  const T* kb = a.pg.k + (int64_t)hk * a.pg.head_stride + sub * VEC;
  const T* vb = a.pg.v + (int64_t)hk * a.pg.head_stride + sub * VEC;
  for (int i0 = wbeg; i0 < wend; i0 += KS * KPT) {
    uint4 kr[KPT], vr[KPT];
    bool ok[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int i = i0 + u * KS + slot;
      int64_t off = -1;
      if (i < wend) off = key_offset(a.pg, trow, vis.key(i));
      ok[u] = off >= 0;
      kr[u] = vr[u] = make_uint4(0u, 0u, 0u, 0u);
      if (ok[u]) {
        kr[u] = __ldg(reinterpret_cast<const uint4*>(kb + off));
        vr[u] = __ldg(reinterpret_cast<const uint4*>(vb + off));
      }
    }
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      float s[KPT], cm = -CUDART_INF_F;
#pragma unroll
      for (int u = 0; u < KPT; ++u) {
        const T* e = reinterpret_cast<const T*>(&kr[u]);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) dot = fmaf(qv[g][j], to_f(e[j]), dot);
#pragma unroll
        for (int o = 1; o < LPK; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        s[u] = ok[u] ? dot : -CUDART_INF_F;
        cm = fmaxf(cm, s[u]);
      }
      const float mn = fmaxf(m[g], cm);
      const float sub_m = mn == -CUDART_INF_F ? 0.f : mn;
      const float corr = ex2_f32(m[g] - sub_m);
      l[g] *= corr;
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[g][j] *= corr;
#pragma unroll
      for (int u = 0; u < KPT; ++u) {
        const float p = ok[u] ? ex2_f32(s[u] - sub_m) : 0.f;
        const T* e = reinterpret_cast<const T*>(&vr[u]);
        l[g] += p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[g][j] = fmaf(p, to_f(e[j]), acc[g][j]);
      }
      m[g] = mn;
    }
  }
  // the 32 / LPK lanes of one channel piece hold disjoint keys
#pragma unroll
  for (int g = 0; g < GH; ++g) {
    float M = m[g];
#pragma unroll
    for (int o = LPK; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = m[g] == -CUDART_INF_F ? 0.f : ex2_f32(m[g] - M);
    l[g] *= f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[g][j] *= f;
#pragma unroll
    for (int o = LPK; o < 32; o <<= 1) {
      l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[g][j] += __shfl_xor_sync(0xffffffffu, acc[g][j], o);
    }
    if (lane < LPK) {
      red[warp][g][sub][0] = M;
      red[warp][g][sub][1] = l[g];
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[warp][g][sub][2 + j] = acc[g][j];
    }
  }
  __syncthreads();
  const int64_t Hq = (int64_t)a.kv_heads * a.group;
  const bool whole = vis.n <= a.chunk || a.nsplit == 1;  // this range is all there is
  for (int i = threadIdx.x; i < ng * HD; i += W * 32) {
    const int g = i / HD, d = i - g * HD, p = d / VEC, j = d - p * VEC;
    float M = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, red[w][g][p][0]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = red[w][g][p][0];
      const float f = mw == -CUDART_INF_F ? 0.f : ex2_f32(mw - M);
      L = fmaf(red[w][g][p][1], f, L);
      O = fmaf(red[w][g][p][2 + j], f, O);
    }
    const int64_t row = (int64_t)b * Hq + h0 + g;
    if (whole) {
      a.o[row * HD + d] = round_f<T>(L == 0.f ? 0.f : O / L);  // no visible key: zeros
    } else {
      a.part_o[(row * a.nsplit + c) * HD + d] = O;
      if (d == 0) {
        a.part_ml[(row * a.nsplit + c) * 2] = M;
        a.part_ml[(row * a.nsplit + c) * 2 + 1] = L;
      }
    }
  }
}

// Joins the ranges of each (sequence, head): one warp per row.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const DecodeArgs<T> a) {
  const int lane = threadIdx.x & 31;
  const int64_t Hq = (int64_t)a.kv_heads * a.group;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.B * Hq) return;
  const Visible vis = visible_keys(seq_len(a.pg, (int)(row / Hq)) - 1, a.pg.window, a.pg.sinks);
  if (vis.n <= a.chunk) return;  // written whole
  const int nc = (int)min((int64_t)a.nsplit, ((int64_t)vis.n + a.chunk - 1) / a.chunk);
  const float* ml = a.part_ml + row * a.nsplit * 2;
  const float* po = a.part_o + row * a.nsplit * HD;
  float M = -CUDART_INF_F;
  for (int i = lane; i < nc; i += 32) M = fmaxf(M, ml[2 * i]);
  M = warp_max(M);
  const float sub_m = M == -CUDART_INF_F ? 0.f : M;
  constexpr int DP = HD < 32 ? HD : 32;  // channels per step
  constexpr int SL = 32 / DP;            // ranges per step
  const int d0 = lane % DP, s0 = lane / DP;
  float L = 0.f, O[HD / DP] = {};
  for (int i = s0; i < nc; i += SL) {
    const float f = ex2_f32(ml[2 * i] - sub_m);
    L = fmaf(ml[2 * i + 1], f, L);
#pragma unroll
    for (int k = 0; k < HD / DP; ++k) O[k] = fmaf(po[(int64_t)i * HD + k * DP + d0], f, O[k]);
  }
#pragma unroll
  for (int o = DP; o < 32; o <<= 1) {
    L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int k = 0; k < HD / DP; ++k) O[k] += __shfl_xor_sync(0xffffffffu, O[k], o);
  }
  if (lane < DP)
#pragma unroll
    for (int k = 0; k < HD / DP; ++k) a.o[row * HD + k * DP + d0] = round_f<T>(L == 0.f ? 0.f : O[k] / L);
}

template <typename T, int HD>
static int launch_decode(DecodeArgs<T> a, cudaStream_t s) {
  constexpr int W = 4;
  const int64_t ctas = (int64_t)a.B * a.kv_heads * a.gtiles * a.nsplit;
  if (a.group == 1)
    paged_decode_vec_kernel<T, HD, 1, W><<<(unsigned)ctas, W * 32, 0, s>>>(a);
  else
    paged_decode_vec_kernel<T, HD, 4, W><<<(unsigned)ctas, W * 32, 0, s>>>(a);
  if (const int r = launch_status()) return r;
  if (a.nsplit > 1) {
    const int64_t rows = (int64_t)a.B * a.kv_heads * a.group;
    paged_join_kernel<T, HD><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(a);
    return launch_status();
  }
  return WALSH_OK;
}

// How a call is cut: enough ranges to fill the GPU when there are few (sequence,
// head) units, none shorter than 256 keys.
struct DecodePlan {
  int gtiles, nsplit, chunk;
};
static DecodePlan decode_plan(const walsh_paged_kv* kv, int B, int q_heads, int max_len) {
  const int group = q_heads / kv->kv_heads;
  DecodePlan p;
  p.gtiles = group == 1 ? 1 : (group + 3) / 4;
  const int64_t units = (int64_t)B * kv->kv_heads * p.gtiles;
  int64_t n = max_len;
  if (kv->window > 0) n = min64(n, (int64_t)kv->window + kv->sinks);
  const int64_t want = (148 * 8 + units - 1) / units;
  p.nsplit = (int)(n < 256 ? 1 : min64(want, n / 256));
  if (p.nsplit < 1) p.nsplit = 1;
  p.chunk = (int)((n + p.nsplit - 1) / p.nsplit);
  if (p.chunk < 1) p.chunk = 1;
  return p;
}

}  // namespace walsh

using namespace walsh;

static int decode_check(const walsh_paged_kv* kv, int B, int q_heads, int max_len) {
  if (int e = check_pages(kv, true)) return e;
  WALSH_CHECK_SHAPE(B >= 0 && q_heads > 0 && q_heads <= 65535 && q_heads % kv->kv_heads == 0 && max_len >= 0);
  WALSH_CHECK_SHAPE((int64_t)B * q_heads < (1ll << 26));
  return WALSH_OK;
}

extern "C" int64_t walsh_paged_attn_scratch_bytes(const walsh_paged_kv* kv, int B, int q_heads, int max_len) {
  if (decode_check(kv, B, q_heads, max_len) != WALSH_OK) return -1;
  const DecodePlan p = decode_plan(kv, B, q_heads, max_len);
  return p.nsplit > 1 ? (int64_t)B * q_heads * p.nsplit * (kv->head_dim + 2) * 4 : 0;
}

extern "C" walsh_status walsh_paged_attn_fwd(const walsh_paged_kv* kv, const void* q, int64_t q_bs, int64_t q_hs,
                                             int B, int q_heads, int max_len, void* scratch, void* o, void* stream) {
  if (int e = injected("paged_attn_fwd")) return e;
  if (int e = decode_check(kv, B, q_heads, max_len)) return e;
  WALSH_CHECK_ARG(q && o);
  const int64_t vec = kv->dtype == WALSH_F32 ? 4 : 8;
  WALSH_CHECK_SHAPE(q_bs >= 0 && q_hs >= 0);
  if (((((uintptr_t)q) | ((uintptr_t)o) | ((uintptr_t)scratch)) & 15u) != 0 || q_bs % vec || q_hs % vec)
    return WALSH_ERR_ALIGN;
  if (B == 0) return WALSH_OK;
  const DecodePlan p = decode_plan(kv, B, q_heads, max_len);
  WALSH_CHECK_ARG(p.nsplit == 1 || scratch);
  return WALSH_DISPATCH_DTYPE(kv->dtype, ET, [&]() -> int {
    DecodeArgs<ET> a;
    a.pg = make_pages<ET>(kv);
    a.q = (const ET*)q, a.q_bs = q_bs, a.q_hs = q_hs, a.o = (ET*)o;
    a.part_o = (float*)scratch;
    a.part_ml = a.part_o + (int64_t)B * q_heads * p.nsplit * kv->head_dim;
    a.B = B, a.kv_heads = kv->kv_heads, a.group = q_heads / kv->kv_heads;
    a.gtiles = p.gtiles, a.nsplit = p.nsplit, a.chunk = p.chunk;
    a.scale_log2 = kv->scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    switch (kv->head_dim) {
      case 16: return launch_decode<ET, 16>(a, s);
      case 32: return launch_decode<ET, 32>(a, s);
      case 64: return launch_decode<ET, 64>(a, s);
      default: return launch_decode<ET, 128>(a, s);
    }
  }());
}
