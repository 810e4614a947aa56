// Token sampling from logits: temperature, top-k, top-p (nucleus), min-p and
// one draw per row from a given uniform number.
//
//   w_i = exp((l_i - max l) / T)
//   top-k:  the k largest logits (ties: lowest index first)
//   top-p:  of those, in descending order, token r stays while the mass
//           before it is below p times the mass of the top-k set
//   min-p:  w_i >= min_p
//   draw:   the first token in index order whose running mass exceeds u Z
//
// A token at a border is kept or dropped whole, so what decides is held to about
// 2^-45 of the largest weight: exp in double, rounded to a 64-bit integer
// multiple of 2^-44 (sums of integers do not depend on the order they are taken
// in, so neither do the draws).  Float32 sums are used only together with a bound
// of their error, and replaced by exact ones where that bound could change the
// answer.  The vocabulary is limited to 2^18 tokens, which keeps every sum below
// 2^63.
//
// Bytes are the floor (256 rows of 50257 float32 logits: 7.9 us), instructions
// the bound: about 140 thousand warp instructions per row with top-p (one pass
// for the largest logit, one for the total and a histogram, one for the masses
// above the border) run at 60 % of the issue slots, 72.5 us; 1 row with top-k 50
// takes 12.3 us, the barriers and dependent steps of a row.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "mma.cuh"
#include "paged.cuh"
#include "sample_plan.h"

namespace walsh {

constexpr double kWeightOne = 17592186044416.0;  // 2^44

template <typename T>
struct SampleArgs {
  const T* logits;
  int64_t ld;
  int rows, vocab;
  const float* u;
  // one value for all rows, or one per row where the pointer is given
  double temperature, top_p, min_p;
  int top_k;
  const float *temperature_r, *top_p_r, *min_p_r;
  const int* top_k_r;
  int64_t* ids;
  float* logp;
};

// Unsigned order of floats; callers add +0 first, which makes -0 count as +0.
__device__ __forceinline__ uint32_t float_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

using u64 = unsigned long long;
namespace cg = cooperative_groups;

// 2^-x for 0 <= x < 64 in double: 2^-x = 2^-n 2^-1/2 2^g with n = floor x and
// g = n + 1/2 - x in (-1/2, 1/2], the last factor by the Taylor series of
// exp(g ln 2); its first dropped term is (ln 2 / 2)^12 / 12! = 6e-15.
__device__ __forceinline__ double exp2_neg(double x) {
  const int n = (int)x;
  const double g = ((double)n + 0.5 - x) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, g, 1.0 / 3628800.0);
  p = fma(p, g, 1.0 / 362880.0);
  p = fma(p, g, 1.0 / 40320.0);
  p = fma(p, g, 1.0 / 5040.0);
  p = fma(p, g, 1.0 / 720.0);
  p = fma(p, g, 1.0 / 120.0);
  p = fma(p, g, 1.0 / 24.0);
  p = fma(p, g, 1.0 / 6.0);
  p = fma(p, g, 0.5);
  p = fma(p, g, 1.0);
  p = fma(p, g, 1.0);
  return p * (0.70710678118654752440 * __hiloint2double((1023 - n) << 20, 0));
}

// Weight of logit l: exp((l - m) / T) with c = log2(e) / T; l <= m, m finite.
__device__ __forceinline__ double weight(float l, float m, double c) {
  if (l == m) return 1.0;
  if (l == -CUDART_INF_F) return 0.0;
  const double x = ((double)m - (double)l) * c;
  return x < 60.0 ? exp2_neg(x) : 0.0;
}
__device__ __forceinline__ u64 fixed(double w) { return __double2ull_rn(w * kWeightOne); }

constexpr int kBins = 1024;      // bins of the mass histogram
constexpr int kCands = 256;      // tokens resolved one by one at a top-p border
constexpr int kList = 1024;      // tokens of a top-k list
constexpr int kListTopK = 512;   // largest top_k that goes by the list
constexpr int kPairs = 256;      // lists up to this long are ranked by comparing all pairs, longer ones sorted

struct SampleShared {
  union {
    struct {
      uint32_t maxima[2 * kSampleThreads];  // of the halves of a thread's chunks
      uint32_t warp_max[kSampleWarps], oct_max[4 * kSampleWarps];
      u64 list[kList];
    } k;
    struct {
      float queue[kSampleWarps][64];
      uint16_t queue_tok[kSampleWarps][64];  // from the warp's first element
      u64 cand[kCands];  // this CTA's tokens at the border
      union {
        uint32_t hist[kBins];
        struct {
          u64 all[kCands], wt[kCands];  // the whole row's
        };
        u64 mass[256];
      };
    } p;
  };
  u64 w_keep[kSampleWarps], w_all[kSampleWarps], scratch[kSampleWarps], step[kSampleSteps], add[8];
  double w_sum[kSampleWarps];
  // what other CTAs of the cluster read; each sum of a phase has a place of its own,
  // since a CTA may be a phase ahead of one that still reads
  u64 cta_keep, cta_all, cta_ties;
  double cta_bound, cta_z, cta_tail;
  uint32_t cta_max, n, key_lo, key_hi;  // key_lo, key_hi: of the tokens at the border
  // what the CTA that finds it writes into every CTA
  int tie_index, uncertain;
  u64 thr;
};

// bits of two or one -inf values
template <typename T> __device__ __forceinline__ uint32_t neg_inf_word();
template <> __device__ __forceinline__ uint32_t neg_inf_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ uint32_t neg_inf_word<__nv_bfloat16>() { return 0xff80ff80u; }

// One cluster of CS CTAs per row, each with a contiguous part of the row, held in
// shared memory (STAGE) or read again from L2 by each pass; each warp owns a
// contiguous part of that, so index order is (CTA, warp, position).
template <typename T, int CS, bool STAGE>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs<T> a) {
  constexpr int NT = kSampleThreads, NW = kSampleWarps, VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SampleShared sh;
  T* seg = reinterpret_cast<T*>(dyn);
  bool inf_row = false;  // the largest logit is +inf
  bool nans = true;      // the part may hold NaN (in memory)
  const cg::cluster_group cl = cg::this_cluster();
  const int rank = CS == 1 ? 0 : (int)cl.block_rank();
  const int row = blockIdx.x / CS, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  auto all_sync = [&]() {
    if constexpr (CS == 1) __syncthreads();
    else cl.sync();
  };
  auto peer = [&](int r) -> SampleShared* {
    if constexpr (CS == 1) return &sh;
    else return cl.map_shared_rank(&sh, r);
  };
  const double temp = a.temperature_r ? (double)a.temperature_r[row] : a.temperature;
  const double top_p = a.top_p_r ? (double)a.top_p_r[row] : a.top_p;
  const double min_p = fmin(a.min_p_r ? (double)a.min_p_r[row] : a.min_p, 1.0);
  int top_k = a.top_k_r ? a.top_k_r[row] : a.top_k;
  if (top_k <= 0 || top_k > V) top_k = V;
  const bool greedy = !(temp > 0.0) || top_k == 1;
  const double c = temp > 0.0 ? 1.4426950408889634074 / temp : 1.0;
  const float cf = (float)c;
  // float32 weights only where neither c nor a difference of logits that still weighs (60 / c) may leave float32
  const bool approx = c >= 1e-36 && c <= 3e38;
  const bool by_list = top_k < V && top_k <= kListTopK, by_mass = top_k == V && top_p < 1.0 && approx;

  // ---- the row's part of this CTA; chunks of 16 bytes, `mis` elements before the row's first chunk boundary
  const T* lg = a.logits + (int64_t)row * a.ld;
  const int mis = (int)(((uintptr_t)lg & 15) / sizeof(T));
  const int chunks = sample_chunks(V, mis, VEC), per_cta = sample_cta_chunks(chunks, CS);
  const int c0 = rank * per_cta, nch = max(0, min(per_cta, chunks - c0));
  const int per_warp = sample_warp_chunks(nch);
  const int wbeg = min(nch, warp * per_warp), wend = min(nch, wbeg + per_warp);
  const int base = c0 * VEC - mis;  // token of the part's first element (negative: before the row)
  float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
  bool any_nan = false;
  // 16 bytes of the row from its memory, -inf outside the row
  const int in0 = base < 0 ? 1 : 0, in1 = base + nch * VEC > V ? nch - 1 : nch;  // chunks wholly inside
  auto fetch = [&](int ch) -> uint4 {
    const int t0 = base + ch * VEC;
    uint4 raw;
    if (ch >= in0 && ch < in1) {
      raw = STAGE ? __ldcs(reinterpret_cast<const uint4*>(lg + t0)) : __ldg(reinterpret_cast<const uint4*>(lg + t0));
    } else {
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = t0 + j >= 0 && t0 + j < V ? lg[t0 + j] : round_f<T>(-CUDART_INF_F);
    }
    return raw;
  };
  auto clean = [&](uint4 raw) -> uint4 {  // NaN count as -inf
    T* e = reinterpret_cast<T*>(&raw);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = fmaxf(e[j], -CUDART_INF_F);
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      T2* p = reinterpret_cast<T2*>(&raw);
      const uint32_t w = neg_inf_word<T>();
      T2 low;
      memcpy(&low, &w, 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = __hmax2(p[j], low);
    }
    return raw;
  };
  {
    constexpr int U = 4;
    for (int ch0 = wbeg + lane; ch0 < wend; ch0 += 32 * U) {
      uint4 raw[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (ch0 + 32 * i < wend) raw[i] = fetch(ch0 + 32 * i);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int ch = ch0 + 32 * i;
        if (ch >= wend) continue;
        if constexpr (STAGE) raw[i] = clean(raw[i]);
        const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = to_f(e[j]);
          if constexpr (!STAGE) any_nan |= v != v;
          if (j < VEC / 2) mx0 = fmaxf(mx0, v);
          else mx1 = fmaxf(mx1, v);
        }
        if constexpr (STAGE) *reinterpret_cast<uint4*>(seg + (int64_t)ch * VEC) = raw[i];
      }
    }
  }
  // 16 bytes of the part (past a warp's chunks and around the row -inf)
  auto chunk = [&](int ch, int end) -> uint4 {
    const uint32_t w = neg_inf_word<T>();
    uint4 raw = make_uint4(w, w, w, w);
    if (ch < end) {
      if constexpr (STAGE) raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
      else raw = nans ? clean(fetch(ch)) : fetch(ch);
    }
    if (inf_row) {  // the +inf logits share the weight, nothing else has any
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = to_f(e[j]) == CUDART_INF_F ? round_f<T>(0.f) : round_f<T>(-CUDART_INF_F);
    }
    return raw;
  };
  // f(value, token, is one) for the elements of the warp's chunks; every lane makes the same number of calls
  auto each = [&](auto f) {
    uint4 next = chunk(wbeg + lane, wend);  // a step ahead
    for (int ch0 = wbeg; ch0 < wend; ch0 += 32) {
      const int ch = ch0 + lane;
      const uint4 raw = next;
      next = chunk(ch + 32, wend);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int t = base + ch * VEC + j;
        f(to_f(e[j]), t, ch < wend && (unsigned)t < (unsigned)V);
      }
    }
  };
  auto composite = [](float v, int t) { return ((u64)float_key(v + 0.f) << 32) | (0xffffffffu - (unsigned)t); };
  auto warp_sum64 = [&](u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto warp_sumd = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  // sums over the block of one value per thread
  auto block_sum = [&](u64 v) {
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) sh.scratch[warp] = v;
    __syncthreads();
    v = sh.scratch[lane % NW];
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto block_sum32 = [&](unsigned v) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sh.scratch[warp] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, lane < NW ? (unsigned)sh.scratch[lane] : 0u);
  };
  // inclusive prefix sum over the block's threads
  auto block_scan = [&](u64 v, u64* total) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 31) sh.scratch[warp] = v;
    __syncthreads();
    u64 s = 0, before = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w == warp) before = s;
      s += sh.scratch[w];
    }
    *total = s;
    return v + before;
  };

  // ---- maximum of the row, and for top-p a lower bound of Z
  const uint32_t mk0 = float_key(mx0 + 0.f), mk1 = float_key(mx1 + 0.f);
  {
    const uint32_t wm = __reduce_max_sync(0xffffffffu, max(mk0, mk1));
    if (by_list) {
      sh.k.maxima[tid] = mk0;
      sh.k.maxima[NT + tid] = mk1;
      const uint32_t om = __reduce_max_sync(0xffu << (lane & 24), max(mk0, mk1));
      if ((lane & 7) == 0) sh.k.oct_max[tid >> 3] = om;
      if (lane == 0) sh.k.warp_max[warp] = wm;
    }
    if (lane == 0) sh.scratch[warp] = wm;
    if (tid == 0) sh.n = 0, sh.uncertain = 0, sh.key_lo = ~0u, sh.key_hi = 0u;
    if (tid < 8) sh.add[tid] = 0;
    if constexpr (STAGE) __syncthreads();
    else nans = __syncthreads_or(any_nan);
    const uint32_t cm = __reduce_max_sync(0xffffffffu, (uint32_t)sh.scratch[lane % NW]);
    if (tid == 0) sh.cta_max = cm;
    if (by_mass) {  // the sum of the threads' largest weights, relative to this part's largest
      const float f = key_float(cm);
      float z = f > -CUDART_INF_F && f < CUDART_INF_F ? ex2_f32((mx0 - f) * cf) + ex2_f32((mx1 - f) * cf) : 0.f;
      z = warp_sum(z);
      if (lane == 0) sh.w_sum[warp] = z;
      __syncthreads();
      if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < NW; ++w) s += sh.w_sum[w];
        sh.cta_bound = s;
      }
    }
  }
  all_sync();
  uint32_t kmax = 0;
#pragma unroll
  for (int r = 0; r < CS; ++r) kmax = max(kmax, peer(r)->cta_max);
  float m = key_float(kmax);
  if (m == -CUDART_INF_F) {  // no token to draw
    if (rank == 0 && tid == 0) {
      a.ids[row] = -1;
      if (a.logp) a.logp[row] = CUDART_NAN_F;
    }
    all_sync();
    return;
  }
  bool general = top_k < V ? !by_list : top_p < 1.0 && !by_mass;
  float z_low = 0.f, z_high = (float)V;
  if (by_mass) {
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      const float f = key_float(peer(r)->cta_max);
      if (f > -CUDART_INF_F) z_low += (float)peer(r)->cta_bound * ex2_f32((f - m) * cf);
    }
    // Z is at most that sum times the elements behind one of the maxima (of the
    // longest part: every CTA needs the same bound)
    const int steps = sample_steps(sample_warp_chunks(per_cta));
    z_high = fminf(z_high, fmaxf(z_low, 1.f) * 1.001f * (float)(steps * (VEC / 2)));
    z_low = fmaxf(z_low * 0.999f, 1.f);
  }
  if (m == CUDART_INF_F && !greedy) {
    inf_row = true;
    m = 0.f;
    kmax = float_key(0.f);
    z_low = 1.f;
    z_high = (float)V;
    general |= top_k < V;  // (the list's maxima are of the logits as they were)
  }
  const double u = (double)a.u[row];
  auto finish = [&](int id, double w, double z) {
    a.ids[row] = id;
    if (a.logp) a.logp[row] = greedy ? 0.f : (float)log(w / z);
  };

  if (greedy) {  // the first token of the largest logit
    int best = 0x7fffffff;
    each([&](float v, int t, bool in) {
      if (in && float_key(v + 0.f) == kmax) best = min(best, t);
    });
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0) sh.scratch[warp] = (u64)best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < NW; ++w) best = min(best, (int)sh.scratch[w]);
      sh.tie_index = best;
    }
    all_sync();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < CS; ++r) best = min(best, peer(r)->tie_index);
      finish(best, 1.0, 1.0);
    }
    all_sync();
    return;
  }

  auto drawn_mass = [&](u64 z) {  // the running mass that the drawn token is the first to exceed
    const double uz = u * (double)z;
    const u64 t = uz > 0.0 ? (uz < 9.2e18 ? (u64)uz : z - 1) : 0;
    return t < z ? t : z - 1;
  };

  // -----------------------------------------------------------------------
  // top-k by a list: a lower bound t of the k-th largest logit is the k-th
  // largest maximum over disjoint groups of the row (k groups reach it, so k
  // logits do; with at least 2 k groups few more).  The logits from t up are
  // gathered in one CTA, which ranks them and does everything else.
  // -----------------------------------------------------------------------
  if (by_list && !general) {
    uint32_t t = 0;
    if (V > kList) {
      const int groups = 2 * top_k <= NW * CS ? NW : 2 * top_k <= 4 * NW * CS ? 4 * NW : 0;  // of a CTA
      if (groups) {
        uint32_t* vals = reinterpret_cast<uint32_t*>(sh.k.list);
        const int all = groups * CS;
        if (tid < all) {
          const SampleShared* q = peer(tid / groups);
          vals[tid] = groups == NW ? q->k.warp_max[tid % NW] : q->k.oct_max[tid % (4 * NW)];
        }
        __syncthreads();
        const int gs = NT / all, i = tid / gs;  // threads per value (all divides NT)
        const uint32_t mine = vals[i];
        unsigned n = 0;  // values above, and at least, mine
        for (int j = tid % gs; j < all; j += gs) n += (vals[j] > mine) + ((unsigned)(vals[j] >= mine) << 16);
        for (int o = 1; o < min(gs, 32); o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        if ((int)(n & 0xffffu) < top_k && top_k <= (int)(n >> 16)) sh.tie_index = (int)mine;
        __syncthreads();
        t = (uint32_t)sh.tie_index;
      } else {
        uint32_t keys[2 * CS];
#pragma unroll
        for (int r = 0; r < CS; ++r) {
          keys[2 * r] = peer(r)->k.maxima[tid];
          keys[2 * r + 1] = peer(r)->k.maxima[NT + tid];
        }
        uint32_t lo = 0, hi = kmax;  // count(>= lo) >= k; wanted: not many more
        const unsigned enough = (unsigned)top_k + max(16, top_k / 4);
        // a small row has too few half chunks: its logits themselves are counted
        const bool few = CS == 1 && V < top_k * VEC;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          unsigned n = 0;
          if (few) {
            each([&](float v, int, bool in) { n += in && float_key(v + 0.f) >= mid; });
          } else {
#pragma unroll
            for (int i = 0; i < 2 * CS; ++i) n += keys[i] >= mid;
          }
          n = block_sum32(n);
          if (n >= (unsigned)top_k) {
            lo = mid;
            if (n <= enough) break;
          } else {
            hi = mid - 1;
          }
        }
        t = lo;
      }
      __syncthreads();  // (the list takes the place of vals)
    }
    each([&](float v, int tok, bool in) {
      const bool take = in && float_key(v + 0.f) >= t;
      const unsigned bal = __ballot_sync(0xffffffffu, take);
      if (bal) {
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&sh.n, __popc(bal));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(bal & ((1u << lane) - 1));
        if (take && at < kList) sh.k.list[at] = composite(v, tok);
      }
    });
    all_sync();
    unsigned n = 0;
#pragma unroll
    for (int r = 0; r < CS; ++r) n += peer(r)->n;
    if (n <= kList) {
      if (rank == 0) {
        u64* s = reinterpret_cast<u64*>(dyn);  // [kList]; the part itself is no longer needed
        u64* ws = s + kList;                   // [kList]
        unsigned at = 0;
        for (int r = 0; r < CS; ++r) {
          const SampleShared* q = peer(r);
          const unsigned k = q->n;
          for (unsigned i = tid; i < k; i += NT) s[at + i] = q->k.list[i];
          at += k;
        }
        const unsigned k = min(n, (unsigned)top_k);
        if (n <= kPairs) {
          __syncthreads();
          for (unsigned i = tid; i < n; i += NT) ws[i] = fixed(weight(key_float((uint32_t)(s[i] >> 32)), m, c));
          __syncthreads();
          // gs threads per entry: its rank and the mass before it
          unsigned gs = 32;
          while (NT / gs < n) gs >>= 1;
          const unsigned i = tid / gs, part = tid % gs;
          const bool have = i < n;
          const u64 mine = have ? s[i] : 0, w = have ? ws[i] : 0;
          unsigned rk = 0;
          u64 before = 0;
          for (unsigned j = part; j < n; j += gs)
            if (s[j] > mine) ++rk, before += ws[j];
          for (unsigned o = 1; o < gs; o <<= 1) {
            rk += __shfl_xor_sync(0xffffffffu, rk, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
          }
          bool keep = have && rk < k;
          const u64 zk = block_sum(keep && part == 0 ? w : 0);
          if (keep && rk > 0) {
            if (top_p < 1.0) keep = (double)before < top_p * (double)zk;
            if (min_p > 0.0) keep = keep && weight(key_float((uint32_t)(mine >> 32)), m, c) >= min_p;
          }
          __syncthreads();
          if (part == 0 && have) ws[i] = keep ? w : 0;
          const u64 z = block_sum(keep && part == 0 ? w : 0);  // (its barriers order ws)
          // the mass before it by index: a smaller index has a larger complement
          before = 0;
          for (unsigned j = part; j < n; j += gs)
            if ((uint32_t)s[j] > (uint32_t)mine) before += ws[j];
          for (unsigned o = 1; o < gs; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
          const u64 target = drawn_mass(z);
          if (keep && part == 0 && target >= before && target < before + w)
            finish((int)(0xffffffffu - (uint32_t)mine), (double)w, (double)z);
        } else {
          const unsigned size = 1u << (32 - __clz(n - 1));
          for (unsigned i = n + tid; i < size; i += NT) s[i] = 0;
          auto sort_down = [&](unsigned size) {  // bitonic, descending
            for (unsigned k = 2; k <= size; k <<= 1)
              for (unsigned j = k >> 1; j > 0; j >>= 1) {
                __syncthreads();
                for (unsigned i = tid; i < size / 2; i += NT) {
                  const unsigned x = 2 * i - (i & (j - 1)), y = x + j;
                  const u64 p = s[x], q = s[y];
                  if (((x & k) == 0) == (p < q)) s[x] = q, s[y] = p;
                }
              }
            __syncthreads();
          };
          sort_down(size);
          static_assert(kListTopK == NT, "one rank per thread");
          const unsigned r = tid;
          u64 z;
          const double wd = r < k ? weight(key_float((uint32_t)(s[r] >> 32)), m, c) : 0.0;
          const u64 w = fixed(wd);
          u64 before = block_scan(w, &z) - w;
          const double reach = top_p < 1.0 ? top_p * (double)z : 2.0 * (double)z;
          const bool keep = r < k && (r == 0 || ((double)before < reach && wd >= min_p));
          // for the order by index: the complement of the token in the upper half, the rank below
          const u64 entry = keep ? (s[r] << 32) | r : 0;
          const unsigned kept = block_sum32(keep);  // the kept are the leading ranks
          __syncthreads();
          s[r] = entry;
          ws[r] = w;
          sort_down(max(64u, 1u << (32 - __clz(max(kept, 2u) - 1))));
          const u64 wi = r < kept ? ws[(uint32_t)s[r]] : 0;
          before = block_scan(wi, &z) - wi;
          const u64 target = drawn_mass(z);
          if (r < kept && target >= before && target < before + wi)
            finish((int)(0xffffffffu - (uint32_t)(s[r] >> 32)), (double)wi, (double)z);
        }
      }
      all_sync();
      return;
    }
    general = true;  // too many equal logits
  }

  // f(value) for the values for which want(value, token) holds, 32 at a time: they are
  // packed in the warp's queue, since the exact weights cost about 60 instructions each
  auto packed = [&](auto want, auto f) {
    int fill = 0;
    float* q = sh.p.queue[warp];
    each([&](float v, int t, bool in) {
      const bool take = want(v, t) && in;
      const unsigned bal = __ballot_sync(0xffffffffu, take);
      if (take) q[fill + __popc(bal & ((1u << lane) - 1))] = v;
      fill += __popc(bal);
      if (fill >= 32) {
        __syncwarp();
        const float x = q[lane], y = q[32 + lane];
        __syncwarp();
        q[lane] = y;
        __syncwarp();  // before other lanes append over it
        fill -= 32;
        f(x);
      }
    });
    __syncwarp();
    if (lane < fill) f(q[lane]);
    __syncwarp();
  };

  // The last step of every path below: sh.w_keep holds each warp's kept mass and
  // keep_of[r] each CTA's.  In the CTA that holds the drawn mass all warps share
  // the steps of the part that holds it.  sel(value, token): kept; w_of(value):
  // its mass; slack: the uncertainty of the sums (0: exact).  Returns true when
  // the draw is certain (the same in every CTA).
  auto draw = [&](const u64* keep_of, auto sel, auto w_of, u64 slack) -> bool {
    u64 z = 0, mine0 = 0, mine = 0;
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      if (r == rank) mine0 = z, mine = keep_of[r];
      z += keep_of[r];
    }
    const u64 target = drawn_mass(z);
    if (target >= mine0 && target < mine0 + mine) {
      auto find = [&](u64 v, u64* at) {  // first lane whose running sum from *at exceeds the target (32: none, all added)
        u64 incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, *at + incl > target);
        const int l = hit ? __ffs(hit) - 1 : 32;
        *at += __shfl_sync(0xffffffffu, hit ? incl - v : incl, hit ? l : 31);
        return l;
      };
      u64 at = mine0;
      const int hw = find(lane < NW ? sh.w_keep[lane] : 0, &at);
      const int hb = min(nch, hw * per_warp), he = min(nch, hb + per_warp);
      const int steps = sample_steps(he - hb);
      u64 w[VEC], sum = 0;
      auto weigh = [&](int s) {
        const int ch = hb + 32 * s + lane;
        const uint4 raw = chunk(ch, he);
        const T* e = reinterpret_cast<const T*>(&raw);
        sum = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int t = base + ch * VEC + j;
          const bool is = ch < he && (unsigned)t < (unsigned)V && sel(to_f(e[j]), t);
          w[j] = 0;
          if (__any_sync(0xffffffffu, is)) w[j] = is ? w_of(to_f(e[j])) : 0;
          sum += w[j];
        }
      };
      int last = -1;
      for (int s = warp; s < steps; s += NW) {
        weigh(s);
        last = s;
        const u64 t = warp_sum64(sum);
        if (lane == 0) sh.step[s] = t;
      }
      __syncthreads();
      int hs = 0, in = 32;  // the step that holds it is hs + in
      for (; hs < steps; hs += 32)
        if ((in = find(hs + lane < steps ? sh.step[hs + lane] : 0, &at)) < 32) break;
      hs += in;
      if (in == 32 || hw == 32) {  // the approximate sums of the two walks differ by their rounding
        if (tid == 0)
          for (int r = 0; r < CS; ++r) peer(r)->uncertain = 1;
      } else if (hs % NW == warp) {
        if (last != hs) weigh(hs);
        const int l = find(sum, &at);
        if (lane == l) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (target >= at && target < at + w[j]) {
              if (slack == 0 || (target >= at + slack && target + slack < at + w[j])) {
                finish(base + (hb + 32 * hs + lane) * VEC + j, (double)w[j], (double)z);
              } else {
                for (int r = 0; r < CS; ++r) peer(r)->uncertain = 1;
              }
            }
            at += w[j];
          }
        }
      }
    }
    all_sync();
    return sh.uncertain == 0;
  };
  // exact draw among the tokens with composite >= thr and weight >= min_p
  auto exact_of = [&](float v) -> u64 {
    const double w = weight(v, m, c);
    return w >= min_p ? fixed(w) : 0;
  };
  // exact mass of this thread's tokens for which want(value) holds: no packing, independent exponentials
  auto mass_of = [&](auto want) -> u64 {
    u64 acc = 0;
    uint4 next = chunk(wbeg + lane, wend);
    for (int ch = wbeg + lane; ch < wend; ch += 32) {
      const uint4 raw = next;
      next = chunk(ch + 32, wend);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll 1
      for (int h = 0; h < VEC; h += 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = VEC == 4 || h == 0 ? to_f(e[j]) : to_f(e[VEC - 4 + j]);
          const double x = fmin(((double)m - (double)v) * c, 60.0);
          const u64 f = fixed(exp2_neg(x));
          acc += !want(v) ? 0 : v == m ? (u64)kWeightOne : x < 60.0 ? f : 0;
        }
    }
    return acc;
  };
  auto draw_exact = [&](u64 thr) {
    u64 acc = 0;
    if (thr == 0 && min_p <= 0.0) {
      acc = mass_of([](float) { return true; });
    } else {
      packed([&](float v, int t) { return composite(v, t) >= thr; }, [&](float v) { acc += exact_of(v); });
    }
    acc = warp_sum64(acc);
    if (lane == 0) sh.w_keep[warp] = acc;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int w = 0; w < NW; ++w) s += sh.w_keep[w];
      sh.cta_keep = s;
    }
    all_sync();
    u64 keep_of[CS];
#pragma unroll
    for (int r = 0; r < CS; ++r) keep_of[r] = peer(r)->cta_keep;
    draw(keep_of, [&](float v, int t) { return composite(v, t) >= thr; }, exact_of, 0);
  };

  // A weight 2^-x in float32 (ex2.approx, at most 2^-22 off) errs relatively by at
  // most err_1 + x err_x: the difference m - l and the product with c are rounded
  // once each and c itself is off by a known factor, each moving the weight by x
  // ln 2 times its relative error; sums of VEC weights add VEC roundings.  Of a
  // sum S of weights the error is then at most S (err_1 + x0 err_x) and, as t 2^-t
  // is below 0.54, that of the weights beyond x0 V 2^-x0 0.54 err_x more.
  const double err_x = 0.6932 * (0x1p-23 + fabs((double)cf / c - 1.0)), err_1 = (4 + VEC) * 0x1p-24;
  auto sum_error = [&](double s, float x0) {
    return s * (err_1 + x0 * err_x) + 0.54 * V * (double)ex2_f32(-x0) * err_x;
  };
  if (!general && !by_mass) {
    // ---------------------------------------------------------------------
    // no top-k, no top-p: draw from the float32 masses when the drawn mass is
    // farther from the token's borders than their error, else from exact ones;
    // a log probability needs the exact sum anyway
    // ---------------------------------------------------------------------
    if (a.logp || !approx) {
      draw_exact(0);
      return;
    }
    const float x_min = min_p > 0.0 ? (float)(-log2(min_p)) : CUDART_INF_F;
    double sum = 0.0;
    bool border = false;
    uint4 next = chunk(wbeg + lane, wend);
    for (int ch = wbeg + lane; ch < wend; ch += 32) {
      const uint4 raw = next;
      next = chunk(ch + 32, wend);
      const T* e = reinterpret_cast<const T*>(&raw);
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = (m - to_f(e[j])) * cf;
        border |= x_min < CUDART_INF_F && fabsf(x - x_min) <= 1e-6f * (x_min + 1.f);
        s += x <= x_min ? ex2_f32(-x) : 0.f;
      }
      sum += (double)s;
    }
    if (border) atomicOr(&sh.uncertain, 1);
    sum = warp_sumd(sum);
    if (lane == 0) sh.w_keep[warp] = fixed(sum);
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int w = 0; w < NW; ++w) s += sh.w_keep[w];
      sh.cta_keep = s;
      sh.cta_ties = sh.uncertain;
    }
    all_sync();
    u64 keep_of[CS], z = 0;
    bool sure = true;
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      z += keep_of[r] = peer(r)->cta_keep;
      sure &= peer(r)->cta_ties == 0;
    }
    // both the running mass and u Z~ move with the error, and each token's and
    // warp's mass is rounded to the fixed point
    const u64 slack = (u64)(2.0 * sum_error((double)z / kWeightOne, 32.f) * kWeightOne) + (u64)V + 64;
    if (sure)
      sure = draw(keep_of, [&](float v, int) { return (m - v) * cf <= x_min; },
                  [&](float v) { return fixed((double)ex2_f32((v - m) * cf)); }, slack);
    else
      all_sync();  // every CTA has read the sums before they are written again
    if (!sure) draw_exact(0);
    return;
  }

  u64 thr = 0;  // kept: composite >= thr
  bool many = false;  // top-p with many tokens at the border: their keys, the mass above them and the reach
  uint32_t m_lo = 0, m_hi = 0;
  u64 m_above = 0;
  double m_reach = 0.0;
  if (!general) {
    // ---------------------------------------------------------------------
    // top-p.  With z_low <= Z a token below (1 - p) z_low / V cannot stay (all
    // tokens from it down have less than (1 - p) Z).  One pass sums the float32
    // weights to Z~ and makes a histogram over x of the masses that can; the
    // border lies in the one or few bins where the running mass passes p Z~.
    // The next pass sums the masses above those bins exactly and the tail in
    // float32 with its error bound, and the tokens of the bins are taken one
    // by one.  Where the error could move the border, the tail is summed
    // exactly as well.
    // ---------------------------------------------------------------------
    const float rest = fmaxf((float)(1.0 - top_p), 1e-17f);
    const float x_end = fmaxf(log2f((float)V / z_low) - log2f(rest), 0.f) * (1.f + 0x1p-9f) + 0.02f;
    // bin of a logit, as the float 2^23 + bin: adding 2^23 rounds to an integer in
    // the low mantissa bits (no conversion instruction), and falls with v
    const float bin_scale = fminf(cf * ((float)kBins / x_end), 3e38f);
    auto bin_at = [&](float v) { return fmaf(m - v, bin_scale, 8388608.f); };
    // masses in units of at most 2^-22, so that they come out the same way and all of them stay below 2^31
    const float unit = fminf(4194304.f, 2147483648.0f / z_high * (1.f - 1e-3f));
    for (int i = tid; i < kBins; i += NT) sh.p.hist[i] = 0;
    __syncthreads();
    const uint32_t hist_s = smem_addr(sh.p.hist);
    double sum = 0.0;
    uint4 next = chunk(wbeg + lane, wend);
    for (int ch = wbeg + lane; ch < wend; ch += 32) {
      const uint4 raw = next;
      next = chunk(ch + 32, wend);
      const T* e = reinterpret_cast<const T*>(&raw);
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float v = to_f(e[j]), b = bin_at(v), w = ex2_f32((v - m) * cf);
        s += w;
        const uint32_t bin = __float_as_uint(b) - 0x4b000000u;
        const uint32_t mass = __float_as_uint(fmaf(w, unit, 8388608.f)) - 0x4b000000u;
        asm volatile(
            "{\n .reg .pred p;\n setp.lt.u32 p, %0, %1;\n @p red.shared.add.u32 [%2], %3;\n}\n" ::"r"(bin), "n"(kBins),
            "r"(hist_s + 4u * bin), "r"(mass)
            : "memory");
      }
      sum += (double)s;
    }
    sum = warp_sumd(sum);
    if (lane == 0) sh.w_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int w = 0; w < NW; ++w) s += sh.w_sum[w];
      sh.cta_z = s;
    }
    all_sync();
    int blo, bhi;
    {
      static_assert(kBins == 2 * NT, "two bins per thread");
      double z = 0.0;
      uint32_t h0 = 0, h1 = 0;
#pragma unroll
      for (int r = 0; r < CS; ++r) {
        z += peer(r)->cta_z;
        const uint2 h = *reinterpret_cast<const uint2*>(&peer(r)->p.hist[2 * tid]);
        h0 += h.x;
        h1 += h.y;
      }
      // inclusive prefix sums of 32 bits: the masses are below 2^31 in all
      uint32_t incl = h0 + h1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) sh.step[warp] = incl;
      __syncthreads();
      incl += __reduce_add_sync(0xffffffffu, lane < warp ? (uint32_t)sh.step[lane] : 0u);
      const double reach = top_p * z * unit, margin = 0.5 * V + 3e-5 * z * unit;
      const long long below = (long long)floor(reach - margin), past = (long long)ceil(reach + margin);
      // number of bins whose running mass stays at or below either bound
      const unsigned n_lo = ((long long)(incl - h1) <= below) + ((long long)incl <= below);
      const unsigned n_hi = ((long long)(incl - h1) < past) + ((long long)incl < past);
      const unsigned both = block_sum32((n_hi << 16) | n_lo);
      blo = min((int)(both & 0xffffu), kBins - 1);
      bhi = min((int)(both >> 16), kBins - 1);
    }
    const float edge_lo = 8388608.f + (float)blo, edge_hi = 8388608.f + (float)(bhi + 1);
    u64 keep_of[CS];
    u64 acc_keep, acc_all;
    double tail;
    // the pass over the part: the tail in float32; what is above it goes through the
    // warp's queue, 32 at a time, to the exact masses or the bins' tokens
    auto tally = [&]() {
      acc_keep = acc_all = 0;
      tail = 0.0;
      int fill = 0;
      float* q = sh.p.queue[warp];
      uint16_t* qt = sh.p.queue_tok[warp];
      auto take = [&](float v, int t, bool is) {
        const bool border = is && bin_at(v) >= edge_lo;
        if (is && !border) {
          const double w = weight(v, m, c);
          const u64 f = fixed(w);
          acc_all += f;
          if (w >= min_p) acc_keep += f;
        }
        const unsigned bb = __ballot_sync(0xffffffffu, border);
        if (bb) {
          const uint32_t key = float_key(v + 0.f);
          const uint32_t lo = __reduce_min_sync(0xffffffffu, border ? key : ~0u);
          const uint32_t hi = __reduce_max_sync(0xffffffffu, border ? key : 0u);
          unsigned at = 0;
          if (lane == 0) {
            at = atomicAdd(&sh.n, __popc(bb));
            atomicMin(&sh.key_lo, lo);
            atomicMax(&sh.key_hi, hi);
          }
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(bb & ((1u << lane) - 1));
          if (border && at < kCands) sh.p.cand[at] = composite(v, base + wbeg * VEC + t);
        }
      };
      uint4 next = chunk(wbeg + lane, wend);
      for (int ch0 = wbeg; ch0 < wend; ch0 += 32) {
        const int ch = ch0 + lane;
        const uint4 raw = next;
        next = chunk(ch + 32, wend);
        const T* e = reinterpret_cast<const T*>(&raw);
        float s = 0.f;
        unsigned up = 0;  // elements above the tail
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = to_f(e[j]), w = ex2_f32((v - m) * cf);
          const bool in_tail = bin_at(v) >= edge_hi;
          s += in_tail ? w : 0.f;
          up |= in_tail ? 0u : 1u << j;
        }
        tail += (double)s;
        // one element per lane and turn
        for (unsigned bal = __ballot_sync(0xffffffffu, up != 0); bal; bal = __ballot_sync(0xffffffffu, up != 0)) {
          if (up) {
            const int j = __ffs(up) - 1;
            float v = to_f(e[0]);
#pragma unroll
            for (int i = 1; i < VEC; ++i)
              if (i == j) v = to_f(e[i]);
            const int at = fill + __popc(bal & ((1u << lane) - 1));
            q[at] = v;
            qt[at] = (uint16_t)((ch - wbeg) * VEC + j);
            up &= up - 1;
          }
          fill += __popc(bal);
          if (fill >= 32) {
            __syncwarp();
            const float v0 = q[lane], v1 = q[32 + lane];
            const uint16_t t0 = qt[lane], t1 = qt[32 + lane];
            __syncwarp();
            q[lane] = v1;
            qt[lane] = t1;
            __syncwarp();  // before other lanes append over it
            fill -= 32;
            take(v0, t0, true);
          }
        }
      }
      __syncwarp();
      take(q[lane], qt[lane], lane < fill);
      __syncwarp();
    };
    // the tail once more with an error below 1e-9 of it: independent Taylor series
    // of degree 8 in double (the first dropped term is (ln 2 / 2)^9 / 9! = 2e-10)
    auto fine_tail_sum = [&]() -> double {
      const double mc = (double)m * c;
      double acc = 0.0;
      uint4 next = chunk(wbeg + lane, wend);
      for (int ch = wbeg + lane; ch < wend; ch += 32) {
        const uint4 raw = next;
        next = chunk(ch + 32, wend);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll 1
        for (int h = 0; h < VEC; h += 4) {
          double s[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = VEC == 4 || h == 0 ? to_f(e[j]) : to_f(e[VEC - 4 + j]);
            const double x = fma((double)v, -c, mc);
            const bool is = bin_at(v) >= edge_hi && x < 60.0;  // beyond it a mass is nothing
            const double t = (is ? x : 0.0) + 6755399441055744.0;  // 1.5 * 2^52: x to the nearest integer
            const int n = __double2loint(t);
            const double g = (t - 6755399441055744.0) - (is ? x : 0.0);
            // 2^g, |g| <= 1/2, coefficients (ln 2)^k / k!
            double p = 1.3215486790144307e-06;
            p = fma(p, g, 1.5252733804059841e-05);
            p = fma(p, g, 1.5403530393381608e-04);
            p = fma(p, g, 1.3333558146428443e-03);
            p = fma(p, g, 9.6181291076284772e-03);
            p = fma(p, g, 5.5504108664821580e-02);
            p = fma(p, g, 2.4022650695910072e-01);
            p = fma(p, g, 6.9314718055994531e-01);
            p = fma(p, g, 1.0);
            s[j] = is ? __hiloint2double(__double2hiint(p) - (n << 20), __double2loint(p)) : 0.0;
          }
          acc += (s[0] + s[1]) + (s[2] + s[3]);
        }
      }
      return warp_sumd(acc);
    };
    tally();
    acc_keep = warp_sum64(acc_keep);
    acc_all = warp_sum64(acc_all);
    tail = warp_sumd(tail);
    if (lane == 0) {
      sh.w_keep[warp] = acc_keep;
      sh.w_all[warp] = acc_all;
      sh.w_sum[warp] = tail;
    }
    __syncthreads();
    if (tid == 0) {
      u64 k = 0, al = 0;
      double s = 0.0;
      for (int w = 0; w < NW; ++w) k += sh.w_keep[w], al += sh.w_all[w], s += sh.w_sum[w];
      sh.cta_keep = k, sh.cta_all = al, sh.cta_tail = s;
    }
    all_sync();
    u64 above = 0, own = 0;
    double tl = 0.0;
    unsigned n = 0;
    uint32_t key_lo = ~0u, key_hi = 0u;
    int src = -1;
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      const SampleShared* q = peer(r);
      key_lo = min(key_lo, q->key_lo);
      key_hi = max(key_hi, q->key_hi);
      keep_of[r] = q->cta_keep;
      above += q->cta_all;
      tl += q->cta_tail;
      const unsigned k = q->n;
      if (tid >= n && tid < n + k && k <= kCands) own = q->p.cand[tid - n], src = r;
      n += k;
    }
    double te = sum_error(tl, x_end);
    // the tail to 1e-9 of it, on demand: the same answer in every CTA
    auto refine_tail = [&]() {
      const double mine = fine_tail_sum();
      all_sync();  // (every CTA has read the sums)
      if (lane == 0) sh.w_sum[warp] = mine;
      __syncthreads();
      if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < NW; ++w) s += sh.w_sum[w];
        sh.cta_tail = s;
      }
      all_sync();
      tl = 0.0;
#pragma unroll
      for (int r = 0; r < CS; ++r) tl += peer(r)->cta_tail;
      te = 0.0;
    };
    // and exactly
    bool exact_tail = false;
    u64 tail_mass = 0;
    auto take_tail = [&]() {
      const u64 mine = block_sum(mass_of([&](float v) { return bin_at(v) >= edge_hi; }));
      all_sync();  // (every CTA has read what cta_all held)
      if (tid == 0) sh.cta_all = mine;
      all_sync();
#pragma unroll
      for (int r = 0; r < CS; ++r) tail_mass += peer(r)->cta_all;
      exact_tail = true;
    };
    // the mass that has to come before a token for it to be dropped, `in` being the
    // bins' own mass; sign -1, 1: bounds of it
    auto reach_of = [&](u64 in, double sign) {
      if (exact_tail) return top_p * (double)(above + in + tail_mass);
      return top_p * ((double)(above + in) + (tl + sign * te) * kWeightOne * (1.0 + sign * 1e-9) + sign * V);
    };
    bool resolved = false;
    if (n > 0 && n <= kCands) {
      // thread i < n holds token i of the border: its weight for the others
      const double own_w = src >= 0 ? weight(key_float((uint32_t)(own >> 32)), m, c) : 0.0;
      if (src >= 0) {
        sh.p.all[tid] = own;
        sh.p.wt[tid] = fixed(own_w);
      }
      __syncthreads();
      // gs threads per token: its rank in the bins and the mass before it
      unsigned gs = 16;
      while (NT / gs < n) gs >>= 1;
      const unsigned i = tid / gs, part = tid % gs;
      const bool have = i < n;
      const u64 mine = have ? sh.p.all[i] : 0;
      unsigned rk = 0;
      u64 before = 0, cands = 0;
      for (unsigned j = part; j < n; j += gs) {
        const u64 w = sh.p.wt[j];
        cands += w;
        if (sh.p.all[j] > mine) ++rk, before += w;
      }
      for (unsigned o = 1; o < gs; o <<= 1) {
        rk += __shfl_xor_sync(0xffffffffu, rk, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
        cands += __shfl_xor_sync(0xffffffffu, cands, o);
      }
      const bool first = above == 0 && rk == 0;  // the most likely token stays
      before += above;
      // does the error of the tail matter to this token, or to the bins?
      const double all_in = (double)(above + cands);
      auto unsure = [&]() {
        const double lo = reach_of(cands, -1.0), hi = reach_of(cands, 1.0);
        return __syncthreads_or((have && ((double)before < lo) != ((double)before < hi)) || (all_in >= lo) != (all_in >= hi));
      };
      if (unsure()) {
        refine_tail();
        if (unsure()) take_tail();
      }
      const double reach = reach_of(cands, 0.0);
      const bool keep = have && (first || (double)before < reach);
      // the border does lie in these bins (their histogram is approximate)
      if ((above == 0 || (double)above < reach) && all_in >= reach) {
        // threshold: the last kept token, or just above the first of them
        const unsigned kept = block_sum32(keep && part == 0);
        if (part == 0 && have && (kept ? rk == kept - 1 : rk == 0)) sh.thr = kept ? mine : mine + 1;
        // the kept join the masses of their CTAs and of this CTA's warps
        __syncthreads();
        thr = sh.thr;
        if (src >= 0 && own >= thr && own_w >= min_p) {
          const u64 f = fixed(own_w);
          atomicAdd(&sh.add[src], f);
          if (src == rank) atomicAdd(&sh.w_keep[(((int)(0xffffffffu - (uint32_t)own) - base) / VEC) / per_warp], f);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < CS; ++r) keep_of[r] += sh.add[r];
        resolved = true;
      }
    }
    if (resolved) {
      draw(keep_of, [&](float v, int t) { return composite(v, t) >= thr; }, exact_of, 0);
      return;
    }
    if (n > kCands) {  // too many to rank: the border key is sought among theirs, with exact sums
      take_tail();
      u64 in = 0;
      packed([&](float v, int) { const uint32_t k = float_key(v + 0.f); return k >= key_lo && k <= key_hi; },
             [&](float v) { in += fixed(weight(v, m, c)); });
      in = block_sum(in);
      all_sync();  // (and the tail)
      if (tid == 0) sh.cta_all = in;
      all_sync();
      in = 0;
#pragma unroll
      for (int r = 0; r < CS; ++r) in += peer(r)->cta_all;
      m_lo = key_lo, m_hi = key_hi, m_above = above;
      m_reach = reach_of(in, 0.0);
      many = (above == 0 || (double)above < m_reach) && (double)(above + in) >= m_reach;  // (or the bins were wrong)
    }
    all_sync();
  }

  // -----------------------------------------------------------------------
  // general: the border key by radix selection, 8 bits a pass, on exact counts
  // (top-k) and masses (top-p); then the place of the last kept token among
  // those of the border key
  // -----------------------------------------------------------------------
  // largest K in [lo, hi] with `run` (the sum over keys > hi) plus the sum over
  // keys K .. hi reaching `target`; *above = the sum over keys > K
  auto select = [&](bool by_weight, double target, uint32_t lo, uint32_t hi, u64 run, u64* above) -> uint32_t {
    const int first = lo == hi ? -8 : (31 - __clz(lo ^ hi)) / 8 * 8;
    uint32_t prefix = lo == hi ? hi : first == 24 ? 0u : hi & (~0u << (first + 8));
    for (int shift = first; shift >= 0; shift -= 8) {
      const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int i = tid; i < 256; i += NT) sh.p.mass[i] = 0;
      __syncthreads();
      each([&](float v, int, bool in) {
        const uint32_t k = float_key(v + 0.f);
        const bool take = in && k >= lo && k <= hi && (k & mask) == prefix;
        const unsigned act = __ballot_sync(0xffffffffu, take);
        if (!act) return;
        u64 w = 0;
        if (take) w = by_weight ? fixed(weight(v, m, c)) : 1;
        const int b = (k >> shift) & 255, lead = __shfl_sync(0xffffffffu, b, __ffs(act) - 1);
        if (__all_sync(0xffffffffu, !take || b == lead)) {  // one bin: one addition
          w = warp_sum64(w);
          if (lane == 0) atomicAdd(&sh.p.mass[lead], w);
        } else if (take) {
          atomicAdd(&sh.p.mass[b], w);
        }
      });
      all_sync();
      // bins from the top: thread t holds bin 255 - t
      u64 h = 0, total;
      if (tid < 256)
        for (int r = 0; r < CS; ++r) h += peer(r)->p.mass[255 - tid];
      const u64 incl = block_scan(h, &total);
      // bins passed before the target is reached
      const bool passed = tid < 256 && (double)(run + incl) < target;
      const unsigned np = min(block_sum32(passed), 255u);
      __syncthreads();
      if (tid == np) sh.thr = run + incl - h;
      __syncthreads();
      run = sh.thr;
      prefix |= (255u - np) << shift;
      all_sync();  // the histograms have been read
    }
    *above = run;
    return prefix;
  };
  all_sync();  // (a list that was too long has been counted by every CTA)
  uint32_t K = 0;
  u64 ties = ~0ull, above = 0;
  double reach = m_reach;
  bool by_reach = many;  // of the tokens of key K those stay that have less than `reach` before them
  if (many) {
    K = select(true, reach, m_lo, m_hi, m_above, &above);
  } else {
    if (top_k < V) {
      K = select(false, (double)top_k, 0, kmax, 0, &above);
      ties = (u64)top_k - above;
    }
    // mass of the top-k set
    u64 acc = 0, zk = 0;
    packed([&](float v, int) { return float_key(v + 0.f) > K; }, [&](float v) { acc += fixed(weight(v, m, c)); });
    acc = block_sum(acc);
    if (tid == 0) sh.cta_all = acc;
    all_sync();
#pragma unroll
    for (int r = 0; r < CS; ++r) zk += peer(r)->cta_all;
    if (top_k < V) zk += ties * fixed(weight(key_float(K), m, c));
    if (top_p < 1.0) {
      by_reach = true;
      reach = top_p * (double)zk;
      uint32_t kp = select(true, reach, 0, kmax, 0, &above);
      if (reach <= 0.0) kp = kmax, above = 0;
      if (kp > K) {
        K = kp;
        ties = ~0ull;
      } else if (top_k < V) {  // the border lies among the ties of the top-k border
        above = zk - ties * fixed(weight(key_float(K), m, c));
      }
    }
  }
  if (by_reach) {
    const u64 w = fixed(weight(key_float(K), m, c));
    u64 n = w ? (u64)fmin(fmax(0.0, (reach - (double)above) / (double)w), 262144.0) : 0;
    while (n > 0 && (double)(above + (n - 1) * w) >= reach) --n;
    while (n < 262144 && w && (double)(above + n * w) < reach) ++n;
    if (K == kmax && n == 0) n = 1;
    ties = min(ties, n);
  }
  if (ties == 0) {
    thr = ((u64)K + 1) << 32;
  } else if (ties >= 262144) {
    thr = (u64)K << 32;
  } else {
    // index of the ties-th token of key K
    u64 mine = 0, total;
    each([&](float v, int, bool in) { mine += in && float_key(v + 0.f) == K; });
    mine = warp_sum64(mine);
    if (lane == 0) sh.w_all[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int w = 0; w < NW; ++w) s += sh.w_all[w];
      sh.cta_ties = s;
      sh.tie_index = 0x7fffffff;  // fewer ties than that: all of them stay
    }
    all_sync();
    total = 0;
    for (int r = 0; r < rank; ++r) total += peer(r)->cta_ties;
    for (int w = 0; w < warp; ++w) total += sh.w_all[w];
    if (total < ties && total + mine >= ties) {
      u64 run = total;
      for (int ch0 = wbeg; ch0 < wend; ch0 += 32) {
        const int ch = ch0 + lane;
        const uint4 raw = chunk(ch, wend);
        const T* e = reinterpret_cast<const T*>(&raw);
        unsigned n = 0, eq = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int t = base + ch * VEC + j;
          const bool is = ch < wend && (unsigned)t < (unsigned)V && float_key(to_f(e[j]) + 0.f) == K;
          eq |= (unsigned)is << j;
          n += is;
        }
        u64 incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        u64 b = run + incl - n;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if ((eq >> j) & 1) {
            if (++b == ties)
              for (int r = 0; r < CS; ++r) peer(r)->tie_index = base + ch * VEC + j;
          }
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    all_sync();
    thr = sh.tie_index == 0x7fffffff ? (u64)K << 32 : ((u64)K << 32) | (0xffffffffu - (unsigned)sh.tie_index);
  }
  draw_exact(thr);
}

// Parts up to this size are staged: two CTAs then share an SM.
constexpr int kStageBytes = 99 * 1024;
static_assert(kStageBytes >= kList * 16, "a list fits where a part does");

template <typename T, int CS, bool STAGE>
static int launch_sample_as(const SampleArgs<T>& a, int part, cudaStream_t s) {
  const int smem = max(STAGE ? part : 0, kList * 16);  // a list takes the part's place, with its weights
  auto* kern = sample_kernel<T, CS, STAGE>;
  // the most of any call: the limit holds for the whole process, and another thread's call may come between this and the launch
  if (STAGE && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStageBytes) != cudaSuccess)
    return launch_status();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * CS);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CS;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, a);
  return launch_status();
}

template <typename T, int CS>
static int launch_sample(const SampleArgs<T>& a, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int part = sample_cta_chunks(sample_chunks(a.vocab, VEC - 1, VEC), CS) * 16;
  constexpr int most = sample_cta_chunks(sample_chunks(kSampleMaxVocab, VEC - 1, VEC), CS) * 16;  // of any vocabulary
  if constexpr (most > kStageBytes)
    if (part > kStageBytes) return launch_sample_as<T, CS, false>(a, part, s);
  return launch_sample_as<T, CS, true>(a, part, s);
}

}  // namespace walsh

using namespace walsh;

extern "C" walsh_status walsh_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t rows, int vocab,
                                            const float* u, double temperature, int top_k, double top_p, double min_p,
                                            const float* temperature_rows, const int32_t* top_k_rows,
                                            const float* top_p_rows, const float* min_p_rows, int64_t* ids,
                                            float* logp, void* stream) {
  if (int e = injected("sample_tokens")) return e;
  WALSH_CHECK_DTYPE(dtype);
  WALSH_CHECK_SHAPE(rows >= 0 && rows < (1ll << 28) && vocab > 0 && vocab <= kSampleMaxVocab && ld >= 0);
  if (rows == 0) return WALSH_OK;
  WALSH_CHECK_ARG(logits && u && ids);
  WALSH_CHECK_ARG(temperature_rows || temperature >= 0.0);
  WALSH_CHECK_ARG(top_p_rows || top_p == top_p);
  WALSH_CHECK_ARG(min_p_rows || min_p == min_p);
  return WALSH_DISPATCH_DTYPE(dtype, ET, [&]() -> int {
    SampleArgs<ET> a;
    a.logits = (const ET*)logits, a.ld = ld, a.rows = (int)rows, a.vocab = vocab, a.u = u;
    a.temperature = temperature, a.top_p = top_p, a.min_p = min_p, a.top_k = top_k;
    a.temperature_r = temperature_rows, a.top_p_r = top_p_rows, a.min_p_r = min_p_rows, a.top_k_r = top_k_rows;
    a.ids = ids, a.logp = logp;
    cudaStream_t s = (cudaStream_t)stream;
    switch (sample_cluster(rows, vocab)) {
      case 1: return launch_sample<ET, 1>(a, s);
      case 2: return launch_sample<ET, 2>(a, s);
      case 4: return launch_sample<ET, 4>(a, s);
      default: return launch_sample<ET, 8>(a, s);
    }
  }());
}
