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
// A token at a border is kept or dropped whole, so the weights and their sums
// are held to about 2^-45 of the largest weight: exp in double, rounded to a
// 64-bit integer multiple of 2^-44.  Integer sums do not depend on the order
// they are taken in, so neither do the draws.  The vocabulary is limited to
// 2^18 tokens, which keeps every sum below 2^63.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "common.cuh"
#include "mma.cuh"
#include "paged.cuh"

namespace walsh {

constexpr int kSampleMaxVocab = 1 << 18;
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

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 1024;      // bins of the mass histogram
constexpr int kCands = 512;      // tokens resolved one by one at a top-p border
constexpr int kList = 2048;      // tokens of a top-k list (sorted in shared memory)
constexpr int kListTopK = 512;   // largest top_k that goes by the list

struct SampleShared {
  union {
    struct {
      uint32_t maxima[2 * kSampleThreads];
      u64 list[kList];
    } k;
    struct {
      uint32_t hist[kBins];
      u64 cand[kCands], all[kCands];
      uint8_t from[kCands];
    } p;
    struct {
      u64 mass[256];
      uint32_t count[256];
    } r;
  };
  float queue[kSampleWarps][64];
  u64 w_keep[kSampleWarps], w_all[kSampleWarps], scratch[kSampleWarps];
  double w_sum[kSampleWarps], w_err[kSampleWarps];
  // what other CTAs of the cluster read
  u64 cta_keep, cta_all, cta_ties;
  double cta_sum, cta_err;
  uint32_t cta_max, n;
  // what the CTA that finds it writes into every CTA
  int tie_index, uncertain;
};

// One cluster of CS CTAs per row, each holding a contiguous part of the row in
// shared memory; each warp owns a contiguous part of that, so index order is
// (CTA, warp, position).
template <typename T, int CS>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs<T> a) {
  constexpr int NT = kSampleThreads, NW = kSampleWarps, VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SampleShared sh;
  T* seg = reinterpret_cast<T*>(dyn);
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
  const float cf = fminf(fmaxf((float)c, 1.2e-38f), 3e38f);

  // ---- the row's part of this CTA; chunks of 16 bytes, `mis` elements before the row's first chunk boundary
  const T* lg = a.logits + (int64_t)row * a.ld;
  const int mis = (int)(((uintptr_t)lg & 15) / sizeof(T));
  const int chunks = (mis + V + VEC - 1) / VEC, per_cta = (chunks + CS - 1) / CS;
  const int c0 = rank * per_cta, nch = max(0, min(per_cta, chunks - c0));
  const int per_warp = (nch + NW - 1) / NW;
  const int wbeg = min(nch, warp * per_warp), wend = min(nch, wbeg + per_warp);
  const int base = c0 * VEC - mis;  // token of the part's first element (negative: before the row)
  float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
  {
    constexpr int U = 4;
    for (int ch0 = wbeg + lane; ch0 < wend; ch0 += 32 * U) {
      uint4 raw[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int ch = ch0 + 32 * i, t0 = base + ch * VEC;
        if (ch >= wend) continue;
        if (t0 >= 0 && t0 + VEC <= V) {
          raw[i] = __ldcs(reinterpret_cast<const uint4*>(lg + t0));
        } else {
          T* e = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
          for (int j = 0; j < VEC; ++j) e[j] = t0 + j >= 0 && t0 + j < V ? lg[t0 + j] : round_f<T>(-CUDART_INF_F);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int ch = ch0 + 32 * i;
        if (ch >= wend) continue;
        T* e = reinterpret_cast<T*>(&raw[i]);
        bool nan = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = to_f(e[j]);
          nan |= v != v;
          if (j < VEC / 2) mx0 = fmaxf(mx0, v);
          else mx1 = fmaxf(mx1, v);
        }
        if (nan) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (to_f(e[j]) != to_f(e[j])) e[j] = round_f<T>(-CUDART_INF_F);
        }
        *reinterpret_cast<uint4*>(seg + (int64_t)ch * VEC) = raw[i];
      }
    }
  }
  // f(value, token) for this lane's elements of the warp's part, in order of the
  // warp's steps; every lane makes the same number of calls (in = false: no element)
  auto each = [&](auto f) {
    for (int ch0 = wbeg; ch0 < wend; ch0 += 32) {
      const int ch = ch0 + lane;
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      if (ch < wend) raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int t = base + ch * VEC + j;
        f(to_f(e[j]), t, ch < wend && (unsigned)t < (unsigned)V);
      }
    }
  };
  auto composite = [](float v, int t) { return ((u64)float_key(v + 0.f) << 32) | (0xffffffffu - (unsigned)t); };

  // ---- maximum of the row
  const uint32_t mk0 = float_key(mx0 + 0.f), mk1 = float_key(mx1 + 0.f);
  {
    const uint32_t wm = __reduce_max_sync(0xffffffffu, max(mk0, mk1));
    sh.k.maxima[tid] = mk0;
    sh.k.maxima[NT + tid] = mk1;
    if (lane == 0) sh.scratch[warp] = wm;
    if (tid == 0) sh.n = 0, sh.uncertain = 0;
    __syncthreads();
    if (warp == 0) {
      const uint32_t cm = __reduce_max_sync(0xffffffffu, lane < NW ? (uint32_t)sh.scratch[lane] : 0u);
      if (lane == 0) sh.cta_max = cm;
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
  if (m == CUDART_INF_F && !greedy) {  // the +inf logits share the weight, nothing else has any
    for (int i = tid; i < nch * VEC; i += NT)
      seg[i] = to_f(seg[i]) == CUDART_INF_F ? round_f<T>(0.f) : round_f<T>(-CUDART_INF_F);
    m = 0.f;
    kmax = float_key(0.f);
    const bool i0 = mx0 == CUDART_INF_F, i1 = mx1 == CUDART_INF_F;
    all_sync();
    sh.k.maxima[tid] = float_key(i0 ? 0.f : -CUDART_INF_F);
    sh.k.maxima[NT + tid] = float_key(i1 ? 0.f : -CUDART_INF_F);
    all_sync();
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

  // sum over the block of one value per thread
  auto block_sum = [&](u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh.scratch[warp] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += sh.scratch[w];
    return s;
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
  auto drawn_mass = [&](u64 z) {  // the running mass that the drawn token is the first to exceed
    const double uz = u * (double)z;
    const u64 t = uz > 0.0 ? (uz < 9.2e18 ? (u64)uz : z - 1) : 0;
    return t < z ? t : z - 1;
  };

  // -----------------------------------------------------------------------
  // top-k by a list: a lower bound t of the k-th largest logit comes from the
  // maxima of half chunks (k of those reach t, so k logits do), the logits from
  // t up are gathered and sorted, and everything else happens on the list.
  // -----------------------------------------------------------------------
  bool general = top_k < V;
  if (top_k < V && top_k <= kListTopK) {
    uint32_t t = 0;
    if (V > kList) {
      uint32_t keys[2 * CS];
#pragma unroll
      for (int r = 0; r < CS; ++r) {
        keys[2 * r] = peer(r)->k.maxima[tid];
        keys[2 * r + 1] = peer(r)->k.maxima[NT + tid];
      }
      uint32_t lo = 0, hi = kmax;  // count(>= lo) >= k; wanted: not many more
      const unsigned enough = (unsigned)top_k + max(16, top_k / 4);
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        unsigned n = 0;
#pragma unroll
        for (int i = 0; i < 2 * CS; ++i) n += keys[i] >= mid;
        n = (unsigned)block_sum(n);
        if (n >= (unsigned)top_k) {
          lo = mid;
          if (n <= enough) break;
        } else {
          hi = mid - 1;
        }
      }
      t = lo;
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
        u64* s = reinterpret_cast<u64*>(dyn);  // the part itself is no longer needed
        const unsigned size = n <= 64 ? 64 : 1u << (32 - __clz(n - 1));
        __syncthreads();
        unsigned at = 0;
        for (int r = 0; r < CS; ++r) {
          const SampleShared* q = peer(r);
          const unsigned k = q->n;
          for (unsigned i = tid; i < k; i += NT) s[at + i] = q->k.list[i];
          at += k;
        }
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
        const unsigned k = min(n, (unsigned)top_k);
        constexpr int PER = kListTopK / NT;  // ranks per thread, consecutive
        u64 w[PER], mine = 0, z;
        double wd[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned r = tid * PER + i;
          wd[i] = r < k ? weight(key_float((uint32_t)(s[r] >> 32)), m, c) : 0.0;
          w[i] = fixed(wd[i]);
          mine += w[i];
        }
        u64 before = block_scan(mine, &z) - mine;
        const double reach = top_p < 1.0 ? top_p * (double)z : 2.0 * (double)z;
        unsigned kept = 0;
        u64 entry[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned r = tid * PER + i;
          const bool keep = r < k && (r == 0 || ((double)before < reach && wd[i] >= min_p));
          kept += keep;
          // for the order by index: token in the upper half (its complement sorts it), rank below
          entry[i] = keep ? (s[r] << 32) | r : 0;
          before += w[i];
        }
        kept = (unsigned)block_sum(kept);
        __syncthreads();
        u64* wr = sh.k.list;  // weights by rank; every CTA's list has been read
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          s[tid * PER + i] = entry[i];
          wr[tid * PER + i] = w[i];
        }
        // the kept are the leading ranks
        const unsigned size2 = kept <= 64 ? 64 : 1u << (32 - __clz(kept - 1));
        sort_down(size2);  // descending complement of the index: ascending index
        mine = 0;
        u64 wi[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned r = tid * PER + i;
          wi[i] = r < kept ? wr[(uint32_t)s[r]] : 0;
          mine += wi[i];
        }
        before = block_scan(mine, &z) - mine;
        const u64 target = drawn_mass(z);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned r = tid * PER + i;
          if (r < kept && target >= before && target < before + wi[i]) {
            const int tok = (int)(0xffffffffu - (uint32_t)(s[r] >> 32));
            finish(tok, (double)wi[i], (double)z);
          }
          before += wi[i];
        }
      }
      all_sync();
      return;
    }
  }

  // f(value) for the values for which want(value, token) holds, 32 at a time: they are
  // packed in the warp's queue, since the exact weights cost about 60 instructions each
  auto packed = [&](auto want, auto f) {
    int fill = 0;
    float* q = sh.queue[warp];
    each([&](float v, int t, bool in) {
      const bool take = in && want(v, t);
      const unsigned bal = __ballot_sync(0xffffffffu, take);
      if (take) q[fill + __popc(bal & ((1u << lane) - 1))] = v;
      fill += __popc(bal);
      if (fill >= 32) {
        __syncwarp();
        const float x = q[lane], y = q[32 + lane];
        __syncwarp();
        q[lane] = y;
        fill -= 32;
        f(x);
      }
    });
    __syncwarp();
    if (lane < fill) f(q[lane]);
    __syncwarp();
  };
  auto warp_sum64 = [&](u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };

  // The last step of every path below: sh.w_keep holds each warp's kept mass and
  // keep_of[r] each CTA's; the warp that holds the drawn mass walks its part.
  // w_of(value, token) is a token's kept mass; slack the uncertainty of the sums
  // (0: exact).  Returns true when the draw is certain (the same in every CTA).
  auto draw = [&](const u64* keep_of, auto w_of, u64 slack) -> bool {
    u64 z = 0, mine0 = 0;
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      if (r == rank) mine0 = z;
      z += keep_of[r];
    }
    const u64 target = drawn_mass(z);
    if (target >= mine0 && target < mine0 + keep_of[rank]) {
      u64 acc = mine0;
      for (int w = 0; w < warp; ++w) acc += sh.w_keep[w];
      if (target >= acc && target < acc + sh.w_keep[warp]) {
        bool done = false;
        for (int ch0 = wbeg; ch0 < wend && !done; ch0 += 32) {
          const int ch = ch0 + lane;
          uint4 raw = make_uint4(0u, 0u, 0u, 0u);
          if (ch < wend) raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
          const T* e = reinterpret_cast<const T*>(&raw);
          u64 w[VEC], s = 0;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int t = base + ch * VEC + j;
            w[j] = ch < wend && (unsigned)t < (unsigned)V ? w_of(to_f(e[j]), t) : 0;
            s += w[j];
          }
          u64 incl = s;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, acc + incl > target);
          if (hit) {
            done = true;
            if (lane == __ffs(hit) - 1) {
              u64 b = acc + incl - s;
#pragma unroll
              for (int j = 0; j < VEC; ++j) {
                if (target >= b && target < b + w[j]) {
                  const bool sure = slack == 0 || (target >= b + slack && target + slack < b + w[j]);
                  if (sure) {
                    finish(base + ch * VEC + j, (double)w[j], (double)z);
                  } else {
                    for (int r = 0; r < CS; ++r) peer(r)->uncertain = 1;
                  }
                }
                b += w[j];
              }
            }
          }
          acc += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (!done && lane == 0)  // the approximate sums of the two walks may differ by their rounding
          for (int r = 0; r < CS; ++r) peer(r)->uncertain = 1;
      }
    }
    all_sync();
    return sh.uncertain == 0;
  };
  // exact draw among the tokens with composite >= thr and weight >= min_p
  auto draw_exact = [&](u64 thr) {
    u64 acc = 0;
    packed([&](float v, int t) { return composite(v, t) >= thr; },
           [&](float v) {
             const double w = weight(v, m, c);
             if (w >= min_p) acc += fixed(w);
           });
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
    draw(keep_of,
         [&](float v, int t) -> u64 {
           if (composite(v, t) < thr) return 0;
           const double w = weight(v, m, c);
           return w >= min_p ? fixed(w) : 0;
         },
         0);
  };

  // Sum of the weights in float32 (ex2.approx, at most 2 ulp): Z~, and a bound of
  // its error: x = (m - l) c carries 3 roundings, each moving the weight by
  // x 2^-24 ln 2; the exponential 2^-22; sums of VEC weights VEC roundings.
  const float err_x = 3.f * 0.7f * 5.9604645e-8f, err_1 = (4.f + VEC) * 5.9604645e-8f;
  if (!general && !(top_p < 1.0)) {
    // ---------------------------------------------------------------------
    // no top-k, no top-p: draw from the float32 masses when the drawn mass is
    // farther from the token's borders than their error, else from exact ones;
    // a log probability needs the exact sum anyway
    // ---------------------------------------------------------------------
    if (a.logp) {
      draw_exact(0);
      return;
    }
    const float x_min = min_p > 0.0 ? (float)(-log2(min_p)) : CUDART_INF_F;
    double sum = 0.0, err = 0.0;
    bool border = false;
    for (int ch = wbeg + lane; ch < wend; ch += 32) {
      const uint4 raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
      const T* e = reinterpret_cast<const T*>(&raw);
      float s = 0.f, se = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = (m - to_f(e[j])) * cf;
        const float w = x <= x_min ? ex2_f32(-x) : 0.f;
        border |= x_min < CUDART_INF_F && fabsf(x - x_min) <= 1e-6f * (x_min + 1.f);
        s += w;
        if (w > 0.f) se = fmaf(w, fmaf(x, err_x, err_1), se);
      }
      sum += (double)s;
      err += (double)se;
    }
    if (border) atomicOr(&sh.uncertain, 1);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      err += __shfl_xor_sync(0xffffffffu, err, o);
    }
    if (lane == 0) {
      sh.w_keep[warp] = fixed(sum);
      sh.w_err[warp] = err;
    }
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      double e = 0.0;
      for (int w = 0; w < NW; ++w) s += sh.w_keep[w], e += sh.w_err[w];
      sh.cta_keep = s;
      sh.cta_err = e;
      sh.cta_ties = sh.uncertain;
    }
    all_sync();
    u64 keep_of[CS];
    double e = 0.0;
    bool sure = true;
#pragma unroll
    for (int r = 0; r < CS; ++r) {
      keep_of[r] = peer(r)->cta_keep;
      e += peer(r)->cta_err;
      sure &= peer(r)->cta_ties == 0;
    }
    // both the running mass and u Z~ move with the error, and each token's and
    // warp's mass is rounded to the fixed point
    const u64 slack = (u64)(2.0 * e * kWeightOne) + (u64)V + 64;
    if (sure)
      sure = draw(keep_of,
                  [&](float v, int) -> u64 {
                    const float x = (m - v) * cf;
                    return x <= x_min ? fixed((double)ex2_f32(-x)) : 0;
                  },
                  slack);
    else
      all_sync();  // every CTA has read the sums before they are written again
    if (!sure) draw_exact(0);
    return;
  }

  u64 thr = 0;  // kept: composite >= thr
  if (!general) {
    // ---------------------------------------------------------------------
    // top-p.  Z~ bounds the weights that can stay (a token below (1 - p) Z / V
    // cannot: all tokens from it down would have less than (1 - p) Z); a
    // histogram of their float32 masses over x gives a few bins that hold the
    // border; the masses above those bins are summed exactly, the tail in
    // float32 with its error bound, and the tokens of the bins are taken one
    // by one.  Where the error could move the border, the tail is summed
    // exactly as well.
    // ---------------------------------------------------------------------
    double sum = 0.0;
    for (int ch = wbeg + lane; ch < wend; ch += 32) {
      const uint4 raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
      const T* e = reinterpret_cast<const T*>(&raw);
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += ex2_f32((to_f(e[j]) - m) * cf);
      sum += (double)s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.w_sum[warp] = sum;
    // (the maxima of the union are not read any more: no list was made)
    for (int i = tid; i < kBins; i += NT) sh.p.hist[i] = 0;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int w = 0; w < NW; ++w) s += sh.w_sum[w];
      sh.cta_sum = s;
    }
    all_sync();
    double z = 0.0;
#pragma unroll
    for (int r = 0; r < CS; ++r) z += peer(r)->cta_sum;
    const double rest = fmax(1.0 - top_p, 1e-17);
    const float x_end = (float)fmax(log2((double)V / (rest * z)), 0.0) + 0.01f;
    const float bin_scale = (float)kBins / x_end, unit = (float)(2147483648.0 / z * (1.0 - 1e-4));
    auto bin_of = [&](float v) { return min((m - v) * cf * bin_scale, (float)kBins + 1.f); };  // monotone in v
    each([&](float v, int, bool in) {
      const float b = bin_of(v);
      if (in && b < (float)kBins) atomicAdd(&sh.p.hist[(int)b], __float2uint_rn(ex2_f32((v - m) * cf) * unit));
    });
    all_sync();
    int blo, bhi;
    {
      static_assert(kBins == 2 * NT, "two bins per thread");
      u64 h0 = 0, h1 = 0, total;
#pragma unroll
      for (int r = 0; r < CS; ++r) {
        h0 += peer(r)->p.hist[2 * tid];
        h1 += peer(r)->p.hist[2 * tid + 1];
      }
      const u64 incl = block_scan(h0 + h1, &total);
      const double reach = top_p * z * unit, margin = 0.5 * V + 3e-5 * z * unit;
      // number of bins whose running mass stays at or below either bound
      const unsigned n_lo = ((double)(incl - h1) <= reach - margin) + ((double)incl <= reach - margin);
      const unsigned n_hi = ((double)(incl - h1) < reach + margin) + ((double)incl < reach + margin);
      const u64 both = block_sum(((u64)n_hi << 32) | n_lo);
      blo = min((int)(both & 0xffffffffu), kBins - 1);
      bhi = min((int)(both >> 32), kBins - 1);
    }
    all_sync();  // every CTA has read the histograms: the union is free
    const float edge_lo = (float)blo, edge_hi = (float)(bhi + 1);
    bool exact_tail = false, resolved = false;
    u64 keep_of[CS];
    for (;;) {
      if (tid == 0) sh.n = 0;
      __syncthreads();
      u64 acc_keep = 0, acc_all = 0, acc_tail = 0;
      double tail = 0.0, tail_err = 0.0;
      packed(
          [&](float v, int t) {
            const float b = bin_of(v);
            if (b >= edge_lo && b < edge_hi) {
              const unsigned at = atomicAdd(&sh.n, 1u);
              if (at < kCands) sh.p.cand[at] = composite(v, t);
            }
            return b < edge_lo || (exact_tail && b >= edge_hi);
          },
          [&](float v) {
            const double w = weight(v, m, c);
            const u64 f = fixed(w);
            if (bin_of(v) < edge_lo) {
              acc_all += f;
              if (w >= min_p) acc_keep += f;
            } else {
              acc_tail += f;
            }
          });
      if (!exact_tail) {
        for (int ch = wbeg + lane; ch < wend; ch += 32) {
          const uint4 raw = *reinterpret_cast<const uint4*>(seg + (int64_t)ch * VEC);
          const T* e = reinterpret_cast<const T*>(&raw);
          float s = 0.f, se = 0.f;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float v = to_f(e[j]), x = (m - v) * cf;
            const float w = bin_of(v) >= edge_hi ? ex2_f32(-x) : 0.f;
            s += w;
            if (w > 0.f) se = fmaf(w, fmaf(x, err_x, err_1), se);
          }
          tail += (double)s;
          tail_err += (double)se;
        }
      }
      acc_keep = warp_sum64(acc_keep);
      acc_all = warp_sum64(acc_all);
      acc_tail = warp_sum64(acc_tail);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        tail += __shfl_xor_sync(0xffffffffu, tail, o);
        tail_err += __shfl_xor_sync(0xffffffffu, tail_err, o);
      }
      if (lane == 0) {
        sh.w_keep[warp] = acc_keep;
        sh.w_all[warp] = acc_all;
        sh.w_sum[warp] = exact_tail ? (double)acc_tail / kWeightOne : tail;
        sh.w_err[warp] = tail_err;
      }
      __syncthreads();
      if (tid == 0) {
        u64 k = 0, al = 0;
        double s = 0.0, e = 0.0;
        for (int w = 0; w < NW; ++w) k += sh.w_keep[w], al += sh.w_all[w], s += sh.w_sum[w], e += sh.w_err[w];
        sh.cta_keep = k, sh.cta_all = al, sh.cta_sum = s, sh.cta_err = e;
      }
      all_sync();
      u64 above = 0;
      double tl = 0.0, te = 0.0;
      unsigned n = 0;
#pragma unroll
      for (int r = 0; r < CS; ++r) {
        const SampleShared* q = peer(r);
        keep_of[r] = q->cta_keep;
        above += q->cta_all;
        tl += q->cta_sum;
        te += q->cta_err;
        n += q->n;
      }
      if (n == 0 || n > kCands) break;  // too many tokens at the border: the general way
      unsigned at = 0;
      for (int r = 0; r < CS; ++r) {
        const SampleShared* q = peer(r);
        const unsigned k = q->n;
        for (unsigned i = tid; i < k; i += NT) {
          sh.p.all[at + i] = q->p.cand[i];
          sh.p.from[at + i] = (uint8_t)r;
        }
        at += k;
      }
      __syncthreads();
      // this thread's candidate: the mass before it
      static_assert(kCands == NT, "one candidate per thread");
      const bool have = tid < n;
      const u64 mine = have ? sh.p.all[tid] : 0;
      const double wd = have ? weight(key_float((uint32_t)(mine >> 32)), m, c) : 0.0;
      const u64 wf = fixed(wd);
      u64 before = above;
      const u64 cands = block_sum(wf);
      for (unsigned i0 = 0; i0 < n; i0 += 32) {
        // 32 candidates at a time, their weights computed by this warp's lanes
        const u64 other = i0 + lane < n ? sh.p.all[i0 + lane] : 0;
        const u64 ow = other ? fixed(weight(key_float((uint32_t)(other >> 32)), m, c)) : 0;
#pragma unroll 4
        for (int i = 0; i < 32; ++i) {
          const u64 oc = __shfl_sync(0xffffffffu, other, i), w = __shfl_sync(0xffffffffu, ow, i);
          if (oc > mine) before += w;
        }
      }
      const double zx = (double)(above + cands);
      const double reach_lo = top_p * (zx + (tl - te) * kWeightOne * (1.0 - 1e-9) - V);
      const double reach_hi = top_p * (zx + (tl + te) * kWeightOne * (1.0 + 1e-9) + V);
      const double reach = top_p * (zx + tl * kWeightOne);
      const bool first = before == 0 && mine >> 32 == kmax;  // the most likely token stays
      bool keep = have && (first || (double)before < reach);
      if (!exact_tail) {
        const bool unsure = have && ((double)before < reach_lo) != ((double)before < reach_hi);
        if (__syncthreads_or(unsure)) {
          exact_tail = true;
          all_sync();  // the lists and sums have been read by every CTA
          continue;
        }
      }
      // threshold: the last kept candidate, or just above the first of them
      u64 lowest = keep ? mine : ~0ull, highest = mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, o));
        highest = max(highest, __shfl_xor_sync(0xffffffffu, highest, o));
      }
      __syncthreads();
      if (lane == 0) sh.scratch[warp] = lowest;
      __syncthreads();
      for (int w = 0; w < NW; ++w) lowest = min(lowest, sh.scratch[w]);
      __syncthreads();
      if (lane == 0) sh.scratch[warp] = highest;
      __syncthreads();
      for (int w = 0; w < NW; ++w) highest = max(highest, sh.scratch[w]);
      thr = lowest != ~0ull ? lowest : highest + 1;
      // the kept candidates join the masses of their CTAs and of this CTA's warps
      const bool counts = keep && wd >= min_p;
      const int src = have ? sh.p.from[tid] : -1;
#pragma unroll
      for (int r = 0; r < CS; ++r) keep_of[r] += block_sum(counts && src == r ? wf : 0);
      if (counts && src == rank) {
        const int t = (int)(0xffffffffu - (uint32_t)mine);
        atomicAdd(&sh.w_keep[((t - base) / VEC) / per_warp], wf);
      }
      __syncthreads();
      resolved = true;
      break;
    }
    if (resolved) {
      draw(keep_of,
           [&](float v, int t) -> u64 {
             if (composite(v, t) < thr) return 0;
             const double w = weight(v, m, c);
             return w >= min_p ? fixed(w) : 0;
           },
           0);
      return;
    }
    all_sync();
  }

  // -----------------------------------------------------------------------
  // general: the border key by radix selection, 8 bits a pass, on exact counts
  // (top-k) and masses (top-p); then the place of the last kept token among
  // those of the border key
  // -----------------------------------------------------------------------
  // largest K with sum over keys >= K reaching `target` (of counts, or of masses
  // while the running value is below it); *above = the sum over keys > K
  auto select = [&](bool by_mass, double target, u64* above) -> uint32_t {
    uint32_t prefix = 0;
    u64 run = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += NT) sh.r.mass[i] = 0;
      __syncthreads();
      each([&](float v, int, bool in) {
        const uint32_t k = float_key(v + 0.f);
        const bool take = in && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
        const unsigned act = __ballot_sync(0xffffffffu, take);
        if (!act) return;
        u64 w = 0;
        if (take) w = by_mass ? fixed(weight(v, m, c)) : 1;
        const int b = (k >> shift) & 255, lead = __shfl_sync(0xffffffffu, b, __ffs(act) - 1);
        if (__all_sync(0xffffffffu, !take || b == lead)) {  // one bin: one addition
          w = warp_sum64(w);
          if (lane == 0) atomicAdd(&sh.r.mass[lead], w);
        } else if (take) {
          atomicAdd(&sh.r.mass[b], w);
        }
      });
      all_sync();
      // bins from the top: thread t holds bin 255 - t
      u64 h = 0, total;
      if (tid < 256)
        for (int r = 0; r < CS; ++r) h += peer(r)->r.mass[255 - tid];
      const u64 incl = block_scan(h, &total);
      // bins passed before the target is reached
      const bool passed = tid < 256 && (double)(run + incl) < target;
      const unsigned np = min((unsigned)block_sum(passed), 255u);
      __syncthreads();
      if (tid == np) sh.scratch[0] = run + incl - h;
      __syncthreads();
      run = sh.scratch[0];
      prefix |= (255u - np) << shift;
      all_sync();  // the histograms have been read
    }
    *above = run;
    return prefix;
  };
  uint32_t K = 0;
  u64 ties = ~0ull, above = 0, zk;
  if (top_k < V) {
    K = select(false, (double)top_k, &above);
    ties = (u64)top_k - above;
  }
  {  // mass of the top-k set
    u64 acc = 0;
    packed([&](float v, int) { return float_key(v + 0.f) > K; }, [&](float v) { acc += fixed(weight(v, m, c)); });
    acc = block_sum(acc);
    if (tid == 0) sh.cta_all = acc;
    all_sync();
    zk = 0;
#pragma unroll
    for (int r = 0; r < CS; ++r) zk += peer(r)->cta_all;
    if (top_k < V) zk += ties * fixed(weight(key_float(K), m, c));
  }
  if (top_p < 1.0) {
    const double reach = top_p * (double)zk;
    uint32_t kp = select(true, reach, &above);
    if (kp > kmax || reach <= 0.0) kp = kmax, above = 0;
    if (kp > K) {
      K = kp;
      ties = ~0ull;
    } else if (top_k < V) {  // the border lies among the ties of the top-k border
      above = zk - ties * fixed(weight(key_float(K), m, c));
    }
    // of the ties those stay that have less than the reach before them
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
        unsigned n = 0, eq = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int t = base + ch * VEC + j;
          const bool is = ch < wend && (unsigned)t < (unsigned)V && float_key(to_f(seg[(int64_t)ch * VEC + j]) + 0.f) == K;
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

template <typename T, int CS>
static int launch_sample(const SampleArgs<T>& a, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int per_cta = ((VEC - 1 + a.vocab + VEC - 1) / VEC + CS - 1) / CS;
  const int smem = max(per_cta * 16, kList * 8);
  auto* kern = sample_kernel<T, CS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
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

// CTAs per row: as many as keep a part at 56 KB (three CTAs per SM), then more
// while the rows alone do not fill the GPU and a thread still has eight tokens.
template <typename T>
static int sample_cluster(int64_t rows, int vocab) {
  int cs = 1;
  while (cs < 8 && (int64_t)vocab * (int)sizeof(T) > cs * 57344ll) cs *= 2;
  while (cs < 8 && rows * cs < 148 * 2 && vocab / cs > kSampleThreads * 8) cs *= 2;
  return cs;
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
    switch (sample_cluster<ET>(rows, vocab)) {
      case 1: return launch_sample<ET, 1>(a, s);
      case 2: return launch_sample<ET, 2>(a, s);
      case 4: return launch_sample<ET, 4>(a, s);
      default: return launch_sample<ET, 8>(a, s);
    }
  }());
}
