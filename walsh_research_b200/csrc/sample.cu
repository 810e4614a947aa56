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
#include <math_constants.h>

#include "common.cuh"
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

// Unsigned order of floats (-0 counts as +0, NaN as -inf).
__device__ __forceinline__ float clean_logit(float v) { return v != v ? -CUDART_INF_F : v + 0.f; }
__device__ __forceinline__ uint32_t float_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// Weight of logit l as a double (exp of the 64-bit difference).
__device__ __forceinline__ double weight(float l, float m, double inv_t) {
  if (l == m) return 1.0;
  if (l == -CUDART_INF_F || m == CUDART_INF_F) return 0.0;
  return exp(((double)l - (double)m) * inv_t);
}
__device__ __forceinline__ unsigned long long fixed(double w) { return __double2ull_rn(w * kWeightOne); }

template <int NT>
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < NT / 32; ++i) v += buf[i];
  return v;
}

// One CTA per row; the threshold key is found by bisection over the 32 key bits.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_rows_kernel(const SampleArgs<T> a) {
  __shared__ unsigned long long buf[NT / 32];
  __shared__ unsigned long long wsum[NT / 32];
  __shared__ unsigned wtie[NT / 32];
  __shared__ int found;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  const T* lg = a.logits + (int64_t)r * a.ld;
  auto key_at = [&](int i) { return float_key(clean_logit(to_f(lg[i]))); };
  const double temp = a.temperature_r ? (double)a.temperature_r[r] : a.temperature;
  const double top_p = a.top_p_r ? (double)a.top_p_r[r] : a.top_p;
  const double min_p = fmin(a.min_p_r ? (double)a.min_p_r[r] : a.min_p, 1.0);
  int top_k = a.top_k_r ? a.top_k_r[r] : a.top_k;
  if (top_k <= 0 || top_k > V) top_k = V;
  if (!(temp > 0.0)) top_k = 1;  // greedy
  const double inv_t = temp > 0.0 ? 1.0 / temp : 1.0;
  uint32_t kmax = 0;
  for (int i = tid; i < V; i += NT) kmax = max(kmax, key_at(i));
  {
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) wtie[warp] = kmax;
    __syncthreads();
    for (int i = 0; i < NT / 32; ++i) kmax = max(kmax, wtie[i]);
  }
  const float m = key_float(kmax);
  if (m == -CUDART_INF_F) {  // no token to draw
    if (tid == 0) {
      a.ids[r] = -1;
      if (a.logp) a.logp[r] = CUDART_NAN_F;
    }
    return;
  }
  // count and mass of the keys >= K
  auto above = [&](uint32_t K, unsigned long long* mass) {
    unsigned long long n = 0, w = 0;
    for (int i = tid; i < V; i += NT) {
      const uint32_t k = key_at(i);
      if (k >= K) {
        ++n;
        w += fixed(weight(key_float(k), m, inv_t));
      }
    }
    *mass = block_sum<NT>(w, buf);
    return block_sum<NT>(n, buf);
  };
  // kept: key > K, and the first `ties` (index order) of those equal to K
  uint32_t K = 0;
  unsigned long long ties = V, mass;
  unsigned long long Z;
  if (top_k < V) {
    uint32_t lo = 0;  // the largest K with count(key >= K) >= top_k
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = lo | (1u << bit);
      if (above(t, &mass) >= (unsigned long long)top_k) lo = t;
    }
    K = lo;
    const unsigned long long gt = K == 0xffffffffu ? 0 : above(K + 1, &mass);
    ties = top_k - gt;
    Z = mass + ties * fixed(weight(key_float(K), m, inv_t));
  } else {
    above(0, &Z);
  }
  if (top_p < 1.0) {
    const double P = top_p * (double)Z;
    // the largest K with mass(key >= K) >= P; keys below the top-k border count as reached
    uint32_t best = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = best | (1u << bit);
      if (t > kmax) continue;
      if (t <= K) {
        best = t;
        continue;
      }
      above(t, &mass);
      if ((double)mass >= P) best = t;
    }
    const uint32_t Kp = max(best, K);
    if (Kp > K) ties = V;
    K = Kp;
    if (K < kmax) above(K + 1, &mass); else mass = 0;
    const unsigned long long w = fixed(weight(key_float(K), m, inv_t));
    unsigned long long c = w ? (unsigned long long)fmax(0.0, (P - (double)mass) / (double)w) : 0;
    while (c > 0 && (double)(mass + (c - 1) * w) >= P) --c;
    while (c < (unsigned long long)V && w && (double)(mass + c * w) < P) ++c;
    if (K == kmax && c == 0) c = 1;  // the most likely token always stays
    ties = min(ties, c);
  }
  // draw: every warp owns a run of the row; masses and tie counts before it by prefix sums
  const int run = ((V + NT / 32 - 1) / (NT / 32) + 31) / 32 * 32;
  const int i0 = min(V, warp * run), i1 = min(V, i0 + run);
  unsigned nt = 0;
  for (int i = i0 + lane; i < i1; i += 32) nt += key_at(i) == K;
  nt = __reduce_add_sync(0xffffffffu, nt);
  __syncthreads();
  if (lane == 0) wtie[warp] = nt;
  __syncthreads();
  unsigned long long tie0 = 0;
  for (int w = 0; w < warp; ++w) tie0 += wtie[w];
  // one pass over the run: its kept mass, or with `hunt` the first token whose running mass exceeds `t`
  auto pass = [&](bool hunt, unsigned long long t, unsigned long long acc) {
    unsigned long long tie = tie0;
    for (int i = i0; i < i1; i += 32) {
      const bool in = i + lane < i1;
      const uint32_t k = in ? key_at(i + lane) : 0u;
      const unsigned eq = __ballot_sync(0xffffffffu, in && k == K);
      const bool keep = in && (k > K || (k == K && tie + __popc(eq & ((1u << lane) - 1)) < ties));
      tie += __popc(eq);
      unsigned long long w = 0;
      if (keep) {
        const double x = weight(key_float(k), m, inv_t);
        if (x >= min_p) w = fixed(x);
      }
      unsigned long long s = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      if (hunt) {
        const unsigned hit = __ballot_sync(0xffffffffu, acc + s > t);
        if (hit) {
          if (lane == __ffs(hit) - 1) found = i + lane;
          return acc;
        }
      }
      acc += __shfl_sync(0xffffffffu, s, 31);
    }
    return acc;
  };
  const unsigned long long mine = pass(false, 0, 0);
  if (lane == 0) wsum[warp] = mine;
  __syncthreads();
  unsigned long long before = 0;
  Z = 0;
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += wsum[w];
    Z += wsum[w];
  }
  const double uz = (double)a.u[r] * (double)Z;
  unsigned long long t = uz > 0.0 ? (unsigned long long)uz : 0;  // u outside [0, 1) or NaN: the nearest end
  if (t > Z - 1) t = Z - 1;
  if (t >= before && t < before + mine) pass(true, t, before);
  __syncthreads();
  if (tid == 0) {
    a.ids[r] = found;
    if (a.logp) {
      const double w = temp > 0.0 ? weight(key_float(key_at(found)), m, inv_t) : 1.0;
      a.logp[r] = top_k == 1 ? 0.f : (float)log(w * kWeightOne / (double)Z);
    }
  }
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
  WALSH_CHECK_SHAPE(rows >= 0 && rows < (1ll << 31) && vocab > 0 && vocab <= kSampleMaxVocab && ld >= 0);
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
    sample_rows_kernel<ET, 1024><<<(unsigned)rows, 1024, 0, (cudaStream_t)stream>>>(a);
    return launch_status();
  }());
}
