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
// (float32), joined through shared memory.  A few ranges are joined by a cluster
// of their CTAs; more leave (m, l, o) in the workspace for paged_join_kernel.
// Both combine them in order of the ranges, so results do not depend on timing.
// Measured (of the HBM copy rate): 256 sequences of up to 1024 keys, 32 heads of
// 16 channels, 50.8 us (0.82); 12 of up to 32768, 8 shared heads of 64, 81 us
// (0.91); 48 under a window of 1000, 64 heads of 32, 61.4 us (0.90).
#include <cooperative_groups.h>
#include <math_constants.h>

#include "mma.cuh"
#include "paged.cuh"

namespace walsh {

namespace cg = cooperative_groups;

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

// The ranges of one unit joined through distributed shared memory: the CTAs of a
// cluster hold their range's (m, l, o) in cj [rows][HD + 2] and each combines a
// share of the outputs, in order of the ranges.
template <typename T, int HD>
__device__ __forceinline__ void cluster_join(const DecodeArgs<T>& a, float* cj, int c, int ng, int64_t row0) {
  const cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  for (int i = c * blockDim.x + threadIdx.x; i < ng * HD; i += a.nsplit * blockDim.x) {
    const int r = i / HD, d = i - r * HD;
    float M = -CUDART_INF_F, L = 0.f, O = 0.f;
    for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, cl.map_shared_rank(cj, s)[r * (HD + 2) + HD]);
    const float sub = M == -CUDART_INF_F ? 0.f : M;
    for (int s = 0; s < a.nsplit; ++s) {
      const float* q = cl.map_shared_rank(cj, s) + r * (HD + 2);
      const float f = ex2_f32(q[HD] - sub);
      L = fmaf(q[HD + 1], f, L);
      O = fmaf(q[d], f, O);
    }
    a.o[(row0 + r) * HD + d] = round_f<T>(L == 0.f ? 0.f : O / L);
  }
  cl.sync();  // no CTA leaves while its memory is read
}

// ---------------------------------------------------------------------------
// CUDA-core form for float32.  LPK lanes share one key, 16 bytes of it each; a
// warp step covers 32 / LPK keys and KPT steps are in flight.
// ---------------------------------------------------------------------------
template <typename T, int HD, int GH, int W, bool CL>
__global__ void __launch_bounds__(W * 32) paged_decode_vec_kernel(const DecodeArgs<T> a) {
  constexpr int VEC = 16 / (int)sizeof(T), LPK = HD / VEC, KS = 32 / LPK, KPT = 4;
  __shared__ float red[W][GH][LPK][VEC + 2];
  __shared__ float cj[CL ? GH * (HD + 2) : 1];
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
  if (!CL && beg >= end && c > 0) return;
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
  const int64_t row0 = (int64_t)b * Hq + h0;
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
    if constexpr (CL) {
      cj[(row - row0) * (HD + 2) + d] = O;
      if (d == 0) {
        cj[(row - row0) * (HD + 2) + HD] = M;
        cj[(row - row0) * (HD + 2) + HD + 1] = L;
      }
    } else if (whole) {
      a.o[row * HD + d] = round_f<T>(L == 0.f ? 0.f : O / L);  // no visible key: zeros
    } else {
      a.part_o[(row * a.nsplit + c) * HD + d] = O;
      if (d == 0) {
        a.part_ml[(row * a.nsplit + c) * 2] = M;
        a.part_ml[(row * a.nsplit + c) * 2 + 1] = L;
      }
    }
  }
  if constexpr (CL) cluster_join<T, HD>(a, cj, c, ng, row0);
}

// ---------------------------------------------------------------------------
// Tensor-core form for 16-bit types.  A CTA of W warps takes one range of one
// (sequence, key/value head); each warp streams its slice through its own ring
// of NS stages of KT keys (16-byte asynchronous copies; no CTA barrier until
// the join), page lookups made a stage ahead, one key row per lane.  The heads
// of the group are the rows of the MMAs: S = Q K^T and O += P V (m16n8k16).
// P enters as two 16-bit terms, rounded and what that left over, so it keeps 16
// (bf16) to 22 bits: with up to 8 heads the rows 8 - 15 carry the second term at
// no cost, with 9 to 16 heads it takes MMAs of its own (64 x 4000 keys,
// 64 heads on 4 of 64 channels 54 -> 56 us, 64 on 4 of 16 17 -> 19.5, 32 on 2 of 128
// 60 -> 64.5).  Rows that come out as NaN are computed again.
// ---------------------------------------------------------------------------
template <int HD>
__device__ __forceinline__ int dec_swz(int r, int c) {  // 16-byte piece c of row r: its place in the row
  if constexpr (HD == 16) return c ^ ((r >> 2) & 1);
  else if constexpr (HD == 32) return c ^ ((r >> 1) & 3);
  else return c ^ (r & 7);
}
template <typename T> __device__ __forceinline__ uint32_t dec_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t dec_pack<__half>(float lo, float hi) { return pack_f16(lo, hi); }
template <> __device__ __forceinline__ uint32_t dec_pack<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }

// One row of a warp's slice again in float32, over the n keys from number beg on:
// a probability that is nothing in 16 bits makes NaN of an infinite value, which
// float32 keeps infinite.  (m, l, o) go where the warps are joined.  (The kernel's
// arguments are a __grid_constant__: passed on by reference they would be copied to
// local memory, 256 x 1024 keys 56.5 us against 50.7.)
template <typename T, int HD>
__device__ __noinline__ void decode_row_again(const DecodeArgs<T>& a, const Visible vis, int b, int hk, int h, int beg,
                                              int n, float* jo, float* jm) {
  constexpr int DL = (HD + 31) / 32;
  const int lane = threadIdx.x & 31;
  float m, l, acc[DL];
  attend_row<T, HD>(a.pg, b, hk, a.q + (int64_t)b * a.q_bs + (int64_t)h * a.q_hs, vis, beg, n, a.scale_log2, &m, &l, acc);
#pragma unroll
  for (int i = 0; i < DL; ++i)
    if (i * 32 + lane < HD) jo[i * 32 + lane] = acc[i];
  if (lane == 0) jm[0] = m, jm[1] = l;
}

// RH: halves of the 16 MMA rows in use (1: up to 8 heads, 2: up to 16)
template <typename T, int HD, int RH, int W, int KT, int NS, bool CL>
__global__ void __launch_bounds__(W * 32) paged_decode_mma_kernel(const __grid_constant__ DecodeArgs<T> a) {
  constexpr int CH = HD / 8, STAGE = 2 * KT * HD, RI = 32 / CH;  // RI: rows per copy instruction
  constexpr int OL = HD + 4;                                     // padded row of the join buffer
  extern __shared__ __align__(16) unsigned char smb[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
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
  if (!CL && beg >= end && c > 0) return;
  const int ng = min(8 * RH, a.group - gt * 8 * RH), h0 = hk * a.group + gt * 8 * RH;
  const int per = ((end - beg + W - 1) / W + 15) / 16 * 16;
  const int wbeg = min(end, beg + warp * per), n = min(end, wbeg + per) - wbeg;  // this warp's keys
  const int nst = (n + KT - 1) / KT;
  T* ring = reinterpret_cast<T*>(smb) + warp * (NS * STAGE);  // a warp's own
  const int* trow = a.pg.table + (int64_t)b * a.pg.table_stride;
  const T* kb = a.pg.k + (int64_t)hk * a.pg.head_stride + (lane % CH) * 8;
  const T* vb = a.pg.v + (int64_t)hk * a.pg.head_stride + (lane % CH) * 8;

  constexpr int RL = (KT + 31) / 32;  // rows looked up per lane
  int64_t off[RL];
  auto lookup = [&](int st) {
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int x = st * KT + i * 32 + lane;
      off[i] = -1;
      if ((KT >= 32 || lane < KT) && x < n) off[i] = key_offset(a.pg, trow, vis.key(wbeg + x));
    }
  };
  // bit r: row r of the stage holds a key
  uint32_t okq[NS][RL];
  auto load = [&](int buf) {
    T* dst = ring + buf * STAGE;
#pragma unroll
    for (int i = 0; i < KT / RI; ++i) {
      const int r = i * RI + lane / CH, ch = lane % CH;
      const int64_t o = __shfl_sync(0xffffffffu, off[(i * RI) / 32], r % 32);
      const int at = r * HD + dec_swz<HD>(r, ch) * 8;
      cp_async16(dst + at, kb + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
      cp_async16(dst + KT * HD + at, vb + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
    }
  };
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int j = 0; j < RL; ++j) okq[i][j] = 0;
  if (n > 0) {
    lookup(0);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      if (s < nst) load(s);
#pragma unroll
      for (int j = 0; j < RL; ++j) okq[s][j] = __ballot_sync(0xffffffffu, s < nst && off[j] >= 0);
      cp_async_commit();
      lookup(s + 1);
    }
  }
  // Q fragments; rows past the tile's heads are zero
  uint32_t qf[HD / 16][4];
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = g + (j & 1) * 8;
      qf[ks][j] = 0u;
      if (r < ng)
        qf[ks][j] = __ldg(reinterpret_cast<const uint32_t*>(a.q + (int64_t)b * a.q_bs + (int64_t)(h0 + r) * a.q_hs) +
                          ks * 8 + t4 + (j >> 1) * 4);
    }
  float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f}, acc[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  const float sc = a.scale_log2;
  auto compute = [&](const T* kt_s, const uint32_t* ok) {
    const T* vt_s = kt_s + KT * HD;
    float s[KT / 8][4];
#pragma unroll
    for (int i = 0; i < KT / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int np = 0; np < KT / 16; ++np) {
        uint32_t kf[4];
        const int r = np * 16 + (lane & 7) + ((lane >> 4) << 3), ch = ks * 2 + ((lane >> 3) & 1);
        ldsm_x4(kf, kt_s + r * HD + dec_swz<HD>(r, ch) * 8);
        mma16<T>(s[2 * np], qf[ks], kf[0], kf[1]);
        mma16<T>(s[2 * np + 1], qf[ks], kf[2], kf[3]);
      }
    bool full = true;
#pragma unroll
    for (int j = 0; j < RL; ++j) full &= ok[j] == (KT >= 32 ? 0xffffffffu : (1u << (KT & 31)) - 1u);
    if (!full) {
#pragma unroll
      for (int i = 0; i < KT / 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (!((ok[i >> 2] >> ((i & 3) * 8 + 2 * t4 + e)) & 1u)) s[i][e] = s[i][2 + e] = -CUDART_INF_F;
    }
    uint32_t pf[KT / 16][4], pl[RH == 2 ? KT / 16 : 1][4];
#pragma unroll
    for (int h = 0; h < RH; ++h) {
      float mt = -CUDART_INF_F;
#pragma unroll
      for (int i = 0; i < KT / 8; ++i) mt = fmax3(mt, s[i][2 * h], s[i][2 * h + 1]);
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float mn = fmaxf(m[h], mt), sub = mn == -CUDART_INF_F ? 0.f : mn * sc;
      const float corr = ex2_f32(m[h] * sc - sub);
      m[h] = mn;
      float rs = 0.f;
#pragma unroll
      for (int i = 0; i < KT / 8; ++i) {
        const float p0 = ex2_f32(fmaf(s[i][2 * h], sc, -sub)), p1 = ex2_f32(fmaf(s[i][2 * h + 1], sc, -sub));
        rs += p0 + p1;
        const uint32_t hi = dec_pack<T>(p0, p1);
        pf[i >> 1][(i & 1) * 2 + h] = hi;
        const float2 hf = unpack2<T>(hi);
        const uint32_t rest = dec_pack<T>(p0 - hf.x, p1 - hf.y);
        if constexpr (RH == 1) pf[i >> 1][(i & 1) * 2 + 1] = rest;
        else pl[i >> 1][(i & 1) * 2 + h] = rest;
      }
      l[h] = l[h] * corr + rs;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        acc[i][2 * h] *= corr, acc[i][2 * h + 1] *= corr;
        if constexpr (RH == 1) acc[i][2] *= corr, acc[i][3] *= corr;
      }
    }
#pragma unroll
    for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
      for (int dp = 0; dp < HD / 16; ++dp) {
        uint32_t vf[4];
        const int r = kk * 16 + (lane & 15), ch = dp * 2 + (lane >> 4);
        ldsm_x4_t(vf, vt_s + r * HD + dec_swz<HD>(r, ch) * 8);
        mma16<T>(acc[2 * dp], pf[kk], vf[0], vf[1]);
        mma16<T>(acc[2 * dp + 1], pf[kk], vf[2], vf[3]);
        if constexpr (RH == 2) {
          mma16<T>(acc[2 * dp], pl[kk], vf[0], vf[1]);
          mma16<T>(acc[2 * dp + 1], pl[kk], vf[2], vf[3]);
        }
      }
  };
  for (int st0 = 0; st0 < nst; st0 += NS) {
#pragma unroll
    for (int u = 0; u < NS; ++u) {  // stage st0 + u lies in buffer u
      const int st = st0 + u;
      if (st >= nst) break;
      // the buffer that the stage before this one left takes stage st + NS - 1
      constexpr int NB = NS - 1;
      const int nb = (u + NB) % NS;
      if (st + NB < nst) load(nb);
#pragma unroll
      for (int j = 0; j < RL; ++j) okq[nb][j] = __ballot_sync(0xffffffffu, st + NB < nst && off[j] >= 0);
      cp_async_commit();
      lookup(st + NS);
      cp_async_wait<NS - 1>();
      __syncwarp();
      compute(ring + u * STAGE, okq[u]);
      __syncwarp();
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < RH; ++h)
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
  if constexpr (RH == 1) {  // the leftovers' part (an infinite sum is complete without it)
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (fabsf(acc[i][e]) < CUDART_INF_F) acc[i][e] += acc[i][2 + e];
  }
  // join the warps: rows of the ring are free
  float* jo = reinterpret_cast<float*>(smb);             // [W][8 RH][OL]
  float* jm = jo + W * 8 * RH * OL;                      // [W][8 RH][2]
  float* cj = jm + W * 8 * RH * 2;                       // [8 RH][HD + 2], cluster join
  if constexpr (W > 1) __syncthreads();
#pragma unroll
  for (int h = 0; h < RH; ++h) {
    const int r = g + 8 * h;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
      nan |= r < ng && (acc[i][2 * h] != acc[i][2 * h] || acc[i][2 * h + 1] != acc[i][2 * h + 1]);
    unsigned again = __ballot_sync(0xffffffffu, nan);
    if (r < ng && !(again & (15u << (lane & 28)))) {
      float* row = jo + (warp * 8 * RH + r) * OL;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<float2*>(row + i * 8 + 2 * t4) = make_float2(acc[i][2 * h], acc[i][2 * h + 1]);
      if (t4 == 0) {
        jm[(warp * 8 * RH + r) * 2] = m[h] * sc;
        jm[(warp * 8 * RH + r) * 2 + 1] = l[h];
      }
    }
    while (again) {
      const int q = (__ffs(again) - 1) >> 2, at = warp * 8 * RH + q + 8 * h;  // the lane quad of a row
      again &= ~(15u << (4 * q));
      decode_row_again<T, HD>(a, vis, b, hk, h0 + q + 8 * h, wbeg, n, jo + at * OL, jm + at * 2);
    }
  }
  if constexpr (W > 1) __syncthreads();
  else __syncwarp();
  const int64_t Hq = (int64_t)a.kv_heads * a.group;
  const int64_t row0 = (int64_t)b * Hq + h0;
  const bool whole = vis.n <= a.chunk || a.nsplit == 1;  // this range is all there is
  for (int i = threadIdx.x; i < ng * HD; i += W * 32) {
    const int r = i / HD, d = i - r * HD;
    float M = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, jm[(w * 8 * RH + r) * 2]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = jm[(w * 8 * RH + r) * 2];
      const float f = mw == -CUDART_INF_F ? 0.f : ex2_f32(mw - M);
      L = fmaf(jm[(w * 8 * RH + r) * 2 + 1], f, L);
      O = fmaf(jo[(w * 8 * RH + r) * OL + d], f, O);
    }
    const int64_t row = (int64_t)b * Hq + h0 + r;
    if constexpr (CL) {
      cj[(row - row0) * (HD + 2) + d] = O;
      if (d == 0) {
        cj[(row - row0) * (HD + 2) + HD] = M;
        cj[(row - row0) * (HD + 2) + HD + 1] = L;
      }
    } else if (whole) {
      a.o[row * HD + d] = round_f<T>(L == 0.f ? 0.f : O / L);  // no visible key: zeros
    } else {
      a.part_o[(row * a.nsplit + c) * HD + d] = O;
      if (d == 0) {
        a.part_ml[(row * a.nsplit + c) * 2] = M;
        a.part_ml[(row * a.nsplit + c) * 2 + 1] = L;
      }
    }
  }
  if constexpr (CL) cluster_join<T, HD>(a, cj, c, ng, row0);
}

// Joins the ranges of each (sequence, head): one CTA per row, its warps take
// every fourth group of ranges with four loads in flight.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const DecodeArgs<T> a) {
  constexpr int DP = HD < 32 ? HD : 32, DN = HD / DP, SL = 32 / DP;  // channels and ranges per step of a warp
  __shared__ float red[4][HD + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x, Hq = (int64_t)a.kv_heads * a.group;
  const Visible vis = visible_keys(seq_len(a.pg, (int)(row / Hq)) - 1, a.pg.window, a.pg.sinks);
  if (vis.n <= a.chunk) return;  // written whole
  const int nc = (int)min((int64_t)a.nsplit, ((int64_t)vis.n + a.chunk - 1) / a.chunk);
  const float* ml = a.part_ml + row * a.nsplit * 2;
  const float* po = a.part_o + row * a.nsplit * HD;
  float M = -CUDART_INF_F;
  for (int i = lane; i < nc; i += 32) M = fmaxf(M, ml[2 * i]);
  M = warp_max(M);
  const float sub_m = M == -CUDART_INF_F ? 0.f : M;
  const int d0 = lane % DP, s0 = lane / DP;
  float L = 0.f, O[DN] = {};
#pragma unroll 4
  for (int i = warp * SL + s0; i < nc; i += 4 * SL) {
    const float f = ex2_f32(ml[2 * i] - sub_m);
    L = fmaf(ml[2 * i + 1], f, L);
#pragma unroll
    for (int k = 0; k < DN; ++k) O[k] = fmaf(po[(int64_t)i * HD + k * DP + d0], f, O[k]);
  }
#pragma unroll
  for (int o = DP; o < 32; o <<= 1) {
    L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
    for (int k = 0; k < DN; ++k) O[k] += __shfl_xor_sync(0xffffffffu, O[k], o);
  }
  if (lane < DP) {
#pragma unroll
    for (int k = 0; k < DN; ++k) red[warp][k * DP + d0] = O[k];
    if (lane == 0) red[warp][HD] = L;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += 128) {
    const float l = red[0][HD] + red[1][HD] + red[2][HD] + red[3][HD];
    const float o = red[0][d] + red[1][d] + red[2][d] + red[3][d];
    a.o[row * HD + d] = round_f<T>(l == 0.f ? 0.f : o / l);
  }
}

// Launches CTAs, in clusters of `cluster` when that is more than one.
template <typename K, typename A>
static int launch_ctas(K* kern, const A& a, int64_t ctas, int threads, int smem, int cluster, cudaStream_t s) {
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status();
  if (cluster <= 1) {
    kern<<<(unsigned)ctas, threads, smem, s>>>(a);
    return launch_status();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, a);
  return launch_status();
}

template <typename T, int HD, int RH, int W, bool CL>
static int launch_decode_mma(const DecodeArgs<T>& a, int64_t ctas, cudaStream_t s) {
  // 8 KB of K and V per stage (4 KB for 16 channels)
  constexpr int KT = HD <= 32 ? 64 : HD == 64 ? 32 : 16;
  // two stages in flight and the warps' number cover the latency; the smaller
  // ring leaves room for more warps (256 x up to 1024 keys, 16 channels: 2 stages
  // 50.7 us, 3 51.8, 4 61.7; 12 x up to 32768, 64 channels: 81.2, 84.1, 112)
  constexpr int NS = 2;
  constexpr int ring = W * NS * 2 * KT * HD * 2, join = (W * 8 * RH * (HD + 4 + 2) + (CL ? 8 * RH * (HD + 2) : 0)) * 4;
  return launch_ctas(paged_decode_mma_kernel<T, HD, RH, W, KT, NS, CL>, a, ctas, W * 32, ring > join ? ring : join,
                     CL ? a.nsplit : 1, s);
}

template <typename T, int HD, int W, bool CL>
static int launch_decode(const DecodeArgs<T>& a, cudaStream_t s) {
  const int64_t ctas = (int64_t)a.B * a.kv_heads * a.gtiles * a.nsplit;
  int r;
  if constexpr (sizeof(T) == 2) {
    r = a.group <= 8 ? launch_decode_mma<T, HD, 1, W, CL>(a, ctas, s) : launch_decode_mma<T, HD, 2, W, CL>(a, ctas, s);
  } else {
    const int cl = CL ? a.nsplit : 1;
    r = a.group == 1 ? launch_ctas(paged_decode_vec_kernel<T, HD, 1, W, CL>, a, ctas, W * 32, 0, cl, s)
                     : launch_ctas(paged_decode_vec_kernel<T, HD, 4, W, CL>, a, ctas, W * 32, 0, cl, s);
  }
  if (r || CL) return r;
  if (a.nsplit > 1) {
    const int64_t rows = (int64_t)a.B * a.kv_heads * a.group;
    paged_join_kernel<T, HD><<<(unsigned)rows, 128, 0, s>>>(a);
    return launch_status();
  }
  return WALSH_OK;
}

// How a call is cut: `warps` per CTA, `nsplit` ranges of `chunk` visible keys per
// unit (sequence, key/value head, head tile), by the bytes of its longest.
struct DecodePlan {
  int warps, gtiles, nsplit, chunk;
  bool cluster;  // the ranges' CTAs join through distributed shared memory
};
constexpr int64_t kRangeBytes = 256 << 10;  // longer ranges are cut for the balance between sequences
constexpr int64_t kRangeLeast = 32 << 10;   // shorter ones cost more to join than they save
// from so many units up to so many bytes each, a warp per unit.  32 heads of 16,
// lengths up to the one named: 256 x 1024 keys (8192 units of 64 KB) 50.6 us against
// 58.2 with four, 100 x 200 8.8 against 13.9, 100 x 600 17.6 against 20.5; about
// even at 100 x 1200 (77 KB) 28.8 and 29.1, 100 x 1500 (96 KB) 33.6 and 32.8, 64 x
// 1024 (2048 units) 21.0 and 19.3, 62 x 1024 19.9 and 18.7; all of one length they
// pass earlier, 100 x 1200 50.5 and 44.2, 100 x 2000 79 and 65
constexpr int kSingleUnits = 2000;
constexpr int64_t kSingleBytes = 100000;
static DecodePlan decode_plan(const walsh_paged_kv* kv, int B, int q_heads, int max_len) {
  const int group = q_heads / kv->kv_heads, tile = kv->dtype == WALSH_F32 ? 4 : group <= 8 ? 8 : 16;
  DecodePlan p;
  p.gtiles = group == 1 ? 1 : (group + tile - 1) / tile;
  const int64_t units = (int64_t)B * kv->kv_heads * p.gtiles;
  int64_t n = max_len;
  if (kv->window > 0) n = min64(n, (int64_t)kv->window + kv->sinks);
  const int64_t bytes = n * 2 * kv->head_dim * (kv->dtype == WALSH_F32 ? 4 : 2);  // of a unit
  // one warp per unit when there are enough units for the GPU, or nothing to share
  p.warps = (units >= kSingleUnits && bytes <= kSingleBytes) || bytes < (8 << 10) ? 1 : 4;
  // CTAs of four warps that run together, so that no range waits for another: their
  // rings of 64 KB leave room for 3 on an SM (2 x 20000 keys, 32 on 8 heads of 64
  // channels, 3 per SM 21.1 us, 4 25.1, 5 25.0; 32 on 4 of 32, 3 11.4, 4 15.5, 5
  // 16.0; but 37 x 4000 of these 27.4 against 23.1 with 5, whose ranges are too many
  // for clusters); with 16 channels and 32 KB 4 do best (4 x 4000, 32 heads, 3 11.5,
  // 4 10.2, 5 12.7)
  const int ctas = 148 * (kv->head_dim == 16 ? 4 : 3);
  int64_t split = units > 0 ? ctas / units : 1;
  if (split < bytes / kRangeBytes) split = bytes / kRangeBytes;
  split = min64(split, bytes / kRangeLeast);
  if (units > 0) split = min64(split, ((1ll << 31) - 1) / units);  // the grid counts CTAs in 31 bits
  p.nsplit = p.warps == 1 || split < 1 ? 1 : (int)split;
  p.chunk = (int)((n + p.nsplit - 1) / p.nsplit);
  if (p.chunk < 1) p.chunk = 1;
  // the clusters' one launch saves the joining kernel and its scratch (1 x 4099 keys
  // of 32 heads of 16 8.0 -> 7.1 us, 4 x 4000 11.6 -> 10.2; but 8 x 8000, 32 on 8 of
  // 64, 31.4 -> 34.2, in clusters of 6) while all of them run at once; beyond that
  // CTAs that wait for their cluster keep others out (48 x 4000, 16 on 2 of 128: 44.9
  // us against 43.0)
  p.cluster = p.nsplit > 1 && p.nsplit <= 8 && units * p.nsplit <= 148 * 4;
  return p;
}

template <typename T, int HD>
static int launch_decode_plan(const DecodeArgs<T>& a, const DecodePlan& p, cudaStream_t s) {
  if (p.cluster) return launch_decode<T, HD, 4, true>(a, s);
  return p.warps == 1 ? launch_decode<T, HD, 1, false>(a, s) : launch_decode<T, HD, 4, false>(a, s);
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
  return p.nsplit > 1 && !p.cluster ? (int64_t)B * q_heads * p.nsplit * (kv->head_dim + 2) * 4 : 0;
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
  WALSH_CHECK_ARG(p.nsplit == 1 || p.cluster || scratch);
  return WALSH_DISPATCH_DTYPE(kv->dtype, ET, [&]() -> int {
    DecodeArgs<ET> a;
    a.pg = make_pages<ET>(kv);
    a.q = (const ET*)q, a.q_bs = q_bs, a.q_hs = q_hs, a.o = (ET*)o;
    a.part_o = (float*)scratch;
    a.part_ml = scratch ? a.part_o + (int64_t)B * q_heads * p.nsplit * kv->head_dim : nullptr;
    a.B = B, a.kv_heads = kv->kv_heads, a.group = q_heads / kv->kv_heads;
    a.gtiles = p.gtiles, a.nsplit = p.nsplit, a.chunk = p.chunk;
    a.scale_log2 = kv->scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    switch (kv->head_dim) {
      case 16: return launch_decode_plan<ET, 16>(a, p, s);
      case 32: return launch_decode_plan<ET, 32>(a, p, s);
      case 64: return launch_decode_plan<ET, 64>(a, p, s);
      default: return launch_decode_plan<ET, 128>(a, p, s);
    }
  }());
}
