// Paged key/value cache: addressing shared by the append and attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "mma.cuh"

namespace walsh {

// n / d for 0 <= n < 2^31 as one 64-bit multiply: with s = floor(log2 d) and
// m = floor(2^(32+s) / d) + 1, the excess m d - 2^(32+s) is at most d, so the
// quotient is exact while n d < 2^(32+s), which n < 2^31 and d < 2^(s+1) give.
struct FastDiv {
  uint32_t d, sh;
  uint64_t m;
};
static inline FastDiv make_fastdiv(uint32_t d) {
  FastDiv f;
  f.d = d;
  uint32_t s = 0;
  while ((2ull << s) <= d) ++s;
  f.sh = 32 + s;
  f.m = (1ull << f.sh) / d + 1;
  return f;
}
__device__ __forceinline__ uint32_t fdiv(uint32_t n, const FastDiv& f) { return (uint32_t)(((uint64_t)n * f.m) >> f.sh); }

// float -> storage type, round to nearest; unlike from_f, fp16 keeps infinities and NaN
template <typename T> __device__ __forceinline__ T round_f(float v);
template <> __device__ __forceinline__ float round_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 round_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half round_f<__half>(float v) { return __float2half_rn(v); }

// One layer's pages as the kernels see them.
template <typename T>
struct Pages {
  const T* k;
  const T* v;
  int64_t page_stride, head_stride, row_stride;  // elements
  const int* table;
  int64_t table_stride;
  int table_cols, n_pages;
  FastDiv ps;  // page size
  const int* lens;
  int window, sinks;
  int* err;
};

// Length of sequence b: a length outside [0, table_cols * page size] is
// reported and clamped, so no later index leaves the table.
template <typename T>
__device__ __forceinline__ int seq_len(const Pages<T>& p, int b) {
  const int64_t cap = (int64_t)p.table_cols * p.ps.d;
  const int n = p.lens[b];
  if (n < 0 || n > cap) {
    if (p.err) atomicExch(p.err, (int)WALSH_ERR_INDEX);
    return n < 0 ? 0 : (int)cap;
  }
  return n;
}

// Element offset of key `key` (< seq_len) of the head at head_off, or -1 (and
// a report) when its page id is outside the pool.
template <typename T>
__device__ __forceinline__ int64_t key_offset(const Pages<T>& p, const int* trow, int key) {
  const uint32_t pi = fdiv((uint32_t)key, p.ps);
  const int id = __ldg(trow + pi);
  if ((uint32_t)id >= (uint32_t)p.n_pages) {
    if (p.err) atomicExch(p.err, (int)WALSH_ERR_INDEX);
    return -1;
  }
  return (int64_t)id * p.page_stride + (int64_t)(key - (int)(pi * p.ps.d)) * p.row_stride;
}

// The keys a query at position pos sees, numbered from 0: first the sinks
// that lie before the window, then the window itself.
struct Visible {
  int n, nsink, lo;  // key of number i: i < nsink ? i : lo + i - nsink
  __device__ __forceinline__ int key(int i) const { return i < nsink ? i : lo + (i - nsink); }
};
__device__ __forceinline__ Visible visible_keys(int pos, int window, int sinks) {
  Visible v;
  v.lo = window > 0 ? max(0, pos + 1 - window) : 0;
  v.nsink = min(sinks, v.lo);
  v.n = v.nsink + (pos + 1 - v.lo);
  return v;
}

// One query row (qp, of the group of kv head hk) over the n keys from number beg
// on, by one warp in float32: running maximum m (of the scores times log2 e), sum l
// and the lane's channels i * 32 + lane of o, undivided.
template <typename T, int HD>
__device__ __forceinline__ void attend_row(const Pages<T>& p, int b, int hk, const T* qp, const Visible& vis, int beg,
                                           int n, float scale_log2, float* m_out, float* l_out, float* acc) {
  constexpr int DL = (HD + 31) / 32;  // channels per lane
  const int lane = threadIdx.x & 31;
  const int* trow = p.table + (int64_t)b * p.table_stride;
  const T* kb = p.k + (int64_t)hk * p.head_stride;
  const T* vb = p.v + (int64_t)hk * p.head_stride;
  float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int i = 0; i < DL; ++i) acc[i] = 0.f;
  for (int x0 = 0; x0 < n; x0 += 32) {
    int64_t off = -1;
    float s = -CUDART_INF_F;
    if (x0 + lane < n) off = key_offset(p, trow, vis.key(beg + x0 + lane));
    if (off >= 0) {
      float dot = 0.f;
      for (int d = 0; d < HD; ++d) dot = fmaf(to_f(qp[d]), to_f(kb[off + d]), dot);
      s = dot * scale_log2;
    }
    const float mn = fmaxf(m, warp_max(s)), sub = mn == -CUDART_INF_F ? 0.f : mn;
    const float corr = ex2_f32(m - sub), w = off >= 0 ? ex2_f32(s - sub) : 0.f;
    m = mn;
    l = l * corr + warp_sum(w);
#pragma unroll
    for (int i = 0; i < DL; ++i) acc[i] *= corr;
    unsigned todo = __ballot_sync(0xffffffffu, off >= 0);
    while (todo) {
      const int j = __ffs(todo) - 1;
      todo &= todo - 1;
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int64_t oj = __shfl_sync(0xffffffffu, off, j);
#pragma unroll
      for (int i = 0; i < DL; ++i)
        if (i * 32 + lane < HD) acc[i] = fmaf(wj, to_f(vb[oj + i * 32 + lane]), acc[i]);
    }
  }
  *m_out = m, *l_out = l;
}

// Host: fills Pages<T> from the C description.
template <typename T>
static inline Pages<T> make_pages(const walsh_paged_kv* kv) {
  Pages<T> p;
  p.k = (const T*)kv->k_pages;
  p.v = (const T*)kv->v_pages;
  p.page_stride = kv->page_stride;
  p.head_stride = kv->head_stride;
  p.row_stride = kv->row_stride;
  p.table = kv->page_table;
  p.table_stride = kv->table_stride;
  p.table_cols = kv->table_cols;
  p.n_pages = kv->n_pages;
  p.ps = make_fastdiv((uint32_t)kv->page_size);
  p.lens = kv->kv_lens;
  p.window = kv->window;
  p.sinks = kv->sinks;
  p.err = kv->err;
  return p;
}

// Host: checks of the description that every paged entry point makes.
static inline int check_pages(const walsh_paged_kv* kv, bool table) {
  WALSH_CHECK_ARG(kv && kv->k_pages && kv->v_pages);
  WALSH_CHECK_DTYPE(kv->dtype);
  const int hd = kv->head_dim;
  if (hd != 16 && hd != 32 && hd != 64 && hd != 128) return WALSH_ERR_SHAPE;
  WALSH_CHECK_SHAPE(kv->n_pages > 0 && kv->kv_heads > 0 && kv->kv_heads <= 65535 && kv->page_size > 0 &&
                    (int64_t)kv->n_pages * kv->page_size < (1ll << 40) && kv->page_size < (1 << 30));
  WALSH_CHECK_SHAPE(kv->page_stride >= 0 && kv->head_stride >= 0 && kv->row_stride >= hd);
  const int64_t vec = kv->dtype == WALSH_F32 ? 4 : 8;
  if (((((uintptr_t)kv->k_pages) | ((uintptr_t)kv->v_pages)) & 15u) != 0 || kv->page_stride % vec ||
      kv->head_stride % vec || kv->row_stride % vec)
    return WALSH_ERR_ALIGN;
  if (table) {
    WALSH_CHECK_ARG(kv->page_table && kv->kv_lens && kv->window >= 0 && kv->sinks >= 0 && kv->scale > 0.f && kv->scale < 3.0e38f);
    WALSH_CHECK_SHAPE(kv->table_cols > 0 && kv->table_stride >= 0 &&
                      (int64_t)kv->table_cols * kv->page_size < (1ll << 31));
  }
  return WALSH_OK;
}

}  // namespace walsh
