// Append of new tokens to a paged key/value cache: per-head RMS norm of q and
// k, rotation at each token's position, and the scatter of k and v into their
// slots, in one pass.
//
//   n = x / sqrt(mean_d(x^2) + eps) * w          (when a norm weight is given)
//   (y_2i, y_2i+1) = (n_2i c - n_2i+1 s, n_2i s + n_2i+1 c),  c, s = cos, sin[pos][i]
//
// Bytes bound it: every element is read once and written once and the
// arithmetic is a few operations per element.  A thread owns one 16-byte
// piece of one head row, so a row's norm is a shuffle reduction over the
// hd * size / 16 (2 to 32) lanes that hold it and both the reads and the
// rows of q_out are whole 16-byte accesses of consecutive lanes.
#include "paged.cuh"

namespace walsh {

template <typename T>
struct AppendArgs {
  const T *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  int ntok, q_heads, kv_heads;
  FastDiv per_tok;  // rows of a token: q_heads (when q is given) + 2 kv_heads
  const void* slots;
  const void* positions;  // null: no rotation
  int idx64;              // slots and positions are int64 (else int32)
  int64_t n_slots;
  int n_pos;
  const float *cos, *sin, *q_norm, *k_norm;
  float eps;
  T *q_out, *k_pages, *v_pages;
  int64_t page_stride, head_stride, row_stride;
  FastDiv ps;
  int* err;
};

template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs<T> a) {
  constexpr int VEC = 16 / (int)sizeof(T), LPR = HD / VEC;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(i % LPR) * VEC;  // first element of this thread's piece
  const int64_t row = i / LPR;
  const bool in = row < (int64_t)a.ntok * a.per_tok.d;
  const uint32_t tok = in ? fdiv((uint32_t)row, a.per_tok) : 0u;
  int h = in ? (int)((uint32_t)row - tok * a.per_tok.d) : 0;
  // role: 0 query, 1 key, 2 value
  const int nq = a.q ? a.q_heads : 0;
  int role = 0;
  if (h >= nq) {
    h -= nq;
    role = 1;
    if (h >= a.kv_heads) {
      h -= a.kv_heads;
      role = 2;
    }
  }
  const T* src = role == 0   ? a.q + (int64_t)tok * a.q_ts + (int64_t)h * a.q_hs
                 : role == 1 ? a.k + (int64_t)tok * a.k_ts + (int64_t)h * a.k_hs
                             : a.v + (int64_t)tok * a.v_ts + (int64_t)h * a.v_hs;
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  if (in) raw = *reinterpret_cast<const uint4*>(src + c);
  int64_t slot = -1, pos = 0;
  bool bad = false;
  if (in) {
    if (role != 0) slot = a.idx64 ? ((const int64_t*)a.slots)[tok] : (int64_t)((const int*)a.slots)[tok];
    if (a.positions) {  // a value too: a token is stored whole or not at all
      pos = a.idx64 ? ((const int64_t*)a.positions)[tok] : (int64_t)((const int*)a.positions)[tok];
      if (pos < 0 || pos >= a.n_pos) bad = true;
    }
    if (slot >= a.n_slots) bad = true;
    if (bad && a.err) atomicExch(a.err, (int)WALSH_ERR_INDEX);
  }
  const float* nw = role == 0 ? a.q_norm : role == 1 ? a.k_norm : nullptr;
  const bool rot = a.positions != nullptr && role != 2;
  float x[VEC];
  {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = to_f(e[j]);
  }
  if (a.q_norm || a.k_norm) {  // the whole warp takes part in the reduction
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (nw) {
      const float r = 1.0f / sqrtf(ss * (1.0f / HD) + a.eps);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = x[j] * r * nw[c + j];
    }
  }
  if (!in) return;
  if (rot && !bad) {
    const float* cp = a.cos + pos * (HD / 2) + c / 2;
    const float* sp = a.sin + pos * (HD / 2) + c / 2;
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float cc = cp[j / 2], sn = sp[j / 2], u = x[j], w = x[j + 1];
      x[j] = u * cc - w * sn;
      x[j + 1] = u * sn + w * cc;
    }
  }
  if (nw || rot) {  // otherwise the bits are copied as they are
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = round_f<T>(x[j]);
  }
  if (role == 0) {
    if (bad) raw = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(a.q_out + ((int64_t)tok * a.q_heads + h) * HD + c) = raw;
    return;
  }
  if (slot < 0 || bad) return;
  // a slot may pass 2^31 in a large pool
  const int64_t page = slot < (1ll << 31) ? (int64_t)fdiv((uint32_t)slot, a.ps) : slot / a.ps.d;
  const int64_t off = page * a.page_stride + (int64_t)h * a.head_stride + (slot - page * a.ps.d) * a.row_stride + c;
  *reinterpret_cast<uint4*>((role == 1 ? a.k_pages : a.v_pages) + off) = raw;
}

template <typename T>
static int launch_append(AppendArgs<T> a, int hd, int64_t ntok, cudaStream_t s) {
  const int lpr = hd * (int)sizeof(T) / 16;
  // rows are numbered in 31 bits: more tokens go in several launches
  const int64_t most = ((1ll << 31) - 1) / a.per_tok.d;
  for (int64_t t0 = 0; t0 < ntok; t0 += most) {
    const int64_t n = min64(most, ntok - t0);
    AppendArgs<T> b = a;
    b.ntok = (int)n;
    if (b.q) b.q += t0 * b.q_ts, b.q_out += t0 * (int64_t)b.q_heads * hd;
    b.k += t0 * b.k_ts;
    b.v += t0 * b.v_ts;
    const int64_t ib = t0 * (b.idx64 ? 8 : 4);
    b.slots = (const char*)b.slots + ib;
    if (b.positions) b.positions = (const char*)b.positions + ib;
    const int64_t blocks = (n * b.per_tok.d * lpr + 255) / 256;
    switch (hd) {
      case 16: paged_append_kernel<T, 16><<<(unsigned)blocks, 256, 0, s>>>(b); break;
      case 32: paged_append_kernel<T, 32><<<(unsigned)blocks, 256, 0, s>>>(b); break;
      case 64: paged_append_kernel<T, 64><<<(unsigned)blocks, 256, 0, s>>>(b); break;
      default: paged_append_kernel<T, 128><<<(unsigned)blocks, 256, 0, s>>>(b); break;
    }
    if (const int r = launch_status()) return r;
  }
  return WALSH_OK;
}

}  // namespace walsh

using namespace walsh;

extern "C" walsh_status walsh_paged_append(const walsh_paged_kv* kv, const void* q, int64_t q_ts, int64_t q_hs,
                                           const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts,
                                           int64_t v_hs, int64_t ntok, int q_heads, const void* slots,
                                           const void* positions, int idx64, const float* rope_cos,
                                           const float* rope_sin, int64_t n_pos, const float* q_norm,
                                           const float* k_norm, float eps, void* q_out, void* stream) {
  if (int e = injected("paged_append")) return e;
  if (int e = check_pages(kv, false)) return e;
  WALSH_CHECK_ARG(k && v && slots && (q == nullptr) == (q_out == nullptr));
  WALSH_CHECK_ARG((positions == nullptr) == (rope_cos == nullptr) && (positions == nullptr) == (rope_sin == nullptr));
  WALSH_CHECK_ARG(q || !q_norm);
  WALSH_CHECK_ARG(!(q_norm || k_norm) || eps >= 0.f);
  WALSH_CHECK_SHAPE(ntok >= 0 && ntok < (1ll << 31) && (!q || (q_heads > 0 && q_heads <= 65535)));
  WALSH_CHECK_SHAPE(!positions || (n_pos > 0 && n_pos < (1ll << 31)));
  const int64_t vec = kv->dtype == WALSH_F32 ? 4 : 8;
  const int64_t strides[6] = {q ? q_ts : 0, q ? q_hs : 0, k_ts, k_hs, v_ts, v_hs};
  for (int64_t st : strides)
    if (st < 0 || st % vec) return st < 0 ? WALSH_ERR_SHAPE : WALSH_ERR_ALIGN;
  if (((((uintptr_t)q) | ((uintptr_t)k) | ((uintptr_t)v) | ((uintptr_t)q_out)) & 15u) != 0) return WALSH_ERR_ALIGN;
  if (ntok == 0) return WALSH_OK;
  const int per_tok = (q ? q_heads : 0) + 2 * kv->kv_heads;
  return WALSH_DISPATCH_DTYPE(kv->dtype, ET, [&]() -> int {
    AppendArgs<ET> a;
    a.q = (const ET*)q, a.k = (const ET*)k, a.v = (const ET*)v;
    a.q_ts = q_ts, a.q_hs = q_hs, a.k_ts = k_ts, a.k_hs = k_hs, a.v_ts = v_ts, a.v_hs = v_hs;
    a.ntok = 0, a.q_heads = q_heads, a.kv_heads = kv->kv_heads;
    a.per_tok = make_fastdiv((uint32_t)per_tok);
    a.slots = slots, a.positions = positions, a.idx64 = idx64;
    a.n_slots = (int64_t)kv->n_pages * kv->page_size;
    a.n_pos = (int)n_pos;
    a.cos = rope_cos, a.sin = rope_sin, a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.q_out = (ET*)q_out, a.k_pages = (ET*)kv->k_pages, a.v_pages = (ET*)kv->v_pages;
    a.page_stride = kv->page_stride, a.head_stride = kv->head_stride, a.row_stride = kv->row_stride;
    a.ps = make_fastdiv((uint32_t)kv->page_size);
    a.err = kv->err;
    return launch_append<ET>(a, kv->head_dim, ntok, (cudaStream_t)stream);
  }());
}
