// Append of new tokens to a paged key/value cache: per-head RMS norm of q and
// k, rotation at each token's position, and the scatter of k and v into their
// slots, in one pass.
//
//   n = x / sqrt(mean_d(x^2) + eps) * w          (when a norm weight is given)
//   (y_2i, y_2i+1) = (n_2i c - n_2i+1 s, n_2i s + n_2i+1 c),  c, s = cos, sin[pos][i]
//
// Bytes bound it: every element is read once and written once and the
// arithmetic is a few operations per element.  A thread owns 32 bytes of one
// head row, so a row's norm is a sum within the thread and over the hd * size /
// 32 (1 to 16) lanes that hold it.  With 16 bytes per thread the index and
// address arithmetic (about 280 instructions per thread in all) bounded it:
// 121 us at 65536 tokens of 3 x 32 heads of 16 channels.
#include "mma.cuh"
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
  int n_pos, vec_rope;  // vec_rope: the tables' rows lie on 16-byte boundaries
  int wide;             // every row read or written lies on a 32-byte boundary
  const float *cos, *sin, *q_norm, *k_norm;
  float eps;
  T *q_out, *k_pages, *v_pages;
  int64_t page_stride, head_stride, row_stride;
  FastDiv ps;
  int* err;
};

__device__ __forceinline__ uint32_t round_pair(const __half*, float lo, float hi) { return pack_f16(lo, hi); }
__device__ __forceinline__ uint32_t round_pair(const __nv_bfloat16*, float lo, float hi) { return pack_bf16(lo, hi); }

// 32 bytes in one access (both ends on 32-byte boundaries) or two
__device__ __forceinline__ void load32(const void* p, uint4* r, bool wide) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0].x), "=r"(r[0].y), "=r"(r[0].z), "=r"(r[0].w), "=r"(r[1].x), "=r"(r[1].y), "=r"(r[1].z),
                   "=r"(r[1].w)
                 : "l"(p));
  } else {
    r[0] = reinterpret_cast<const uint4*>(p)[0];
    r[1] = reinterpret_cast<const uint4*>(p)[1];
  }
}
__device__ __forceinline__ void store32(void* p, const uint4* r, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p), "r"(r[0].x), "r"(r[0].y), "r"(r[0].z),
                 "r"(r[0].w), "r"(r[1].x), "r"(r[1].y), "r"(r[1].z), "r"(r[1].w)
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = r[0];
    reinterpret_cast<uint4*>(p)[1] = r[1];
  }
}

// four values of a rotation table (whose rows need not lie on 16-byte boundaries)
__device__ __forceinline__ float4 load_rope(const float* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const float4*>(p));
  return make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
}

// 32 bytes as floats, and back with one rounding each
template <typename T>
__device__ __forceinline__ void piece_to_f(const uint4* raw, float* x) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        x[4 * i + j] = __uint_as_float(w[j]);
      } else {
        const float2 f = unpack2<T>(w[j]);
        x[8 * i + 2 * j] = f.x, x[8 * i + 2 * j + 1] = f.y;
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ void f_to_piece(const float* x, uint4* raw) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(x[4 * i + j]);
      else w[j] = round_pair((const T*)nullptr, x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
    }
    raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs<T> a) {
  constexpr int VEC = 32 / (int)sizeof(T), LPR = HD / VEC;
  const uint32_t row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = (int)(threadIdx.x % LPR) * VEC;  // first element of this thread's piece
  const bool in = row < (uint32_t)a.ntok * a.per_tok.d;
  const uint32_t tok = in ? fdiv(row, a.per_tok) : 0u;
  int h = in ? (int)(row - tok * a.per_tok.d) : 0;
  const int nq = a.q ? a.q_heads : 0;
  // role: 0 query, 1 key, 2 value
  int role = 0;
  const T* src = a.q + (int64_t)tok * a.q_ts + (int64_t)h * a.q_hs;
  if (h >= nq) {
    h -= nq;
    role = 1;
    src = a.k + (int64_t)tok * a.k_ts + (int64_t)h * a.k_hs;
    if (h >= a.kv_heads) {
      h -= a.kv_heads;
      role = 2;
      src = a.v + (int64_t)tok * a.v_ts + (int64_t)h * a.v_hs;
    }
  }
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  int64_t slot = -1, pos = 0;
  if (in) {
    load32(src + c, raw, a.wide);
    if (role != 0) slot = a.idx64 ? ((const int64_t*)a.slots)[tok] : (int64_t)((const int*)a.slots)[tok];
    if (a.positions)  // a value's too: a token is stored whole or not at all
      pos = a.idx64 ? ((const int64_t*)a.positions)[tok] : (int64_t)((const int*)a.positions)[tok];
  }
  const bool bad = (a.positions && (pos < 0 || pos >= a.n_pos)) || slot >= a.n_slots;
  const float* nw = role == 0 ? a.q_norm : role == 1 ? a.k_norm : nullptr;
  const bool rot = a.positions != nullptr && role != 2;
  if (LPR > 1 ? (a.q_norm || a.k_norm || rot) : (nw || rot)) {  // the shuffles need the whole warp where a row spans lanes
    float x[VEC];
    piece_to_f<T>(raw, x);
    if (a.q_norm || a.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss = fmaf(x[j], x[j], ss);
      if constexpr (LPR > 1) {
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      }
      if (nw) {
        const float r = rsqrtf(ss * (1.0f / HD) + a.eps);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = x[j] * r * __ldg(nw + c + j);
      }
    }
    if (rot && !bad) {
      const float* cp = a.cos + pos * (HD / 2) + c / 2;
      const float* sp = a.sin + pos * (HD / 2) + c / 2;
#pragma unroll
      for (int j = 0; j < VEC; j += 8) {  // rows of the tables are 32 bytes or more
        const float4 cv = load_rope(cp + j / 2, a.vec_rope), sv = load_rope(sp + j / 2, a.vec_rope);
        const float cc[4] = {cv.x, cv.y, cv.z, cv.w}, sn[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x[j + 2 * i], q = x[j + 2 * i + 1];
          x[j + 2 * i] = p * cc[i] - q * sn[i];
          x[j + 2 * i + 1] = p * sn[i] + q * cc[i];
        }
      }
    }
    if (nw || rot) f_to_piece<T>(x, raw);  // otherwise the bits are copied as they are
  }
  if (!in) return;
  if (bad && a.err) atomicExch(a.err, (int)WALSH_ERR_INDEX);
  T* dst;
  if (role == 0) {
    if (bad) raw[0] = raw[1] = make_uint4(0u, 0u, 0u, 0u);
    dst = a.q_out + ((int64_t)tok * a.q_heads + h) * HD + c;
  } else {
    if (slot < 0 || bad) return;
    // a slot may pass 2^31 in a large pool
    const int64_t page = slot < (1ll << 31) ? (int64_t)fdiv((uint32_t)slot, a.ps) : slot / a.ps.d;
    dst = (role == 1 ? a.k_pages : a.v_pages) + page * a.page_stride + (int64_t)h * a.head_stride +
          (slot - page * a.ps.d) * a.row_stride + c;
  }
  store32(dst, raw, a.wide);
}

template <typename T, int HD>
static void launch_append_rows(const AppendArgs<T>& b, int64_t rows, cudaStream_t s) {
  constexpr int RPB = 256 / (HD * (int)sizeof(T) / 32);  // rows per block
  paged_append_kernel<T, HD><<<(unsigned)((rows + RPB - 1) / RPB), 256, 0, s>>>(b);
}

template <typename T>
static int launch_append(AppendArgs<T> a, int hd, int64_t ntok, cudaStream_t s) {
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
    switch (hd) {
      case 16: launch_append_rows<T, 16>(b, n * b.per_tok.d, s); break;
      case 32: launch_append_rows<T, 32>(b, n * b.per_tok.d, s); break;
      case 64: launch_append_rows<T, 64>(b, n * b.per_tok.d, s); break;
      default: launch_append_rows<T, 128>(b, n * b.per_tok.d, s); break;
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
    int64_t all = (int64_t)((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)kv->k_pages |
                            (uintptr_t)kv->v_pages);
    for (int64_t st : strides) all |= st * (int64_t)sizeof(ET);
    all |= (kv->page_stride | kv->head_stride | kv->row_stride) * (int64_t)sizeof(ET);
    a.wide = all % 32 == 0;
    a.vec_rope = ((((uintptr_t)rope_cos) | ((uintptr_t)rope_sin)) & 15u) == 0;
    a.cos = rope_cos, a.sin = rope_sin, a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.q_out = (ET*)q_out, a.k_pages = (ET*)kv->k_pages, a.v_pages = (ET*)kv->v_pages;
    a.page_stride = kv->page_stride, a.head_stride = kv->head_stride, a.row_stride = kv->row_stride;
    a.ps = make_fastdiv((uint32_t)kv->page_size);
    a.err = kv->err;
    return launch_append<ET>(a, kv->head_dim, ntok, (cudaStream_t)stream);
  }());
}
