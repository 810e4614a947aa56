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

#include <type_traits>

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

// One row again by one warp, over the keys it sees and no others.  A tile
// multiplies hidden keys by a probability of 0, which is no use when the value
// is infinite or NaN (a later token's, say): rows that come out as NaN are not
// stored but computed once more by this, so that only what a row sees reaches it
// (o may be q: a row of it is read before any lane stores its own part).
template <typename T, int HD>
__device__ __noinline__ void prefill_row_again(const PrefillArgs<T>& a, int b, int hk, const T* qp, int pos, T* op) {
  constexpr int DL = (HD + 31) / 32;
  const int lane = threadIdx.x & 31;
  const Visible vis = visible_keys(pos, a.pg.window, a.pg.sinks);
  float m, l, acc[DL];
  attend_row<T, HD>(a.pg, b, hk, qp, vis, 0, vis.n, a.scale_log2, &m, &l, acc);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < DL; ++i)
    if (i * 32 + lane < HD) op[i * 32 + lane] = round_f<T>(l == 0.f ? 0.f : acc[i] / l);
}

// CUDA-core form for float32: 64 rows x KT keys a step, 256 threads; a half warp owns four
// rows (scores, softmax and accumulator), so only K and V tiles need barriers.
// Shared-memory loads bound it: a thread's KT / 16 x 4 scores and its four rows of P V
// read operands as float4 (KT = 64; 32 for 128 channels, whose tiles fill the memory).
// 4 x 1000 tokens: 64 heads of 32 753 us, 16 on 2 heads of 128 673.
template <typename T, int HD, int KT>
__global__ void __launch_bounds__(256) paged_prefill_vec_kernel(const PrefillArgs<T> a) {
  constexpr int QT = 64, KJ = KT / 16, LD = HD + 4, LP = KT + 4, VEC = 16 / (int)sizeof(T), CH = HD / VEC;
  static_assert(sizeof(T) == 4, "16-bit types take the tensor-core form");
  extern __shared__ __align__(16) float sm[];
  float* Qs = sm;             // [QT][LD]
  float* Ks = Qs + QT * LD;   // [KT][LD]
  float* Vs = Ks + KT * LD;   // [KT][LD]
  float* Ps = Vs + KT * LD;   // [QT][LP]
  // key of each row of a tile (-1: none, or in a bad page) and its offset, looked up a tile ahead
  __shared__ int okk[2][KT];
  __shared__ int64_t offs[2][KT];
  const int b = blockIdx.z, hk = blockIdx.y, tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  int64_t first;
  const int T_ = query_span(a, b, &first);
  const int G = (int)a.group.d;
  const int64_t nrows = (int64_t)T_ * G;
  const int len = seq_len(a.pg, b), pos0 = len - T_;
  const int* trow = a.pg.table + (int64_t)b * a.pg.table_stride;
  const int64_t hoff = (int64_t)hk * a.pg.head_stride;
  const int64_t tiles = (nrows + QT - 1) / QT;
  // the grid covers max_q tokens, latest (longest) tiles first; tiles of a longer span follow in further turns
  for (int64_t turn = blockIdx.x; turn < tiles; turn += gridDim.x) {
    const int64_t r0 = (tiles - 1 - turn) * QT;
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
    auto lookup = [&](int k0, int buf) {
      if (tid < KT) {
        const int x = k0 + tid, key = x < nsink ? x : lo + (x - nsink);
        const int64_t off = x < n ? key_offset(a.pg, trow, key) : -1;
        offs[buf][tid] = off;
        okk[buf][tid] = off >= 0 ? key : -1;
      }
    };
    lookup(0, 0);
    for (int k0 = 0, buf = 0; k0 < n; k0 += KT, buf ^= 1) {
      __syncthreads();
      for (int i = tid; i < KT * CH; i += 256) {
        const int r = i / CH, c = i - r * CH;
        const int64_t off = offs[buf][r];
        uint4 kr = make_uint4(0u, 0u, 0u, 0u), vr = kr;
        if (off >= 0) {
          kr = __ldg(reinterpret_cast<const uint4*>(a.pg.k + hoff + off + c * VEC));
          vr = __ldg(reinterpret_cast<const uint4*>(a.pg.v + hoff + off + c * VEC));
        }
        *reinterpret_cast<uint4*>(&Ks[r * LD + c * VEC]) = kr;
        *reinterpret_cast<uint4*>(&Vs[r * LD + c * VEC]) = vr;
      }
      lookup(k0 + KT, buf ^ 1);
      __syncthreads();
      float s[4][KJ] = {};
      for (int d = 0; d < HD; d += 4) {
        float4 q4[4], k4[KJ];
#pragma unroll
        for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(&Qs[(ty * 4 + i) * LD + d]);
#pragma unroll
        for (int j = 0; j < KJ; ++j) k4[j] = *reinterpret_cast<const float4*>(&Ks[(tx + 16 * j) * LD + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < KJ; ++j)
            s[i][j] = fmaf(q4[i].x, k4[j].x, fmaf(q4[i].y, k4[j].y, fmaf(q4[i].z, k4[j].z, fmaf(q4[i].w, k4[j].w, s[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bool see[KJ];
        float mt = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const int key = okk[buf][tx + 16 * j];
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
        for (int j = 0; j < KJ; ++j) {
          const float p = see[j] ? ex2_f32(s[i][j] - sub_m) : 0.f;
          l[i] += p;
          Ps[(ty * 4 + i) * LP + tx + 16 * j] = p;
        }
      }
      __syncwarp();
      for (int j = 0; j < KT; j += 4) {
        float4 p4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p4[i] = *reinterpret_cast<const float4*>(&Ps[(ty * 4 + i) * LP + j]);
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          const float* vp = &Vs[j * LD + tx + 16 * d];
          const float v0 = vp[0], v1 = vp[LD], v2 = vp[2 * LD], v3 = vp[3 * LD];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[i][d] = fmaf(p4[i].w, v3, fmaf(p4[i].z, v2, fmaf(p4[i].y, v1, fmaf(p4[i].x, v0, acc[i][d]))));
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
      bool nan = false;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        acc[i][d] = L == 0.f ? 0.f : acc[i][d] / L;
        nan |= r < nr && acc[i][d] != acc[i][d];
      }
      const unsigned again = __ballot_sync(0xffffffffu, nan);
      if (r < nr && !(again & (0xffffu << (16 * (ty & 1))))) {
        const uint32_t t = fdiv((uint32_t)(r0 + r), a.group), g = (uint32_t)(r0 + r) - t * G;
        T* op = a.o + ((first + t) * Hq + (int64_t)hk * G + g) * HD;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) op[tx + 16 * d] = round_f<T>(acc[i][d]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (again & (0xffffu << (16 * h))) {
          const uint32_t x = (uint32_t)(r0 + (ty & ~1) * 4 + h * 4 + i), t = fdiv(x, a.group), g = x - t * G;
          prefill_row_again<T, HD>(a, b, hk, a.q + (first + t) * a.q_ts + (int64_t)(hk * G + g) * a.q_hs, pos0 + (int)t,
                                   a.o + ((first + t) * Hq + (int64_t)hk * G + g) * HD);
        }
    }
  }
}

// Tensor-core form for 16-bit types (mma.sync m16n8k16, float32 accumulation):
// W warps of MT x 16 rows; stages of KS keys double-buffered in shared memory by
// 16-byte asynchronous copies, one page lookup per key row and thread, made a
// stage ahead; steps of KT keys within a stage without barriers, and only those
// that some row of the warp sees.  Per step and warp: S - m = Q K^T - m (m is the
// MMAs' addend), P = 2^(c (S - m)) in float32, row sums of the float32 P, and O
// += P V.  TWO: P enters as two 16-bit terms, rounded to the type and what that left
// over, rounded again: good to 2^-18 (bf16) or 2^-22 (fp16, down to its smallest
// step) of each probability, below the output's own rounding.  Otherwise P is
// rounded once, as in the dense attention kernels, for callers that ask for it: half
// of these MMAs and no splitting (150 against 179 us in the case below, 199 against
// 256 with 32 channels), but two outputs of five move by a step.  m, O and the row
// sums move only when a row's maximum has grown by more than 8 powers of two (P <=
// 2^8).
// With 16 channels the exponentials are the floor (16 per clock and SM), with 32
// they and the MMAs take the same time; instructions bound it (8 x 2048 tokens,
// 32 heads of 16, window 512: 179 us; the floor 55).
template <typename T> __device__ __forceinline__ uint32_t pack_p(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_p<__half>(float lo, float hi) { return pack_f16(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack_p<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }

// two probabilities as the pair rounded to T and what that left over, rounded to T
template <typename T>
__device__ __forceinline__ void split_p(uint64_t p, uint32_t* hi, uint32_t* rest) {
  *hi = pack_p<T>(f2_lo(p), f2_hi(p));
  const float2 h = unpack2<T>(*hi);
  const uint64_t r = f2_fma(f2_pack(h.x, h.y), f2_dup(-1.f), p);
  *rest = pack_p<T>(f2_lo(r), f2_hi(r));
}

template <int HD>
__device__ __forceinline__ int row_swz(int r, int c) {  // 16-byte piece c of row r: its place in the row
  if constexpr (HD == 16) return c ^ ((r >> 2) & 1);
  else if constexpr (HD == 32) return c ^ ((r >> 1) & 3);
  else return c ^ (r & 7);
}

// d = a b + (c_lo, c_lo, c_hi, c_hi)
template <typename T>
__device__ __forceinline__ void mma_rowc(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c_lo, float c_hi);
template <>
__device__ __forceinline__ void mma_rowc<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c_lo,
                                                 float c_hi) {
  mma_f16_rowc(d, a, b0, b1, c_lo, c_hi);
}
template <>
__device__ __forceinline__ void mma_rowc<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c_lo,
                                                        float c_hi) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%11,%11};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c_lo), "f"(c_hi));
}

template <typename T, int HD, int W, int MT, int KT, int KS, int MINB, bool TWO>
__global__ void __launch_bounds__(W * 32, MINB) paged_prefill_mma_kernel(const PrefillArgs<T> a) {
  constexpr int QT = W * MT * 16, NT = W * 32, CH = HD / 8, STAGE = KS * HD;
  extern __shared__ __align__(16) unsigned char smb[];
  T* Ks = reinterpret_cast<T*>(smb);  // [2][KS][HD]
  T* Vs = Ks + 2 * STAGE;             // [2][KS][HD]
  // offsets of a stage's key rows (-1: none, or in a bad page), looked up a stage ahead, one row per thread
  __shared__ int64_t offs[3][KS];
  const int b = blockIdx.z, hk = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  int64_t first;
  const int T_ = query_span(a, b, &first);
  const int G = (int)a.group.d;
  const int64_t nrows = (int64_t)T_ * G, Hq = (int64_t)a.kv_heads * G;
  const int len = seq_len(a.pg, b), pos0 = len - T_;
  const int window = a.pg.window, sinks = a.pg.sinks;
  const int* trow = a.pg.table + (int64_t)b * a.pg.table_stride;
  const T* kb = a.pg.k + (int64_t)hk * a.pg.head_stride;
  const T* vb = a.pg.v + (int64_t)hk * a.pg.head_stride;
  const float c = a.scale_log2, slack = 8.f / c;
  const int64_t tiles = (nrows + QT - 1) / QT;
  // the grid covers max_q tokens, latest (longest) tiles first; tiles of a longer span follow in further turns
  for (int64_t turn = blockIdx.x; turn < tiles; turn += gridDim.x) {
    const int64_t r0 = (tiles - 1 - turn) * QT;
    const int nr = (int)min64(QT, nrows - r0);
    const int pos_first = pos0 + (int)fdiv((uint32_t)r0, a.group);
    const int pos_last = pos0 + (int)fdiv((uint32_t)(r0 + nr - 1), a.group);
    // the tile's keys are numbered: sinks before the first row's window, then lo .. pos_last.
    // In these numbers a row at pos sees x < end and (x >= end - window or x < sinks), with
    // end = pos + 1 - shift, shift = lo - nsink.
    const int lo = window > 0 ? max(0, pos_first + 1 - window) : 0;
    const int nsink = min(sinks, lo), n = nsink + max(0, pos_last + 1 - lo), shift = lo - nsink;
    const int nst = (n + KS - 1) / KS;

    auto lookup = [&](int st) {
      for (int r = tid; r < KS; r += NT) {
        const int x = st * KS + r;
        offs[st % 3][r] = x < n ? key_offset(a.pg, trow, x < nsink ? x : x + shift) : -1;
      }
    };
    // starts the copies of stage st; returns whether one of its keys lies in a bad page
    constexpr int RPT = KS * CH / NT;  // 16-byte pieces per thread and matrix
    static_assert(KS * CH % NT == 0 && NT % CH == 0, "whole pieces");
    const int pr = tid / CH, pc = tid - pr * CH;
    auto load = [&](int st) {
      const int buf = st & 1;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = pr + i * (NT / CH);
        const int64_t off = offs[st % 3][r];
        const bool in = off >= 0;
        const int64_t o = (in ? off : 0) + pc * 8;
        const int at = buf * STAGE + r * HD + row_swz<HD>(r, pc) * 8;
        cp_async16(Ks + at, kb + o, in ? 16 : 0);
        cp_async16(Vs + at, vb + o, in ? 16 : 0);
        bad |= !in && st * KS + r < n;
      }
      cp_async_commit();
      return bad;
    };
    __syncthreads();  // the buffers of the turn before are free
    lookup(0);
    lookup(1);
    __syncthreads();
    bool bad_next = load(0);

    // Q fragments and bounds of this thread's rows: tile mt of the warp, halves g and g + 8
    uint32_t qf[MT][HD / 16][4];
    int end[MT][2];
    const int wr0 = warp * MT * 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = wr0 + mt * 16 + g + 8 * h;
        const uint32_t x = (uint32_t)(r0 + min(r, nr - 1)), t = fdiv(x, a.group), gi = x - t * G;
        const uint32_t* qp =
            reinterpret_cast<const uint32_t*>(a.q + (first + t) * a.q_ts + (int64_t)(hk * G + gi) * a.q_hs);
        const int pos = pos0 + (int)t;
        end[mt][h] = r < nr && pos >= 0 ? pos + 1 - shift : 0;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j) qf[mt][ks][2 * j + h] = r < nr ? __ldg(qp + ks * 8 + t4 + j * 4) : 0u;
      }
    // numbers that every row of the warp sees: beg_all <= x < end_all (and x < sinks); that some row sees: beg_any, end_any
    const int wr1 = min(nr, wr0 + MT * 16) - 1;
    int beg_any = 0, end_any = 0, beg_all = -1, end_all = 0;
    if (wr0 < nr) {
      end_all = max(0, pos0 + (int)fdiv((uint32_t)(r0 + wr0), a.group) + 1 - shift);
      end_any = max(0, pos0 + (int)fdiv((uint32_t)(r0 + wr1), a.group) + 1 - shift);
      if (window > 0) {
        beg_any = end_all - window;
        beg_all = end_any - window;
      }
    }

    // nm: minus the score a row's exponents refer to.  It is the MMAs' addend, so
    // scores come out relative to it; 0 until the row's first key (thr = -inf)
    float nm[MT][2], thr[MT][2], thr_min = -CUDART_INF_F, l[MT][2], acc[MT][HD / 8][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) nm[mt][h] = l[mt][h] = 0.f, thr[mt][h] = -CUDART_INF_F;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) acc[mt][i][0] = acc[mt][i][1] = acc[mt][i][2] = acc[mt][i][3] = 0.f;
    }

    // this lane's ldmatrix rows within 16 keys, in bytes from a step's first row
    uint32_t k_lane[HD / 16], v_lane[HD / 16];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      const int kr = (lane & 7) + ((lane >> 4) << 3), vr = lane & 15;
      k_lane[i] = (kr * HD + row_swz<HD>(kr, i * 2 + ((lane >> 3) & 1)) * 8) * 2;
      v_lane[i] = (vr * HD + row_swz<HD>(vr, i * 2 + (lane >> 4)) * 8) * 2;
    }
    const uint64_t c2 = f2_dup(c), one2 = f2_dup(1.f);
    // one step of KT keys from number x0; EDGE: some row does not see all of them
    auto step = [&](auto edge_tag, const int x0, const int st, const bool bad) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      const int row0 = x0 - st * KS;
      const unsigned char* kt_s = smb + ((st & 1) * STAGE + row0 * HD) * 2;
      const unsigned char* vt_s = kt_s + 2 * STAGE * 2;
      float s[MT][KT / 8][4];
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int np = 0; np < KT / 16; ++np) {
          uint32_t kf[4];
          ldsm_x4(kf, kt_s + k_lane[ks] + np * 16 * HD * 2);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float* d = s[mt][2 * np + j];
              if (ks == 0) mma_rowc<T>(d, qf[mt][0], kf[2 * j], kf[2 * j + 1], nm[mt][0], nm[mt][1]);
              else mma16<T>(d, qf[mt][ks], kf[2 * j], kf[2 * j + 1]);
            }
        }
      if constexpr (EDGE) {
        if (x0 + KT > end_all) {  // keys after some row
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int e_lo = end[mt][0] - x0 - 2 * t4, e_hi = end[mt][1] - x0 - 2 * t4;
#pragma unroll
            for (int i = 0; i < KT / 8; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (i * 8 + e >= e_lo) s[mt][i][e] = -CUDART_INF_F;
                if (i * 8 + e >= e_hi) s[mt][i][2 + e] = -CUDART_INF_F;
              }
          }
        }
        if (window > 0 && x0 < beg_all) {  // keys before some row's window; sinks stay
          const int sk = max(sinks - x0, 0) - 2 * t4;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int b_lo = end[mt][0] - window - x0 - 2 * t4, b_hi = end[mt][1] - window - x0 - 2 * t4;
#pragma unroll
            for (int i = 0; i < KT / 8; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (i * 8 + e < b_lo && i * 8 + e >= sk) s[mt][i][e] = -CUDART_INF_F;
                if (i * 8 + e < b_hi && i * 8 + e >= sk) s[mt][i][2 + e] = -CUDART_INF_F;
              }
          }
        }
        if (bad) {
#pragma unroll
          for (int i = 0; i < KT / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (offs[st % 3][row0 + i * 8 + 2 * t4 + e] < 0) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][i][e] = s[mt][i][2 + e] = -CUDART_INF_F;
              }
        }
      }
      // a row's reference moves when its maximum is more than the slack above it
      float mx[MT][2], top = -CUDART_INF_F;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mx[mt][0] = mx[mt][1] = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < KT / 8; ++i) {
          mx[mt][0] = fmax3(mx[mt][0], s[mt][i][0], s[mt][i][1]);
          mx[mt][1] = fmax3(mx[mt][1], s[mt][i][2], s[mt][i][3]);
        }
        top = fmax3(top, mx[mt][0], mx[mt][1]);
      }
      if (__any_sync(0xffffffffu, top > thr_min)) {
        thr_min = CUDART_INF_F;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = mx[mt][h];
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const bool mv = x > thr[mt][h], fresh = thr[mt][h] == -CUDART_INF_F;
            const float d = mv ? x : 0.f;
            // before a row's first key O and l are zero and any finite factor will do
            const float f = mv && !fresh ? ex2_f32(-d * c) : 1.f;
            l[mt][h] *= f;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) acc[mt][i][2 * h] *= f, acc[mt][i][2 * h + 1] *= f;
#pragma unroll
            for (int i = 0; i < KT / 8; ++i) s[mt][i][2 * h] -= d, s[mt][i][2 * h + 1] -= d;
            if (mv) {
              nm[mt][h] -= d;
              thr[mt][h] = slack;
            }
            thr_min = fminf(thr_min, thr[mt][h]);
          }
      }
      uint32_t pf[MT][KT / 16][4], pl[MT][TWO ? KT / 16 : 1][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint64_t rs0 = 0, rs1 = 0;
#pragma unroll
        for (int i = 0; i < KT / 8; ++i) {
          const uint64_t x = f2_mul(f2_pack(s[mt][i][0], s[mt][i][1]), c2), y = f2_mul(f2_pack(s[mt][i][2], s[mt][i][3]), c2);
          const uint64_t p0 = f2_pack(ex2_f32(f2_lo(x)), ex2_f32(f2_hi(x))), p1 = f2_pack(ex2_f32(f2_lo(y)), ex2_f32(f2_hi(y)));
          rs0 = f2_fma(p0, one2, rs0);
          rs1 = f2_fma(p1, one2, rs1);
          const int kk = i >> 1, j = (i & 1) * 2;
          if constexpr (TWO) {
            split_p<T>(p0, &pf[mt][kk][j], &pl[mt][kk][j]);
            split_p<T>(p1, &pf[mt][kk][j + 1], &pl[mt][kk][j + 1]);
          } else {
            pf[mt][kk][j] = pack_p<T>(f2_lo(p0), f2_hi(p0));
            pf[mt][kk][j + 1] = pack_p<T>(f2_lo(p1), f2_hi(p1));
          }
        }
        l[mt][0] += f2_lo(rs0) + f2_hi(rs0);
        l[mt][1] += f2_lo(rs1) + f2_hi(rs1);
      }
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
        for (int dp = 0; dp < HD / 16; ++dp) {
          uint32_t vf[4];
          ldsm_x4_t(vf, vt_s + v_lane[dp] + kk * 16 * HD * 2);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<T>(acc[mt][2 * dp], pf[mt][kk], vf[0], vf[1]);
            mma16<T>(acc[mt][2 * dp + 1], pf[mt][kk], vf[2], vf[3]);
            if constexpr (TWO) {
              mma16<T>(acc[mt][2 * dp], pl[mt][kk], vf[0], vf[1]);
              mma16<T>(acc[mt][2 * dp + 1], pl[mt][kk], vf[2], vf[3]);
            }
          }
        }
    };
    for (int st = 0; st < nst; ++st) {
      const bool bad_mine = bad_next;
      if (st + 1 < nst) {
        if (st > 0) __syncthreads();  // the other buffer is free
        bad_next = load(st + 1);
        lookup(st + 2);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      const bool bad = __syncthreads_or(bad_mine);
      // steps some row of the warp sees: from its rows' windows (or the sinks) to their ends
      const int x_end = min(end_any, (st + 1) * KS);
#pragma unroll 1
      for (int x0 = st * KS; x0 < x_end; x0 += KT) {
        if (x0 + KT <= beg_any && x0 >= sinks) continue;
        if (x0 + KT > end_all || x0 < beg_all || bad) step(std::true_type{}, x0, st, bad);
        else step(std::false_type{}, x0, st, false);
      }
    }
    cp_async_wait<0>();  // (a tile whose rows see nothing has started its first stage all the same)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float L = l[mt][h];
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const int r = wr0 + mt * 16 + g + 8 * h;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          const float u = acc[mt][i][2 * h] *= inv, w = acc[mt][i][2 * h + 1] *= inv;
          nan |= r < nr && (u != u || w != w);
        }
        unsigned again = __ballot_sync(0xffffffffu, nan);
        if (r < nr && !(again & (15u << (lane & 28)))) {
          const uint32_t x = (uint32_t)(r0 + r), t = fdiv(x, a.group), gi = x - t * G;
          T* op = a.o + ((first + t) * Hq + (int64_t)hk * G + gi) * HD;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            T pair[2] = {round_f<T>(acc[mt][i][2 * h]), round_f<T>(acc[mt][i][2 * h + 1])};
            *reinterpret_cast<uint32_t*>(op + i * 8 + 2 * t4) = *reinterpret_cast<uint32_t*>(pair);
          }
        }
        while (again) {
          const int q = (__ffs(again) - 1) >> 2;  // the lane quad of a row
          again &= ~(15u << (4 * q));
          const uint32_t x = (uint32_t)(r0 + wr0 + mt * 16 + 8 * h + q), t = fdiv(x, a.group), gi = x - t * G;
          prefill_row_again<T, HD>(a, b, hk, a.q + (first + t) * a.q_ts + (int64_t)(hk * G + gi) * a.q_hs, pos0 + (int)t,
                                   a.o + ((first + t) * Hq + (int64_t)hk * G + gi) * HD);
        }
      }
  }
}

template <typename T, int HD, int W, int MT, int KT, int KS, int MINB>
static int launch_prefill_tile(const PrefillArgs<T>& a, int B, int max_q, bool two, cudaStream_t s) {
  constexpr int smem = 4 * KS * HD * 2;
  auto* kern = two ? paged_prefill_mma_kernel<T, HD, W, MT, KT, KS, MINB, true>
                   : paged_prefill_mma_kernel<T, HD, W, MT, KT, KS, MINB, false>;
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status();
  const int64_t tiles = ((int64_t)max_q * a.group.d + W * MT * 16 - 1) / (W * MT * 16);
  kern<<<dim3((unsigned)tiles, a.kv_heads, B), W * 32, smem, s>>>(a);
  return launch_status();
}

// Warps, 16-row tiles per warp, keys per step and per stage, CTAs per SM.
// Measured with two terms, replayed from a graph: 16 channels (8 x 2048 tokens, 32 heads, window
// 512): (4, 1, 64, 128, 5) 179 us, (4, 1, 64, 128, 4) 178, (8, 1, 32, 256, 3) 184,
// (4, 2, 32, 256, 4) 165, but 5.8 against 4.8 us for a few short prompts; 32
// channels (3 later parts up to 3500, 64 heads, window 1024): (4, 2, 32, 256, 3)
// 256 us, (4, 2, 32, 128, 4) 281, (4, 1, 64, 128, 4) 269; 64 channels (8 x 1000, 32
// on 8 heads): (4, 1, 64, 128, 3) 195 us, (4, 1, 64, 64, 3) 201, (4, 1, 64, 128, 2)
// 211; 128 (8 x 800, 16 on 2): (4, 1, 64, 64, 2) 130, (4, 1, 32, 64, 2) 131, (8, 1,
// 64, 64, 1) 143.
template <typename T, int HD>
static int launch_prefill_mma(const PrefillArgs<T>& a, int B, int max_q, bool two, cudaStream_t s) {
  if constexpr (HD == 16) return launch_prefill_tile<T, HD, 4, 1, 64, 128, 5>(a, B, max_q, two, s);
  else if constexpr (HD == 32) return launch_prefill_tile<T, HD, 4, 2, 32, 256, 3>(a, B, max_q, two, s);
  else if constexpr (HD == 64) return launch_prefill_tile<T, HD, 4, 1, 64, 128, 3>(a, B, max_q, two, s);
  else return launch_prefill_tile<T, HD, 4, 1, 64, 64, 2>(a, B, max_q, two, s);
}

template <typename T, int HD>
static int launch_prefill(const PrefillArgs<T>& a, int B, int max_q, bool two, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    return launch_prefill_mma<T, HD>(a, B, max_q, two, s);
  } else {
    constexpr int QT = 64, KT = HD == 128 ? 32 : 64, LD = HD + 4;
    constexpr int smem = ((QT + 2 * KT) * LD + QT * (KT + 4)) * 4;
    auto* kern = paged_prefill_vec_kernel<T, HD, KT>;
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return launch_status();
    const int64_t tiles = ((int64_t)max_q * a.group.d + QT - 1) / QT;
    kern<<<dim3((unsigned)tiles, a.kv_heads, B), 256, smem, s>>>(a);
    return launch_status();
  }
}

}  // namespace walsh

using namespace walsh;

static int prefill_fwd(const walsh_paged_kv* kv, const void* q, int64_t q_ts, int64_t q_hs, int64_t q_rows,
                       const int32_t* q_offsets, int B, int q_heads, int max_q, bool two, void* o, void* stream) {
  if (int e = injected("paged_prefill_fwd")) return e;
  if (int e = check_pages(kv, true)) return e;
  WALSH_CHECK_ARG(q && q_offsets && o);
  WALSH_CHECK_SHAPE(B >= 0 && B <= 65535 && q_heads > 0 && q_heads <= 65535 && q_heads % kv->kv_heads == 0);
  WALSH_CHECK_SHAPE(q_rows >= 0 && q_rows < (1ll << 31) && max_q >= 0 && (int64_t)max_q * q_heads < (1ll << 31) &&
                    q_rows * (q_heads / kv->kv_heads) < (1ll << 31));
  const int64_t vec = kv->dtype == WALSH_F32 ? 4 : 8;
  WALSH_CHECK_SHAPE(q_ts >= 0 && q_hs >= 0);
  if (((((uintptr_t)q) | ((uintptr_t)o)) & 15u) != 0 || q_ts % vec || q_hs % vec) return WALSH_ERR_ALIGN;
  if (B == 0 || q_rows == 0) return WALSH_OK;
  if (max_q == 0) max_q = 1;  // (longer spans are still computed)
  return WALSH_DISPATCH_DTYPE(kv->dtype, ET, [&]() -> int {
    PrefillArgs<ET> a;
    a.pg = make_pages<ET>(kv);
    a.q = (const ET*)q, a.q_ts = q_ts, a.q_hs = q_hs, a.q_rows = q_rows, a.q_off = q_offsets, a.o = (ET*)o;
    a.kv_heads = kv->kv_heads;
    a.group = make_fastdiv((uint32_t)(q_heads / kv->kv_heads));
    a.scale_log2 = kv->scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    switch (kv->head_dim) {
      case 16: return launch_prefill<ET, 16>(a, B, max_q, two, s);
      case 32: return launch_prefill<ET, 32>(a, B, max_q, two, s);
      case 64: return launch_prefill<ET, 64>(a, B, max_q, two, s);
      default: return launch_prefill<ET, 128>(a, B, max_q, two, s);
    }
  }());
}

extern "C" walsh_status walsh_paged_prefill_fwd(const walsh_paged_kv* kv, const void* q, int64_t q_ts, int64_t q_hs,
                                                int64_t q_rows, const int32_t* q_offsets, int B, int q_heads,
                                                int max_q, void* o, void* stream) {
  return prefill_fwd(kv, q, q_ts, q_hs, q_rows, q_offsets, B, q_heads, max_q, true, o, stream);
}

extern "C" walsh_status walsh_paged_prefill_rounded_fwd(const walsh_paged_kv* kv, const void* q, int64_t q_ts,
                                                        int64_t q_hs, int64_t q_rows, const int32_t* q_offsets, int B,
                                                        int q_heads, int max_q, void* o, void* stream) {
  return prefill_fwd(kv, q, q_ts, q_hs, q_rows, q_offsets, B, q_heads, max_q, false, o, stream);
}
