// Linear attention with a decay for each head.  A head keeps a matrix state S [K, V]:
//
//   S[t] = e^{g[t]} S[t-1] + k[t] v[t]^T,      y[t] = scale S[t]^T q[t]
//
// Prompts and training run over chunks of C tokens.  With G[i] the sum of g in the chunk up to i, n its last token:
//
//   y[i]  = scale (sum_{j <= i} (q[i].k[j]) e^{G[i] - G[j]} v[j] + e^{G[i]} S_in^T q[i])
//   S_out = e^{G[n]} S_in + sum_j e^{G[n] - G[j]} k[j] v[j]^T
//
// so that nearly all of the work is matrix products.  Every exponent is a difference of sums, at most zero where the
// log decays are: nothing overflows, whatever the decays.  The sums are pairs of floats (Sum): a difference of two
// plain ones is off by 2^-24 of the sums, which a token that clears the state makes large.
//
// The products run on bf16 matrix instructions for all three types: a bf16 value is one bf16, an fp16 value is the
// sum of two, exactly, an fp32 value of three (8 + 8 + 8 bits), and a product of two such sums is the products of
// their parts, without those below fp32's last bit.  An fp32 product of six parts takes 96 cycles a 16 x 16 x 32 tile,
// where fp32 matrix instructions would take 256.  Sums and states are fp32.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace lng {
namespace {

constexpr int MAX_D = 128;  // of keys and values
constexpr int VT = 64;      // columns of values a block takes
constexpr int PAD = 8;      // elements behind a row in LDS

// Planes: bf16 parts of an input; PREC: parts of a computed operand of a product whose result is rounded to the type.
template <typename T>
struct Traits;
template <>
struct Traits<bf16> {
  static constexpr int planes = 1, prec = 2, chunk = 64;
};
template <>
struct Traits<_Float16> {
  static constexpr int planes = 2, prec = 2, chunk = 32;
};
template <>
struct Traits<float> {
  static constexpr int planes = 3, prec = 3, chunk = 32;
};

// ------------------------------------------------------------------ arguments
struct Args {
  int64_t B, T;
  int H, Hq, Hk, Hv, K, V, vts, segs, seg_chunks, chunks;
  float scale;
  const void *q, *k, *v, *dy;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, yb, yt, yh;
  bool qvec, kvec, vvec, yvec;  // rows that 16-byte loads take
  const float* g;
  int64_t gb, gt;
  const float* start;    // [B, H, K, V] or null
  const int* lengths;    // [B] or null
  void* y;               // [B, T, H, V]
  float* end;            // [B, H, K, V] or null
  float* ckpt;           // the state before every chunk [B, H, chunks, K, V], or null
  float* seg_state;      // [B, H, segs, K, V] what a segment adds, then the state before it
  float* seg_decay;      // [B, H, segs] log2 of a segment's decay
  // backward
  const float* dend;
  float* dstart;
  void *dq, *dk, *dv;    // in the type, or fp32 partial sums of each head (and value tile)
  bool dq32, dk32, dv32;
  float* dg;             // [B, T, H * vts]
};

struct Unit {  // one block's work
  int64_t b;
  int h, vt, seg;
  int len;       // the sequence's own tokens
};

__device__ __forceinline__ Unit unit_of(const Args& a, int segs, int first_seg) {
  int64_t u = blockIdx.x;
  Unit r;
  r.vt = static_cast<int>(u % a.vts), u /= a.vts;
  r.h = static_cast<int>(u % a.H), u /= a.H;
  r.seg = first_seg + static_cast<int>(u % segs);
  r.b = u / segs;
  r.len = static_cast<int>(a.T);
  if (a.lengths) r.len = min(max(a.lengths[r.b], 0), static_cast<int>(a.T));
  return r;
}

// ------------------------------------------------------------------ sums of log decays
struct Sum {
  float hi, lo;
};
__device__ __forceinline__ Sum add(Sum a, Sum b) {
  const float s = a.hi + b.hi, bb = s - a.hi;
  const float lo = ((a.hi - (s - bb)) + (b.hi - bb)) + (a.lo + b.lo);
  const float hi = s + lo;
  return {hi, lo - (hi - s)};
}
// 2^(a - b)
__device__ __forceinline__ float exp2_gap(float ahi, float alo, float bhi, float blo) {
  return __builtin_amdgcn_exp2f((ahi - bhi) + (alo - blo));
}
// A log decay in powers of two.  Below -300 the decay is zero in fp32 whatever the rest: it counts as -300, minus
// infinity too, so that a difference of two such sums is no NaN.
__device__ __forceinline__ Sum log2_decay(float g) {
  constexpr float REST = 1.92596303e-8f;  // log2 e - LOG2E
  g = g < -300.f ? -300.f : g;
  const float p = g * LOG2E;
  return {p, fmaf(g, REST, fmaf(g, LOG2E, -p))};
}
// Inclusive sums over the first n lanes' tokens
__device__ __forceinline__ Sum scan_sum(Sum v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const Sum o{__shfl_up(v.hi, off, 64), __shfl_up(v.lo, off, 64)};
    if (lane >= off) v = add(o, v);
  }
  return v;
}

// ------------------------------------------------------------------ operands
// x as the sum of N bf16 values; what is no finite bf16 value stands in the first part alone
template <int N>
__device__ __forceinline__ void split(float x, bf16 (&out)[N]) {
  float r = x;
#pragma unroll
  for (int p = 0; p < N; ++p) {
    out[p] = static_cast<bf16>(r);
    const float f = static_cast<float>(out[p]);
    if (p + 1 < N) r = fabsf(f) < INFINITY ? r - f : 0.f;
  }
}

template <int N>
struct Frag {
  bf16x8 p[N];
};

template <int N>
__device__ __forceinline__ void put(Frag<N>& f, int i, float x) {
  bf16 t[N];
  split<N>(x, t);
#pragma unroll
  for (int p = 0; p < N; ++p) f.p[p][i] = t[p];
}

// acc += a . b without the products of parts that add to LIM or more
template <int LIM, int NA, int NB>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<NA>& a, const Frag<NB>& b) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < LIM) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
}

// Lane l of a 16 x 16 x 32 product: row (column) l % 16 of an operand, and of its 32 products' index the values
// 4 g + 0..3 and 16 + 4 g + 0..3 with g = l / 16.  (Any order will do that both operands share; this one is that of
// two stacked result tiles, whose rows 4 g + 0..3 a lane holds, so that results are operands as they are.)
//
// From LDS, rows of `stride` elements, planes `plane` elements apart.  by_row: row r0 + l % 16, index along the row.
template <int N>
__device__ __forceinline__ Frag<N> by_row(const bf16* s, int stride, int plane, int r0, int c0) {
  const int lane = threadIdx.x & 63;
  const bf16* at = s + (r0 + (lane & 15)) * stride + c0 + 4 * (lane >> 4);
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(at + p * plane);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(at + p * plane + 16);
    f.p[p] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}
// by_col: column c0 + l % 16, index along the rows from r0: the transposing read gives lane i of each 16-lane group
// element i % 4 of the 8-byte chunks that lanes i / 4 + 4 c address (c = 0..3).
template <int N>
__device__ __forceinline__ Frag<N> by_col(const bf16* s, int stride, int plane, int r0, int c0) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const bf16* at = s + (r0 + 4 * g + (i >> 2)) * stride + c0 + 4 * (i & 3);
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) bf16x4*)(at + p * plane));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) bf16x4*)(at + p * plane + 16 * stride));
    f.p[p] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}
template <int N>
__device__ __forceinline__ float value(const Frag<N>& f, int i) {
  float x = 0.f;
#pragma unroll
  for (int p = N - 1; p >= 0; --p) x += static_cast<float>(f.p[p][i]);
  return x;
}
// Four neighbouring values of a row
template <int N>
__device__ __forceinline__ void four(const bf16* at, int plane, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = 0.f;
#pragma unroll
  for (int p = N - 1; p >= 0; --p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(at + p * plane);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += static_cast<float>(a[i]);
  }
}
// a lane's four values of a result tile into row-major LDS planes
template <int N>
__device__ __forceinline__ void put_four(bf16* at, int plane, const float (&x)[4]) {
  bf16 t[4][N];
#pragma unroll
  for (int i = 0; i < 4; ++i) split<N>(x[i], t[i]);
#pragma unroll
  for (int p = 0; p < N; ++p) *reinterpret_cast<bf16x4*>(at + p * plane) = bf16x4{t[0][p], t[1][p], t[2][p], t[3][p]};
}

// ------------------------------------------------------------------ rows from memory to LDS
template <typename T>
struct Eight {  // neighbouring values of a row as they are in memory
  T x[8] __attribute__((aligned(16)));
};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* row, int c, int D, bool vec) {
  Eight<T> e;
  u32x4* w = reinterpret_cast<u32x4*>(&e);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = u32x4{0, 0, 0, 0};
  if (vec) {
    if (c < D) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = reinterpret_cast<const u32x4*>(row + c)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < D) e.x[i] = row[c + i];
  }
  return e;
}

// The rows of one tensor of a chunk, held by a block's threads: C rows of W columns
template <typename T, int C, int W, int THREADS>
struct Stage {
  static constexpr int N = (C * W / 8 + THREADS - 1) / THREADS, PER = W / 8;
  static constexpr bool WHOLE = C * W % (8 * THREADS) == 0;  // else some threads have a group less
  Eight<T> e[N];
  // rows t0 .. t0 + n - 1 of the tensor; the others are zero
  __device__ __forceinline__ void load(const T* base, int64_t stride, int t0, int n, int c0, int D, bool vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * THREADS, r = at / PER, c = at % PER * 8;
      if (r < n)
        e[i] = load_eight<T>(base + (t0 + r) * stride + c0, c, D - c0, vec);
      else {
        u32x4* w = reinterpret_cast<u32x4*>(&e[i]);
        for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) w[k] = u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void store(bf16* s, int stride, int plane) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * THREADS, r = at / PER, c = at % PER * 8;
      if (!WHOLE && r >= C) continue;
      bf16* to = s + r * stride + c;
      if constexpr (std::is_same<T, bf16>::value) {
        *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(&e[i]);
      } else {
        Frag<Traits<T>::planes> f;
#pragma unroll
        for (int k = 0; k < 8; ++k) put(f, k, to_f32(e[i].x[k]));
#pragma unroll
        for (int p = 0; p < Traits<T>::planes; ++p) *reinterpret_cast<bf16x8*>(to + p * plane) = f.p[p];
      }
    }
  }
};

// What a chunk's decays give: sums (in powers of two), e^{G[i]} scale, e^{G[n] - G[j]}
template <int C>
struct Decays {
  float hi[C], lo[C], from[C], left[C];
  float whole;     // e^{G[n]}
  Sum total;
  float pad;
};
// by one whole wave; g: this lane's token's log decay (0 behind the sequence's end)
template <int C>
__device__ __forceinline__ void decays(Decays<C>& d, float g, float scale) {
  const int lane = threadIdx.x & 63;
  const Sum s = scan_sum(log2_decay(g), lane);
  const Sum t{__shfl(s.hi, C - 1, 64), __shfl(s.lo, C - 1, 64)};
  if (lane < C) {
    d.hi[lane] = s.hi, d.lo[lane] = s.lo;
    d.from[lane] = __builtin_amdgcn_exp2f(s.hi + s.lo) * scale;
    d.left[lane] = exp2_gap(t.hi, t.lo, s.hi, s.lo);
  }
  if (lane == 0) d.whole = __builtin_amdgcn_exp2f(t.hi + t.lo), d.total = t;
}
__device__ __forceinline__ float load_decay(const Args& a, const Unit& u, int t0, int n) {
  const int lane = threadIdx.x & 63;
  return lane < n ? a.g[u.b * a.gb + (t0 + lane) * a.gt + u.h] : 0.f;
}

// four neighbouring values of a row of an output, as far as it goes
template <typename T>
__device__ __forceinline__ void store_four(T* at, int left, bool vec, const float (&x)[4]) {
  if (vec && left >= 4) {
    struct alignas(4 * sizeof(T)) Four {
      T x[4];
    };
    Four f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.x[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Four*>(at) = f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) at[i] = from_f32<T>(x[i]);
  }
}

// ------------------------------------------------------------------ a state in a wave's registers
// Tile t holds rows 16 t + 4 g + 0..3 (keys) of column c0 + l % 16 (values) of a [K, V] matrix
template <int TK>
__device__ __forceinline__ void load_state(f32x4 (&s)[TK], const float* m, int K, int V, int c0) {
  const int lane = threadIdx.x & 63, c = c0 + (lane & 15), r0 = 4 * (lane >> 4);
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + r0 + i;
      s[t][i] = r < K && c < V ? m[r * V + c] : 0.f;
    }
}
template <int TK>
__device__ __forceinline__ void store_state(const f32x4 (&s)[TK], float* m, int K, int V, int c0) {
  const int lane = threadIdx.x & 63, c = c0 + (lane & 15), r0 = 4 * (lane >> 4);
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + r0 + i;
      if (r < K && c < V) m[r * V + c] = s[t][i];
    }
}

// S <- whole S + X^T (f Y): rows of X (sX, keys) and Y (sY, values) of a chunk, f a factor a row.  The scaled operand is
// fp32 in three parts: the states are the results that stay in fp32.
template <int C, int TK, int NX>
__device__ __forceinline__ void update_state(f32x4 (&s)[TK], const bf16* sX, int xstride, int xplane, const Frag<NX> (&y)[C / 32],
                                             const float* f, float whole) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < TK; ++t) s[t] *= whole;
#pragma unroll
  for (int st = 0; st < C / 32; ++st) {
    Frag<3> fy;
#pragma unroll
    for (int i = 0; i < 8; ++i) put(fy, i, value(y[st], i) * f[32 * st + (i < 4 ? 0 : 16) + 4 * g + (i & 3)]);
#pragma unroll
    for (int t = 0; t < TK; ++t) mma<3>(s[t], by_col<NX>(sX, xstride, xplane, 32 * st, 16 * t), fy);
  }
}

// ------------------------------------------------------------------ forward
template <typename T, int DK, int NW>
struct FwdLds {
  using Tr = Traits<T>;
  static constexpr int C = Tr::chunk, KS = DK + PAD, VS = 16 * NW + PAD, PS = C + PAD;
  bf16 q[Tr::planes][C][KS];
  bf16 k[Tr::planes][C][KS];
  bf16 v[Tr::planes][C][VS];
  bf16 p[Tr::prec][C][PS];
  Decays<C> d[2];
};

// A block of NW waves takes a head's 16 NW value columns over a segment of chunks; a wave holds 16 columns of the
// state.  ENDS: only what the segment adds to the state, into seg_state, with its decay.
template <typename T, int DK, int NW, bool ENDS>
__global__ __launch_bounds__(64 * NW) void k_la_fwd(Args a) {
  using L = FwdLds<T, DK, NW>;
  using Tr = Traits<T>;
  constexpr int C = L::C, TK = DK / 16, TI = C / 16, NP = Tr::planes, PR = Tr::prec, THREADS = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  L& lds = *reinterpret_cast<L*>(lds_raw);
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Unit u = unit_of(a, ENDS ? a.segs - 1 : a.segs, 0);
  const int c_first = u.seg * a.seg_chunks, c_last = min(c_first + a.seg_chunks, a.chunks);
  const int v0 = u.vt * VT, vc = v0 + 16 * w;  // the block's and the wave's first column
  const int64_t bh = u.b * a.H + u.h;
  const int64_t KV = int64_t{a.K} * a.V;
  const T* q = static_cast<const T*>(a.q) + u.b * a.qb + u.h / (a.H / a.Hq) * a.qh;
  const T* k = static_cast<const T*>(a.k) + u.b * a.kb + u.h / (a.H / a.Hk) * a.kh;
  const T* v = static_cast<const T*>(a.v) + u.b * a.vb + u.h / (a.H / a.Hv) * a.vh;
  T* y = static_cast<T*>(a.y) + (u.b * a.T * a.H + u.h) * a.V;

  f32x4 s[TK];
  if (!ENDS && a.segs > 1)
    load_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
  else if (!ENDS && a.start)
    load_state(s, a.start + bh * KV, a.K, a.V, vc);
  else
    for (int t = 0; t < TK; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  Stage<T, C, DK, THREADS> rq, rk;
  Stage<T, C, 16 * NW, THREADS> rv;
  float rg = 0.f;
  auto fetch = [&](int c) {
    const int t0 = c * C, n = min(C, u.len - t0);
    if (!ENDS) rq.load(q, a.qt, t0, n, 0, a.K, a.qvec);
    rk.load(k, a.kt, t0, n, 0, a.K, a.kvec);
    rv.load(v, a.vt, t0, n, v0, a.V, a.vvec);
    if (w == 0) rg = load_decay(a, u, t0, n);
  };
  const int c_end = min(c_last, (u.len + C - 1) / C);  // chunks with tokens
  if (c_first < c_end) {
    fetch(c_first);
    if (!ENDS)  // the tiles above the diagonal stay zero
      for (int i = threadIdx.x; i < static_cast<int>(sizeof(lds.p) / 16); i += THREADS)
        reinterpret_cast<u32x4*>(&lds.p)[i] = u32x4{0, 0, 0, 0};
    if (w == 0) decays(lds.d[c_first & 1], rg, a.scale);
  }
  Sum seg{0.f, 0.f};
  for (int c = c_first; c < c_end; ++c) {
    const int t0 = c * C, n = min(C, u.len - t0);
    const Decays<C>& d = lds.d[c & 1];
    if (!ENDS) rq.store(&lds.q[0][0][0], L::KS, C * L::KS);
    rk.store(&lds.k[0][0][0], L::KS, C * L::KS);
    rv.store(&lds.v[0][0][0], L::VS, C * L::VS);
    __syncthreads();
    if (c + 1 < c_end) fetch(c + 1);
    if (!ENDS && a.ckpt) store_state(s, a.ckpt + (bh * a.chunks + c) * KV, a.K, a.V, vc);

    const int tiles = (n + 15) / 16;
    if (!ENDS) {
      // the scores' tiles on and below the diagonal, transposed: column i, rows j
      for (int idx = w; idx < tiles * (tiles + 1) / 2; idx += NW) {
        const int it = idx >= 6 ? 3 : idx >= 3 ? 2 : idx >= 1 ? 1 : 0, jt = idx - it * (it + 1) / 2;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st)
          mma<3>(acc, by_row<NP>(&lds.k[0][0][0], L::KS, C * L::KS, 16 * jt, 32 * st),
                 by_row<NP>(&lds.q[0][0][0], L::KS, C * L::KS, 16 * it, 32 * st));
        const int i = 16 * it + li, j0 = 16 * jt + 4 * lg;
        const f32x4 jh = *reinterpret_cast<const f32x4*>(&d.hi[j0]), jl = *reinterpret_cast<const f32x4*>(&d.lo[j0]);
        const float ih = d.hi[i], il = d.lo[i];
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          p[r] = j0 + r <= i ? acc[r] * exp2_gap(ih, il, jh[r], jl[r]) * a.scale : 0.f;
        put_four<PR>(&lds.p[0][i][j0], C * L::PS, p);
      }
      __syncthreads();
    }
    if (w == 0 && c + 1 < c_end) decays(lds.d[(c + 1) & 1], rg, a.scale);

    Frag<NP> fv[C / 32];
    float odd = 0.f;
#pragma unroll
    for (int st = 0; st < C / 32; ++st) {
      fv[st] = by_col<NP>(&lds.v[0][0][0], L::VS, C * L::VS, 32 * st, 16 * w);
#pragma unroll
      for (int i = 0; i < 8; ++i) odd = fmaf(static_cast<float>(fv[st].p[0][i]), 0.f, odd);
    }
    if (!ENDS) {
      // an infinity or NaN among the values may not reach the tokens before it, with a weight of zero
      const bool careful = __ballot(!(odd == 0.f)) != 0ull;
      Frag<PR> fs[DK / 32];
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) put(fs[t / 2], 4 * (t & 1) + r, s[t][r]);
#pragma unroll
      for (int it = 0; it < TI; ++it) {
        if (it >= tiles) break;
        const int i = 16 * it + li;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st)
          mma<PR>(acc, fs[st], by_row<NP>(&lds.q[0][0][0], L::KS, C * L::KS, 16 * it, 32 * st));
        acc *= d.from[i];
        if (!careful) {
#pragma unroll
          for (int st = 0; st <= it / 2; ++st)
            mma<PR>(acc, fv[st], by_row<PR>(&lds.p[0][0][0], L::PS, C * L::PS, 16 * it, 32 * st));
        } else {
          for (int j = 0; j <= i; ++j) {
            float p = 0.f, x[4];
            for (int b = PR - 1; b >= 0; --b) p += static_cast<float>(lds.p[b][i][j]);
            four<NP>(&lds.v[0][j][16 * w + 4 * lg], C * L::VS, x);
            for (int r = 0; r < 4; ++r) acc[r] = fmaf(p, x[r], acc[r]);
          }
        }
        const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
        const int col = vc + 4 * lg;
        if (i < n) store_four(y + int64_t{t0 + i} * a.H * a.V + col, a.V - col, a.yvec, out);
      }
    }
    update_state<C, TK, NP>(s, &lds.k[0][0][0], L::KS, C * L::KS, fv, d.left, d.whole);
    if (ENDS && threadIdx.x == 0) seg = add(seg, d.total);
    __syncthreads();
  }
  if (ENDS) {
    store_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
    if (threadIdx.x == 0 && u.vt == 0) a.seg_decay[bh * a.segs + u.seg] = seg.hi + seg.lo;
    return;
  }
  // positions behind the sequence's end
  const int from = max(u.len, c_first * C), to = static_cast<int>(min(static_cast<int64_t>(c_last) * C, a.T));
  const int cols = min(16 * NW, a.V - v0);
  for (int64_t i = threadIdx.x; i < int64_t{to - from} * cols; i += THREADS)
    y[(from + i / cols) * a.H * a.V + v0 + i % cols] = from_f32<T>(0.f);
  if (a.end && u.seg == a.segs - 1) store_state(s, a.end + bh * KV, a.K, a.V, vc);
}

// Segments one after the other: what each adds becomes the state before it (BACK: the gradient of the state behind it)
template <bool BACK>
__global__ __launch_bounds__(256) void k_la_join(Args a) {
  const int64_t KV = int64_t{a.K} * a.V;
  const int64_t blocks = (KV + 255) / 256;
  const int64_t bh = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
  if (e >= KV) return;
  const float* from = BACK ? a.dend : a.start;
  float s = from ? from[bh * KV + e] : 0.f;
  for (int i = 0; i < a.segs; ++i) {
    const int seg = BACK ? a.segs - 1 - i : i;
    float* at = a.seg_state + (bh * a.segs + seg) * KV + e;
    const float add = i + 1 < a.segs ? *at : 0.f;
    *at = s;
    if (i + 1 < a.segs) s = fmaf(s, __builtin_amdgcn_exp2f(a.seg_decay[bh * a.segs + seg]), add);
  }
}

// ------------------------------------------------------------------ backward
//
// With R = dL/dS behind the chunk, P[i,j] = scale e^{G[i]-G[j]} (q[i].k[j]), A[i,j] = scale e^{G[i]-G[j]} (dy[i].v[j]):
//
//   dq[i] = sum_{j <= i} A[i,j] k[j] + scale e^{G[i]} S_in dy[i]
//   dk[j] = sum_{i >= j} A[i,j] q[i] + e^{G[n]-G[j]} R v[j]
//   dv[j] = sum_{i >= j} P[i,j] dy[i] + e^{G[n]-G[j]} R^T k[j]
//   R_in  = e^{G[n]} R + scale sum_i e^{G[i]} q[i] dy[i]^T
//   dg[t] = sum_{j < t <= i} P[i,j] (dy[i].v[j]) + sum_{i >= t} q[i].(scale e^{G[i]} S_in dy[i])
//           + sum_{j < t} v[j].(e^{G[n]-G[j]} R^T k[j]) + e^{G[n]} <S_in, R>
//
// A decay's gradient is every pair and every state that it stands between.  The shorter form, the sum behind t of
// q.dq - k.dk, takes large terms from each other along the whole sequence; this one only within a chunk.
//
// One pass from the last chunk to the first reads q, k, v and dy once, and the states before the chunks, which the
// forward pass kept.  Everything is linear in the value columns: a block takes up to 64 of them, and dq, dk and dg of
// several such tiles are summed afterwards, as the gradients of shared heads are.
template <typename T, int DK>
struct BwdLds {
  using Tr = Traits<T>;
  static constexpr int C = Tr::chunk, KS = DK + PAD, VS = VT + PAD, PS = C + PAD, NR = Tr::planes > 2 ? 3 : 2;
  bf16 q[Tr::planes][C][KS];
  bf16 k[Tr::planes][C][KS];
  bf16 v[Tr::planes][C][VS];
  bf16 o[Tr::planes][C][VS];  // dy
  bf16 p[Tr::prec][C][PS];
  bf16 a[Tr::prec][C][PS];
  bf16 r[NR][DK][VS];
  Decays<C> d[2];
  float row[C / 16][C];       // sums over a tile's j of P (dy.v), below the diagonal
  float col[C / 16][C];       // over its i
  float qs[DK / 16][C];       // q[i].(scale e^{G[i]} S_in dy[i]) over 16 keys
  float kr[4][C];             // v[j].(e^{G[n]-G[j]} R^T k[j]) over a wave's columns
  float sr[4];                // a wave's share of <S_in, R>
};

constexpr int BW = 4, BTHREADS = 64 * BW;  // waves and threads of a backward block

// Sum over the 16 lanes of a row of the wave, in all of them
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = 1; m < 16; m *= 2) v += __shfl_xor(v, m, 64);
  return v;
}

// What the columns v0 .. v0 + 63 of the values add to the gradients; ENDS: only what the segment adds to the state's
// gradient.
template <typename T, int DK, bool ENDS>
__global__ __launch_bounds__(BTHREADS) void k_la_bwd(Args a) {
  using L = BwdLds<T, DK>;
  using Tr = Traits<T>;
  constexpr int C = L::C, TK = DK / 16, TI = C / 16, NP = Tr::planes, PR = Tr::prec, NR = L::NR;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  L& lds = *reinterpret_cast<L*>(lds_raw);
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Unit u = unit_of(a, ENDS ? a.segs - 1 : a.segs, ENDS ? 1 : 0);
  const int c_first = u.seg * a.seg_chunks, c_last = min(c_first + a.seg_chunks, a.chunks);
  const int v0 = u.vt * VT, vc = v0 + 16 * w;
  const int64_t bh = u.b * a.H + u.h;
  const int64_t KV = int64_t{a.K} * a.V;
  const T* q = static_cast<const T*>(a.q) + u.b * a.qb + u.h / (a.H / a.Hq) * a.qh;
  const T* k = static_cast<const T*>(a.k) + u.b * a.kb + u.h / (a.H / a.Hk) * a.kh;
  const T* v = static_cast<const T*>(a.v) + u.b * a.vb + u.h / (a.H / a.Hv) * a.vh;
  const T* dy = static_cast<const T*>(a.dy) + u.b * a.yb + u.h * a.yh;
  const int hv = u.h * a.vts + u.vt;  // of the heads' value tiles

  f32x4 s[TK];  // R: rows of keys, this wave's 16 columns
  if (!ENDS && a.segs > 1)
    load_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
  else if (!ENDS && a.dend)
    load_state(s, a.dend + bh * KV, a.K, a.V, vc);
  else
    for (int t = 0; t < TK; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  Stage<T, C, DK, BTHREADS> rq, rk;
  Stage<T, C, VT, BTHREADS> rv, ro;
  float rg = 0.f;
  auto fetch = [&](int c) {
    const int t0 = c * C, n = min(C, u.len - t0);
    rq.load(q, a.qt, t0, n, 0, a.K, a.qvec);
    ro.load(dy, a.yt, t0, n, v0, a.V, a.yvec);
    if (!ENDS) {
      rk.load(k, a.kt, t0, n, 0, a.K, a.kvec);
      rv.load(v, a.vt, t0, n, v0, a.V, a.vvec);
    }
    if (w == 0) rg = load_decay(a, u, t0, n);
  };
  const int c_end = min(c_last, (u.len + C - 1) / C);  // chunks with tokens
  if (c_first < c_end) {
    fetch(c_end - 1);
    if (!ENDS)  // the tiles above the diagonal stay zero
      for (int i = threadIdx.x; i < static_cast<int>((sizeof(lds.p) + sizeof(lds.a)) / 16); i += BTHREADS)
        reinterpret_cast<u32x4*>(&lds.p)[i] = u32x4{0, 0, 0, 0};
    if (w == 0) decays(lds.d[(c_end - 1) & 1], rg, a.scale);
  }
  Sum seg{0.f, 0.f};
  for (int c = c_end - 1; c >= c_first; --c) {
    const int t0 = c * C, n = min(C, u.len - t0), tiles = (n + 15) / 16;
    const Decays<C>& d = lds.d[c & 1];
    rq.store(&lds.q[0][0][0], L::KS, C * L::KS);
    ro.store(&lds.o[0][0][0], L::VS, C * L::VS);
    if (!ENDS) {
      rk.store(&lds.k[0][0][0], L::KS, C * L::KS);
      rv.store(&lds.v[0][0][0], L::VS, C * L::VS);
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bf16 x[NR];
          split<NR>(s[t][r], x);
#pragma unroll
          for (int b = 0; b < NR; ++b) lds.r[b][16 * t + 4 * lg + r][16 * w + li] = x[b];
        }
    }
    __syncthreads();
    if (c > c_first) fetch(c - 1);

    if (!ENDS) {
      for (int idx = w; idx < tiles * (tiles + 1) / 2; idx += BW) {
        const int it = idx >= 6 ? 3 : idx >= 3 ? 2 : idx >= 1 ? 1 : 0, jt = idx - it * (it + 1) / 2;
        f32x4 qk{0.f, 0.f, 0.f, 0.f}, ov{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st)
          mma<3>(qk, by_row<NP>(&lds.k[0][0][0], L::KS, C * L::KS, 16 * jt, 32 * st),
                 by_row<NP>(&lds.q[0][0][0], L::KS, C * L::KS, 16 * it, 32 * st));
#pragma unroll
        for (int st = 0; st < VT / 32; ++st)
          mma<3>(ov, by_row<NP>(&lds.v[0][0][0], L::VS, C * L::VS, 16 * jt, 32 * st),
                 by_row<NP>(&lds.o[0][0][0], L::VS, C * L::VS, 16 * it, 32 * st));
        const int i = 16 * it + li, j0 = 16 * jt + 4 * lg;
        const f32x4 jh = *reinterpret_cast<const f32x4*>(&d.hi[j0]), jl = *reinterpret_cast<const f32x4*>(&d.lo[j0]);
        const float ih = d.hi[i], il = d.lo[i];
        float p[4], x[4], pair[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float dec = exp2_gap(ih, il, jh[r], jl[r]) * a.scale;
          p[r] = j0 + r <= i ? qk[r] * dec : 0.f;
          x[r] = j0 + r <= i ? ov[r] * dec : 0.f;
          pair[r] = j0 + r < i ? p[r] * ov[r] : 0.f;
        }
        put_four<PR>(&lds.p[0][i][j0], C * L::PS, p);
        put_four<PR>(&lds.a[0][i][j0], C * L::PS, x);
        float rows = (pair[0] + pair[1]) + (pair[2] + pair[3]);
        rows += __shfl_xor(rows, 16, 64);
        rows += __shfl_xor(rows, 32, 64);
        if (lg == 0) lds.row[jt][i] = rows;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float cols = row_sum(pair[r]);
          if (li == 0) lds.col[it][j0 + r] = cols;
        }
      }
      __syncthreads();
    }
    if (w == 0 && c > c_first) decays(lds.d[(c - 1) & 1], rg, a.scale);

    if (!ENDS) {
      // dq and dk: tiles of 16 keys and 16 tokens, a wave's share of the keys (of the tokens, where keys are few)
      constexpr int SHARE = TK >= BW ? 1 : BW / TK, KT = TK >= BW ? TK / BW : 1, IT = TI / SHARE > 0 ? TI / SHARE : 1;
      const float* s_in = a.ckpt + (bh * a.chunks + c) * KV;
      const int part = w % SHARE;
#pragma unroll 1
      for (int kk = 0; kk < KT; ++kk) {
        const int kt = w / SHARE * KT + kk;
        if (part * IT >= tiles) break;
        Frag<3> fs[VT / 32];  // S_in, rows of keys, index of values
        const int row = 16 * kt + li;
#pragma unroll
        for (int st = 0; st < VT / 32; ++st)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int col = v0 + 32 * st + (i < 4 ? 0 : 16) + 4 * lg + (i & 3);
            put(fs[st], i, row < a.K && col < a.V ? s_in[row * a.V + col] : 0.f);
          }
        Frag<NR> fr[VT / 32];
#pragma unroll
        for (int st = 0; st < VT / 32; ++st) fr[st] = by_row<NR>(&lds.r[0][0][0], L::VS, DK * L::VS, 16 * kt, 32 * st);
        for (int ii = 0; ii < IT; ++ii) {
          const int it = part * IT + ii;
          if (it >= tiles) break;
          const int i = 16 * it + li, key = 16 * kt + 4 * lg;
          f32x4 acc{0.f, 0.f, 0.f, 0.f};
          float x[4], sum = 0.f;
#pragma unroll
          for (int st = 0; st < VT / 32; ++st)
            mma<3>(acc, fs[st], by_row<NP>(&lds.o[0][0][0], L::VS, C * L::VS, 16 * it, 32 * st));
          acc *= d.from[i];
          four<NP>(&lds.q[0][i][key], C * L::KS, x);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum = fmaf(x[r], acc[r], sum);
          sum += __shfl_xor(sum, 16, 64);
          sum += __shfl_xor(sum, 32, 64);
          if (lg == 0) lds.qs[kt][i] = sum;
          for (int st = 0; st <= it / 2; ++st)
            mma<PR>(acc, by_col<NP>(&lds.k[0][0][0], L::KS, C * L::KS, 32 * st, 16 * kt),
                    by_row<PR>(&lds.a[0][0][0], L::PS, C * L::PS, 16 * it, 32 * st));
          const int64_t token = u.b * a.T + t0 + i;
          if (i < n) {
            const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
            if (a.dq32)
              store_four(static_cast<float*>(a.dq) + (token * a.H * a.vts + hv) * a.K + key, a.K - key, a.K % 4 == 0, out);
            else
              store_four(static_cast<T*>(a.dq) + (token * a.H + u.h) * a.K + key, a.K - key, a.K % 4 == 0, out);
          }
          acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < VT / 32; ++st)
            mma<NR>(acc, fr[st], by_row<NP>(&lds.v[0][0][0], L::VS, C * L::VS, 16 * it, 32 * st));
          acc *= d.left[i];
          for (int st = it / 2; st < C / 32; ++st)
            mma<PR>(acc, by_col<NP>(&lds.q[0][0][0], L::KS, C * L::KS, 32 * st, 16 * kt),
                    by_col<PR>(&lds.a[0][0][0], L::PS, C * L::PS, 32 * st, 16 * it));
          if (i < n) {
            const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
            if (a.dk32)
              store_four(static_cast<float*>(a.dk) + (token * a.H * a.vts + hv) * a.K + key, a.K - key, a.K % 4 == 0, out);
            else
              store_four(static_cast<T*>(a.dk) + (token * a.H + u.h) * a.K + key, a.K - key, a.K % 4 == 0, out);
          }
        }
      }
    }
    Frag<NP> fo[C / 32];
#pragma unroll
    for (int st = 0; st < C / 32; ++st) fo[st] = by_col<NP>(&lds.o[0][0][0], L::VS, C * L::VS, 32 * st, 16 * w);
    if (!ENDS) {
      // dv: this wave's 16 columns
      Frag<3> fs[DK / 32];
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) put(fs[t / 2], 4 * (t & 1) + r, s[t][r]);
#pragma unroll
      for (int jt = 0; jt < TI; ++jt) {
        if (jt >= tiles) break;
        const int j = 16 * jt + li;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st)
          mma<3>(acc, fs[st], by_row<NP>(&lds.k[0][0][0], L::KS, C * L::KS, 16 * jt, 32 * st));
        acc *= d.left[j];
        float x[4], sum = 0.f;
        four<NP>(&lds.v[0][j][16 * w + 4 * lg], C * L::VS, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) sum = fmaf(x[r], acc[r], sum);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lg == 0) lds.kr[w][j] = sum;
#pragma unroll
        for (int st = jt / 2; st < C / 32; ++st)
          mma<PR>(acc, fo[st], by_col<PR>(&lds.p[0][0][0], L::PS, C * L::PS, 32 * st, 16 * jt));
        if (j < n) {
          const float out[4] = {acc[0], acc[1], acc[2], acc[3]};
          const int col = vc + 4 * lg;
          const int64_t token = u.b * a.T + t0 + j;
          if (a.dv32)
            store_four(static_cast<float*>(a.dv) + (token * a.H + u.h) * a.V + col, a.V - col, a.V % 4 == 0, out);
          else
            store_four(static_cast<T*>(a.dv) + (token * a.H + u.h) * a.V + col, a.V - col, a.V % 4 == 0, out);
        }
      }
      // <S_in, R> over this wave's columns
      const float* s_in = a.ckpt + (bh * a.chunks + c) * KV;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * t + 4 * lg + r, col = vc + li;
          if (row < a.K && col < a.V) sum = fmaf(s_in[row * a.V + col], s[t][r], sum);
        }
      sum = wave_sum(sum);
      if (lane == 0) lds.sr[w] = sum;
    }
    update_state<C, TK, NP>(s, &lds.q[0][0][0], L::KS, C * L::KS, fo, d.from, d.whole);
    if (ENDS && threadIdx.x == 0) seg = add(seg, d.total);
    __syncthreads();
    if (!ENDS && w == BW - 1) {
      // the decays' gradients: a lane a token
      double later = 0., kept = 0.;  // what is summed from t on, and before t
      if (lane < n) {
        for (int t = 0; t <= lane / 16; ++t) later += lds.row[t][lane];
        for (int t = lane / 16; t < tiles; ++t) later -= lds.col[t][lane];
        for (int t = 0; t < TK; ++t) later += lds.qs[t][lane];
        for (int t = 0; t < BW; ++t) kept += lds.kr[t][lane];
      }
      double total = kept;
#pragma unroll
      for (int off = 1; off < 64; off *= 2) {
        const double x = __shfl_down(later, off, 64), y = __shfl_up(total, off, 64);
        if (lane + off < 64) later += x;
        if (lane >= off) total += y;
      }
      if (lane < n)
        a.dg[(u.b * a.T + t0 + lane) * a.H * a.vts + hv] = static_cast<float>(
            later + (total - kept) + double(d.whole) * ((double(lds.sr[0]) + lds.sr[1]) + (double(lds.sr[2]) + lds.sr[3])));
    }
  }
  if (ENDS) {
    store_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
    if (threadIdx.x == 0 && u.vt == 0) a.seg_decay[bh * a.segs + u.seg] = seg.hi + seg.lo;
    return;
  }
  // positions behind the sequence's end
  const int from = max(u.len, c_first * C), to = static_cast<int>(min(static_cast<int64_t>(c_last) * C, a.T));
  const int cols = min(VT, a.V - v0);
  auto clear = [&](void* out, bool f32, int64_t head, int64_t heads, int d, int c0, int width) {
    for (int64_t i = threadIdx.x; i < int64_t{to - from} * width; i += BTHREADS) {
      const int64_t at = ((u.b * a.T + from + i / width) * heads + head) * d + c0 + i % width;
      if (f32)
        static_cast<float*>(out)[at] = 0.f;
      else
        static_cast<T*>(out)[at] = from_f32<T>(0.f);
    }
  };
  clear(a.dq, a.dq32, a.dq32 ? hv : u.h, a.dq32 ? a.H * a.vts : a.H, a.K, 0, a.K);
  clear(a.dk, a.dk32, a.dk32 ? hv : u.h, a.dk32 ? a.H * a.vts : a.H, a.K, 0, a.K);
  clear(a.dv, a.dv32, u.h, a.H, a.V, v0, cols);
  clear(a.dg, true, hv, a.H * a.vts, 1, 0, 1);
  if (a.dstart && u.seg == 0) store_state(s, a.dstart + bh * KV, a.K, a.V, vc);
}

// Sums of `share` neighbouring rows of d values: [rows, share, d] in fp32 -> [rows, d]
template <typename T>
__global__ __launch_bounds__(256) void k_la_shared(const float* part, int64_t n, int share, int d, T* out) {
  const int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x;
  if (i >= n) return;
  const float* p = part + i / d * share * d + i % d;
  float s = 0.f;
  for (int k = 0; k < share; ++k) s += p[int64_t{k} * d];
  out[i] = from_f32<T>(s);
}

// Column sums of [rows, cols] in two steps: blocks over ranges of rows, then a thread a head over the blocks' sums and
// its `share` neighbouring columns.
__global__ __launch_bounds__(256) void k_la_columns(const float* x, int64_t rows, int cols, int64_t per, float* out) {
  __shared__ double part[4][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r0 = blockIdx.x * per, r1 = min(rows, r0 + per);
  for (int c0 = 0; c0 < cols; c0 += 64) {
    double s = 0.;
    if (c0 + lane < cols)
      for (int64_t r = r0 + w; r < r1; r += 4) s += x[r * cols + c0 + lane];
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && c0 + lane < cols)
      out[int64_t{blockIdx.x} * cols + c0 + lane] =
          static_cast<float>((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
    __syncthreads();
  }
}
__global__ __launch_bounds__(64) void k_la_column_ends(const float* part, int blocks, int heads, int share, float* out) {
  const int h = blockIdx.x;
  double s = 0.;
  for (int i = threadIdx.x; i < blocks * share; i += 64)
    s += part[int64_t{i / share} * heads * share + h * share + i % share];
#pragma unroll
  for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m, 64);
  if (threadIdx.x == 0) out[h] = static_cast<float>(s);
}

// ------------------------------------------------------------------ one token
// A wave takes 64 value columns of a head: lane l four of them, and of the keys every fourth part.  All of a lane's
// state is asked for at once; the state is read and written where it stands, so that it may move on in place.
template <typename T, int NB, bool VEC>
__global__ __launch_bounds__(256) void k_la_step(Args a, int64_t waves) {
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int64_t u = int64_t{blockIdx.x} * 4 + (threadIdx.x >> 6);
  if (u >= waves) return;
  const int64_t bh = u / a.vts, b = bh / a.H;
  const int h = static_cast<int>(bh % a.H), c = static_cast<int>(u % a.vts) * VT + 4 * li, r0 = 8 * NB * lg;
  const float* from = a.start + bh * a.K * a.V;
  float* to = a.end + bh * a.K * a.V;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h / (a.H / a.Hq) * a.qh;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + h / (a.H / a.Hk) * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + h / (a.H / a.Hv) * a.vh;
  f32x4 s[8 * NB];
  Eight<T> ek[NB], eq[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    ek[n] = load_eight<T>(k, r0 + 8 * n, a.K, a.kvec);
    eq[n] = load_eight<T>(q, r0 + 8 * n, a.K, a.qvec);
  }
  float g = a.g[b * a.gb + h], vv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vv[i] = c + i < a.V ? to_f32(v[c + i]) : 0.f;
#pragma unroll
  for (int n = 0; n < 8 * NB; ++n) {
    const int r = r0 + n;
    s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < a.K) {
      if constexpr (VEC) {
        if (c < a.V) s[n] = *reinterpret_cast<const f32x4*>(from + r * a.V + c);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < a.V) s[n][i] = from[r * a.V + c + i];
      }
    }
  }
  const Sum d = log2_decay(g);
  const float e = __builtin_amdgcn_exp2f(d.hi), decay = fmaf(e, d.lo * 0.69314718f, e);
  f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < 8 * NB; ++n) {
    const float kk = to_f32(ek[n / 8].x[n % 8]), qq = to_f32(eq[n / 8].x[n % 8]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[n][i] = fmaf(decay, s[n][i], kk * vv[i]);
      y[i] = fmaf(qq, s[n][i], y[i]);
    }
    const int r = r0 + n;
    if (r < a.K) {
      if constexpr (VEC) {
        if (c < a.V) *reinterpret_cast<f32x4*>(to + r * a.V + c) = s[n];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < a.V) to[r * a.V + c + i] = s[n][i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] += __shfl_xor(y[i], 16, 64);
    y[i] += __shfl_xor(y[i], 32, 64);
  }
  const float out[4] = {y[0] * a.scale, y[1] * a.scale, y[2] * a.scale, y[3] * a.scale};
  if (lg == 0) store_four(static_cast<T*>(a.y) + bh * a.V + c, a.V - c, VEC, out);
}

// ------------------------------------------------------------------ host
int chunk_of(int dtype) { return dtype == LNG_BF16 ? Traits<bf16>::chunk : Traits<float>::chunk; }

bool vector_rows(const void* p, int es, int64_t batch, int64_t token, int64_t head, int d) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && batch * es % 16 == 0 && token * es % 16 == 0 && head * es % 16 == 0 &&
         d % 8 == 0;
}

// Blocks that a launch should have: a segment more costs the keys and values (the queries and dy) of all but one
// segment a second time.
constexpr int64_t FWD_BLOCKS = 1024, BWD_BLOCKS = 512;

Args make_args(const lng_linear_attention& l, bool grad) {
  Args a{};
  a.B = l.B, a.T = l.T, a.H = l.H, a.Hq = l.Hq, a.Hk = l.Hk, a.Hv = l.Hv, a.K = l.K, a.V = l.V, a.scale = l.scale;
  a.q = l.q, a.k = l.k, a.v = l.v;
  a.qb = l.q_batch, a.qt = l.q_token, a.qh = l.q_head, a.kb = l.k_batch, a.kt = l.k_token, a.kh = l.k_head;
  a.vb = l.v_batch, a.vt = l.v_token, a.vh = l.v_head;
  const int es = dtype_size(l.dtype);
  a.qvec = vector_rows(a.q, es, a.qb, a.qt, a.qh, a.K), a.kvec = vector_rows(a.k, es, a.kb, a.kt, a.kh, a.K);
  a.vvec = vector_rows(a.v, es, a.vb, a.vt, a.vh, a.V);
  a.g = l.decay, a.gb = l.decay_batch, a.gt = l.decay_token;
  a.start = l.state, a.lengths = l.lengths, a.y = l.y, a.end = l.state_out, a.ckpt = l.checkpoints;
  a.yvec = a.V % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * es) == 0;
  a.vts = static_cast<int>(cdiv(a.V, VT));
  a.chunks = static_cast<int>(cdiv(a.T, chunk_of(l.dtype)));
  const int64_t units = a.B * a.H * a.vts, want = grad ? BWD_BLOCKS : FWD_BLOCKS;
  int64_t segs = units * 2 > want ? 1 : std::min<int64_t>(cdiv(want, std::max<int64_t>(units, 1)), cdiv(a.chunks, 2));
  a.seg_chunks = static_cast<int>(cdiv(a.chunks, std::max<int64_t>(segs, 1)));
  a.segs = a.seg_chunks ? static_cast<int>(cdiv(a.chunks, a.seg_chunks)) : 1;
  return a;
}

// floats of the workspace
struct Space {
  int64_t seg_state = 0, seg_decay = 0, dq = 0, dk = 0, dv = 0, dg = 0, cols = 0, total = 0;
  int64_t col_blocks = 0;
  Space(const Args& a, bool grad, bool token_decay) {
    auto take = [&](int64_t n) {
      const int64_t at = total;
      total += cdiv(n, 16) * 16;
      return at;
    };
    if (a.segs > 1) seg_state = take(a.B * a.H * a.segs * a.K * a.V), seg_decay = take(a.B * a.H * a.segs);
    if (!grad) return;
    const int64_t rows = a.B * a.T, hv = int64_t{a.H} * a.vts;
    if (hv > a.Hq) dq = take(rows * hv * a.K);
    if (hv > a.Hk) dk = take(rows * hv * a.K);
    if (a.H > a.Hv) dv = take(rows * a.H * a.V);
    if (a.vts > 1 || !token_decay) dg = take(rows * hv);
    col_blocks = std::min<int64_t>(256, cdiv(rows, 64));
    if (!token_decay) cols = take(col_blocks * hv);
  }
};

int check_args(const char* what, const lng_linear_attention* l) {
  if (!l) return fail(LNG_E_ARG, std::string(what) + ": null arguments");
  if (l->dtype != LNG_F32 && l->dtype != LNG_BF16 && l->dtype != LNG_F16)
    return fail(LNG_E_DTYPE, std::string(what) + ": fp32, bf16 or fp16 tensors");
  if (l->K < 1 || l->K > MAX_D || l->V < 1 || l->V > MAX_D)
    return fail(LNG_E_ARG, std::string(what) + ": heads of 1 to 128 keys and values");
  if (l->H < 1 || l->H > (1 << 16) || l->Hq < 1 || l->Hk < 1 || l->Hv < 1 || l->H % l->Hq || l->H % l->Hk || l->H % l->Hv)
    return fail(LNG_E_ARG, std::string(what) + ": the heads of q, k and v divide those of the decays");
  if (l->B < 0 || l->T < 0 || l->B > (int64_t{1} << 24) || l->T > (int64_t{1} << 30) ||
      l->B * l->T > (int64_t{1} << 40) / l->H / MAX_D)
    return fail(LNG_E_ARG, std::string(what) + ": bad shape");
  if (l->B * l->T > 0 && (!l->q || !l->k || !l->v || !l->decay))
    return fail(LNG_E_ARG, std::string(what) + ": null pointer");
  return LNG_OK;
}

int check_threads(const char* what, int64_t blocks, int threads) {
  if (blocks * threads <= MOST_THREADS) return LNG_OK;
  return fail(LNG_E_ARG, std::string(what) + ": too many sequences, heads or tokens for one launch; split the batch");
}

template <typename F>
int launch(F* kernel, unsigned blocks, unsigned threads, size_t lds, hipStream_t st, const Args& a, const char* what) {
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return fail(LNG_E_HIP, std::string(what) + ": " + hipGetErrorString(e));
  }
  kernel<<<blocks, threads, lds, st>>>(a);
  return check_launch(what);
}

template <bool BACK>
int run_join(const Args& a, hipStream_t st) {
  k_la_join<BACK><<<static_cast<unsigned>(a.B * a.H * cdiv(int64_t{a.K} * a.V, 256)), 256, 0, st>>>(a);
  return check_launch("linear_attention");
}

template <typename T, int DK, int NW>
int run_fwd(const Args& a, hipStream_t st) {
  constexpr size_t lds = sizeof(FwdLds<T, DK, NW>);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  const int64_t units = a.B * a.H * a.vts;
  if (a.segs > 1) {
    if (int rc = launch(&k_la_fwd<T, DK, NW, true>, static_cast<unsigned>(units * (a.segs - 1)), 64 * NW, lds, st, a,
                        "linear_attention"))
      return rc;
    if (int rc = run_join<false>(a, st)) return rc;
  }
  return launch(&k_la_fwd<T, DK, NW, false>, static_cast<unsigned>(units * a.segs), 64 * NW, lds, st, a,
                "linear_attention");
}

template <typename T, int DK>
int run_bwd(const Args& a, hipStream_t st) {
  constexpr size_t lds = sizeof(BwdLds<T, DK>);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  const int64_t units = a.B * a.H * a.vts;
  if (a.segs > 1) {
    if (int rc = launch(&k_la_bwd<T, DK, true>, static_cast<unsigned>(units * (a.segs - 1)), BTHREADS, lds, st, a,
                        "linear_attention_grad"))
      return rc;
    if (int rc = run_join<true>(a, st)) return rc;
  }
  return launch(&k_la_bwd<T, DK, false>, static_cast<unsigned>(units * a.segs), BTHREADS, lds, st, a,
                "linear_attention_grad");
}

template <typename T>
int run_shared(const float* part, int64_t rows, int heads, int share, int d, T* out, hipStream_t st) {
  const int64_t n = rows * heads * d;
  if (int rc = check_threads("linear_attention_grad", cdiv(n, 256), 256)) return rc;
  k_la_shared<T><<<static_cast<unsigned>(cdiv(n, 256)), 256, 0, st>>>(part, n, share, d, out);
  return check_launch("linear_attention_grad");
}

template <typename F>
int with_type(int dtype, F f) {
  if (dtype == LNG_F32) return f(float{});
  if (dtype == LNG_BF16) return f(bf16{});
  return f(_Float16{});
}
template <typename F>
int with_keys(int K, F f) {
  if (K <= 32) return f(std::integral_constant<int, 32>{});
  if (K <= 64) return f(std::integral_constant<int, 64>{});
  return f(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace lng

using namespace lng;

extern "C" {

size_t lng_linear_attention_size(void) { return sizeof(lng_linear_attention); }
size_t lng_linear_attention_grad_size(void) { return sizeof(lng_linear_attention_grad); }

size_t lng_linear_attention_workspace_bytes(const lng_linear_attention* args, int grad) {
  if (check_args("linear_attention_workspace_bytes", args) || args->B == 0 || args->T == 0) return 0;
  const Args a = make_args(*args, grad != 0);
  return static_cast<size_t>(Space(a, grad != 0, args->token_decay != 0).total) * 4;
}

int64_t lng_linear_attention_checkpoints(int64_t B, int64_t T, int32_t H, int32_t K, int32_t V, int dtype) {
  if (B <= 0 || T <= 0 || H <= 0 || K <= 0 || V <= 0) return 0;
  return B * H * cdiv(T, chunk_of(dtype)) * K * V;
}

int lng_linear_attention_scan(const lng_linear_attention* args, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "linear_attention";
  if (int rc = check_args(what, args)) return rc;
  if (args->B == 0 || args->T == 0) return LNG_OK;
  if (!args->y) return fail(LNG_E_ARG, "linear_attention: null pointer");
  Args a = make_args(*args, false);
  const Space s(a, false, args->token_decay != 0);
  if (s.total && (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 ||
                  reinterpret_cast<uintptr_t>(workspace) % 64))
    return fail(LNG_E_ARG, "linear_attention: the workspace is too small or not 64-byte aligned");
  if (int rc = check_threads(what, a.B * a.H * std::max<int64_t>(a.vts * a.segs, cdiv(int64_t{a.K} * a.V, 256)), 256))
    return rc;
  float* const ws = static_cast<float*>(workspace);
  a.seg_state = ws + s.seg_state, a.seg_decay = ws + s.seg_decay;
  return with_type(args->dtype, [&](auto t) {
    return with_keys(a.K, [&](auto dk) {
      using T = decltype(t);
      constexpr int DK = decltype(dk)::value;
      return a.V <= 32 ? run_fwd<T, DK, 2>(a, as_stream(stream)) : run_fwd<T, DK, 4>(a, as_stream(stream));
    });
  });
}

int lng_linear_attention_scan_grad(const lng_linear_attention* args, const lng_linear_attention_grad* grads,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "linear_attention_grad";
  if (int rc = check_args(what, args)) return rc;
  if (!grads) return fail(LNG_E_ARG, "linear_attention_grad: null arguments");
  const lng_linear_attention_grad& g = *grads;
  if (args->B == 0 || args->T == 0) return fail(LNG_E_ARG, "linear_attention_grad: no tokens");
  if (!args->checkpoints || !g.dy || !g.dq || !g.dk || !g.dv || !g.ddecay)
    return fail(LNG_E_ARG, "linear_attention_grad: null pointer");
  Args a = make_args(*args, true);
  const bool token = args->token_decay != 0;
  const Space s(a, true, token);
  if (s.total && (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 ||
                  reinterpret_cast<uintptr_t>(workspace) % 64))
    return fail(LNG_E_ARG, "linear_attention_grad: the workspace is too small or not 64-byte aligned");
  const int64_t rows = a.B * a.T, hv = int64_t{a.H} * a.vts;
  if (int rc = check_threads(what, a.B * a.H * std::max<int64_t>(a.vts * a.segs, cdiv(int64_t{a.K} * a.V, 256)), 256))
    return rc;
  if (int rc = check_threads(what, cdiv(rows * a.H * std::max(a.K, a.V), 256), 256)) return rc;
  float* const ws = static_cast<float*>(workspace);
  a.seg_state = ws + s.seg_state, a.seg_decay = ws + s.seg_decay;
  a.dy = g.dy, a.yb = g.dy_batch, a.yt = g.dy_token, a.yh = g.dy_head;
  a.yvec = vector_rows(a.dy, dtype_size(args->dtype), a.yb, a.yt, a.yh, a.V);
  a.dend = g.dstate_out, a.dstart = g.dstate;
  a.dq32 = hv > a.Hq, a.dk32 = hv > a.Hk, a.dv32 = a.H > a.Hv;
  a.dq = a.dq32 ? ws + s.dq : g.dq, a.dk = a.dk32 ? ws + s.dk : g.dk, a.dv = a.dv32 ? ws + s.dv : g.dv;
  const bool dg_part = a.vts > 1 || !token;
  a.dg = dg_part ? ws + s.dg : g.ddecay;
  hipStream_t st = as_stream(stream);
  return with_type(args->dtype, [&](auto t) {
    using T = decltype(t);
    if (int rc = with_keys(a.K, [&](auto dk) { return run_bwd<T, decltype(dk)::value>(a, st); })) return rc;
    if (a.dq32)
      if (int rc = run_shared<T>(ws + s.dq, rows, a.Hq, static_cast<int>(hv / a.Hq), a.K, static_cast<T*>(g.dq), st)) return rc;
    if (a.dk32)
      if (int rc = run_shared<T>(ws + s.dk, rows, a.Hk, static_cast<int>(hv / a.Hk), a.K, static_cast<T*>(g.dk), st)) return rc;
    if (a.dv32)
      if (int rc = run_shared<T>(ws + s.dv, rows, a.Hv, a.H / a.Hv, a.V, static_cast<T*>(g.dv), st)) return rc;
    if (!dg_part) return static_cast<int>(LNG_OK);
    if (token) return run_shared<float>(ws + s.dg, rows, a.H, a.vts, 1, g.ddecay, st);
    k_la_columns<<<static_cast<unsigned>(s.col_blocks), 256, 0, st>>>(ws + s.dg, rows, static_cast<int>(hv),
                                                                     cdiv(rows, s.col_blocks), ws + s.cols);
    if (int rc = check_launch(what)) return rc;
    k_la_column_ends<<<static_cast<unsigned>(a.H), 64, 0, st>>>(ws + s.cols, static_cast<int>(s.col_blocks), a.H, a.vts,
                                                              g.ddecay);
    return check_launch(what);
  });
}

int lng_linear_attention_step(const lng_linear_attention* args, void* stream) {
  const char* what = "linear_attention_step";
  if (int rc = check_args(what, args)) return rc;
  if (args->T != 1) return fail(LNG_E_ARG, "linear_attention_step: one token of every sequence (T = 1)");
  if (args->B == 0) return LNG_OK;
  if (!args->state || !args->state_out || !args->y) return fail(LNG_E_ARG, "linear_attention_step: null pointer");
  const Args a = make_args(*args, false);
  const int64_t waves = a.B * a.H * a.vts, blocks = cdiv(waves, 4);
  if (int rc = check_threads(what, blocks, 256)) return rc;
  const bool vec = a.yvec && reinterpret_cast<uintptr_t>(a.start) % 16 == 0 && reinterpret_cast<uintptr_t>(a.end) % 16 == 0;
  return with_type(args->dtype, [&](auto t) {
    return with_keys(a.K, [&](auto dk) {
      using T = decltype(t);
      constexpr int NB = decltype(dk)::value / 32;
      hipStream_t st = as_stream(stream);
      if (vec)
        k_la_step<T, NB, true><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, waves);
      else
        k_la_step<T, NB, false><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a, waves);
      return check_launch(what);
    });
  });
}

}  // extern "C"
