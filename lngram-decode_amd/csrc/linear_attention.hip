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
constexpr int VT = 64;      // columns of values that four waves take

// Planes: bf16 parts of an input.  What is computed (scores, states, their gradients) enters products in PARTS whatever the
// type, so that a 16-bit result is what fp32 sums give, rounded once.  Two parts are short of up to 2^-16 of a value, which
// turns the rounding of one bf16 result in a thousand (1.2e-4 of the norm instead of 3e-5); they would take 107 us instead of
// 114 at 8 x 4096 x 16 x 64, bf16, and 200 instead of 214 in the training of 8 x 2048 x 16 x 64.
//
// Chunk: tokens of one.  bf16 in chunks of 64 and of 32: 8 x 4096 x 16 x 64 127 us and 139, its training 404 and 461, 4 x
// 2048 x 16 x 128 86 and 101, 284 and 365, 64 x 40 x 16 x 64 19 and 18.  fp16 in chunks of 32 and of 64: 170 and 173, 543 and
// 634, 125 and 111, 20 and 25; fp32 217 and 283, 707 and 1104.  Chunks of 64 tokens with 128 keys and values fit into LDS in
// neither direction in fp32, and not in the backward one in fp16.
constexpr int PARTS = 3;
template <typename T>
struct Traits;
template <>
struct Traits<bf16> {
  static constexpr int planes = 1, chunk = 64;
};
template <>
struct Traits<_Float16> {
  static constexpr int planes = 2, chunk = 32;
};
template <>
struct Traits<float> {
  static constexpr int planes = 3, chunk = 32;
};

// ------------------------------------------------------------------ arguments
struct Args {
  int64_t B, T;
  int H, Hq, Hk, Hv, K, V, vts, segs, seg_chunks, chunks;
  float scale;
  const void *q, *k, *v, *dy;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, yb, yt, yh;
  bool qvec, kvec, vvec, yvec;  // rows that 16-byte loads take (y: stores of four values)
  int Kp, Vp;                   // keys and values a row of q, k, v and dy holds, zeros behind K and V
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
  // Blocks go to the eight XCDs in turn: each is given neighbouring units, whose heads share keys and values in its L2.
  const uint32_t each = gridDim.x / 8, more = gridDim.x % 8, xcd = blockIdx.x % 8;
  int64_t u = xcd * each + min(xcd, more) + blockIdx.x / 8;
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
// 2^(a - b) of two sums, each the sum of two floats
__device__ __forceinline__ float exp2_gap(float ahi, float alo, float bhi, float blo) {
  return __builtin_amdgcn_exp2f((ahi - bhi) + (alo - blo));
}
__device__ __forceinline__ float exp2_sum(double x) {
  const float hi = static_cast<float>(x), e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, static_cast<float>(x - hi) * 0.69314718f, e);
}
// A log decay in powers of two.  Below -300 the decay is zero in fp32 whatever the rest: it counts as -300, minus
// infinity too, so that a difference of two such sums is no NaN.
__device__ __forceinline__ double log2_decay(float g) {
  g = g < -300.f ? -300.f : g;
  return static_cast<double>(g) * 1.4426950408889634;
}

// ------------------------------------------------------------------ operands
// x as the sum of N bf16 values.  An fp16 value is two parts exactly, an fp32 value three.  The first part is cut off, so
// that the largest finite values stay finite.  ROUND: the others are rounded, so that the products that are left out (second
// part times third: 2^-23 of the whole at most) are of either sign and add up to nothing.  Cut off as well they all have the
// whole's sign: an fp32 product is short of 2^-24 of it on average, y and the gradients of 1.4 * 2^-24 of themselves instead of
// 0.1, in 1 to 4 % less time.  Against bf16 values, one part each, nothing is left out.  (What is not finite comes out as NaN.)
template <int PLANES>
constexpr bool NEAREST = PLANES > 1;  // by the parts of the other operand, which is an input
__device__ __forceinline__ float top(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u); }

template <int N>
struct Frag {
  bf16x8 p[N];
};

// two neighbouring values of an operand
template <bool ROUND, int N>
__device__ __forceinline__ void put2(Frag<N>& f, int i, float x, float y) {
  u32x4* w[N];
#pragma unroll
  for (int p = 0; p < N; ++p) {
    w[p] = reinterpret_cast<u32x4*>(&f.p[p]);
    if (p + 1 < N && !(ROUND && p)) {
      (*w[p])[i / 2] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
      x -= top(x), y -= top(y);
    } else {
      const uint32_t both = __builtin_bit_cast(uint32_t, bf16x2{static_cast<bf16>(x), static_cast<bf16>(y)});
      (*w[p])[i / 2] = both;
      x -= __builtin_bit_cast(float, both << 16), y -= __builtin_bit_cast(float, both & 0xffff0000u);
    }
  }
}

// acc += a . b without the products of the smallest parts
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<NA>& a, const Frag<NB>& b) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < PARTS) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
}

// The same for n results that do not wait for each other: acc[k] += a(k) . b(k)
template <int NA, int NB, int N>
__device__ __forceinline__ void mma_n(f32x4 (&acc)[N], const Frag<NA> (&a)[N], const Frag<NB>& b) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < PARTS)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k].p[i], b.p[j], acc[k], 0, 0, 0);
}
template <int NA, int NB, int N>
__device__ __forceinline__ void mma_n(f32x4 (&acc)[N], const Frag<NA>& a, const Frag<NB> (&b)[N]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < PARTS)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b[k].p[j], acc[k], 0, 0, 0);
}
template <int NA, int NB, int N>
__device__ __forceinline__ void mma_n(f32x4 (&acc)[N], const Frag<NA> (&a)[N], const Frag<NB> (&b)[N]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < PARTS)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k].p[i], b[k].p[j], acc[k], 0, 0, 0);
}

// Lane l of a 16 x 16 x 32 product: row (column) l % 16 of an operand, and of its 32 products' index the values
// 4 g + 0..3 and 16 + 4 g + 0..3 with g = l / 16.  (Any order will do that both operands share; this one is that of
// two stacked result tiles, whose rows 4 g + 0..3 a lane holds, so that results are operands as they are.)
//
// Matrices stand in LDS as tiles of 16 x 16, 512 bytes each; in row r of a tile the four pieces of four values are
// swapped by r / 4, so that 16 lanes' 8-byte pieces of one column or of four rows cover all banks once, whichever way a
// matrix is read.  Whatever the matrix, a lane's place in a tile is one of two: the rest are constants.
constexpr int TILE = 256;  // elements
__device__ __forceinline__ int row_place() {  // row l % 16, piece g
  const int lane = threadIdx.x & 63, i = lane & 15;
  return i * 16 + (((lane >> 4) ^ (i >> 2)) << 2);
}
__device__ __forceinline__ int col_place() {  // row 4 g + i / 4, piece i % 4
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  return (4 * g + (i >> 2)) * 16 + (((i & 3) ^ g) << 2);
}
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ bf16x4 piece(const bf16* at) { return *reinterpret_cast<const bf16x4*>(at); }
// the transposing read: lane i of each 16-lane group gets element i % 4 of the pieces that lanes i / 4 + 4 c address
__device__ __forceinline__ bf16x4 piece_tr(const bf16* at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(at));
}
// A matrix of W columns in N planes: by_row: row r0 + l % 16, index along the row from c0; by_col: column c0 + l % 16,
// index along the rows from r0.
template <int N, int W>
__device__ __forceinline__ Frag<N> by_row(const bf16* s, int plane, int r0, int c0) {
  const bf16* at = s + ((r0 / 16) * (W / 16) + c0 / 16) * TILE + row_place();
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) f.p[p] = join(piece(at + p * plane), piece(at + p * plane + TILE));
  return f;
}
template <int N, int W>
__device__ __forceinline__ Frag<N> by_col(const bf16* s, int plane, int r0, int c0) {
  const bf16* at = s + ((r0 / 16) * (W / 16) + c0 / 16) * TILE + col_place();
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) f.p[p] = join(piece_tr(at + p * plane), piece_tr(at + p * plane + (W / 16) * TILE));
  return f;
}
// A lower triangle of tiles: (it, jt) with jt <= it
__device__ __forceinline__ constexpr int tri(int it, int jt) { return (it * (it + 1) / 2 + jt) * TILE; }
template <int N>
__device__ __forceinline__ Frag<N> tri_by_row(const bf16* s, int plane, int it, int st) {  // columns 32 st ..; 2 st <= it
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16* at = s + p * plane + row_place();
    f.p[p] = join(piece(at + tri(it, 2 * st)), 2 * st + 1 <= it ? piece(at + tri(it, 2 * st + 1)) : bf16x4{});
  }
  return f;
}
template <int N>
__device__ __forceinline__ Frag<N> tri_by_col(const bf16* s, int plane, int st, int jt) {  // rows 32 st ..; jt <= 2 st + 1
  Frag<N> f;
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16* at = s + p * plane + col_place();
    f.p[p] = join(2 * st >= jt ? piece_tr(at + tri(2 * st, jt)) : bf16x4{}, piece_tr(at + tri(2 * st + 1, jt)));
  }
  return f;
}
template <int N>
__device__ __forceinline__ float value(const Frag<N>& f, int i) {
  float x = 0.f;
#pragma unroll
  for (int p = N - 1; p >= 0; --p) x = p == N - 1 ? static_cast<float>(f.p[p][i]) : x + static_cast<float>(f.p[p][i]);
  return x;
}
// The four values of a tile's row l % 16 from column 4 g on, as a result tile's lane holds them (transposed)
template <int N>
__device__ __forceinline__ void four(const bf16* tile, int plane, float (&x)[4]) {
#pragma unroll
  for (int p = N - 1; p >= 0; --p) {
    const bf16x4 a = piece(tile + p * plane + row_place());
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p == N - 1 ? static_cast<float>(a[i]) : x[i] + static_cast<float>(a[i]);
  }
}
template <bool ROUND, int N>
__device__ __forceinline__ void put_four(bf16* tile, int plane, const float (&x)[4]) {
  Frag<N> f;
  put2<ROUND>(f, 0, x[0], x[1]);
  put2<ROUND>(f, 2, x[2], x[3]);
#pragma unroll
  for (int p = 0; p < N; ++p)
    *reinterpret_cast<bf16x4*>(tile + p * plane + row_place()) = __builtin_shufflevector(f.p[p], f.p[p], 0, 1, 2, 3);
}
// ------------------------------------------------------------------ rows from memory to LDS
// Eight neighbouring values of a row as they are in memory, element by element where 16-byte loads do not do
template <typename T>
struct Eight {
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

// The rows of one tensor of a chunk, held by a block's threads: C rows of W columns.  16 neighbouring threads take eight
// rows of half a tile, so that they write to all banks; a wave reads whole lines.
template <typename T, int C, int W, int THREADS>
struct Stage {
  static constexpr int GROUPS = C * W / 8, N = (GROUPS + THREADS - 1) / THREADS, TILES = W / 16;
  static constexpr bool WHOLE = GROUPS % THREADS == 0;  // else some threads have a group less
  Eight<T> e[N];
  static __device__ __forceinline__ void place(int i, int& r, int& c) {
    const int at = static_cast<int>(threadIdx.x) + i * THREADS;
    r = ((at >> 1) & 7) + (at >> 4) / TILES * 8;
    c = ((at >> 4) % TILES) * 16 + (at & 1) * 8;
  }
  // rows 0 .. n - 1 from `base`, `stride` bytes apart (the same in every lane), c0 their first column; else zeros
  __device__ __forceinline__ void load(const T* base, uint32_t stride, int n, int c0, int Dp) {
    const __amdgpu_buffer_rsrc_t rs = dev_buf(base, 0x7ffffff0u);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int r, c;
      place(i, r, c);
      // an offset past the descriptor's range reads zeros
      const uint32_t off = r < n && c0 + c < Dp ? static_cast<uint32_t>(r) * stride + (c0 + c) * sizeof(T) : 0x7ffffff0u;
      u32x4* w = reinterpret_cast<u32x4*>(&e[i]);
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k)
        w[k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * k, 0, 0));
    }
  }
  __device__ __forceinline__ void store(bf16* s, int plane) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int r, c;
      place(i, r, c);
      if (!WHOLE && r >= C) continue;
      bf16* tile = s + ((r / 16) * TILES + c / 16) * TILE + (r & 15) * 16;
      const int u = (c >> 2) & 3, h = (r >> 2) & 3;
      Frag<Traits<T>::planes> f;
      if constexpr (std::is_same<T, bf16>::value) {
        f.p[0] = *reinterpret_cast<const bf16x8*>(&e[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; k += 2) put2<true>(f, k, to_f32(e[i].x[k]), to_f32(e[i].x[k + 1]));
      }
#pragma unroll
      for (int p = 0; p < Traits<T>::planes; ++p) {
        *reinterpret_cast<bf16x4*>(tile + p * plane + ((u ^ h) << 2)) = __builtin_shufflevector(f.p[p], f.p[p], 0, 1, 2, 3);
        *reinterpret_cast<bf16x4*>(tile + p * plane + (((u + 1) ^ h) << 2)) =
            __builtin_shufflevector(f.p[p], f.p[p], 4, 5, 6, 7);
      }
    }
  }
};

// What a chunk's decays give: sums (in powers of two), e^{G[i]} scale, e^{G[n] - G[j]}
template <int C>
struct Decays {
  float hi[C], lo[C], from[C], left[C];
  float whole;     // e^{G[n]}
  float pad;
  double total;
};
// by one whole wave; g: this lane's token's log decay (0 behind the sequence's end)
template <int C>
__device__ __forceinline__ void decays(Decays<C>& d, float g, float scale) {
  const int lane = threadIdx.x & 63;
  double s = log2_decay(g);
#pragma unroll
  for (int off = 1; off < C; off *= 2) {
    const double o = __shfl_up(s, off, 64);
    s += lane >= off ? o : 0.;
  }
  const double t = __shfl(s, C - 1, 64);
  if (lane < C) {
    const float hi = static_cast<float>(s);
    d.hi[lane] = hi, d.lo[lane] = static_cast<float>(s - hi);
    d.from[lane] = exp2_sum(s) * scale;
    d.left[lane] = exp2_sum(t - s);
  }
  if (lane == 0) d.whole = exp2_sum(t), d.total = t;
}
__device__ __forceinline__ float load_decay(const float* g, int64_t stride, int n) {
  const int lane = threadIdx.x & 63;
  return lane < n ? g[lane * stride] : 0.f;
}

// Reads and writes through buffer descriptors: an offset past the range reads zero and writes nothing, so that no lane
// has to leave the others.  `base` is the same in every lane.
constexpr uint32_t NOWHERE = 0x7ffffff0u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t from(const void* base) { return dev_buf(base, NOWHERE); }

// A value that is formed anew where it is used: the places of results, the same in every chunk, would take dozens of
// registers through the whole loop, and spilling others costs a wait for all stores on their way.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// four neighbouring values of a row of an output, as far as it goes (left > 0 in some lane at most)
template <typename T, bool VECTOR>
__device__ __forceinline__ void store_four(__amdgpu_buffer_rsrc_t rs, uint32_t off, int left, const f32x4& x) {
  if constexpr (VECTOR) {  // whole pieces of four
    const uint32_t at = left > 0 ? off : NOWHERE;
    if constexpr (sizeof(T) == 4) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rs, at, 0, 0);
    } else {
      typedef T T4 __attribute__((ext_vector_type(4)));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const T4 t{from_f32<T>(x[0]), from_f32<T>(x[1]), from_f32<T>(x[2]), from_f32<T>(x[3])};
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, t), rs, at, 0, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = i < left ? off + i * sizeof(T) : NOWHERE;
      const float v = x[i];  // a bit cast of a vector's element itself comes out as element 0
      if constexpr (sizeof(T) == 4)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rs, at, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, from_f32<T>(v)), rs, at, 0, 0);
    }
  }
}

// ------------------------------------------------------------------ a state in a wave's registers
// Tile t holds rows 16 t + 4 g + 0..3 (keys) of column c0 + l % 16 (values) of a [K, V] matrix
__device__ __forceinline__ uint32_t state_place(int V, int c0) {
  const int lane = threadIdx.x & 63, c = c0 + (lane & 15);
  return c < V ? 4u * (4 * (lane >> 4) * V + c) : NOWHERE / 2;
}
template <int TK>
__device__ __forceinline__ void load_state(f32x4 (&s)[TK], const float* m, int K, int V, int c0) {
  const __amdgpu_buffer_rsrc_t rs = dev_buf(m, 4u * K * V);
  const uint32_t at = anew(state_place(V, c0));
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s[t][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at + 4u * (16 * t + i) * V, 0, 0));
}
template <int TK>
__device__ __forceinline__ void store_state(const f32x4 (&s)[TK], float* m, int K, int V, int c0) {
  const __amdgpu_buffer_rsrc_t rs = dev_buf(m, 4u * K * V);
  const uint32_t at = anew(state_place(V, c0));
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = s[t][i];
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rs, at + 4u * (16 * t + i) * V, 0, 0);
    }
}

// A state's tile in LDS, which a lane writes four keys of a value and reads four values of a key: key r's row stands at
// place 4 (r % 4) + r / 4, its four pieces of four swapped by r % 4, so that both take all banks once.
__device__ __forceinline__ void put_state(float* tile, const f32x4& s) {
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) tile[(4 * i + lg) * 16 + (((li >> 2) ^ i) << 2) + (li & 3)] = s[i];
}
__device__ __forceinline__ f32x4 get_state(const float* tile) {
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  return *reinterpret_cast<const f32x4*>(tile + (4 * (li & 3) + (li >> 2)) * 16 + ((lg ^ (li & 3)) << 2));
}

// S <- whole S + X^T (f Y): rows of X (sX, W keys) and Y (values, this wave's columns) of a chunk, f a factor a row.  The
// scaled operand is fp32 in three parts: the states are the results that stay in fp32.
template <int C, int TK, int W, int NX>
__device__ __forceinline__ void update_state(f32x4 (&s)[TK], const bf16* sX, int xplane, const Frag<NX> (&y)[C / 32],
                                             const float* f, float whole) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int t = 0; t < TK; ++t) s[t] *= whole;
#pragma unroll
  for (int st = 0; st < C / 32; ++st) {
    Frag<PARTS> fy;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 fr = *reinterpret_cast<const f32x4*>(f + 32 * st + 16 * h + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        put2<NEAREST<NX>>(fy, 4 * h + i, value(y[st], 4 * h + i) * fr[i], value(y[st], 4 * h + i + 1) * fr[i + 1]);
    }
    Frag<NX> fx[TK];
#pragma unroll
    for (int t = 0; t < TK; ++t) fx[t] = by_col<NX, W>(sX, xplane, 32 * st, 16 * t);
    mma_n(s, fx, fy);
  }
}
// The state as the operand whose index runs over keys
template <bool ROUND, int TK, int N>
__device__ __forceinline__ void state_frags(const f32x4 (&s)[TK], Frag<N> (&f)[TK / 2]) {
#pragma unroll
  for (int t = 0; t < TK; ++t)
#pragma unroll
    for (int r = 0; r < 4; r += 2) put2<ROUND>(f[t / 2], 4 * (t & 1) + r, s[t][r], s[t][r + 1]);
}

// ------------------------------------------------------------------ forward
template <typename T, int DK, int NW>
struct FwdLds {
  using Tr = Traits<T>;
  static constexpr int C = Tr::chunk, W = 16 * NW;
  bf16 k[Tr::planes][C * DK];
  bf16 v[Tr::planes][C * W];
  Decays<C> d[2];
  bf16 q[Tr::planes][C * DK];  // from here on: not for a segment's ends
  bf16 p[PARTS][tri(C / 16, 0)];
};

// What bounds it: at 8 x 4096 x 16 x 64 (bf16) 84 us for 281 MB, 3.3 TB/s, and at 1 x 16384 x 16 x 128 103 us, with the vector
// unit busy for 43 % and the matrix unit for 19 and 27 %: waits, at two waves a SIMD (more segments cost more than a third wave
// gains).  The segments' ends: 34 us for 109 MB, and 45 us for 49 MB.
//
// A block of NW waves takes a head's values, up to 16 NW columns, over a segment of chunks; a wave holds 16 columns of the
// state.  ENDS: only what the segment adds to the state, into seg_state, with its decay.
template <typename T, int DK, int NW, bool ENDS>
__global__ __launch_bounds__(64 * NW, ENDS && NW == 4 ? (DK <= 64 ? 4 : 3) : 2) void k_la_fwd(Args a) {
  using L = FwdLds<T, DK, NW>;
  using Tr = Traits<T>;
  constexpr int C = L::C, W = L::W, TK = DK / 16, TI = C / 16, NP = Tr::planes, THREADS = 64 * NW;
  constexpr int KP = C * DK, VP = C * W, PP = tri(C / 16, 0);  // elements of a plane
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  L& lds = *reinterpret_cast<L*>(lds_raw);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the same in all lanes: scalar arithmetic
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Unit u = unit_of(a, ENDS ? a.segs - 1 : a.segs, 0);
  const int c_first = u.seg * a.seg_chunks, c_last = min(c_first + a.seg_chunks, a.chunks);
  const int vc = 16 * w;  // the wave's first column
  const int64_t bh = u.b * a.H + u.h;
  const int64_t KV = int64_t{a.K} * a.V;
  const T* q = static_cast<const T*>(a.q) + u.b * a.qb + u.h / (a.H / a.Hq) * a.qh;
  const T* k = static_cast<const T*>(a.k) + u.b * a.kb + u.h / (a.H / a.Hk) * a.kh;
  const T* v = static_cast<const T*>(a.v) + u.b * a.vb + u.h / (a.H / a.Hv) * a.vh;
  const float* g = a.g + u.b * a.gb + u.h;
  T* y = static_cast<T*>(a.y) + (u.b * a.T * a.H + u.h) * a.V;
  const int yrow = a.H * a.V;

  f32x4 s[TK];
  if (!ENDS && a.segs > 1)
    load_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
  else if (!ENDS && a.start)
    load_state(s, a.start + bh * KV, a.K, a.V, vc);
  else
    for (int t = 0; t < TK; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int c_end = min(c_last, (u.len + C - 1) / C);  // chunks with tokens
  Stage<T, C, DK, THREADS> rq, rk;
  Stage<T, C, W, THREADS> rv;
  // one wave's: the next chunk's log decays, asked for a chunk before the rows are, so that their sums wait for nothing
  float rg = 0.f;
  g += int64_t{c_first} * C * a.gt, q += int64_t{c_first} * C * a.qt;
  k += int64_t{c_first} * C * a.kt, v += int64_t{c_first} * C * a.vt;
  auto fetch_decay = [&](int c) {
    if (w == NW - 1 && c < c_end) rg = load_decay(g, a.gt, min(C, u.len - c * C));
    g += C * a.gt;
  };
  auto fetch = [&](int c) {
    const int n = min(C, u.len - c * C);
    if (!ENDS) rq.load(q, static_cast<uint32_t>(a.qt) * sizeof(T), n, 0, a.Kp);
    rk.load(k, static_cast<uint32_t>(a.kt) * sizeof(T), n, 0, a.Kp);
    rv.load(v, static_cast<uint32_t>(a.vt) * sizeof(T), n, 0, a.Vp);
    q += C * a.qt, k += C * a.kt, v += C * a.vt;
  };
  if (c_first < c_end) {
    fetch_decay(c_first);
    fetch(c_first);
    if (w == NW - 1) decays(lds.d[c_first & 1], rg, a.scale);
    fetch_decay(c_first + 1);
  }
  double seg = 0.;
  for (int c = c_first; c < c_end; ++c) {
    const int t0 = c * C, n = min(C, u.len - t0);
    const Decays<C>& d = lds.d[c & 1];
    if (!ENDS) rq.store(lds.q[0], KP);
    rk.store(lds.k[0], KP);
    rv.store(lds.v[0], VP);
    __syncthreads();
    const float g_next = rg;
    fetch_decay(c + 2);
    if (c + 1 < c_end) fetch(c + 1);
    if (!ENDS && a.ckpt) store_state(s, a.ckpt + (bh * a.chunks + c) * KV, a.K, a.V, vc);

    if (!ENDS) {
      // the scores' tiles on and below the diagonal, transposed: column i, rows j.  A wave's tiles do not wait for each
      // other; one too many is done twice.
      auto scores = [&](auto count, int first, int all) {
        constexpr int N = decltype(count)::value;
        f32x4 acc[N];
        int it[N], idx[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          idx[k] = first + k * NW < all ? first + k * NW : first;
          it[k] = idx[k] >= 6 ? 3 : idx[k] >= 3 ? 2 : idx[k] >= 1 ? 1 : 0;
          acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int st = 0; st < DK / 32; ++st) {
          Frag<NP> fk[N], fq[N];
#pragma unroll
          for (int k = 0; k < N; ++k) {
            fk[k] = by_row<NP, DK>(lds.k[0], KP, 16 * (idx[k] - it[k] * (it[k] + 1) / 2), 32 * st);
            fq[k] = by_row<NP, DK>(lds.q[0], KP, 16 * it[k], 32 * st);
          }
          mma_n(acc, fk, fq);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int jt = idx[k] - it[k] * (it[k] + 1) / 2, i = 16 * it[k] + li, j0 = 16 * jt + 4 * lg;
          const f32x4 jh = *reinterpret_cast<const f32x4*>(&d.hi[j0]), jl = *reinterpret_cast<const f32x4*>(&d.lo[j0]);
          const float ih = d.hi[i], il = d.lo[i];
          float p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[r] = acc[k][r] * (exp2_gap(ih, il, jh[r], jl[r]) * a.scale);
            p[r] = j0 + r <= i ? p[r] : 0.f;
          }
          put_four<NEAREST<NP>, PARTS>(lds.p[0] + idx[k] * TILE, PP, p);
        }
      };
      constexpr int ALL = TI * (TI + 1) / 2, EACH = (ALL + NW - 1) / NW;
      scores(std::integral_constant<int, EACH>{}, w < ALL ? w : 0, ALL);
      __syncthreads();
    }
    if (w == NW - 1 && c + 1 < c_end) decays(lds.d[(c + 1) & 1], g_next, a.scale);

    Frag<NP> fv[C / 32];
    float odd = 0.f;
#pragma unroll
    for (int st = 0; st < C / 32; ++st) {
      fv[st] = by_col<NP, W>(lds.v[0], VP, 32 * st, 16 * w);
#pragma unroll
      for (int i = 0; i < 8; ++i) odd = fmaf(static_cast<float>(fv[st].p[0][i]), 0.f, odd);
    }
    // A weight of zero would carry an infinity or NaN among the values to the tokens before it.  It counts as zero in the
    // products, and what follows it in its column becomes NaN.
    int bad = C;  // the first such token of column l % 16
    const bool careful = __ballot(!(odd == 0.f)) != 0ull;
    if (careful) {
#pragma unroll
      for (int st = 0; st < C / 32; ++st)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = static_cast<float>(fv[st].p[0][i]);
          if (!(fabsf(f) < INFINITY)) {
            bad = min(bad, 32 * st + (i < 4 ? 0 : 16) + 4 * lg + (i & 3));
#pragma unroll
            for (int p = 0; p < NP; ++p) fv[st].p[p][i] = static_cast<bf16>(0.f);
          }
        }
      bad = min(bad, __shfl_xor(bad, 16, 64));
      bad = min(bad, __shfl_xor(bad, 32, 64));
    }
    if (!ENDS) {
      Frag<PARTS> fs[TK / 2];
      state_frags<NEAREST<NP>>(s, fs);
      const __amdgpu_buffer_rsrc_t yc = from(y + int64_t{t0} * yrow);
      const int col = anew(vc + 4 * lg);
      auto outputs = [&](auto count, int first) {
        constexpr int N = decltype(count)::value;
        f32x4 acc[N];
        Frag<NP> fq[N];
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st) {
#pragma unroll
          for (int k = 0; k < N; ++k) fq[k] = by_row<NP, DK>(lds.q[0], KP, 16 * (first + k), 32 * st);
          mma_n(acc, fs[st], fq);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] *= d.from[16 * (first + k) + li];
#pragma unroll
        for (int st = 0; st < C / 32; ++st)
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (2 * st <= first + k) mma(acc[k], fv[st], tri_by_row<PARTS>(lds.p[0], PP, first + k, st));
        if (careful)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int from_here = __shfl(bad, 4 * lg + r, 64);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k][r] = 16 * (first + k) + li >= from_here ? NAN : acc[k][r];
          }
        if (a.yvec) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int i = 16 * (first + k) + li;
            store_four<T, true>(yc, static_cast<uint32_t>(i * yrow + col) * sizeof(T), i < n ? a.V - col : 0, acc[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int i = 16 * (first + k) + li;
            store_four<T, false>(yc, static_cast<uint32_t>(i * yrow + col) * sizeof(T), i < n ? a.V - col : 0, acc[k]);
          }
        }
      };
      outputs(std::integral_constant<int, TI>{}, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    update_state<C, TK, DK, NP>(s, lds.k[0], KP, fv, d.left, d.whole);
    if (careful && bad < C)
#pragma unroll
      for (int t = 0; t < TK; ++t) s[t] = f32x4{NAN, NAN, NAN, NAN};
    if (ENDS && threadIdx.x == 0) seg += d.total;
    __syncthreads();
  }
  if (ENDS) {
    store_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
    if (threadIdx.x == 0) a.seg_decay[bh * a.segs + u.seg] = static_cast<float>(seg);
    return;
  }
  // positions behind the sequence's end
  const int start = max(u.len, c_first * C), to = static_cast<int>(min(static_cast<int64_t>(c_last) * C, a.T));
  const int cols = a.V;
  for (int64_t i = threadIdx.x; i < int64_t{to - start} * cols; i += THREADS)
    y[(start + i / cols) * a.H * a.V + i % cols] = from_f32<T>(0.f);
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
  // eight segments' terms asked for at once: the loads do not wait for each other
  constexpr int N = 8;
  for (int first = 0; first < a.segs; first += N) {
    float* at[N];
    float add[N], decay[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = min(first + n, a.segs - 1), seg = BACK ? a.segs - 1 - i : i;
      at[n] = a.seg_state + (bh * a.segs + seg) * KV + e;
      const bool has = i + 1 < a.segs;  // the last one's end is nobody's start
      add[n] = has ? *at[n] : 0.f;
      decay[n] = has ? a.seg_decay[bh * a.segs + seg] : 0.f;
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (first + n < a.segs) {
        *at[n] = s;
        s = fmaf(s, __builtin_amdgcn_exp2f(decay[n]), add[n]);
      }
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
// forward pass kept.  Everything is linear in the value columns: a block takes 16 BW of them, and dq, dk and dg of
// several such tiles are summed afterwards, as the gradients of shared heads are.  P and A take the same place in LDS, one
// after the other, A in registers meanwhile: three parts of both and R would leave room for one block a CU.
//
// 8 x 2048 x 16 x 64, bf16: 117 us for 313 MB; the vector unit is busy for 35 %, the matrix unit for 15 %: waits, at two waves
// a SIMD.  Registers decide: the scores' tiles go one by one and operands are split where they are used, since a spill waits
// for the stores in flight (a third more time).
template <typename T, int DK, int BW>
struct BwdLds {
  using Tr = Traits<T>;
  static constexpr int C = Tr::chunk, W = 16 * BW;
  bf16 q[Tr::planes][C * DK];
  bf16 o[Tr::planes][C * W];  // dy
  Decays<C> d[2];
  bf16 k[Tr::planes][C * DK];  // from here on: not for a segment's ends
  bf16 v[Tr::planes][C * W];
  bf16 p[PARTS][tri(C / 16, 0)];  // P for dv, then A for dq and dk
  float r[W * DK];             // R for dk: tiles of 16 values and 16 keys
  float row[C / 16][C];        // sums over a tile's j of P (dy.v), below the diagonal
  float col[C / 16][C];        // over its i
  float qs[DK / 16][C];        // q[i].(scale e^{G[i]} S_in dy[i]) over 16 keys
  float kr[BW][C];             // v[j].(e^{G[n]-G[j]} R^T k[j]) over a wave's columns
  float sr[BW];                // a wave's share of <S_in, R>
};

// Sum over the 16 lanes of a row of the wave, in all of them
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = 1; m < 16; m *= 2) v += __shfl_xor(v, m, 64);
  return v;
}
// Sum over the four rows of the wave, in all of them
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// What a block's 16 BW columns of the values add to the gradients; ENDS: only what the segment adds to the state's
// gradient.
template <typename T, int DK, int BW, bool ENDS>
__global__ __launch_bounds__(64 * BW, BW == 8 ? 2 : DK <= 64 ? (ENDS ? 4 : 2) : (ENDS ? 3 : 1)) void k_la_bwd(Args a) {
  using L = BwdLds<T, DK, BW>;
  using Tr = Traits<T>;
  constexpr int C = L::C, W = L::W, BTHREADS = 64 * BW, TK = DK / 16, TI = C / 16, NP = Tr::planes;
  constexpr int KP = C * DK, VP = C * W, PP = tri(C / 16, 0);  // elements of a plane
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  L& lds = *reinterpret_cast<L*>(lds_raw);
  // scalar: transposing reads need all lanes, which a branch on a wave's number in a vector register does not promise
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Unit u = unit_of(a, ENDS ? a.segs - 1 : a.segs, ENDS ? 1 : 0);
  const int c_first = u.seg * a.seg_chunks, c_last = min(c_first + a.seg_chunks, a.chunks);
  const int v0 = u.vt * W, vc = v0 + 16 * w;
  const int64_t bh = u.b * a.H + u.h;
  const int64_t KV = int64_t{a.K} * a.V;
  const T* q = static_cast<const T*>(a.q) + u.b * a.qb + u.h / (a.H / a.Hq) * a.qh;
  const T* k = static_cast<const T*>(a.k) + u.b * a.kb + u.h / (a.H / a.Hk) * a.kh;
  const T* v = static_cast<const T*>(a.v) + u.b * a.vb + u.h / (a.H / a.Hv) * a.vh;
  const T* dy = static_cast<const T*>(a.dy) + u.b * a.yb + u.h * a.yh;
  const float* g = a.g + u.b * a.gb + u.h;
  const int hv = u.h * a.vts + u.vt;  // of the heads' value tiles

  f32x4 s[TK];  // R: rows of keys, this wave's 16 columns
  if (!ENDS && a.segs > 1)
    load_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
  else if (!ENDS && a.dend)
    load_state(s, a.dend + bh * KV, a.K, a.V, vc);
  else
    for (int t = 0; t < TK; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int c_end = min(c_last, (u.len + C - 1) / C);  // chunks with tokens
  Stage<T, C, DK, BTHREADS> rq, rk;
  Stage<T, C, W, BTHREADS> rv, ro;
  float rg = 0.f;  // one wave's: the log decays of the chunk before, asked for a chunk ahead of its rows
  g += int64_t{c_end - 1} * C * a.gt, q += int64_t{c_end - 1} * C * a.qt, dy += int64_t{c_end - 1} * C * a.yt;
  k += int64_t{c_end - 1} * C * a.kt, v += int64_t{c_end - 1} * C * a.vt;
  auto fetch_decay = [&](int c) {
    if (w == BW - 1 && c >= c_first) rg = load_decay(g, a.gt, min(C, u.len - c * C));
    g -= C * a.gt;
  };
  auto fetch = [&](int c) {
    const int n = min(C, u.len - c * C);
    rq.load(q, static_cast<uint32_t>(a.qt) * sizeof(T), n, 0, a.Kp);
    ro.load(dy, static_cast<uint32_t>(a.yt) * sizeof(T), n, v0, a.Vp);
    if (!ENDS) {
      rk.load(k, static_cast<uint32_t>(a.kt) * sizeof(T), n, 0, a.Kp);
      rv.load(v, static_cast<uint32_t>(a.vt) * sizeof(T), n, v0, a.Vp);
    }
    q -= C * a.qt, dy -= C * a.yt, k -= C * a.kt, v -= C * a.vt;
  };
  if (c_first < c_end) {
    fetch_decay(c_end - 1);
    fetch(c_end - 1);
    if (w == BW - 1) decays(lds.d[(c_end - 1) & 1], rg, a.scale);
    fetch_decay(c_end - 2);
  }
  // rows of the outputs, in elements
  const int qrow = (a.dq32 ? a.H * a.vts : a.H) * a.K, krow = (a.dk32 ? a.H * a.vts : a.H) * a.K, vrow = a.H * a.V;
  const int qcol = (a.dq32 ? hv : u.h) * a.K, kcol = (a.dk32 ? hv : u.h) * a.K;
  const bool k4 = a.K % 4 == 0, v4 = a.V % 4 == 0;
  // a lane's four values of a token's output: in the type, or in fp32 to be summed with others
  auto emit = [&](void* out, bool f32, int64_t first, int row, int i, int col, int left, bool vec, const f32x4& x) {
    const uint32_t es = f32 ? 4 : sizeof(T), at = static_cast<uint32_t>(i * row + col) * es;
    const __amdgpu_buffer_rsrc_t rs = from(static_cast<char*>(out) + first * row * es);
    if (f32)
      vec ? store_four<float, true>(rs, at, left, x) : store_four<float, false>(rs, at, left, x);
    else
      vec ? store_four<T, true>(rs, at, left, x) : store_four<T, false>(rs, at, left, x);
  };
  double seg = 0.;
  for (int c = c_end - 1; c >= c_first; --c) {
    const int t0 = c * C, n = min(C, u.len - t0);
    const int64_t token = u.b * a.T + t0;
    const Decays<C>& d = lds.d[c & 1];
    rq.store(lds.q[0], KP);
    ro.store(lds.o[0], VP);
    if (!ENDS) {
      rk.store(lds.k[0], KP);
      rv.store(lds.v[0], VP);
#pragma unroll
      for (int t = 0; t < TK; ++t) put_state(lds.r + (w * TK + t) * TILE, s[t]);
    }
    __syncthreads();
    const float g_next = rg;
    fetch_decay(c - 2);
    if (c > c_first) fetch(c - 1);

    constexpr int ALL = TI * (TI + 1) / 2, EACH = (ALL + BW - 1) / BW;
    float held[EACH][4];  // this wave's tiles of A: they take the place of P's when dv has been formed
    if (!ENDS) {
      // a wave's tiles one after the other: side by side their operands would spill
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const int idx = w + k * BW;
        if (idx >= ALL) continue;
        const int it = idx >= 6 ? 3 : idx >= 3 ? 2 : idx >= 1 ? 1 : 0, jt = idx - it * (it + 1) / 2;
        f32x4 qk{0.f, 0.f, 0.f, 0.f}, ov{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st)
          mma(qk, by_row<NP, DK>(lds.k[0], KP, 16 * jt, 32 * st), by_row<NP, DK>(lds.q[0], KP, 16 * it, 32 * st));
#pragma unroll
        for (int st = 0; st < W / 32; ++st)
          mma(ov, by_row<NP, W>(lds.v[0], VP, 16 * jt, 32 * st), by_row<NP, W>(lds.o[0], VP, 16 * it, 32 * st));
        const int i = 16 * it + li, j0 = 16 * jt + 4 * lg;
        const f32x4 jh = *reinterpret_cast<const f32x4*>(&d.hi[j0]), jl = *reinterpret_cast<const f32x4*>(&d.lo[j0]);
        const float ih = d.hi[i], il = d.lo[i];
        float p[4], pair[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float dec = exp2_gap(ih, il, jh[r], jl[r]) * a.scale;
          p[r] = j0 + r <= i ? qk[r] * dec : 0.f;
          held[k][r] = j0 + r <= i ? ov[r] * dec : 0.f;
          pair[r] = j0 + r < i ? p[r] * ov[r] : 0.f;
        }
        put_four<NEAREST<NP>, PARTS>(lds.p[0] + idx * TILE, PP, p);
        const float rows = col_sum((pair[0] + pair[1]) + (pair[2] + pair[3]));
        if (lg == 0) lds.row[jt][i] = rows;
#pragma unroll
        for (int r = 0; r < 4; ++r) pair[r] = row_sum(pair[r]);
        if (li == 0) *reinterpret_cast<f32x4*>(&lds.col[it][j0]) = f32x4{pair[0], pair[1], pair[2], pair[3]};
        __builtin_amdgcn_sched_barrier(0);
      }
      __syncthreads();
    }
    if (w == BW - 1 && c > c_first) decays(lds.d[(c - 1) & 1], g_next, a.scale);

    if (!ENDS) {
      // <S_in, R> of this wave's columns, in 32 bits: as the state lies in registers
      f32x4 in[TK];
      float sr = 0.f;
      load_state(in, a.ckpt + (bh * a.chunks + c) * KV, a.K, a.V, vc);
#pragma unroll
      for (int t = 0; t < TK; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sr = fmaf(in[t][r], s[t][r], sr);
      sr = wave_sum(sr);
      if (lane == 0) lds.sr[w] = sr;
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);
    Frag<NP> fo[C / 32];  // dy: this wave's columns
#pragma unroll
    for (int st = 0; st < C / 32; ++st) fo[st] = by_col<NP, W>(lds.o[0], VP, 32 * st, 16 * w);
    if (!ENDS) {
      // dv: this wave's 16 columns
      const int col = anew(vc + 4 * lg);
      auto values = [&](auto count, int first) {
        constexpr int N = decltype(count)::value;
        f32x4 acc[N];
        Frag<NP> fj[N];
#pragma unroll
        for (int m = 0; m < N; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < DK / 32; ++st) {
#pragma unroll
          for (int m = 0; m < N; ++m) fj[m] = by_row<NP, DK>(lds.k[0], KP, 16 * (first + m), 32 * st);
          Frag<PARTS> fs;  // R, index of keys
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; r += 2) put2<NEAREST<NP>>(fs, 4 * t + r, s[2 * st + t][r], s[2 * st + t][r + 1]);
          mma_n(acc, fs, fj);
        }
#pragma unroll
        for (int m = 0; m < N; ++m) {
          const int j = 16 * (first + m) + li;
          float x[4], sum = 0.f;
          acc[m] *= d.left[j];
          four<NP>(lds.v[0] + ((first + m) * (W / 16) + w) * TILE, VP, x);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum = fmaf(x[r], acc[m][r], sum);
          sum = col_sum(sum);
          if (lg == 0) lds.kr[w][j] = sum;
        }
#pragma unroll
        for (int st = 0; st < C / 32; ++st)
#pragma unroll
          for (int m = 0; m < N; ++m)
            if (2 * st + 1 >= first + m)
              mma(acc[m], fo[st], tri_by_col<PARTS>(lds.p[0], PP, st, first + m));
#pragma unroll
        for (int m = 0; m < N; ++m) {
          const int j = 16 * (first + m) + li;
          emit(a.dv, a.dv32, token, vrow, j, u.h * a.V + col, j < n ? a.V - col : 0, v4, acc[m]);
        }
      };
      values(std::integral_constant<int, TI>{}, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!ENDS) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < EACH; ++k)
        if (w + k * BW < ALL) put_four<NEAREST<NP>, PARTS>(lds.p[0] + (w + k * BW) * TILE, PP, held[k]);
    }
    update_state<C, TK, DK, NP>(s, lds.q[0], KP, fo, d.from, d.whole);
    if (ENDS && threadIdx.x == 0) seg += d.total;
    if (!ENDS) {
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      // dq and dk: tiles of 16 keys and 16 tokens, a wave's share of the keys (of the tokens, where keys are few)
      constexpr int SHARE = TK >= BW ? 1 : BW / TK, KT = TK >= BW ? TK / BW : 1, IT = TI / SHARE > 0 ? TI / SHARE : 1;
      const __amdgpu_buffer_rsrc_t si = dev_buf(a.ckpt + (bh * a.chunks + c) * KV, 4u * a.K * a.V);
      const int part = w % SHARE;
#pragma unroll 1
      for (int kk = 0; kk < KT; ++kk) {
        const int kt = w / SHARE * KT + kk;
        f32x4 in[W / 32][2];  // S_in, rows of keys, index of values
        const int row = 16 * kt + li;
#pragma unroll
        for (int st = 0; st < W / 32; ++st)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = v0 + 32 * st + 16 * h + 4 * lg;
            const uint32_t at = 4u * (row * a.V + col);
            if (v4) {
              in[st][h] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(si, col < a.V ? at : NOWHERE, 0, 0));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                in[st][h][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(si, col + i < a.V ? at + 4 * i : NOWHERE, 0, 0));
            }
          }
        const int key = anew(16 * kt + 4 * lg);
        auto tokens = [&](auto count, int first) {  // the tiles of tokens from `first` on
          constexpr int N = decltype(count)::value;
          f32x4 acc[N];
          Frag<NP> fi[N];
#pragma unroll
          for (int m = 0; m < N; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < W / 32; ++st) {
#pragma unroll
            for (int m = 0; m < N; ++m) fi[m] = by_row<NP, W>(lds.o[0], VP, 16 * (first + m), 32 * st);
            Frag<PARTS> fs;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x[4] = {in[st][h][0], in[st][h][1], in[st][h][2], in[st][h][3]};
              put2<NEAREST<NP>>(fs, 4 * h, x[0], x[1]);
              put2<NEAREST<NP>>(fs, 4 * h + 2, x[2], x[3]);
            }
            mma_n(acc, fs, fi);
            if (DK > 64) __builtin_amdgcn_sched_barrier(0);  // one operand at a time: registers
          }
#pragma unroll
          for (int m = 0; m < N; ++m) {
            const int i = 16 * (first + m) + li;
            float x[4], sum = 0.f;
            acc[m] *= d.from[i];
            four<NP>(lds.q[0] + ((first + m) * TK + kt) * TILE, KP, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum = fmaf(x[r], acc[m][r], sum);
            sum = col_sum(sum);
            if (lg == 0) lds.qs[kt][i] = sum;
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int st = 0; st < C / 32; ++st) {
            if (2 * st > first + N - 1) continue;
            const Frag<NP> fk = by_col<NP, DK>(lds.k[0], KP, 32 * st, 16 * kt);
#pragma unroll
            for (int m = 0; m < N; ++m)
              if (2 * st <= first + m) mma(acc[m], fk, tri_by_row<PARTS>(lds.p[0], PP, first + m, st));
          }
#pragma unroll
          for (int m = 0; m < N; ++m) {
            const int i = 16 * (first + m) + li;
            emit(a.dq, a.dq32, token, qrow, i, qcol + key, i < n ? a.K - key : 0, k4, acc[m]);
            acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int st = 0; st < W / 32; ++st) {
#pragma unroll
            for (int m = 0; m < N; ++m) fi[m] = by_row<NP, W>(lds.v[0], VP, 16 * (first + m), 32 * st);
            const f32x4 r0 = get_state(lds.r + (2 * st * TK + kt) * TILE), r1 = get_state(lds.r + ((2 * st + 1) * TK + kt) * TILE);
            Frag<PARTS> fr;  // R, index of values
#pragma unroll
            for (int r = 0; r < 4; r += 2) put2<NEAREST<NP>>(fr, r, r0[r], r0[r + 1]), put2<NEAREST<NP>>(fr, 4 + r, r1[r], r1[r + 1]);
            mma_n(acc, fr, fi);
          }
#pragma unroll
          for (int m = 0; m < N; ++m) acc[m] *= d.left[16 * (first + m) + li];
#pragma unroll
          for (int st = 0; st < C / 32; ++st) {
            const Frag<NP> fq = by_col<NP, DK>(lds.q[0], KP, 32 * st, 16 * kt);
#pragma unroll
            for (int m = 0; m < N; ++m)
              if (2 * st + 1 >= first + m)
                mma(acc[m], fq, tri_by_col<PARTS>(lds.p[0], PP, st, first + m));
          }
#pragma unroll
          for (int m = 0; m < N; ++m) {
            const int i = 16 * (first + m) + li;
            emit(a.dk, a.dk32, token, krow, i, kcol + key, i < n ? a.K - key : 0, k4, acc[m]);
          }
        };
        if (part * IT < TI) tokens(std::integral_constant<int, IT>{}, SHARE == 1 ? 0 : part * IT);
      }
    }
    __syncthreads();
    if (!ENDS && w == BW - 1) {
      // the decays' gradients: a lane a token
      double later = 0., kept = 0., sr = 0.;  // what is summed from t on, before t, and for all
      for (int t = 0; t < BW; ++t) sr += lds.sr[t];
      if (lane < n) {
        for (int t = 0; t <= lane / 16; ++t) later += lds.row[t][lane];
        for (int t = lane / 16; t < TI; ++t) later -= lds.col[t][lane];
        for (int t = 0; t < TK; ++t) later += lds.qs[t][lane];
        for (int t = 0; t < BW; ++t) kept += lds.kr[t][lane];
      }
      double total = kept;
#pragma unroll
      for (int off = 1; off < C; off *= 2) {
        const double x = __shfl_down(later, off, 64), y = __shfl_up(total, off, 64);
        if (lane + off < 64) later += x;
        if (lane >= off) total += y;
      }
      if (lane < n)
        a.dg[(token + lane) * a.H * a.vts + hv] = static_cast<float>(
            later + (total - kept) + double(d.whole) * sr);
    }
  }
  if (ENDS) {
    store_state(s, a.seg_state + (bh * a.segs + u.seg) * KV, a.K, a.V, vc);
    if (threadIdx.x == 0 && u.vt == 0) a.seg_decay[bh * a.segs + u.seg] = static_cast<float>(seg);
    return;
  }
  // positions behind the sequence's end
  const int start = max(u.len, c_first * C), to = static_cast<int>(min(static_cast<int64_t>(c_last) * C, a.T));
  const int cols = min(W, a.V - v0);
  auto clear = [&](void* out, bool f32, int64_t head, int64_t heads, int d, int c0, int width) {
    for (int64_t i = threadIdx.x; i < int64_t{to - start} * width; i += BTHREADS) {
      const int64_t at = ((u.b * a.T + start + i / width) * heads + head) * d + c0 + i % width;
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

// ------------------------------------------------------------------ rows for 16-byte loads
// [B, T, heads, D] -> [B, T, heads, Dp] in neighbouring rows, zeros behind D: what rows of other widths, addresses or
// distances go through first
template <typename T>
__global__ __launch_bounds__(256) void k_la_pack(const T* x, int64_t batch, int64_t token, int64_t head, int64_t tokens, int heads,
                                                 int D, int Dp, int64_t groups, T* out) {
  const int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x;
  if (i >= groups) return;
  const int per = Dp / 8, c = static_cast<int>(i % per) * 8;
  int64_t r = i / per;
  const int h = static_cast<int>(r % heads);
  r /= heads;
  const T* row = x + r / tokens * batch + r % tokens * token + h * head;
  const Eight<T> e = load_eight<T>(row, c, D, false);
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k)
    reinterpret_cast<u32x4*>(out + i * 8)[k] = reinterpret_cast<const u32x4*>(&e)[k];
}

// ------------------------------------------------------------------ one token
// A wave takes 64 value columns of a head: lane l four of them, and of the keys every fourth part.  All of a lane's
// state is asked for at once; the state is read and written where it stands, so that it may move on in place.  512 x 16 x
// 64 x 64, bf16 rows: 57 us for 273 MB, 4.8 TB/s.
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
  const float decay = exp2_sum(log2_decay(g));
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
  if (lg) return;
  T* out = static_cast<T*>(a.y) + bh * a.V + c;
  if constexpr (VEC) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    y *= a.scale;
    if (c < a.V) *reinterpret_cast<T4*>(out) = T4{from_f32<T>(y[0]), from_f32<T>(y[1]), from_f32<T>(y[2]), from_f32<T>(y[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < a.V) out[i] = from_f32<T>(y[i] * a.scale);
  }
}

// ------------------------------------------------------------------ host
int chunk_of(int dtype) { return dtype == LNG_BF16 ? Traits<bf16>::chunk : Traits<float>::chunk; }

// Rows in 16-byte pieces, a chunk's within 32-bit offsets; a distance of what there is one of does not count.
bool vector_rows(const void* p, int es, const Args& a, int heads, int64_t batch, int64_t token, int64_t head, int d) {
  if (a.B == 1) batch = 0;
  if (a.T == 1) token = 0;
  if (heads == 1) head = 0;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && batch * es % 16 == 0 && token * es % 16 == 0 && head * es % 16 == 0 &&
         d % 8 == 0 && token >= 0 && token * es < (int64_t{1} << 25);
}

// Blocks of four waves that a launch should have, two for each CU (of eight, one): a segment more costs the keys and
// values (the queries and dy) of all but one segment a second time.  8 x 4096 x 16 x 64 in 128, 256, 384, 512, 768, 1024
// blocks: 213, 162, 133, 114, 107, 113 us; 1 x 16384 x 16 x 128 in 256, 384, 512, 768, 1024: 234, 174, 139, 182, 151; the
// training of 8 x 2048 x 16 x 64 with its backward pass in 128, 256, 384, 512, 768: 451, 299, 247, 214, 242.  Segments of
// one chunk gain nothing: 3 x 777 x 6 x 40 from one chunk, two, three, four on: 28, 29, 33, 37 us.
constexpr int64_t BLOCKS = 512;

Args make_args(const lng_linear_attention& l, bool grad) {
  Args a{};
  a.B = l.B, a.T = l.T, a.H = l.H, a.Hq = l.Hq, a.Hk = l.Hk, a.Hv = l.Hv, a.K = l.K, a.V = l.V, a.scale = l.scale;
  a.q = l.q, a.k = l.k, a.v = l.v;
  a.qb = l.q_batch, a.qt = l.q_token, a.qh = l.q_head, a.kb = l.k_batch, a.kt = l.k_token, a.kh = l.k_head;
  a.vb = l.v_batch, a.vt = l.v_token, a.vh = l.v_head;
  const int es = dtype_size(l.dtype);
  a.qvec = vector_rows(a.q, es, a, a.Hq, a.qb, a.qt, a.qh, a.K), a.kvec = vector_rows(a.k, es, a, a.Hk, a.kb, a.kt, a.kh, a.K);
  a.vvec = vector_rows(a.v, es, a, a.Hv, a.vb, a.vt, a.vh, a.V);
  a.g = l.decay, a.gb = l.decay_batch, a.gt = l.decay_token;
  a.start = l.state, a.lengths = l.lengths, a.y = l.y, a.end = l.state_out, a.ckpt = l.checkpoints;
  a.yvec = a.V % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * es) == 0;
  a.Kp = static_cast<int>(cdiv(a.K, 8)) * 8, a.Vp = static_cast<int>(cdiv(a.V, 8)) * 8;
  a.vts = grad && l.dtype != LNG_F32 ? 1 : static_cast<int>(cdiv(a.V, VT));  // blocks of value columns
  a.chunks = static_cast<int>(cdiv(a.T, chunk_of(l.dtype)));
  const int64_t units = std::max<int64_t>(1, a.B * a.H * cdiv(a.V, VT));
  const int64_t segs = std::min<int64_t>((BLOCKS + units / 2) / units, cdiv(a.chunks, 2));
  a.seg_chunks = static_cast<int>(cdiv(a.chunks, std::max<int64_t>(segs, 1)));
  a.segs = a.seg_chunks ? static_cast<int>(cdiv(a.chunks, a.seg_chunks)) : 1;
  return a;
}

// floats of the workspace
struct Space {
  int64_t seg_state = 0, seg_decay = 0, q = 0, k = 0, v = 0, dy = 0, dq = 0, dk = 0, dv = 0, dg = 0, cols = 0, total = 0;
  int64_t col_blocks = 0;
  Space(const Args& a, int es, bool grad, bool token_decay) {
    auto take = [&](int64_t n) {
      const int64_t at = total;
      total += cdiv(n, 16) * 16;
      return at;
    };
    if (a.segs > 1) seg_state = take(a.B * a.H * a.segs * a.K * a.V), seg_decay = take(a.B * a.H * a.segs);
    auto rows_of = [&](int heads, int width) { return take(cdiv(a.B * a.T * heads * width * es, 4)); };
    if (!a.qvec) q = rows_of(a.Hq, a.Kp);
    if (!a.kvec) k = rows_of(a.Hk, a.Kp);
    if (!a.vvec) v = rows_of(a.Hv, a.Vp);
    if (!grad) return;
    if (a.V % 8) dy = rows_of(a.H, a.Vp);
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
  if (l->H < 1 || l->H > (1 << 14) || l->Hq < 1 || l->Hk < 1 || l->Hv < 1 || l->H % l->Hq || l->H % l->Hk || l->H % l->Hv)
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

// Every launch of a call, before its first
int check_launches(const char* what, const Args& a, bool grad) {
  const int64_t rows = a.B * a.T;
  int64_t most = a.B * a.H * std::max<int64_t>(cdiv(a.V, VT) * a.segs, cdiv(int64_t{a.K} * a.V, 256));
  auto packed = [&](bool vec, int heads, int width) {
    if (!vec) most = std::max(most, cdiv(rows * heads * (width / 8), 256));
  };
  packed(a.qvec, a.Hq, a.Kp), packed(a.kvec, a.Hk, a.Kp), packed(a.vvec, a.Hv, a.Vp);
  if (grad) packed(a.V % 8 == 0, a.H, a.Vp), most = std::max(most, cdiv(rows * a.H * std::max(a.K, a.V), 256));
  return check_threads(what, most, 256);
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

// A tensor's rows into the workspace; from there on they are the tensor
template <typename T>
int pack(const void*& x, int64_t& batch, int64_t& token, int64_t& head, int64_t B, int64_t tokens, int heads, int D, int Dp,
         float* to, hipStream_t st) {
  const int64_t groups = B * tokens * heads * (Dp / 8);
  k_la_pack<T><<<static_cast<unsigned>(cdiv(groups, 256)), 256, 0, st>>>(static_cast<const T*>(x), batch, token, head, tokens,
                                                                       heads, D, Dp, groups, reinterpret_cast<T*>(to));
  x = to, head = Dp, token = int64_t{heads} * Dp, batch = tokens * token;
  return check_launch("linear_attention");
}
template <typename T>
int pack_inputs(Args& a, const Space& s, float* ws, hipStream_t st) {
  if (!a.qvec)
    if (int rc = pack<T>(a.q, a.qb, a.qt, a.qh, a.B, a.T, a.Hq, a.K, a.Kp, ws + s.q, st)) return rc;
  if (!a.kvec)
    if (int rc = pack<T>(a.k, a.kb, a.kt, a.kh, a.B, a.T, a.Hk, a.K, a.Kp, ws + s.k, st)) return rc;
  if (!a.vvec)
    if (int rc = pack<T>(a.v, a.vb, a.vt, a.vh, a.B, a.T, a.Hv, a.V, a.Vp, ws + s.v, st)) return rc;
  return LNG_OK;
}

template <typename T, int DK, int NW>
int run_fwd(const Args& args, hipStream_t st) {
  using L = FwdLds<T, DK, NW>;
  constexpr size_t lds = sizeof(L);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  Args a = args;
  a.vts = 1;  // a block takes all columns
  const int64_t units = a.B * a.H;
  if (a.segs > 1) {
    if (int rc = launch(&k_la_fwd<T, DK, NW, true>, static_cast<unsigned>(units * (a.segs - 1)), 64 * NW,
                        offsetof(L, q), st, a, "linear_attention"))
      return rc;
    if (int rc = run_join<false>(a, st)) return rc;
  }
  return launch(&k_la_fwd<T, DK, NW, false>, static_cast<unsigned>(units * a.segs), 64 * NW, lds, st, a,
                "linear_attention");
}

template <typename T, int DK, int BW>
int run_bwd(const Args& a, hipStream_t st) {
  using L = BwdLds<T, DK, BW>;
  constexpr size_t lds = sizeof(L);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  const int64_t units = a.B * a.H * a.vts;
  if (a.segs > 1) {
    if (int rc = launch(&k_la_bwd<T, DK, BW, true>, static_cast<unsigned>(units * (a.segs - 1)), 64 * BW,
                        offsetof(L, k), st, a, "linear_attention_grad"))
      return rc;
    if (int rc = run_join<true>(a, st)) return rc;
  }
  return launch(&k_la_bwd<T, DK, BW, false>, static_cast<unsigned>(units * a.segs), 64 * BW, lds, st, a,
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
  return static_cast<size_t>(Space(a, dtype_size(args->dtype), grad != 0, args->token_decay != 0).total) * 4;
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
  const Space s(a, dtype_size(args->dtype), false, args->token_decay != 0);
  if (s.total && (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 ||
                  reinterpret_cast<uintptr_t>(workspace) % 64))
    return fail(LNG_E_ARG, "linear_attention: the workspace is too small or not 64-byte aligned");
  if (int rc = check_launches(what, a, false)) return rc;
  float* const ws = static_cast<float*>(workspace);
  a.seg_state = ws + s.seg_state, a.seg_decay = ws + s.seg_decay;
  return with_type(args->dtype, [&](auto t) {
    if (int rc = pack_inputs<decltype(t)>(a, s, ws, as_stream(stream))) return rc;
    return with_keys(a.K, [&](auto dk) {
      using T = decltype(t);
      constexpr int DK = decltype(dk)::value;
      // Eight waves compute the scores of 128 columns once, and twice if they are blocks of four.  1 x 8192 tokens, 16
      // heads of 64 keys and 128 values, bf16: 63 us and 67, of 128 keys 82 and 90, in fp32 108 and 110, 152 and 161.  Up to
      // 64 columns they would leave half of the waves without work: 64 and 46.
      return a.V <= 64 ? run_fwd<T, DK, 4>(a, as_stream(stream)) : run_fwd<T, DK, 8>(a, as_stream(stream));
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
  const int es = dtype_size(args->dtype);
  const Space s(a, es, true, token);
  if (s.total && (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 ||
                  reinterpret_cast<uintptr_t>(workspace) % 64))
    return fail(LNG_E_ARG, "linear_attention_grad: the workspace is too small or not 64-byte aligned");
  const int64_t rows = a.B * a.T, hv = int64_t{a.H} * a.vts;
  if (int rc = check_launches(what, a, true)) return rc;
  a.dy = g.dy, a.yb = g.dy_batch, a.yt = g.dy_token, a.yh = g.dy_head;
  if (a.V % 8 == 0 && !vector_rows(a.dy, es, a, a.H, a.yb, a.yt, a.yh, a.V))
    return fail(LNG_E_ARG, "linear_attention_grad: rows of dy in 16-byte pieces, less than 2^25 bytes apart");
  float* const ws = static_cast<float*>(workspace);
  a.seg_state = ws + s.seg_state, a.seg_decay = ws + s.seg_decay;
  a.dend = g.dstate_out, a.dstart = g.dstate;
  a.dq32 = hv > a.Hq, a.dk32 = hv > a.Hk, a.dv32 = a.H > a.Hv;
  a.dq = a.dq32 ? ws + s.dq : g.dq, a.dk = a.dk32 ? ws + s.dk : g.dk, a.dv = a.dv32 ? ws + s.dv : g.dv;
  const bool dg_part = a.vts > 1 || !token;
  a.dg = dg_part ? ws + s.dg : g.ddecay;
  hipStream_t st = as_stream(stream);
  return with_type(args->dtype, [&](auto t) {
    using T = decltype(t);
    if (int rc = pack_inputs<T>(a, s, ws, st)) return rc;
    if (a.V % 8)
      if (int rc = pack<T>(a.dy, a.yb, a.yt, a.yh, a.B, a.T, a.H, a.V, a.Vp, ws + s.dy, st)) return rc;
    if (int rc = with_keys(a.K, [&](auto dk) {
          constexpr int DK = decltype(dk)::value;
          // Eight waves for 128 columns spare partial results of dq and dk, and a second product of q and k.  4 x 2048 x 16,
          // bf16, both passes: 32 keys and 128 values 164 us and 194, 64 199 and 278, 128 288 and 545; fp16, 128: 425
          // and 693.  In fp32 three parts of 128 keys and of 128 values do not fit into LDS.
          if constexpr (!std::is_same_v<T, float>)
            if (a.V > VT) return run_bwd<T, DK, 8>(a, st);
          return run_bwd<T, DK, 4>(a, st);
        }))
      return rc;
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
