// Layer norm over the last dimension and its backward pass with the weight's and bias' gradients
// (nn.LayerNorm, the LayerNorm choice of build_lngram_norm, ffnmem/memory/lngram_v2.py:56-71).
//
//   xn = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xn * w + b
//   g = dy * w,  dx = rstd * (g - mean(g) - xn * mean(g * xn)),  dw = sum_rows dy * xn,  db = sum_rows dy
//
// Both directions are bound by memory: a row is read once and stays in registers between its statistics
// and its output (the variance is formed from the centred row, so rows with a large mean lose nothing).
// LPR lanes hold a row, 8 elements a load.  A block walks over many rows, so that the weights are read
// once per block, and in the backward pass the weight gradients of a thread's columns stay in registers
// over all of the block's rows: they leave as one partial row per block, summed in a fixed order by
// k_norm_partials (no atomics: the result of a call does not vary).
// bf16: 16384 x 1024 13 us (67 MB) forward, 19 backward (68 MB read, 38 written, 5.5 TB/s) and 4 for the partial rows;
// 421911 x 256 78 us, 5.5 TB/s.  Every input byte is read once; a copy, which runs past the Infinity Cache, reaches 4.9.
#include "common.h"

namespace lng {
namespace {

constexpr int VEC = 8;

// V neighbouring elements: eight, aligned to 16 bytes, or one.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 2) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 r = *reinterpret_cast<const T8*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(r[i]);
  } else {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 2) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r[i] = from_f32<T>(v[i]);
    *reinterpret_cast<T8*>(p) = r;
  } else {
    f32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = v[i], b[i] = v[i + 4];
    reinterpret_cast<f32x4*>(p)[0] = a, reinterpret_cast<f32x4*>(p)[1] = b;
  }
}

// Sum over the LPR threads that hold a row, in every one of them.  LPR > 64: the whole block, through
// `red` (one float per wave; the barriers also separate successive uses).
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (LPR < 64) {
#pragma unroll
    for (int m = LPR / 2; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
  } else if constexpr (LPR == 64) {
    return wave_sum(v);
  } else {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < LPR / 64; ++i) s += red[i];
    return s;
  }
}

// A thread's columns of a row: element i of chunk j is column (lane + LPR * j) * V + i.  Single elements are
// asked for without branches (the last one again behind a row's end), so that all are on their way together.
template <typename T, int LPR, int NV, int V>
__device__ __forceinline__ void load_row(const T* p, int lane, int chunks, float (&v)[NV][V]) {
  if constexpr (V == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) load_v<T, V>(p + (lane + LPR * j < chunks ? lane + LPR * j : chunks - 1), v[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j][0] = lane + LPR * j < chunks ? v[j][0] : 0.f;
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + LPR * j;
    if (c < chunks) {
      load_v<T, V>(p + c * V, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = 0.f;
    }
  }
}

template <typename T, typename W, int LPR, int NV, int V>
__global__ __launch_bounds__(256) void k_layer_norm(const T* __restrict__ x, int64_t rows, int d, int64_t xs,
                                                    const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                    T* __restrict__ y, float* __restrict__ mean_out,
                                                    float* __restrict__ rstd_out) {
  constexpr int RPB = 256 / LPR;
  __shared__ float red[4];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR, chunks = d / V;
  const float inv_d = 1.f / static_cast<float>(d);
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) wv[j][i] = 1.f, bv[j][i] = 0.f;
  if (w) load_row<W, LPR, NV, V>(w, lane, chunks, wv);
  if (b) load_row<W, LPR, NV, V>(b, lane, chunks, bv);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * RPB; base < rows; base += static_cast<int64_t>(gridDim.x) * RPB) {
    const bool ok = base + slot < rows;
    const int64_t row = ok ? base + slot : rows - 1;
    float v[NV][V];
    load_row<T, LPR, NV, V>(x + row * xs, lane, chunks, v);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    const float mean = row_sum<LPR>(s, red) * inv_d;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (lane + LPR * j < chunks) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] -= mean, s += v[j][i] * v[j][i];
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<LPR>(s, red) * inv_d + eps);
    if (ok) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = lane + LPR * j;
        if (c < chunks) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * rstd * wv[j][i] + bv[j][i];
          store_v<T, V>(y + row * d + c * V, v[j]);
        }
      }
      if (lane == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
    }
  }
}

// One block per row, any width and alignment: the row is read three times (the second and third from the
// caches).  Widths past 8192 (2048 x 8200 46 us forward, 124 with its backward; 2048 x 8192 18 and 56).
template <typename T, typename W>
__global__ __launch_bounds__(256) void k_layer_norm_any(const T* __restrict__ x, int64_t rows, int64_t d, int64_t xs,
                                                        const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                        T* __restrict__ y, float* __restrict__ mean_out,
                                                        float* __restrict__ rstd_out) {
  __shared__ float red[4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* p = x + row * xs;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += 256) s += to_f32(p[c]);
    const float mean = row_sum<256>(s, red) / static_cast<float>(d);
    s = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += 256) {
      const float v = to_f32(p[c]) - mean;
      s += v * v;
    }
    const float rstd = 1.f / sqrtf(row_sum<256>(s, red) / static_cast<float>(d) + eps);
    for (int64_t c = threadIdx.x; c < d; c += 256) {
      const float xn = (to_f32(p[c]) - mean) * rstd;
      y[row * d + c] = from_f32<T>(xn * (w ? to_f32(w[c]) : 1.f) + (b ? to_f32(b[c]) : 0.f));
    }
    if (threadIdx.x == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <typename T, typename W, int LPR, int NV, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void k_layer_norm_grad(const T* __restrict__ dy, int64_t dys,
                                                             const T* __restrict__ x, int64_t xs, int64_t rows, int d,
                                                             const W* __restrict__ w, const float* __restrict__ mean_in,
                                                             const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                             float* __restrict__ partial) {
  constexpr int RPB = THREADS / LPR;
  __shared__ float red[2][THREADS / 64];
  __shared__ float cols[RPB > 1 ? THREADS * NV * V : 1];
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR, chunks = d / V;
  const float inv_d = 1.f / static_cast<float>(d);
  float wv[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) wv[j][i] = 1.f, dw[j][i] = 0.f, db[j][i] = 0.f;
  if (w) load_row<W, LPR, NV, V>(w, lane, chunks, wv);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * RPB; base < rows; base += static_cast<int64_t>(gridDim.x) * RPB) {
    const bool ok = base + slot < rows;
    const int64_t row = ok ? base + slot : rows - 1;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float v[NV][V], g[NV][V];
    load_row<T, LPR, NV, V>(x + row * xs, lane, chunks, v);
    load_row<T, LPR, NV, V>(dy + row * dys, lane, chunks, g);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xn = (v[j][i] - mean) * rstd, gy = ok ? g[j][i] : 0.f;
        dw[j][i] += gy * xn;
        db[j][i] += gy;
        g[j][i] *= wv[j][i];
        s1 += g[j][i];
        s2 += g[j][i] * xn;
        v[j][i] = xn;
      }
    s1 = row_sum<LPR>(s1, red[0]) * inv_d;
    s2 = row_sum<LPR>(s2, red[1]) * inv_d;
    if (ok && dx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = lane + LPR * j;
        if (c < chunks) {
#pragma unroll
          for (int i = 0; i < V; ++i) g[j][i] = rstd * (g[j][i] - s1 - v[j][i] * s2);
          store_v<T, V>(dx + row * d + c * V, g[j]);
        }
      }
    }
  }
  if (!partial) return;
  float* const out = partial + static_cast<int64_t>(blockIdx.x) * 2 * d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (RPB == 1) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (lane + LPR * j < chunks) store_v<float, V>(out + which * d + (lane + LPR * j) * V, which ? db[j] : dw[j]);
    } else {
      // the block's row slots are merged in LDS, each column by one thread, in the order of the slots
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j) store_v<float, V>(cols + (slot * LPR * NV + lane + LPR * j) * V, which ? db[j] : dw[j]);
      __syncthreads();
      for (int c = threadIdx.x; c < d; c += THREADS) {
        float s = 0.f;
        for (int r = 0; r < RPB; ++r) s += cols[r * LPR * NV * V + c];
        out[which * d + c] = s;
      }
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void k_layer_norm_grad_any(const T* __restrict__ dy, int64_t dys,
                                                             const T* __restrict__ x, int64_t xs, int64_t rows,
                                                             int64_t d, const W* __restrict__ w,
                                                             const float* __restrict__ mean_in,
                                                             const float* __restrict__ rstd_in, T* __restrict__ dx) {
  __shared__ float red[2][4];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *p = x + row * xs, *q = dy + row * dys;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += 256) {
      const float g = to_f32(q[c]) * (w ? to_f32(w[c]) : 1.f);
      s1 += g;
      s2 += g * ((to_f32(p[c]) - mean) * rstd);
    }
    s1 = row_sum<256>(s1, red[0]) / static_cast<float>(d);
    s2 = row_sum<256>(s2, red[1]) / static_cast<float>(d);
    for (int64_t c = threadIdx.x; c < d; c += 256) {
      const float g = to_f32(q[c]) * (w ? to_f32(w[c]) : 1.f), xn = (to_f32(p[c]) - mean) * rstd;
      dx[row * d + c] = from_f32<T>(rstd * (g - s1 - xn * s2));
    }
  }
}

// Column sums of dy * xn and dy over a slice of the rows: block (x: 256 columns, y: slice).
template <typename T>
__global__ __launch_bounds__(256) void k_layer_norm_cols_any(const T* __restrict__ dy, int64_t dys,
                                                             const T* __restrict__ x, int64_t xs, int64_t rows,
                                                             int64_t d, const float* __restrict__ mean_in,
                                                             const float* __restrict__ rstd_in,
                                                             float* __restrict__ partial) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= d) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float g = to_f32(dy[row * dys + c]);
    dw += g * ((to_f32(x[row * xs + c]) - mean_in[row]) * rstd_in[row]);
    db += g;
  }
  float* const out = partial + static_cast<int64_t>(blockIdx.y) * 2 * d;
  out[c] = dw;
  out[d + c] = db;
}

// dw[c], db[c] = the sums over the P partial rows [P, 2, d]: 16 columns a block, 16 threads a column.
template <typename W>
__global__ __launch_bounds__(256) void k_norm_partials(const float* __restrict__ partial, int P, int64_t d,
                                                       W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float part[16][17];
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + col;
  float s = 0.f;
  if (m < 2 * d) {
#pragma unroll 8
    for (int p = grp; p < P; p += 16) s += partial[static_cast<int64_t>(p) * 2 * d + m];
  }
  part[grp][col] = s;
  __syncthreads();
  if (grp == 0 && m < 2 * d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][col];
    if (m < d) {
      if (dw) dw[m] = from_f32<W>(s);
    } else if (db) {
      db[m - d] = from_f32<W>(s);
    }
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Whether 8-element loads serve these rows.
bool vector_rows(const void* p, int64_t stride, int64_t d, int es) {
  return aligned16(p) && stride * es % 16 == 0 && d % VEC == 0;
}

constexpr int64_t MAX_ROW_D = 8192;  // a row in the registers of 256 threads
constexpr int64_t GRAD_BLOCKS = 512;  // two blocks of 8 waves per CU

// Blocks of the backward pass, each leaving one partial row of the weight gradients.
int64_t grad_blocks(int64_t rows, int64_t d) {
  const int64_t rpb = d <= 32 ? 128 : d <= 128 ? 32 : d <= 256 ? 16 : d <= 2048 ? 8 : 1;
  const int64_t most = std::min(GRAD_BLOCKS, (int64_t{1} << 26) / d);  // very wide rows: partial rows of 512 MB at most
  return std::max<int64_t>(1, std::min(cdiv(rows, rpb), most));
}

struct Rows {  // one call's rows
  const void *x, *dy, *w, *b;
  int64_t xs, dys, rows, d;
  float eps;
  void *y, *dx, *dw, *db;
  float *mean, *rstd, *partial;
  hipStream_t st;
};

template <typename T, typename W, int LPR, int NV, int V>
void launch_fwd(const Rows& r) {
  constexpr int rpb = 256 / LPR;
  const int64_t grid = std::min<int64_t>(cdiv(r.rows, rpb), 2048);
  k_layer_norm<T, W, LPR, NV, V><<<static_cast<unsigned>(grid), 256, 0, r.st>>>(
      static_cast<const T*>(r.x), r.rows, static_cast<int>(r.d), r.xs, static_cast<const W*>(r.w),
      static_cast<const W*>(r.b), r.eps, static_cast<T*>(r.y), r.mean, r.rstd);
}

template <typename T, typename W, int LPR, int NV, int V>
void launch_bwd(const Rows& r) {
  constexpr int threads = LPR > 64 ? LPR : 512;
  k_layer_norm_grad<T, W, LPR, NV, V, threads><<<static_cast<unsigned>(grad_blocks(r.rows, r.d)), threads, 0, r.st>>>(
      static_cast<const T*>(r.dy), r.dys, static_cast<const T*>(r.x), r.xs, r.rows, static_cast<int>(r.d),
      static_cast<const W*>(r.w), r.mean, r.rstd, static_cast<T*>(r.dx), r.partial);
}

// VECTOR: 8 elements a load.  Else one, for other widths or alignments: 100000 x 37 11 us, where a block a row took
// 80, 16384 x 1001 19 and 47, the training of 100000 x 37 25 and 216.
template <typename T, typename W, bool BWD, bool VECTOR>
void launch_shape(const Rows& r) {
#define LNG_NORM_SHAPE(limit, LPR, NV, V) \
  if (r.d <= limit) {                     \
    if constexpr (BWD)                    \
      launch_bwd<T, W, LPR, NV, V>(r);    \
    else                                  \
      launch_fwd<T, W, LPR, NV, V>(r);    \
    return;                               \
  }
  if constexpr (VECTOR) {
    LNG_NORM_SHAPE(32, 4, 1, VEC)
    LNG_NORM_SHAPE(128, 16, 1, VEC)
    LNG_NORM_SHAPE(256, 32, 1, VEC)
    LNG_NORM_SHAPE(512, 64, 1, VEC)
    LNG_NORM_SHAPE(1024, 64, 2, VEC)
    LNG_NORM_SHAPE(2048, 64, 4, VEC)
    LNG_NORM_SHAPE(4096, 256, 2, VEC)
    LNG_NORM_SHAPE(8192, 256, 4, VEC)
  } else {
    LNG_NORM_SHAPE(16, 16, 1, 1)
    LNG_NORM_SHAPE(64, 16, 4, 1)
    LNG_NORM_SHAPE(256, 64, 4, 1)
    LNG_NORM_SHAPE(512, 64, 8, 1)
    LNG_NORM_SHAPE(1024, 64, 16, 1)
    LNG_NORM_SHAPE(2048, 256, 8, 1)
    LNG_NORM_SHAPE(4096, 256, 16, 1)
    LNG_NORM_SHAPE(8192, 256, 32, 1)
  }
#undef LNG_NORM_SHAPE
}

template <typename T, typename W>
int run_fwd(const Rows& r) {
  const bool vec = vector_rows(r.x, r.xs, r.d, sizeof(T)) && aligned16(r.y) && aligned16(r.w) &&
                   aligned16(r.b);
  if (r.d <= MAX_ROW_D && vec)
    launch_shape<T, W, false, true>(r);
  else if (r.d <= MAX_ROW_D)
    launch_shape<T, W, false, false>(r);
  else
    k_layer_norm_any<T, W><<<static_cast<unsigned>(std::min<int64_t>(r.rows, 8192)), 256, 0, r.st>>>(
        static_cast<const T*>(r.x), r.rows, r.d, r.xs, static_cast<const W*>(r.w), static_cast<const W*>(r.b), r.eps,
        static_cast<T*>(r.y), r.mean, r.rstd);
  return check_launch("layer_norm");
}

template <typename T, typename W>
int run_bwd(const Rows& r) {
  const bool vec = vector_rows(r.x, r.xs, r.d, sizeof(T)) &&
                   vector_rows(r.dy, r.dys, r.d, sizeof(T)) && aligned16(r.dx) && aligned16(r.w);
  int64_t P = grad_blocks(r.rows, r.d);
  if (r.d <= MAX_ROW_D && vec) {
    launch_shape<T, W, true, true>(r);
  } else if (r.d <= MAX_ROW_D) {
    launch_shape<T, W, true, false>(r);
  } else {
    const T *dy = static_cast<const T*>(r.dy), *x = static_cast<const T*>(r.x);
    if (r.dx) {
      k_layer_norm_grad_any<T, W><<<static_cast<unsigned>(std::min<int64_t>(r.rows, 8192)), 256, 0, r.st>>>(
          dy, r.dys, x, r.xs, r.rows, r.d, static_cast<const W*>(r.w), r.mean, r.rstd, static_cast<T*>(r.dx));
      if (int rc = check_launch("layer_norm_grad")) return rc;
    }
    if (r.partial)
      k_layer_norm_cols_any<T><<<dim3(static_cast<unsigned>(cdiv(r.d, 256)), static_cast<unsigned>(P)), 256, 0, r.st>>>(
          dy, r.dys, x, r.xs, r.rows, r.d, r.mean, r.rstd, r.partial);
  }
  if (int rc = check_launch("layer_norm_grad")) return rc;
  if (!r.partial) return LNG_OK;
  k_norm_partials<W><<<static_cast<unsigned>(cdiv(2 * r.d, 16)), 256, 0, r.st>>>(
      r.partial, static_cast<int>(P), r.d, static_cast<W*>(r.dw), static_cast<W*>(r.db));
  return check_launch("layer_norm_grad");
}

int check_rows(const char* what, int dtype, int w_dtype, int64_t rows, int64_t d, int64_t xs) {
  if (dtype != LNG_F32 && dtype != LNG_BF16 && dtype != LNG_F16)
    return fail(LNG_E_DTYPE, std::string(what) + ": fp32, bf16 or fp16 rows");
  if (w_dtype != dtype && w_dtype != LNG_F32)
    return fail(LNG_E_DTYPE, std::string(what) + ": weights in the rows' type or fp32");
  if (rows < 0 || d <= 0 || d > (int64_t{1} << 24) || (rows > 1 && xs < 0))
    return fail(LNG_E_ARG, std::string(what) + ": bad shape");
  return LNG_OK;
}

template <typename F>
int with_types(int dtype, int w_dtype, F f) {
  if (dtype == LNG_F32) return f(float{}, float{});
  if (dtype == LNG_BF16) return w_dtype == LNG_F32 ? f(bf16{}, float{}) : f(bf16{}, bf16{});
  return w_dtype == LNG_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
}

}  // namespace
}  // namespace lng

using namespace lng;

extern "C" {

int lng_layer_norm(const void* x, int dtype, int64_t rows, int64_t d, int64_t x_stride, const void* w, const void* b,
                   int w_dtype, float eps, void* y, float* mean, float* rstd, void* stream) {
  if (int rc = check_rows("layer_norm", dtype, w_dtype, rows, d, x_stride)) return rc;
  if (rows == 0) return LNG_OK;
  if (!x || !y || !mean != !rstd) return fail(LNG_E_ARG, "layer_norm: null pointer");
  Rows r{x, nullptr, w, b, x_stride, 0, rows, d, eps, y, nullptr, nullptr, nullptr, mean, rstd, nullptr,
         as_stream(stream)};
  return with_types(dtype, w_dtype, [&](auto t, auto wt) { return run_fwd<decltype(t), decltype(wt)>(r); });
}

size_t lng_layer_norm_grad_workspace_bytes(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return static_cast<size_t>(grad_blocks(rows, d)) * 2 * static_cast<size_t>(d) * 4;
}

int lng_layer_norm_grad(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int dtype, int64_t rows,
                        int64_t d, const void* w, int w_dtype, const float* mean, const float* rstd, void* workspace,
                        size_t workspace_bytes, void* dx, void* dw, void* db, void* stream) {
  if (int rc = check_rows("layer_norm_grad", dtype, w_dtype, rows, d, x_stride)) return rc;
  if (rows > 1 && dy_stride < 0) return fail(LNG_E_ARG, "layer_norm_grad: bad shape");
  hipStream_t st = as_stream(stream);
  const bool cols = dw || db;
  if (rows == 0) {  // no rows: the weights' gradients are zero, formed from no partial rows
    if (!cols) return LNG_OK;
    const unsigned grid = static_cast<unsigned>(cdiv(2 * d, 16));
    return with_types(dtype, w_dtype, [&](auto, auto wt) {
      using W = decltype(wt);
      k_norm_partials<W><<<grid, 256, 0, st>>>(nullptr, 0, d, static_cast<W*>(dw), static_cast<W*>(db));
      return check_launch("layer_norm_grad");
    });
  }
  if (!dy || !x || !mean || !rstd) return fail(LNG_E_ARG, "layer_norm_grad: null pointer");
  if (cols && (!workspace || !aligned16(workspace) || workspace_bytes < lng_layer_norm_grad_workspace_bytes(rows, d)))
    return fail(LNG_E_ARG, "layer_norm_grad: the workspace is too small or not 16-byte aligned");
  Rows r{x, dy, w, nullptr, x_stride, dy_stride, rows, d, 0.f, nullptr, dx, dw, db, const_cast<float*>(mean),
         const_cast<float*>(rstd), cols ? static_cast<float*>(workspace) : nullptr, st};
  return with_types(dtype, w_dtype, [&](auto t, auto wt) { return run_bwd<decltype(t), decltype(wt)>(r); });
}

}  // extern "C"
