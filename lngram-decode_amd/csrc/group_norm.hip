// Group norm with an activation, channels last, and its backward pass: LayerNorm's choice for groups of channels
// (nn.GroupNorm on rows whose channels lie together), over all positions of a sample.
//
//   x [N, L, C], a group of cg = C / G neighbouring channels, statistics over its L cg values of a sample
//   xn = (x - mean) rstd,  z = xn w + b,  y = z or silu(z)
//   dz = dy silu'(z),  h = dz w,  dx = rstd (h - mean(h) - xn mean(h xn)),  dw = sum dz xn,  db = sum dz
//
// All of it is bound by memory.  Three forms:
// - one position a sample (a token's heads, each normed on its own): a group is a short row, held by LPR lanes as layer
//   norm holds its rows; a lane keeps the same channels of the same group from sample to sample, so that weights are
//   read, and their gradients added up, in registers.  32768 x 1024 in 16 groups, bf16, with silu: 28 us, 4.8 TB/s (a copy:
//   5.1); the backward of 16384 x 1024 27 us, 4.1 TB/s with its partial rows.
// - samples that a block's registers hold: threads over positions and channels, statistics through LDS, one pass.
// - larger ones: blocks over ranges of positions leave (mean, sum of squares around it) of their values, a small launch
//   joins them, and the second pass finds part of what the first one read in the caches.  8 x 4096 x 320 in 32 groups: 11 +
//   6 + 11 us, 1.9 TB/s in the first pass, 4.0 in the second.  (Joined by every block of the second pass for itself they
//   took longer than the launch.)
// The variance is always formed around a mean, never as a difference of squares.  Sums are fp32 in a fixed order: no
// atomics, equal calls give equal bits.
#include "common.h"

#include <algorithm>

namespace lng {
namespace {

constexpr int VEC = 8;
constexpr int MAX_ROW = 8192;           // channels of a group held by a block's threads
constexpr int MOST_CHUNKS = 1024;       // a sample's ranges of positions

struct Gn {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float *mean, *rstd;   // [N, G]
  float* stats;         // [N, chunks, G + slabs, 2]: group g's part of slab s at g + s (a slab's first group may be shared)
  float* cols;          // [P, 2, C] partial gradients of w and b
  int64_t N, L, xs, xl, dys, dyl;
  int C, G, cg, wdt;
  bool act;
  float eps;
  // blocks over positions and channels
  int slab, slabs, chunks;
  int64_t chunk_rows;
  __host__ __device__ int64_t parts() const { return int64_t{G} + slabs; }  // of a chunk: a place for each group and boundary
};

template <typename T, int V>
struct Raw {
  T v[V] __attribute__((aligned(sizeof(T) * V)));
};
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  if constexpr (V == 1) {
    return {{*p}};
  } else {
    Raw<T, V> r;
    u32x4* to = reinterpret_cast<u32x4*>(&r);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) to[i] = reinterpret_cast<const u32x4*>(p)[i];
    return r;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_raw(T* p, const float (&v)[V]) {
  Raw<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = from_f32<T>(v[i]);
  if constexpr (V == 1) {
    *p = r.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i)
      reinterpret_cast<u32x4*>(p)[i] = reinterpret_cast<const u32x4*>(&r)[i];
  }
}
__device__ __forceinline__ float weight(const void* w, int dt, int64_t i, float none) {
  if (!w) return none;
  if (dt == LNG_F32) return static_cast<const float*>(w)[i];
  if (dt == LNG_BF16) return to_f32(static_cast<const bf16*>(w)[i]);
  return to_f32(static_cast<const _Float16*>(w)[i]);
}
// V neighbouring weights, 16 bytes at a time where they allow it; `none` where there are none
template <int V>
__device__ __forceinline__ void weights(const void* w, int dt, int64_t i, float none, float (&v)[V]) {
  if constexpr (V > 1) {
    if (w && reinterpret_cast<uintptr_t>(w) % 16 == 0) {
      if (dt == LNG_F32) {
        const Raw<float, V> r = load_raw<float, V>(static_cast<const float*>(w) + i);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = r.v[k];
      } else if (dt == LNG_BF16) {
        const Raw<bf16, V> r = load_raw<bf16, V>(static_cast<const bf16*>(w) + i);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = to_f32(r.v[k]);
      } else {
        const Raw<_Float16, V> r = load_raw<_Float16, V>(static_cast<const _Float16*>(w) + i);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = to_f32(r.v[k]);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = weight(w, dt, i + k, none);
}
// dy silu'(z)
__device__ __forceinline__ float slope(float dy, float z) {
  const float s = sigmoid(z);
  return dy * s * fmaf(z, 1.f - s, 1.f);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (LPR < 64) {
#pragma unroll
    for (int m = LPR / 2; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
  } else if constexpr (LPR == 64) {
    return wave_sum(v);
  } else {  // the whole block; the barriers also separate successive uses
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

// ------------------------------------------------------------------ one position a sample
// A block's slots of LPR lanes: `gs` groups of `si` samples; blocks over slabs of gs groups and over samples.
struct Slots {
  int gs, per, slabs;  // groups and samples of a block at a time, slabs of groups
  __host__ __device__ Slots(int G, int slots) : gs(G < slots ? G : slots), per(slots / gs), slabs((G + gs - 1) / gs) {}
};

// A lane's part of a group as it is in memory: the next one is asked for before this one is worked on
template <typename T, int LPR, int NV, int V>
struct Held {
  Raw<T, V> r[NV];
  __device__ __forceinline__ void load(const T* p, int lane, int vecs) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + LPR * j;
      r[j] = load_raw<T, V>(p + (c < vecs ? c : 0) * V);  // no branch: all of them on their way together
    }
  }
  __device__ __forceinline__ void values(int lane, int vecs, float (&v)[NV][V]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = lane + LPR * j < vecs ? to_f32(r[j].v[i]) : 0.f;
  }
};

template <typename T, int LPR, int NV, int V>
__global__ __launch_bounds__(256) void k_gn_rows(Gn a) {
  __shared__ float red[4];
  const Slots sl(a.G, 256 / LPR);
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR, vecs = a.cg / V;
  const int64_t first = int64_t{blockIdx.x} / sl.slabs * sl.per + slot / sl.gs;
  const int64_t step = int64_t{gridDim.x} / sl.slabs * sl.per;
  const int g = static_cast<int>(blockIdx.x % sl.slabs) * sl.gs + slot % sl.gs;
  if (slot >= sl.per * sl.gs || g >= a.G || first >= a.N) return;  // LPR > 64 has one slot: nobody leaves a barrier behind
  const float inv = 1.f / static_cast<float>(a.cg);
  const T* x = static_cast<const T*>(a.x) + int64_t{g} * a.cg;
  Held<T, LPR, NV, V> next;
  next.load(x + first * a.xs, lane, vecs);
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + LPR * j < vecs ? (lane + LPR * j) * V : 0;
    weights<V>(a.w, a.wdt, int64_t{g} * a.cg + c, 1.f, wv[j]);
    weights<V>(a.b, a.wdt, int64_t{g} * a.cg + c, 0.f, bv[j]);
  }
  for (int64_t n = first; n < a.N; n += step) {
    float v[NV][V];
    next.values(lane, vecs, v);
    if (n + step < a.N) next.load(x + (n + step) * a.xs, lane, vecs);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    const float mean = row_sum<LPR>(s, red) * inv;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool own = lane + LPR * j < vecs;
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = own ? v[j][i] - mean : 0.f, s = fmaf(v[j][i], v[j][i], s);
    }
    const float rstd = 1.f / sqrtf(fmaf(row_sum<LPR>(s, red), inv, a.eps));
    T* y = static_cast<T*>(a.y) + n * a.C + int64_t{g} * a.cg;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (lane + LPR * j >= vecs) break;
      float out[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = fmaf(v[j][i] * rstd, wv[j][i], bv[j][i]);
        out[i] = a.act ? silu<T>(z) : z;
      }
      store_raw<T, V>(y + (lane + LPR * j) * V, out);
    }
    if (a.mean && lane == 0) a.mean[n * a.G + g] = mean, a.rstd[n * a.G + g] = rstd;
  }
}

template <typename T, int LPR, int NV, int V>
__global__ __launch_bounds__(256) void k_gn_rows_grad(Gn a) {
  __shared__ float red[4];
  extern __shared__ float sums[];  // [2][256 NV V]
  const Slots sl(a.G, 256 / LPR);
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR, vecs = a.cg / V;
  const int64_t first = int64_t{blockIdx.x} / sl.slabs * sl.per + slot / sl.gs;
  const int64_t step = int64_t{gridDim.x} / sl.slabs * sl.per;
  const int g = static_cast<int>(blockIdx.x % sl.slabs) * sl.gs + slot % sl.gs;
  const bool on = slot < sl.per * sl.gs && g < a.G && first < a.N;
  const float inv = 1.f / static_cast<float>(a.cg);
  const T *x = static_cast<const T*>(a.x) + int64_t{g} * a.cg, *dy = static_cast<const T*>(a.dy) + int64_t{g} * a.cg;
  float wv[NV][V], bv[NV][V], dw[NV][V], db[NV][V];
  Held<T, LPR, NV, V> nx, nd;
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t n) {
    nx.load(x + n * a.xs, lane, vecs), nd.load(dy + n * a.dys, lane, vecs);
    nmean = a.mean[n * a.G + g], nrstd = a.rstd[n * a.G + g];
  };
  if (on) fetch(first);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + LPR * j < vecs ? (lane + LPR * j) * V : 0, gc = on ? g : 0;
    weights<V>(a.w, a.wdt, int64_t{gc} * a.cg + c, 1.f, wv[j]);
    weights<V>(a.b, a.wdt, int64_t{gc} * a.cg + c, 0.f, bv[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  for (int64_t n = on ? first : a.N; n < a.N; n += step) {
    float v[NV][V], h[NV][V];
    nx.values(lane, vecs, v), nd.values(lane, vecs, h);  // dy is zero behind the group's end
    const float mean = nmean, rstd = nrstd;
    if (n + step < a.N) fetch(n + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] = (v[j][i] - mean) * rstd;
        const float dz = a.act ? slope(h[j][i], fmaf(v[j][i], wv[j][i], bv[j][i])) : h[j][i];
        dw[j][i] = fmaf(dz, v[j][i], dw[j][i]), db[j][i] += dz;
        h[j][i] = dz * wv[j][i];
        s1 += h[j][i], s2 = fmaf(h[j][i], v[j][i], s2);
      }
    s1 = row_sum<LPR>(s1, red) * inv;
    s2 = row_sum<LPR>(s2, red) * inv;
    if (a.dx) {
      T* dx = static_cast<T*>(a.dx) + n * a.C + int64_t{g} * a.cg;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (lane + LPR * j >= vecs) break;
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = rstd * (h[j][i] - s1 - v[j][i] * s2);
        store_raw<T, V>(dx + (lane + LPR * j) * V, out);
      }
    }
  }
  if (!a.cols) return;
  // the samples of a block, slot by slot, into its partial row
  constexpr int W = LPR * NV * V, HALF = 256 / LPR * W;
  if constexpr (LPR <= 64) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int at = slot * W + (lane + LPR * j) * V + i;
        sums[at] = dw[j][i], sums[HALF + at] = db[j][i];
      }
    __syncthreads();
  }
  if (slot >= sl.gs || g >= a.G) return;
  float* to = a.cols + int64_t{blockIdx.x} / sl.slabs * 2 * a.C + int64_t{g} * a.cg;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + LPR * j) * V + i;
      if (c >= a.cg) continue;
      float x = dw[j][i], y = db[j][i];
      if constexpr (LPR <= 64)
        for (int k = 1; k < sl.per; ++k) x += sums[(slot + k * sl.gs) * W + c], y += sums[HALF + (slot + k * sl.gs) * W + c];
      to[c] = x, to[a.C + c] = y;
    }
}

// ------------------------------------------------------------------ blocks over positions and channels
// A block's slab, range of positions and sample
struct Place {
  int slab, chunk;
  int64_t n;
  __device__ explicit Place(const Gn& a) {
    const uint32_t slabs = a.slabs, chunks = a.chunks, u = blockIdx.x / slabs;
    slab = blockIdx.x - u * slabs, n = u / chunks, chunk = u - static_cast<uint32_t>(n) * chunks;
  }
};

// A thread has V neighbouring channels of a slab and every RL-th position.
template <int V>
struct Tile {
  int c0, width, cv, rl, RL;  // first channel and channels of the slab; this thread's vector and first position
  int g0, groups;             // groups that the slab touches
  bool on;
  int c;                      // this thread's first channel
  int gk[V];                  // its channels' groups, from g0
  __device__ Tile(const Gn& a, int slab) {
    c0 = slab * a.slab, width = min(a.slab, a.C - c0);
    const int CV = width / V;
    RL = 256 / CV, cv = static_cast<int>(threadIdx.x) % CV, rl = static_cast<int>(threadIdx.x) / CV, on = rl < RL;
    g0 = c0 / a.cg, groups = (c0 + width - 1) / a.cg - g0 + 1;
    c = c0 + cv * V;
    int g = c / a.cg, rest = c - g * a.cg;  // one division: they are slow
#pragma unroll
    for (int i = 0; i < V; ++i) {
      gk[i] = g - g0;
      if (++rest == a.cg) rest = 0, ++g;
    }
  }
  // channels of group gi within the slab: [from, to)
  __device__ int from(const Gn& a, int gi) const { return max((g0 + gi) * a.cg - c0, 0); }
  __device__ int to(const Gn& a, int gi) const { return min((g0 + gi + 1) * a.cg - c0, width); }
};

template <int V>
struct TileLds {
  alignas(16) float one[256 * V], two[256 * V];    // values a (position lane, channel), of two kinds
  float mean[256 * V], m2[256 * V];    // of a group: mean and sum of squares around it (or sums of two kinds)
};

// V neighbouring floats into LDS, 16 bytes at a time (one by one they would meet on the same banks)
template <int V>
__device__ __forceinline__ void put_row(float* at, const float (&v)[V]) {
  if constexpr (V == 1) {
    *at = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<f32x4*>(at + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  }
}

// Two values a (position, channel), summed over the positions: into lds.one and lds.two by channel
template <int V>
__device__ __forceinline__ void channel_sums(TileLds<V>& lds, const Tile<V>& t, const float (&x)[V], const float (&y)[V]) {
  __syncthreads();
  if (t.on) {
    put_row<V>(&lds.one[t.rl * t.width + t.cv * V], x);
    put_row<V>(&lds.two[t.rl * t.width + t.cv * V], y);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < t.width; c += 256) {
    float s = lds.one[c], u = lds.two[c];
#pragma unroll 8
    for (int r = 1; r < t.RL; ++r) s += lds.one[r * t.width + c], u += lds.two[r * t.width + c];
    lds.one[c] = s, lds.two[c] = u;  // this thread's column
  }
  __syncthreads();
}
// f(group, sums of lds.one and lds.two over the group's channels in the slab, times w), by one thread each
template <int V, typename F>
__device__ __forceinline__ void group_sums(const TileLds<V>& lds, const Tile<V>& t, const Gn& a, F f) {
  const int lg = a.cg >= 256 ? 64 : 16, lane = threadIdx.x % lg;
  for (int gi = threadIdx.x / lg; gi < t.groups; gi += 256 / lg) {
    float s = 0.f, u = 0.f;
    const int to = t.to(a, gi);
    for (int c = t.from(a, gi) + lane; c < to; c += lg) {
      const float w = weight(a.w, a.wdt, t.c0 + c, 1.f);
      s = fmaf(lds.one[c], w, s), u = fmaf(lds.two[c], w, u);
    }
    for (int m = lg / 2; m; m >>= 1) s += __shfl_xor(s, m), u += __shfl_xor(u, m);
    if (lane == 0) f(gi, s, u);
  }
}

// A sample's positions l0 + rl, l0 + rl + RL, .. (R of them) in a thread's registers
template <typename T, int V, int R>
__device__ __forceinline__ void load_tile(Raw<T, V> (&v)[R], const T* x, int64_t stride, const Tile<V>& t, int64_t l0, int64_t l1) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t l = l0 + t.rl + int64_t{i} * t.RL;
    if (t.on && l < l1)
      v[i] = load_raw<T, V>(x + l * stride + t.c);
    else
#pragma unroll
      for (int k = 0; k < V; ++k) v[i].v[k] = from_f32<T>(0.f);
  }
}

// Mean and sum of squares around it of the groups in a tile of positions: lds.mean, lds.m2.  Each thread forms both of its
// positions of a channel, a group's lanes join them: one exchange for the two steps.
template <typename T, int V, int R>
__device__ __forceinline__ void tile_stats(TileLds<V>& lds, const Tile<V>& t, const Gn& a, const Raw<T, V> (&v)[R], int64_t l0,
                                           int64_t l1) {
  const int rows = static_cast<int>(l1 - l0);
  const int all = rows / t.RL, more = rows - all * t.RL;  // position lane r has `all` of them, the first `more` one more
  const int mine = all + (t.rl < more);
  const float inv = mine ? 1.f / static_cast<float>(mine) : 0.f;
  __syncthreads();
  if (t.on) {
    float m[V], q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      m[k] = q[k] = 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i) m[k] += to_f32(v[i].v[k]);
      m[k] *= inv;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float d = to_f32(v[i].v[k]) - m[k];
        q[k] = i < mine ? fmaf(d, d, q[k]) : q[k];
      }
    }
    put_row<V>(&lds.one[t.rl * t.width + t.cv * V], m);
    put_row<V>(&lds.two[t.rl * t.width + t.cv * V], q);
  }
  __syncthreads();
  const int lg = a.cg >= 256 ? 64 : 16, lane = threadIdx.x % lg, used = min(t.RL, rows);
  for (int gi = threadIdx.x / lg; gi < t.groups; gi += 256 / lg) {
    const int c0 = t.from(a, gi), c1 = t.to(a, gi);
    const float count = static_cast<float>(rows) * static_cast<float>(c1 - c0);
    float m = 0.f, q = 0.f;
    for (int c = c0 + lane; c < c1; c += lg)
#pragma unroll 8
      for (int r = 0; r < used; ++r) m = fmaf(lds.one[r * t.width + c], static_cast<float>(all + (r < more)), m);

    for (int k = lg / 2; k; k >>= 1) m += __shfl_xor(m, k);
    m /= count;
    for (int c = c0 + lane; c < c1; c += lg)
#pragma unroll 8
      for (int r = 0; r < used; ++r) {
        const float d = lds.one[r * t.width + c] - m;
        q += fmaf(d * d, static_cast<float>(all + (r < more)), lds.two[r * t.width + c]);
      }
    for (int k = lg / 2; k; k >>= 1) q += __shfl_xor(q, k);
    if (lane == 0) lds.mean[gi] = m, lds.m2[gi] = q;
  }
  __syncthreads();
}

template <typename T, int V>
struct Weights {
  float w[V], b[V];
  __device__ Weights(const Gn& a, const Tile<V>& t) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = b[i] = 0.f;
    if (!t.on) return;
    weights<V>(a.w, a.wdt, t.c, 1.f, w);
    weights<V>(a.b, a.wdt, t.c, 0.f, b);
  }
};

template <typename T, int V>
__device__ __forceinline__ void write_row(const Gn& a, const Weights<T, V>& wt, const Raw<T, V>& x, const float (&mean)[V],
                                          const float (&rstd)[V], T* y) {
  float out[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float z = fmaf((to_f32(x.v[k]) - mean[k]) * rstd[k], wt.w[k], wt.b[k]);
    out[k] = a.act ? silu<T>(z) : z;
  }
  store_raw<T, V>(y, out);
}

// Samples that the registers hold
template <typename T, int V, int R>
__global__ __launch_bounds__(256) void k_gn_samples(Gn a) {
  __shared__ TileLds<V> lds;
  const Tile<V> t(a, blockIdx.x % a.slabs);
  const Weights<T, V> wt(a, t);
  const float count = static_cast<float>(a.L) * static_cast<float>(a.cg);
  for (int64_t n = blockIdx.x / a.slabs; n < a.N; n += gridDim.x / a.slabs) {
    Raw<T, V> v[R];
    load_tile(v, static_cast<const T*>(a.x) + n * a.xs, a.xl, t, 0, a.L);
    tile_stats(lds, t, a, v, 0, a.L);
    float mean[V], rstd[V];
#pragma unroll
    for (int k = 0; k < V; ++k) mean[k] = lds.mean[t.gk[k]], rstd[k] = 1.f / sqrtf(lds.m2[t.gk[k]] / count + a.eps);
    if (a.mean)
      for (int gi = threadIdx.x; gi < t.groups; gi += 256) {
        a.mean[n * a.G + t.g0 + gi] = lds.mean[gi];
        a.rstd[n * a.G + t.g0 + gi] = 1.f / sqrtf(lds.m2[gi] / count + a.eps);
      }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t l = t.rl + int64_t{i} * t.RL;
      if (t.on && l < a.L) write_row<T, V>(a, wt, v[i], mean, rstd, static_cast<T*>(a.y) + (n * a.L + l) * a.C + t.c);
    }
  }
}

// Statistics of a range of positions of a slab: (mean, sum of squares around it) a group
template <typename T, int V, int R>
__global__ __launch_bounds__(256) void k_gn_stats(Gn a) {
  __shared__ TileLds<V> lds;
  const Place at(a);
  const Tile<V> t(a, at.slab);
  const int chunk = at.chunk;
  const int64_t n = at.n, l0 = chunk * a.chunk_rows, l1 = min(l0 + a.chunk_rows, a.L);
  float* to = a.stats + ((n * a.chunks + chunk) * a.parts() + at.slab) * 2;
  for (int64_t l = l0; l < l1; l += int64_t{R} * t.RL) {
    const int64_t e = min(l + int64_t{R} * t.RL, l1);
    Raw<T, V> v[R];
    load_tile(v, static_cast<const T*>(a.x) + n * a.xs, a.xl, t, l, e);
    tile_stats(lds, t, a, v, l, e);
    const float before = static_cast<float>(l - l0), rows = static_cast<float>(e - l);
    for (int gi = threadIdx.x; gi < t.groups; gi += 256) {  // joined with the tiles before, which this thread wrote
      float* own = to + 2 * (t.g0 + gi);
      const float width = static_cast<float>(t.to(a, gi) - t.from(a, gi));
      if (l == l0) {
        own[0] = lds.mean[gi], own[1] = lds.m2[gi];
      } else {
        const float d = lds.mean[gi] - own[0], part = rows / (before + rows);
        own[0] = fmaf(d, part, own[0]);
        own[1] += fmaf(d * d, before * part * width, lds.m2[gi]);
      }
    }
  }
}

// Positions of chunk i
__device__ __forceinline__ float chunk_size(const Gn& a, int64_t i) {
  return static_cast<float>(min(a.chunk_rows, a.L - i * a.chunk_rows));
}
// The slabs that hold channels of group g: [first, last]
__device__ __forceinline__ int first_slab(const Gn& a, int g) { return a.slabs == 1 ? 0 : g * a.cg / a.slab; }
__device__ __forceinline__ int last_slab(const Gn& a, int g) { return a.slabs == 1 ? 0 : ((g + 1) * a.cg - 1) / a.slab; }
__device__ __forceinline__ float slab_part(const Gn& a, int g, int s) {  // channels of group g in slab s
  return static_cast<float>(min((g + 1) * a.cg, (s + 1) * a.slab) - max(g * a.cg, s * a.slab));
}

template <int V>
__device__ __forceinline__ void load_stats(const Gn& a, const Tile<V>& t, int64_t n, float (&mean)[V], float (&rstd)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    mean[k] = t.on ? a.mean[n * a.G + t.g0 + t.gk[k]] : 0.f;
    rstd[k] = t.on ? a.rstd[n * a.G + t.g0 + t.gk[k]] : 0.f;
  }
}

// Between the passes: 16 lanes join a group's ranges.  Statistics become mean and rstd; GRAD: sums of h and h xn become
// their means over the group, in the place of its first range.
template <bool GRAD>
__global__ __launch_bounds__(256) void k_gn_join(Gn a, int64_t pairs) {
  const int64_t i = int64_t{blockIdx.x} * 16 + threadIdx.x / 16;
  if (i >= pairs) return;
  const int lane = threadIdx.x & 15;
  const int64_t n = i / a.G;
  const int g = static_cast<int>(i - n * a.G), s0 = first_slab(a, g), ns = last_slab(a, g) - s0 + 1, parts = a.chunks * ns;
  float2* const at = reinterpret_cast<float2*>(a.stats) + n * a.chunks * a.parts() + s0 + g;
  const float count = static_cast<float>(a.L) * static_cast<float>(a.cg);
  const float full = static_cast<float>(a.chunk_rows), last = chunk_size(a, a.chunks - 1);
  auto part = [&](int k, float& size) {
    const int ch = ns == 1 ? k : k / ns, sb = k - ch * ns;
    size = (ch + 1 < a.chunks ? full : last) * (ns == 1 ? static_cast<float>(a.cg) : slab_part(a, g, s0 + sb));
    return at[ch * a.parts() + sb];
  };
  float one = 0.f, two = 0.f, size;
  if constexpr (GRAD) {
#pragma unroll 8
    for (int k = lane; k < parts; k += 16) {
      const float2 p = part(k, size);
      one += p.x, two += p.y;
    }
  } else {
#pragma unroll 8
    for (int k = lane; k < parts; k += 16) {
      const float2 p = part(k, size);
      one = fmaf(p.x, size / count, one);
    }
#pragma unroll
    for (int k = 8; k; k >>= 1) one += __shfl_xor(one, k);
#pragma unroll 8
    for (int k = lane; k < parts; k += 16) {
      const float2 p = part(k, size);
      two += fmaf((p.x - one) * (p.x - one), size, p.y);
    }
  }
#pragma unroll
  for (int k = 8; k; k >>= 1) {
    if (GRAD) one += __shfl_xor(one, k);
    two += __shfl_xor(two, k);
  }
  if (lane) return;
  if (GRAD)
    *at = float2{one / count, two / count};
  else
    a.mean[i] = one, a.rstd[i] = 1.f / sqrtf(two / count + a.eps);
}

// The second pass
template <typename T, int V, int R>
__global__ __launch_bounds__(256) void k_gn_apply(Gn a) {
  const Place at(a);
  const Tile<V> t(a, at.slab);
  if (!t.on) return;
  const int64_t n = at.n, l0 = at.chunk * a.chunk_rows, l1 = min(l0 + a.chunk_rows, a.L);
  const T* x = static_cast<const T*>(a.x) + n * a.xs;
  Raw<T, V> v[R];
  load_tile(v, x, a.xl, t, l0, l1);
  const Weights<T, V> wt(a, t);
  float mean[V], rstd[V];
  load_stats(a, t, n, mean, rstd);
  T* y = static_cast<T*>(a.y) + n * a.L * a.C + t.c;
  for (int64_t l = l0; l < l1; l += int64_t{R} * t.RL) {
    Raw<T, V> now[R];
#pragma unroll
    for (int i = 0; i < R; ++i) now[i] = v[i];
    if (l + int64_t{R} * t.RL < l1) load_tile(v, x, a.xl, t, l + int64_t{R} * t.RL, l1);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = l + t.rl + int64_t{i} * t.RL;
      if (row < l1) write_row<T, V>(a, wt, now[i], mean, rstd, y + row * a.C);
    }
  }
}

// ------------------------------------------------------------------ their backward pass
template <typename T, int V>
struct GradRow {
  float xn[V], dz[V];
  __device__ GradRow(const Gn& a, const Weights<T, V>& wt, const Raw<T, V>& x, const Raw<T, V>& dy, const float (&mean)[V],
                     const float (&rstd)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      xn[k] = (to_f32(x.v[k]) - mean[k]) * rstd[k];
      const float d = to_f32(dy.v[k]);
      dz[k] = a.act ? slope(d, fmaf(xn[k], wt.w[k], wt.b[k])) : d;
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void write_dx(const Weights<T, V>& wt, const GradRow<T, V>& r, const float (&rstd)[V],
                                         const float (&s1)[V], const float (&s2)[V], T* dx) {
  float out[V];
#pragma unroll
  for (int k = 0; k < V; ++k) out[k] = rstd[k] * (r.dz[k] * wt.w[k] - s1[k] - r.xn[k] * s2[k]);
  store_raw<T, V>(dx, out);
}
// Samples that the registers hold; a block's samples leave one partial row of dw and db
template <typename T, int V, int R>
__global__ __launch_bounds__(256) void k_gn_samples_grad(Gn a) {
  __shared__ TileLds<V> lds;
  const Tile<V> t(a, blockIdx.x % a.slabs);
  const Weights<T, V> wt(a, t);
  const float inv = 1.f / (static_cast<float>(a.L) * static_cast<float>(a.cg));
  float dw[V], db[V];
#pragma unroll
  for (int k = 0; k < V; ++k) dw[k] = db[k] = 0.f;
  for (int64_t n = blockIdx.x / a.slabs; n < a.N; n += gridDim.x / a.slabs) {
    Raw<T, V> x[R], dy[R];
    float mean[V], rstd[V], sa[V], sb[V];
    load_tile(x, static_cast<const T*>(a.x) + n * a.xs, a.xl, t, 0, a.L);
    load_tile(dy, static_cast<const T*>(a.dy) + n * a.dys, a.dyl, t, 0, a.L);
    load_stats(a, t, n, mean, rstd);
#pragma unroll
    for (int k = 0; k < V; ++k) sa[k] = sb[k] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (!t.on || t.rl + int64_t{i} * t.RL >= a.L) continue;
      const GradRow<T, V> r(a, wt, x[i], dy[i], mean, rstd);
#pragma unroll
      for (int k = 0; k < V; ++k) sa[k] = fmaf(r.dz[k], r.xn[k], sa[k]), sb[k] += r.dz[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) dw[k] += sa[k], db[k] += sb[k];
    channel_sums(lds, t, sb, sa);
    group_sums(lds, t, a, [&](int gi, float s, float u) { lds.mean[gi] = s * inv, lds.m2[gi] = u * inv; });
    __syncthreads();
    float s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s1[k] = lds.mean[t.gk[k]], s2[k] = lds.m2[t.gk[k]];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t l = t.rl + int64_t{i} * t.RL;
      if (!a.dx || !t.on || l >= a.L) continue;
      const GradRow<T, V> r(a, wt, x[i], dy[i], mean, rstd);
      write_dx<T, V>(wt, r, rstd, s1, s2, static_cast<T*>(a.dx) + (n * a.L + l) * a.C + t.c);
    }
  }
  if (!a.cols) return;
  float* to = a.cols + int64_t{blockIdx.x} / a.slabs * 2 * a.C + t.c0;
  channel_sums(lds, t, dw, db);
  for (int c = threadIdx.x; c < t.width; c += 256) to[c] = lds.one[c], to[a.C + c] = lds.two[c];
}

// A range of positions of a slab: sums of dz xn and dz by channel into a partial row, times w by group into stats
template <typename T, int V>
__global__ __launch_bounds__(256) void k_gn_grad_sums(Gn a) {
  __shared__ TileLds<V> lds;
  const Place at(a);
  const int slab = at.slab, chunk = at.chunk;
  const Tile<V> t(a, slab);
  const int64_t n = at.n, l0 = chunk * a.chunk_rows, l1 = min(l0 + a.chunk_rows, a.L);
  const Weights<T, V> wt(a, t);
  float mean[V], rstd[V], sa[V], sb[V];
  load_stats(a, t, n, mean, rstd);
#pragma unroll
  for (int k = 0; k < V; ++k) sa[k] = sb[k] = 0.f;
  const T *x = static_cast<const T*>(a.x) + n * a.xs + t.c, *dy = static_cast<const T*>(a.dy) + n * a.dys + t.c;
  // Where there are samples enough to fill the card a range is a whole sample: 32 positions at a time, whose sums a thread
  // adds up in LDS (registers would leave three waves a SIMD instead of four: 2 x 100000 x 64 84 us in training, not 80).
  float *const la = lds.one + threadIdx.x * V, *const lb = lds.two + threadIdx.x * V;
  bool more = false;
  if (t.on)
    for (int64_t l = l0 + t.rl; l < l1;) {
      if (more) {
#pragma unroll
        for (int k = 0; k < V; ++k) la[k] = sa[k], lb[k] = sb[k], sa[k] = sb[k] = 0.f;
      }
#pragma unroll 4
      for (const int64_t e = min(l + 32 * t.RL, l1); l < e; l += t.RL) {
        const GradRow<T, V> r(a, wt, load_raw<T, V>(x + l * a.xl), load_raw<T, V>(dy + l * a.dyl), mean, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k) sa[k] = fmaf(r.dz[k], r.xn[k], sa[k]), sb[k] += r.dz[k];
      }
      if (more) {
#pragma unroll
        for (int k = 0; k < V; ++k) sa[k] += la[k], sb[k] += lb[k];
      }
      more = true;
    }
  float* to = a.cols + (n * a.chunks + chunk) * 2 * a.C + t.c0;
  float* groups = a.stats + ((n * a.chunks + chunk) * a.parts() + slab) * 2;
  channel_sums(lds, t, sa, sb);
  for (int c = threadIdx.x; c < t.width; c += 256) to[c] = lds.one[c], to[a.C + c] = lds.two[c];
  group_sums(lds, t, a, [&](int gi, float s, float u) { groups[2 * (t.g0 + gi) + 1] = s, groups[2 * (t.g0 + gi)] = u; });
}

template <typename T, int V, int R>
__global__ __launch_bounds__(256) void k_gn_grad_apply(Gn a) {
  const Place at(a);
  const Tile<V> t(a, at.slab);
  if (!t.on) return;
  const int64_t n = at.n, l0 = at.chunk * a.chunk_rows, l1 = min(l0 + a.chunk_rows, a.L);
  const T *px = static_cast<const T*>(a.x) + n * a.xs, *pd = static_cast<const T*>(a.dy) + n * a.dys;
  Raw<T, V> x[R], dy[R];
  load_tile(x, px, a.xl, t, l0, l1);
  load_tile(dy, pd, a.dyl, t, l0, l1);
  const Weights<T, V> wt(a, t);
  float mean[V], rstd[V], s1[V], s2[V];
  load_stats(a, t, n, mean, rstd);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int g = t.g0 + t.gk[k];
    const float2 s = reinterpret_cast<const float2*>(a.stats)[n * a.chunks * a.parts() + first_slab(a, g) + g];
    s1[k] = s.x, s2[k] = s.y;
  }
  T* dx = static_cast<T*>(a.dx) + n * a.L * a.C + t.c;
  for (int64_t l = l0; l < l1; l += int64_t{R} * t.RL) {
    Raw<T, V> nx[R], nd[R];
#pragma unroll
    for (int i = 0; i < R; ++i) nx[i] = x[i], nd[i] = dy[i];
    if (l + int64_t{R} * t.RL < l1) {
      load_tile(x, px, a.xl, t, l + int64_t{R} * t.RL, l1);
      load_tile(dy, pd, a.dyl, t, l + int64_t{R} * t.RL, l1);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t row = l + t.rl + int64_t{i} * t.RL;
      if (row >= l1) continue;
      const GradRow<T, V> r(a, wt, nx[i], nd[i], mean, rstd);
      write_dx<T, V>(wt, r, rstd, s1, s2, dx + row * a.C);
    }
  }
}

// dw[c], db[c] = the sums over the P partial rows [P, 2, C]: 16 columns a block, 16 threads a column
__global__ __launch_bounds__(256) void k_gn_cols(const float* __restrict__ partial, int64_t P, int C, int wdt, void* dw,
                                                 void* db) {
  __shared__ float part[16][17];
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + col;
  float s = 0.f;
  if (m < 2 * C) {
#pragma unroll 8
    for (int64_t p = grp; p < P; p += 16) s += partial[p * 2 * C + m];
  }
  part[grp][col] = s;
  __syncthreads();
  if (grp || m >= 2 * C) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += part[i][col];
  void* to = m < C ? dw : db;
  if (!to) return;
  const int64_t c = m < C ? m : m - C;
  if (wdt == LNG_F32)
    static_cast<float*>(to)[c] = s;
  else if (wdt == LNG_BF16)
    static_cast<bf16*>(to)[c] = from_f32<bf16>(s);
  else
    static_cast<_Float16*>(to)[c] = from_f32<_Float16>(s);
}

// ------------------------------------------------------------------ host
enum class Form { rows, samples, passes };
constexpr int FWD_R = 8, BWD_R = 4;  // positions a thread holds

struct Plan {
  Form form;
  bool vec;
  int lpr;             // rows: lanes a group
  int64_t blocks;
  int64_t P;           // partial rows of the weights' gradients
  int64_t stats, cols; // floats of the workspace
  int64_t own;         // where among the first are mean and rstd
};

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Lanes that hold a group of one position (LPR of the kernels' table below)
int lanes_of(int cg, bool vec) {
  if (vec) return cg <= 32 ? 4 : cg <= 64 ? 8 : cg <= 128 ? 16 : cg <= 256 ? 32 : cg <= 2048 ? 64 : 256;
  return cg <= 4 ? 4 : cg <= 64 ? 16 : cg <= 1024 ? 64 : 256;
}

// vec, es: 16-byte loads and the rows' element size.  The plan's workspace goes by the shape alone: 16-byte loads
// never need more of it.
Plan make_plan(Gn& a, bool vec, bool grad) {
  Plan p{};
  const int64_t N = a.N, L = a.L;
  if (L == 1 && a.cg <= MAX_ROW) {
    p.form = Form::rows;
    p.vec = vec && a.cg % VEC == 0;
    p.lpr = lanes_of(a.cg, p.vec);
    const Slots sl(a.G, 256 / p.lpr);
    // Enough blocks to fill the card; in the backward pass each leaves a partial row.  32768 x 1024 in 16 groups, bf16, in
    // 512, 1024, 2048, 4096, 8192, 16384 blocks: 34, 29, 29, 28, 30, 37 us; the training of 65536 x 1024 with 256, 512, 1024,
    // 2048, 4096 in the backward: 202, 155, 142, 149, 167.
    const int64_t per_slab = std::max<int64_t>(1, (grad ? 1024 : 4096) / sl.slabs);
    const int64_t bx = std::max<int64_t>(1, std::min<int64_t>(cdiv(N, sl.per), per_slab));
    p.blocks = bx * sl.slabs, p.P = bx;
  } else {
    p.vec = vec;
    const int V = vec ? VEC : 1, cap = 256 * V;
    if (a.C <= cap)
      a.slab = a.C;
    else if (a.cg % V == 0 && a.cg <= cap)
      a.slab = cap / a.cg * a.cg;
    else
      a.slab = cap;
    a.slabs = static_cast<int>(cdiv(a.C, a.slab));
    const int64_t rl = 256 / (std::min(a.slab, a.C) / V);
    if (a.slab % a.cg == 0 && L <= rl * (grad ? BWD_R : FWD_R)) {
      // One pass and one launch: 64 x 64 x 256 in 8 groups 18 us and in two passes 19, 512 x 64 x 256 19 and 24, the training of
      // 64 x 32 x 256 26 and 34, of 512 x 32 x 256 32 and 42, of 2048 x 32 x 256 90 and 90.  Where there are samples for several
      // rounds of blocks the first pass' loads hide the launches: 2048 x 64 x 256 54 and 49.  That is given away.
      p.form = Form::samples;
      const int64_t bx = std::min<int64_t>(N, std::max<int64_t>(1, (grad ? 1024 : 4096) / a.slabs));
      p.blocks = bx * a.slabs, p.P = bx;
    } else {
      p.form = Form::passes;
      // Whole tiles of positions, as many blocks as fill the card.  8 x 4096 x 320 in 256, 512, 1024, 2048 blocks: 39, 32, 26, 26
      // us; 2 x 100000 x 64: 49, 34, 30, 30.  With four positions a thread instead of eight both take a sixth longer.
      const int64_t tile = rl * FWD_R, tiles = cdiv(L, tile);
      const int64_t want = std::min<int64_t>({tiles, MOST_CHUNKS, std::max<int64_t>(1, cdiv(2048, N * a.slabs))});
      a.chunk_rows = cdiv(tiles, want) * tile;
      a.chunks = static_cast<int>(cdiv(L, a.chunk_rows));
      p.blocks = N * a.chunks * a.slabs, p.P = N * a.chunks;
      p.stats = N * a.chunks * a.parts() * 2;
      if (!grad) p.own = cdiv(p.stats, 16) * 16, p.stats = p.own + 2 * N * a.G;  // mean and rstd, where the caller wants none
    }
  }
  p.cols = grad ? p.P * 2 * a.C : 0;
  return p;
}

int64_t space_of(const Plan& p) { return cdiv(p.stats, 16) * 16 + p.cols; }

template <typename T, bool GRAD, int LPR, int NV, int V>
int launch_rows(const Gn& a, const Plan& p, hipStream_t st) {
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  if constexpr (GRAD) {
    constexpr size_t lds = LPR <= 64 ? size_t{2} * 256 * NV * V * 4 : 0;
    static_assert(lds <= 64 * 1024, "LDS of a block without a larger limit");
    k_gn_rows_grad<T, LPR, NV, V><<<blocks, 256, lds, st>>>(a);
  } else {
    k_gn_rows<T, LPR, NV, V><<<blocks, 256, 0, st>>>(a);
  }
  return check_launch(GRAD ? "group_norm_grad" : "group_norm");
}

template <typename T, bool GRAD>
int run_rows(const Gn& a, const Plan& p, hipStream_t st) {
#define LNG_GN_ROWS(limit, LPR, NV, V) \
  if (a.cg <= limit) return launch_rows<T, GRAD, LPR, NV, V>(a, p, st);
  if (p.vec) {
    LNG_GN_ROWS(32, 4, 1, VEC)
    LNG_GN_ROWS(64, 8, 1, VEC)
    LNG_GN_ROWS(128, 16, 1, VEC)
    LNG_GN_ROWS(256, 32, 1, VEC)
    LNG_GN_ROWS(512, 64, 1, VEC)
    LNG_GN_ROWS(1024, 64, 2, VEC)
    LNG_GN_ROWS(2048, 64, 4, VEC)
    LNG_GN_ROWS(4096, 256, 2, VEC)
    LNG_GN_ROWS(MAX_ROW, 256, 4, VEC)
  } else {
    LNG_GN_ROWS(4, 4, 1, 1)
    LNG_GN_ROWS(16, 16, 1, 1)
    LNG_GN_ROWS(64, 16, 4, 1)
    LNG_GN_ROWS(256, 64, 4, 1)
    LNG_GN_ROWS(1024, 64, 16, 1)
    LNG_GN_ROWS(4096, 256, 16, 1)
    LNG_GN_ROWS(MAX_ROW, 256, 32, 1)
  }
#undef LNG_GN_ROWS
  return fail(LNG_E_ARG, "group_norm: bad shape");
}

int64_t join_blocks(const Gn& a) { return cdiv(a.N * a.G, 16); }
template <bool GRAD>
int run_join(const Gn& a, hipStream_t st) {
  k_gn_join<GRAD><<<static_cast<unsigned>(join_blocks(a)), 256, 0, st>>>(a, a.N * a.G);
  return check_launch("group_norm");
}

template <typename T, int V>
int run_fwd(const Gn& a, const Plan& p, hipStream_t st) {
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  if (p.form == Form::samples) {
    k_gn_samples<T, V, FWD_R><<<blocks, 256, 0, st>>>(a);
    return check_launch("group_norm");
  }
  k_gn_stats<T, V, FWD_R><<<blocks, 256, 0, st>>>(a);
  if (int rc = check_launch("group_norm")) return rc;
  if (int rc = run_join<false>(a, st)) return rc;
  k_gn_apply<T, V, 2><<<blocks, 256, 0, st>>>(a);
  return check_launch("group_norm");
}

template <typename T, int V>
int run_bwd(const Gn& a, const Plan& p, hipStream_t st) {
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  if (p.form == Form::samples) {
    k_gn_samples_grad<T, V, BWD_R><<<blocks, 256, 0, st>>>(a);
    return check_launch("group_norm_grad");
  }
  k_gn_grad_sums<T, V><<<blocks, 256, 0, st>>>(a);
  if (int rc = check_launch("group_norm_grad")) return rc;
  if (!a.dx) return LNG_OK;
  if (int rc = run_join<true>(a, st)) return rc;
  k_gn_grad_apply<T, V, 2><<<blocks, 256, 0, st>>>(a);
  return check_launch("group_norm_grad");
}

template <typename T>
int run(const Gn& a, const Plan& p, bool grad, hipStream_t st) {
  if (p.form == Form::rows) return grad ? run_rows<T, true>(a, p, st) : run_rows<T, false>(a, p, st);
  if (p.vec) return grad ? run_bwd<T, VEC>(a, p, st) : run_fwd<T, VEC>(a, p, st);
  return grad ? run_bwd<T, 1>(a, p, st) : run_fwd<T, 1>(a, p, st);
}

int dispatch(int dtype, const Gn& a, const Plan& p, bool grad, hipStream_t st) {
  if (dtype == LNG_F32) return run<float>(a, p, grad, st);
  if (dtype == LNG_BF16) return run<bf16>(a, p, grad, st);
  return run<_Float16>(a, p, grad, st);
}

int check_args(const char* what, int dtype, int w_dtype, int64_t N, int64_t L, int32_t C, int32_t G, int64_t xs, int64_t xl) {
  if (dtype != LNG_F32 && dtype != LNG_BF16 && dtype != LNG_F16)
    return fail(LNG_E_DTYPE, std::string(what) + ": fp32, bf16 or fp16 rows");
  if (w_dtype != dtype && w_dtype != LNG_F32)
    return fail(LNG_E_DTYPE, std::string(what) + ": weights in the rows' type or fp32");
  if (N < 0 || L < 0 || C < 1 || C > (1 << 24) || G < 1 || C % G || N > (int64_t{1} << 40) || L > (int64_t{1} << 40) ||
      (N && L > (int64_t{1} << 44) / N / C) || xs < 0 || xl < 0)
    return fail(LNG_E_ARG, std::string(what) + ": bad shape (groups that divide the channels)");
  return LNG_OK;
}

// Blocks past 2^32 threads: more samples and slabs of channels than one launch counts, or more groups than the one between
// the passes
int check_blocks(const char* what, const Gn& a, const Plan& p) {
  if (std::max(p.blocks, p.form == Form::passes ? join_blocks(a) : 0) * 256 <= MOST_THREADS) return LNG_OK;
  return fail(LNG_E_ARG, std::string(what) + ": too many samples or channels for one launch; split the batch");
}

Gn make_args(const void* x, int64_t N, int64_t L, int32_t C, int32_t G, int64_t xs, int64_t xl, const void* w, const void* b,
             int w_dtype, float eps, int silu) {
  Gn a{};
  a.x = x, a.w = w, a.b = b, a.N = N, a.L = L, a.xs = xs, a.xl = xl, a.C = C, a.G = G, a.cg = C / G, a.wdt = w_dtype;
  a.act = silu != 0, a.eps = eps, a.slab = C, a.slabs = a.chunks = 1, a.chunk_rows = L;
  return a;
}

bool vector_rows(const void* p, int64_t s, int64_t l, int64_t N, int64_t L, int es) {
  return aligned(p, 16) && (N == 1 || s * es % 16 == 0) && (L == 1 || l * es % 16 == 0);
}

}  // namespace
}  // namespace lng

using namespace lng;

extern "C" {

size_t lng_group_norm_workspace_bytes(int64_t N, int64_t L, int32_t C, int32_t G, int grad) {
  if (N <= 0 || L <= 0 || C <= 0 || G <= 0 || C % G) return 0;
  int64_t most = 0;
  for (const bool vec : {false, true}) {
    if (vec && C % VEC) continue;
    Gn a = make_args(nullptr, N, L, C, G, 0, 0, nullptr, nullptr, LNG_F32, 0.f, 0);
    most = std::max(most, space_of(make_plan(a, vec, grad != 0)));
  }
  return static_cast<size_t>(most) * 4;
}

int lng_group_norm(const void* x, int dtype, int64_t N, int64_t L, int32_t C, int32_t G, int64_t x_sample, int64_t x_row,
                   const void* w, const void* b, int w_dtype, float eps, int silu, void* workspace, size_t workspace_bytes,
                   void* y, float* mean, float* rstd, void* stream) {
  const char* what = "group_norm";
  if (int rc = check_args(what, dtype, w_dtype, N, L, C, G, x_sample, x_row)) return rc;
  if (N == 0 || L == 0) return LNG_OK;
  if (!x || !y || !mean != !rstd) return fail(LNG_E_ARG, "group_norm: null pointer");
  Gn a = make_args(x, N, L, C, G, x_sample, x_row, w, b, w_dtype, eps, silu);
  a.y = y, a.mean = mean, a.rstd = rstd;
  const int es = dtype_size(dtype);
  const Plan p = make_plan(a, C % VEC == 0 && vector_rows(x, x_sample, x_row, N, L, es) && aligned(y, 16), false);
  if (int rc = check_blocks(what, a, p)) return rc;
  const size_t need = lng_group_norm_workspace_bytes(N, L, C, G, 0);
  if (need && (!workspace || !aligned(workspace, 64) || workspace_bytes < need))
    return fail(LNG_E_ARG, "group_norm: the workspace is too small or not 64-byte aligned");
  a.stats = static_cast<float*>(workspace);
  if (p.form == Form::passes && !mean) a.mean = a.stats + p.own, a.rstd = a.mean + N * G;
  return dispatch(dtype, a, p, false, as_stream(stream));
}

int lng_group_norm_grad(const void* dy, int64_t dy_sample, int64_t dy_row, const void* x, int64_t x_sample, int64_t x_row,
                        int dtype, int64_t N, int64_t L, int32_t C, int32_t G, const void* w, const void* b, int w_dtype,
                        int silu, const float* mean, const float* rstd, void* workspace, size_t workspace_bytes, void* dx,
                        void* dw, void* db, void* stream) {
  const char* what = "group_norm_grad";
  if (int rc = check_args(what, dtype, w_dtype, N, L, C, G, x_sample, x_row)) return rc;
  if (dy_sample < 0 || dy_row < 0) return fail(LNG_E_ARG, "group_norm_grad: bad shape");
  hipStream_t st = as_stream(stream);
  const unsigned col_blocks = static_cast<unsigned>(cdiv(2 * int64_t{C}, 16));
  const bool cols = dw || db;
  if (N == 0 || L == 0) {  // no values: the weights' gradients are zero, formed from no partial rows
    if (!cols) return LNG_OK;
    k_gn_cols<<<col_blocks, 256, 0, st>>>(nullptr, 0, C, w_dtype, dw, db);
    return check_launch(what);
  }
  if (!dy || !x || !mean || !rstd) return fail(LNG_E_ARG, "group_norm_grad: null pointer");
  Gn a = make_args(x, N, L, C, G, x_sample, x_row, w, b, w_dtype, 0.f, silu);
  a.dy = dy, a.dys = dy_sample, a.dyl = dy_row, a.dx = dx, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  const int es = dtype_size(dtype);
  const Plan p = make_plan(a, C % VEC == 0 && vector_rows(x, x_sample, x_row, N, L, es) &&
                                  vector_rows(dy, dy_sample, dy_row, N, L, es) && aligned(dx, 16), true);
  if (int rc = check_blocks(what, a, p)) return rc;
  if (!workspace || !aligned(workspace, 64) || workspace_bytes < lng_group_norm_workspace_bytes(N, L, C, G, 1))
    return fail(LNG_E_ARG, "group_norm_grad: the workspace is too small or not 64-byte aligned");
  a.stats = static_cast<float*>(workspace);
  a.cols = cols || p.form == Form::passes ? a.stats + cdiv(p.stats, 16) * 16 : nullptr;
  if (int rc = dispatch(dtype, a, p, true, st)) return rc;
  if (!cols) return LNG_OK;
  k_gn_cols<<<col_blocks, 256, 0, st>>>(a.cols, p.P, C, w_dtype, dw, db);
  return check_launch(what);
}

}  // extern "C"
