// Short causal depthwise convolution with bias, activation, dilation, a history and ragged lengths, its
// backward pass, and its step for one new token of every sequence (the conv of
// DepthwiseCausalConv.forward / forward_incremental, ffnmem/memory/lngram_v2.py:273-311, on rows that a
// caller has normalised itself, and the token mixer's conv of a selective state space).
//
//   pre[t, c] = bias[c] + sum_j w[c, j] * ext[t + j * dil, c],   y = pre * sigmoid(pre) (SiLU) or pre
//
// ext: the history's (K - 1) * dil rows (zeros without one), then the sequence.  A sequence of n < T tokens
// leaves zeros behind its end and never reads what stands there; the next history is ext's rows
// n .. n + (K - 1) * dil - 1.
//
// Backward, with dpre = dy * act'(pre): d ext[e] = sum_j w[j] dpre[e - j * dil] (+ the next history's
// gradient), dw[c, j] = sum dpre[t] ext[t + j * dil], dbias = sum dpre.
//
// Bound by memory.  The positions of one residue class of t mod dil see a conv without dilation, so a
// thread takes VEC channels and TT consecutive positions of one class and holds the taps' rows in
// registers: every row is read 1 + (K - 1) / TT times, and the loads of a thread's rows go out together.
// The backward pass forms pre again from x (K multiply-adds) instead of reading it.  Weight gradients are
// summed in registers over all of a thread's tiles, over a block's threads in LDS, and over blocks by
// k_conv_partials in a fixed order.
// bf16, 4 taps, SiLU: 8 x 4096 x 1024 33 us (75 MB read, 67 written, 4.4 TB/s), 3 x 777 x 1024 6.4; training of
// 8 x 2048 x 1024 20 us forward, 35 backward and 4 for the partial rows.  The backward pass moves 77 and 39 MB, 24 us
// of memory, and keeps the vector unit busy 47 % of its time, 17 us: a thread's 25 rows arrive before it computes, and
// four waves a SIMD do not hide all of either.  1 and 5 to 8 taps take a row after the other (training of the same
// size 89 us with 1 tap, 151 with 5, 225 with 8; 56 with 4).
#include "common.h"

namespace lng {
namespace {

constexpr int MAX_TAPS = 8;

// N neighbouring elements; aligned to the largest power of two that divides their size, 16 at most.
constexpr int pack_align(int bytes) { return (bytes & -bytes) < 16 ? (bytes & -bytes) : 16; }
template <typename T, int N>
struct alignas(pack_align(sizeof(T) * N)) Pack {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[N]) {
  const Pack<T, N> r = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(r.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[N]) {
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = r;
}

struct ConvArgs {
  const void *x, *w, *bias, *hist, *dy, *dhist_out;
  const int32_t* lengths;
  int64_t B, T, xb, xt, dyb, dyt, tiles;
  int C, K, dil, act, classes;  // classes: residue classes of t mod dil that the launch's positions fall into
  void *y, *hist_out, *dx, *dhist;
  float* partial;

  __device__ __forceinline__ int lp() const { return (K - 1) * dil; }
  __device__ __forceinline__ int64_t len(int64_t b) const {
    if (!lengths) return T;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
  }
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& r, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(r.v[i]);
}

// Row of a sequence at position pos: x, the history below 0, zeros below the history and from `end` on.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack_at(const ConvArgs& a, int64_t b, int64_t pos, int64_t end, int c) {
  const T* p = nullptr;
  if (pos >= 0) {
    if (pos < end) p = static_cast<const T*>(a.x) + b * a.xb + pos * a.xt + c;
  } else if (a.hist && pos >= -a.lp()) {
    p = static_cast<const T*>(a.hist) + (b * a.lp() + a.lp() + pos) * a.C + c;
  }
  Pack<T, VEC> r{};
  if (p) r = *reinterpret_cast<const Pack<T, VEC>*>(p);
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void load_at(const ConvArgs& a, int64_t b, int64_t pos, int64_t end, int c, float (&v)[VEC]) {
  unpack<T, VEC>(pack_at<T, VEC>(a, b, pos, end, c), v);
}

// w[j + KM - K][i]: tap j of channel c + i, so that the last register is the tap of the position itself.
// KT > 0: K taps known at compile time, read as 16-byte pieces (VEC * KT weights of neighbouring channels
// lie side by side).
template <typename W, int VEC, int KT, int KM>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int c, float (&w)[KM][VEC], float (&bias)[VEC]) {
  const W* p = static_cast<const W*>(a.w) + static_cast<int64_t>(c) * a.K;
  if constexpr (KT > 0 && VEC > 1) {
    float flat[VEC * KT];
    load_pack<W, VEC * KT>(p, flat);
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[j][i] = flat[i * KT + j];
  } else {
#pragma unroll
    for (int j = 0; j < KM; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[j][i] = j >= KM - a.K ? to_f32(p[i * a.K + j - (KM - a.K)]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) bias[i] = a.bias ? to_f32(static_cast<const W*>(a.bias)[c + i]) : 0.f;
}

// d silu / dv = s (1 + v (1 - s)), s = sigmoid(v)
template <typename T>
__device__ __forceinline__ float silu_grad(float v) {
  const float s = sizeof(T) == 2 ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-v * LOG2E)) : sigmoid(v);
  return s * fmaf(v, 1.f - s, 1.f);
}

// Threads [0, B * tiles * classes * C / VEC): outputs; behind them B * lp * C / VEC threads copy the next history.
template <typename T, typename W, int VEC, int KT, int TT>
__global__ __launch_bounds__(256) void k_short_conv(ConvArgs a) {
  constexpr int KM = KT > 0 ? KT : MAX_TAPS;
  const int64_t ncv = a.C / VEC;
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n_out = a.B * a.tiles * a.classes * ncv;
  if (i >= n_out) {
    i -= n_out;
    const int lp = a.lp();
    if (!a.hist_out || i >= a.B * lp * ncv) return;
    const int c = static_cast<int>(i % ncv) * VEC;
    const int64_t row = i / ncv, b = row / lp, n = a.len(b);
    float v[VEC];
    load_at<T, VEC>(a, b, n + row % lp - lp, n, c, v);
    store_pack<T, VEC>(static_cast<T*>(a.hist_out) + row * a.C + c, v);
    return;
  }
  const int c = static_cast<int>(i % ncv) * VEC;
  const int64_t rest = i / ncv, tr = rest % (a.tiles * a.classes), b = rest / (a.tiles * a.classes);
  const int64_t pos0 = tr / a.classes * TT * a.dil + tr % a.classes;  // first position, the others dil apart
  if (pos0 >= a.T) return;
  const int64_t n = a.len(b);
  // the registers of absent taps are skipped, not multiplied by zero: what their rows hold may be infinite
  const int skip = KT > 0 ? 0 : KM - a.K;
  // x[m]: position pos0 + (m - (KM - 1)) * dil, kept as stored until it enters the window
  Pack<T, VEC> x[TT + KM - 1];
  const int64_t first = pos0 - static_cast<int64_t>(a.K - 1) * a.dil, last = pos0 + static_cast<int64_t>(TT - 1) * a.dil;
  const bool inside = first >= 0 && last < n;  // no history, no padding: loads without a choice go out together
  if (inside) {
    const T* p = static_cast<const T*>(a.x) + b * a.xb + c;
#pragma unroll
    for (int m = 0; m < TT + KM - 1; ++m)
      if (m >= skip) x[m] = *reinterpret_cast<const Pack<T, VEC>*>(p + (pos0 + static_cast<int64_t>(m - (KM - 1)) * a.dil) * a.xt);
  } else {
#pragma unroll
    for (int m = 0; m < TT + KM - 1; ++m)
      if (m >= skip) x[m] = pack_at<T, VEC>(a, b, pos0 + static_cast<int64_t>(m - (KM - 1)) * a.dil, n, c);
  }
  float w[KM][VEC], bias[VEC], win[TT + KM - 1][VEC];
  load_weights<W, VEC, KT, KM>(a, c, w, bias);
#pragma unroll
  for (int m = 0; m < KM - 1; ++m) unpack<T, VEC>(x[m], win[m]);
  T* const y = static_cast<T*>(a.y) + (b * a.T + pos0) * a.C + c;
#pragma unroll
  for (int m = 0; m < TT; ++m) {
    unpack<T, VEC>(x[m + KM - 1], win[m + KM - 1]);
    const int64_t pos = pos0 + static_cast<int64_t>(m) * a.dil;
    float v[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = bias[k];
#pragma unroll
    for (int j = 0; j < KM; ++j) {
      if (j < skip) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = fmaf(w[j][k], win[m + j][k], v[k]);
    }
    if (a.act) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = silu<T>(v[k]);
    }
    if (!inside) {
      if (pos >= a.T) break;
      if (pos >= n) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = 0.f;
      }
    }
    store_pack<T, VEC>(y + static_cast<int64_t>(m) * a.dil * a.C, v);
  }
}

// Block: cx threads over the channels (blockIdx.x), 256 / cx over tiles; blockIdx.y strides over the tiles
// of all sequences.  A tile is TT positions q of one residue class from tile * TT - (K - 1) on, so that the
// first one begins with the history's rows: d ext of q needs dpre of q .. q + K - 1, formed here again
// ((K - 1) / TT more than once each), and the weights' gradients take each dpre where its position is one
// of the tile's own.
template <typename T, typename W, int VEC, int KT, int TT>
__global__ __launch_bounds__(256) void k_short_conv_grad(ConvArgs a, int cx) {
  constexpr int KM = KT > 0 ? KT : MAX_TAPS;
  __shared__ float sums[256 * VEC];
  const int tx = threadIdx.x % cx, ty = threadIdx.x / cx, py = 256 / cx;
  const int c = (static_cast<int>(blockIdx.x) * cx + tx) * VEC;
  const bool own = c < a.C;
  const int skip = KT > 0 ? 0 : KM - a.K, lp = a.lp();
  float w[KM][VEC], wl[KM][VEC], bias[VEC], dw[KM][VEC], db[VEC];  // wl[j]: tap j
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    db[k] = 0.f;
#pragma unroll
    for (int j = 0; j < KM; ++j) dw[j][k] = 0.f;
  }
  if (own) {
    load_weights<W, VEC, KT, KM>(a, c, w, bias);
#pragma unroll
    for (int j = 0; j < KM; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        wl[j][k] = KT > 0 ? w[j][k] : j < a.K ? to_f32(static_cast<const W*>(a.w)[int64_t{c + k} * a.K + j]) : 0.f;
    const int64_t total = a.B * a.tiles * a.dil;
    for (int64_t it = static_cast<int64_t>(blockIdx.y) * py + ty; it < total; it += static_cast<int64_t>(gridDim.y) * py) {
      const int64_t tr = it % (a.tiles * a.dil), b = it / (a.tiles * a.dil), n = a.len(b);
      const int64_t q0 = tr / a.dil * TT - (a.K - 1);
      const int64_t pos0 = q0 * a.dil + tr % a.dil;
      if (pos0 >= a.T) continue;
      // one position's dpre from the window's rows (the newest last), and its share of the weights' gradients
      auto slope = [&](const float (&x)[KM][VEC], const float (&dy)[VEC], bool own_pos, float (&g)[VEC]) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float v = bias[k];
#pragma unroll
          for (int j = 0; j < KM; ++j)
            if (j >= skip) v = fmaf(w[j][k], x[j][k], v);
          g[k] = a.act ? dy[k] * silu_grad<T>(v) : dy[k];
        }
        if (own_pos) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            db[k] += g[k];
#pragma unroll
            for (int j = 0; j < KM; ++j)
              if (j >= skip) dw[j][k] = fmaf(g[k], x[j][k], dw[j][k]);
          }
        }
      };
      // d ext of the row K - 1 steps back, which then has all its uses
      auto gather = [&](const float (&dp)[KM][VEC], float (&g)[VEC]) {
#pragma unroll
        for (int j = 0; j < KM; ++j) {
          if (j >= (KT > 0 ? KT : a.K)) continue;
#pragma unroll
          for (int k = 0; k < VEC; ++k) g[k] = fmaf(wl[j][k], dp[KM - 1 - j][k], g[k]);
        }
      };
      float x[KM][VEC], dp[KM][VEC];  // the last KM rows and their dpre; the newest at KM - 1
#pragma unroll
      for (int j = 0; j < KM; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dp[j][k] = 0.f;
      auto shift = [&] {
#pragma unroll
        for (int j = 0; j < KM - 1; ++j)
#pragma unroll
          for (int k = 0; k < VEC; ++k) x[j][k] = x[j + 1][k], dp[j][k] = dp[j + 1][k];
      };
      const int64_t last = pos0 + static_cast<int64_t>(TT + a.K - 2) * a.dil;
      if (KT > 0 && pos0 - lp >= 0 && last < n && a.dx) {
        // neither history nor padding: every row is asked for at once
        constexpr int XS = TT + 2 * (KM - 1), YS = TT + KM - 1;
        Pack<T, VEC> xr[XS], yr[YS];
        const T* const xp = static_cast<const T*>(a.x) + b * a.xb + (pos0 - lp) * a.xt + c;
        const T* const yp = static_cast<const T*>(a.dy) + b * a.dyb + pos0 * a.dyt + c;
#pragma unroll
        for (int m = 0; m < XS; ++m) xr[m] = *reinterpret_cast<const Pack<T, VEC>*>(xp + static_cast<int64_t>(m) * a.dil * a.xt);
#pragma unroll
        for (int m = 0; m < YS; ++m) yr[m] = *reinterpret_cast<const Pack<T, VEC>*>(yp + static_cast<int64_t>(m) * a.dil * a.dyt);
        T* const out = static_cast<T*>(a.dx) + (b * a.T + pos0) * a.C + c;
#pragma unroll
        for (int j = 1; j < KM; ++j) unpack<T, VEC>(xr[j - 1], x[j]);
#pragma unroll
        for (int m = 0; m < YS; ++m) {
          float dy[VEC];
          shift();
          unpack<T, VEC>(xr[m + KM - 1], x[KM - 1]);
          unpack<T, VEC>(yr[m], dy);
          slope(x, dy, m < TT, dp[KM - 1]);
          if (m >= KM - 1) {
            float g[VEC] = {};
            gather(dp, g);
            store_pack<T, VEC>(out + static_cast<int64_t>(m - (KM - 1)) * a.dil * a.C, g);
          }
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < KM; ++j)
        if (j > skip) load_at<T, VEC>(a, b, pos0 + static_cast<int64_t>(j - KM) * a.dil, n, c, x[j]);
#pragma unroll 1
      for (int m = 0; m < TT + a.K - 1; ++m) {
        const int64_t pos = pos0 + static_cast<int64_t>(m) * a.dil;
        shift();
        load_at<T, VEC>(a, b, pos, n, c, x[KM - 1]);
        if (pos >= 0 && pos < n) {
          float dy[VEC];
          load_pack<T, VEC>(static_cast<const T*>(a.dy) + b * a.dyb + pos * a.dyt + c, dy);
          slope(x, dy, m < TT, dp[KM - 1]);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) dp[KM - 1][k] = 0.f;
        }
        const int64_t at = pos - lp;
        if (m >= a.K - 1 && at < a.T && (at >= 0 ? a.dx != nullptr : a.dhist != nullptr)) {
          float g[VEC] = {};
          const int64_t slot = pos - n;  // of the next history
          if (a.dhist_out && slot >= 0 && slot < lp)
            load_pack<T, VEC>(static_cast<const T*>(a.dhist_out) + (b * lp + slot) * a.C + c, g);
          if (at < n) gather(dp, g);
          T* const out = at >= 0 ? static_cast<T*>(a.dx) + (b * a.T + at) * a.C
                                 : static_cast<T*>(a.dhist) + (b * lp + lp + at) * a.C;
          store_pack<T, VEC>(out + c, g);
        }
      }
    }
  }
  if (!a.partial) return;
  float* const out = a.partial + static_cast<int64_t>(blockIdx.y) * (a.K + 1) * a.C;
#pragma unroll
  for (int j = 0; j <= KM; ++j) {
    if (j < skip) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VEC; ++k) sums[threadIdx.x * VEC + k] = j == KM ? db[k] : dw[j < KM ? j : 0][k];
    __syncthreads();
    for (int i = threadIdx.x; i < cx * VEC; i += 256) {
      const int col = static_cast<int>(blockIdx.x) * cx * VEC + i;
      if (col >= a.C) continue;
      float s = 0.f;
      for (int r = 0; r < py; ++r) s += sums[r * cx * VEC + i];
      out[static_cast<int64_t>(j - skip) * a.C + col] = s;
    }
  }
}

// dw[c, j], dbias[c] = the sums over the P partial rows [P, K + 1, C]: 16 columns a block, 16 threads a column.
template <typename W>
__global__ __launch_bounds__(256) void k_conv_partials(const float* __restrict__ partial, int P, int K, int C,
                                                       W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float part[16][17];
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t M = int64_t{K + 1} * C, m = static_cast<int64_t>(blockIdx.x) * 16 + col;
  float s = 0.f;
  if (m < M) {
#pragma unroll 8
    for (int p = grp; p < P; p += 16) s += partial[p * M + m];
  }
  part[grp][col] = s;
  __syncthreads();
  if (grp == 0 && m < M) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][col];
    const int64_t j = m / C, c = m % C;
    if (j < K) {
      if (dw) dw[c * K + j] = from_f32<W>(s);
    } else if (db) {
      db[c] = from_f32<W>(s);
    }
  }
}

// One new token of every sequence: a thread owns VEC channels of a sequence, so the history may move in
// place (hist_out == hist): each of its rows is read before the thread writes the row in front of it.  NEAR:
// without dilation the window has at most MAX_TAPS rows, which are all asked for together (512 x 2048, 4 taps: 5 us
// instead of 12 with one row after the other).  With dilation 3 its nine rows, one after the other, take 15.
template <typename T, typename W, int VEC, int KT, bool NEAR>
__global__ __launch_bounds__(256) void k_short_conv_step(ConvArgs a) {
  constexpr int KM = KT > 0 ? KT : MAX_TAPS;
  const int64_t ncv = a.C / VEC, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.B * ncv) return;
  const int c = static_cast<int>(i % ncv) * VEC, lp = a.lp();
  const int64_t b = i / ncv;
  const T* const h = static_cast<const T*>(a.hist) + b * lp * a.C + c;
  T* const ho = static_cast<T*>(a.hist_out) + b * lp * a.C + c;
  float x[VEC], v[VEC];
  load_pack<T, VEC>(static_cast<const T*>(a.x) + b * a.xb + c, x);
  if constexpr (NEAR) {
    const int skip = KT > 0 ? 0 : KM - a.K;  // row e of the window and its weight in registers e + skip, the token's last
    float r[KM][VEC], w[KM][VEC];
#pragma unroll
    for (int j = 0; j < KM - 1; ++j)
      if (j >= skip) load_pack<T, VEC>(h + static_cast<int64_t>(j - skip) * a.C, r[j]);
    load_weights<W, VEC, KT, KM>(a, c, w, v);  // v: the bias
#pragma unroll
    for (int j = 0; j < KM - 1; ++j) {
      if (j < skip) continue;
      if (j > skip) store_pack<T, VEC>(ho + static_cast<int64_t>(j - skip - 1) * a.C, r[j]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = fmaf(w[j][k], r[j][k], v[k]);
    }
    if (lp > 0) store_pack<T, VEC>(ho + static_cast<int64_t>(lp - 1) * a.C, x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = fmaf(w[KM - 1][k], x[k], v[k]);
  } else {
    const W *wp = static_cast<const W*>(a.w) + static_cast<int64_t>(c) * a.K, *bp = static_cast<const W*>(a.bias);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = bp ? to_f32(bp[c + k]) : 0.f;
    for (int e = 0; e <= lp; ++e) {  // the window's rows: the history, then the token
      float r[VEC];
      if (e < lp) {
        load_pack<T, VEC>(h + static_cast<int64_t>(e) * a.C, r);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) r[k] = x[k];
      }
      if (e > 0) store_pack<T, VEC>(ho + static_cast<int64_t>(e - 1) * a.C, r);
      if (e % a.dil == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = fmaf(to_f32(wp[k * a.K + e / a.dil]), r[k], v[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = a.act ? silu<T>(v[k]) : v[k];
  store_pack<T, VEC>(static_cast<T*>(a.y) + b * a.C + c, v);
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether VEC-channel accesses serve every tensor of a call.
bool vector_ok(const ConvArgs& a, int vec, int es) {
  const int bytes = vec * es;
  return a.C % vec == 0 && aligned(a.x, bytes) && a.xb % vec == 0 && a.xt % vec == 0 && aligned(a.dy, bytes) &&
         a.dyb % vec == 0 && a.dyt % vec == 0 && aligned(a.w, 16) && aligned(a.hist, bytes) && aligned(a.y, bytes) &&
         aligned(a.hist_out, bytes) && aligned(a.dx, bytes) && aligned(a.dhist, bytes) && aligned(a.dhist_out, bytes);
}

// 16 positions a thread re-read fewest rows; 4 where 16 would leave the 1024 SIMDs less than two waves each.
int tile_rows(const ConvArgs& a, int vec) {
  return a.B * a.T / 16 * cdiv(a.C, vec) >= 1024 * 2 * 64 ? 16 : 4;
}

int too_many(const char* what) {
  return fail(LNG_E_ARG, std::string(what) + ": too many rows and channels for one launch; split the batch");
}

template <typename T, typename W, int VEC, int KT, int TT>
int launch_conv(ConvArgs a, hipStream_t st) {
  a.tiles = cdiv(cdiv(a.T, a.dil), TT);
  a.classes = static_cast<int>(std::min<int64_t>(a.dil, a.T));
  const int64_t rows = a.B * (a.tiles * a.classes + (a.hist_out ? (a.K - 1) * a.dil : 0));
  const int64_t threads = rows * (a.C / VEC);
  if (cdiv(threads, 256) * 256 > MOST_THREADS) return too_many("short_conv");
  if (threads) k_short_conv<T, W, VEC, KT, TT><<<static_cast<unsigned>(cdiv(threads, 256)), 256, 0, st>>>(a);
  return check_launch("short_conv");
}

struct GradGrid {
  int tt, vec, cx;
  int64_t tiles, gx, gy;
  GradGrid(int64_t B, int64_t T, int C, int K, int dil, int vec_) : vec(vec_) {
    tt = B * T / 16 * cdiv(C, vec) >= 1024 * 64 ? 8 : 4;
    tiles = cdiv(cdiv(T, dil) + K - 1, tt);
    const int64_t ncv = cdiv(C, vec);
    for (cx = 1; cx < 64 && cx < ncv; cx *= 2) {}
    gx = cdiv(ncv, cx);
    gy = std::max<int64_t>(1, std::min(cdiv(B * tiles * dil, 256 / cx), std::max<int64_t>(1, 1024 / gx)));
  }
};

template <typename T, typename W, int VEC, int KT, int TT>
void launch_grad(const ConvArgs& a, const GradGrid& g, hipStream_t st) {
  k_short_conv_grad<T, W, VEC, KT, TT><<<dim3(static_cast<unsigned>(g.gx), static_cast<unsigned>(g.gy)), 256, 0, st>>>(
      a, g.cx);
}

template <typename T, typename W, int VEC, int KT>
void grad_tile(const ConvArgs& a, const GradGrid& g, hipStream_t st) {
  if (g.tt == 8)
    launch_grad<T, W, VEC, KT, 8>(a, g, st);
  else
    launch_grad<T, W, VEC, KT, 4>(a, g, st);
}

template <typename T, typename W, int V, int KT>
int conv_tile(const ConvArgs& a, hipStream_t st) {
  return tile_rows(a, V) == 16 ? launch_conv<T, W, V, KT, 16>(a, st) : launch_conv<T, W, V, KT, 4>(a, st);
}

// Two to four taps as compile-time counts, for single channels too (4 x 2048 x 1001 with 4 taps 14 us and its
// training 45; 22 and 85 with eight taps of which the call's own are run).
template <typename T, typename W, int V>
int conv_taps(const ConvArgs& a, hipStream_t st) {
  switch (a.K) {
    case 2: return conv_tile<T, W, V, 2>(a, st);
    case 3: return conv_tile<T, W, V, 3>(a, st);
    case 4: return conv_tile<T, W, V, 4>(a, st);
    default: return launch_conv<T, W, V, 0, 4>(a, st);
  }
}
template <typename T, typename W, int V>
void grad_taps(const ConvArgs& a, const GradGrid& g, hipStream_t st) {
  switch (a.K) {
    case 2: grad_tile<T, W, V, 2>(a, g, st); break;
    case 3: grad_tile<T, W, V, 3>(a, g, st); break;
    case 4: grad_tile<T, W, V, 4>(a, g, st); break;
    default: grad_tile<T, W, V, 0>(a, g, st);
  }
}

template <typename T, typename W>
int run_conv(const ConvArgs& a, hipStream_t st) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  return vector_ok(a, V, sizeof(T)) ? conv_taps<T, W, V>(a, st) : conv_taps<T, W, 1>(a, st);
}

template <typename T, typename W>
int run_grad(ConvArgs a, void* dw, void* db, hipStream_t st) {
  const bool vec = vector_ok(a, 4, sizeof(T));
  const GradGrid g(a.B, a.T, a.C, a.K, a.dil, vec ? 4 : 1);
  a.tiles = g.tiles;
  if (vec)
    grad_taps<T, W, 4>(a, g, st);
  else
    grad_taps<T, W, 1>(a, g, st);
  if (int rc = check_launch("short_conv_grad")) return rc;
  if (!a.partial) return LNG_OK;
  k_conv_partials<W><<<static_cast<unsigned>(cdiv(int64_t{a.K + 1} * a.C, 16)), 256, 0, st>>>(
      a.partial, static_cast<int>(g.gy), a.K, a.C, static_cast<W*>(dw), static_cast<W*>(db));
  return check_launch("short_conv_grad");
}

template <typename T, typename W, int VEC>
int launch_step(const ConvArgs& a, hipStream_t st) {
  const int64_t n = cdiv(a.B * (a.C / VEC), 256);
  if (n * 256 > MOST_THREADS) return too_many("short_conv_step");
  const unsigned blocks = static_cast<unsigned>(n);
  if (a.dil == 1 && a.K == 4)
    k_short_conv_step<T, W, VEC, 4, true><<<blocks, 256, 0, st>>>(a);
  else if (a.dil == 1)
    k_short_conv_step<T, W, VEC, 0, true><<<blocks, 256, 0, st>>>(a);
  else
    k_short_conv_step<T, W, VEC, 0, false><<<blocks, 256, 0, st>>>(a);
  return check_launch("short_conv_step");
}

template <typename T, typename W>
int run_step(const ConvArgs& a, hipStream_t st) {
  // few channels in all: one a thread, so that more waves wait for memory at once
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  return a.B * a.C > 65536 && vector_ok(a, V, sizeof(T)) ? launch_step<T, W, V>(a, st) : launch_step<T, W, 1>(a, st);
}

int check_conv(const char* what, int dtype, int w_dtype, int64_t B, int64_t T, int32_t C, int32_t K, int32_t dil,
               int act) {
  if (dtype != LNG_F32 && dtype != LNG_BF16 && dtype != LNG_F16)
    return fail(LNG_E_DTYPE, std::string(what) + ": fp32, bf16 or fp16 rows");
  if (w_dtype != dtype && w_dtype != LNG_F32)
    return fail(LNG_E_DTYPE, std::string(what) + ": weights in the rows' type or fp32");
  if (B < 0 || T < 0 || C <= 0 || K < 1 || K > MAX_TAPS || dil < 1 || dil > 4096 || (act != 0 && act != 1) ||
      C > (1 << 24) || B > (int64_t{1} << 24) || T > (int64_t{1} << 31) ||
      B * (T + int64_t{K - 1} * dil) > (int64_t{1} << 36) / C)
    return fail(LNG_E_ARG, std::string(what) + ": bad shape (1 to 8 taps, dilation up to 4096, 2^36 elements with "
                                               "the history)");
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

int lng_short_conv(const void* x, int dtype, int64_t B, int64_t T, int32_t C, int64_t x_batch_stride, int64_t x_stride,
                   const void* w, const void* bias, int w_dtype, int32_t K, int32_t dilation, int silu,
                   const void* hist, const int32_t* lengths, void* y, void* hist_out, void* stream) {
  if (int rc = check_conv("short_conv", dtype, w_dtype, B, T, C, K, dilation, silu)) return rc;
  if (B == 0 || (T == 0 && (!hist_out || K == 1))) return LNG_OK;
  if (!w || (T > 0 && (!x || !y))) return fail(LNG_E_ARG, "short_conv: null pointer");
  if (hist_out && hist_out == hist) return fail(LNG_E_ARG, "short_conv: the next history needs memory of its own");
  ConvArgs a{};
  a.x = x, a.w = w, a.bias = bias, a.hist = hist, a.lengths = lengths, a.B = B, a.T = T, a.xb = x_batch_stride;
  a.xt = x_stride, a.C = C, a.K = K, a.dil = dilation, a.act = silu, a.y = y, a.hist_out = hist_out;
  return with_types(dtype, w_dtype,
                    [&](auto t, auto wt) { return run_conv<decltype(t), decltype(wt)>(a, as_stream(stream)); });
}

size_t lng_short_conv_grad_workspace_bytes(int64_t B, int64_t T, int32_t C, int32_t K, int32_t dilation) {
  if (B <= 0 || T < 0 || C <= 0 || K < 1 || K > MAX_TAPS || dilation < 1) return 0;
  const int64_t rows = std::max(GradGrid(B, T, C, K, dilation, 4).gy, GradGrid(B, T, C, K, dilation, 1).gy);
  return static_cast<size_t>(rows) * (K + 1) * static_cast<size_t>(C) * 4;
}

int lng_short_conv_grad(const void* dy, int64_t dy_batch_stride, int64_t dy_stride, const void* x,
                        int64_t x_batch_stride, int64_t x_stride, int dtype, int64_t B, int64_t T, int32_t C,
                        const void* w, const void* bias, int w_dtype, int32_t K, int32_t dilation, int silu,
                        const void* hist, const int32_t* lengths, const void* dhist_out, void* workspace,
                        size_t workspace_bytes, void* dx, void* dw, void* dbias, void* dhist, void* stream) {
  if (int rc = check_conv("short_conv_grad", dtype, w_dtype, B, T, C, K, dilation, silu)) return rc;
  const bool wts = dw || dbias;
  if (!w || (B * T > 0 && (!x || !dy))) return fail(LNG_E_ARG, "short_conv_grad: null pointer");
  if (wts && B > 0 &&
      (!workspace || workspace_bytes < lng_short_conv_grad_workspace_bytes(B, T, C, K, dilation)))
    return fail(LNG_E_ARG, "short_conv_grad: the workspace is too small");
  ConvArgs a{};
  a.x = x, a.w = w, a.bias = bias, a.hist = hist, a.lengths = lengths, a.B = B, a.T = T, a.xb = x_batch_stride;
  a.xt = x_stride, a.dy = dy, a.dyb = dy_batch_stride, a.dyt = dy_stride, a.dhist_out = dhist_out, a.C = C, a.K = K;
  a.dil = dilation, a.act = silu, a.dx = dx, a.dhist = dhist, a.partial = wts ? static_cast<float*>(workspace) : nullptr;
  hipStream_t st = as_stream(stream);
  return with_types(dtype, w_dtype, [&](auto t, auto wt) {
    using W = decltype(wt);
    if (B > 0) return run_grad<decltype(t), W>(a, dw, dbias, st);
    if (!wts) return static_cast<int>(LNG_OK);
    k_conv_partials<W><<<static_cast<unsigned>(cdiv(int64_t{K + 1} * C, 16)), 256, 0, st>>>(
        nullptr, 0, K, C, static_cast<W*>(dw), static_cast<W*>(dbias));
    return check_launch("short_conv_grad");
  });
}

int lng_short_conv_step(const void* x, int dtype, int64_t B, int32_t C, int64_t x_stride, const void* w,
                        const void* bias, int w_dtype, int32_t K, int32_t dilation, int silu, const void* hist,
                        void* hist_out, void* y, void* stream) {
  if (int rc = check_conv("short_conv_step", dtype, w_dtype, B, 1, C, K, dilation, silu)) return rc;
  if (B == 0) return LNG_OK;
  if (!x || !w || !y || (K > 1 && (!hist || !hist_out))) return fail(LNG_E_ARG, "short_conv_step: null pointer");
  ConvArgs a{};
  a.x = x, a.w = w, a.bias = bias, a.hist = hist, a.B = B, a.T = 1, a.xb = x_stride, a.C = C, a.K = K;
  a.dil = dilation, a.act = silu, a.y = y, a.hist_out = hist_out;
  return with_types(dtype, w_dtype,
                    [&](auto t, auto wt) { return run_step<decltype(t), decltype(wt)>(a, as_stream(stream)); });
}

}  // extern "C"
