// Selective state space scan: the diagonal recurrence of DiagonalSSM (ffnmem/memory/ssm.py:22-91) with N
// states a channel and with step sizes, inputs and outputs that the token chooses, its backward pass, and
// its step for one new token of every sequence.
//
//   s[t, c] = softplus(dt[t, c] + dt_bias[c])  (or dt + dt_bias)
//   h[t, c, n] = exp(s[t, c] A[c, n]) h[t-1, c, n] + s[t, c] u[t, c] B[t, g, n]      (g: the channel's group)
//   y[t, c] = (sum_n C[t, g, n] h[t, c, n] + D[c] u[t, c]) * silu(z[t, c])
//
// Backward, with e = dy silu(z) and q the gradient of h (q[t] = e[t] C[t] + exp(s[t+1] A) q[t+1]):
//   dC[t, n] = sum_c e h,  dB[t, n] = sum_c q s u,  du = s sum_n q B + e D,
//   ds = u sum_n q B + sum_n q exp(s A) h[t-1] A,  dA = sum_t q exp(s A) h[t-1] s,  d dt = ds softplus'(dt)
//
// Bound by the vector ALU: an exponential and some five multiply-adds for every (token, channel, state), on
// 8 bytes a (token, channel).  An exponential and four of the others take a SIMD 25 cycles a wave, so one pass
// over 8 x 4096 x 256 x 16 states is 21 us of all SIMDs' time (30 with softplus, gate and conversions) and its
// bytes are 14 us; it takes 53, and 39 more for the chunks' ends (the vector unit busy 57 % of either).  States kept
// in registers instead of LDS, or tiles read from LDS instead of through the scalar unit, take the same times.  A
// training step of 8 x 2048 x 1024 x 16: forward 108 and 74, backward 245 (the vector unit busy 81 %) and 77 us, 503
// with all.
//
// A lane holds one channel, so u, dt, z and y move as whole rows, and what all of a wave's channels share (B
// and C of a token) comes through the scalar unit: k_sel_tiles lays B and C out as fp32 tiles of SEG tokens
// per state, and a tile's row of 2 * SEG values is one scalar load for 64 * SEG state updates.  A segment of
// SEG tokens stays in registers (step sizes, inputs, outputs) while the loop runs over the states, whose
// values rest in LDS in between, so every N runs in the same registers.
// All sums and states are fp32.
//
// Where batch * channels gives too few waves, the time axis is cut into chunks: the chunks' own end states
// (from zero) and total step sizes, then their start states from one short pass over the chunks, then every
// chunk from its start.  The backward pass does the same for q, backwards, and takes the states of
// every GSEG tokens' start from the forward pass (N / GSEG floats a (token, channel)).  Short prompts of up to
// 64 states are not cut: k_sel_rows gives every state a lane instead (rows_serve says when).
#include <type_traits>

#include "common.h"

namespace lng {
namespace {

constexpr int SEG = 16;   // tokens of a tile, and of the forward pass's segments
constexpr int GSEG = 8;   // tokens of the backward pass's segments, whose first states the forward pass leaves
constexpr int WAVES = 4;  // waves of a block: neighbouring channels of one chunk
constexpr int MAX_N = 256;

typedef const float __attribute__((address_space(4))) cfloat;  // read through the scalar unit where uniform

struct Dims {
  int64_t B;
  int T, chunk, segs, gsegs;  // chunk: tokens of a chunk, a multiple of SEG; segs, gsegs: a sequence's segments
  int C, N, G, chunks, cbg;  // cbg: channel blocks of 64 in a group
  int np;                    // states of a tile: N, or N and zero rows up to whole sixteens
  int softplus;
  int rows;                  // a tile's values in the order of a state a lane: fours of tokens, then states
};

struct Ptrs {
  const void *u, *dt, *z, *Bm, *Cm, *dy;
  int64_t ub, ut, dtb, dtt, zb, zt, Bb, Bt, Bg, Cb, Ct, Cg, dyb, dyt;
  const float *A, *D, *bias, *start, *dend;
  const int32_t* lengths;
  void* y;
  float *end, *ckpt;
  const float* ckpt_in;
  // workspace
  float *tiles, *at, *hloc, *ssum, *pA, *pD, *pBC;
  void *du, *ddt, *dz;
  float* dstart;
};

// log(1 + exp(x)) with log1p by 2 atanh(e / (2 + e)): exact to about an ulp over the whole range, which
// log(1 + e) is not for the small steps that training starts from.  The series' first term left out is below
// 2^-26 at e = 1.
__device__ __forceinline__ float softplus(float x) {
  const float e = exp_minus_abs(x), s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float p = 1.f / 13.f;
  p = fmaf(p, q, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  p = fmaf(p, q, 1.f);
  return fmaf(2.f * s, p, fmaxf(x, 0.f));
}

// A decay rate without a bound (minus infinity keeps nothing of a state) as one that is still finite times log2 e:
// the steps of zero behind a sequence's end would make a NaN of it, while it ends every own token's state as well.
__device__ __forceinline__ float rate(float a) {
  constexpr float LEAST = -2e38f;
  return a < LEAST ? LEAST : a;
}

// The own tokens of sequence b (the same in every lane that asks for the same b).
__device__ __forceinline__ int seq_len(const int32_t* lengths, int64_t b, int T) {
  if (!lengths) return T;
  const int n = lengths[b];
  return n < 0 ? 0 : n > T ? T : n;
}

// B and C as fp32 tiles [b][g][seg][n][B: SEG, C: SEG] (zeros behind a sequence), and A transposed [N][C].
template <typename T>
__global__ __launch_bounds__(256) void k_sel_tiles(Dims d, Ptrs p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n_tiles = d.B * d.G * d.segs * SEG * d.np;
  if (i < n_tiles) {
    const int n = static_cast<int>(i % d.np), k = static_cast<int>(i / d.np % SEG);
    const int64_t seg = i / d.np / SEG % d.segs, bg = i / d.np / SEG / d.segs, g = bg % d.G, b = bg / d.G;
    const int64_t t = seg * SEG + k;
    float bv = 0.f, cv = 0.f;
    if (n < d.N && t < seq_len(p.lengths, b, d.T)) {
      bv = to_f32(static_cast<const T*>(p.Bm)[b * p.Bb + t * p.Bt + g * p.Bg + n]);
      cv = to_f32(static_cast<const T*>(p.Cm)[b * p.Cb + t * p.Ct + g * p.Cg + n]);
    }
    float* const tile = p.tiles + (bg * d.segs + seg) * d.np * 2 * SEG;
    if (d.rows) {
      float* const o = tile + n / 16 * 32 * SEG + k / 4 * 64 + n % 16 * 4 + k % 4;
      o[0] = bv;
      o[SEG * 16] = cv;
    } else {
      float* const o = tile + n * 2 * SEG + k;
      o[0] = bv;
      o[SEG] = cv;
    }
  } else if (i - n_tiles < static_cast<int64_t>(d.C) * d.N) {
    const int64_t j = i - n_tiles, c = j % d.C, n = j / d.C;
    p.at[j] = rate(p.A[c * d.N + n]);
  }
}

// A wave's share of a launch: 64 channels of one group, one sequence, one chunk.
struct Unit {
  int64_t b, bg, u;       // sequence, sequence and group, sequence and chunk
  int t0, t1, end;        // tokens [t0, t1) of the chunk; end: the sequence's length
  int c, lane, wave, chunk;
  bool ok;   // this lane has a channel
  bool any;  // the wave has one
  __device__ __forceinline__ Unit(const Dims& d, const int32_t* lengths) {
    // blocks: channel block groups fastest, then chunks, then sequences
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned waves = blockDim.x >> 6, bpg = (d.cbg + waves - 1) / waves;  // blocks of a group's channels
    const unsigned x = blockIdx.x, cb = x % (bpg * d.G), bs = x / (bpg * d.G);
    const int g = cb / bpg;
    chunk = bs % d.chunks;
    b = bs / d.chunks;
    bg = b * d.G + g;
    u = bs;
    const int cg = d.C / d.G, in = ((cb % bpg) * waves + wave) * 64;
    any = in < cg;
    ok = in + lane < cg;
    c = g * cg + (ok ? in + lane : cg - 1);
    t0 = chunk * d.chunk;
    t1 = t0 + d.chunk < d.T ? t0 + d.chunk : d.T;
    end = __builtin_amdgcn_readfirstlane(seq_len(lengths, b, d.T));
  }
  // The lane's byte offset in a row of T; lanes without a channel write nowhere (past every buffer's end).
  template <typename T>
  __device__ __forceinline__ int in(bool store = false) const {
    return store && !ok ? static_cast<int>(0x80000000u) : c * static_cast<int>(sizeof(T));
  }
};

// Rows of C channels behind one scalar address, reached by a lane's offset and a scalar one, so that no lane
// holds addresses.  The buffer's bounds hold a lane's offset (which is how lanes without a channel write
// nothing), not the scalar one: `load` and `store` take rows that exist.
template <typename T>
struct Rows {
  __amdgpu_buffer_rsrc_t buf;
  int stride;  // bytes
  // `rows` rows from `row` on, `token` elements apart
  __device__ __forceinline__ Rows(const void* row, int64_t token, int rows, int C)
      : stride(static_cast<int>(token) * static_cast<int>(sizeof(T))) {
    buf = dev_buf(row, static_cast<uint32_t>((rows - 1) * stride + C * static_cast<int>(sizeof(T))));
  }
  // The value's bits in a register of its own: a load into half a register would be waited for at once.
  __device__ __forceinline__ unsigned load(int lane, int i) const {
    if constexpr (sizeof(T) == 2)
      return static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(buf, lane, i * stride, 0));
    else
      return __builtin_amdgcn_raw_buffer_load_b32(buf, lane, i * stride, 0);
  }
  __device__ __forceinline__ void store(int lane, int i, float v) const {
    const T t = from_f32<T>(v);
    if constexpr (sizeof(T) == 2)
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, t), buf, lane, i * stride, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, t), buf, lane, i * stride, 0);
  }
};

// The first n of a segment's values into contiguous rows from `row` on.
template <typename T, int S>
__device__ __forceinline__ void put_seg(void* base, int64_t row, int n, int C, int lane, const float (&v)[S]) {
  const Rows<T> rows(static_cast<T*>(base) + row, C, n, C);
  if (n == S) {
#pragma unroll
    for (int i = 0; i < S; ++i) rows.store(lane, i, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < n) rows.store(lane, i, v[i]);
  }
}

template <typename T>
__device__ __forceinline__ float value(unsigned bits) {
  if constexpr (sizeof(T) == 4)
    return __builtin_bit_cast(float, bits);
  else
    return to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
}

template <int S>
__device__ __forceinline__ int live(int t, int end) {
  return end - t < S ? end - t : S;
}

// A segment's values of one tensor, as stored: loads that go out together.  Tokens at and behind `end`
// (which is past t) read the last own one; `widen` and `steps` put zeros in their place.
template <typename T, int S>
__device__ __forceinline__ void fetch(const void* base, int64_t batch, int64_t token, int t, int end, int C, int lane,
                                      unsigned (&v)[S]) {
  const int n = live<S>(t, end);
  const Rows<T> rows(static_cast<const T*>(base) + batch + t * token, token, n, C);
#pragma unroll
  for (int i = 0; i < S; ++i) v[i] = rows.load(lane, i < n ? i : n - 1);
}
template <typename T, int S>
__device__ __forceinline__ void widen(const unsigned (&r)[S], int t, int end, float (&v)[S]) {
#pragma unroll
  for (int i = 0; i < S; ++i) v[i] = value<T>(r[i]);
  if (t + S > end) {
#pragma unroll
    for (int i = 0; i < S; ++i) v[i] = t + i < end ? v[i] : 0.f;
  }
}

// Step sizes from dt; no time passes behind a sequence's end.
template <typename T, int S>
__device__ __forceinline__ void steps(const Dims& d, const unsigned (&r)[S], int t, int end, float bias, float (&s)[S]) {
#pragma unroll
  for (int i = 0; i < S; ++i) s[i] = value<T>(r[i]) + bias;
  if (d.softplus) {
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] = softplus(s[i]);
  }
  if (t + S > end) {
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] = t + i < end ? s[i] : 0.f;
  }
}

template <int S>
struct Row {  // B and C of one state over S of a tile's tokens
  float B[S], C[S];
};
template <int S>
__device__ __forceinline__ Row<S> load_row(const float* tiles, int64_t at) {
  cfloat* const q = (cfloat*)(uintptr_t)(tiles + at);
  Row<S> r;
#pragma unroll
  for (int i = 0; i < S; ++i) r.B[i] = q[i], r.C[i] = q[SEG + i];
  return r;
}

// Reads a word of each of a tile's 128-byte rows through the vector unit, a segment ahead of their scalar
// loads: those then find them in the XCD's L2 and not 2000 cycles away in memory, longer than a row's SEG
// tokens take.  `done` uses the words once they are there.
struct Warm {
  float got = 0.f;
  __device__ __forceinline__ void start(const float* tiles, int64_t tile, int N, int lane) {
    got = 0.f;
    for (int n = lane; n < N; n += 64) got += tiles[tile + n * 2 * SEG];
  }
  __device__ __forceinline__ void done() {
    asm volatile("" ::"v"(got));
  }
};

// Scalar loads come back in any order, so a wait for one is a wait for all: it stands in front of the next
// row's load, where what it waits for was asked for a whole row's work ago (behind that load, where the
// compiler would put it, every row waits for memory: 20 us more for the outputs of 8 x 4096 x 256, now 53).
constexpr int WAITCNT_LGKM0 = 0xC07F;  // s_waitcnt lgkmcnt(0), the other counts left open
__device__ __forceinline__ void rows_arrived() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(WAITCNT_LGKM0);
  __builtin_amdgcn_sched_barrier(0);
}

// A lane's per-state values (a state or its gradient, and the decay exponent A log2 e): the lane's columns of
// [N][64] arrays in LDS.  They could stay in registers only with the walk over the states unrolled for each N,
// which is no faster (56 us against 55 for the outputs of 8 x 4096 x 256); one loop serves any N.
struct States {
  float *v, *a;
  __device__ __forceinline__ States(float* lds, int wave, int lane, int N) {
    v = lds + wave * 2 * N * 64 + lane;
    a = v + N * 64;
  }
  // f(row, value, exponent, n) for every state, which updates the value: two rows in turn, the next state's
  // row and values on their way while f runs over the S tokens, and the last state's value on its way back.
  template <int S, typename F>
  __device__ __forceinline__ void walk(const float* tiles, int64_t tile, int N, F f) {
    Row<S> r0 = load_row<S>(tiles, tile), r1;
    float v0 = v[0], a0 = a[0], v1, a1, done = v0;
    float* back = v;
    for (int n = 0; n < N; n += 2) {
      int m = n + 1 < N ? n + 1 : n;
      rows_arrived();
      r1 = load_row<S>(tiles, tile + m * 2 * SEG);
      v1 = v[m * 64], a1 = a[m * 64];
      *back = done;
      f(r0, v0, a0, n);
      done = v0, back = v + n * 64;
      if (n + 1 >= N) break;
      m = n + 2 < N ? n + 2 : n;
      rows_arrived();
      r0 = load_row<S>(tiles, tile + m * 2 * SEG);
      v0 = v[m * 64], a0 = a[m * 64];
      *back = done;
      f(r1, v1, a1, n + 1);
      done = v1, back = v + (n + 1) * 64;
    }
    *back = done;
  }
};

// AGG: the chunk's end state from zero and its total step size.  Else: y, the final state (its last chunk)
// and, where wanted, the states at every segment's start.
template <typename T, bool AGG>
__global__ __launch_bounds__(64 * WAVES) void k_sel_scan(Dims d, Ptrs p) {
  extern __shared__ float lds[];
  const Unit w(d, p.lengths);
  if (!w.any || (AGG && w.chunk == d.chunks - 1)) return;
  const int stop = w.t1 < w.end ? w.t1 : w.end;  // behind it: zeros, and the states stay
  const int in = w.in<T>(), out = w.in<T>(true), out32 = w.in<float>(true);
  unsigned ur[SEG], dr[SEG], zr[SEG];
  auto read = [&](int t) {
    fetch<T>(p.u, w.b * p.ub, p.ut, t, stop, d.C, in, ur);
    fetch<T>(p.dt, w.b * p.dtb, p.dtt, t, stop, d.C, in, dr);
    if constexpr (!AGG)
      if (p.z) fetch<T>(p.z, w.b * p.zb, p.zt, t, stop, d.C, in, zr);
  };
  Warm warm;
  auto tile_of = [&](int t) { return (w.bg * d.segs + t / SEG) * d.np * 2 * SEG; };
  if (w.t0 < stop) {
    warm.start(p.tiles, tile_of(w.t0), d.N, w.lane);
    read(w.t0);
  }
  States states(lds, w.wave, w.lane, d.N);
#pragma unroll 8
  for (int n = 0; n < d.N; ++n) {
    const int64_t at = static_cast<int64_t>(n) * d.C + w.c;
    float h = 0.f;
    if constexpr (!AGG) {
      if (d.chunks > 1)
        h = p.hloc[w.u * d.N * d.C + at];
      else if (p.start)
        h = p.start[(w.b * d.C + w.c) * d.N + n];
    }
    states.v[n * 64] = h;
    states.a[n * 64] = p.at[at] * LOG2E;
  }
  const float bias = p.bias ? p.bias[w.c] : 0.f, dskip = !AGG && p.D ? p.D[w.c] : 0.f;
  float total = 0.f;
  for (int t = w.t0; t < stop; t += SEG) {
    float s[SEG], x[SEG], y[SEG], gate[SEG];
    widen<T>(ur, t, stop, x);
    steps<T>(d, dr, t, stop, bias, s);
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
      if constexpr (AGG) total += s[i];
      y[i] = p.D ? dskip * x[i] : 0.f;  // nothing of u without a skip, were it infinite
      x[i] *= s[i];
      gate[i] = 1.f;
    }
    if constexpr (!AGG) {
      if (p.z) {
        widen<T>(zr, t, stop, gate);
#pragma unroll
        for (int i = 0; i < SEG; ++i) gate[i] = silu<T>(gate[i]);
      }
    }
    warm.done();
    if (t + SEG < stop) {  // the next segment's values arrive while this one is computed
      warm.start(p.tiles, tile_of(t + SEG), d.N, w.lane);
      read(t + SEG);
    }
    const int64_t ck = (w.b * d.gsegs + t / GSEG) * d.N * d.C;
    const Rows<float> first(p.ckpt + ck, d.C, d.N, d.C), second(p.ckpt + ck + static_cast<int64_t>(d.N) * d.C, d.C, d.N, d.C);
    const bool both = t + GSEG < stop;
    states.walk<SEG>(p.tiles, tile_of(t), d.N, [&](const Row<SEG>& r, float& h, float a, int n) {
      if (!AGG && p.ckpt) first.store(out32, n, h);
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
        if (!AGG && i == GSEG && p.ckpt && both) second.store(out32, n, h);
        h = fmaf(__builtin_amdgcn_exp2f(s[i] * a), h, x[i] * r.B[i]);
        if constexpr (!AGG) y[i] = fmaf(r.C[i], h, y[i]);
      }
    });
    if constexpr (!AGG) {
#pragma unroll
      for (int i = 0; i < SEG; ++i) y[i] *= gate[i];
      put_seg<T>(p.y, (w.b * d.T + t) * d.C, live<SEG>(t, stop), d.C, out, y);
    }
  }
  if (!w.ok) return;
  if constexpr (AGG) {
    for (int n = 0; n < d.N; ++n) p.hloc[(w.u * d.N + n) * d.C + w.c] = states.v[n * 64];
    p.ssum[w.u * d.C + w.c] = total;
  } else {
    for (int64_t t = w.t0 < stop ? stop : w.t0; t < w.t1; ++t)
      static_cast<T*>(p.y)[(w.b * d.T + t) * d.C + w.c] = from_f32<T>(0.f);
    if (p.end && w.chunk == d.chunks - 1)
      for (int n = 0; n < d.N; ++n) p.end[(w.b * d.C + w.c) * d.N + n] = states.v[n * 64];
  }
}

// The chunks' start values from their own ends, in place: hloc[b, chunk, n, c] <- the value that enters the
// chunk.  Forward: from the first chunk on, starting with the given state.  BACK: the gradient that enters
// a chunk from behind, from the last chunk on, starting with the final state's gradient.  Block: 64 (b, n, c)
// by up to 16 waves, each of which holds the values of JOIN neighbouring chunks in registers: their loads go
// out together, their joint end and decay meet the other waves' in LDS, and longer sequences take another
// round (64 chunks of 8 x 16 x 256 states: 22 us one after the other, 9 with 16 loads at a time, 6 so).
constexpr int JOIN = 8;
template <bool BACK>
__global__ __launch_bounds__(1024) void k_sel_join(Dims d, Ptrs p) {
  __shared__ float ends[16][64], decays[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t total = d.B * d.N * d.C, i0 = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const int64_t i = i0 < total ? i0 : total - 1;
  const int64_t c = i % d.C, n = i / d.C % d.N, b = i / d.C / d.N;
  const float a = p.at[n * d.C + c] * LOG2E;
  const float* const first = BACK ? p.dend : p.start;
  float carry = first ? first[(b * d.C + c) * d.N + n] : 0.f;
  for (int k0 = 0; k0 < d.chunks; k0 += waves * JOIN) {
    float own[JOIN], decay[JOIN];
    auto unit = [&](int j) {
      const int k = k0 + wave * JOIN + j;
      return b * d.chunks + (BACK ? d.chunks - 1 - k : k);
    };
#pragma unroll
    for (int j = 0; j < JOIN; ++j) {
      own[j] = 0.f, decay[j] = 0.f;  // the last chunk's own values are not used
      if (k0 + wave * JOIN + j < d.chunks - 1) {
        own[j] = p.hloc[(unit(j) * d.N + n) * d.C + c];
        decay[j] = p.ssum[unit(j) * d.C + c];
      }
    }
    float h = 0.f, steps = 0.f;
#pragma unroll
    for (int j = 0; j < JOIN; ++j) {
      steps += decay[j];
      decay[j] = __builtin_amdgcn_exp2f(decay[j] * a);
      h = fmaf(decay[j], h, own[j]);
    }
    ends[wave][lane] = h;
    decays[wave][lane] = __builtin_amdgcn_exp2f(steps * a);
    __syncthreads();
    h = carry;
    for (int k = 0; k < waves; ++k) {
      if (k == wave) {
        float g = h;
#pragma unroll
        for (int j = 0; j < JOIN; ++j) {
          if (k0 + wave * JOIN + j < d.chunks && i0 < total) p.hloc[(unit(j) * d.N + n) * d.C + c] = g;
          g = fmaf(decay[j], g, own[j]);
        }
      }
      h = fmaf(decays[k][lane], h, ends[k][lane]);
    }
    carry = h;
    __syncthreads();
  }
}

// ------------------------------------------------------------------ a state a lane
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ float swap_add(bool high, float a, float b) {  // low lanes keep a's sum, high lanes b's
  const float keep = high ? b : a, give = high ? a : b;
  return keep + dpp_move<CTRL>(give);
}
// The sum over a row of 16 lanes of each of 16 values, in 45 operations: lane j of the row receives value j's.
__device__ __forceinline__ float row_sums(float (&v)[16], int j) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = swap_add<0x128>(j & 8, v[i], v[i + 8]);  // row_ror:8
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = swap_add<0x141>(j & 4, v[i], v[i + 4]);  // row_half_mirror
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = swap_add<0x4E>(j & 2, v[i], v[i + 2]);   // quad_perm 2 3 0 1
  return swap_add<0xB1>(j & 1, v[0], v[1]);                                   // quad_perm 1 0 3 2
}

// What the wave's lanes wrote to LDS before is what they read behind it.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int I, int S, typename F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (I < S) {
    f(std::integral_constant<int, I>{});
    unrolled<I + 1, S>(f);
  }
}

// Prompts in one pass, without a cut in time: a wave holds four channels, a row of 16 lanes each, and lane j of
// a row holds states j, j + 16, .. (K of them) of its channel.  What a (token, channel) needs once (step size, input, gate,
// output) is read, made and written by lane 4 * token + channel, so that a load's neighbours are neighbours in
// memory (token-major lanes took 1.37 us a segment instead of 1.15 with two waves a SIMD: 64 lines a load);
// step sizes and inputs reach the rows through LDS, and a segment's 16 outputs are summed over a row's states in
// 45 operations.  The next segment's tile and the inputs after it are asked for before this segment is run.
// A wave needs 0.65 us a segment whatever its neighbours do (1.1 for two states a lane, 1.4 for four), so few and
// short sequences are what it is for (rows_serve).
struct RowTile {  // B and C of a lane's state over a segment
  f32x4 B[4], C[4];
};
struct RowOwn {  // u, dt and z of a lane's (token, channel), as stored
  unsigned u, dt, z;
};
template <typename T, int K, bool CKPT>
__global__ __launch_bounds__(64 * WAVES) void k_sel_rows(Dims d, Ptrs p) {
  __shared__ f32x4 lds[WAVES][5][9];  // a channel's 16 step sizes and 16 inputs; the fifth row: zeros
  const int lane = threadIdx.x & 63, r = lane >> 4, j = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned waves = blockDim.x >> 6;
  const int cg = d.C / d.G;
  const unsigned bpg = (cg + 4 * waves - 1) / (4 * waves), x = blockIdx.x, cb = x % (bpg * d.G);
  const int64_t b = x / (bpg * d.G);
  const int g = cb / bpg, in0 = ((cb % bpg) * waves + wave) * 4;
  if (in0 >= cg) return;
  const bool ok = in0 + r < cg;
  const int c = g * cg + (ok ? in0 + r : cg - 1), es = sizeof(T);
  const int64_t bg = b * d.G + g;
  const int end = __builtin_amdgcn_readfirstlane(seq_len(p.lengths, b, d.T));
  float a[K], h[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = j + 16 * k;
    const bool real = n < d.N;
    a[k] = real ? rate(p.A[static_cast<int64_t>(c) * d.N + n]) * LOG2E : 0.f;
    h[k] = real && p.start ? p.start[(b * d.C + c) * d.N + n] : 0.f;
  }
  // a token's four channels in neighbouring lanes for what a (token, channel) needs once
  const int lt = lane >> 2, lr = lane & 3;
  const bool lok = in0 + lr < cg;
  const int lc = g * cg + (lok ? in0 + lr : cg - 1);
  const float bias = p.bias ? p.bias[lc] : 0.f, dskip = p.D ? p.D[lc] : 0.f;
  const int ou = lt * static_cast<int>(p.ut) * es + lc * es, od = lt * static_cast<int>(p.dtt) * es + lc * es;
  // loads without a branch, so that a wait counts exactly the ones it is for: without a gate z reads u
  const T* const zp = p.z ? static_cast<const T*>(p.z) + b * p.zb : static_cast<const T*>(p.u) + b * p.ub;
  const int64_t zt = p.z ? p.zt : p.ut;
  const int oz = lt * static_cast<int>(zt) * es + lc * es;
  const int oy = lok ? (lt * d.C + lc) * es : static_cast<int>(0x80000000u);
  float* const own_lds = reinterpret_cast<float*>(&lds[wave][0][0]) + lr * 36 + lt;
  // lanes without a state take the zeros, so that what isn't finite in a row stays out of its sums
  const f32x4* const row_lds = &lds[wave][j < d.N ? r : 4][0];
  if (lane < 9) lds[wave][4][lane] = f32x4{};
  const int last = end > 0 ? (end - 1) / SEG * SEG : 0;
  auto read_own = [&](int t, RowOwn& s) {
    t = t < last ? t : last;
    const int n = live<SEG>(t, end);
    s.u = Rows<T>(static_cast<const T*>(p.u) + b * p.ub + t * p.ut, p.ut, n, d.C).load(ou, 0);
    s.dt = Rows<T>(static_cast<const T*>(p.dt) + b * p.dtb + t * p.dtt, p.dtt, n, d.C).load(od, 0);
    s.z = Rows<T>(zp + t * zt, zt, n, d.C).load(oz, 0);
  };
  auto read_tile = [&](int t, int k, RowTile& s) {
    t = t < last ? t : last;
    const f32x4* const q = reinterpret_cast<const f32x4*>(
        p.tiles + ((bg * d.segs + static_cast<unsigned>(t) / SEG) * K + k) * 32 * SEG);
#pragma unroll
    for (int i = 0; i < 4; ++i) s.B[i] = q[i * 16 + j], s.C[i] = q[64 + i * 16 + j];
  };
  // `even`: the tile of the lane's first state, which is there or on its way; each further state's, and at last the
  // next segment's first, is asked for while the one before it is run, into the other of the two
  auto run = [&](int t, RowOwn& in, RowTile& even, RowTile& odd) {
    unsigned ub = in.u, db = in.dt, zb = in.z;
    asm volatile("" : "+v"(ub), "+v"(db), "+v"(zb));  // converted here, not where they are asked for
    const bool own = t + lt < end;
    const float u = own ? value<T>(ub) : 0.f;
    float s = value<T>(db) + bias;
    if (d.softplus) s = softplus(s);
    s = own ? s : 0.f;
    const float xs = s * u;
    wave_order();
    own_lds[0] = s;
    own_lds[16] = xs;
    wave_order();
    f32x4 ss[4], xx[4];
    float v[SEG];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const RowTile& in_k = k % 2 ? odd : even;
      RowTile& next = k % 2 ? even : odd;
      if (k + 1 < K)
        read_tile(t, k + 1, next);
      else
        read_tile(t + SEG, 0, next);
      if (k == 0) {
        read_own(t + 2 * SEG, in);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[i] = row_lds[i], xx[i] = row_lds[4 + i];
      }
      __builtin_amdgcn_sched_barrier(0);
      unrolled<0, SEG>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (CKPT && i % GSEG == 0) {
          const int seg = (t + i) / GSEG;
          const Rows<float> ck(p.ckpt + (b * d.gsegs + (seg < d.gsegs ? seg : 0)) * d.N * d.C, d.C, d.N, d.C);
          const int n = lt + 16 * k;  // four channels in neighbouring lanes, as the other rows are written
          const int kept = __builtin_amdgcn_ds_bpermute((lr * 16 + lt) * 4, __builtin_bit_cast(int, h[k]));
          ck.store(lok && n < d.N && t + i < end ? (n * d.C + lc) * 4 : static_cast<int>(0x80000000u), 0,
                   __builtin_bit_cast(float, kept));
        }
        h[k] = fmaf(__builtin_amdgcn_exp2f(ss[i / 4][i % 4] * a[k]), h[k], xx[i / 4][i % 4] * in_k.B[i / 4][i % 4]);
        if (k)
          v[i] = j + 16 * k < d.N ? fmaf(in_k.C[i / 4][i % 4], h[k], v[i]) : v[i];
        else
          v[i] = in_k.C[i / 4][i % 4] * h[k];
      });
    }
    const float sum = __builtin_bit_cast(
        float, __builtin_amdgcn_ds_bpermute((lr * 16 + lt) * 4, __builtin_bit_cast(int, row_sums(v, j))));
    float y = p.D ? fmaf(dskip, u, sum) : sum;
    if (p.z) y *= silu<T>(value<T>(zb));
    const Rows<T> out(static_cast<T*>(p.y) + (b * d.T + t) * d.C, d.C, live<SEG>(t, d.T), d.C);
    out.store(oy, 0, own ? y : 0.f);
  };
  int t = 0;
  if (end > 0) {
    RowOwn o0, o1;
    RowTile t0, t1;
    read_own(0, o0);
    __builtin_amdgcn_sched_barrier(0);
    read_tile(0, 0, t0);
    __builtin_amdgcn_sched_barrier(0);
    read_own(SEG, o1);
    __builtin_amdgcn_sched_barrier(0);
    for (;;) {
      run(t, o0, t0, t1);
      t += SEG;
      if (t > last) break;
      if constexpr (K == 1)
        run(t, o1, t1, t0);
      else
        run(t, o1, t0, t1);
      t += SEG;
      if (t > last) break;
    }
  }
  for (; t < d.T; t += SEG) {
    const Rows<T> out(static_cast<T*>(p.y) + (b * d.T + t) * d.C, d.C, live<SEG>(t, d.T), d.C);
    out.store(oy, 0, 0.f);
  }
  if (p.end && ok) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + 16 * k < d.N) p.end[(b * d.C + c) * d.N + j + 16 * k] = h[k];
  }
}

// A chunk's own gradient of the state in front of it (nothing from behind) and its total step size.
template <typename T>
__global__ __launch_bounds__(64 * WAVES) void k_sel_grad_ends(Dims d, Ptrs p) {
  extern __shared__ float lds[];
  const Unit w(d, p.lengths);
  if (!w.any || w.chunk == 0) return;
  const int stop = w.t1 < w.end ? w.t1 : w.end, in = w.in<T>();
  unsigned er[SEG], dr[SEG], zr[SEG];
  auto read = [&](int t) {
    fetch<T>(p.dy, w.b * p.dyb, p.dyt, t, stop, d.C, in, er);
    fetch<T>(p.dt, w.b * p.dtb, p.dtt, t, stop, d.C, in, dr);
    if (p.z) fetch<T>(p.z, w.b * p.zb, p.zt, t, stop, d.C, in, zr);
  };
  const int last = stop > w.t0 ? (stop - 1) / SEG * SEG : w.t0 - SEG;
  Warm warm;
  auto tile_of = [&](int t) { return (w.bg * d.segs + t / SEG) * d.np * 2 * SEG; };
  if (last >= w.t0) {
    warm.start(p.tiles, tile_of(last), d.N, w.lane);
    read(last);
  }
  States states(lds, w.wave, w.lane, d.N);
#pragma unroll 8
  for (int n = 0; n < d.N; ++n) {
    states.v[n * 64] = 0.f;
    states.a[n * 64] = p.at[static_cast<int64_t>(n) * d.C + w.c] * LOG2E;
  }
  const float bias = p.bias ? p.bias[w.c] : 0.f;
  float total = 0.f;
  for (int t = last; t >= w.t0; t -= SEG) {
    float s[SEG], e[SEG];
    widen<T>(er, t, stop, e);
    steps<T>(d, dr, t, stop, bias, s);
    if (p.z) {
      float z[SEG];
      widen<T>(zr, t, stop, z);
#pragma unroll
      for (int i = 0; i < SEG; ++i) e[i] *= z[i] * sigmoid(z[i]);
    }
    warm.done();
    if (t > w.t0) {
      warm.start(p.tiles, tile_of(t - SEG), d.N, w.lane);
      read(t - SEG);
    }
#pragma unroll
    for (int i = 0; i < SEG; ++i) total += s[i];
    states.walk<SEG>(p.tiles, tile_of(t), d.N, [&](const Row<SEG>& r, float& q, float a, int) {
#pragma unroll
      for (int i = SEG - 1; i >= 0; --i) q = fmaf(e[i], r.C[i], q) * __builtin_amdgcn_exp2f(s[i] * a);
    });
  }
  if (!w.ok) return;
  for (int n = 0; n < d.N; ++n) p.hloc[(w.u * d.N + n) * d.C + w.c] = states.v[n * 64];
  p.ssum[w.u * d.C + w.c] = total;
}

// The sum over the wave's 64 lanes of each of 16 values, in 35 operations instead of 16 * 7: every round
// halves the values that a lane carries by handing the other half to its partner.  Lane l receives the sum
// of value l / 4.
// The two halves of a swap's result, added.  (Through integers of their own: a bit cast of a vector's element
// takes the vector's first one.)
__device__ __forceinline__ float sum_of(unsigned a, unsigned b) {
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float lane_sums(float (&v)[16], int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v[i]),
                                                    __builtin_bit_cast(unsigned, v[i + 8]), false, false);
    v[i] = sum_of(r[0], r[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v[i]),
                                                    __builtin_bit_cast(unsigned, v[i + 4]), false, false);
    v[i] = sum_of(r[0], r[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = swap_add<0x128>(lane & 8, v[i], v[i + 2]);  // row_ror:8
  v[0] = swap_add<0x141>(lane & 4, v[0], v[1]);                                  // row_half_mirror
  v[0] += dpp_move<0x4E>(v[0]);                                                  // quad_perm 2 3 0 1
  return v[0] + dpp_move<0xB1>(v[0]);                                            // quad_perm 1 0 3 2
}

// The backward pass of one chunk, segment by segment from its end.  pBC[cb][b][g][t][2][N] receives the
// block's share of dB and dC (its channels' sum), pA[unit][n][c] and pD[unit][2][c] the chunk's share of dA,
// dD and d dt_bias.
template <typename T>
__global__ __launch_bounds__(64 * WAVES, 3) void k_sel_grad(Dims d, Ptrs p) {
  extern __shared__ float lds[];
  const Unit w(d, p.lengths);
  const int waves = blockDim.x >> 6, N = d.N;
  States grads(lds, w.wave, w.lane, N);  // the gradients from behind, and dA in the place of the exponents
  float *const qs = grads.v, *const ga = grads.a;
  float* const sums = lds + waves * 2 * N * 64;          // [wave][n][B: GSEG, C: GSEG]
  const float bias = p.bias ? p.bias[w.c] : 0.f, dskip = p.D ? p.D[w.c] : 0.f;
  float dD = 0.f, dbias = 0.f;
  for (int n = 0; n < N; ++n) {
    const int64_t at = static_cast<int64_t>(n) * d.C + w.c;
    float q = 0.f;
    if (d.chunks > 1)
      q = p.hloc[w.u * N * d.C + at];
    else if (p.dend)
      q = p.dend[(w.b * d.C + w.c) * N + n];
    qs[n * 64] = w.ok ? q : 0.f;
    ga[n * 64] = 0.f;
  }
  const int bpg = (d.cbg + waves - 1) / waves;
  const int64_t cb = blockIdx.x % bpg;  // this block's place among those of its group
  const int in = w.in<T>(), out_t = w.in<T>(true), in32 = w.in<float>();
  const Rows<float> at(p.at, d.C, N, d.C);
  Warm warm;
  auto tile_of = [&](int t) { return (w.bg * d.segs + t / SEG) * d.np * 2 * SEG + t % SEG; };
  warm.start(p.tiles, tile_of(w.t1 - 1), N, w.lane);
  for (int t = (w.t1 - 1) / GSEG * GSEG; t >= w.t0; t -= GSEG) {
    const int64_t row = (w.b * d.T + t) * d.C;
    const int rows = live<GSEG>(t, w.t1);  // tokens that the tensors have
    if (t < w.end) {
      if (w.any) {
        // inputs, step sizes and their slopes, gated gradients, dz without its y; sums over the states
        float u[GSEG], s[GSEG], slope[GSEG], e[GSEG], dz[GSEG], y[GSEG], gb[GSEG], gs[GSEG];
        {
          unsigned ur[GSEG], dr[GSEG], er[GSEG], zr[GSEG];
          fetch<T>(p.u, w.b * p.ub, p.ut, t, w.end, d.C, in, ur);
          fetch<T>(p.dt, w.b * p.dtb, p.dtt, t, w.end, d.C, in, dr);
          fetch<T>(p.dy, w.b * p.dyb, p.dyt, t, w.end, d.C, in, er);
          if (p.z) fetch<T>(p.z, w.b * p.zb, p.zt, t, w.end, d.C, in, zr);
          widen<T>(ur, t, w.end, u);
          steps<T>(d, dr, t, w.end, bias, s);
          widen<T>(er, t, w.end, e);
#pragma unroll
          for (int i = 0; i < GSEG; ++i) slope[i] = 1.f, dz[i] = 0.f;
          if (d.softplus) {
#pragma unroll
            for (int i = 0; i < GSEG; ++i) slope[i] = sigmoid(value<T>(dr[i]) + bias);
          }
          if (p.z) {
            float z[GSEG];
            widen<T>(zr, t, w.end, z);
#pragma unroll
            for (int i = 0; i < GSEG; ++i) {
              const float sg = sigmoid(z[i]);
              dz[i] = e[i] * sg * fmaf(z[i], 1.f - sg, 1.f);
              e[i] *= z[i] * sg;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < GSEG; ++i) {
          e[i] = w.ok ? e[i] : 0.f;  // lanes without a channel add nothing to the sums over channels
          y[i] = gb[i] = gs[i] = 0.f;
        }
        warm.done();
        if (t > w.t0) warm.start(p.tiles, tile_of(t - GSEG), N, w.lane);
        const int64_t tile = tile_of(t);
        const Rows<float> ckpt(p.ckpt_in + (w.b * d.gsegs + t / GSEG) * N * d.C, d.C, N, d.C);
        float an_next = value<float>(at.load(in32, 0)), h0_next = value<float>(ckpt.load(in32, 0));
        grads.walk<GSEG>(p.tiles, tile, N, [&](const Row<GSEG>& r, float& q, float dA, int n) {
          const int m = n + 1 < N ? n + 1 : n;
          const float an = an_next, h0 = h0_next, a2 = an * LOG2E;
          an_next = value<float>(at.load(in32, m)), h0_next = value<float>(ckpt.load(in32, m));
          float a[GSEG], h[GSEG], v[2 * GSEG];
#pragma unroll
          for (int i = 0; i < GSEG; ++i) {
            a[i] = __builtin_amdgcn_exp2f(s[i] * a2);
            h[i] = fmaf(a[i], i ? h[i - 1] : h0, s[i] * u[i] * r.B[i]);
            y[i] = fmaf(r.C[i], h[i], y[i]);
            v[GSEG + i] = e[i] * h[i];
          }
#pragma unroll
          for (int i = GSEG - 1; i >= 0; --i) {
            q = fmaf(e[i], r.C[i], q);
            v[i] = q * (s[i] * u[i]);
            gb[i] = fmaf(q, r.B[i], gb[i]);
            q *= a[i];
            const float through = q * (i ? h[i - 1] : h0);
            gs[i] = fmaf(through, an, gs[i]);
            dA = fmaf(through, s[i], dA);
          }
          ga[n * 64] = dA;
          const float total = lane_sums(v, w.lane);
          if ((w.lane & 3) == 0) sums[(w.wave * N + n) * 2 * GSEG + (w.lane >> 2)] = total;
        });
#pragma unroll
        for (int i = 0; i < GSEG; ++i) {
          dD = fmaf(e[i], u[i], dD);
          dz[i] *= p.D ? fmaf(dskip, u[i], y[i]) : y[i];
          gs[i] = fmaf(gb[i], u[i], gs[i]) * slope[i];  // d dt
          gb[i] = fmaf(gb[i], s[i], p.D ? e[i] * dskip : 0.f);      // du
        }
        if (t + GSEG > w.end) {
#pragma unroll
          for (int i = 0; i < GSEG; ++i)
            if (t + i >= w.end) gb[i] = gs[i] = dz[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < GSEG; ++i) dbias += gs[i];
        put_seg<T>(p.du, row, rows, d.C, out_t, gb);
        put_seg<T>(p.ddt, row, rows, d.C, out_t, gs);
        if (p.z) put_seg<T>(p.dz, row, rows, d.C, out_t, dz);
      } else {
        for (int i = w.lane; i < N * 2 * GSEG; i += 64) sums[w.wave * N * 2 * GSEG + i] = 0.f;
      }
    } else {
      const float none[GSEG] = {};
      put_seg<T>(p.du, row, rows, d.C, out_t, none);
      put_seg<T>(p.ddt, row, rows, d.C, out_t, none);
      if (p.z) put_seg<T>(p.dz, row, rows, d.C, out_t, none);
    }
    __syncthreads();
    float* const out = p.pBC + ((cb * d.B * d.G + w.bg) * d.T + t) * 2 * N;
    for (int j = threadIdx.x; j < rows * 2 * N; j += blockDim.x) {
      const int n = j % N, which = j / N & 1, i = j / N / 2;
      float v = 0.f;
      if (t + i < w.end)
        for (int k = 0; k < waves; ++k) v += sums[(k * N + n) * 2 * GSEG + which * GSEG + i];
      out[j] = v;
    }
    __syncthreads();
  }
  if (!w.ok) return;
  for (int n = 0; n < N; ++n) {
    p.pA[(w.u * N + n) * d.C + w.c] = ga[n * 64];
    if (p.dstart && w.chunk == 0) p.dstart[(w.b * d.C + w.c) * N + n] = qs[n * 64];
  }
  p.pD[w.u * 2 * d.C + w.c] = dD;
  p.pD[(w.u * 2 + 1) * d.C + w.c] = dbias;
}

// dB, dC [B, T, G, N] from the channel blocks' shares.
template <typename T>
__global__ __launch_bounds__(256) void k_sel_grad_bc(Dims d, const float* __restrict__ pBC, int parts,
                                                     T* __restrict__ dB, T* __restrict__ dC) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t total = d.B * d.G * d.T * 2 * d.N;
  if (i >= total) return;
  float v = 0.f;
  for (int k = 0; k < parts; ++k) v += pBC[k * total + i];
  const int64_t n = i % d.N, which = i / d.N & 1, t = i / d.N / 2 % d.T, bg = i / d.N / 2 / d.T, g = bg % d.G;
  (which ? dC : dB)[((bg / d.G * d.T + t) * d.G + g) * d.N + n] = from_f32<T>(v);
}

// dA [C, N], dD [C] and d dt_bias [C] from the chunks' shares: 64 columns a block, 4 threads a column.
__global__ __launch_bounds__(256) void k_sel_grad_a(Dims d, const float* __restrict__ pA, const float* __restrict__ pD,
                                                    float* __restrict__ dA, float* __restrict__ dD,
                                                    float* __restrict__ dbias) {
  __shared__ float part[4][64];
  const int col = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int64_t NC = static_cast<int64_t>(d.N) * d.C, m = static_cast<int64_t>(blockIdx.x) * 64 + col;
  const int64_t units = d.B * d.chunks;
  float s = 0.f;
  if (m < NC) {
#pragma unroll 8
    for (int64_t k = grp; k < units; k += 4) s += pA[k * NC + m];
  } else if (m < NC + 2 * d.C) {
#pragma unroll 8
    for (int64_t k = grp; k < units; k += 4) s += pD[k * 2 * d.C + m - NC];
  }
  part[grp][col] = s;
  __syncthreads();
  if (grp || m >= NC + 2 * d.C) return;
  s = (part[0][col] + part[1][col]) + (part[2][col] + part[3][col]);
  if (m < NC) {
    if (dA) dA[m % d.C * d.N + m / d.C] = s;
  } else if (m < NC + d.C) {
    if (dD) dD[m - NC] = s;
  } else if (dbias) {
    dbias[m - NC - d.C] = s;
  }
}

// One new token of every sequence: LPC neighbouring lanes hold a channel, four states (16 bytes) each and a
// round; the output is summed over the lanes.  `end` may be the state that is read.  Bound by memory, which is
// the state read and written: 512 x 2048 x 16 134 MB in 32 us, 4.2 TB/s; 8 x 1024 x 16 3.6 us.
template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(256) void k_sel_step(Dims d, Ptrs p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t total = d.B * d.C, j = i / LPC < total ? i / LPC : total - 1;
  const bool ok = i / LPC < total;
  const int part = static_cast<int>(i % LPC);
  const int64_t b = j / d.C;
  const int c = static_cast<int>(j % d.C), g = c / (d.C / d.G);
  const float u = to_f32(static_cast<const T*>(p.u)[b * p.ub + c]);
  float s = to_f32(static_cast<const T*>(p.dt)[b * p.dtb + c]) + (p.bias ? p.bias[c] : 0.f);
  if (d.softplus) s = softplus(s);
  const float x = s * u;
  const float *h = p.start + j * d.N, *A = p.A + static_cast<int64_t>(c) * d.N;
  float* const out = p.end + j * d.N;
  const T *Bm = static_cast<const T*>(p.Bm) + b * p.Bb + g * p.Bg, *Cm = static_cast<const T*>(p.Cm) + b * p.Cb + g * p.Cg;
  float y = 0.f;
  for (int n0 = part * 4; n0 < d.N; n0 += LPC * 4) {
    float hv[4], av[4];
    if constexpr (VEC) {
      const f32x4 hq = *reinterpret_cast<const f32x4*>(h + n0), aq = *reinterpret_cast<const f32x4*>(A + n0);
#pragma unroll
      for (int k = 0; k < 4; ++k) hv[k] = hq[k], av[k] = aq[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) hv[k] = n0 + k < d.N ? h[n0 + k] : 0.f, av[k] = n0 + k < d.N ? A[n0 + k] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (VEC || n0 + k < d.N) {
        hv[k] = fmaf(__builtin_amdgcn_exp2f(s * (rate(av[k]) * LOG2E)), hv[k], x * to_f32(Bm[n0 + k]));
        y = fmaf(to_f32(Cm[n0 + k]), hv[k], y);
      }
    }
    if (!ok) continue;
    if constexpr (VEC) {
      f32x4 hq;
#pragma unroll
      for (int k = 0; k < 4; ++k) hq[k] = hv[k];
      *reinterpret_cast<f32x4*>(out + n0) = hq;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n0 + k < d.N) out[n0 + k] = hv[k];
    }
  }
#pragma unroll
  for (int m = 1; m < LPC; m *= 2) y += __shfl_xor(y, m);
  if (!ok || part) return;
  if (p.D) y = fmaf(p.D[c], u, y);
  if (p.z) {
    const float z = to_f32(static_cast<const T*>(p.z)[b * p.zb + c]);
    y *= z * sigmoid(z);
  }
  static_cast<T*>(p.y)[j] = from_f32<T>(y);
}

// ------------------------------------------------------------------ host
int waves_for(const Dims& d, bool grad) {
  // a wave's states take 512 N bytes of LDS (the backward pass 128 N more): blocks of two waves past 32
  // states, of one past 128, leave a CU several blocks
  const int by_n = d.N <= 32 ? WAVES : d.N <= 128 ? 2 : 1;
  return std::min(by_n, d.cbg);
}

int rows_states(const Dims& d) { return d.N <= 16 ? 16 : d.N <= 32 ? 32 : 64; }  // of a padded tile

// Whether a state a lane serves a forward call: its time grows with a sequence's segments alone until every SIMD
// has its waves, the chunks' with all tokens behind 30 us of their own, and with more than 32 states they have few
// waves.  Measured, rows against chunks, us of a call replayed from a graph (bf16, with the tiles):
//   16 states: 1 x 64 x 2048 9 and 41, 16 x 128 x 1024 27 and 47, 1 x 512 x 512 29 and 41, 3 x 777 x 1000 44 and 59,
//     4 x 1024 x 2048 80 and 98; 2 x 1024 x 1024 53 and 46, 1 x 1024 x 512 52 and 42, 8 x 4096 x 256 183 and 100
//   32 states: 1 x 512 x 1024 33 and 65, 8 x 1024 x 1024 106 and 157
//   64 states: 1 x 64 x 2048 13 and 106, 1 x 512 x 512 49 and 107, 4 x 1024 x 1024 98 and 275
//   4 states (half of a row has nothing to do): 1 x 256 x 512 18 and 25, 8 x 128 x 2048 25 and 27, 4 x 512 x 1024 31 and 27
// Far more waves pay each wave's beginning: 64 x 16 x 2048 with 16 states 39 and 22.  2 x 1024 x 1024 is on the rule's
// slower side.
bool rows_serve(const Dims& d) {
  const int64_t lanes = d.B * d.C;
  if (d.N <= 8) return lanes <= 16384 && d.T <= 256;
  return d.N <= 64 && lanes <= 65536 && (d.T <= 512 || (d.T <= 1024 && (lanes >= 2048 || d.N > 32)));
}

Dims make_dims(const lng_selective& a, bool grad) {
  Dims d{};
  d.B = a.B, d.T = static_cast<int>(a.T), d.C = a.C, d.N = a.N, d.np = a.N, d.G = a.G, d.softplus = a.softplus;
  d.cbg = static_cast<int>(cdiv(a.C / a.G, 64));
  d.segs = static_cast<int>(cdiv(a.T, SEG)), d.gsegs = static_cast<int>(cdiv(a.T, GSEG));
  // chunks of at least four segments, for two waves on each of the 1024 SIMDs (the backward pass, whose waves
  // wait more, four: 553 -> 511 us for a training step of 8 x 2048 x 1024); of two segments where even those
  // leave SIMDs idle (3 x 777 x 1000: 80 -> 55 us)
  const int64_t units = a.B * a.G * d.cbg, goal = grad ? 4096 : 2048;
  int64_t want = std::min<int64_t>(cdiv(goal, std::max<int64_t>(units, 1)), std::max(1, d.segs / 4));
  if (units * want < 2048) want = std::min<int64_t>(cdiv(2048, std::max<int64_t>(units, 1)), std::max(1, d.segs / 2));
  d.chunk = static_cast<int>(std::max<int64_t>(1, cdiv(d.segs, std::max<int64_t>(want, 1)))) * SEG;
  d.chunks = static_cast<int>(std::max<int64_t>(1, cdiv(a.T, d.chunk)));
  d.rows = !grad && rows_serve(d);
  if (d.rows) d.np = rows_states(d);
  return d;
}

struct Space {  // workspace offsets in floats
  int64_t tiles, at, hloc, ssum, pA = 0, pD = 0, pBC = 0, total = 0;
  int64_t take(int64_t n) {
    const int64_t p = total;
    total += (n + 63) & ~int64_t{63};
    return p;
  }
  Space(const Dims& d, bool grad) {
    const int64_t NC = int64_t{d.N} * d.C, units = d.B * d.chunks;
    // room for padded tiles in either direction, so that what serves a shape's backward pass serves its forward
    tiles = take(d.B * d.G * d.segs * SEG * 2 * (rows_serve(d) ? rows_states(d) : d.N));
    at = take(NC);
    hloc = take(d.chunks > 1 ? units * NC : 0);
    ssum = take(d.chunks > 1 ? units * d.C : 0);
    if (!grad) return;
    pA = take(units * NC);
    pD = take(units * 2 * d.C);
    pBC = take(cdiv(d.cbg, waves_for(d, true)) * d.B * d.G * d.T * 2 * d.N);
  }
};

Ptrs make_ptrs(const lng_selective& a) {
  Ptrs p{};
  p.u = a.u, p.dt = a.dt, p.z = a.z, p.Bm = a.Bm, p.Cm = a.Cm;
  p.ub = a.u_batch, p.ut = a.u_token, p.dtb = a.dt_batch, p.dtt = a.dt_token, p.zb = a.z_batch, p.zt = a.z_token;
  p.Bb = a.B_batch, p.Bt = a.B_token, p.Bg = a.B_group, p.Cb = a.C_batch, p.Ct = a.C_token, p.Cg = a.C_group;
  p.A = a.A, p.D = a.D, p.bias = a.dt_bias, p.start = a.state, p.lengths = a.lengths;
  p.y = a.y, p.end = a.state_out, p.ckpt = a.checkpoints;
  return p;
}

int check_args(const char* what, const lng_selective* a) {
  if (!a) return fail(LNG_E_ARG, std::string(what) + ": null arguments");
  if (a->dtype != LNG_F32 && a->dtype != LNG_BF16 && a->dtype != LNG_F16)
    return fail(LNG_E_DTYPE, std::string(what) + ": fp32, bf16 or fp16 tensors");
  if (a->B < 0 || a->T < 0 || a->C <= 0 || a->N <= 0 || a->N > MAX_N || a->G <= 0 || a->C % a->G ||
      a->C > (1 << 20) || a->T > (int64_t{1} << 30) || a->B > (int64_t{1} << 24) ||
      a->B * a->T > (int64_t{1} << 38) / a->C / a->N)
    return fail(LNG_E_ARG, std::string(what) + ": bad shape (1 to 256 states, groups that divide the channels)");
  // a segment's rows are reached by 32-bit offsets from its first one
  const int64_t far = (int64_t{1} << 26) / dtype_size(a->dtype);
  for (const int64_t token : {a->u_token, a->dt_token, a->z_token})
    if (token < 0 || token > far)
      return fail(LNG_E_ARG, std::string(what) + ": rows of u, dt and z are 0 to 2^26 bytes apart");
  if (a->B * a->T > 0 && (!a->u || !a->dt || !a->Bm || !a->Cm || !a->A || (!a->y && !a->checkpoints_in)))
    return fail(LNG_E_ARG, std::string(what) + ": null pointer");
  return LNG_OK;
}

void place(Ptrs& p, const Space& s, void* ws) {
  float* const w = static_cast<float*>(ws);
  p.tiles = w + s.tiles, p.at = w + s.at, p.hloc = w + s.hloc, p.ssum = w + s.ssum, p.pA = w + s.pA, p.pD = w + s.pD;
  p.pBC = w + s.pBC;
}

unsigned grid256(int64_t n) { return static_cast<unsigned>(cdiv(n, 256)); }
int64_t unit_blocks(const Dims& d, int waves) { return cdiv(d.cbg, waves) * d.G * d.chunks * d.B; }
int64_t tile_threads(const Dims& d) { return d.B * d.G * d.segs * SEG * d.np + int64_t{d.C} * d.N; }
int step_lanes(const Dims& d) {  // of a channel
  int lpc = 1;
  while (lpc < 16 && lpc * 4 < d.N) lpc *= 2;
  return lpc;
}

// The launches whose threads grow with the batch.  The others stay below: k_sel_rows serves 2^16 channels of all
// sequences (rows_serve), k_sel_join runs where these give fewer than 4096 waves, k_sel_grad_a has 4 (N + 2) C threads.
int check_threads(const char* what, int64_t threads) {
  if (cdiv(threads, 256) * 256 <= MOST_THREADS) return LNG_OK;
  return fail(LNG_E_ARG, std::string(what) + ": too many tokens, groups or channels for one launch; split the batch");
}
int check_launches(const char* what, const Dims& d, bool grad) {
  const int waves = waves_for(d, grad);
  int64_t most = std::max(tile_threads(d), unit_blocks(d, waves) * 64 * waves);
  if (grad) most = std::max(most, d.B * d.G * d.T * 2 * d.N);
  return check_threads(what, most);
}

unsigned states_lds(const Dims& d, int waves) { return waves * 2 * d.N * 64 * 4; }

template <bool BACK>
void launch_join(const Dims& d, const Ptrs& p, hipStream_t st) {
  const int waves = static_cast<int>(std::min<int64_t>(16, cdiv(d.chunks, JOIN)));
  k_sel_join<BACK><<<static_cast<unsigned>(cdiv(d.B * d.N * d.C, 64)), 64 * waves, 0, st>>>(d, p);
}

template <typename T>
int run_scan(const Dims& d, Ptrs p, hipStream_t st) {
  if (d.rows) {
    k_sel_tiles<T><<<grid256(tile_threads(d)), 256, 0, st>>>(d, p);
    const int cg = d.C / d.G, waves = static_cast<int>(std::min<int64_t>(WAVES, cdiv(cg, 4)));
    const unsigned blocks = static_cast<unsigned>(cdiv(cg, 4 * waves) * d.G * d.B);
    auto launch = [&](auto ck) {
      constexpr bool CK = decltype(ck)::value;
      if (d.np == 16)
        k_sel_rows<T, 1, CK><<<blocks, 64 * waves, 0, st>>>(d, p);
      else if (d.np == 32)
        k_sel_rows<T, 2, CK><<<blocks, 64 * waves, 0, st>>>(d, p);
      else
        k_sel_rows<T, 4, CK><<<blocks, 64 * waves, 0, st>>>(d, p);
    };
    if (p.ckpt)
      launch(std::true_type{});
    else
      launch(std::false_type{});
    return check_launch("selective_scan");
  }
  const int waves = waves_for(d, false);
  const unsigned blocks = static_cast<unsigned>(unit_blocks(d, waves));
  k_sel_tiles<T><<<grid256(tile_threads(d)), 256, 0, st>>>(d, p);
  if (d.chunks > 1) {
    k_sel_scan<T, true><<<blocks, 64 * waves, states_lds(d, waves), st>>>(d, p);
    launch_join<false>(d, p, st);
  }
  k_sel_scan<T, false><<<blocks, 64 * waves, states_lds(d, waves), st>>>(d, p);
  return check_launch("selective_scan");
}

template <typename T>
int run_grad(const Dims& d, Ptrs p, const lng_selective_grad& g, hipStream_t st) {
  const int waves = waves_for(d, true);
  const unsigned blocks = static_cast<unsigned>(unit_blocks(d, waves));
  k_sel_tiles<T><<<grid256(tile_threads(d)), 256, 0, st>>>(d, p);
  if (d.chunks > 1) {
    k_sel_grad_ends<T><<<blocks, 64 * waves, states_lds(d, waves), st>>>(d, p);
    launch_join<true>(d, p, st);
  }
  k_sel_grad<T><<<blocks, 64 * waves, states_lds(d, waves) + waves * d.N * 2 * GSEG * 4, st>>>(d, p);
  k_sel_grad_bc<T><<<grid256(d.B * d.G * d.T * 2 * d.N), 256, 0, st>>>(
      d, p.pBC, static_cast<int>(cdiv(d.cbg, waves)), static_cast<T*>(g.dB), static_cast<T*>(g.dC));
  k_sel_grad_a<<<static_cast<unsigned>(cdiv(int64_t{d.N + 2} * d.C, 64)), 256, 0, st>>>(d, p.pA, p.pD, g.dA, g.dD,
                                                                                       g.ddt_bias);
  return check_launch("selective_scan_grad");
}

template <typename T>
int run_step(const Dims& d, const Ptrs& p, hipStream_t st) {
  const bool vec = d.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.start) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.end) % 16 == 0 && reinterpret_cast<uintptr_t>(p.A) % 16 == 0;
  const int lpc = step_lanes(d);
  const unsigned blocks = grid256(d.B * d.C * lpc);
#define LNG_SEL_STEP(L)                                       \
  if (lpc == L) {                                             \
    if (vec)                                                  \
      k_sel_step<T, L, true><<<blocks, 256, 0, st>>>(d, p);   \
    else                                                      \
      k_sel_step<T, L, false><<<blocks, 256, 0, st>>>(d, p);  \
  }
  LNG_SEL_STEP(1)
  LNG_SEL_STEP(2)
  LNG_SEL_STEP(4)
  LNG_SEL_STEP(8)
  LNG_SEL_STEP(16)
#undef LNG_SEL_STEP
  return check_launch("selective_step");
}

template <typename F>
int with_type(int dtype, F f) {
  if (dtype == LNG_F32) return f(float{});
  if (dtype == LNG_BF16) return f(bf16{});
  return f(_Float16{});
}

}  // namespace
}  // namespace lng

using namespace lng;

extern "C" {

size_t lng_selective_size(void) { return sizeof(lng_selective); }
size_t lng_selective_grad_size(void) { return sizeof(lng_selective_grad); }

size_t lng_selective_workspace_bytes(int64_t B, int64_t T, int32_t C, int32_t N, int32_t G, int grad) {
  lng_selective a{};
  a.B = B, a.T = T, a.C = C, a.N = N, a.G = G, a.dtype = LNG_F32;
  if (B <= 0 || T <= 0 || C <= 0 || N <= 0 || N > MAX_N || G <= 0 || C % G) return 0;
  return static_cast<size_t>(Space(make_dims(a, grad != 0), grad != 0).total) * 4;
}

int64_t lng_selective_checkpoints(int64_t B, int64_t T, int32_t C, int32_t N) {
  if (B <= 0 || T <= 0 || C <= 0 || N <= 0) return 0;
  return B * cdiv(T, GSEG) * N * C;
}

int lng_selective_scan(const lng_selective* args, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_args("selective_scan", args)) return rc;
  const lng_selective& a = *args;
  if (a.B == 0 || a.T == 0) return LNG_OK;
  if (!a.y) return fail(LNG_E_ARG, "selective_scan: null pointer");
  const Dims d = make_dims(a, false);
  if (int rc = check_launches("selective_scan", d, false)) return rc;
  const Space s(d, false);
  if (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 || reinterpret_cast<uintptr_t>(workspace) % 64)
    return fail(LNG_E_ARG, "selective_scan: the workspace is too small or not 64-byte aligned");
  Ptrs p = make_ptrs(a);
  place(p, s, workspace);
  return with_type(a.dtype, [&](auto t) { return run_scan<decltype(t)>(d, p, as_stream(stream)); });
}

int lng_selective_scan_grad(const lng_selective* args, const lng_selective_grad* grads, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = check_args("selective_scan_grad", args)) return rc;
  const lng_selective& a = *args;
  if (!grads) return fail(LNG_E_ARG, "selective_scan_grad: null arguments");
  const lng_selective_grad& g = *grads;
  if (a.B == 0 || a.T == 0) return fail(LNG_E_ARG, "selective_scan_grad: no tokens");
  if (!a.checkpoints_in || !g.dy || !g.du || !g.ddt || !g.dB || !g.dC || (a.z && !g.dz))
    return fail(LNG_E_ARG, "selective_scan_grad: null pointer");
  if (g.dy_token < 0 || g.dy_token > (int64_t{1} << 26) / dtype_size(a.dtype))
    return fail(LNG_E_ARG, "selective_scan_grad: rows of dy are 0 to 2^26 bytes apart");
  const Dims d = make_dims(a, true);
  if (int rc = check_launches("selective_scan_grad", d, true)) return rc;
  const Space s(d, true);
  if (!workspace || workspace_bytes < static_cast<size_t>(s.total) * 4 || reinterpret_cast<uintptr_t>(workspace) % 64)
    return fail(LNG_E_ARG, "selective_scan_grad: the workspace is too small or not 64-byte aligned");
  Ptrs p = make_ptrs(a);
  place(p, s, workspace);
  p.ckpt_in = a.checkpoints_in, p.dy = g.dy, p.dyb = g.dy_batch, p.dyt = g.dy_token, p.dend = g.dstate_out;
  p.du = g.du, p.ddt = g.ddt, p.dz = g.dz, p.dstart = g.dstate;
  return with_type(a.dtype, [&](auto t) { return run_grad<decltype(t)>(d, p, g, as_stream(stream)); });
}

int lng_selective_step(const lng_selective* args, void* stream) {
  if (int rc = check_args("selective_step", args)) return rc;
  const lng_selective& a = *args;
  if (a.T != 1) return fail(LNG_E_ARG, "selective_step: one token of every sequence (T = 1)");
  if (a.B == 0) return LNG_OK;
  if (!a.state || !a.state_out || !a.y) return fail(LNG_E_ARG, "selective_step: null pointer");
  const Dims d = make_dims(a, false);
  if (int rc = check_threads("selective_step", d.B * d.C * step_lanes(d))) return rc;
  const Ptrs p = make_ptrs(a);
  return with_type(a.dtype, [&](auto t) { return run_step<decltype(t)>(d, p, as_stream(stream)); });
}

}  // extern "C"
