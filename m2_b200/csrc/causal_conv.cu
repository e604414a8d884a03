// Short causal convolution of every channel with its own W <= 8 taps, in front of a scan:
//     v_t = bias + sum_i w_i x_{t-W+1+i},      y_t = v_t or silu(v_t),
// its gradients, and one token at a time.  x_{-W+1} .. x_{-1} are the inputs that earlier calls left.  (The reference's short convolution,
// bert/src/mm/monarch_mixer_sequence_mixer.py:118-121, has three taps around a token and lies inside m2_longconv_fwd.)
//
// Bound: memory, x in and y out (gradients: x and dy in, dx out).  A thread walks through a chunk of tokens of a few adjacent channels with the last W - 1
// inputs in registers, so that a token is read once but for the W - 1 in front of a chunk; the next four tokens are under way while four are computed,
// in pairs of channels.
#include "common.cuh"

namespace m2 {
namespace cc {

constexpr int THREADS = 128;
constexpr int MAX_TAPS = 8;

// Blocks that an SM holds at least, by the registers of their taps and windows: what the kernels are bounded to, and what a thread's chunk goes by.  With four
// taps the bound costs spills: 32 bytes forwards (float32 28), 44 in bf16's gradients.
__host__ __device__ constexpr int fwd_blocks(int size, int v, int taps) {
  return taps <= 4 || (size == 4 && v > 1) ? 5 : v == 1 ? (taps <= 7 ? 5 : 4) : taps <= 6 ? 4 : 3;
}
__host__ __device__ constexpr int back_blocks(int size, int taps) { return taps <= 4 || size == 4 ? 3 : 2; }

struct Args {
  int batch, len, dim, taps, silu, chunk, chunks;
  const void* x; long long x_sb, x_st;
  const float *w, *bias;
  const long long* lengths;
  const void* state_in;                  // (batch, taps - 1, dim), packed, oldest first
  void *y, *state_out;
};
struct Grads {
  const void* dy; long long y_sb, y_st;
  const void* d_state_out;
  void *dx, *d_state_in;
  float* part;                           // (parts, taps + 1, dim)
  float *dw, *d_bias;
};

// V adjacent channels as they lie in memory, and as P pairs of float32
template <typename T, int V> struct Vec {
  static constexpr int BYTES = V * (int)sizeof(T), P = (V + 1) / 2, WORDS = (BYTES + 3) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (BYTES == 16) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void get(f32x2 (&f)[P]) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < P; ++i) f[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) f[i] = f2_pack(__uint_as_float(w[2 * i]), V > 1 ? __uint_as_float(w[(2 * i + 1) % WORDS]) : 0.f);
    }
  }
  static __device__ __forceinline__ void put(T* p, const f32x2 (&f)[P]) {
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float x, y;
      f2_unpack(f[i], x, y);
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        w[2 * i] = __float_as_uint(x);
        if constexpr (V > 1) w[2 * i + 1] = __float_as_uint(y);
      }
    }
    if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
};

// a number of each of V channels, step apart
template <int V> __device__ __forceinline__ void channels(const float* p, int step, f32x2 (&f)[(V + 1) / 2]) {
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) f[i] = p ? f2_pack(__ldg(p + 2 * i * step), V > 1 ? __ldg(p + (2 * i + 1) * step) : 0.f) : 0;
}
// the taps of V channels, (dim, W): four at once where they are on 16 bytes
template <int V, int W> __device__ __forceinline__ void taps_of(const float* p, f32x2 (&w)[W][(V + 1) / 2]) {
  if constexpr (W % 4 == 0 && V > 1) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
#pragma unroll
        for (int k = 0; k < W; k += 4) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(p + 2 * i * W + k)), b = __ldg(reinterpret_cast<const float4*>(p + (2 * i + 1) * W + k));
          w[k][i] = f2_pack(a.x, b.x); w[k + 1][i] = f2_pack(a.y, b.y); w[k + 2][i] = f2_pack(a.z, b.z); w[k + 3][i] = f2_pack(a.w, b.w);
        }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < W; ++k) channels<V>(p + k, W, w[k]);
}

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + lp::ex2(-v * lp::LOG2E)); }
__device__ __forceinline__ f32x2 sigmoid2(f32x2 v) {
  float x, y;
  f2_unpack(v, x, y);
  return f2_pack(sigmoid(x), sigmoid(y));
}
__device__ __forceinline__ int text_length(const Args& a, int b) {
  if (!a.lengths) return a.len;
  const long long n = a.lengths[b];
  return (int)(n < 0 ? 0 : n > a.len ? a.len : n);
}

// x_t of a sequence, t >= -(W-1): the inputs that earlier calls left, then the sequence's own; zero behind its end
template <typename T, int V, int W> struct Line {
  const T *x, *before;
  long long st; int dim, n;
  __device__ Line(const Args& a, int b, int c, int n_) : x(static_cast<const T*>(a.x) + b * a.x_sb + c),
      before(a.state_in ? static_cast<const T*>(a.state_in) + (long long)b * (W - 1) * a.dim + c : nullptr), st(a.x_st), dim(a.dim), n(n_) {}
  __device__ __forceinline__ const T* at(int t) const {                // NULL: zero
    return t >= 0 && t < n ? x + t * st : t < 0 && t > -W && before ? before + (long long)(t + W - 1) * dim : nullptr;
  }
  __device__ __forceinline__ void get(int t, f32x2 (&f)[(V + 1) / 2]) const {
    Vec<T, V> v;
    const T* p = at(t);
    if (p) v.load(p);
    else v.clear();
    v.get(f);
  }
};

// The next tokens of a thread, U at a time: copies under way into its own part of shared memory, a ring of R stages of which one is being used, one was
// used before and is asked for anew, and the others are under way; or (pieces below 8 bytes) U of them in registers.
constexpr int U = 4, R = 5;
template <typename T, int V> struct Ring {
  static constexpr bool ASYNC = Vec<T, V>::BYTES >= 8;
  static constexpr int DEPTH = ASYNC ? R : 1, UNDER_WAY = ASYNC ? R - 1 : 1, WORDS = Vec<T, V>::WORDS, SIZE = ASYNC ? R * U * THREADS * WORDS : 1;     // words of shared memory
  uint32_t* sm;
  Vec<T, V> reg[ASYNC ? 1 : U];
  __device__ __forceinline__ Ring(uint32_t* s) : sm(s + threadIdx.x * WORDS) {}
  __device__ __forceinline__ uint32_t* at(int stage, int u) const { return sm + (stage * U + u) * THREADS * WORDS; }
  __device__ __forceinline__ void put(int stage, int u, const T* from) {       // NULL: zero
    if constexpr (ASYNC) {
      uint32_t* to = at(stage, u);
      if (from) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(Vec<T, V>::BYTES) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) to[i] = 0;
      }
    } else {
      if (from) reg[u].load(from);
      else reg[u].clear();
    }
  }
  __device__ __forceinline__ void get(int stage, int u, f32x2 (&f)[Vec<T, V>::P]) const {
    if constexpr (ASYNC) {
      Vec<T, V> v;
      const uint32_t* from = at(stage, u);
      if constexpr (WORDS == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(from);
        v.w[0] = w.x; v.w[1] = w.y; v.w[2] = w.z; v.w[3] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(from);
        v.w[0] = w.x; v.w[1] = w.y;
      }
      v.get(f);
    } else {
      reg[u].get(f);
    }
  }
};
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <bool B> struct Const { static constexpr bool value = B; };

struct Place { int b, chunk, c; bool live; };
template <int V> __device__ __forceinline__ Place place_of(const Args& a) {       // lanes go over channels first
  const int cols = (a.dim + V - 1) / V;
  const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
  Place p;
  p.c = (int)(i % cols) * V;
  const long long r = i / cols;
  p.chunk = (int)(r % a.chunks);
  p.live = r / a.chunks < a.batch;
  p.b = p.live ? (int)(r / a.chunks) : 0;
  return p;
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS, fwd_blocks(sizeof(T), V, W))
conv_kernel(const Args a) {
  constexpr int P = (V + 1) / 2;
  using X = Vec<T, V>;
  pdl_wait();
  const Place p = place_of<V>(a);
  if (!p.live) return;
  const int n = text_length(a, p.b);
  const Line<T, V, W> line(a, p.b, p.c, n);
  const int first = p.chunk * a.chunk, end = min(first + a.chunk, a.len), last = min(end, n);
  constexpr int D = Ring<T, V>::DEPTH, M = Ring<T, V>::UNDER_WAY, AHEAD = M * U;
  __shared__ __align__(16) uint32_t s_ring[Ring<T, V>::SIZE];
  Ring<T, V> next(s_ring);
  const T* x_at = line.x + first * a.x_st;
  int stage = 0;
  for (int s = 0; s < M; ++s) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + s * U + u < last) next.put(s, u, x_at + u * a.x_st);
    x_at += U * a.x_st;
    copies_end();
  }
  f32x2 x[W - 1 + U][P];
#pragma unroll
  for (int i = 0; i < W - 1; ++i) line.get(first - (W - 1) + i, x[i]);
  f32x2 w[W][P], bias[P];
  channels<V>(a.bias ? a.bias + p.c : nullptr, 1, bias);
  taps_of<V, W>(a.w + (long long)p.c * W, w);
  T* y = static_cast<T*>(a.y) + ((long long)p.b * a.len + first) * a.dim + p.c;
  // ALL: neither these U tokens nor those that are asked for now end the chunk
  auto tokens = [&](int t, auto all) {
    constexpr bool ALL = decltype(all)::value;
    copies_but<M - 1>();
#pragma unroll
    for (int u = 0; u < U; ++u) next.get(stage, u, x[W - 1 + u]);
    const int used = stage > 0 ? stage - 1 : D - 1;          // by the tokens before these
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ALL || t + AHEAD + u < last) next.put(used, u, x_at + u * a.x_st);
    copies_end();
    x_at += U * a.x_st;
    stage = stage + 1 < D ? stage + 1 : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!ALL && t + u >= last) break;
      f32x2 v[P];
#pragma unroll
      for (int j = 0; j < P; ++j) {
        v[j] = bias[j];
#pragma unroll
        for (int i = 0; i < W; ++i) v[j] = f2_fma(w[i][j], x[u + i][j], v[j]);
        if (a.silu) v[j] = f2_mul(v[j], sigmoid2(v[j]));
      }
      X::put(y + u * a.dim, v);
    }
    y += U * a.dim;
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) x[i][j] = x[i + U][j];
  };
  int t = first;
  for (; t + AHEAD + U <= last; t += U) tokens(t, Const<true>());
  for (; t < last; t += U) tokens(t, Const<false>());
  const f32x2 zero[P] = {};
  y = static_cast<T*>(a.y) + (long long)p.b * a.len * a.dim + p.c;
  for (t = max(first, last); t < end; ++t) X::put(y + (long long)t * a.dim, zero);
  if (a.state_out && p.chunk == 0) {
    T* s = static_cast<T*>(a.state_out) + (long long)p.b * (W - 1) * a.dim + p.c;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      f32x2 v[P];
      line.get(n - (W - 1) + i, v);
      X::put(s + (long long)i * a.dim, v);
    }
  }
}

// dx_s = sum_i w_i dv_{s+W-1-i}, dv = dy silu'(v), with v computed again; a chunk's tokens s and the W - 1 behind them are walked through, so that
// every chunk has all that its own dx need.  A thread's sums of dw and dbias are its chunk's part.
template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS, back_blocks(sizeof(T), W))
back_kernel(const Args a, const Grads g) {
  constexpr int P = (V + 1) / 2;
  using X = Vec<T, V>;
  pdl_wait();
  const Place p = place_of<V>(a);
  if (!p.live) return;
  const int n = text_length(a, p.b);
  const Line<T, V, W> line(a, p.b, p.c, n);
  const T* dy = static_cast<const T*>(g.dy) + p.b * g.y_sb + p.c;
  const T* ds = g.d_state_out ? static_cast<const T*>(g.d_state_out) + (long long)p.b * (W - 1) * a.dim + p.c : nullptr;
  const int first = p.chunk * a.chunk, end = min(first + a.chunk, a.len), last = min(end, n);
  // the first chunk also has the inputs in front of the sequence
  const int lo = p.chunk == 0 ? -(W - 1) : first;
  const int stop = max(last, p.chunk == 0 ? 0 : first) + W - 1;        // the last s whose gradient is not zero by its place, and what it needs
  constexpr int D = Ring<T, V>::DEPTH, M = Ring<T, V>::UNDER_WAY, AHEAD = M * U;
  __shared__ __align__(16) uint32_t s_x[Ring<T, V>::SIZE], s_y[Ring<T, V>::SIZE];
  Ring<T, V> next_x(s_x), next_y(s_y);
  auto ask = [&](int stage, int t0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u;
      next_x.put(stage, u, t < stop ? line.at(t) : nullptr);
      next_y.put(stage, u, t >= 0 && t < n && t < stop ? dy + t * g.y_st : nullptr);
    }
    copies_end();
  };
  for (int s = 0; s < M; ++s) ask(s, lo + s * U);
  int stage = 0;
  f32x2 w[W][P], bias[P], dw[W][P], db[P];
  channels<V>(a.bias ? a.bias + p.c : nullptr, 1, bias);
  taps_of<V, W>(a.w + (long long)p.c * W, w);
  f32x2 x[W - 1 + U][P], dv[W - 1 + U][P];                             // x_{t-W+1} .. x_{t+U-1} and dv of the same
#pragma unroll
  for (int i = 0; i < W - 1; ++i) {
    line.get(p.chunk == 0 ? n : lo - (W - 1) + i, x[i]);               // in front of what lies in front of a text: zero
#pragma unroll
    for (int j = 0; j < P; ++j) dv[i][j] = 0;
  }
#pragma unroll
  for (int j = 0; j < P; ++j) {
    db[j] = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) dw[i][j] = 0;
  }
  T* dx = static_cast<T*>(g.dx) + (long long)p.b * a.len * a.dim + p.c;
  T* d_before = g.d_state_in ? static_cast<T*>(g.d_state_in) + (long long)p.b * (W - 1) * a.dim + p.c : nullptr;
  // ALL: these U tokens, the W - 1 in front of them and those that are asked for now are the chunk's own
  const T *x_at = line.x + (lo + AHEAD) * a.x_st, *y_at = dy + (lo + AHEAD) * g.y_st;
  T* o_at = dx + (long long)(lo - (W - 1)) * a.dim;
  auto tokens = [&](int t0, auto all) {
    constexpr bool ALL = decltype(all)::value;
    copies_but<M - 1>();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next_x.get(stage, u, x[W - 1 + u]);
      next_y.get(stage, u, dv[W - 1 + u]);
    }
    const int used = stage > 0 ? stage - 1 : D - 1;          // by the tokens before these
    if constexpr (ALL) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        next_x.put(used, u, x_at + u * a.x_st);
        next_y.put(used, u, y_at + u * g.y_st);
      }
      copies_end();
    } else {
      ask(used, t0 + AHEAD);
    }
    stage = stage + 1 < D ? stage + 1 : 0;
    x_at += U * a.x_st;
    y_at += U * g.y_st;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u;
      if (!ALL && t >= stop) break;
      const bool own = ALL || (t >= max(first, 0) && t < last);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        f32x2 e = dv[W - 1 + u][j];                                    // dy, 0 where there is none
        if (a.silu) {
          f32x2 v = bias[j];
#pragma unroll
          for (int i = 0; i < W; ++i) v = f2_fma(w[i][j], x[u + i][j], v);
          const f32x2 s = sigmoid2(v);
          // silu' = s (1 + v (1 - s))
          const f32x2 rest = f2_fma(s, f2_splat(-1.f), f2_splat(1.f));
          const f32x2 slope = f2_mul(s, f2_fma(v, rest, f2_splat(1.f)));
          if (ALL || (t >= 0 && t < n)) e = f2_mul(e, slope);          // elsewhere x may be anything
          dv[W - 1 + u][j] = e;
        }
        if (own) {
          db[j] = f2_add(db[j], e);
#pragma unroll
          for (int i = 0; i < W; ++i) dw[i][j] = f2_fma(e, x[u + i][j], dw[i][j]);
        }
      }
      const int s = t - (W - 1);
      if (ALL || (s >= lo && (s >= 0 || d_before))) {
        f32x2 o[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          o[j] = f2_mul(w[0][j], dv[W - 1 + u][j]);
#pragma unroll
          for (int i = 1; i < W; ++i) o[j] = f2_fma(w[i][j], dv[W - 1 + u - i][j], o[j]);
        }
        if (!ALL && ds && s >= n - (W - 1) && s < n) {
          X v;
          f32x2 q[P];
          v.load(ds + (long long)(s - n + W - 1) * a.dim);
          v.get(q);
#pragma unroll
          for (int j = 0; j < P; ++j) o[j] = f2_add(o[j], q[j]);
        }
        if (ALL || s >= 0) { if (ALL || s < last) X::put(o_at + u * a.dim, o); }
        else X::put(d_before + (long long)(s + W - 1) * a.dim, o);
      }
    }
    o_at += U * a.dim;
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) { x[i][j] = x[i + U][j]; dv[i][j] = dv[i + U][j]; }
  };
  int t0 = lo;
  for (; t0 < max(lo, 0) + W - 1 && t0 < stop; t0 += U) tokens(t0, Const<false>());
  for (; t0 + AHEAD + U <= last; t0 += U) tokens(t0, Const<true>());
  for (; t0 < stop; t0 += U) tokens(t0, Const<false>());
  const f32x2 zero[P] = {};
  for (int t = max(first, last); t < end; ++t) X::put(dx + (long long)t * a.dim, zero);
  float* part = g.part + ((long long)p.b * a.chunks + p.chunk) * (W + 1) * a.dim + p.c;
#pragma unroll
  for (int i = 0; i <= W; ++i) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float f[2];
      f2_unpack(i < W ? dw[i % W][j] : db[j], f[0], f[1]);
      part[(long long)i * a.dim + 2 * j] = f[0];
      if (V > 1) part[(long long)i * a.dim + 2 * j + 1] = f[1];
    }
  }
}

// Sums of the chunks' parts: 32 columns a block, 8 threads a column, eight parts of each at a time in float32, these in 64 bits and in order.
__global__ void __launch_bounds__(256)
sum_kernel(const float* __restrict__ part, float* dw, float* d_bias, int parts, int taps, int dim) {
  __shared__ double s[8][32];
  pdl_wait();
  const long long i = blockIdx.x * 32LL + (threadIdx.x & 31), n = (long long)(taps + 1) * dim;
  const int y = threadIdx.x >> 5;
  double v = 0.0;
  if (i < n) {
    for (int k = y; k < parts; k += 64) {
      float eight = 0.f;
#pragma unroll
      for (int j = 0; j < 64; j += 8) eight += k + j < parts ? part[(k + j) * n + i] : 0.f;
      v += eight;
    }
  }
  s[y][threadIdx.x & 31] = v;
  __syncthreads();
  if (y || i >= n) return;
  v = s[0][threadIdx.x];
#pragma unroll
  for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
  const int tap = (int)(i / dim), c = (int)(i % dim);
  if (tap < taps) { if (dw) dw[(long long)c * taps + tap] = (float)v; }
  else if (d_bias) d_bias[c] = (float)v;
}

struct StepArgs {
  int batch, dim, taps, silu;
  const void* x; long long x_sb;
  const float *w, *bias;
  void* state; long long s_b;
  void* y;
};

template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
step_kernel(const StepArgs a) {
  pdl_wait();
  const int cols = (a.dim + V - 1) / V;
  const long long i = blockIdx.x * (long long)THREADS + threadIdx.x;
  if (i >= (long long)a.batch * cols) return;
  const int b = (int)(i / cols), c = (int)(i % cols) * V, W = a.taps;
  constexpr int P = (V + 1) / 2;
  using X = Vec<T, V>;
  T* s = static_cast<T*>(a.state) + b * a.s_b + c;
  X x[MAX_TAPS], last;
#pragma unroll
  for (int k = 0; k < MAX_TAPS - 1; ++k)
    if (k < W - 1) x[k].load(s + (long long)k * a.dim);
  last.load(static_cast<const T*>(a.x) + b * a.x_sb + c);
  f32x2 v[P];
  channels<V>(a.bias ? a.bias + c : nullptr, 1, v);
  auto add = [&](const X& in, int k) {
    f32x2 f[P], w[P];
    in.get(f);
    channels<V>(a.w + (long long)c * W + k, W, w);
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = f2_fma(w[j], f[j], v[j]);
  };
#pragma unroll
  for (int k = 0; k < MAX_TAPS - 1; ++k)
    if (k < W - 1) add(x[k], k);
  add(last, W - 1);
  if (a.silu) {
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = f2_mul(v[j], sigmoid2(v[j]));
  }
  X::put(static_cast<T*>(a.y) + (long long)b * a.dim + c, v);
  auto keep = [&](const X& in, int k) {
    f32x2 f[P];
    in.get(f);
    X::put(s + (long long)k * a.dim, f);
  };
#pragma unroll
  for (int k = 1; k < MAX_TAPS - 1; ++k)
    if (k < W - 1) keep(x[k], k - 1);
  if (W > 1) keep(last, W - 2);
}

// ---- host ------------------------------------------------------------------------------------------------------------
// Tokens of a thread: as many as let all threads run at once (a block that starts waits for its taps and its first tokens: 16 x 2048 x 1536 in four
// rounds of 32 tokens took 55 us), but 8 at least, as W - 1 in front of them are read twice.
static int chunk_of(int batch, int len, int dim, int v, int an_sm, int least) {
  const long long cols = (dim + v - 1) / v, threads = (long long)an_sm * THREADS * m2_sm_count();
  long long chunks = threads / (batch * cols);
  if (chunks < 1) chunks = 1;
  const long long chunk = (len + chunks - 1) / chunks;
  return chunk < least ? least : (int)chunk;
}
// Of the gradients: their parameters' sums leave W + 1 numbers a channel and chunk, and each chunk walks W - 1 tokens further.  The width of a
// thread goes by the tensors' alignment, chunks do not, as the bits of the parameters' sums go by them: they are those of the widest thread of the type (size bytes a value).
// A thread adds at most 256 tokens one by one: 8192 in one round of threads were off by 1e-4 where all roundings go one way (and slower: 64 x 8192 x 1536 bf16 in chunks of
// 4096 took 1123 us, in chunks of 256 1079).
static int back_chunk_of(int batch, int len, int dim, int taps, int size) {
  const int chunk = chunk_of(batch, len, dim, 8 / size, back_blocks(size, taps), 16), rounds = (chunk + 255) / 256;
  return (chunk + rounds - 1) / rounds;
}
static int chunks_of(int len, int chunk) { return len > 0 ? (len + chunk - 1) / chunk : 1; }

// channels of a thread: 8 bytes (float32 forward with few taps 16); one where a row does not allow it
static bool wide(const void* p, long long sb, long long st, int dim, int size, int bytes) {
  return !p || (m2_aligned(p, bytes) && sb * size % bytes == 0 && st * size % bytes == 0 && (long long)dim * size % bytes == 0);
}

template <typename T, int V, int W> static int forward(const Args& a, cudaStream_t st) {
  const long long threads = (long long)a.batch * a.chunks * ((a.dim + V - 1) / V), blocks = (threads + THREADS - 1) / THREADS;
  M2_REQUIRE(blocks <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_causal_conv_fwd: %d sequences of %d tokens are more than the grid takes", a.batch, a.len);
  return m2_launch("m2_causal_conv_fwd", (long long)a.batch * a.len * a.dim, conv_kernel<T, V, W>, dim3((unsigned)blocks), THREADS, 0, st, a);
}
template <typename T, int V, int W> static int backward(const Args& a, const Grads& g, cudaStream_t st) {
  const long long threads = (long long)a.batch * a.chunks * ((a.dim + V - 1) / V), blocks = (threads + THREADS - 1) / THREADS;
  M2_REQUIRE(blocks <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_causal_conv_bwd: %d sequences of %d tokens are more than the grid takes", a.batch, a.len);
  const long long size = (long long)a.batch * a.len * a.dim;
  if (int rc = m2_launch("m2_causal_conv_bwd", size, back_kernel<T, V, W>, dim3((unsigned)blocks), THREADS, 0, st, a, g)) return rc;
  if (!g.dw && !g.d_bias) return M2_OK;
  const long long n = (long long)(W + 1) * a.dim;
  return m2_launch("m2_causal_conv_bwd", size, sum_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, st, g.part, g.dw, g.d_bias, a.batch * a.chunks, W, a.dim);
}

// FEW channels a thread with up to 4 taps, MANY taps with fewer; one where the rows are in no such pieces
template <typename T, int FEW, int MANY, bool BACK> static int by_taps(const Args& a, const Grads& g, cudaStream_t st) {
#define M2_CC_CASE(W_) case W_: { constexpr int V = W_ <= 4 ? FEW : MANY; if constexpr (BACK) return backward<T, V, W_>(a, g, st); else return forward<T, V, W_>(a, st); }
  switch (a.taps) {
    M2_CC_CASE(1) M2_CC_CASE(2) M2_CC_CASE(3) M2_CC_CASE(4) M2_CC_CASE(5) M2_CC_CASE(6) M2_CC_CASE(7) M2_CC_CASE(8)
  }
#undef M2_CC_CASE
  return M2_ERR_UNSUPPORTED;
}

static int check(const char* name, const m2_causal_conv_args& g, Args& a) {
  M2_REQUIRE(g.batch >= 0 && g.seq_len >= 0 && g.dim >= 1 && g.taps >= 1, M2_ERR_ARG, "%s: %d sequences of %d tokens, %d channels, %d taps", name, g.batch,
             g.seq_len, g.dim, g.taps);
  M2_REQUIRE(g.taps <= MAX_TAPS, M2_ERR_UNSUPPORTED, "%s: %d taps (at most %d)", name, g.taps, MAX_TAPS);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: tensors are float32 or bf16", name);
  M2_REQUIRE(g.seq_len <= 1 << 28 && g.dim <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: %d tokens of %d channels", name, g.seq_len, g.dim);
  a = Args{};
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.weight && (g.x || g.seq_len == 0), M2_ERR_ARG, "%s: x or weight is NULL", name);
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.x, size) && m2_aligned(g.state_in, size) && m2_aligned(g.y, size) && m2_aligned(g.state_out, size) && m2_aligned(g.lengths, 8),
             M2_ERR_ALIGN, "%s: a tensor is not aligned to its type", name);
  a.batch = g.batch; a.len = g.seq_len; a.dim = g.dim; a.taps = g.taps; a.silu = g.silu; a.x = g.x; a.x_sb = g.x_sb; a.x_st = g.x_st;
  a.w = g.weight; a.bias = g.bias; a.lengths = (const long long*)g.lengths; a.state_in = g.taps > 1 ? g.state_in : nullptr;
  a.y = g.y; a.state_out = g.taps > 1 ? g.state_out : nullptr;
  return M2_OK;
}

}  // namespace cc
}  // namespace m2

extern "C" long long m2_causal_conv_workspace(int batch, int seq_len, int dim, int taps) {
  using namespace m2::cc;
  if (batch <= 0 || seq_len < 0 || dim <= 0 || taps <= 0 || taps > MAX_TAPS) return 0;
  const int few = chunks_of(seq_len, back_chunk_of(batch, seq_len, dim, taps, 4)), many = chunks_of(seq_len, back_chunk_of(batch, seq_len, dim, taps, 2));
  return 4LL * batch * (few > many ? few : many) * (taps + 1) * dim;       // of either type
}

extern "C" int m2_causal_conv_fwd(const m2_causal_conv_args* args, void* stream) {
  using namespace m2::cc;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_causal_conv_fwd: args is NULL");
  const m2_causal_conv_args& g = *args;
  Args a;
  if (int rc = check("m2_causal_conv_fwd", g, a)) return rc;
  if (g.batch == 0 || (g.seq_len == 0 && !a.state_out)) return M2_OK;
  M2_REQUIRE(g.y || g.seq_len == 0, M2_ERR_ARG, "m2_causal_conv_fwd: y is NULL");
  const int size = g.dtype == M2_F32 ? 4 : 2;
  const cudaStream_t st = (cudaStream_t)stream;
  const int bytes = g.dtype == M2_F32 && g.taps <= 4 ? 16 : 8;
  const bool vec = wide(g.x, g.x_sb, g.x_st, g.dim, size, bytes) && wide(a.state_in, 0, 0, g.dim, size, bytes) && wide(g.y, 0, 0, g.dim, size, bytes) &&
                   wide(a.state_out, 0, 0, g.dim, size, bytes);
  const int v = vec ? bytes / size : 1;
  a.chunk = chunk_of(g.batch, g.seq_len, g.dim, v, fwd_blocks(size, v, g.taps), 8);
  a.chunks = chunks_of(g.seq_len, a.chunk);
  const Grads none = {};
  if (g.dtype == M2_F32) return vec ? by_taps<float, 4, 2, false>(a, none, st) : by_taps<float, 1, 1, false>(a, none, st);
  return vec ? by_taps<__nv_bfloat16, 4, 4, false>(a, none, st) : by_taps<__nv_bfloat16, 1, 1, false>(a, none, st);
}

extern "C" int m2_causal_conv_bwd(const m2_causal_conv_args* args, const m2_causal_conv_grads* grads, void* stream) {
  using namespace m2::cc;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_causal_conv_bwd: args or grads is NULL");
  const m2_causal_conv_args& g = *args;
  const m2_causal_conv_grads& o = *grads;
  Args a;
  if (int rc = check("m2_causal_conv_bwd", g, a)) return rc;
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.seq_len == 0 || (o.d_y && o.d_x), M2_ERR_ARG, "m2_causal_conv_bwd: d_y or d_x is NULL");
  const long long need = m2_causal_conv_workspace(g.batch, g.seq_len, g.dim, g.taps);
  M2_REQUIRE(o.workspace && o.workspace_bytes >= need, M2_ERR_ARG, "m2_causal_conv_bwd: the workspace has %lld bytes of %lld",
             o.workspace ? o.workspace_bytes : 0, need);
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(o.d_y, size) && m2_aligned(o.d_x, size) && m2_aligned(o.d_state_out, size) && m2_aligned(o.d_state_in, size) && m2_aligned(o.workspace, 16),
             M2_ERR_ALIGN, "m2_causal_conv_bwd: a gradient is not aligned to its type, or the workspace not to 16 bytes");
  const Grads r = {o.d_y, o.y_sb, o.y_st, g.taps > 1 ? o.d_state_out : nullptr, o.d_x, g.taps > 1 ? o.d_state_in : nullptr, o.workspace, o.d_weight, o.d_bias};
  const int bytes = 8;
  const bool vec = wide(g.x, g.x_sb, g.x_st, g.dim, size, bytes) && wide(a.state_in, 0, 0, g.dim, size, bytes) && wide(o.d_y, o.y_sb, o.y_st, g.dim, size, bytes) &&
                   wide(o.d_x, 0, 0, g.dim, size, bytes) && wide(r.d_state_out, 0, 0, g.dim, size, bytes) && wide(r.d_state_in, 0, 0, g.dim, size, bytes);
  a.chunk = back_chunk_of(g.batch, g.seq_len, g.dim, g.taps, size);
  a.chunks = chunks_of(g.seq_len, a.chunk);
  const cudaStream_t st = (cudaStream_t)stream;
  if (g.dtype == M2_F32) return vec ? by_taps<float, 2, 2, true>(a, r, st) : by_taps<float, 1, 1, true>(a, r, st);
  return vec ? by_taps<__nv_bfloat16, 4, 4, true>(a, r, st) : by_taps<__nv_bfloat16, 1, 1, true>(a, r, st);
}

extern "C" int m2_causal_conv_step(const m2_causal_conv_step_args* args, void* stream) {
  using namespace m2::cc;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_causal_conv_step: args is NULL");
  const m2_causal_conv_step_args& g = *args;
  M2_REQUIRE(g.batch >= 0 && g.dim >= 1 && g.taps >= 1, M2_ERR_ARG, "m2_causal_conv_step: %d sequences, %d channels, %d taps", g.batch, g.dim, g.taps);
  M2_REQUIRE(g.taps <= MAX_TAPS, M2_ERR_UNSUPPORTED, "m2_causal_conv_step: %d taps (at most %d)", g.taps, MAX_TAPS);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "m2_causal_conv_step: tensors are float32 or bf16");
  M2_REQUIRE(g.dim <= 1 << 24 && ((long long)g.batch * g.dim + THREADS - 1) / THREADS <= 0x7fffffffLL, M2_ERR_UNSUPPORTED,
             "m2_causal_conv_step: %d sequences of %d channels are more than the grid takes", g.batch, g.dim);
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.x && g.weight && g.y && (g.state || g.taps == 1), M2_ERR_ARG, "m2_causal_conv_step: a tensor is NULL");
  M2_REQUIRE(g.batch == 1 || g.taps == 1 || g.s_b >= (long long)(g.taps - 1) * g.dim, M2_ERR_ARG, "m2_causal_conv_step: states overlap");
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.x, size) && m2_aligned(g.state, size) && m2_aligned(g.y, size), M2_ERR_ALIGN, "m2_causal_conv_step: a tensor is not aligned to its type");
  const StepArgs a = {g.batch, g.dim, g.taps, g.silu, g.x, g.x_sb, g.weight, g.bias, g.state, g.s_b, g.y};
  const bool vec = wide(g.x, g.x_sb, 0, g.dim, size, 8) && wide(g.taps > 1 ? g.state : nullptr, g.s_b, 0, g.dim, size, 8) && wide(g.y, 0, 0, g.dim, size, 8);
  const int v = vec ? 8 / size : 1;
  const long long blocks = ((long long)g.batch * ((g.dim + v - 1) / v) + THREADS - 1) / THREADS, elements = (long long)g.batch * g.dim * g.taps;
  const cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return m2_launch("m2_causal_conv_step", elements, kernel, dim3((unsigned)blocks), THREADS, 0, st, a); };
  if (g.dtype == M2_F32) return vec ? go(step_kernel<float, 2>) : go(step_kernel<float, 1>);
  return vec ? go(step_kernel<__nv_bfloat16, 4>) : go(step_kernel<__nv_bfloat16, 1>);
}
