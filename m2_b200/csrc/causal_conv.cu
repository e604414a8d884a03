// Short causal convolution of every channel with its own W <= 8 taps, in front of a scan:
//     v_t = bias + sum_i w_i x_{t-W+1+i},      y_t = v_t or silu(v_t),
// its gradients, and one token at a time.  x_{-W+1} .. x_{-1} are the inputs that earlier calls left.  (The reference's short convolution,
// bert/src/mm/monarch_mixer_sequence_mixer.py:118-121, has three taps around a token and lies inside m2_longconv_fwd.)
//
// Bound: memory, x in and y out (gradients: x and dy in, dx out).  A thread walks through CHUNK tokens of a few adjacent channels with the last W - 1
// inputs in registers, so that a token is read once but for the W - 1 in front of a chunk.
#include "common.cuh"

namespace m2 {
namespace cc {

constexpr int THREADS = 128;
constexpr int MAX_TAPS = 8;

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

template <typename T, int V> struct Vec {                              // V adjacent channels
  static constexpr int BYTES = V * (int)sizeof(T);
  static __device__ __forceinline__ void get(const T* p, float (&f)[V]) {
    if constexpr (BYTES == 16) {
      lp::Piece<T>::get(__ldg(reinterpret_cast<const uint4*>(p)), f);
    } else if constexpr (BYTES == 8) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      if constexpr (sizeof(T) == 2) {
        f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
        f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
      } else {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = lp::load1(p + j);
    }
  }
  static __device__ __forceinline__ void put(T* p, const float (&f)[V]) {
    if constexpr (BYTES == 16) {
      *reinterpret_cast<uint4*>(p) = lp::Piece<T>::put(f);
    } else if constexpr (BYTES == 8) {
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      } else {
        *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) st_from_float(p + j, f[j]);
    }
  }
};

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + lp::ex2(-v * lp::LOG2E)); }
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
  __device__ __forceinline__ void get(int t, float (&f)[V]) const {
    if (t >= 0 && t < n) { Vec<T, V>::get(x + t * st, f); return; }
    if (t < 0 && before) { Vec<T, V>::get(before + (long long)(t + W - 1) * dim, f); return; }
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = 0.f;
  }
};

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
__global__ void __launch_bounds__(THREADS)
conv_kernel(const Args a) {
  constexpr int U = 4;                   // tokens whose loads are under way together
  pdl_wait();
  const Place p = place_of<V>(a);
  if (!p.live) return;
  const int n = text_length(a, p.b);
  const Line<T, V, W> line(a, p.b, p.c, n);
  const int first = p.chunk * a.chunk, end = min(first + a.chunk, a.len), last = min(end, n);
  float w[W][V], bias[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bias[j] = a.bias ? __ldg(a.bias + p.c + j) : 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) w[i][j] = __ldg(a.w + (long long)(p.c + j) * W + i);
  }
  float x[W - 1 + U][V];
#pragma unroll
  for (int i = 0; i < W - 1; ++i) line.get(first - (W - 1) + i, x[i]);
  T* y = static_cast<T*>(a.y) + (long long)p.b * a.len * a.dim + p.c;
  for (int t = first; t < last; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) line.get(t + u < last ? t + u : n, x[W - 1 + u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= last) break;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = bias[j];
#pragma unroll
        for (int i = 0; i < W; ++i) v[j] = fmaf(w[i][j], x[u + i][j], v[j]);
        if (a.silu) v[j] *= sigmoid(v[j]);
      }
      Vec<T, V>::put(y + (long long)(t + u) * a.dim, v);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = x[i + U][j];
  }
  const float zero[V] = {};
  for (int t = max(first, last); t < end; ++t) Vec<T, V>::put(y + (long long)t * a.dim, zero);
  if (a.state_out && p.chunk == 0) {
    T* s = static_cast<T*>(a.state_out) + (long long)p.b * (W - 1) * a.dim + p.c;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      float v[V];
      line.get(n - (W - 1) + i, v);
      Vec<T, V>::put(s + (long long)i * a.dim, v);
    }
  }
}

// dx_s = sum_i w_i dv_{s+W-1-i}, dv = dy silu'(v), with v computed again; a chunk's tokens s and the W - 1 behind them are walked through, so that
// every chunk has all that its own dx need.  Sums of dw and dbias over a block's chunks of one column of channels, then over the blocks.
template <typename T, int V, int W>
__global__ void __launch_bounds__(THREADS)
back_kernel(const Args a, const Grads g) {
  pdl_wait();
  const Place p = place_of<V>(a);
  if (!p.live) return;
  const int n = text_length(a, p.b);
  const Line<T, V, W> line(a, p.b, p.c, n);
  const T* dy = static_cast<const T*>(g.dy) + p.b * g.y_sb + p.c;
  const T* ds = g.d_state_out ? static_cast<const T*>(g.d_state_out) + (long long)p.b * (W - 1) * a.dim + p.c : nullptr;
  const int first = p.chunk * a.chunk, end = min(first + a.chunk, a.len), last = min(end, n);
  float w[W][V], bias[V], dw[W][V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bias[j] = a.bias ? __ldg(a.bias + p.c + j) : 0.f;
    db[j] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      w[i][j] = __ldg(a.w + (long long)(p.c + j) * W + i);
      dw[i][j] = 0.f;
    }
  }
  T* dx = static_cast<T*>(g.dx) + (long long)p.b * a.len * a.dim + p.c;
  T* d_before = g.d_state_in ? static_cast<T*>(g.d_state_in) + (long long)p.b * (W - 1) * a.dim + p.c : nullptr;
  // the first chunk also has the inputs in front of the sequence
  const int lo = p.chunk == 0 ? -(W - 1) : first;
  float x[W][V], dv[W][V];               // x_{t-W+1} .. x_t; dv_{t-W+1} .. dv_t
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i > 0) line.get(lo - W + i < -(W - 1) ? n : lo - W + i, x[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (i == 0 || lo - W + i < -(W - 1)) x[i][j] = 0.f;
      dv[i][j] = 0.f;
    }
  }
  const int stop = max(last, p.chunk == 0 ? 0 : first);                // one behind the last s whose gradient is not zero by its place
  for (int t = lo; t < stop + W - 1; ++t) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) { x[i][j] = x[i + 1][j]; dv[i][j] = dv[i + 1][j]; }
    line.get(t, x[W - 1]);
    const bool in = t >= 0 && t < n, own = in && t >= first && t < last;
    float d[V];
    if (in) Vec<T, V>::get(dy + t * g.y_st, d);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float e = 0.f;
      if (in) {
        e = d[j];
        if (a.silu) {
          float v = bias[j];
#pragma unroll
          for (int i = 0; i < W; ++i) v = fmaf(w[i][j], x[i][j], v);
          const float s = sigmoid(v);
          e *= s * fmaf(v, 1.f - s, 1.f);
        }
      }
      dv[W - 1][j] = e;
      if (own) {
        db[j] += e;
#pragma unroll
        for (int i = 0; i < W; ++i) dw[i][j] = fmaf(e, x[i][j], dw[i][j]);
      }
    }
    const int s = t - (W - 1);
    if (s >= lo && (s >= 0 || d_before)) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        o[j] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) o[j] = fmaf(w[i][j], dv[W - 1 - i][j], o[j]);
      }
      if (ds && s >= n - (W - 1) && s < n) {
        float q[V];
        Vec<T, V>::get(ds + (long long)(s - n + W - 1) * a.dim, q);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += q[j];
      }
      if (s >= 0) { if (s < last) Vec<T, V>::put(dx + (long long)s * a.dim, o); }
      else Vec<T, V>::put(d_before + (long long)(s + W - 1) * a.dim, o);
    }
  }
  const float zero[V] = {};
  for (int t = max(first, last); t < end; ++t) Vec<T, V>::put(dx + (long long)t * a.dim, zero);
  float* part = g.part + ((long long)p.b * a.chunks + p.chunk) * (W + 1) * a.dim + p.c;
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int i = 0; i < W; ++i) part[(long long)i * a.dim + j] = dw[i][j];
    part[(long long)W * a.dim + j] = db[j];
  }
}

// Sums of the chunks' parts: 32 columns a block, 8 parts side by side, then these in order.
__global__ void __launch_bounds__(256)
sum_kernel(const float* __restrict__ part, float* dw, float* d_bias, int parts, int taps, int dim) {
  __shared__ float s[8][32];
  pdl_wait();
  const long long i = blockIdx.x * 32LL + (threadIdx.x & 31), n = (long long)(taps + 1) * dim;
  const int y = threadIdx.x >> 5;
  float v = 0.f;
  if (i < n)
    for (int k = y; k < parts; k += 8) v += part[k * n + i];
  s[y][threadIdx.x & 31] = v;
  __syncthreads();
  if (y || i >= n) return;
  v = s[0][threadIdx.x];
#pragma unroll
  for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
  const int tap = (int)(i / dim), c = (int)(i % dim);
  if (tap < taps) { if (dw) dw[(long long)c * taps + tap] = v; }
  else if (d_bias) d_bias[c] = v;
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
  T* s = static_cast<T*>(a.state) + b * a.s_b + c;
  float x[MAX_TAPS][V], v[V];
#pragma unroll
  for (int k = 0; k < MAX_TAPS; ++k) {
    if (k < W - 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = 0.f;
      Vec<T, V>::get(s + (long long)k * a.dim, x[k]);
    }
  }
  float last[V];
  Vec<T, V>::get(static_cast<const T*>(a.x) + b * a.x_sb + c, last);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    v[j] = a.bias ? __ldg(a.bias + c + j) : 0.f;
#pragma unroll
    for (int k = 0; k < MAX_TAPS; ++k)
      if (k < W - 1) v[j] = fmaf(__ldg(a.w + (long long)(c + j) * W + k), x[k][j], v[j]);
    v[j] = fmaf(__ldg(a.w + (long long)(c + j) * W + W - 1), last[j], v[j]);
    if (a.silu) v[j] *= sigmoid(v[j]);
  }
  Vec<T, V>::put(static_cast<T*>(a.y) + (long long)b * a.dim + c, v);
#pragma unroll
  for (int k = 1; k < MAX_TAPS; ++k)
    if (k < W - 1) Vec<T, V>::put(s + (long long)(k - 1) * a.dim, x[k]);
  if (W > 1) Vec<T, V>::put(s + (long long)(W - 2) * a.dim, last);
}

// ---- host ------------------------------------------------------------------------------------------------------------
// Tokens of a thread: 32, fewer where that leaves SMs without 8 warps (two of 128 tokens have W - 1 in front of them read twice).
static int chunk_of(int batch, int len, int dim, int v) {
  const long long cols = (dim + v - 1) / v;
  int chunk = 32;
  while (chunk > 4 && (long long)batch * cols * ((len + chunk - 1) / chunk) < 256LL * m2_sm_count()) chunk /= 2;
  return chunk;
}
// Of the gradients: their parameters' sums leave W + 1 numbers a channel and chunk.
static int back_chunk_of(int batch, int len, int dim) {
  int chunk = 256;
  while (chunk > 16 && (long long)batch * dim / 4 * ((len + chunk - 1) / chunk) < 512LL * m2_sm_count()) chunk /= 2;
  return chunk;
}

// channels of a thread: 16 bytes, fewer with many taps and in the gradient (registers); one where a row does not allow it
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
  const int chunk = back_chunk_of(batch, seq_len, dim), chunks = seq_len > 0 ? (seq_len + chunk - 1) / chunk : 1;
  return 4LL * batch * chunks * (taps + 1) * dim;
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
  const int bytes = g.taps <= 4 ? 16 : 8;
  const bool vec = wide(g.x, g.x_sb, g.x_st, g.dim, size, bytes) && wide(a.state_in, 0, 0, g.dim, size, bytes) && wide(g.y, 0, 0, g.dim, size, bytes) &&
                   wide(a.state_out, 0, 0, g.dim, size, bytes);
  a.chunk = chunk_of(g.batch, g.seq_len, g.dim, vec ? bytes / size : 1);
  a.chunks = g.seq_len > 0 ? (g.seq_len + a.chunk - 1) / a.chunk : 1;
  const Grads none = {};
  if (g.dtype == M2_F32) return vec ? by_taps<float, 4, 2, false>(a, none, st) : by_taps<float, 1, 1, false>(a, none, st);
  return vec ? by_taps<__nv_bfloat16, 8, 4, false>(a, none, st) : by_taps<__nv_bfloat16, 1, 1, false>(a, none, st);
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
  a.chunk = back_chunk_of(g.batch, g.seq_len, g.dim);
  a.chunks = g.seq_len > 0 ? (g.seq_len + a.chunk - 1) / a.chunk : 1;
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
