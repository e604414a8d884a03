// Selective state space scan: every channel d has a state of N numbers that fade and are fed by the token itself,
//     s_t = softplus(delta_t + bias)  (or delta_t),     h_t[n] = exp(s_t a[d,n]) h_{t-1}[n] + s_t x_t b_t[n],
//     y_t = (sum_n c_t[n] h_t[n] + skip x_t) silu(z_t),
// its gradients, and one token at a time.  No counterpart in the reference, whose mixer is the long convolution
// (bert/src/mm/monarch_mixer_sequence_mixer.py:100-154).
#include "common.cuh"

namespace m2 {
namespace ss {

constexpr int THREADS = 128;
constexpr int CT = 64;                   // channels of a block: 16 a warp, two a thread
constexpr int QL = 4;                    // lanes that share a channel's states
constexpr int MAX_STATES = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;

__host__ __device__ constexpr int tile_of(int per_lane) { return per_lane == 16 ? 16 : 32; }       // tokens of a tile

struct Rows { const void* p; long long sb, st; int vec; };           // vec: 16-byte pieces
struct Group { const void* p; long long sb, st, sg; };

struct Args {
  int batch, len, dim, states, groups, per_group, tiles, softplus;   // per_group: channels of a group; tiles: blocks that share them
  Rows x, delta, z;
  Group b, c;
  const float *a, *skip, *bias;
  const long long* lengths;
  const float* state_in;
  void* y;
  float *state_out, *saves;
  int segs, seg_tiles;                   // the axis in segments of seg_tiles tiles
  float *seg_state, *seg_steps;          // (batch, segs, dim, NP) and (batch, segs, dim)
  int y_vec;
};

struct Grads {
  Rows dy;
  const float* d_state_out;
  void *dx, *d_delta, *dz;
  int vec;                               // packed outputs in 16-byte pieces
  float *part_b, *part_c;                // (tiles, batch, len, groups, NP)
  float *part_a, *part_skip, *part_bias; // (batch * segs, dim, NP), (batch * segs, dim) twice
  void *db, *dc;
  float *da, *d_skip, *d_bias, *d_state_in;
};

using lp::Piece;
using lp::ex2;

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + ex2(-v * LOG2E)); }
__device__ __forceinline__ float step_of(float v, int softplus) {
  return softplus ? fmaxf(v, 0.f) + log1pf(ex2(-fabsf(v) * LOG2E)) : v;
}

template <typename T> __device__ __forceinline__ uint4 load_piece(const T* p, int valid, bool vec) {
  constexpr int E = Piece<T>::N;
  if (vec && valid >= E) return __ldg(reinterpret_cast<const uint4*>(p));
  float f[E];
#pragma unroll
  for (int j = 0; j < E; ++j) f[j] = j < valid ? lp::load1(p + j) : 0.f;
  return Piece<T>::put(f);
}
template <typename T> __device__ __forceinline__ void store_piece(T* p, const float (&f)[Piece<T>::N], int valid, bool vec) {
  constexpr int E = Piece<T>::N;
  if (vec && valid >= E) { *reinterpret_cast<uint4*>(p) = Piece<T>::put(f); return; }
#pragma unroll
  for (int j = 0; j < E; ++j)
    if (j < valid) st_from_float(p + j, f[j]);
}
template <int E> __device__ __forceinline__ void to_shared(float* p, const float (&f)[E]) {
#pragma unroll
  for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
}
template <int E> __device__ __forceinline__ void from_shared(const float* p, float (&f)[E]) {
#pragma unroll
  for (int j = 0; j < E; j += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + j);
    f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w;
  }
}
__device__ __forceinline__ f32x2 ld2(const float* p) { return *reinterpret_cast<const f32x2*>(p); }
__device__ __forceinline__ f32x2 ex2_pair(f32x2 v) {
  float x, y;
  f2_unpack(v, x, y);
  return f2_pack(ex2(x), ex2(y));
}
template <int S> __device__ __forceinline__ void ld_dup(const float* p, f32x2 (&v)[S]) {      // pairs of equal numbers
#pragma unroll
  for (int i = 0; i < S; i += 2) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p + 2 * i);
    v[i] = u.x; v[i + 1] = u.y;
  }
}
// The sum over the lanes of a channel's states of (v, w), a pair of channels each: lane bit 0 ends with the channel, bit 1 with v or w.
__device__ __forceinline__ float sum_states(f32x2 v, f32x2 w, int lane) {
  float v0, v1, w0, w1;
  f2_unpack(v, v0, v1);
  f2_unpack(w, w0, w1);
  const bool hi = lane & 1, sec = lane & 2;
  const float p = (hi ? v1 : v0) + __shfl_xor_sync(~0u, hi ? v0 : v1, 1);
  const float q = (hi ? w1 : w0) + __shfl_xor_sync(~0u, hi ? w0 : w1, 1);
  return (sec ? q : p) + __shfl_xor_sync(~0u, sec ? p : q, 2);
}

// Where a block works: blocks of one sequence and segment lie side by side, as they read the same b and c
struct Place { int b, seg, g, tile, c0, valid, ch0; };
__device__ __forceinline__ Place place_of(const Args& a) {
  Place p;
  unsigned i = blockIdx.x;
  p.tile = i % a.tiles; i /= a.tiles;
  p.g = i % a.groups; i /= a.groups;
  p.seg = i % a.segs;
  p.b = i / a.segs;
  p.c0 = p.tile * CT;                                                  // first channel within the group
  p.valid = min(CT, a.per_group - p.c0);
  p.ch0 = p.g * a.per_group + p.c0;
  return p;
}
__device__ __forceinline__ int text_length(const Args& a, int b) {
  if (!a.lengths) return a.len;
  const long long n = a.lengths[b];
  return (int)(n < 0 ? 0 : n > a.len ? a.len : n);
}

// b and c of a tile, as pairs of equal numbers in shared memory
template <typename T, int S, int TT> struct Coeffs {
  static constexpr int NP = QL * S, PER = TT * NP / THREADS;
  float v[PER];
  __device__ __forceinline__ void fetch(const Group& r, const Place& p, int t0, int n, int states) {
    const T* base = static_cast<const T*>(r.p) + p.b * r.sb + p.g * r.sg;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = threadIdx.x + i * THREADS, t = t0 + at / NP, s = at % NP;
      v[i] = t < n && s < states ? lp::load1(base + t * r.st + s) : 0.f;
    }
  }
  __device__ __forceinline__ void put(float* sm) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) *reinterpret_cast<float2*>(sm + 2 * (threadIdx.x + i * THREADS)) = make_float2(v[i], v[i]);
  }
};

template <typename T, int TT> struct Pieces {                           // a thread's part of a tile of x, delta, z or a gradient
  static constexpr int E = Piece<T>::N, PPR = CT / E, ROWS = THREADS / PPR, P = TT / ROWS;
  uint4 v[P];
  __device__ __forceinline__ void fetch(const Rows& r, const Place& p, int t0, int n) {
    const int col = threadIdx.x % PPR * E, row = threadIdx.x / PPR;
    const T* base = static_cast<const T*>(r.p) + p.b * r.sb + p.ch0 + col;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int t = t0 + row + i * ROWS;
      v[i] = t < n ? load_piece<T>(base + t * r.st, p.valid - col, r.vec) : make_uint4(0, 0, 0, 0);
    }
  }
};

// A segment's part of y, or (SUMS) its own contribution to the state and the sum of its steps.
template <typename T, int S, bool SUMS>
__global__ void __launch_bounds__(THREADS, S == 4 ? 4 : 2)
scan_kernel(const Args a) {
  constexpr int TT = tile_of(S), NP = QL * S;
  using Px = Pieces<T, TT>;
  constexpr int E = Px::E;
  __shared__ __align__(16) float s_dt[TT][CT], s_dx[TT][CT], s_y[TT][CT], s_b[TT][2 * NP], s_c[TT][2 * NP], s_bias[CT], s_skip[CT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place p = place_of(a);
  pdl_wait();
  const int n = text_length(a, p.b);
  if (tid < CT) {
    s_bias[tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
    s_skip[tid] = a.skip && tid < p.valid ? a.skip[p.ch0 + tid] : 0.f;
  }
  const int cl = warp * 16 + (lane >> 2) * 2, q0 = (lane & 3) * S;      // the thread's two channels and S states
  f32x2 h[S], A[S];
  const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float v[2], w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool real = cl + j < p.valid && q0 + i < a.states;
      const long long ch = p.ch0 + cl + j;
      v[j] = real ? a.a[ch * a.states + q0 + i] * LOG2E : 0.f;
      w[j] = 0.f;
      if (!SUMS && real) {
        if (a.segs > 1) w[j] = a.seg_state[(row_n + cl + j) * NP + q0 + i];
        else if (a.state_in) w[j] = a.state_in[((long long)p.b * a.dim + ch) * a.states + q0 + i];
      }
    }
    A[i] = f2_pack(v[0], v[1]);
    h[i] = f2_pack(w[0], w[1]);
  }
  const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles, last = min(first + a.seg_tiles, total);
  const int used = min(last, (n + TT - 1) / TT);
  const int col = tid % Px::PPR * E, row = tid / Px::PPR;
  T* y = static_cast<T*>(a.y) + (long long)p.b * a.len * a.dim + p.ch0 + col;
  Px x, delta, z;
  Coeffs<T, S, TT> fb, fc;
  auto fetch = [&](int k) {
    x.fetch(a.x, p, k * TT, n);
    delta.fetch(a.delta, p, k * TT, n);
    fb.fetch(a.b, p, k * TT, n, a.states);
    if constexpr (!SUMS) {
      if (a.z.p) z.fetch(a.z, p, k * TT, n);
      fc.fetch(a.c, p, k * TT, n, a.states);
    }
  };
  float steps[2] = {0.f, 0.f};
  if (first < used) fetch(first);
  __syncthreads();
  for (int k = first; k < used; ++k) {
    if (!SUMS && a.saves) {              // the state in front of the tile, for the gradient
      float* to = a.saves + (((long long)p.b * total + k) * a.dim + p.ch0 + cl) * NP + q0;
#pragma unroll
      for (int i = 0; i < S; i += 4) {
        float f[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f2_unpack(h[i + j], f[0][j], f[1][j]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (cl + j < p.valid) *reinterpret_cast<float4*>(to + j * NP + i) = make_float4(f[j][0], f[j][1], f[j][2], f[j][3]);
      }
    }
    Px x_now = x, z_now = z;
    {
      float bias[E];
      from_shared(s_bias + col, bias);
#pragma unroll
      for (int i = 0; i < Px::P; ++i) {
        const int t = row + i * Px::ROWS;
        const bool in = k * TT + t < n;
        float f[E], d[E];
        Piece<T>::get(x.v[i], f);
        Piece<T>::get(delta.v[i], d);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          d[j] = in ? step_of(d[j] + bias[j], a.softplus) : 0.f;
          f[j] *= d[j];
        }
        to_shared(&s_dt[t][col], d);
        to_shared(&s_dx[t][col], f);
      }
    }
    fb.put(&s_b[0][0]);
    if constexpr (!SUMS) fc.put(&s_c[0][0]);
    __syncthreads();
    if (k + 1 < used) fetch(k + 1);
#pragma unroll 2
    for (int t = 0; t < TT; t += 2) {
      f32x2 sum[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x2 dt = ld2(&s_dt[t + u][cl]), dx = ld2(&s_dx[t + u][cl]);
        f32x2 B[S], C[S];
        ld_dup<S>(&s_b[t + u][2 * q0], B);
        if constexpr (!SUMS) ld_dup<S>(&s_c[t + u][2 * q0], C);
        sum[u] = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          h[i] = f2_fma(ex2_pair(f2_mul(dt, A[i])), h[i], f2_mul(dx, B[i]));
          if constexpr (!SUMS) sum[u] = f2_fma(h[i], C[i], sum[u]);
        }
        if constexpr (SUMS) {
          float d0, d1;
          f2_unpack(dt, d0, d1);
          steps[0] += d0;
          steps[1] += d1;
        }
      }
      if constexpr (!SUMS) s_y[t + ((lane >> 1) & 1)][cl + (lane & 1)] = sum_states(sum[0], sum[1], lane);
    }
    __syncthreads();
    if constexpr (!SUMS) {
      float skip[E];
      from_shared(s_skip + col, skip);
#pragma unroll
      for (int i = 0; i < Px::P; ++i) {
        const int t = k * TT + row + i * Px::ROWS;
        if (t >= a.len) continue;
        float f[E], u[E];
        from_shared(&s_y[row + i * Px::ROWS][col], f);
        Piece<T>::get(x_now.v[i], u);
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = fmaf(skip[j], u[j], f[j]);
        if (a.z.p) {
          Piece<T>::get(z_now.v[i], u);
#pragma unroll
          for (int j = 0; j < E; ++j) f[j] *= u[j] * sigmoid(u[j]);
        }
        if (t >= n) {
#pragma unroll
          for (int j = 0; j < E; ++j) f[j] = 0.f;
        }
        store_piece<T>(y + (long long)t * a.dim, f, p.valid - col, a.y_vec);
      }
    }
  }
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      float f[2];
      f2_unpack(h[i], f[0], f[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (cl + j < p.valid) a.seg_state[(row_n + cl + j) * NP + q0 + i] = f[j];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if ((lane & 3) == 0 && cl + j < p.valid) a.seg_steps[row_n + cl + j] = steps[j];
  } else {
    for (int t = max(used, first) * TT + row; t < min(last * TT, a.len); t += Px::ROWS) {      // behind the text
      const float f[E] = {};
      store_piece<T>(y + (long long)t * a.dim, f, p.valid - col, a.y_vec);
    }
    if (a.state_out && p.seg == a.segs - 1) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        float f[2];
        f2_unpack(h[i], f[0], f[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (cl + j < p.valid && q0 + i < a.states) a.state_out[((long long)p.b * a.dim + p.ch0 + cl + j) * a.states + q0 + i] = f[j];
      }
    }
  }
}

// What a segment hands on, from the segments' own sums: forwards the state in front of each (from state_in), backwards the gradient of the state behind each.
__global__ void __launch_bounds__(256)
join_kernel(const float* __restrict__ a, float* __restrict__ seg_state, const float* __restrict__ seg_steps, const float* __restrict__ edge,
            int batch, int segs, int dim, int states, int np, int reverse) {
  pdl_wait();
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= (long long)batch * dim * np) return;
  const int s = (int)(i % np), d = (int)(i / np % dim), b = (int)(i / np / dim);
  const bool real = s < states;
  const float A = real ? a[(long long)d * states + s] * LOG2E : 0.f;
  float h = real && edge ? edge[((long long)b * dim + d) * states + s] : 0.f;
  for (int k = 0; k < segs; ++k) {
    const long long at = ((long long)b * segs + (reverse ? segs - 1 - k : k)) * dim + d;
    const float own = seg_state[at * np + s];
    seg_state[at * np + s] = h;
    h = fmaf(exp2f(A * seg_steps[at]), h, own);
  }
}

// The contribution of a segment's outputs to the gradient of the state in front of it, and the sum of its steps.
template <typename T, int S>
__global__ void __launch_bounds__(THREADS, S == 4 ? 4 : 2)
back_sums_kernel(const Args a, const Grads g) {
  constexpr int TT = tile_of(S), NP = QL * S;
  using Px = Pieces<T, TT>;
  constexpr int E = Px::E;
  __shared__ __align__(16) float s_dt[TT][CT], s_e[TT][CT], s_c[TT][2 * NP], s_bias[CT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place p = place_of(a);
  pdl_wait();
  const int n = text_length(a, p.b);
  if (tid < CT) s_bias[tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
  const int cl = warp * 16 + (lane >> 2) * 2, q0 = (lane & 3) * S;
  f32x2 G[S], A[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      v[j] = cl + j < p.valid && q0 + i < a.states ? a.a[(long long)(p.ch0 + cl + j) * a.states + q0 + i] * LOG2E : 0.f;
    A[i] = f2_pack(v[0], v[1]);
    G[i] = 0;
  }
  const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles;
  const int used = min(min(first + a.seg_tiles, total), (n + TT - 1) / TT);
  const int col = tid % Px::PPR * E, row = tid / Px::PPR;
  Px delta, dy, z;
  Coeffs<T, S, TT> fc;
  float steps[2] = {0.f, 0.f};
  __syncthreads();
  for (int k = used - 1; k >= first; --k) {
    delta.fetch(a.delta, p, k * TT, n);
    dy.fetch(g.dy, p, k * TT, n);
    if (a.z.p) z.fetch(a.z, p, k * TT, n);
    fc.fetch(a.c, p, k * TT, n, a.states);
    float bias[E];
    from_shared(s_bias + col, bias);
#pragma unroll
    for (int i = 0; i < Px::P; ++i) {
      const int t = row + i * Px::ROWS;
      const bool in = k * TT + t < n;
      float d[E], e[E];
      Piece<T>::get(delta.v[i], d);
      Piece<T>::get(dy.v[i], e);
      if (a.z.p) {
        float u[E];
        Piece<T>::get(z.v[i], u);
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] *= u[j] * sigmoid(u[j]);
      }
#pragma unroll
      for (int j = 0; j < E; ++j) d[j] = in ? step_of(d[j] + bias[j], a.softplus) : 0.f;
      to_shared(&s_dt[t][col], d);
      to_shared(&s_e[t][col], e);
    }
    fc.put(&s_c[0][0]);
    __syncthreads();
#pragma unroll 2
    for (int t = TT - 1; t >= 0; --t) {
      const f32x2 dt = ld2(&s_dt[t][cl]), e = ld2(&s_e[t][cl]);
      f32x2 C[S];
      ld_dup<S>(&s_c[t][2 * q0], C);
#pragma unroll
      for (int i = 0; i < S; ++i) G[i] = f2_mul(ex2_pair(f2_mul(dt, A[i])), f2_fma(e, C[i], G[i]));
      float d0, d1;
      f2_unpack(dt, d0, d1);
      steps[0] += d0;
      steps[1] += d1;
    }
    __syncthreads();
  }
  const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float f[2];
    f2_unpack(G[i], f[0], f[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (cl + j < p.valid) a.seg_state[(row_n + cl + j) * NP + q0 + i] = f[j];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if ((lane & 3) == 0 && cl + j < p.valid) a.seg_steps[row_n + cl + j] = steps[j];
}

template <int TT, int NP> struct BackShared {
  float dt[TT][CT], dx[TT][CT], e[TT][CT], y[TT][CT], q[TT][CT], gb[TT][CT];
  float b[TT][2 * NP], c[TT][2 * NP];
  float db[4][TT][NP], dc[4][TT][NP];    // of each warp's channels
  float bias[CT], skip[CT];
};

// Sums over a warp's channels of S values in each of two steps (pairs of channels), into out[state] of the steps.
template <int S> __device__ __forceinline__ void sum_channels(const f32x2 (&v)[S], const f32x2 (&w)[S], int lane, float* to_v, float* to_w) {
  float f[2 * S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float x, y;
    f2_unpack(v[i], x, y);
    f[i] = x + y;
    f2_unpack(w[i], x, y);
    f[S + i] = x + y;
  }
  constexpr int H = S;                   // of 2 S values half stay, a quarter, an eighth
  const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
#pragma unroll
  for (int i = 0; i < H; ++i) f[i] = (b4 ? f[H + i] : f[i]) + __shfl_xor_sync(~0u, b4 ? f[i] : f[H + i], 16);
#pragma unroll
  for (int i = 0; i < H / 2; ++i) f[i] = (b3 ? f[H / 2 + i] : f[i]) + __shfl_xor_sync(~0u, b3 ? f[i] : f[H / 2 + i], 8);
#pragma unroll
  for (int i = 0; i < H / 4; ++i) f[i] = (b2 ? f[H / 4 + i] : f[i]) + __shfl_xor_sync(~0u, b2 ? f[i] : f[H / 4 + i], 4);
  float* to = (b4 ? to_w : to_v) + (lane & 3) * S + (b3 ? S / 2 : 0) + (b2 ? S / 4 : 0);
#pragma unroll
  for (int i = 0; i < H / 4; ++i) to[i] = f[i];
}

// Gradients, a tile at a time from the last to the first.  With v_t = h_t c_t, e_t the gradient of sum c h, g_t that of h_t:
//   forwards   h_t again from the saved state in front of the tile: y, dc_t = sum_d h_t e_t, and q_t = sum_n a v_t
//   backwards  g_t = c_t e_t + exp(s a)_{t+1} g_{t+1}: gb_t = sum_n g_t b_t, db_t = sum_d g_t s x, and p_t = sum_n a g_t b_t
// The gradient of s_t needs w_t = g_t exp(s_t a) h_{t-1} for every state, so h and g at one time.  But w_{t+1} = w_t + g_t b_t s x - v_t e_t, so that inside
// a tile sum_n a w_t is a sum of scalars of a channel from its end, where h and g are both at hand:
//   sum_n a w_t = sum_n a g h (end) + sum_{r >= t} (q_r e_r - p_r s x),       da = sum_t s_t w_t = g h S + sum_r S_r (v_r e_r - g_r b_r s x)
// with S_r the sum of the tile's steps up to r.
template <typename T, int S>
__global__ void __launch_bounds__(THREADS, S == 4 ? 3 : S == 8 ? 2 : 1)
back_kernel(const Args a, const Grads g) {
  constexpr int TT = tile_of(S), NP = QL * S;
  using Px = Pieces<T, TT>;
  constexpr int E = Px::E;
  extern __shared__ __align__(16) unsigned char raw[];
  BackShared<TT, NP>& sh = *reinterpret_cast<BackShared<TT, NP>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place p = place_of(a);
  pdl_wait();
  const int n = text_length(a, p.b);
  if (tid < CT) {
    sh.bias[tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
    sh.skip[tid] = a.skip && tid < p.valid ? a.skip[p.ch0 + tid] : 0.f;
  }
  const int cl = warp * 16 + (lane >> 2) * 2, q0 = (lane & 3) * S;
  const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
  f32x2 G[S], A[S], dA[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float v[2], w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool real = cl + j < p.valid && q0 + i < a.states;
      const long long ch = p.ch0 + cl + j;
      v[j] = real ? a.a[ch * a.states + q0 + i] * LOG2E : 0.f;
      w[j] = 0.f;
      if (real && a.segs > 1) w[j] = a.seg_state[(row_n + cl + j) * NP + q0 + i];
      else if (real && g.d_state_out) w[j] = g.d_state_out[((long long)p.b * a.dim + ch) * a.states + q0 + i];
    }
    A[i] = f2_pack(v[0], v[1]);
    G[i] = f2_pack(w[0], w[1]);
    dA[i] = 0;
  }
  const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles, last = min(first + a.seg_tiles, total);
  const int used = min(last, (n + TT - 1) / TT);
  const int col = tid % Px::PPR * E, row = tid / Px::PPR;
  const long long out0 = (long long)p.b * a.len * a.dim + p.ch0 + col;
  T *dx = static_cast<T*>(g.dx) + out0, *dd = static_cast<T*>(g.d_delta) + out0, *dz = static_cast<T*>(g.dz) + out0;
  float d_skip[E], d_bias[E];
#pragma unroll
  for (int j = 0; j < E; ++j) d_skip[j] = d_bias[j] = 0.f;
  for (int t = max(used, first) * TT + row; t < min(last * TT, a.len); t += Px::ROWS) {       // behind the text
    const float f[E] = {};
    store_piece<T>(dx + (long long)t * a.dim, f, p.valid - col, g.vec);
    store_piece<T>(dd + (long long)t * a.dim, f, p.valid - col, g.vec);
    if (g.dz) store_piece<T>(dz + (long long)t * a.dim, f, p.valid - col, g.vec);
  }
  Px x, delta, z, dy;
  Coeffs<T, S, TT> fb, fc;
  auto fetch = [&](int k) {
    x.fetch(a.x, p, k * TT, n);
    delta.fetch(a.delta, p, k * TT, n);
    dy.fetch(g.dy, p, k * TT, n);
    if (a.z.p) z.fetch(a.z, p, k * TT, n);
    fb.fetch(a.b, p, k * TT, n, a.states);
    fc.fetch(a.c, p, k * TT, n, a.states);
  };
  __syncthreads();
  for (int k = used - 1; k >= first; --k) {
    fetch(k);
    f32x2 h[S];
    {
      const float* from = a.saves + (((long long)p.b * total + k) * a.dim + p.ch0 + cl) * NP + q0;
#pragma unroll
      for (int i = 0; i < S; i += 4) {
        float4 f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) f[j] = cl + j < p.valid ? *reinterpret_cast<const float4*>(from + j * NP + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        h[i] = f2_pack(f[0].x, f[1].x); h[i + 1] = f2_pack(f[0].y, f[1].y); h[i + 2] = f2_pack(f[0].z, f[1].z); h[i + 3] = f2_pack(f[0].w, f[1].w);
      }
    }
    {
      float bias[E];
      from_shared(sh.bias + col, bias);
#pragma unroll
      for (int i = 0; i < Px::P; ++i) {
        const int t = row + i * Px::ROWS;
        const bool in = k * TT + t < n;
        float f[E], d[E], e[E];
        Piece<T>::get(x.v[i], f);
        Piece<T>::get(delta.v[i], d);
        Piece<T>::get(dy.v[i], e);
        if (a.z.p) {
          float u[E];
          Piece<T>::get(z.v[i], u);
#pragma unroll
          for (int j = 0; j < E; ++j) e[j] *= u[j] * sigmoid(u[j]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
          d[j] = in ? step_of(d[j] + bias[j], a.softplus) : 0.f;
          f[j] *= d[j];
        }
        to_shared(&sh.dt[t][col], d);
        to_shared(&sh.dx[t][col], f);
        to_shared(&sh.e[t][col], e);
      }
    }
    fb.put(&sh.b[0][0]);
    fc.put(&sh.c[0][0]);
    __syncthreads();
    const int own_row = (lane >> 1) & 1, own_ch = cl + (lane & 1);
    f32x2 cum = 0;
    for (int t = 0; t < TT; t += 2) {
      f32x2 U[2][S];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x2 dt = ld2(&sh.dt[t + u][cl]), xs = ld2(&sh.dx[t + u][cl]), e = ld2(&sh.e[t + u][cl]);
        f32x2 B[S], C[S];
        ld_dup<S>(&sh.b[t + u][2 * q0], B);
        ld_dup<S>(&sh.c[t + u][2 * q0], C);
        cum = f2_add(cum, dt);
        const f32x2 ec = f2_mul(e, cum);
        f32x2 y = 0, q = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          h[i] = f2_fma(ex2_pair(f2_mul(dt, A[i])), h[i], f2_mul(xs, B[i]));
          U[u][i] = f2_mul(h[i], e);
          const f32x2 v = f2_mul(h[i], C[i]);
          y = f2_add(y, v);
          q = f2_fma(v, A[i], q);
          dA[i] = f2_fma(v, ec, dA[i]);
        }
        const float r = sum_states(y, q, lane);
        (own_row ? sh.q : sh.y)[t + u][own_ch] = r;
      }
      sum_channels<S>(U[0], U[1], lane, sh.dc[warp][t], sh.dc[warp][t + 1]);
    }
    f32x2 end = 0;                       // sum a g h behind the tile's last token
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const f32x2 w = f2_mul(G[i], h[i]);
      end = f2_fma(w, A[i], end);
      dA[i] = f2_fma(w, cum, dA[i]);
    }
    const float w_end = sum_states(end, 0, lane);          // lanes with bit 1 clear
    for (int t = TT - 2; t >= 0; t -= 2) {
      f32x2 U[2][S];
#pragma unroll
      for (int u = 1; u >= 0; --u) {
        const f32x2 dt = ld2(&sh.dt[t + u][cl]), xs = ld2(&sh.dx[t + u][cl]), e = ld2(&sh.e[t + u][cl]);
        f32x2 B[S], C[S];
        ld_dup<S>(&sh.b[t + u][2 * q0], B);
        ld_dup<S>(&sh.c[t + u][2 * q0], C);
        const f32x2 xc = f2_mul(f2_mul(xs, cum), f2_splat(-1.f));
        cum = f2_fma(dt, f2_splat(-1.f), cum);
        f32x2 gb = 0, q = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
          G[i] = f2_fma(e, C[i], G[i]);
          U[u][i] = f2_mul(G[i], xs);
          const f32x2 v = f2_mul(G[i], B[i]);
          gb = f2_add(gb, v);
          q = f2_fma(v, A[i], q);
          dA[i] = f2_fma(v, xc, dA[i]);
          G[i] = f2_mul(ex2_pair(f2_mul(dt, A[i])), G[i]);
        }
        const float r = sum_states(gb, q, lane);
        if (own_row) sh.q[t + u][own_ch] = sh.q[t + u][own_ch] * sh.e[t + u][own_ch] - r * sh.dx[t + u][own_ch];
        else sh.gb[t + u][own_ch] = r;
      }
      sum_channels<S>(U[0], U[1], lane, sh.db[warp][t], sh.db[warp][t + 1]);
    }
    __syncwarp();
    if (own_row == 0 && (lane & 3) == (lane & 1)) {        // a channel's sums from the tile's end
      float w = w_end;
      for (int t = TT - 1; t >= 0; --t) {
        w += sh.q[t][own_ch];
        sh.q[t][own_ch] = w * LN2;
      }
    }
    __syncthreads();
    for (int i = tid; i < TT * NP; i += THREADS) {
      const int t = k * TT + i / NP;
      if (t < n) {
        const long long at = ((((long long)p.tile * a.batch + p.b) * a.len + t) * a.groups + p.g) * NP + i % NP;
        g.part_b[at] = (&sh.db[0][0][0])[i] + (&sh.db[1][0][0])[i] + (&sh.db[2][0][0])[i] + (&sh.db[3][0][0])[i];
        g.part_c[at] = (&sh.dc[0][0][0])[i] + (&sh.dc[1][0][0])[i] + (&sh.dc[2][0][0])[i] + (&sh.dc[3][0][0])[i];
      }
    }
    {
      float bias[E], skip[E];
      from_shared(sh.bias + col, bias);
      from_shared(sh.skip + col, skip);
#pragma unroll
      for (int i = 0; i < Px::P; ++i) {
        const int r = row + i * Px::ROWS, t = k * TT + r;
        if (t >= a.len) continue;
        const bool in = t < n;
        float u[E], e[E], gb[E], f[E], o[E];
        Piece<T>::get(x.v[i], u);
        from_shared(&sh.e[r][col], e);
        if (g.dz) {
          float zz[E], dout[E];
          Piece<T>::get(z.v[i], zz);
          Piece<T>::get(dy.v[i], dout);
          from_shared(&sh.y[r][col], f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const float s = sigmoid(zz[j]), yy = fmaf(skip[j], u[j], f[j]);
            o[j] = in ? dout[j] * yy * s * (1.f + zz[j] * (1.f - s)) : 0.f;
          }
          store_piece<T>(dz + (long long)t * a.dim, o, p.valid - col, g.vec);
        }
        from_shared(&sh.gb[r][col], gb);
        from_shared(&sh.dt[r][col], f);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          o[j] = in ? fmaf(f[j], gb[j], skip[j] * e[j]) : 0.f;
          d_skip[j] = fmaf(e[j], u[j], d_skip[j]);
        }
        store_piece<T>(dx + (long long)t * a.dim, o, p.valid - col, g.vec);
        from_shared(&sh.q[r][col], f);
        float d[E];
        Piece<T>::get(delta.v[i], d);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          o[j] = fmaf(gb[j], u[j], f[j]);
          if (a.softplus) o[j] *= sigmoid(d[j] + bias[j]);
          if (!in) o[j] = 0.f;
          d_bias[j] += o[j];
        }
        store_piece<T>(dd + (long long)t * a.dim, o, p.valid - col, g.vec);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    float f[2], w[2];
    f2_unpack(dA[i], f[0], f[1]);
    f2_unpack(G[i], w[0], w[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (cl + j < p.valid) {
        g.part_a[(row_n + cl + j) * NP + q0 + i] = f[j];
        if (g.d_state_in && p.seg == 0 && q0 + i < a.states) g.d_state_in[((long long)p.b * a.dim + p.ch0 + cl + j) * a.states + q0 + i] = w[j];
      }
    }
  }
  float* sums = &sh.dt[0][0];            // [2][ROWS][CT]
  static_assert(2 * Px::ROWS <= 6 * TT, "sums of the parameters");
  to_shared(sums + row * CT + col, d_skip);
  to_shared(sums + (Px::ROWS + row) * CT + col, d_bias);
  __syncthreads();
  const int c = tid % CT, which = tid / CT;
  float v = 0.f;
  for (int r = 0; r < Px::ROWS; ++r) v += sums[(which * Px::ROWS + r) * CT + c];
  if (c < p.valid) (which ? g.part_bias : g.part_skip)[row_n + c] = v;
}

// The blocks' parts of the gradients of b, c and of the parameters, added in one order.
template <typename T>
__global__ void __launch_bounds__(256)
finish_kernel(const Args a, const Grads g, int np, unsigned bc_blocks) {
  pdl_wait();
  if (blockIdx.x < bc_blocks) {
    const long long rows = (long long)a.batch * a.len * a.groups, i = blockIdx.x * 256LL + threadIdx.x;
    if (i >= rows * a.states) return;
    const long long r = i / a.states;
    const int s = (int)(i - r * a.states);
    const int t = (int)(r / a.groups % a.len), b = (int)(r / a.groups / a.len);
    float vb = 0.f, vc = 0.f;
    if (t < text_length(a, b)) {
      for (int k = 0; k < a.tiles; ++k) {
        vb += g.part_b[(k * rows + r) * np + s];
        vc += g.part_c[(k * rows + r) * np + s];
      }
    }
    st_from_float(static_cast<T*>(g.db) + i, vb);
    st_from_float(static_cast<T*>(g.dc) + i, vc);
    return;
  }
  const long long i = (blockIdx.x - bc_blocks) * 256LL + threadIdx.x, d = i / (a.states + 2);
  const int s = (int)(i - d * (a.states + 2)), parts = a.batch * a.segs;
  if (d >= a.dim) return;
  float v = 0.f;
  if (s < a.states) {
    if (!g.da) return;
    for (int k = 0; k < parts; ++k) v += g.part_a[((long long)k * a.dim + d) * np + s];
    g.da[d * a.states + s] = v;
  } else {
    const float* from = s == a.states ? g.part_skip : g.part_bias;
    float* to = s == a.states ? g.d_skip : g.d_bias;
    if (!to) return;
    for (int k = 0; k < parts; ++k) v += from[(long long)k * a.dim + d];
    to[d] = v;
  }
}

// One token: four threads a channel, a piece of its states each.
struct StepArgs {
  int batch, dim, states, groups, per_group, softplus;
  const void *x, *delta, *z, *b, *c;
  long long x_sb, d_sb, z_sb, b_sb, b_sg, c_sb, c_sg;
  const float *a, *skip, *bias;
  float* state; long long s_b;
  void* y;
};

template <typename T>
__global__ void __launch_bounds__(256)
step_kernel(const StepArgs a) {
  pdl_wait();
  const long long i = blockIdx.x * 64LL + threadIdx.x / 4;
  const int part = threadIdx.x % 4;
  const bool live = i < (long long)a.batch * a.dim;
  const int b = live ? (int)(i / a.dim) : 0, d = live ? (int)(i % a.dim) : 0, grp = d / a.per_group;
  const float x = lp::load1(static_cast<const T*>(a.x) + b * a.x_sb + d);
  const float dt = step_of(lp::load1(static_cast<const T*>(a.delta) + b * a.d_sb + d) + (a.bias ? a.bias[d] : 0.f), a.softplus);
  const float dx = dt * x;
  const T* B = static_cast<const T*>(a.b) + b * a.b_sb + grp * a.b_sg;
  const T* C = static_cast<const T*>(a.c) + b * a.c_sb + grp * a.c_sg;
  float* h = a.state + b * a.s_b + (long long)d * a.states;
  const float* A = a.a + (long long)d * a.states;
  float y = 0.f;
  auto one = [&](float hh, float aa, int s) {
    hh = fmaf(ex2(dt * (aa * LOG2E)), hh, dx * lp::load1(B + s));
    y = fmaf(hh, lp::load1(C + s), y);
    return hh;
  };
  if (live) {
    if (a.states % 4 == 0 && ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(A)) & 15) == 0) {
      for (int s = part * 4; s < a.states; s += 16) {
        float4 v = *reinterpret_cast<float4*>(h + s);
        const float4 w = __ldg(reinterpret_cast<const float4*>(A + s));
        v.x = one(v.x, w.x, s); v.y = one(v.y, w.y, s + 1); v.z = one(v.z, w.z, s + 2); v.w = one(v.w, w.w, s + 3);
        *reinterpret_cast<float4*>(h + s) = v;
      }
    } else {
      for (int s = part; s < a.states; s += 4) h[s] = one(h[s], A[s], s);
    }
  }
  y += __shfl_xor_sync(~0u, y, 1);
  y += __shfl_xor_sync(~0u, y, 2);
  if (!live || part) return;
  if (a.skip) y = fmaf(a.skip[d], x, y);
  if (a.z) {
    const float z = lp::load1(static_cast<const T*>(a.z) + b * a.z_sb + d);
    y *= z * sigmoid(z);
  }
  st_from_float(static_cast<T*>(a.y) + i, y);
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int per_lane(int states) { return states <= 16 ? 4 : states <= 32 ? 8 : 16; }

struct Plan { int per_lane, np, tile, total, tiles, per_group, segs, seg_tiles; };
// The axis is cut into segments where sequences and channels alone leave SMs without two blocks: what a segment adds to the state is then computed
// first, at the price of a second exp for each token, channel and state.
static Plan plan_of(int batch, int len, int dim, int states, int groups) {
  Plan p;
  p.per_lane = per_lane(states);
  p.np = QL * p.per_lane;
  p.tile = tile_of(p.per_lane);
  p.total = (len + p.tile - 1) / p.tile;
  p.per_group = dim / groups;
  p.tiles = (p.per_group + CT - 1) / CT;
  const long long blocks = (long long)batch * groups * p.tiles, want = 4LL * m2_sm_count();
  p.segs = 1;
  if (blocks < m2_sm_count() && p.total >= 8) {
    long long s = want / (blocks > 0 ? blocks : 1);
    if (s > p.total / 2) s = p.total / 2;
    p.segs = s > 1 ? (int)s : 1;
  }
  p.seg_tiles = p.total > 0 ? (p.total + p.segs - 1) / p.segs : 1;
  p.segs = p.total > 0 ? (p.total + p.seg_tiles - 1) / p.seg_tiles : 1;
  return p;
}

static long long seg_floats(const Plan& p, int batch, int dim) { return p.segs > 1 ? (long long)batch * p.segs * dim * (p.np + 1) : 0; }
static long long saves_floats(const Plan& p, int batch, int dim) { return (long long)batch * p.total * dim * p.np; }
static long long grad_floats(const Plan& p, int batch, int len, int dim, int groups) {
  return seg_floats(p, batch, dim) + 2LL * p.tiles * batch * len * groups * p.np + (long long)batch * p.segs * dim * (p.np + 2);
}

template <typename T, int S> static int forward(const Args& a, const Plan& p, cudaStream_t st) {
  const long long blocks = (long long)a.batch * p.segs * a.groups * p.tiles, size = (long long)a.batch * a.len * a.dim;
  if (p.segs > 1) {
    if (int rc = m2_launch("m2_selective_scan_fwd", size, scan_kernel<T, S, true>, dim3((unsigned)blocks), THREADS, 0, st, a)) return rc;
    const long long n = (long long)a.batch * a.dim * p.np;
    if (int rc = m2_launch("m2_selective_scan_fwd", size, join_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a.a, a.seg_state, a.seg_steps,
                           a.state_in, a.batch, p.segs, a.dim, a.states, p.np, 0)) return rc;
  }
  return m2_launch("m2_selective_scan_fwd", size, scan_kernel<T, S, false>, dim3((unsigned)blocks), THREADS, 0, st, a);
}

template <typename T, int S> static int backward(const Args& a, const Grads& g, const Plan& p, cudaStream_t st) {
  const long long blocks = (long long)a.batch * p.segs * a.groups * p.tiles, size = (long long)a.batch * a.len * a.dim;
  if (p.segs > 1) {
    if (int rc = m2_launch("m2_selective_scan_bwd", size, back_sums_kernel<T, S>, dim3((unsigned)blocks), THREADS, 0, st, a, g)) return rc;
    const long long n = (long long)a.batch * a.dim * p.np;
    if (int rc = m2_launch("m2_selective_scan_bwd", size, join_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a.a, a.seg_state, a.seg_steps,
                           g.d_state_out, a.batch, p.segs, a.dim, a.states, p.np, 1)) return rc;
  }
  constexpr size_t smem = sizeof(BackShared<tile_of(S), QL * S>);
  M2_SMEM_ONCE((back_kernel<T, S>), smem);
  if (int rc = m2_launch("m2_selective_scan_bwd", size, back_kernel<T, S>, dim3((unsigned)blocks), THREADS, smem, st, a, g)) return rc;
  const long long bc = ((long long)a.batch * a.len * a.groups * a.states + 255) / 256, par = ((long long)a.dim * (a.states + 2) + 255) / 256;
  return m2_launch("m2_selective_scan_bwd", size, finish_kernel<T>, dim3((unsigned)(bc + par)), 256, 0, st, a, g, p.np, (unsigned)bc);
}

static bool in_pieces(const void* p, long long sb, long long st, int per_group, int size) {
  return m2_aligned(p, 16) && sb * size % 16 == 0 && st * size % 16 == 0 && (long long)per_group * size % 16 == 0;
}

static int check(const char* name, const m2_selective_scan_args& g, Args& a, Plan& p) {
  M2_REQUIRE(g.batch >= 0 && g.seq_len >= 0 && g.dim >= 1 && g.states >= 1 && g.groups >= 1 && g.dim % g.groups == 0, M2_ERR_ARG,
             "%s: %d sequences of %d tokens, %d channels, %d states, %d groups", name, g.batch, g.seq_len, g.dim, g.states, g.groups);
  M2_REQUIRE(g.states <= MAX_STATES, M2_ERR_UNSUPPORTED, "%s: %d states (at most %d)", name, g.states, MAX_STATES);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: tensors are float32 or bf16", name);
  M2_REQUIRE(g.seq_len <= 1 << 28 && g.dim <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: %d tokens of %d channels", name, g.seq_len, g.dim);
  p = plan_of(g.batch, g.seq_len, g.dim, g.states, g.groups);
  M2_REQUIRE((long long)g.batch * p.segs * g.groups * p.tiles <= 0x7fffffffLL && ((long long)g.batch * g.dim * p.np + 255) / 256 <= 0x7fffffffLL &&
                 ((long long)g.batch * g.seq_len * g.groups * g.states + 255) / 256 <= 0x3fffffffLL,
             M2_ERR_UNSUPPORTED, "%s: %d sequences of %d channels are more than the grid takes", name, g.batch, g.dim);
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.a && (g.seq_len == 0 || (g.x && g.delta && g.b && g.c)), M2_ERR_ARG, "%s: x, delta, a, b or c is NULL", name);
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.x, size) && m2_aligned(g.delta, size) && m2_aligned(g.gate, size) && m2_aligned(g.b, size) && m2_aligned(g.c, size) &&
                 m2_aligned(g.lengths, 8) && m2_aligned(g.saves, 16) && m2_aligned(g.workspace, 16),
             M2_ERR_ALIGN, "%s: a tensor is not aligned to its type, or saves or the workspace not to 16 bytes", name);
  auto rows = [&](const void* q, long long sb, long long st) { return Rows{q, sb, st, in_pieces(q, sb, st, p.per_group, size)}; };
  a = Args{};
  a.batch = g.batch; a.len = g.seq_len; a.dim = g.dim; a.states = g.states; a.groups = g.groups; a.per_group = p.per_group; a.tiles = p.tiles;
  a.softplus = g.softplus;
  a.x = rows(g.x, g.x_sb, g.x_st); a.delta = rows(g.delta, g.d_sb, g.d_st); a.z = rows(g.gate, g.z_sb, g.z_st);
  a.b = {g.b, g.b_sb, g.b_st, g.b_sg}; a.c = {g.c, g.c_sb, g.c_st, g.c_sg};
  a.a = g.a; a.skip = g.skip; a.bias = g.delta_bias; a.lengths = (const long long*)g.lengths; a.state_in = g.state_in;
  a.y = g.y; a.state_out = g.state_out; a.saves = g.saves; a.segs = p.segs; a.seg_tiles = p.seg_tiles;
  a.seg_state = g.workspace; a.seg_steps = g.workspace ? g.workspace + (long long)g.batch * p.segs * g.dim * p.np : nullptr;
  a.y_vec = in_pieces(g.y, 0, g.dim, p.per_group, size) && (long long)g.seq_len * g.dim * size % 16 == 0;
  return M2_OK;
}

}  // namespace ss
}  // namespace m2

extern "C" long long m2_selective_scan_saves(int batch, int seq_len, int dim, int states, int groups) {
  using namespace m2::ss;
  if (batch <= 0 || seq_len <= 0 || dim <= 0 || states <= 0 || states > MAX_STATES || groups <= 0 || dim % groups) return 0;
  return 4 * saves_floats(plan_of(batch, seq_len, dim, states, groups), batch, dim);
}

extern "C" long long m2_selective_scan_workspace(int batch, int seq_len, int dim, int states, int groups, int backward) {
  using namespace m2::ss;
  if (batch <= 0 || seq_len <= 0 || dim <= 0 || states <= 0 || states > MAX_STATES || groups <= 0 || dim % groups) return 0;
  const Plan p = plan_of(batch, seq_len, dim, states, groups);
  return 4 * (backward ? grad_floats(p, batch, seq_len, dim, groups) : seg_floats(p, batch, dim));
}

#define M2_SS_DISPATCH(fn, ...)                                                                                           \
  (g.dtype == M2_F32 ? (p.per_lane == 4 ? fn<float, 4>(__VA_ARGS__) : p.per_lane == 8 ? fn<float, 8>(__VA_ARGS__) : fn<float, 16>(__VA_ARGS__)) \
                     : (p.per_lane == 4 ? fn<__nv_bfloat16, 4>(__VA_ARGS__) : p.per_lane == 8 ? fn<__nv_bfloat16, 8>(__VA_ARGS__)               \
                                                                                     : fn<__nv_bfloat16, 16>(__VA_ARGS__)))

extern "C" int m2_selective_scan_fwd(const m2_selective_scan_args* args, void* stream) {
  using namespace m2::ss;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_selective_scan_fwd: args is NULL");
  const m2_selective_scan_args& g = *args;
  Args a;
  Plan p;
  if (int rc = check("m2_selective_scan_fwd", g, a, p)) return rc;
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.y || g.seq_len == 0, M2_ERR_ARG, "m2_selective_scan_fwd: y is NULL");
  const long long need = 4 * seg_floats(p, g.batch, g.dim), keep = 4 * saves_floats(p, g.batch, g.dim);
  M2_REQUIRE(need == 0 || (g.workspace && g.workspace_bytes >= need), M2_ERR_ARG, "m2_selective_scan_fwd: the workspace has %lld bytes of %lld",
             g.workspace ? g.workspace_bytes : 0, need);
  M2_REQUIRE(!g.saves || g.saves_bytes >= keep, M2_ERR_ARG, "m2_selective_scan_fwd: saves has %lld bytes of %lld", g.saves_bytes, keep);
  const cudaStream_t st = (cudaStream_t)stream;
  return M2_SS_DISPATCH(forward, a, p, st);
}

extern "C" int m2_selective_scan_bwd(const m2_selective_scan_args* args, const m2_selective_scan_grads* grads, void* stream) {
  using namespace m2::ss;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_selective_scan_bwd: args or grads is NULL");
  const m2_selective_scan_args& g = *args;
  const m2_selective_scan_grads& o = *grads;
  Args a;
  Plan p;
  if (int rc = check("m2_selective_scan_bwd", g, a, p)) return rc;
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.seq_len == 0 || (o.d_y && o.d_x && o.d_delta && o.d_b && o.d_c && (!g.gate == !o.d_gate)), M2_ERR_ARG,
             "m2_selective_scan_bwd: d_y or a gradient is NULL");
  const long long need = 4 * grad_floats(p, g.batch, g.seq_len, g.dim, g.groups), keep = 4 * saves_floats(p, g.batch, g.dim);
  M2_REQUIRE(g.workspace && g.workspace_bytes >= need, M2_ERR_ARG, "m2_selective_scan_bwd: the workspace has %lld bytes of %lld",
             g.workspace ? g.workspace_bytes : 0, need);
  M2_REQUIRE(keep == 0 || (g.saves && g.saves_bytes >= keep), M2_ERR_ARG, "m2_selective_scan_bwd: saves has %lld bytes of %lld",
             g.saves ? g.saves_bytes : 0, keep);
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(o.d_y, size) && m2_aligned(o.d_x, size) && m2_aligned(o.d_delta, size) && m2_aligned(o.d_gate, size) && m2_aligned(o.d_b, size) &&
                 m2_aligned(o.d_c, size), M2_ERR_ALIGN, "m2_selective_scan_bwd: a gradient is not aligned to its type");
  Grads r = {};
  r.dy = {o.d_y, o.y_sb, o.y_st, in_pieces(o.d_y, o.y_sb, o.y_st, p.per_group, size)};
  r.d_state_out = o.d_state_out;
  r.dx = o.d_x; r.d_delta = o.d_delta; r.dz = o.d_gate;
  r.vec = m2_aligned(o.d_x, 16) && m2_aligned(o.d_delta, 16) && m2_aligned(o.d_gate, 16) && (long long)p.per_group * size % 16 == 0;
  float* w = g.workspace + seg_floats(p, g.batch, g.dim);
  const long long bc = (long long)p.tiles * g.batch * g.seq_len * g.groups * p.np, parts = (long long)g.batch * p.segs * g.dim;
  r.part_b = w; r.part_c = w + bc; r.part_a = w + 2 * bc; r.part_skip = r.part_a + parts * p.np; r.part_bias = r.part_skip + parts;
  r.db = o.d_b; r.dc = o.d_c; r.da = o.d_a; r.d_skip = o.d_skip; r.d_bias = o.d_delta_bias; r.d_state_in = o.d_state_in;
  const cudaStream_t st = (cudaStream_t)stream;
  return M2_SS_DISPATCH(backward, a, r, p, st);
}

extern "C" int m2_selective_scan_step(const m2_selective_scan_step_args* args, void* stream) {
  using namespace m2::ss;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_selective_scan_step: args is NULL");
  const m2_selective_scan_step_args& g = *args;
  M2_REQUIRE(g.batch >= 0 && g.dim >= 1 && g.states >= 1 && g.groups >= 1 && g.dim % g.groups == 0, M2_ERR_ARG,
             "m2_selective_scan_step: %d sequences, %d channels, %d states, %d groups", g.batch, g.dim, g.states, g.groups);
  M2_REQUIRE(g.states <= MAX_STATES, M2_ERR_UNSUPPORTED, "m2_selective_scan_step: %d states (at most %d)", g.states, MAX_STATES);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "m2_selective_scan_step: tensors are float32 or bf16");
  const long long blocks = ((long long)g.batch * g.dim + 63) / 64;
  M2_REQUIRE(blocks <= 0x7fffffffLL && g.dim <= 1 << 24, M2_ERR_UNSUPPORTED, "m2_selective_scan_step: %d sequences of %d channels are more than the grid takes", g.batch, g.dim);
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.x && g.delta && g.a && g.b && g.c && g.state && g.y, M2_ERR_ARG, "m2_selective_scan_step: a tensor is NULL");
  M2_REQUIRE(g.batch == 1 || g.s_b >= (long long)g.dim * g.states, M2_ERR_ARG, "m2_selective_scan_step: states overlap");
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.x, size) && m2_aligned(g.delta, size) && m2_aligned(g.gate, size) && m2_aligned(g.b, size) && m2_aligned(g.c, size) &&
                 m2_aligned(g.y, size) && m2_aligned(g.state, 4), M2_ERR_ALIGN, "m2_selective_scan_step: a tensor is not aligned to its type");
  const StepArgs a = {g.batch, g.dim, g.states, g.groups, g.dim / g.groups, g.softplus, g.x, g.delta, g.gate, g.b, g.c,
                      g.x_sb, g.d_sb, g.z_sb, g.b_sb, g.b_sg, g.c_sb, g.c_sg, g.a, g.skip, g.delta_bias, g.state, g.s_b, g.y};
  const long long elements = (long long)g.batch * g.dim * g.states;
  const cudaStream_t st = (cudaStream_t)stream;
  return g.dtype == M2_F32 ? m2_launch("m2_selective_scan_step", elements, step_kernel<float>, dim3((unsigned)blocks), 256, 0, st, a)
                           : m2_launch("m2_selective_scan_step", elements, step_kernel<__nv_bfloat16>, dim3((unsigned)blocks), 256, 0, st, a);
}
