// Norms after and before a block, fused with the block's gate and the residual's scale:
//     r = a x + g N1(y),      h = N2(r),      N(v) = (v - mean) rstd w + b   (LayerNorm)   or   v rstd w + b   (RMS norm)
// and its gradient.  Generalises the post-norm of m2_add_layernorm_fwd (bert/src/bert_layers.py:506, which is a = g = 1, no N1,
// and h alone) to pre-, post- and sandwich-norm blocks.
//
// With u = dr + N2'(dh):  dx = a u,  da = sum x u,  dn = g u,  dg = u N1(y),  dy = N1'(dn), and for a norm with normalised values v^
//     N'(d) = rstd (d w - mean(d w) - v^ mean(d w v^)),      dw = sum d v^,      db = sum d      (no mean(d w) for the RMS norm).
//
// Bound: every tensor crosses HBM once in each direction.  Forward: a warp has a row (forward_warp_kernel), 131072 x 1536 with a
// float32 stream and a gate per token 500 to 550 us, 5.1 to 5.6 TB/s or 0.78 to 0.86 of the measured copy rate.  Gradient, and rows of
// other lengths: a block of ceil(n / 256) warps walks over rows and a thread owns the same 8 columns of each: weights stay in its
// registers, and so do the column sums of the gradient, which meet in a second, small launch that adds the blocks' sums in a fixed
// order (no atomics: two runs give the same bits); 32768 x 768 144 to 150 us, 3.1 TB/s: 168 registers a thread, 48 of them the six
// column sums whether or not they are asked for, admit 12 warps an SM, whose two sums over the row then show (with the parameters in
// shared memory and 96 registers it spilled, 346 us).  Rows to come are copied ahead (cp.async).
// Everything is float32 until the one rounding of each output.
#include "common.cuh"

namespace m2 {
namespace rn {

constexpr int VEC = 8;
constexpr int MAX_N = 1024 * VEC;
enum { G_NONE = 0, G_CHANNEL = 1, G_SEQUENCE = 2, G_TOKEN = 3 };
enum { S_W1 = 0, S_B1, S_W2, S_B2, S_GATE, S_SCALE, S_COUNT };         // the column sums

struct Args {
  const void *x, *y, *g;
  long long ldx, ldy, ldg;
  long long rows, seq_len;
  int n, gate, g_f32, rms, norm1, norm2;
  float scale;
  const float *a, *w1, *b1, *w2, *b2;
  float eps;
  void *r, *h;
  float* stats;                          // rows x (mean1, rstd1, mean2, rstd2)
  // gradient
  const void *dr, *dh;
  void *dx, *dy, *dg;
  float* sums;                           // (blocks, S_COUNT, n)
  float* gate_sums;                      // (sequences * splits, n), or NULL where a sequence is one unit
  int splits;                            // units per sequence
};

// 8 columns as 4 packed pairs (two float32 operations an instruction)
struct V8 {
  f32x2 p[4];
  __device__ __forceinline__ float2 pair(int i) const { float2 f; f2_unpack(p[i], f.x, f.y); return f; }
};
__device__ __forceinline__ V8 splat8(float v) { return {{f2_splat(v), f2_splat(v), f2_splat(v), f2_splat(v)}}; }
__device__ __forceinline__ V8 fma8(const V8& a, const V8& b, const V8& c) { return {{f2_fma(a.p[0], b.p[0], c.p[0]), f2_fma(a.p[1], b.p[1], c.p[1]), f2_fma(a.p[2], b.p[2], c.p[2]), f2_fma(a.p[3], b.p[3], c.p[3])}}; }
__device__ __forceinline__ V8 mul8(const V8& a, const V8& b) { return {{f2_mul(a.p[0], b.p[0]), f2_mul(a.p[1], b.p[1]), f2_mul(a.p[2], b.p[2]), f2_mul(a.p[3], b.p[3])}}; }
__device__ __forceinline__ V8 add8(const V8& a, const V8& b) { return {{f2_add(a.p[0], b.p[0]), f2_add(a.p[1], b.p[1]), f2_add(a.p[2], b.p[2]), f2_add(a.p[3], b.p[3])}}; }
__device__ __forceinline__ float sum8(const V8& a) {
  const f32x2 s = f2_add(f2_add(a.p[0], a.p[1]), f2_add(a.p[2], a.p[3]));
  float x, y;
  f2_unpack(s, x, y);
  return x + y;
}
__device__ __forceinline__ V8 first8(const V8& a, int m) {           // zero from column m on
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = a.pair(i); r.p[i] = f2_pack(2 * i < m ? f.x : 0.f, 2 * i + 1 < m ? f.y : 0.f); }
  return r;
}

// How rows are read.  FULL: 16-byte pieces, n a multiple of 256, so that every thread has 8 columns; WIDE: 16-byte pieces, threads
// with 8 columns or none; PLAIN: any alignment, any n.
enum { PLAIN = 0, WIDE = 1, FULL = 2 };

__device__ __forceinline__ V8 from_bf16(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  V8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.p[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  return v;
}
__device__ __forceinline__ V8 from_f32(const uint4& u, const uint4& w) {
  return {{f2_pack(__uint_as_float(u.x), __uint_as_float(u.y)), f2_pack(__uint_as_float(u.z), __uint_as_float(u.w)),
           f2_pack(__uint_as_float(w.x), __uint_as_float(w.y)), f2_pack(__uint_as_float(w.z), __uint_as_float(w.w))}};
}
template <typename T> __device__ __forceinline__ V8 load_plain(const T* p, int m) {
  V8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.p[i] = f2_pack(2 * i < m ? (float)p[2 * i] : 0.f, 2 * i + 1 < m ? (float)p[2 * i + 1] : 0.f);
  return v;
}
template <int MODE> __device__ __forceinline__ void store8(__nv_bfloat16* p, const V8& v, int m) {
  if constexpr (MODE == PLAIN) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < m) p[i] = __float2bfloat16_rn(i & 1 ? v.pair(i / 2).y : v.pair(i / 2).x);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __float22bfloat162_rn(v.pair(i));
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <int MODE> __device__ __forceinline__ void store8(float* p, const V8& v, int m) {
  if constexpr (MODE == PLAIN) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < m) p[i] = i & 1 ? v.pair(i / 2).y : v.pair(i / 2).x;
  } else {
    const float2 a = v.pair(0), b = v.pair(1), c = v.pair(2), d = v.pair(3);
    reinterpret_cast<float4*>(p)[0] = make_float4(a.x, a.y, b.x, b.y);
    reinterpret_cast<float4*>(p)[1] = make_float4(c.x, c.y, d.x, d.y);
  }
}

// Rows ahead of their use: every thread copies the 16-byte pieces of its own columns into its own places of shared memory, so that
// no barrier is needed and no register is held.
template <int STAGES> struct Ring {
  uint32_t base, piece, stage;           // shared address of this thread's first place; distances of pieces and of stages
  uint32_t in, out;                      // the stages to be filled and to be read, as distances
  __device__ __forceinline__ Ring(void* mem, int pieces) {
    base = (uint32_t)__cvta_generic_to_shared(mem) + threadIdx.x * 16;
    piece = blockDim.x * 16;
    stage = pieces * piece;
    in = out = 0;
  }
  __device__ __forceinline__ void next(uint32_t& at) const { at = at + stage == STAGES * stage ? 0 : at + stage; }
  // 8 columns of either type; the place behind them
  __device__ __forceinline__ uint32_t put(uint32_t to, const char* src, bool f32) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + to), "l"(src) : "memory");
    if (f32) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + to + piece), "l"(src + 16) : "memory");
    return to + (f32 ? 2 * piece : piece);
  }
  __device__ __forceinline__ uint4 piece_at(uint32_t at) const {
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(base + at) : "memory");
    return u;
  }
  __device__ __forceinline__ V8 get(uint32_t at, bool f32) const { return f32 ? from_f32(piece_at(at), piece_at(at + piece)) : from_bf16(piece_at(at)); }
  __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }
};
// A tensor's rows one after the other, from this thread's columns on
struct Walk {
  const char* p; long long step;
  __device__ __forceinline__ Walk(const void* base, long long ld, long long row, int c0, int size, long long rows_a_step)
      : p(static_cast<const char*>(base) + (row * ld + c0) * size), step(rows_a_step * ld * size) {}
  __device__ __forceinline__ const char* go() { const char* q = p; p += step; return q; }
};
template <typename T> constexpr bool is_f32 = sizeof(T) == 4;
template <int MAXT> constexpr int stages = MAXT == 192 ? 3 : 2;      // as many as shared memory has room for

// Sums over the block of two values at once.  Two buffers by turns: one barrier a call.
template <int MAXT> struct Reduce {
  static constexpr int CAP = MAXT == 192 ? 6 : 32;     // warps at most: few of them are added without a loop
  float2 (*buf)[32];
  int turn;
  __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(~0u, a, o);
      b += __shfl_xor_sync(~0u, b, o);
    }
    const int nw = blockDim.x >> 5;
    if (nw == 1) return make_float2(a, b);
    if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = buf[turn][0];
#pragma unroll(CAP <= 6 ? CAP - 1 : 1)
    for (int w = 1; w < CAP; ++w) {
      if (w >= nw) break;
      const float2 q = buf[turn][w];
      s.x += q.x;
      s.y += q.y;
    }
    turn ^= 1;
    return s;
  }
  // mean and sum of squared distances to it over blocks of 256 columns a warp, in one pass: halves of equal size are joined,
  //   mean = (a + b) / 2,   M = Ma + Mb + (a - b)^2 size / 2,
  // which loses nothing where the mean is far from zero (sums of squares would)
  __device__ __forceinline__ float2 moments(const V8& v) {
    float mean = sum8(v) * 0.125f;
    const V8 d = add8(v, splat8(-mean));
    float m2 = sum8(mul8(d, d));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float b = __shfl_xor_sync(~0u, mean, o), q = __shfl_xor_sync(~0u, m2, o), e = b - mean;
      mean = fmaf(0.5f, e, mean);
      m2 = fmaf(e * e, 4.f * o, m2 + q);
    }
    const int nw = blockDim.x >> 5;
    if (nw == 1) return make_float2(mean, m2);
    if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = make_float2(mean, m2);
    __syncthreads();
    // all warps' means against the first one's: distances are as small as the row's spread
    const float2 f = buf[turn][0];
    float d1 = 0.f, d2 = 0.f;
    m2 = f.y;
#pragma unroll(CAP <= 6 ? CAP - 1 : 1)
    for (int w = 1; w < CAP; ++w) {
      if (w >= nw) break;
      const float2 q = buf[turn][w];
      const float e = q.x - f.x;
      d1 += e;
      d2 = fmaf(e, e, d2);
      m2 += q.y;
    }
    d1 /= nw;
    mean = f.x + d1;
    m2 += 256.f * fmaf(-nw * d1, d1, d2);
    turn ^= 1;
    return make_float2(mean, m2);
  }
};

// s / n from inv_n = 1 / n rounded, and one step of Newton's method on what is left: exact where the quotient is a float32 number, so
// that a row of equal values (whose sum is exact) has exactly their mean.  s * inv_n is one step off for n = 56 or 1000, say, which at
// eps 1e-12 became values of 0.1.  A division took 3 to 6 % longer, 32768 x 600 88 -> 92 us.
__device__ __forceinline__ float quotient(float s, float n, float inv_n) {
  const float q = s * inv_n;
  return fmaf(fmaf(-q, n, s), inv_n, q);
}

// mean and 1 / deviation of a row whose columns beyond n (m of this thread's 8 are inside) hold 0
template <int MODE, int MAXT> __device__ __forceinline__ float2 row_stats(Reduce<MAXT>& red, const V8& v, int m, float inv_n, float n, float eps, bool rms) {
  if (rms) return make_float2(0.f, rsqrtf(fmaf(red(sum8(mul8(v, v)), 0.f).x, inv_n, eps)));
  if constexpr (MODE == FULL) {
    const float2 s = red.moments(v);
    return make_float2(s.x, rsqrtf(fmaf(s.y, inv_n, eps)));
  }
  const float mean = quotient(red(sum8(v), 0.f).x, n, inv_n);
  const V8 d = first8(add8(v, splat8(-mean)), m);
  return make_float2(mean, rsqrtf(fmaf(red(sum8(mul8(d, d)), 0.f).x, inv_n, eps)));
}
__device__ __forceinline__ V8 normal(const V8& v, float mean, float rstd) { return mul8(add8(v, splat8(-mean)), splat8(rstd)); }

__device__ __forceinline__ V8 param(const float* p, int c0, int m, float otherwise) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = p && i < m ? __ldg(p + c0 + i) : otherwise;
  return {{f2_pack(f[0], f[1]), f2_pack(f[2], f[3]), f2_pack(f[4], f[5]), f2_pack(f[6], f[7])}};
}
__device__ __forceinline__ V8 channel_gate(const Args& a, int c0, int m) {
  if (a.gate != G_CHANNEL || m == 0) return splat8(1.f);
  return a.g_f32 ? load_plain(static_cast<const float*>(a.g) + c0, m) : load_plain(static_cast<const __nv_bfloat16*>(a.g) + c0, m);
}
__device__ __forceinline__ V8 gate_plain(const Args& a, long long at, int m) {
  return a.g_f32 ? load_plain(static_cast<const float*>(a.g) + at, m) : load_plain(static_cast<const __nv_bfloat16*>(a.g) + at, m);
}

template <typename TX, typename TY, int MODE, int MAXT>
__global__ void __launch_bounds__(MAXT)
forward_kernel(const Args a) {
  extern __shared__ uint4 ring_mem[];
  __shared__ float2 buf[2][32];
  pdl_wait();
  Reduce<MAXT> red = {buf, 0};
  const int c0 = threadIdx.x * VEC;
  const int m = MODE == FULL ? VEC : max(0, min(VEC, a.n - c0));        // this thread's columns
  const bool live = MODE == FULL || m > 0;
  const float inv_n = 1.f / a.n;
  const V8 w1 = param(a.w1, c0, m, 1.f), b1 = param(a.b1, c0, m, 0.f), w2 = param(a.w2, c0, m, 1.f), b2 = param(a.b2, c0, m, 0.f);
  const V8 sc = param(a.a, c0, m, a.scale);
  const bool by_row = a.gate >= G_SEQUENCE;
  V8 gc = channel_gate(a, c0, m);
  constexpr int STAGES = stages<MAXT>;
  constexpr int PX = is_f32<TX> ? 2 : 1, PY = is_f32<TY> ? 2 : 1;
  Ring<STAGES> ring(ring_mem, PX + PY + (by_row ? (a.g_f32 ? 2 : 1) : 0));
  Walk wx(a.x, a.ldx, blockIdx.x, c0, sizeof(TX), gridDim.x), wy(a.y, a.ldy, blockIdx.x, c0, sizeof(TY), gridDim.x);
  Walk wr(a.r, a.n, blockIdx.x, c0, sizeof(TX), gridDim.x), wh(a.h, a.n, blockIdx.x, c0, sizeof(TY), gridDim.x);
  auto gate_at = [&](long long row) { return ((a.gate == G_TOKEN ? row : row / a.seq_len) * a.ldg + c0); };
  long long ahead = blockIdx.x;          // the next row to be copied
  auto fetch = [&]() {
    if (MODE == PLAIN) return;
    if (live && ahead < a.rows) {
      uint32_t to = ring.put(ring.in, wx.go(), is_f32<TX>);
      to = ring.put(to, wy.go(), is_f32<TY>);
      if (by_row) ring.put(to, static_cast<const char*>(a.g) + (gate_at(ahead) << (a.g_f32 ? 2 : 1)), a.g_f32);
    }
    ahead += gridDim.x;
    ring.next(ring.in);
    ring.commit();
  };
  for (int s = 0; s < STAGES - 1; ++s) fetch();
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    V8 x = splat8(0.f), v = x, g = gc;
    if constexpr (MODE == PLAIN) {
      if (live) {
        x = load_plain(reinterpret_cast<const TX*>(wx.go()), m);
        v = load_plain(reinterpret_cast<const TY*>(wy.go()), m);
        if (by_row) g = gate_plain(a, gate_at(row), m);
      }
    } else {
      ring.wait();
      if (live) {
        x = ring.get(ring.out, is_f32<TX>);
        v = ring.get(ring.out + PX * ring.piece, is_f32<TY>);
        if (by_row) g = ring.get(ring.out + (PX + PY) * ring.piece, a.g_f32);
      }
      ring.next(ring.out);
      fetch();
    }
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (a.norm1) {
      s1 = row_stats<MODE, MAXT>(red, v, m, inv_n, a.n, a.eps, a.rms);
      v = fma8(normal(v, s1.x, s1.y), w1, b1);
    }
    v = fma8(g, v, mul8(sc, x));
    if (MODE != FULL) v = first8(v, m);
    TX* to = reinterpret_cast<TX*>(const_cast<char*>(wr.go()));
    if (live) store8<MODE>(to, v, m);
    if (a.norm2) {
      s2 = row_stats<MODE, MAXT>(red, v, m, inv_n, a.n, a.eps, a.rms);
      v = fma8(normal(v, s2.x, s2.y), w2, b2);
      TY* to = reinterpret_cast<TY*>(const_cast<char*>(wh.go()));
      if (live) store8<MODE>(to, v, m);
    }
    if (a.stats && threadIdx.x == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

// Forward of rows of 256 K columns, K <= 8: a warp has a row, 8 columns of each 256 a lane, so that nothing waits for a barrier and
// the 5 steps of a sum over lanes serve the whole row (with 8 columns a thread and a block per row they were half of the
// instructions: 598 us at 131072 x 1536).  y goes to registers; x and the gate wait in the lane's own places of shared memory until
// N_after is done, the parameters lie beside them.
constexpr int WARP_ROWS = 8;             // warps of a block
template <typename TX, typename TY, int K>
__global__ void __launch_bounds__(32 * WARP_ROWS, 2)
forward_warp_kernel(const Args a) {
  extern __shared__ uint4 ring_mem[];
  constexpr int N = 256 * K, PX = is_f32<TX> ? 2 : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inv_n = 1.f / N;
  const bool by_row = a.gate >= G_SEQUENCE, a_channel = a.a != nullptr, g_channel = a.gate == G_CHANNEL;
  pdl_wait();
  // parameters: columns 8 l .. 8 l + 3 of every lane, then the others, so that a load meets every bank once
  float4* par = reinterpret_cast<float4*>(ring_mem);
  constexpr int PLANE = N / 4;
  for (int e = threadIdx.x; e < PLANE; e += 32 * WARP_ROWS) {
    const int half = e / (32 * K), k = e / 32 % K, l = e & 31, c = k * 256 + l * 8 + half * 4;
    auto get = [&](const float* p, float otherwise) {
      return p ? make_float4(__ldg(p + c), __ldg(p + c + 1), __ldg(p + c + 2), __ldg(p + c + 3)) : make_float4(otherwise, otherwise, otherwise, otherwise);
    };
    par[e] = get(a.w1, 1.f);
    par[PLANE + e] = get(a.b1, 0.f);
    par[2 * PLANE + e] = get(a.w2, 1.f);
    par[3 * PLANE + e] = get(a.b2, 0.f);
    if (a_channel) par[4 * PLANE + e] = get(a.a, 0.f);
    if (g_channel) {
      float4 f;
      if (a.g_f32) f = get(static_cast<const float*>(a.g), 0.f);
      else {
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.g) + c;
        f = make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]), __bfloat162float(p[3]));
      }
      par[5 * PLANE + e] = f;
    }
  }
  __syncthreads();
  auto param8 = [&](int i, int k) -> V8 {
    const float4 f = par[i * PLANE + k * 32 + lane], g = par[i * PLANE + (K + k) * 32 + lane];
    return {{f2_pack(f.x, f.y), f2_pack(f.z, f.w), f2_pack(g.x, g.y), f2_pack(g.z, g.w)}};
  };
  // this lane's pieces of x and the gate: 32 lanes apart
  const int gp = by_row ? (a.g_f32 ? 2 : 1) : 0;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring_mem) + 6 * N * 4 + (warp * K * (PX + gp) * 32 + lane) * 16;
  auto copy = [&](int piece, const char* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + piece * 512), "l"(src) : "memory");
  };
  auto piece = [&](int i) {
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(mine + i * 512) : "memory");
    return u;
  };
  const int c0 = lane * 8;
  auto stats = [&](const V8 (&v)[K]) -> float2 {
    if (a.rms) {
      V8 q = mul8(v[0], v[0]);
#pragma unroll
      for (int k = 1; k < K; ++k) q = fma8(v[k], v[k], q);
      float s = sum8(q);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) s += __shfl_xor_sync(~0u, s, o);
      return make_float2(0.f, rsqrtf(fmaf(s, inv_n, a.eps)));
    }
    V8 t = v[0];
#pragma unroll
    for (int k = 1; k < K; ++k) t = add8(t, v[k]);
    float mean = quotient(sum8(t), 8.f * K, 1.f / (8 * K));
    const V8 back = splat8(-mean);
    t = splat8(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) { const V8 d = add8(v[k], back); t = fma8(d, d, t); }
    float m2 = sum8(t);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {   // halves of 8 K o values, as in Reduce::moments
      const float b = __shfl_xor_sync(~0u, mean, o), q = __shfl_xor_sync(~0u, m2, o), e = b - mean;
      mean = fmaf(0.5f, e, mean);
      m2 = fmaf(e * e, 4.f * K * o, m2 + q);
    }
    return make_float2(mean, rsqrtf(fmaf(m2, inv_n, a.eps)));
  };
  for (long long row = (long long)blockIdx.x * WARP_ROWS + warp; row < a.rows; row += (long long)gridDim.x * WARP_ROWS) {
    const char* px = static_cast<const char*>(a.x) + (row * a.ldx + c0) * (long long)sizeof(TX);
    const char* py = static_cast<const char*>(a.y) + (row * a.ldy + c0) * (long long)sizeof(TY);
    uint4 raw[K][is_f32<TY> ? 2 : 1];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      raw[k][0] = *reinterpret_cast<const uint4*>(py + k * 256 * sizeof(TY));
      if (is_f32<TY>) raw[k][is_f32<TY> ? 1 : 0] = *reinterpret_cast<const uint4*>(py + k * 256 * sizeof(TY) + 16);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      copy(k * PX, px + k * 256 * sizeof(TX));
      if (PX == 2) copy(k * PX + 1, px + k * 256 * sizeof(TX) + 16);
    }
    if (by_row) {
      const char* pg = static_cast<const char*>(a.g) + (((a.gate == G_TOKEN ? row : row / a.seq_len) * a.ldg + c0) << (a.g_f32 ? 2 : 1));
#pragma unroll
      for (int k = 0; k < K; ++k) {
        copy(K * PX + k * gp, pg + (k * 256 << (a.g_f32 ? 2 : 1)));
        if (a.g_f32) copy(K * PX + k * gp + 1, pg + (k * 256 << 2) + 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    V8 v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = is_f32<TY> ? from_f32(raw[k][0], raw[k][is_f32<TY> ? 1 : 0]) : from_bf16(raw[k][0]);
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (a.norm1) {
      s1 = stats(v);
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = fma8(normal(v[k], s1.x, s1.y), param8(0, k), param8(1, k));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    TX* pr = static_cast<TX*>(a.r) + row * N + c0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const V8 x = is_f32<TX> ? from_f32(piece(k * PX), piece(k * PX + PX - 1)) : from_bf16(piece(k * PX));
      V8 g = v[k];
      if (by_row) g = mul8(g, a.g_f32 ? from_f32(piece(K * PX + 2 * k), piece(K * PX + 2 * k + 1)) : from_bf16(piece(K * PX + k)));
      else if (g_channel) g = mul8(g, param8(5, k));
      v[k] = fma8(a_channel ? param8(4, k) : splat8(a.scale), x, g);
      store8<FULL>(pr + k * 256, v[k], 8);
    }
    if (a.norm2) {
      s2 = stats(v);
      TY* ph = static_cast<TY*>(a.h) + row * N + c0;
#pragma unroll
      for (int k = 0; k < K; ++k) store8<FULL>(ph + k * 256, fma8(normal(v[k], s2.x, s2.y), param8(2, k), param8(3, k)), 8);
    }
    if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

// MAXT: 192 threads, up to 1536 columns, are the most of which two blocks an SM have 168 registers a thread (65,536 / 384); that form
// spills 24 bytes.  512 threads have 128 and spill 384 to 480 bytes, 1024 have 64 and spill 1272; neither has been made to fit.  As rows
// get wider than the first form, 32768 x 1536 267 us becomes 757 at 2048 columns; 8192 x 8192 takes 1328 (floors 139, 185 and 185).
template <typename TX, typename TY, int MODE, int MAXT>
__global__ void __launch_bounds__(MAXT, (MAXT == 192 ? 2 : 1))
backward_kernel(const Args a) {
  extern __shared__ uint4 ring_mem[];
  __shared__ float2 buf[2][32];
  pdl_wait();
  Reduce<MAXT> red = {buf, 0};
  const int c0 = threadIdx.x * VEC;
  const int m = MODE == FULL ? VEC : max(0, min(VEC, a.n - c0));
  const bool live = MODE == FULL || m > 0;
  const float inv_n = 1.f / a.n;
  const V8 w1 = param(a.w1, c0, m, 1.f), b1 = param(a.b1, c0, m, 0.f), w2 = param(a.w2, c0, m, 1.f), sc = param(a.a, c0, m, a.scale);
  V8 gc = channel_gate(a, c0, m);
  V8 sum[S_COUNT];
#pragma unroll
  for (int k = 0; k < S_COUNT; ++k) sum[k] = splat8(0.f);
  const bool by_row = a.gate >= G_SEQUENCE, has_r = a.dr != nullptr, has_h = a.dh != nullptr;
  constexpr int PX = is_f32<TX> ? 2 : 1, PY = is_f32<TY> ? 2 : 1, STAGES = stages<MAXT>;
  const long long per = (a.seq_len + a.splits - 1) / a.splits;            // rows of a unit
  const long long units = a.rows / a.seq_len * a.splits;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long seq = unit / a.splits, first = seq * a.seq_len;
    const long long row0 = first + min(a.seq_len, (unit - seq * a.splits) * per), row1 = min(first + a.seq_len, row0 + per);
    Ring<STAGES> ring(ring_mem, 2 * PX + 2 * PY + (by_row ? (a.g_f32 ? 2 : 1) : 0));
    Walk wx(a.x, a.ldx, row0, c0, sizeof(TX), 1), wy(a.y, a.ldy, row0, c0, sizeof(TY), 1), wdr(a.dr, a.n, row0, c0, sizeof(TX), 1);
    Walk wdh(a.dh, a.n, row0, c0, sizeof(TY), 1), wg(a.g, a.gate == G_TOKEN ? a.ldg : 0, row0, c0, a.g_f32 ? 4 : 2, 1);
    if (a.gate == G_SEQUENCE) wg.p += (seq * a.ldg) << (a.g_f32 ? 2 : 1);
    Walk wdx(a.dx, a.n, row0, c0, sizeof(TX), 1), wdy(a.dy, a.n, row0, c0, sizeof(TY), 1), wdg(a.dg, a.n, row0, c0, a.g_f32 ? 4 : 2, 1);
    long long ahead = row0;
    auto fetch = [&]() {
      if (MODE == PLAIN) return;
      if (live && ahead < row1) {
        uint32_t to = ring.put(ring.in, wx.go(), is_f32<TX>);
        to = ring.put(to, wy.go(), is_f32<TY>);
        if (has_r) ring.put(to, wdr.go(), is_f32<TX>);
        to += PX * ring.piece;
        if (has_h) ring.put(to, wdh.go(), is_f32<TY>);
        to += PY * ring.piece;
        if (by_row) ring.put(to, wg.go(), a.g_f32);
      }
      ++ahead;
      ring.next(ring.in);
      ring.commit();
    };
    auto stats_of = [&](long long row) { return *reinterpret_cast<const float4*>(a.stats + 4 * row); };
    for (int s = 0; s < STAGES - 1; ++s) fetch();
    float4 next = row0 < row1 ? stats_of(row0) : make_float4(0.f, 1.f, 0.f, 1.f);
    for (long long row = row0; row < row1; ++row) {
      V8 x = splat8(0.f), yh = x, g = gc, u = x, dh = x;
      const float4 s = next;
      if (row + 1 < row1) next = stats_of(row + 1);
      if constexpr (MODE == PLAIN) {
        if (live) {
          x = load_plain(reinterpret_cast<const TX*>(wx.go()), m);
          yh = load_plain(reinterpret_cast<const TY*>(wy.go()), m);
          if (has_r) u = load_plain(reinterpret_cast<const TX*>(wdr.go()), m);
          if (has_h) dh = load_plain(reinterpret_cast<const TY*>(wdh.go()), m);
          if (by_row) g = gate_plain(a, (a.gate == G_TOKEN ? row : seq) * a.ldg + c0, m);
        }
      } else {
        ring.wait();
        if (live) {
          x = ring.get(ring.out, is_f32<TX>);
          yh = ring.get(ring.out + PX * ring.piece, is_f32<TY>);
          if (has_r) u = ring.get(ring.out + (PX + PY) * ring.piece, is_f32<TX>);
          if (has_h) dh = ring.get(ring.out + (2 * PX + PY) * ring.piece, is_f32<TY>);
          if (by_row) g = ring.get(ring.out + (2 * PX + 2 * PY) * ring.piece, a.g_f32);
        }
        ring.next(ring.out);
        fetch();
      }
      V8 n1 = yh;
      if (a.norm1) {
        yh = normal(yh, s.x, s.y);
        n1 = fma8(yh, w1, b1);
      }
      if (has_h) {
        V8 rh = normal(fma8(g, n1, mul8(sc, x)), s.z, s.w);
        if (MODE != FULL) rh = first8(rh, m);
        const V8 d = mul8(dh, w2);
        sum[S_W2] = fma8(dh, rh, sum[S_W2]);
        sum[S_B2] = add8(sum[S_B2], dh);
        const float2 t = red(sum8(d), sum8(mul8(d, rh)));
        // u += rstd (d - mean(d) - r^ mean(d r^))
        u = fma8(splat8(s.w), fma8(rh, splat8(-t.y * inv_n), add8(d, splat8(a.rms ? 0.f : -t.x * inv_n))), u);
        if (MODE != FULL) u = first8(u, m);
      }
      sum[S_SCALE] = fma8(x, u, sum[S_SCALE]);
      const V8 dg = mul8(u, n1);
      if (a.gate != G_TOKEN) sum[S_GATE] = add8(sum[S_GATE], dg);
      V8 d = mul8(g, u);
      char* to = const_cast<char*>(wdx.go());
      if (live && a.dx) store8<MODE>(reinterpret_cast<TX*>(to), mul8(sc, u), m);
      if (live && a.gate == G_TOKEN && a.dg) {
        to = const_cast<char*>(wdg.go());
        if (a.g_f32) store8<MODE>(reinterpret_cast<float*>(to), dg, m);
        else store8<MODE>(reinterpret_cast<__nv_bfloat16*>(to), dg, m);
      }
      if (a.norm1) {
        sum[S_W1] = fma8(d, yh, sum[S_W1]);
        sum[S_B1] = add8(sum[S_B1], d);
        d = mul8(d, w1);
        V8 q = mul8(d, yh);
        if (MODE != FULL) q = first8(q, m);
        const float2 t = red(sum8(d), sum8(q));                             // d is 0 in dead columns, as u is
        d = mul8(splat8(s.y), fma8(yh, splat8(-t.y * inv_n), add8(d, splat8(a.rms ? 0.f : -t.x * inv_n))));
      }
      to = const_cast<char*>(wdy.go());
      if (live && a.dy) store8<MODE>(reinterpret_cast<TY*>(to), d, m);
    }
    if (a.gate == G_SEQUENCE && a.dg) {                                   // this unit's share of the sequence's gate
      if (live) {
        if (a.gate_sums) store8<PLAIN>(a.gate_sums + unit * a.n + c0, sum[S_GATE], m);
        else if (a.g_f32) store8<PLAIN>(static_cast<float*>(a.dg) + seq * a.n + c0, sum[S_GATE], m);
        else store8<PLAIN>(static_cast<__nv_bfloat16*>(a.dg) + seq * a.n + c0, sum[S_GATE], m);
      }
      sum[S_GATE] = splat8(0.f);
    }
  }
  if (live && a.sums) {
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k) store8<PLAIN>(a.sums + ((long long)blockIdx.x * S_COUNT + k) * a.n + c0, sum[k], m);
  }
}

// Column sums over the blocks' (or a sequence's units') shares in a fixed order: 32 columns x 16 lanes a block.
struct JoinArgs {
  const float* sums; int blocks, n;
  float* out[S_COUNT];
  const float* gate_sums; int splits; long long seqs;
  void* dg; int g_f32;
  void* channel_dg;                       // the channel gate's gradient in the gate's type
};
__global__ void __launch_bounds__(512)
join_kernel(const JoinArgs j) {
  __shared__ float part[16][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const long long what = blockIdx.y;      // a column sum, or S_COUNT + a sequence (or 16 of them: few units each)
  if (what >= S_COUNT && j.splits <= 16) {
    const long long seq = (what - S_COUNT) * 16 + ty;
    if (seq >= j.seqs || c >= j.n) return;
    const float* p = j.gate_sums + seq * j.splits * (long long)j.n + c;
    float s = 0.f;
    for (int i = 0; i < j.splits; ++i) s += p[(long long)i * j.n];
    if (j.g_f32) static_cast<float*>(j.dg)[seq * j.n + c] = s;
    else st_from_float(static_cast<__nv_bfloat16*>(j.dg) + seq * j.n + c, s);
    return;
  }
  const bool seq = what >= S_COUNT;
  if (!seq && !j.out[what] && !(what == S_GATE && j.channel_dg)) return;
  const float* p = seq ? j.gate_sums + (what - S_COUNT) * j.splits * (long long)j.n : j.sums + what * j.n;
  const long long step = seq ? j.n : (long long)S_COUNT * j.n;
  const int count = seq ? j.splits : j.blocks;
  float s = 0.f;
  if (c < j.n) {
#pragma unroll 4
    for (int i = ty; i < count; i += 16) s += p[i * step + c];
  }
  part[ty][lane] = s;
  __syncthreads();
  if (ty == 0 && c < j.n) {
    for (int i = 1; i < 16; ++i) s += part[i][lane];
    void* to = seq ? j.dg : j.channel_dg;
    const long long at = seq ? (what - S_COUNT) * j.n + c : c;
    if (!seq && j.out[what]) j.out[what][c] = s;
    else if (j.g_f32) static_cast<float*>(to)[at] = s;
    else st_from_float(static_cast<__nv_bfloat16*>(to) + at, s);
  }
}

struct Plan { int threads, blocks, splits; long long units; };
// blocks: as many as the SMs hold at once by their registers (up to 128 and 168 a thread), no more than there are units.  Sequences are cut
// into units where that fills the blocks better; without a gate per sequence all rows are one sequence.
static Plan plan_of(long long rows, long long seq_len, int n, bool backward) {
  Plan p;
  p.threads = ((n + VEC - 1) / VEC + 31) / 32 * 32;
  const int per_sm = p.threads > 512 ? 1 : max(1, min(16, (backward ? 384 : 512) / p.threads));
  const long long most = (long long)m2_sm_count() * per_sm;
  const long long seqs = rows / seq_len;
  // the number of units a sequence whose rows, round after round of blocks, take the least time (256 sequences on 592 blocks: 2)
  long long splits = 1, best = -1;
  const long long top = seqs < most ? (most / seqs < seq_len ? most / seqs : seq_len) : seqs >= 4 * most ? 1 : (seq_len < 4 ? seq_len : 4);
  for (long long s = seqs < most ? top : 1; s <= top; ++s) {
    const long long time = (seqs * s + most - 1) / most * ((seq_len + s - 1) / s);
    if (best < 0 || time < best) { best = time; splits = s; }
  }
  p.splits = (int)splits;
  p.units = seqs * splits;
  p.blocks = (int)(p.units < most ? p.units : most);
  return p;
}

constexpr int SMEM_MOST = 226 * 1024;
template <typename TX, typename TY> static int smem_of(const Args& a, int ring_stages, bool backward, int threads) {
  const int gate = a.gate >= G_SEQUENCE ? (a.g_f32 ? 2 : 1) : 0;
  return ring_stages * (((is_f32<TX> ? 2 : 1) + (is_f32<TY> ? 2 : 1)) * (backward ? 2 : 1) + gate) * threads * 16;
}
template <typename TX, typename TY, int MODE, int MAXT, bool BACK> static int launch_t(const Args& a, int blocks, int threads, cudaStream_t st) {
  const int smem = smem_of<TX, TY>(a, MODE == PLAIN ? 0 : stages<MAXT>, BACK, threads);
  if constexpr (BACK) {
    if (MODE != PLAIN) M2_SMEM_ONCE((backward_kernel<TX, TY, MODE, MAXT>), SMEM_MOST);
    return m2_launch("m2_residual_norm_bwd", a.rows * a.n, backward_kernel<TX, TY, MODE, MAXT>, dim3(blocks), threads, smem, st, a);
  } else {
    if (MODE != PLAIN) M2_SMEM_ONCE((forward_kernel<TX, TY, MODE, MAXT>), SMEM_MOST);
    return m2_launch("m2_residual_norm_fwd", a.rows * a.n, forward_kernel<TX, TY, MODE, MAXT>, dim3(blocks), threads, smem, st, a);
  }
}
template <typename TX, typename TY, int K> static int launch_warp_k(const Args& a, cudaStream_t st) {
  const int gate = a.gate >= G_SEQUENCE ? (a.g_f32 ? 2 : 1) : 0;
  const int smem = 6 * 256 * K * 4 + WARP_ROWS * K * ((is_f32<TX> ? 2 : 1) + gate) * 512;
  constexpr int most = 6 * 256 * K * 4 + WARP_ROWS * K * 4 * 512;
  M2_SMEM_ONCE((forward_warp_kernel<TX, TY, K>), most);
  const long long blocks = (a.rows + WARP_ROWS - 1) / WARP_ROWS, held = (long long)m2_sm_count() * (K == 1 ? 4 : smem > 112 * 1024 ? 1 : 2);
  return m2_launch("m2_residual_norm_fwd", a.rows * a.n, forward_warp_kernel<TX, TY, K>, dim3((unsigned)(blocks < held ? blocks : held)), 32 * WARP_ROWS, smem, st, a);
}
template <typename TX, typename TY> static int launch_warp(const Args& a, cudaStream_t st) {
  switch (a.n / 256) {
    case 1: return launch_warp_k<TX, TY, 1>(a, st);
    case 2: return launch_warp_k<TX, TY, 2>(a, st);
    case 3: return launch_warp_k<TX, TY, 3>(a, st);
    case 4: return launch_warp_k<TX, TY, 4>(a, st);
    case 5: return launch_warp_k<TX, TY, 5>(a, st);
    case 6: return launch_warp_k<TX, TY, 6>(a, st);
    case 7: return launch_warp_k<TX, TY, 7>(a, st);
    default: return launch_warp_k<TX, TY, 8>(a, st);
  }
}
// Rows in 16-byte pieces: forward, a warp a row where a warp's registers hold it; else a block a row through the ring, up to 4096
// columns.  Longer rows, and rows in no pieces, are loaded value by value: 8192 x 8192 with a float32 stream takes 833 us, 16384 x 4096
// through the ring 283.  (Two stages of 8192 columns would fit into shared memory forward, and backward where the types and the gate
// leave 226 KB; there is no such form.)  Widths that are no multiple of 256 take the gradient's form of 512 threads even where 192
// would do: 32768 x 96 81 us, x 1000 319.
template <typename TX, typename TY, bool BACK> static int launch_n(const Args& a, bool wide, int blocks, int threads, cudaStream_t st) {
  if (threads > 512) return launch_t<TX, TY, PLAIN, 1024, BACK>(a, blocks, threads, st);
  if (!wide) return launch_t<TX, TY, PLAIN, 512, BACK>(a, blocks, threads, st);
  if (a.n % 256) return launch_t<TX, TY, WIDE, 512, BACK>(a, blocks, threads, st);
  if constexpr (BACK) {
    if (threads <= 192) return launch_t<TX, TY, FULL, 192, true>(a, blocks, threads, st);
  } else {
    if (a.n <= 2048) return launch_warp<TX, TY>(a, st);
  }
  return launch_t<TX, TY, FULL, 512, BACK>(a, blocks, threads, st);
}
template <bool BACK> static int launch_types(const Args& a, int xt, int yt, bool wide, int blocks, int threads, cudaStream_t st) {
  typedef __nv_bfloat16 B;
  if (xt == M2_F32) return yt == M2_F32 ? launch_n<float, float, BACK>(a, wide, blocks, threads, st) : launch_n<float, B, BACK>(a, wide, blocks, threads, st);
  return yt == M2_F32 ? launch_n<B, float, BACK>(a, wide, blocks, threads, st) : launch_n<B, B, BACK>(a, wide, blocks, threads, st);
}
static int fill(const char* name, Args& a, const m2_residual_norm_args& g) {
  M2_REQUIRE(g.n >= 1 && g.rows >= 0 && g.seq_len >= 1 && g.rows % g.seq_len == 0, M2_ERR_ARG, "%s: %lld rows of %d columns in sequences of %lld", name,
             g.rows, g.n, g.seq_len);
  M2_REQUIRE(g.n <= MAX_N, M2_ERR_UNSUPPORTED, "%s: rows of up to %d columns, got %d", name, MAX_N, g.n);
  M2_REQUIRE((g.x_dtype == M2_F32 || g.x_dtype == M2_BF16) && (g.y_dtype == M2_F32 || g.y_dtype == M2_BF16) &&
             (g.gate_kind == 0 || g.gate_dtype == M2_F32 || g.gate_dtype == M2_BF16), M2_ERR_UNSUPPORTED, "%s: tensors are float32 or bf16", name);
  M2_REQUIRE(g.gate_kind >= 0 && g.gate_kind <= 3, M2_ERR_ARG, "%s: gate_kind %d", name, g.gate_kind);
  M2_REQUIRE(g.rows == 0 || (g.x && g.y && (g.gate_kind == 0 || g.gate)), M2_ERR_ARG, "%s: x, y or the gate is NULL", name);
  M2_REQUIRE(g.eps >= 0.f, M2_ERR_ARG, "%s: eps %g", name, g.eps);
  M2_REQUIRE(g.rows <= 1 || (g.ldx >= 0 && g.ldy >= 0 && (g.gate_kind < G_SEQUENCE || g.ldg >= 0)), M2_ERR_ARG, "%s: a row stride is negative", name);
  a = Args{};
  a.x = g.x; a.y = g.y; a.g = g.gate; a.ldx = g.ldx; a.ldy = g.ldy; a.ldg = g.ldg;
  a.rows = g.rows;
  a.n = g.n; a.gate = g.gate_kind; a.g_f32 = g.gate_dtype == M2_F32; a.rms = g.rms != 0;
  a.seq_len = g.gate_kind == G_SEQUENCE ? g.seq_len : (g.rows > 0 ? g.rows : 1);
  a.norm1 = g.norm_after != 0; a.norm2 = g.norm_before != 0;
  a.scale = g.scale; a.a = g.scale_channel; a.eps = g.eps;
  a.w1 = a.norm1 ? g.after_weight : nullptr; a.b1 = a.norm1 ? g.after_bias : nullptr;
  a.w2 = a.norm2 ? g.before_weight : nullptr; a.b2 = a.norm2 ? g.before_bias : nullptr;
  return M2_OK;
}
static bool wide_rows(const m2_residual_norm_args& g) {
  return g.n % VEC == 0 && m2_aligned(g.x, 16) && m2_aligned(g.y, 16) && g.ldx % VEC == 0 && g.ldy % VEC == 0 &&
         (g.gate_kind < G_SEQUENCE || (m2_aligned(g.gate, 16) && g.ldg % VEC == 0));
}

}  // namespace rn
}  // namespace m2

extern "C" int m2_residual_norm_fwd(const m2_residual_norm_args* args, void* stream) {
  using namespace m2::rn;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_residual_norm_fwd: args is NULL");
  const m2_residual_norm_args& g = *args;
  Args a;
  if (int rc = fill("m2_residual_norm_fwd", a, g)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.r && (!a.norm2 || g.h), M2_ERR_ARG, "m2_residual_norm_fwd: an output is NULL");
  M2_REQUIRE(m2_aligned(g.stats, 16), M2_ERR_ALIGN, "m2_residual_norm_fwd: stats is not on a 16-byte boundary");
  a.r = g.r; a.h = g.h; a.stats = g.stats;
  const Plan p = plan_of(g.rows, g.rows, g.n, false);
  if (int rc = launch_types<false>(a, g.x_dtype, g.y_dtype, wide_rows(g) && m2_aligned(g.r, 16) && m2_aligned(g.h, 16), p.blocks, p.threads, (cudaStream_t)stream))
    return rc;
  return M2_OK;
}

extern "C" long long m2_residual_norm_workspace(long long rows, long long seq_len, int n, int gate_kind) {
  using namespace m2::rn;
  if (rows < 1 || n < 1 || n > MAX_N || seq_len < 1 || rows % seq_len) return 0;
  const Plan p = plan_of(rows, gate_kind == G_SEQUENCE ? seq_len : rows, n, true);
  const long long gate = gate_kind == G_SEQUENCE && p.splits > 1 ? p.units : 0;
  return ((long long)p.blocks * S_COUNT + gate) * n * (long long)sizeof(float);
}

extern "C" int m2_residual_norm_bwd(const m2_residual_norm_args* args, const m2_residual_norm_grads* grads, void* stream) {
  using namespace m2::rn;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_residual_norm_bwd: args or grads is NULL");
  const m2_residual_norm_args& g = *args;
  const m2_residual_norm_grads& d = *grads;
  Args a;
  if (int rc = fill("m2_residual_norm_bwd", a, g)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.stats && m2_aligned(g.stats, 16), M2_ERR_ARG, "m2_residual_norm_bwd: stats of the forward pass, on a 16-byte boundary, are needed");
  M2_REQUIRE(d.workspace && m2_aligned(d.workspace, 16), M2_ERR_ARG, "m2_residual_norm_bwd: a workspace on a 16-byte boundary is needed");
  a.stats = g.stats; a.dr = d.d_r; a.dh = a.norm2 ? d.d_h : nullptr; a.dx = d.d_x; a.dy = d.d_y; a.dg = d.d_gate;
  const long long need = m2_residual_norm_workspace(g.rows, g.gate_kind == G_SEQUENCE ? g.seq_len : g.rows, g.n, g.gate_kind);
  M2_REQUIRE(d.workspace_bytes >= need, M2_ERR_ARG, "m2_residual_norm_bwd: a workspace of %lld bytes, on this device the shape needs %lld", d.workspace_bytes, need);
  const Plan p = plan_of(a.rows, a.seq_len, a.n, true);
  a.splits = p.splits;
  a.sums = d.workspace;
  a.gate_sums = a.gate == G_SEQUENCE && p.splits > 1 ? d.workspace + (long long)p.blocks * S_COUNT * a.n : nullptr;
  const bool wide = wide_rows(g) && m2_aligned(d.d_r, 16) && m2_aligned(d.d_h, 16) && m2_aligned(d.d_x, 16) && m2_aligned(d.d_y, 16) && m2_aligned(d.d_gate, 16);
  const cudaStream_t st = (cudaStream_t)stream;
  if (int rc = launch_types<true>(a, g.x_dtype, g.y_dtype, wide, p.blocks, p.threads, st)) return rc;
  JoinArgs j = {};
  j.sums = a.sums; j.blocks = p.blocks; j.n = a.n;
  j.out[S_W1] = d.d_after_weight; j.out[S_B1] = d.d_after_bias; j.out[S_W2] = d.d_before_weight; j.out[S_B2] = d.d_before_bias; j.out[S_SCALE] = d.d_scale;
  j.channel_dg = a.gate == G_CHANNEL ? a.dg : nullptr;
  j.g_f32 = a.g_f32;
  const bool seq = a.gate_sums && a.dg;
  if (seq) { j.gate_sums = a.gate_sums; j.splits = p.splits; j.seqs = a.rows / a.seq_len; j.dg = a.dg; }
  if (seq || j.channel_dg || d.d_after_weight || d.d_after_bias || d.d_before_weight || d.d_before_bias || d.d_scale) {
    const long long ys = S_COUNT + (!seq ? 0 : j.splits <= 16 ? (j.seqs + 15) / 16 : j.seqs);
    return m2_launch("m2_residual_norm_bwd (sums)", a.rows * a.n, join_kernel, dim3((a.n + 31) / 32, (unsigned)ys), 512, 0, st, j);
  }
  return M2_OK;
}
