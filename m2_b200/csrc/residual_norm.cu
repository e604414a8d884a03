// Norms after and before a block, fused with the block's gate and the residual's scale:
//     r = a x + g N1(y),      h = N2(r),      N(v) = (v - mean) rstd w + b   (LayerNorm)   or   v rstd w + b   (RMS norm)
// and its gradient.  Generalises the post-norm of m2_add_layernorm_fwd (bert/src/bert_layers.py:506, which is a = g = 1, no N1,
// and h alone) to pre-, post- and sandwich-norm blocks.
//
// With u = dr + N2'(dh):  dx = a u,  da = sum x u,  dn = g u,  dg = u N1(y),  dy = N1'(dn), and for a norm with normalised values v^
//     N'(d) = rstd (d w - mean(d w) - v^ mean(d w v^)),      dw = sum d v^,      db = sum d      (no mean(d w) for the RMS norm).
//
// Bound: every tensor crosses HBM once in each direction.  A block of ceil(n / 256) warps walks over rows and a thread owns the
// same 8 columns of each: weights stay in its registers, and so do the column sums of the gradient, which meet in a second, small
// launch that adds the blocks' sums in a fixed order (no atomics: two runs give the same bits).  The next row is loaded while the
// present one is reduced.  Everything is float32 until the one rounding of each output.
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

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 columns of a row as they lie in memory, so that the next row costs few registers
template <typename T, bool WIDE> struct Cols;
template <> struct Cols<__nv_bfloat16, true> {
  uint4 u;
  __device__ void load(const __nv_bfloat16* p, int) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ void get(float (&f)[8]) const { unpack8(u, f); }
  __device__ static void store(__nv_bfloat16* p, const float (&f)[8], int) { *reinterpret_cast<uint4*>(p) = pack8(f); }
};
template <> struct Cols<float, true> {
  float4 u, v;
  __device__ void load(const float* p, int) { u = reinterpret_cast<const float4*>(p)[0]; v = reinterpret_cast<const float4*>(p)[1]; }
  __device__ void get(float (&f)[8]) const { f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w; }
  __device__ static void store(float* p, const float (&f)[8], int) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <typename T> struct Cols<T, false> {      // any alignment and any number of columns
  float e[8];
  __device__ void load(const T* p, int m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < m ? (float)p[i] : 0.f;
  }
  __device__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = e[i];
  }
  __device__ static void store(T* p, const float (&f)[8], int m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < m) st_from_float(p + i, f[i]);
  }
};
// a gate of either type
template <bool WIDE> struct GateCols {
  Cols<float, WIDE> f;
  Cols<__nv_bfloat16, WIDE> b;
  __device__ void load(const void* p, long long at, bool f32, int m) {
    if (f32) f.load(static_cast<const float*>(p) + at, m); else b.load(static_cast<const __nv_bfloat16*>(p) + at, m);
  }
  __device__ void get(float (&v)[8], bool f32) const { if (f32) f.get(v); else b.get(v); }
};

// Sums over the block of two values at once.  Two buffers by turns: one barrier a call.
struct Reduce {
  float2 (*buf)[32];
  int turn;
  __device__ float2 operator()(float a, float b) {
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
    for (int w = 1; w < nw; ++w) { const float2 q = buf[turn][w]; s.x += q.x; s.y += q.y; }
    turn ^= 1;
    return s;
  }
};

// mean and 1 / deviation of a row whose columns beyond n (m of this thread's 8 are inside) hold 0
__device__ __forceinline__ float2 row_stats(Reduce& red, const float (&v)[8], int m, float inv_n, float eps, bool rms) {
  float mean = 0.f, s = 0.f;
  if (!rms) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
    mean = red(s, 0.f).x * inv_n;
  }
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const float d = i < m ? v[i] - mean : 0.f; s = fmaf(d, d, s); }
  return make_float2(mean, rsqrtf(fmaf(red(s, 0.f).x, inv_n, eps)));
}

__device__ __forceinline__ void param(float (&f)[8], const float* p, int c0, int m, float otherwise) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = p && i < m ? __ldg(p + c0 + i) : otherwise;
}

template <typename TX, typename TY, bool WIDE, int MAXT>
__global__ void __launch_bounds__(MAXT)
forward_kernel(const Args a) {
  __shared__ float2 buf[2][32];
  Reduce red = {buf, 0};
  const int c0 = threadIdx.x * VEC;
  const int m = max(0, min(VEC, a.n - c0));                             // this thread's columns
  const bool live = m > 0;
  const float inv_n = 1.f / a.n;
  float w1[8], b1[8], w2[8], b2[8], sc[8], gc[8];
  param(w1, a.w1, c0, m, 1.f); param(b1, a.b1, c0, m, 0.f);
  param(w2, a.w2, c0, m, 1.f); param(b2, a.b2, c0, m, 0.f);
  param(sc, a.a, c0, m, a.scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) gc[i] = 1.f;
  if (a.gate == G_CHANNEL && live) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < m) gc[i] = a.g_f32 ? static_cast<const float*>(a.g)[c0 + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.g)[c0 + i]);
  }
  const bool by_row = a.gate >= G_SEQUENCE;
  Cols<TX, WIDE> cx;
  Cols<TY, WIDE> cy;
  GateCols<WIDE> cg;
  auto fetch = [&](long long row) {
    if (!live) return;
    cx.load(static_cast<const TX*>(a.x) + row * a.ldx + c0, m);
    cy.load(static_cast<const TY*>(a.y) + row * a.ldy + c0, m);
    if (by_row) cg.load(a.g, (a.gate == G_TOKEN ? row : row / a.seq_len) * a.ldg + c0, a.g_f32, m);
  };
  if ((long long)blockIdx.x < a.rows) fetch(blockIdx.x);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float x[8] = {}, v[8] = {}, g[8];
    if (live) { cx.get(x); cy.get(v); }
    if (by_row && live) {
      cg.get(g, a.g_f32);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = gc[i];
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    float2 s1 = make_float2(0.f, 1.f), s2 = s1;
    if (a.norm1) {
      s1 = row_stats(red, v, m, inv_n, a.eps, a.rms);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf((v[i] - s1.x) * s1.y, w1[i], b1[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < m ? fmaf(g[i], v[i], sc[i] * x[i]) : 0.f;
    if (live) Cols<TX, WIDE>::store(static_cast<TX*>(a.r) + row * a.n + c0, v, m);
    if (a.norm2) {
      s2 = row_stats(red, v, m, inv_n, a.eps, a.rms);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf((v[i] - s2.x) * s2.y, w2[i], b2[i]);
      if (live) Cols<TY, WIDE>::store(static_cast<TY*>(a.h) + row * a.n + c0, v, m);
    }
    if (a.stats && threadIdx.x == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

template <typename TX, typename TY, bool WIDE, int MAXT>
__global__ void __launch_bounds__(MAXT)
backward_kernel(const Args a) {
  __shared__ float2 buf[2][32];
  Reduce red = {buf, 0};
  const int c0 = threadIdx.x * VEC;
  const int m = max(0, min(VEC, a.n - c0));
  const bool live = m > 0;
  const float inv_n = 1.f / a.n;
  float w1[8], b1[8], w2[8], sc[8], gc[8];
  param(w1, a.w1, c0, m, 1.f); param(b1, a.b1, c0, m, 0.f);
  param(w2, a.w2, c0, m, 1.f);
  param(sc, a.a, c0, m, a.scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) gc[i] = 1.f;
  if (a.gate == G_CHANNEL && live) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < m) gc[i] = a.g_f32 ? static_cast<const float*>(a.g)[c0 + i] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.g)[c0 + i]);
  }
  float sum[S_COUNT][8] = {};
  const bool by_row = a.gate >= G_SEQUENCE;
  const long long per = (a.seq_len + a.splits - 1) / a.splits;            // rows of a unit
  const long long units = a.rows / a.seq_len * a.splits;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long seq = unit / a.splits, first = seq * a.seq_len;
    const long long row0 = first + min(a.seq_len, (unit - seq * a.splits) * per), row1 = min(first + a.seq_len, row0 + per);
    Cols<TX, WIDE> cx, cdr;
    Cols<TY, WIDE> cy, cdh;
    GateCols<WIDE> cg;
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    auto fetch = [&](long long row) {
      st = *reinterpret_cast<const float4*>(a.stats + 4 * row);
      if (!live) return;
      cx.load(static_cast<const TX*>(a.x) + row * a.ldx + c0, m);
      cy.load(static_cast<const TY*>(a.y) + row * a.ldy + c0, m);
      if (by_row) cg.load(a.g, (a.gate == G_TOKEN ? row : seq) * a.ldg + c0, a.g_f32, m);
      if (a.dr) cdr.load(static_cast<const TX*>(a.dr) + row * a.n + c0, m);
      if (a.dh) cdh.load(static_cast<const TY*>(a.dh) + row * a.n + c0, m);
    };
    if (row0 < row1) fetch(row0);
    for (long long row = row0; row < row1; ++row) {
      float x[8] = {}, yh[8] = {}, g[8], u[8] = {}, dh[8] = {};
      const float4 s = st;
      if (live) {
        cx.get(x);
        cy.get(yh);
        if (a.dr) cdr.get(u);
        if (a.dh) cdh.get(dh);
      }
      if (by_row && live) {
        cg.get(g, a.g_f32);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = gc[i];
      }
      if (row + 1 < row1) fetch(row + 1);
      float n1[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.norm1) yh[i] = (yh[i] - s.x) * s.y;
        n1[i] = a.norm1 ? fmaf(yh[i], w1[i], b1[i]) : yh[i];
      }
      if (a.norm2 && a.dh) {
        float rh[8], p = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          rh[i] = i < m ? (fmaf(g[i], n1[i], sc[i] * x[i]) - s.z) * s.w : 0.f;
          const float d = dh[i] * w2[i];
          sum[S_W2][i] = fmaf(dh[i], rh[i], sum[S_W2][i]);
          sum[S_B2][i] += dh[i];
          p += d;
          q = fmaf(d, rh[i], q);
        }
        const float2 t = red(p, q);
        const float mp = a.rms ? 0.f : t.x * inv_n, mq = t.y * inv_n;
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = i < m ? fmaf(s.w, fmaf(-rh[i], mq, fmaf(dh[i], w2[i], -mp)), u[i]) : 0.f;
      }
      float d[8], dg[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[S_SCALE][i] = fmaf(x[i], u[i], sum[S_SCALE][i]);
        dg[i] = u[i] * n1[i];
        if (a.gate != G_TOKEN) sum[S_GATE][i] += dg[i];
        d[i] = g[i] * u[i];
        x[i] = sc[i] * u[i];
      }
      if (live && a.dx) Cols<TX, WIDE>::store(static_cast<TX*>(a.dx) + row * a.n + c0, x, m);
      if (live && a.gate == G_TOKEN && a.dg) {
        if (a.g_f32) Cols<float, WIDE>::store(static_cast<float*>(a.dg) + row * a.n + c0, dg, m);
        else Cols<__nv_bfloat16, WIDE>::store(static_cast<__nv_bfloat16*>(a.dg) + row * a.n + c0, dg, m);
      }
      if (a.norm1) {
        float p = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum[S_W1][i] = fmaf(d[i], yh[i], sum[S_W1][i]);
          sum[S_B1][i] += d[i];
          d[i] *= w1[i];
          p += i < m ? d[i] : 0.f;
          q = i < m ? fmaf(d[i], yh[i], q) : q;
        }
        const float2 t = red(p, q);
        const float mp = a.rms ? 0.f : t.x * inv_n, mq = t.y * inv_n;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = s.y * fmaf(-yh[i], mq, d[i] - mp);
      }
      if (live && a.dy) Cols<TY, WIDE>::store(static_cast<TY*>(a.dy) + row * a.n + c0, d, m);
    }
    if (a.gate == G_SEQUENCE && a.dg) {                                   // this unit's share of the sequence's gate
      if (live) {
        if (a.gate_sums) Cols<float, false>::store(a.gate_sums + unit * a.n + c0, sum[S_GATE], m);
        else if (a.g_f32) Cols<float, false>::store(static_cast<float*>(a.dg) + seq * a.n + c0, sum[S_GATE], m);
        else Cols<__nv_bfloat16, false>::store(static_cast<__nv_bfloat16*>(a.dg) + seq * a.n + c0, sum[S_GATE], m);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[S_GATE][i] = 0.f;
    }
  }
  if (live && a.sums) {
#pragma unroll
    for (int k = 0; k < S_COUNT; ++k)
      Cols<float, false>::store(a.sums + ((long long)blockIdx.x * S_COUNT + k) * a.n + c0, sum[k], m);
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
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const long long what = blockIdx.y;      // a column sum, or S_COUNT + a sequence
  const bool seq = what >= S_COUNT;
  if (!seq && !j.out[what] && !(what == S_GATE && j.channel_dg)) return;
  const float* p = seq ? j.gate_sums + (what - S_COUNT) * j.splits * (long long)j.n : j.sums + what * j.n;
  const long long step = seq ? j.n : (long long)S_COUNT * j.n;
  const int count = seq ? j.splits : j.blocks;
  float s = 0.f;
  if (c < j.n) for (int i = ty; i < count; i += 16) s += p[i * step + c];
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
// blocks: as many as the SMs hold at once (about 120 registers a thread), no more than there are units.  Sequences are cut into
// units where there are fewer of them than blocks; without a gate per sequence all rows are one sequence.
static Plan plan_of(long long rows, long long seq_len, int n, bool backward) {
  Plan p;
  p.threads = ((n + VEC - 1) / VEC + 31) / 32 * 32;
  const int per_sm = p.threads > 512 ? 1 : max(1, min(16, (backward ? 384 : 512) / p.threads));
  const long long most = (long long)m2_sm_count() * per_sm;
  const long long seqs = rows / seq_len;
  long long splits = (most + seqs - 1) / seqs;
  if (splits > seq_len) splits = seq_len;
  p.splits = (int)splits;
  p.units = seqs * splits;
  p.blocks = (int)(p.units < most ? p.units : most);
  return p;
}

template <typename TX, typename TY, bool WIDE> static void launch_t(const Args& a, bool backward, int blocks, int threads, cudaStream_t st) {
  if (threads <= 256) {
    if (backward) backward_kernel<TX, TY, WIDE, 256><<<blocks, threads, 0, st>>>(a);
    else forward_kernel<TX, TY, WIDE, 256><<<blocks, threads, 0, st>>>(a);
  } else {
    if (backward) backward_kernel<TX, TY, WIDE, 1024><<<blocks, threads, 0, st>>>(a);
    else forward_kernel<TX, TY, WIDE, 1024><<<blocks, threads, 0, st>>>(a);
  }
}
static void launch(const Args& a, int xt, int yt, bool wide, bool backward, int blocks, int threads, cudaStream_t st) {
  typedef __nv_bfloat16 B;
  if (wide) {
    if (xt == M2_F32) yt == M2_F32 ? launch_t<float, float, true>(a, backward, blocks, threads, st) : launch_t<float, B, true>(a, backward, blocks, threads, st);
    else yt == M2_F32 ? launch_t<B, float, true>(a, backward, blocks, threads, st) : launch_t<B, B, true>(a, backward, blocks, threads, st);
  } else {
    if (xt == M2_F32) yt == M2_F32 ? launch_t<float, float, false>(a, backward, blocks, threads, st) : launch_t<float, B, false>(a, backward, blocks, threads, st);
    else yt == M2_F32 ? launch_t<B, float, false>(a, backward, blocks, threads, st) : launch_t<B, B, false>(a, backward, blocks, threads, st);
  }
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
  M2_REQUIRE((g.ldx >= g.n || g.ldx == 0 || g.rows <= 1) && (g.ldy >= g.n || g.ldy == 0 || g.rows <= 1), M2_ERR_ARG, "%s: a row stride is smaller than a row", name);
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
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_residual_norm_fwd: args is NULL");
  const m2_residual_norm_args& g = *args;
  Args a;
  if (int rc = fill("m2_residual_norm_fwd", a, g)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.r && (!a.norm2 || g.h), M2_ERR_ARG, "m2_residual_norm_fwd: an output is NULL");
  M2_REQUIRE(m2_aligned(g.stats, 16), M2_ERR_ALIGN, "m2_residual_norm_fwd: stats is not on a 16-byte boundary");
  a.r = g.r; a.h = g.h; a.stats = g.stats;
  const Plan p = plan_of(g.rows, g.rows, g.n, false);
  launch(a, g.x_dtype, g.y_dtype, wide_rows(g) && m2_aligned(g.r, 16) && m2_aligned(g.h, 16), false, p.blocks, p.threads, (cudaStream_t)stream);
  M2_LAUNCH_CHECK("m2_residual_norm_fwd");
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
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_residual_norm_bwd: args or grads is NULL");
  const m2_residual_norm_args& g = *args;
  const m2_residual_norm_grads& d = *grads;
  Args a;
  if (int rc = fill("m2_residual_norm_bwd", a, g)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.stats && m2_aligned(g.stats, 16), M2_ERR_ARG, "m2_residual_norm_bwd: stats of the forward pass, on a 16-byte boundary, are needed");
  M2_REQUIRE(d.workspace && m2_aligned(d.workspace, 16), M2_ERR_ARG, "m2_residual_norm_bwd: a workspace on a 16-byte boundary is needed");
  a.stats = g.stats; a.dr = d.d_r; a.dh = a.norm2 ? d.d_h : nullptr; a.dx = d.d_x; a.dy = d.d_y; a.dg = d.d_gate;
  const Plan p = plan_of(a.rows, a.seq_len, a.n, true);
  a.splits = p.splits;
  a.sums = d.workspace;
  a.gate_sums = a.gate == G_SEQUENCE && p.splits > 1 ? d.workspace + (long long)p.blocks * S_COUNT * a.n : nullptr;
  const bool wide = wide_rows(g) && m2_aligned(d.d_r, 16) && m2_aligned(d.d_h, 16) && m2_aligned(d.d_x, 16) && m2_aligned(d.d_y, 16) && m2_aligned(d.d_gate, 16);
  const cudaStream_t st = (cudaStream_t)stream;
  launch(a, g.x_dtype, g.y_dtype, wide, true, p.blocks, p.threads, st);
  M2_LAUNCH_CHECK("m2_residual_norm_bwd");
  JoinArgs j = {};
  j.sums = a.sums; j.blocks = p.blocks; j.n = a.n;
  j.out[S_W1] = d.d_after_weight; j.out[S_B1] = d.d_after_bias; j.out[S_W2] = d.d_before_weight; j.out[S_B2] = d.d_before_bias; j.out[S_SCALE] = d.d_scale;
  j.channel_dg = a.gate == G_CHANNEL ? a.dg : nullptr;
  j.g_f32 = a.g_f32;
  const bool seq = a.gate_sums && a.dg;
  if (seq) { j.gate_sums = a.gate_sums; j.splits = p.splits; j.seqs = a.rows / a.seq_len; j.dg = a.dg; }
  if (seq || j.channel_dg || d.d_after_weight || d.d_after_bias || d.d_before_weight || d.d_before_bias || d.d_scale) {
    const long long ys = S_COUNT + (seq ? j.seqs : 0);
    join_kernel<<<dim3((a.n + 31) / 32, (unsigned)ys), 512, 0, st>>>(j);
    M2_LAUNCH_CHECK("m2_residual_norm_bwd (sums)");
  }
  return M2_OK;
}
