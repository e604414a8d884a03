// Selective state space scan: every channel d has a state of N numbers that fade and are fed by the token itself,
//     s_t = softplus(delta_t + bias)  (or delta_t),     h_t[n] = exp(s_t a[d,n]) h_{t-1}[n] + s_t x_t b_t[n],
//     y_t = (sum_n c_t[n] h_t[n] + skip x_t) silu(z_t),
// its gradients, and one token at a time.  No counterpart in the reference, whose mixer is the long convolution
// (bert/src/mm/monarch_mixer_sequence_mixer.py:100-154).
//
// Bound: one exp for each token, channel and state (the special functions give 16 a cycle and SM), three with the gradients; then the instructions around
// it: 20 packed FMAs, 8 exps, 4 loads from shared memory for 16 channels and 16 states a token, 80 in all, 235 back.  No tensor cores: every channel has
// decays of its own, so that no product shares an operand.  A block has 64 channels and takes 32 tokens at a time: elementwise part (steps, gates) by
// pieces of 16 bytes, then the recurrence with two channels and four states a thread, in registers; y is summed over four lanes.
// Measured (bf16, 16 states): 16 x 2048 x 1536 forward 432 us (exps alone 179), gradients 1460 (447, as half of the exps come twice); 1 x 32768 x 768 forward 336 us in three
// launches (179, as the sums of the segments need the exps too).  Where SMs are full the forward kernel issues in 62 % of the cycles, exps 65 %, shared memory 52 %; back 56, 47
// and 63, in wait for the results of instructions before.  An exp in four as a polynomial on the FMA pipe: 526 us where the exps alone took 481; operands doubled
// in shared memory for packed FMAs: 479 where 465 were; reductions of y and q through shared memory instead of shuffles: 1749 back; the next
// tile's pieces held in registers: 512 where 465 were.
#include "common.cuh"

namespace m2 {
namespace ss {

constexpr int THREADS = 128;
constexpr int TT = 32;                   // tokens of a tile
constexpr int MAX_STATES = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;

// A thread has two channels with S states of each; QL lanes share a channel's states.  4 x 4 for up to 16 states, 8 x 4 up to 32, 8 x 8 up to 64: sixteen
// states a lane were tried and spilled hundreds of bytes.
__host__ __device__ constexpr int channels_of(int ql) { return 256 / ql; }                          // of a block

// Blocks of the gradients' kernel that an SM holds: 168 registers and 74 KB of shared memory up to 16 states, 255 and 90 to 93 beyond; none spills
__host__ __device__ constexpr int back_blocks(int np) { return np == 16 ? 3 : 2; }
// Tokens whose states are at hand at one time: four, or two where a lane has twice the states
__host__ __device__ constexpr int few(int np) { return np == 16 ? 4 : 2; }
constexpr int ASIDE = TT / 4 - 1;        // more than 16 states: places for states in front of every fourth token of a tile but its first
constexpr int PLACES = 4096;             // such blocks, 235 MB (with as many as run at once, 64 ragged texts of 768 channels and 64 states took 1760 us instead of 1610)

struct Rows { const void* p; long long sb, st; int vec; };           // vec: 16-byte pieces
struct Group { const void* p; long long sb, st, sg; int vec; };       // vec: four states at once

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
  float* aside;                          // more than 16 states: (blocks, ASIDE, S, THREADS, 2), each thread's states in front of every fourth token of a tile
  void *db, *dc;
  float *da, *d_skip, *d_bias, *d_state_in;
};

using lp::Piece;
using lp::ex2;

__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.f + ex2(-v * LOG2E)); }
// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|): log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3, and atanh(s) = s + s^3 P(s^2) with P a
// least-squares fit in s^2 <= 1/9 that leaves 5e-9 of s: small steps keep their digits.
__device__ __forceinline__ float step_of(float v, int softplus) {
  if (!softplus) return v;
  const float e = ex2(-fabsf(v) * LOG2E), s = e * rcp(2.f + e), u = s * s;
  float p = fmaf(0.140122298f, u, 0.139995704f);
  p = fmaf(p, u, 0.200108495f);
  p = fmaf(p, u, 0.333332066f);
  return fmaxf(v, 0.f) + 2.f * fmaf(s * u, p, s);
}

template <typename T> __device__ __forceinline__ uint4 load_piece(const T* p, int valid, bool vec) {
  constexpr int E = Piece<T>::N;
  if (vec && valid >= E) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int j = 0; j < E && j < valid; ++j) {
    uint32_t u;
    if constexpr (sizeof(T) == 4) u = __ldg(reinterpret_cast<const uint32_t*>(p) + j);
    else u = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + j) << (j & 1) * 16;
    const int at = j * (int)sizeof(T) / 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] |= q == at ? u : 0;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ void store_piece(T* p, const float (&f)[Piece<T>::N], int valid, bool vec) {
  constexpr int E = Piece<T>::N;
  const uint4 u = Piece<T>::put(f);
  if (vec && valid >= E) { *reinterpret_cast<uint4*>(p) = u; return; }
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll 1
  for (int j = 0; j < E && j < valid; ++j) {
    const uint32_t word = j * sizeof(T) < 4 ? w[0] : j * sizeof(T) < 8 ? w[1] : j * sizeof(T) < 12 ? w[2] : w[3];
    if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[j] = word;
    else reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)(word >> (j & 1) * 16);
  }
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
template <int H> __device__ __forceinline__ void ld_pairs(const float* p, f32x2 (&v)[H]) {
#pragma unroll
  for (int i = 0; i < H; i += 2) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p + 2 * i);
    v[i] = u.x; v[i + 1] = u.y;
  }
}
template <int H> __device__ __forceinline__ void st_pairs(float* p, const f32x2 (&v)[H]) {
#pragma unroll
  for (int i = 0; i < H; i += 2) *reinterpret_cast<ulonglong2*>(p + 2 * i) = make_ulonglong2(v[i], v[i + 1]);
}
// a in units of a factor of two, within float32: a step of 0 fades nothing, also where log2(e) would make an infinity of a (below -2.36e38) or a is one
__device__ __forceinline__ float rate(float a) {
  constexpr float MOST = 3.402823466e38f;
  const float v = a * LOG2E;
  return v < -MOST ? -MOST : v > MOST ? MOST : v;                        // NaN stays
}
// adds to a thread's own numbers in memory; nothing is waited for, and one thread's additions to one place keep their order
template <int H> __device__ __forceinline__ void add_pairs(float* p, const f32x2 (&v)[H]) {
#pragma unroll
  for (int i = 0; i < H; i += 2) {
    float f[4];
    f2_unpack(v[i], f[0], f[1]);
    f2_unpack(v[i + 1], f[2], f[3]);
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + 2 * i), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
  }
}
__device__ __forceinline__ float both(f32x2 v) {
  float x, y;
  f2_unpack(v, x, y);
  return x + y;
}
// What a token brings to a thread.  The loops ask for a token's operands one token ahead, for its step two ahead, and have the next token's decays
// computed while this one's are used, so that neither shared memory nor the exps are waited for.
// H = S / 2 pairs of states; channels one by one.  Shared memory gives four bytes a lane and cycle whatever lanes share, so that b and c lie there
// once, and the channels' numbers are doubled in registers.
template <int H, bool E, bool Cs> struct Token {
  f32x2 x, e, B[H], C[H];                // x, e: of the two channels
  __device__ __forceinline__ void get(const float* dx, const float* ep, const float* b, const float* c) {
    x = ld2(dx);
    if constexpr (E) e = ld2(ep);
    ld_pairs<H>(b, B);
    if constexpr (Cs) ld_pairs<H>(c, C);
  }
};
__device__ __forceinline__ void splat2(f32x2 v, f32x2 (&s)[2]) {
  float x, y;
  f2_unpack(v, x, y);
  s[0] = f2_splat(x);
  s[1] = f2_splat(y);
}
template <int H> __device__ __forceinline__ void decays(f32x2 dt, const f32x2 (&A)[2][H], f32x2 (&d)[2][H]) {
  f32x2 s[2];
  splat2(dt, s);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < H; ++i) d[c][i] = ex2_pair(f2_mul(s[c], A[c][i]));
}
// What was carried, by 2^x for the decays that it met, and what came since.  Nothing carried is nothing, also where states that grow would make infinity of it; a
// factor beyond float32 is met in two halves, as a small state (a large one) may well have grown (faded) by it.
__device__ __forceinline__ float part_of(float x) { return fabsf(x) > 120.f ? 0.5f : 1.f; }
__device__ __forceinline__ float carry(float part, float f, float before, float own) {             // f = 2^(part x)
  return before == 0.f ? own : fmaf(part < 1.f ? before * f : before, f, own);
}
__device__ __forceinline__ float carry(float x, float before, float own) {
  const float part = part_of(x);
  return carry(part, ex2(part * x), before, own);
}
template <int H> __device__ __forceinline__ void carry_pairs(f32x2 dt, const f32x2 (&A)[2][H], f32x2 (&h)[2][H], const f32x2 (&own)[2][H]) {      // h becomes the sum
  float s[2];
  f2_unpack(dt, s[0], s[1]);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < H; ++i) {
      float x[2], b[2], o[2];
      f2_unpack(f2_mul(f2_splat(s[c]), A[c][i]), x[0], x[1]);
      f2_unpack(h[c][i], b[0], b[1]);
      f2_unpack(own[c][i], o[0], o[1]);
      h[c][i] = f2_pack(carry(x[0], b[0], o[0]), carry(x[1], b[1], o[1]));
    }
}

// The sum over the lanes of a channel's states of v and w, of two channels each: lane bit 0 ends with the channel, bit 1 with v or w.
template <int QL> __device__ __forceinline__ float sum_states(float v0, float v1, float w0, float w1, int lane) {
  const bool hi = lane & 1, sec = lane & 2;
  const float p = (hi ? v1 : v0) + __shfl_xor_sync(~0u, hi ? v0 : v1, 1);
  const float q = (hi ? w1 : w0) + __shfl_xor_sync(~0u, hi ? w0 : w1, 1);
  float r = (sec ? q : p) + __shfl_xor_sync(~0u, sec ? p : q, 2);
  if constexpr (QL == 8) r += __shfl_xor_sync(~0u, r, 4);               // two lanes have the same sum
  return r;
}

// Where a block works: blocks of one sequence and segment lie side by side, as they read the same b and c
struct Place { int b, seg, g, tile, c0, valid, ch0; };
template <int CT> __device__ __forceinline__ Place place_of(const Args& a, unsigned i) {
  Place p;
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

template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}

// b or c of a tile: PER times four states of a token a thread
template <typename T, int NP> struct Coeffs {
  static constexpr int PER = TT * NP / 4 / THREADS, WORDS = (int)sizeof(T);           // words of four states
  uint32_t w[PER][WORDS];
  static __device__ __forceinline__ int token(int i) { return (threadIdx.x + i * THREADS) / (NP / 4); }
  static __device__ __forceinline__ int state(int i) { return (threadIdx.x + i * THREADS) % (NP / 4) * 4; }
  static __device__ __forceinline__ const T* at(const Group& r, const Place& p, int t0, int i) {
    return static_cast<const T*>(r.p) + p.b * r.sb + p.g * r.sg + (t0 + token(i)) * r.st + state(i);
  }
  // four states whose rows are in no such pieces, or end among them
  __device__ __forceinline__ void one_by_one(const T* from, int i, int live) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) w[i][j] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= live) continue;
      if constexpr (sizeof(T) == 4) w[i][j] = __ldg(reinterpret_cast<const uint32_t*>(from) + j);
      else w[i][j / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(from) + j) << (j & 1) * 16;
    }
  }
  __device__ __forceinline__ void fetch(const Group& r, const Place& p, int t0, int n, int states) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const T* from = at(r, p, t0, i);
      const int live = t0 + token(i) < n ? states - state(i) : 0;
      if (r.vec && live >= 4) {
        if constexpr (sizeof(T) == 4) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(from));
          w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
        } else {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(from));
          w[i][0] = u.x; w[i][1] = u.y;
        }
      } else {
        one_by_one(from, i, live);
      }
    }
  }
  __device__ __forceinline__ void put(float* sm) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float4 v;
      if constexpr (sizeof(T) == 4) {
        v = make_float4(__uint_as_float(w[i][0]), __uint_as_float(w[i][1]), __uint_as_float(w[i][2]), __uint_as_float(w[i][3]));
      } else {
        v = make_float4(__uint_as_float(w[i][0] << 16), __uint_as_float(w[i][0] & 0xffff0000u), __uint_as_float(w[i][1] << 16), __uint_as_float(w[i][1] & 0xffff0000u));
      }
      *reinterpret_cast<float4*>(sm + 4 * (threadIdx.x + i * THREADS)) = v;
    }
  }
  // under way into a place of the thread's own in shared memory, and out of it
  __device__ __forceinline__ void ask(uint2* slot, const Group& r, const Place& p, int t0, int n, int states) {
    static_assert(sizeof(T) == 2, "float32 is fetched");
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const T* from = at(r, p, t0, i);
      const int live = t0 + token(i) < n ? states - state(i) : 0;
      if (r.vec && live >= 4) {
        copy_async<8>(slot + i * THREADS, from);
      } else {
        one_by_one(from, i, live);
        slot[i * THREADS] = make_uint2(w[i][0], w[i][1]);
      }
    }
  }
  __device__ __forceinline__ void take(const uint2* slot) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint2 u = slot[i * THREADS];
      w[i][0] = u.x; w[i][1] = u.y;
    }
  }
};

template <typename T, int CT, int PARTS = 1> struct Pieces {            // a thread's part of a tile (or of one of PARTS) of x, delta, z or a gradient
  static constexpr int E = Piece<T>::N, PPR = CT / E, ROWS = THREADS / PPR, SPAN = TT / PARTS, P = SPAN / ROWS;
  uint4 v[P];
  __device__ __forceinline__ void fetch(const Rows& r, const Place& p, int t0, int n) {
    const int col = threadIdx.x % PPR * E, row = threadIdx.x / PPR;
    const T* at = static_cast<const T*>(r.p) + p.b * r.sb + p.ch0 + col + (t0 + row) * r.st;
    if (r.vec && p.valid == CT && t0 + SPAN <= n) {                        // for the whole block alike
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(at + i * ROWS * r.st));
    } else {
#pragma unroll 1
      for (int i = 0; i < P; ++i) {
        const uint4 u = t0 + row + i * ROWS < n ? load_piece<T>(at + i * ROWS * r.st, p.valid - col, r.vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (j == i) v[j] = u;
      }
    }
  }
  // under way into a place of the thread's own in shared memory, and out of it
  __device__ __forceinline__ void ask(uint4* slot, const Rows& r, const Place& p, int t0, int n) {
    const int col = threadIdx.x % PPR * E, row = threadIdx.x / PPR;
    const T* at = static_cast<const T*>(r.p) + p.b * r.sb + p.ch0 + col + (t0 + row) * r.st;
    if (r.vec && p.valid == CT && t0 + SPAN <= n) {                        // for the whole block alike
#pragma unroll
      for (int i = 0; i < P; ++i) copy_async<16>(slot + i * THREADS, at + i * ROWS * r.st);
    } else {
#pragma unroll 1
      for (int i = 0; i < P; ++i)
        slot[i * THREADS] = t0 + row + i * ROWS < n ? load_piece<T>(at + i * ROWS * r.st, p.valid - col, r.vec) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void take(const uint4* slot) {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = slot[i * THREADS];
  }
  // into L2, so that fetch() waits less
  static __device__ __forceinline__ void ask(const Rows& r, const Place& p, int t0, int n) {
    const int col = threadIdx.x % PPR * E, row = threadIdx.x / PPR;
    if (threadIdx.x % (PPR < 8 ? PPR : 8) || col >= p.valid) return;        // a line of 128 bytes each
    const T* base = static_cast<const T*>(r.p) + p.b * r.sb + p.ch0 + col;
#pragma unroll
    for (int i = 0; i < P * PARTS; ++i) {
      const int t = t0 + row + i * ROWS;
      if (t >= 0 && t < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(base + t * r.st));
    }
  }
};

// A block's next tile while one is computed: two places in turn for a thread's pieces of x, delta and z and its states of b and c.  (float32 and more states fetch
// theirs when a tile begins: registers and shared memory are full.)
template <typename T, int S, int QL> struct Ahead {
  static constexpr bool USED = sizeof(T) == 2 && S == 4;
  static constexpr int P = Pieces<T, channels_of(QL)>::P, PER = Coeffs<T, QL * S>::PER;
  uint4 rows[2][3][P * THREADS];
  uint2 states[2][2][PER * THREADS];
  static constexpr size_t bytes() { return USED ? sizeof(Ahead) : 0; }
};

// A segment's part of y, or (SUMS) its own contribution to the state and the sum of its steps.
template <typename T, int S, int QL, bool SUMS>
__global__ void __launch_bounds__(THREADS, S == 4 ? 4 : 2)
scan_kernel(const Args a) {
  constexpr int NP = QL * S, CT = channels_of(QL);
  using Px = Pieces<T, CT>;
  constexpr int E = Px::E;
  // two rows and one more than a tile has: what the loop asks for ahead of its end.  y takes the place of s x.
  __shared__ __align__(16) float s_dt[TT + 2][CT], s_dx[TT + 1][CT], s_b[TT + 1][NP], s_c[TT + 1][NP], s_bias[CT], s_skip[CT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place p = place_of<CT>(a, blockIdx.x);
  pdl_wait();
  const int n = text_length(a, p.b);
  if (tid < CT) {
    s_bias[tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
    s_skip[tid] = a.skip && tid < p.valid ? a.skip[p.ch0 + tid] : 0.f;
  }
  const int cl = warp * (CT / 4) + lane / QL * 2, q0 = lane % QL * S;      // the thread's two channels and S states
  constexpr int H = S / 2;
  f32x2 h[2][H], A[2][H];
  const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
      float v[2], w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s = q0 + 2 * i + j;
        const bool real = cl + c < p.valid && s < a.states;
        const long long ch = p.ch0 + cl + c;
        v[j] = real ? rate(a.a[ch * a.states + s]) : 0.f;
        w[j] = 0.f;
        if (!SUMS && real) {
          if (a.segs > 1) w[j] = a.seg_state[(row_n + cl + c) * NP + s];
          else if (a.state_in) w[j] = a.state_in[((long long)p.b * a.dim + ch) * a.states + s];
        }
      }
      A[c][i] = f2_pack(v[0], v[1]);
      h[c][i] = f2_pack(w[0], w[1]);
    }
  }
  const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles, last = min(first + a.seg_tiles, total);
  const int used = min(last, (n + TT - 1) / TT);
  const int col = tid % Px::PPR * E, row = tid / Px::PPR;
  T* y = static_cast<T*>(a.y) + (long long)p.b * a.len * a.dim + p.ch0 + col;
  Px x, delta, z;
  Coeffs<T, NP> fb, fc;
  extern __shared__ __align__(16) unsigned char s_ahead[];
  constexpr bool AHEAD = Ahead<T, S, QL>::USED;
  auto& ahead = *reinterpret_cast<Ahead<T, S, QL>*>(s_ahead);
  auto ask = [&](int k) {
    if constexpr (AHEAD) {
      uint4* rows = &ahead.rows[k & 1][0][tid];
      uint2* states = &ahead.states[k & 1][0][tid];
      constexpr int R = Px::P * THREADS, C = Coeffs<T, NP>::PER * THREADS;
      x.ask(rows, a.x, p, k * TT, n);
      delta.ask(rows + R, a.delta, p, k * TT, n);
      fb.ask(states, a.b, p, k * TT, n, a.states);
      if constexpr (!SUMS) {
        if (a.z.p) z.ask(rows + 2 * R, a.z, p, k * TT, n);
        fc.ask(states + C, a.c, p, k * TT, n, a.states);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  auto fetch = [&](int k) {
    if constexpr (AHEAD) {
      const uint4* rows = &ahead.rows[k & 1][0][tid];
      const uint2* states = &ahead.states[k & 1][0][tid];
      constexpr int R = Px::P * THREADS, C = Coeffs<T, NP>::PER * THREADS;
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      x.take(rows);
      delta.take(rows + R);
      fb.take(states);
      if constexpr (!SUMS) {
        if (a.z.p) z.take(rows + 2 * R);
        fc.take(states + C);
      }
    } else {
      x.fetch(a.x, p, k * TT, n);
      delta.fetch(a.delta, p, k * TT, n);
      fb.fetch(a.b, p, k * TT, n, a.states);
      if constexpr (!SUMS) {
        if (a.z.p) z.fetch(a.z, p, k * TT, n);
        fc.fetch(a.c, p, k * TT, n, a.states);
      }
    }
  };
  f32x2 steps = 0;
  if (first < used) ask(first);
  __syncthreads();
  for (int k = first; k < used; ++k) {
    fetch(k);
    f32x2 h0[2][H], own[2][H], cum = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < H; ++i) { h0[c][i] = h[c][i]; own[c][i] = 0; }
    if (!SUMS && a.saves) {              // the state in front of the tile, for the gradient
      float* to = a.saves + (((long long)p.b * total + k) * a.dim + p.ch0 + cl) * NP + q0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (cl + c < p.valid) st_pairs<H>(to + c * NP, h[c]);
    }
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
    if (k + 1 < used) {
      if constexpr (AHEAD) {             // into the place that the tile before this one had
        ask(k + 1);
      } else {
        Px::ask(a.x, p, (k + 1) * TT, n);
        Px::ask(a.delta, p, (k + 1) * TT, n);
        if (!SUMS && a.z.p) Px::ask(a.z, p, (k + 1) * TT, n);
      }
    }
    {
      constexpr int U = 4;
      Token<H, false, !SUMS> next;
      const float *p_dt = &s_dt[0][cl], *p_dx = &s_dx[0][cl], *p_b = &s_b[0][q0], *p_c = &s_c[0][q0];
      float* p_y = &s_dx[(lane >> 1) & 1][cl + (lane & 1)];
      f32x2 dt = ld2(p_dt), dt_next = ld2(p_dt + CT), d_next[2][H];
      next.get(p_dx, nullptr, p_b, p_c);
      decays<H>(dt, A, d_next);
#pragma unroll 1
      for (int t0 = 0; t0 < TT; t0 += U) {
        float sum[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Token<H, false, !SUMS> now = next;
          f32x2 d[2][H], x[2];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < H; ++i) d[c][i] = d_next[c][i];
          next.get(p_dx + (u + 1) * CT, nullptr, p_b + (u + 1) * NP, p_c + (u + 1) * NP);
          cum = f2_add(cum, dt);
          dt = dt_next;
          dt_next = ld2(p_dt + (u + 2) * CT);
          decays<H>(dt, A, d_next);
          splat2(now.x, x);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            f32x2 y = 0;
#pragma unroll
            for (int i = 0; i < H; ++i) {
              const f32x2 fed = f2_mul(x[c], now.B[i]);
              own[c][i] = f2_fma(d[c][i], own[c][i], fed);
              if constexpr (!SUMS) {
                h[c][i] = f2_fma(d[c][i], h[c][i], fed);
                y = i ? f2_fma(h[c][i], now.C[i], y) : f2_mul(h[c][i], now.C[i]);
              }
            }
            sum[u][c] = both(y);
          }
        }
        if constexpr (!SUMS) {
#pragma unroll
          for (int u = 0; u < U; u += 2) p_y[u * CT] = sum_states<QL>(sum[u][0], sum[u][1], sum[u + 1][0], sum[u + 1][1], lane);
        }
        p_dt += U * CT; p_dx += U * CT; p_b += U * NP; p_c += U * NP; p_y += U * CT;
      }
    }
    // the carried state meets the tile's decays in one product, so that its error grows with the tiles, not with the tokens
    carry_pairs<H>(cum, A, h0, own);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < H; ++i) h[c][i] = h0[c][i];
    steps = f2_add(steps, cum);
    __syncthreads();
    if constexpr (!SUMS) {
      float skip[E];
      from_shared(s_skip + col, skip);
#pragma unroll
      for (int i = 0; i < Px::P; ++i) {
        const int t = k * TT + row + i * Px::ROWS;
        if (t >= a.len) continue;
        float f[E], u[E];
        from_shared(&s_dx[row + i * Px::ROWS][col], f);
        Piece<T>::get(x.v[i], u);
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = fmaf(skip[j], u[j], f[j]);
        if (a.z.p) {
          Piece<T>::get(z.v[i], u);
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
    for (int c = 0; c < 2; ++c)
      if (cl + c < p.valid) st_pairs<H>(a.seg_state + (row_n + cl + c) * NP + q0, h[c]);
    float f[2];
    f2_unpack(steps, f[0], f[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (lane % QL == 0 && cl + j < p.valid) a.seg_steps[row_n + cl + j] = f[j];
  } else {
    for (int t = max(used, first) * TT + row; t < min(last * TT, a.len); t += Px::ROWS) {      // behind the text
      const float f[E] = {};
      store_piece<T>(y + (long long)t * a.dim, f, p.valid - col, a.y_vec);
    }
    if (a.state_out && p.seg == a.segs - 1) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
          float f[2];
          f2_unpack(h[c][i], f[0], f[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (cl + c < p.valid && q0 + 2 * i + j < a.states) a.state_out[((long long)p.b * a.dim + p.ch0 + cl + c) * a.states + q0 + 2 * i + j] = f[j];
        }
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
  const float A = real ? rate(a[(long long)d * states + s]) : 0.f;
  float h = real && edge ? edge[((long long)b * dim + d) * states + s] : 0.f;
  // several segments' loads are under way together
  constexpr int U = 8;
  const long long step = reverse ? -(long long)dim : dim;
  long long at = ((long long)b * segs + (reverse ? segs - 1 : 0)) * dim + d;
  for (int k = 0; k < segs; k += U) {
    float own[U], decay[U], part[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      own[u] = k + u < segs ? seg_state[(at + u * step) * np + s] : 0.f;
      decay[u] = k + u < segs ? seg_steps[at + u * step] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      part[u] = part_of(A * decay[u]);
      decay[u] = ex2(part[u] * (A * decay[u]));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u < segs) {
        seg_state[(at + u * step) * np + s] = h;
        h = carry(part[u], decay[u], h, own[u]);
      }
    }
    at += U * step;
  }
}

// The contribution of a segment's outputs to the gradient of the state in front of it, and the sum of its steps.
template <typename T, int S, int QL>
__global__ void __launch_bounds__(THREADS, S == 4 ? 4 : 2)
back_sums_kernel(const Args a, const Grads g) {
  constexpr int NP = QL * S, CT = channels_of(QL);
  using Px = Pieces<T, CT>;
  constexpr int E = Px::E;
  __shared__ __align__(16) float s_dt[TT][CT], s_e[TT][CT], s_c[TT][NP], s_bias[CT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place p = place_of<CT>(a, blockIdx.x);
  pdl_wait();
  const int n = text_length(a, p.b);
  if (tid < CT) s_bias[tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
  const int cl = warp * (CT / 4) + lane / QL * 2, q0 = lane % QL * S;
  constexpr int H = S / 2;
  f32x2 G[2][H], A[2][H];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
      float v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s = q0 + 2 * i + j;
        v[j] = cl + c < p.valid && s < a.states ? rate(a.a[(long long)(p.ch0 + cl + c) * a.states + s]) : 0.f;
      }
      A[c][i] = f2_pack(v[0], v[1]);
      G[c][i] = 0;
    }
  }
  const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles;
  const int used = min(min(first + a.seg_tiles, total), (n + TT - 1) / TT);
  const int col = tid % Px::PPR * E, row = tid / Px::PPR;
  Px delta, dy, z;
  Coeffs<T, NP> fc;
  f32x2 steps = 0;
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
    f32x2 own[2][H], cum = 0;            // the tile's, as in the forward pass
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < H; ++i) own[c][i] = 0;
#pragma unroll 4
    for (int t = TT - 1; t >= 0; --t) {
      const f32x2 dt = ld2(&s_dt[t][cl]);
      f32x2 C[H], d[2][H], e[2];
      splat2(ld2(&s_e[t][cl]), e);
      ld_pairs<H>(&s_c[t][q0], C);
      decays<H>(dt, A, d);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < H; ++i) own[c][i] = f2_mul(d[c][i], f2_fma(e[c], C[i], own[c][i]));
      cum = f2_add(cum, dt);
    }
    carry_pairs<H>(cum, A, G, own);
    steps = f2_add(steps, cum);
    __syncthreads();
  }
  const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
  float f[2];
  f2_unpack(steps, f[0], f[1]);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (cl + c < p.valid) {
      st_pairs<H>(a.seg_state + (row_n + cl + c) * NP + q0, G[c]);
      if (lane % QL == 0) a.seg_steps[row_n + cl + c] = f[c];
    }
  }
}

template <int S, int QL> struct BackShared {
  static constexpr int NP = QL * S, CT = channels_of(QL), U = 4, FEW = few(QL * S), STEP = 32 / QL * NP + 16;      // STEP: steps side by side meet other banks
  // the loop forwards asks for two tokens more than the tile has: at its end there is other memory of this struct, which is not used
  float bias[2][CT];
  float dt[TT][CT], dx[TT][CT], e[TT][CT], y[TT][CT], q[TT][CT];       // dx becomes gb
  float b[TT][NP], c[TT][NP];
  float part[4][TT][NP];                 // db or dc of each warp's channels
  float mid[4][U * STEP];                // four steps of each pair of channels
  float aside[2][2][S > 4 ? 1 : THREADS][4];          // up to 16 states: each thread's in front of the tile's tokens 8 and 24; then 0 in the place of 24
  float behind[S][THREADS][2];           // the gradient of the state behind the tile
};

// Four steps' values of a warp's pairs of channels are added up through shared memory: half the instructions of shuffles
template <int S, int QL> __device__ __forceinline__ void put_channels(float* mid, const f32x2 (&v)[S / 2], int lane) {
  st_pairs<S / 2>(mid + lane / QL * (QL * S) + lane % QL * S, v);
}
template <int S, int QL> __device__ __forceinline__ void sum_channels(const float* mid, float* to, int lane) {    // to: four rows of NP
  constexpr int NP = QL * S, STEP = BackShared<S, QL>::STEP, C = 32 / QL;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < NP / 16; ++j) {
    const int id = lane + 32 * j, u = id / (NP / 2), at = id % (NP / 2) * 2;
    const float* from = mid + u * STEP + at;
    f32x2 v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = ld2(from + c * NP);
#pragma unroll
    for (int w = C / 2; w > 0; w /= 2)
#pragma unroll
      for (int c = 0; c < w; ++c) v[c] = f2_add(v[c], v[c + w]);
    *reinterpret_cast<f32x2*>(to + u * NP + at) = v[0];
  }
  __syncwarp();
}

// Gradients, a tile at a time from the last to the first.  With v_t = h_t c_t, e_t the gradient of sum c h, g_t that of h_t:
//   forwards   h_t again from the saved state in front of the tile: y and dc_t = sum_d h_t e_t; h in front of every eighth token is put aside
//   backwards  four tokens at a time, f_t = exp(s_t a) h_{t-1} of each from what was put aside, then g_t = c_t e_t + exp(s a)_{t+1} g_{t+1}:
//              gb_t = sum_n g_t b_t, db_t = sum_d g_t s x, and from w_t = g_t f_t both da = sum_t s_t w_t and sum_n a w_t, the part of the step's gradient beside gb_t x_t.
// w is one product of what belongs to its own token.  (w_{t+1} = w_t + g_t b_t s x - v_t e_t, v = c h, makes sum_n a w_t a running sum of scalars and saves the states, but
// what is left of it where a state fades fast, or beside a token that outweighs its neighbours, is the others' roundings: it was off by 1e-5 for a s = -50, by more than
// the gradient itself from -1e6 on.)
// Measured (bf16, 16 states, 16 x 2048 x 1536): 1459 us, the running sum took 1343.  Half of the tokens' h are computed once more on the way from one place to the next
// (73 us; places in front of more tokens do not fit, and those that fit gained nothing); the exps of the next tokens under way while some are computed: spills, 1700.
// With more than 16 states: in front of every fourth token, two tokens at a time.  What is put aside then goes through L2, 57 KB a block, and blocks beyond PLACES
// of them take one piece of work after another.
template <typename T, int S, int QL>
__global__ void __launch_bounds__(THREADS, back_blocks(QL * S))
back_kernel(const Args a, const Grads g, const unsigned work) {
  constexpr int NP = QL * S, CT = channels_of(QL);
  constexpr int PARTS = sizeof(T) / 2;   // float32's twice as many pieces are in registers one half after the other
  using Px = Pieces<T, CT, PARTS>;
  constexpr int E = Px::E;
  extern __shared__ __align__(16) unsigned char raw[];
  BackShared<S, QL>& sh = *reinterpret_cast<BackShared<S, QL>*>(raw);
  float* const far_aside = g.aside + (long long)blockIdx.x * (ASIDE * 2 * S * THREADS) + 4 * threadIdx.x;
  pdl_wait();
  for (unsigned item = blockIdx.x; item < work; item += gridDim.x) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Place p = place_of<CT>(a, item);
    const int n = text_length(a, p.b);
    if (tid < CT) {
      sh.bias[0][tid] = a.bias && tid < p.valid ? a.bias[p.ch0 + tid] : 0.f;
      sh.bias[1][tid] = a.skip && tid < p.valid ? a.skip[p.ch0 + tid] : 0.f;
    }
    const int cl = warp * (CT / 4) + lane / QL * 2, q0 = lane % QL * S;
    const long long row_n = ((long long)p.b * a.segs + p.seg) * a.dim + p.ch0;
    constexpr int H = S / 2;
    f32x2 G[2][H], A[2][H];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        float v[2], w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int s = q0 + 2 * i + j;
          const bool real = cl + c < p.valid && s < a.states;
          const long long ch = p.ch0 + cl + c;
          v[j] = real ? rate(a.a[ch * a.states + s]) : 0.f;
          w[j] = 0.f;
          if (real && a.segs > 1) w[j] = a.seg_state[(row_n + cl + c) * NP + s];
          else if (real && g.d_state_out) w[j] = g.d_state_out[((long long)p.b * a.dim + ch) * a.states + s];
        }
        A[c][i] = f2_pack(v[0], v[1]);
        G[c][i] = f2_pack(w[0], w[1]);
      }
    }
    const int total = (a.len + TT - 1) / TT, first = p.seg * a.seg_tiles, last = min(first + a.seg_tiles, total);
    const int used = min(last, (n + TT - 1) / TT);
    const int col = tid % Px::PPR * E, row = tid / Px::PPR;
    const long long out0 = (long long)p.b * a.len * a.dim + p.ch0 + col;
    T *dx = static_cast<T*>(g.dx) + out0, *dd = static_cast<T*>(g.d_delta) + out0, *dz = static_cast<T*>(g.dz) + out0;
    float sum = 0.f;                       // threads below CT: the gradient of a channel's skip, the next CT: of its delta_bias
    for (int t = max(used, first) * TT + row; t < min(last * TT, a.len); t += Px::ROWS) {       // behind the text
      const float f[E] = {};
      store_piece<T>(dx + (long long)t * a.dim, f, p.valid - col, g.vec);
      store_piece<T>(dd + (long long)t * a.dim, f, p.valid - col, g.vec);
      if (g.dz) store_piece<T>(dz + (long long)t * a.dim, f, p.valid - col, g.vec);
    }
    Px x, delta, z, dy;
    Coeffs<T, NP> fb, fc;
    __syncthreads();
    for (int k = used - 1; k >= first; --k) {
      fb.fetch(a.b, p, k * TT, n, a.states);
      fc.fetch(a.c, p, k * TT, n, a.states);
      const float* saved = a.saves + (((long long)p.b * total + k) * a.dim + p.ch0 + cl) * NP + q0;
      auto in_front = [&](f32x2 (&h)[2][H]) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < H; i += 2) {
            const ulonglong2 u = cl + c < p.valid ? __ldg(reinterpret_cast<const ulonglong2*>(saved + c * NP + 2 * i)) : make_ulonglong2(0, 0);
            h[c][i] = u.x; h[c][i + 1] = u.y;
          }
      };
      f32x2 h[2][H];
      in_front(h);
#pragma unroll 1
      for (int part = 0; part < TT; part += Px::SPAN) {
        x.fetch(a.x, p, k * TT + part, n);
        delta.fetch(a.delta, p, k * TT + part, n);
        dy.fetch(g.dy, p, k * TT + part, n);
        if (a.z.p) z.fetch(a.z, p, k * TT + part, n);
        float bias[E];
        from_shared(sh.bias[0] + col, bias);
#pragma unroll
        for (int i = 0; i < Px::P; ++i) {
          const int t = part + row + i * Px::ROWS;
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
      if (k > first) {
        Px::ask(a.x, p, (k - 1) * TT, n);
        Px::ask(a.delta, p, (k - 1) * TT, n);
        Px::ask(g.dy, p, (k - 1) * TT, n);
        if (a.z.p) Px::ask(a.z, p, (k - 1) * TT, n);
      }
      constexpr int U = BackShared<S, QL>::U, FEW = BackShared<S, QL>::FEW, STEP = BackShared<S, QL>::STEP;
      float* mid = sh.mid[warp];
      // h in front of token t, a multiple of PART: a thread's own loads and stores, 16 bytes each
      constexpr int PART = 2 * FEW;
      auto place = [&](int t, int c) {
        if constexpr (S > 4) return far_aside + (t / PART - 1) * (2 * S * THREADS) + c * (S * THREADS);
        // token 16's lies in the first half of q, in the warp's own columns: by the time that half gets its own numbers it has been used
        else return t == 16 ? &sh.q[c * 8 + lane / 4][warp * (CT / 4) + lane % 4 * 4] : sh.aside[t != 8][c][tid];
      };
      auto put_aside = [&](int t) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float* to = place(t, c);
#pragma unroll
          for (int i = 0; i < H; i += 2) *reinterpret_cast<ulonglong2*>(to + i / 2 * (4 * THREADS)) = make_ulonglong2(h[c][i], h[c][i + 1]);
        }
      };
      auto take_aside = [&](int t) {
        if (S > 4 && t == 0) { in_front(h); return; }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float* from = place(t, c);
#pragma unroll
          for (int i = 0; i < H; i += 2) {
            const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(from + i / 2 * (4 * THREADS));
            h[c][i] = u.x; h[c][i + 1] = u.y;
          }
        }
      };
      {
        Token<H, true, true> next;
        const float *p_dt = &sh.dt[0][cl], *p_dx = &sh.dx[0][cl], *p_e = &sh.e[0][cl], *p_b = &sh.b[0][q0], *p_c = &sh.c[0][q0];
        float* p_y = &sh.y[own_row][own_ch];
        f32x2 dt = ld2(p_dt), dt_next = ld2(p_dt + CT), d_next[2][H];
        next.get(p_dx, p_e, p_b, p_c);
        decays<H>(dt, A, d_next);
#pragma unroll 1
        for (int t0 = 0; t0 < TT; t0 += U) {
          float y[U][2];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (u == 0 && t0 > 0 && t0 % PART == 0) put_aside(t0);
            const Token<H, true, true> now = next;
            f32x2 d[2][H], hs[H], x[2], e[2];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < H; ++i) d[c][i] = d_next[c][i];
            next.get(p_dx + (u + 1) * CT, p_e + (u + 1) * CT, p_b + (u + 1) * NP, p_c + (u + 1) * NP);
            dt = dt_next;
            dt_next = ld2(p_dt + (u + 2) * CT);
            decays<H>(dt, A, d_next);
            splat2(now.x, x);
            splat2(now.e, e);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              f32x2 yy;
#pragma unroll
              for (int i = 0; i < H; ++i) {
                h[c][i] = f2_fma(d[c][i], h[c][i], f2_mul(x[c], now.B[i]));
                hs[i] = c ? f2_fma(h[c][i], e[c], hs[i]) : f2_mul(h[c][i], e[c]);
                yy = i ? f2_fma(h[c][i], now.C[i], yy) : f2_mul(h[c][i], now.C[i]);
              }
              y[u][c] = both(yy);
            }
            put_channels<S, QL>(mid + u * STEP, hs, lane);
          }
#pragma unroll
          for (int u = 0; u < U; u += 2) p_y[u * CT] = sum_states<QL>(y[u][0], y[u][1], y[u + 1][0], y[u + 1][1], lane);
          sum_channels<S, QL>(mid, &sh.part[warp][t0][0], lane);
          p_y += U * CT; p_dt += U * CT; p_dx += U * CT; p_e += U * CT; p_b += U * NP; p_c += U * NP;
        }
      }
      take_aside(TT - PART);
      __syncthreads();
      auto parts_to = [&](float* out) {
        const long long row = (long long)a.groups * NP;
        out += (((long long)p.tile * a.batch + p.b) * a.len + k * TT) * row + p.g * NP + tid % NP;
#pragma unroll
        for (int j = 0; j < TT * NP / THREADS; ++j) {
          const int i = tid + j * THREADS;
          if (k * TT + i / NP < n)
            out[i / NP * row] = ((&sh.part[0][0][0])[i] + (&sh.part[1][0][0])[i]) + ((&sh.part[2][0][0])[i] + (&sh.part[3][0][0])[i]);
        }
      };
      parts_to(g.part_c);
      f32x2 own[2][H], dA[2][H], cum = 0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < H; ++i) {
          *reinterpret_cast<f32x2*>(sh.behind[c * H + i][tid]) = G[c][i];
          own[c][i] = dA[c][i] = 0;
        }
      __syncthreads();
      {
        constexpr int LAST = (TT - U) * CT, LAST_N = (TT - U) * NP;
        const float *p_dt = &sh.dt[0][cl] + LAST, *p_e = &sh.e[0][cl] + LAST, *p_b = &sh.b[0][q0] + LAST_N, *p_c = &sh.c[0][q0] + LAST_N;
        const float* p_dx = &sh.dx[0][cl] + LAST;
        float* to = (own_row ? &sh.q[0][own_ch] : &sh.dx[0][own_ch]) + LAST;
        constexpr int HALVES = PART > U ? 2 : 1;
#pragma unroll 1
        for (int t1 = TT - U; t1 >= 0; t1 -= HALVES * U)
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          const int t0 = t1 - half * U;
#pragma unroll
          for (int u0 = U - FEW; u0 >= 0; u0 -= FEW) {
            f32x2 d[FEW][2][H], f[FEW][2][H];
            float gb[2][2], q[2][2];
            const bool second = PART > U ? half == 0 : u0 > 0;        // half of the part
            if (second) {
#pragma unroll
              for (int v = 0; v < FEW; ++v) {
                const int u = u0 - FEW + v;
                f32x2 x[2], B[H];
                decays<H>(ld2(p_dt + u * CT), A, d[0]);
                splat2(ld2(p_dx + u * CT), x);
                ld_pairs<H>(p_b + u * NP, B);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                  for (int i = 0; i < H; ++i) h[c][i] = f2_fma(d[0][c][i], h[c][i], f2_mul(x[c], B[i]));
              }
            }
#pragma unroll
            for (int v = 0; v < FEW; ++v) {
              const int u = u0 + v;
              f32x2 x[2], B[H];
              decays<H>(ld2(p_dt + u * CT), A, d[v]);
              splat2(ld2(p_dx + u * CT), x);
              ld_pairs<H>(p_b + u * NP, B);
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < H; ++i) {
                  f[v][c][i] = f2_mul(d[v][c][i], h[c][i]);
                  if (v < FEW - 1) h[c][i] = f2_fma(x[c], B[i], f[v][c][i]);
                }
            }
            if constexpr (S == 4) {
              if (t0 == 24) {                                              // its states have been used
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  if (cl + c < p.valid) copy_async<16>(sh.aside[1][c][tid], saved + c * NP);
                  else *reinterpret_cast<float4*>(sh.aside[1][c][tid]) = make_float4(0.f, 0.f, 0.f, 0.f);
                }
              }
              if (t0 == 8) asm volatile("cp.async.wait_all;" ::: "memory");
            }
            if (t0 + u0 > 0) take_aside(t0 + u0 - (second ? FEW : PART));  // under way meanwhile
#pragma unroll
            for (int v = FEW - 1; v >= 0; --v) {
              const int u = u0 + v;
              Token<H, true, true> now;
              now.get(p_dx + u * CT, p_e + u * CT, p_b + u * NP, p_c + u * NP);
              f32x2 gs[H], x[2], e[2], dt[2];
              const f32x2 steps = ld2(p_dt + u * CT);
              cum = f2_add(cum, steps);
              splat2(steps, dt);
              splat2(now.x, x);
              splat2(now.e, e);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                f32x2 bb, qq;
#pragma unroll
                for (int i = 0; i < H; ++i) {
                  const f32x2 fed = f2_fma(e[c], now.C[i], G[c][i]), w = f2_mul(fed, f[v][c][i]);
                  own[c][i] = f2_mul(d[v][c][i], f2_fma(e[c], now.C[i], own[c][i]));
                  gs[i] = c ? f2_fma(fed, x[c], gs[i]) : f2_mul(fed, x[c]);
                  bb = i ? f2_fma(fed, now.B[i], bb) : f2_mul(fed, now.B[i]);
                  qq = i ? f2_fma(w, A[c][i], qq) : f2_mul(w, A[c][i]);
                  dA[c][i] = f2_fma(dt[c], w, dA[c][i]);
                  G[c][i] = f2_mul(d[v][c][i], fed);
                }
                gb[v % 2][c] = both(bb);
                q[v % 2][c] = both(qq);
              }
              put_channels<S, QL>(mid + u * STEP, gs, lane);
              if (v % 2 == 0) {
                __syncwarp();                                              // all of the warp have read these tokens' s x
#pragma unroll
                for (int j = 0; j < 2; ++j) to[(u + j) * CT] = sum_states<QL>(gb[j][0], gb[j][1], q[j][0], q[j][1], lane);
              }
            }
          }
          sum_channels<S, QL>(mid, &sh.part[warp][t0][0], lane);
          to -= U * CT; p_dt -= U * CT; p_dx -= U * CT; p_e -= U * CT; p_b -= U * NP; p_c -= U * NP;
        }
      }
      // a tile's own sum first: 2048 tokens one by one lose half a digit
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (cl + c >= p.valid) continue;
        float* to = g.part_a + (row_n + cl + c) * NP + q0;
        if (k < used - 1) add_pairs<H>(to, dA[c]);
        else st_pairs<H>(to, dA[c]);
      }
      // as in the forward pass: the carried gradient meets the tile's decays once
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < H; ++i) G[c][i] = ld2(sh.behind[c * H + i][tid]);
      carry_pairs<H>(cum, A, G, own);
      __syncthreads();
      parts_to(g.part_b);
#pragma unroll 1
      for (int part = 0; part < TT; part += Px::SPAN) {
        x.fetch(a.x, p, k * TT + part, n);      // again: they would fill 32 registers meanwhile
        delta.fetch(a.delta, p, k * TT + part, n);
        if (a.z.p) {
          dy.fetch(g.dy, p, k * TT + part, n);
          z.fetch(a.z, p, k * TT + part, n);
        }
        float bias[E], skip[E];
        from_shared(sh.bias[0] + col, bias);
        from_shared(sh.bias[1] + col, skip);
#pragma unroll
        for (int i = 0; i < Px::P; ++i) {
          const int r = part + row + i * Px::ROWS, t = k * TT + r;
          const bool in = t < n;
          if (!in) {                         // for the sums
            const float zero[E] = {};
            to_shared(&sh.y[r][col], zero);
            to_shared(&sh.q[r][col], zero);
            if (t < a.len) {
              store_piece<T>(dx + (long long)t * a.dim, zero, p.valid - col, g.vec);
              store_piece<T>(dd + (long long)t * a.dim, zero, p.valid - col, g.vec);
              if (g.dz) store_piece<T>(dz + (long long)t * a.dim, zero, p.valid - col, g.vec);
            }
            continue;
          }
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
              o[j] = dout[j] * yy * s * (1.f + zz[j] * (1.f - s));
            }
            store_piece<T>(dz + (long long)t * a.dim, o, p.valid - col, g.vec);
          }
          from_shared(&sh.dx[r][col], gb);
          from_shared(&sh.dt[r][col], f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            o[j] = fmaf(f[j], gb[j], skip[j] * e[j]);
            e[j] *= u[j];
          }
          to_shared(&sh.y[r][col], e);
          store_piece<T>(dx + (long long)t * a.dim, o, p.valid - col, g.vec);
          from_shared(&sh.q[r][col], f);
          float d[E];
          Piece<T>::get(delta.v[i], d);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            o[j] = fmaf(gb[j], u[j], f[j] * LN2);          // a's unit was a factor of two
            if (a.softplus) o[j] *= sigmoid(d[j] + bias[j]);
          }
          to_shared(&sh.q[r][col], o);
          store_piece<T>(dd + (long long)t * a.dim, o, p.valid - col, g.vec);
        }
      }
      __syncthreads();
      if (tid < 2 * CT) {                  // a tile's own sums
        const float* from = tid < CT ? &sh.y[0][tid] : &sh.q[0][tid - CT];
        float v[4] = {};
#pragma unroll
        for (int r = 0; r < TT; r += 4)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += from[(r + j) * CT];
        sum += (v[0] + v[1]) + (v[2] + v[3]);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (cl + c >= p.valid) continue;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        float w[2];
        f2_unpack(G[c][i], w[0], w[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int s = q0 + 2 * i + j;
          if (used <= first) g.part_a[(row_n + cl + c) * NP + s] = 0.f;
          if (g.d_state_in && p.seg == 0 && s < a.states) g.d_state_in[((long long)p.b * a.dim + p.ch0 + cl + c) * a.states + s] = w[j];
        }
      }
    }
    if (tid < 2 * CT && tid % CT < p.valid) (tid < CT ? g.part_skip : g.part_bias)[row_n + tid % CT] = sum;
    __syncthreads();
  }
}

// The blocks' parts of the gradients of b, c and of the parameters, added in one order; those of the parameters, one for each sequence and segment, in 64 bits.
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
  auto total = [&](const float* from, long long step) {                  // eight at a time, whose loads are under way together
    double v = 0.0;
    for (int k = 0; k < parts; k += 8) {
      float eight = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) eight += k + j < parts ? from[(k + j) * step] : 0.f;
      v += eight;
    }
    return (float)v;
  };
  if (s < a.states) {
    if (g.da) g.da[d * a.states + s] = total(g.part_a + d * np + s, (long long)a.dim * np);
  } else {
    float* to = s == a.states ? g.d_skip : g.d_bias;
    if (to) to[d] = total((s == a.states ? g.part_skip : g.part_bias) + d, a.dim);
  }
}

// One token: four threads a channel, four of its states each at a time.
struct StepArgs {
  int batch, dim, states, groups, per_group, softplus;
  const void *x, *delta, *z, *b, *c;
  long long x_sb, d_sb, z_sb, b_sb, b_sg, c_sb, c_sg;
  const float *a, *skip, *bias;
  float* state; long long s_b;
  void* y;
};

template <typename T> __device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

constexpr int STEP_THREADS = 256, STEP_CHANNELS = STEP_THREADS / 4;      // of a block (two channels a thread: 26 us where one takes 20)

template <typename T, bool VEC>
__global__ void __launch_bounds__(STEP_THREADS)
step_kernel(const StepArgs a) {
  pdl_wait();
  const unsigned tiles = (a.dim + STEP_CHANNELS - 1) / STEP_CHANNELS;
  const long long b = blockIdx.x / tiles;
  const int part = threadIdx.x % 4, at = (int)(blockIdx.x % tiles) * STEP_CHANNELS + threadIdx.x / 4;
  const bool live = at < a.dim;
  const int d = live ? at : 0, grp = a.groups > 1 ? d / a.per_group : 0;
  float* state = a.state + b * a.s_b + (long long)d * a.states;
  const float* decay = a.a + (long long)d * a.states;
  const T *pb = static_cast<const T*>(a.b) + b * a.b_sb + grp * a.b_sg, *pc = static_cast<const T*>(a.c) + b * a.c_sb + grp * a.c_sg;
  float h[4], A[4], B[4], C[4];
  auto load = [&](int s) {
    load4(state + s, h);
    load4(decay + s, A);
    load4(pb + s, B);
    load4(pc + s, C);
  };
  if constexpr (VEC) {
    if (part * 4 < a.states) load(part * 4);                            // under way while the step is computed
  }
  const float x = lp::load1(static_cast<const T*>(a.x) + b * a.x_sb + d);
  const float z = a.z ? lp::load1(static_cast<const T*>(a.z) + b * a.z_sb + d) : 0.f;
  const float dt = step_of(lp::load1(static_cast<const T*>(a.delta) + b * a.d_sb + d) + (a.bias ? a.bias[d] : 0.f), a.softplus), dx = dt * x;
  float y = 0.f;
  if (live) {
    if constexpr (VEC) {
      for (int s = part * 4; s < a.states; s += 16) {
        if (s >= 16) load(s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[j] = fmaf(ex2(dt * rate(A[j])), h[j], dx * B[j]);
          y = fmaf(h[j], C[j], y);
        }
        *reinterpret_cast<float4*>(state + s) = make_float4(h[0], h[1], h[2], h[3]);
      }
    } else {
      for (int s = part; s < a.states; s += 4) {
        const float hh = fmaf(ex2(dt * rate(decay[s])), state[s], dx * lp::load1(pb + s));
        state[s] = hh;
        y = fmaf(hh, lp::load1(pc + s), y);
      }
    }
  }
  y += __shfl_xor_sync(~0u, y, 1);
  y += __shfl_xor_sync(~0u, y, 2);
  if (!live || part) return;
  if (a.skip) y = fmaf(a.skip[d], x, y);
  if (a.z) y *= z * sigmoid(z);
  st_from_float(static_cast<T*>(a.y) + b * a.dim + d, y);
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct Plan { int np, total, tiles, per_group, segs, seg_tiles; };
// The axis is cut into segments where sequences and channels alone are fewer blocks than one and a half times the SMs, into as many as run at once: what a
// segment adds to the state (its gradient) is then computed first, at the price of another exp for each token, channel and state.  With 144 blocks
// (6 x 2048 x 1536) cut: 265 us and 623 back; with 168, cut: 358 and 885, not cut: 356 and 1030; with 240, not cut: 375 and 1038, about what cut ones would take.
static Plan plan_of(int batch, int len, int dim, int states, int groups, bool backward) {
  Plan p;
  p.np = states <= 16 ? 16 : states <= 32 ? 32 : 64;
  p.total = (len + TT - 1) / TT;
  p.per_group = dim / groups;
  const int ct = channels_of(p.np == 64 ? 8 : 4);
  p.tiles = (p.per_group + ct - 1) / ct;
  const long long blocks = (long long)batch * groups * p.tiles, sms = m2_sm_count(), want = (backward ? back_blocks(p.np) : p.np == 16 ? 4 : 2) * sms;
  p.segs = 1;
  if (2 * blocks < 3 * sms && p.total >= 8) {
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
static long long work_of(const Plan& p, int batch, int groups) { return (long long)batch * p.segs * groups * p.tiles; }
static long long back_grid(const Plan& p, int batch, int groups) {
  const long long work = work_of(p, batch, groups);
  return p.np == 16 || work < PLACES ? work : PLACES;
}
static long long aside_floats(const Plan& p, int batch, int groups) { return p.np == 16 ? 0 : back_grid(p, batch, groups) * (ASIDE * 8 * THREADS * 2); }
static long long grad_floats(const Plan& p, int batch, int len, int dim, int groups) {
  return aside_floats(p, batch, groups) + seg_floats(p, batch, dim) + 2LL * p.tiles * batch * len * groups * p.np + (long long)batch * p.segs * dim * (p.np + 2);
}

template <typename T, int S, int QL> static int forward(const Args& a, const Plan& p, cudaStream_t st) {
  constexpr size_t smem = Ahead<T, S, QL>::bytes();
  const long long blocks = (long long)a.batch * p.segs * a.groups * p.tiles, size = (long long)a.batch * a.len * a.dim;
  if (p.segs > 1) {
    if (smem) M2_SMEM_ONCE((scan_kernel<T, S, QL, true>), smem);
    if (int rc = m2_launch("m2_selective_scan_fwd", size, scan_kernel<T, S, QL, true>, dim3((unsigned)blocks), THREADS, smem, st, a)) return rc;
    const long long n = (long long)a.batch * a.dim * p.np;
    if (int rc = m2_launch("m2_selective_scan_fwd", size, join_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a.a, a.seg_state, a.seg_steps,
                           a.state_in, a.batch, p.segs, a.dim, a.states, p.np, 0)) return rc;
  }
  if (smem) M2_SMEM_ONCE((scan_kernel<T, S, QL, false>), smem);
  return m2_launch("m2_selective_scan_fwd", size, scan_kernel<T, S, QL, false>, dim3((unsigned)blocks), THREADS, smem, st, a);
}

template <typename T, int S, int QL> static int backward(const Args& a, const Grads& g, const Plan& p, cudaStream_t st) {
  const long long blocks = (long long)a.batch * p.segs * a.groups * p.tiles, size = (long long)a.batch * a.len * a.dim;
  if (p.segs > 1) {
    if (int rc = m2_launch("m2_selective_scan_bwd", size, back_sums_kernel<T, S, QL>, dim3((unsigned)blocks), THREADS, 0, st, a, g)) return rc;
    const long long n = (long long)a.batch * a.dim * p.np;
    if (int rc = m2_launch("m2_selective_scan_bwd", size, join_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a.a, a.seg_state, a.seg_steps,
                           g.d_state_out, a.batch, p.segs, a.dim, a.states, p.np, 1)) return rc;
  }
  constexpr size_t smem = sizeof(BackShared<S, QL>);
  M2_SMEM_ONCE((back_kernel<T, S, QL>), smem);
  if (int rc = m2_launch("m2_selective_scan_bwd", size, back_kernel<T, S, QL>, dim3((unsigned)back_grid(p, a.batch, a.groups)), THREADS, smem, st, a, g, (unsigned)blocks)) return rc;
  const long long bc = ((long long)a.batch * a.len * a.groups * a.states + 255) / 256, par = ((long long)a.dim * (a.states + 2) + 255) / 256;
  return m2_launch("m2_selective_scan_bwd", size, finish_kernel<T>, dim3((unsigned)(bc + par)), 256, 0, st, a, g, p.np, (unsigned)bc);
}

static bool in_pieces(const void* p, long long sb, long long st, int per_group, int size) {
  return m2_aligned(p, 16) && sb * size % 16 == 0 && st * size % 16 == 0 && (long long)per_group * size % 16 == 0;
}

static int check(const char* name, const m2_selective_scan_args& g, Args& a, Plan& p, bool backward) {
  M2_REQUIRE(g.batch >= 0 && g.seq_len >= 0 && g.dim >= 1 && g.states >= 1 && g.groups >= 1 && g.dim % g.groups == 0, M2_ERR_ARG,
             "%s: %d sequences of %d tokens, %d channels, %d states, %d groups", name, g.batch, g.seq_len, g.dim, g.states, g.groups);
  M2_REQUIRE(g.states <= MAX_STATES, M2_ERR_UNSUPPORTED, "%s: %d states (at most %d)", name, g.states, MAX_STATES);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: tensors are float32 or bf16", name);
  M2_REQUIRE(g.seq_len <= 1 << 28 && g.dim <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: %d tokens of %d channels", name, g.seq_len, g.dim);
  p = plan_of(g.batch, g.seq_len, g.dim, g.states, g.groups, backward);
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
  auto fours = [&](const void* q, long long sb, long long st, long long sg) { return m2_aligned(q, 4 * size) && sb % 4 == 0 && st % 4 == 0 && sg % 4 == 0; };
  a.b = {g.b, g.b_sb, g.b_st, g.b_sg, fours(g.b, g.b_sb, g.b_st, g.b_sg)}; a.c = {g.c, g.c_sb, g.c_st, g.c_sg, fours(g.c, g.c_sb, g.c_st, g.c_sg)};
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
  return 4 * saves_floats(plan_of(batch, seq_len, dim, states, groups, false), batch, dim);
}

extern "C" long long m2_selective_scan_workspace(int batch, int seq_len, int dim, int states, int groups, int backward) {
  using namespace m2::ss;
  if (batch <= 0 || seq_len < 0 || dim <= 0 || states <= 0 || states > MAX_STATES || groups <= 0 || dim % groups) return 0;
  const Plan p = plan_of(batch, seq_len, dim, states, groups, backward != 0);
  return 4 * (backward ? grad_floats(p, batch, seq_len, dim, groups) : seg_floats(p, batch, dim));
}

#define M2_SS_DISPATCH(fn, ...)                                                                                            \
  (g.dtype == M2_F32 ? (p.np == 16 ? fn<float, 4, 4>(__VA_ARGS__) : p.np == 32 ? fn<float, 8, 4>(__VA_ARGS__) : fn<float, 8, 8>(__VA_ARGS__)) \
                     : (p.np == 16 ? fn<__nv_bfloat16, 4, 4>(__VA_ARGS__) : p.np == 32 ? fn<__nv_bfloat16, 8, 4>(__VA_ARGS__) : fn<__nv_bfloat16, 8, 8>(__VA_ARGS__)))

extern "C" int m2_selective_scan_fwd(const m2_selective_scan_args* args, void* stream) {
  using namespace m2::ss;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_selective_scan_fwd: args is NULL");
  const m2_selective_scan_args& g = *args;
  Args a;
  Plan p;
  if (int rc = check("m2_selective_scan_fwd", g, a, p, false)) return rc;
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
  if (int rc = check("m2_selective_scan_bwd", g, a, p, true)) return rc;
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
  // aside, part_a and seg_state on 16 bytes: multiples of that many floats
  const long long bc = (long long)p.tiles * g.batch * g.seq_len * g.groups * p.np, parts = (long long)g.batch * p.segs * g.dim;
  float* w = g.workspace;
  r.aside = w; w += aside_floats(p, g.batch, g.groups);
  r.part_a = w; w += parts * p.np;
  a.seg_state = w; a.seg_steps = w + parts * p.np; w += seg_floats(p, g.batch, g.dim);
  r.part_b = w; r.part_c = w + bc; r.part_skip = w + 2 * bc; r.part_bias = r.part_skip + parts;
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
  const long long blocks = (long long)g.batch * ((g.dim + STEP_CHANNELS - 1) / STEP_CHANNELS);
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
  auto fours = [&](const void* p, long long sb, long long sg, int bytes) { return m2_aligned(p, 4 * bytes) && sb % 4 == 0 && sg % 4 == 0; };
  const bool vec = g.states % 4 == 0 && fours(g.state, g.s_b, 0, 4) && fours(g.a, 0, 0, 4) && fours(g.b, g.b_sb, g.b_sg, size) && fours(g.c, g.c_sb, g.c_sg, size);
  const cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return m2_launch("m2_selective_scan_step", elements, kernel, dim3((unsigned)blocks), STEP_THREADS, 0, st, a); };
  if (g.dtype == M2_F32) return vec ? go(step_kernel<float, true>) : go(step_kernel<float, false>);
  return vec ? go(step_kernel<__nv_bfloat16, true>) : go(step_kernel<__nv_bfloat16, false>);
}
