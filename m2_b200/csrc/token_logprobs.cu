// Log probabilities of given tokens, entropy and the best alternatives of every row of logits, and the gradient with respect to
// the logits: what the loss of the reference's masked-LM head computes behind its decoder (bert/src/bert_layers.py,
// BertForMaskedLM.forward: CrossEntropyLoss over the masked positions), for any given token.
//
// With m = max x, s = sum exp(x_j - m), t = sum (x_j - m) exp(x_j - m):
//     log p_j = (x_j - m) - log s,      H = -sum p log p = log s - t / s
//     dx_j = sum_i g_i (1[j = id_i] - p_j) - g_H p_j (log p_j + H)     over the given token and the alternatives.
//
// Bound: one read of the logits (gradient: one read, one write).  Forward: every thread streams 16-byte pieces and keeps its own
// (m, s, t) in float32, rescaled when a piece raises m; one exp a value.  The alternatives are found without sorting: the k-th
// largest of 64 thread groups' maxima is a lower bound of the row's k-th largest value, so the few threads whose own maximum is not
// below it look at their values once more, collect what is not below it, and these are ranked among one another.  Rows with so many
// equal values that the list overflows are searched k times instead.
// Measured: 8192 x 30528 bf16 106 us (4.7 TB/s, one exp a value keeps the SFUs 60 % busy), with 5 alternatives 125, its gradient 184 to
// 198 us (5.1 to 5.4 TB/s); float32 164 us (6.1 TB/s), with 5 alternatives 188; one row of 30528 bf16 with 20 alternatives 9 us.
// Blocks of 128 threads rather than 256 (a row's start and end overlap with more other rows): 106 against 115 us.
#include "common.cuh"

namespace m2 {
namespace lp {

constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int GROUPS = 64;
constexpr int SHARE = THREADS / GROUPS;   // threads of a group
constexpr int MAX_TOP = 32;              // <= GROUPS
constexpr int CAND = 1024;               // candidates kept per block
constexpr int MAX_SPLIT = 8;             // blocks of a cluster that share a row
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr float LOWEST = -3.402823466e38f;
constexpr int ST_BAD_TARGET = 16;        // M2_DEV_BAD_INDEX

// Rows ld apart, or groups of them (texts of a batch whose last rows are left out, say): up to 2^27 rows, so that 32 bits divide them
struct Rows {
  const void* p; long long ld, ld_group; unsigned group;
  template <typename T> __device__ __forceinline__ const T* at(long long row) const {
    long long to = row * ld;
    if (group) {
      const unsigned g = (unsigned)row / group;
      to = g * ld_group + ((unsigned)row - g * group) * ld;
    }
    return static_cast<const T*>(p) + to;
  }
};

struct Args {
  Rows x;
  const long long* target;
  long long n; int vocab, top, split;
  long long ignore;
  float *logprob, *entropy, *stats, *top_lp;
  long long* top_id;
};

struct BwdArgs {
  Rows x;
  const long long* target;
  long long n; int vocab, top;
  long long ignore;
  const float *stats, *entropy;
  const long long* top_id;
  const float *g_lp, *g_h, *g_top;
  void* dx; long long ldd;
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T> struct Piece;      // 16 bytes of a row
template <> struct Piece<float> {
  static constexpr int N = 4;
  __device__ static void get(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ static uint4 put(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Order of the alternatives: larger value first, NaN before all, equal values (both zeros among them) by ascending id.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long rank_key(float v, int id) {      // larger is better
  return ((unsigned long long)order_key(v) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_id(unsigned long long k) { return (int)~(uint32_t)k; }

// Running (m, s, t) of exp(x - m); m starts at the lowest finite value, so that x - m is never inf - inf for -inf entries.  Distances are cut at -1e4, far beyond
// where exp is 0, so that no 0 * inf arises.
struct Stats { float m, s, t; };
__device__ __forceinline__ void rebase(Stats& a, float m) {         // to the maximum m >= a.m
  const float d = a.m - m, f = ex2(d * LOG2E);
  a.t = f * fmaf(fmaxf(d, -1e4f), a.s, a.t);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  return {m, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ void add_value(Stats& a, float f) {
  if (f > a.m) rebase(a, f);
  const float d = f - a.m, e = ex2(d * LOG2E);                      // -inf: d = -inf, e = 0; NaN stays NaN in s
  a.s += e;
  a.t = fmaf(fmaxf(d, -1e4f), e, a.t);
}
__device__ __forceinline__ float largest(const uint4& u, const float (&f)[4]) { return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])); }
__device__ __forceinline__ float largest(const uint4& u, const float (&f)[8]) {         // pairs of bf16 at once
  auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
  const __nv_bfloat162 m = __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w)));
  return fmaxf(__low2float(m), __high2float(m));
}
// the values of a 16-byte piece, two at a time
template <int N> __device__ __forceinline__ void add_piece(Stats& a, const uint4& u, const float (&f)[N]) {
  const float m = largest(u, f);
  if (m > a.m) rebase(a, m);
  const f32x2 back = f2_splat(-a.m);
  f32x2 s = f2_splat(0.f), t = s;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 d = f2_add(f2_pack(f[i], f[i + 1]), back);
    float d0, d1, x0, x1;
    f2_unpack(d, d0, d1);
    f2_unpack(f2_mul(d, f2_splat(LOG2E)), x0, x1);
    const f32x2 e = f2_pack(ex2(x0), ex2(x1));
    s = f2_add(s, e);
    t = f2_fma(f2_pack(fmaxf(d0, -1e4f), fmaxf(d1, -1e4f)), e, t);
  }
  float x, y;
  f2_unpack(s, x, y);
  a.s += x + y;
  f2_unpack(t, x, y);
  a.t += x + y;
}

// Elements [lo, hi) of a row as scalar ends and 16-byte pieces.
template <typename T> struct Span {
  const T* p;
  int lo, hi, head, pieces;              // [lo, lo + head) scalar, then pieces of N, then scalars up to hi
  __device__ Span(const T* row, int lo_, int hi_) : p(row), lo(lo_), hi(hi_) {
    constexpr int N = Piece<T>::N;
    head = (int)((16 - (reinterpret_cast<uintptr_t>(row + lo) & 15)) & 15) / (int)sizeof(T);
    if (head > hi - lo) head = hi - lo;
    pieces = (hi - lo - head) / N;
  }
  __device__ int body() const { return lo + head; }
  __device__ int tail() const { return lo + head + pieces * Piece<T>::N; }
  // f(value, id) for the scalar ends, one a thread
  template <typename F> __device__ void ends(F&& f) const {
    const int t = threadIdx.x;
    if (t < head) f(load1(p + lo + t), lo + t);
    const int i = tail() + t;
    if (i < hi) f(load1(p + i), i);
  }
};

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename V> __device__ __forceinline__ const V* in_cta(const V* p, uint32_t rank) {     // the same variable in another block
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return reinterpret_cast<const V*>(r);
}

struct Shared {
  Stats warp[WARPS];
  Stats mine;                            // this block's slice
  alignas(16) uint32_t group[GROUPS];
  float bound;
  int count;
  unsigned long long best[MAX_TOP];      // this block's k best, best first; 0 where there are fewer
  unsigned long long cand[CAND];
  unsigned long long found[WARPS];
};

// The k best of [lo, hi) into sh.best.  Called by all threads; vmax: the largest value that this thread saw (LOWEST if none), nan:
// whether it saw a NaN (or an infinity, which makes one in its sum).
template <typename T> __device__ void select_top(Shared& sh, const Span<T>& sp, int k, float vmax, bool nan) {
  constexpr int N = Piece<T>::N;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float g = vmax;
#pragma unroll
  for (int o = 1; o < SHARE; o <<= 1) g = fmaxf(g, __shfl_xor_sync(~0u, g, o));
  if (tid % SHARE == 0) sh.group[tid / SHARE] = order_key(g);
  if (tid < MAX_TOP) sh.best[tid] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  {                                      // a group's threads share the others: how many come before it
    constexpr int PER = GROUPS / SHARE;
    const int g = tid / SHARE, q = tid % SHARE;
    const uint32_t mine = sh.group[g];
    int above = 0;
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(sh.group + q * PER + i);
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) above += w[j] + (q * PER + i + j < g ? 1u : 0u) > mine;      // keys of maxima end below 2^32 - 1
    }
#pragma unroll
    for (int o = 1; o < SHARE; o <<= 1) above += __shfl_xor_sync(~0u, above, o);
    if (q == 0 && above == k - 1) sh.bound = key_value((unsigned long long)mine << 32);
  }
  __syncthreads();
  // a group without values, or with -inf alone, says LOWEST: then everything is a candidate
  const float bound = sh.bound <= LOWEST ? -__int_as_float(0x7f800000) : sh.bound;
  auto offer = [&](float v, int id) {
    if (!(v < bound)) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < CAND) sh.cand[at] = rank_key(v, id);
    }
  };
  const uint4* body = reinterpret_cast<const uint4*>(sp.p + sp.body());
  // few threads have a candidate among their values; the warp looks at those of such threads together, a piece a lane
  const bool mine = nan || !(vmax < bound);
  if (mine) sp.ends(offer);
  for (unsigned need = __ballot_sync(~0u, mine); need;) {
    constexpr int B = 4;                 // such threads at once
    int at[B];
#pragma unroll
    for (int x = 0; x < B; ++x) {
      at[x] = need ? warp * 32 + __ffs(need) - 1 + lane * THREADS : sp.pieces;
      need &= need - 1;
    }
    while (__any_sync(~0u, at[0] < sp.pieces)) {       // the first of them has the lowest places
      uint4 u[B];
#pragma unroll
      for (int x = 0; x < B; ++x)
        if (at[x] < sp.pieces) u[x] = __ldg(body + at[x]);
#pragma unroll
      for (int x = 0; x < B; ++x) {
        if (at[x] < sp.pieces) {
          float f[N];
          Piece<T>::get(u[x], f);
          float m = f[0];
#pragma unroll
          for (int j = 1; j < N; ++j) m = max_nan(m, f[j]);
          if (!(m < bound)) {
#pragma unroll
            for (int j = 0; j < N; ++j) offer(f[j], sp.body() + at[x] * N + j);
          }
        }
        at[x] += 32 * THREADS;
      }
    }
  }
  __syncthreads();
  const int count = sh.count;
  if (count <= CAND) {
    for (int c = tid; c < count; c += THREADS) {
      const unsigned long long mine = sh.cand[c];
      int above = 0;
      for (int i = 0; i < count; ++i) above += sh.cand[i] > mine;          // ids differ: no two are equal
      if (above < k) sh.best[above] = mine;
    }
    __syncthreads();
    return;
  }
  unsigned long long last = ~0ull;                                         // too many equal values: the next best, k times
  for (int r = 0; r < k; ++r) {
    unsigned long long top = 0;
    auto look = [&](float v, int id) {
      const unsigned long long q = rank_key(v, id);
      if ((q < last || r == 0) && q > top) top = q;    // a NaN at id 0 has the largest key there is
    };
    sp.ends(look);
    for (int i = tid; i < sp.pieces; i += THREADS) {
      float f[N];
      Piece<T>::get(body[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) look(f[j], sp.body() + i * N + j);
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long q = __shfl_xor_sync(~0u, top, o);
      top = q > top ? q : top;
    }
    if (lane == 0) sh.found[warp] = top;
    __syncthreads();
    top = 0;
    for (int w = 0; w < WARPS; ++w) top = sh.found[w] > top ? sh.found[w] : top;
    if (tid == 0) sh.best[r] = top;
    last = top;
    __syncthreads();
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
forward_kernel(const Args a) {
  constexpr int N = Piece<T>::N;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = a.split;
  pdl_wait();
  const long long row = blockIdx.x / split;
  const uint32_t part = split > 1 ? cta_rank() : 0;
  const T* x = a.x.at<T>(row);
  const long long target = a.target[row];
  if (target == a.ignore) {                                                // the whole cluster leaves
    if (part == 0) {
      if (tid == 0) {
        a.logprob[row] = 0.f;
        a.entropy[row] = 0.f;
        if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.f;
      }
      if (tid < a.top) { a.top_lp[row * a.top + tid] = 0.f; a.top_id[row * a.top + tid] = -1; }
    }
    return;
  }
  // slices of whole 128-byte lines' worth of ids
  const int per = ((a.vocab + split - 1) / split + 63) / 64 * 64;
  const int lo = min((int)part * per, a.vocab), hi = min(lo + per, a.vocab);
  const Span<T> sp(x, lo, hi);
  Stats st = {LOWEST, 0.f, 0.f};
  sp.ends([&](float v, int) { add_value(st, v); });
  const uint4* body = reinterpret_cast<const uint4*>(x + sp.body());
  // the next pieces are under way while these are summed
  constexpr int U = 4;
  uint4 now[U], next[U];
  auto fetch = [&](uint4 (&u)[U], int i) {
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (i + j * THREADS < sp.pieces) u[j] = __ldg(body + i + j * THREADS);
  };
  fetch(now, tid);
  for (int i = tid; i < sp.pieces; i += U * THREADS) {
    fetch(next, i + U * THREADS);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i + j * THREADS < sp.pieces) {
        float f[N];
        Piece<T>::get(now[j], f);
        add_piece<N>(st, now[j], f);
      }
      now[j] = next[j];
    }
  }
  const float vmax = st.m;
  const bool nan = st.s != st.s;
  for (int o = 16; o > 0; o >>= 1) {
    const Stats b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o), __shfl_xor_sync(~0u, st.t, o)};
    st = join(st, b);
  }
  if (lane == 0) sh.warp[warp] = st;
  __syncthreads();
  if (tid == 0) {
    st = sh.warp[0];
    for (int w = 1; w < WARPS; ++w) st = join(st, sh.warp[w]);
    sh.mine = st;
  }
  if constexpr (TOP) select_top<T>(sh, sp, a.top, vmax, nan);
  if (split > 1) cluster_barrier(); else __syncthreads();
  if (part == 0) {
    st = sh.mine;
    for (int r = 1; r < split; ++r) st = join(st, *in_cta(&sh.mine, r));
    const float log_s = logf(st.s);
    const bool none = st.s == 0.f;                                         // every logit is -inf
    const float minus_inf = -__int_as_float(0x7f800000);
    auto logp = [&](float v) { return none ? minus_inf : (v - st.m) - log_s; };
    if (tid == 0) {
      const bool good = target >= 0 && target < a.vocab;
      if (!good) atomicOr(&m2_dev_status_word, ST_BAD_TARGET);
      a.logprob[row] = good ? logp(load1(x + target)) : __int_as_float(0x7fffffff);
      a.entropy[row] = none ? 0.f : log_s - st.t / st.s;
      if (a.stats) {
        a.stats[2 * row] = st.m;
        a.stats[2 * row + 1] = none ? -minus_inf : log_s;                  // +inf: every probability is 0
      }
    }
    if constexpr (TOP) {
      if (split == 1) {
        if (tid < a.top) {
          const unsigned long long q = sh.best[tid];
          a.top_lp[row * a.top + tid] = logp(key_value(q));
          a.top_id[row * a.top + tid] = key_id(q);
        }
      } else {                                                             // k best of `split` sorted lists
        const int n = split * a.top;
        for (int c = tid; c < n; c += THREADS) sh.cand[c] = in_cta(sh.best, c / a.top)[c % a.top];
        __syncthreads();
        for (int c = tid; c < n; c += THREADS) {
          const unsigned long long q = sh.cand[c];
          int above = 0;
          for (int o = 0; o < n; ++o) above += sh.cand[o] > q;
          if (q != 0 && above < a.top) {
            a.top_lp[row * a.top + above] = logp(key_value(q));
            a.top_id[row * a.top + above] = key_id(q);
          }
        }
      }
    }
  }
  if (split > 1) cluster_barrier();                                        // the other blocks' memory was read
}

constexpr int BWD_PIECES = 8;            // a thread's pieces

template <typename T>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const BwdArgs a, int slices) {
  constexpr int N = Piece<T>::N;
  const long long row = blockIdx.x / slices;
  const int slice = (int)(blockIdx.x % slices);
  constexpr int per = THREADS * BWD_PIECES * N;
  const int lo = slice * per, hi = min(lo + per, a.vocab);
  T* dx = static_cast<T*>(a.dx) + row * a.ldd;
  const int tid = threadIdx.x;
  const long long target = a.target[row];
  if (target == a.ignore) {              // nothing is read: 8192 x 30528 bf16, 85 % of the rows ignored, 101 us; reading them took 183
    const Span<T> z(dx, lo, hi);
    if (tid < z.head) st_from_float(dx + lo + tid, 0.f);
    if (z.tail() + tid < hi) st_from_float(dx + z.tail() + tid, 0.f);
    uint4* out = reinterpret_cast<uint4*>(dx + z.body());
#pragma unroll 4
    for (int i = tid; i < z.pieces; i += THREADS) out[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const T* x = a.x.at<T>(row);
  const bool good = target >= 0 && target < a.vocab;
  const float m = a.stats[2 * row], log_s = a.stats[2 * row + 1];
  const float g_h = a.g_h ? a.g_h[row] : 0.f, h = a.entropy[row];
  const float g_lp = good && a.g_lp ? a.g_lp[row] : 0.f;
  float g = g_lp;
  if (a.g_top) for (int i = 0; i < a.top; ++i) g += a.g_top[row * a.top + i];
  auto grad = [&](float v) {
    const float l = (v - m) - log_s, p = ex2(l * LOG2E);
    return -p * fmaf(g_h, fmaxf(l, -1e4f) + h, g);
  };
  const float c = -fmaf(g_h, h, g);      // -p (g_H (l + H) + g) as p (c - g_H l)
  auto grad2 = [&](float& v, float& w) {
    const f32x2 l = f2_add(f2_add(f2_pack(v, w), f2_splat(-m)), f2_splat(-log_s));
    float l0, l1, x0, x1;
    f2_unpack(l, l0, l1);
    f2_unpack(f2_mul(l, f2_splat(LOG2E)), x0, x1);
    const f32x2 k = f2_fma(f2_splat(-g_h), f2_pack(fmaxf(l0, -1e4f), fmaxf(l1, -1e4f)), f2_splat(c));
    f2_unpack(f2_mul(f2_pack(ex2(x0), ex2(x1)), k), v, w);
  };
  const Span<T> sp(x, lo, hi);
  sp.ends([&](float v, int id) { st_from_float(dx + id, grad(v)); });
  const uint4* body = reinterpret_cast<const uint4*>(x + sp.body());
  T* out = dx + sp.body();
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll 4
  for (int i = tid; i < sp.pieces; i += THREADS) {
    float f[N];
    Piece<T>::get(__ldg(body + i), f);
#pragma unroll
    for (int j = 0; j < N; j += 2) grad2(f[j], f[j + 1]);
    if (wide) {
      reinterpret_cast<uint4*>(out)[i] = Piece<T>::put(f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) st_from_float(out + i * N + j, f[j]);
    }
  }
  __syncthreads();
  // the ids that get a share of their own, written once more with everything in it
  if (tid <= a.top) {
    auto id_of = [&](int i) { return i == a.top ? (good ? target : -1ll) : a.top_id[row * a.top + i]; };
    auto g_of = [&](int i) { return i == a.top ? g_lp : (a.g_top ? a.g_top[row * a.top + i] : 0.f); };
    const long long id = id_of(tid);
    bool first = id >= lo && id < hi;
    for (int i = 0; first && i < tid; ++i) first = id_of(i) != id;
    if (first) {
      float own = 0.f;
      for (int i = tid; i <= a.top; ++i) own += id_of(i) == id ? g_of(i) : 0.f;
      const float v = load1(x + id);
      const bool none = log_s == __int_as_float(0x7f800000);
      st_from_float(dx + id, none ? 0.f : grad(v) + own);
    }
  }
}

template <typename T> static int launch_forward(const Args& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n * a.split));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = a.n * a.vocab <= M2_OVERLAP_ELEMENTS;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  const cudaError_t e = a.top ? cudaLaunchKernelEx(&cfg, forward_kernel<T, true>, a) : cudaLaunchKernelEx(&cfg, forward_kernel<T, false>, a);
  if (e != cudaSuccess) return m2_set_error(M2_ERR_CUDA, "launch of m2_token_logprobs_fwd failed: %s", cudaGetErrorString(e));
  ++m2_launch_count();
  return M2_OK;
}

static int check(const char* name, const void* x, long long ld, long long group, long long ld_group, const void* target, long long n, int vocab, int top, int dtype) {
  M2_REQUIRE(group >= 0 && group <= 1 << 27 && ld_group >= 0, M2_ERR_ARG, "%s: groups of %lld rows, %lld apart", name, group, ld_group);
  M2_REQUIRE(n >= 0 && vocab >= 1 && (ld >= 0 || n <= 1), M2_ERR_ARG, "%s: %lld rows of %d logits, %lld apart", name, n, vocab, ld);
  M2_REQUIRE(top >= 0 && top <= MAX_TOP && top <= vocab, M2_ERR_ARG, "%s: %d alternatives (0 .. %d, at most the %d logits)", name, top, MAX_TOP, vocab);
  M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: logits are float32 or bf16", name);
  M2_REQUIRE(vocab <= 1 << 28 && n <= 1 << 27, M2_ERR_UNSUPPORTED, "%s: %lld rows of %d logits are more than the grid takes", name, n, vocab);
  M2_REQUIRE(n == 0 || (x && target), M2_ERR_ARG, "%s: logits or targets are NULL", name);
  M2_REQUIRE(m2_aligned(x, dtype == M2_F32 ? 4 : 2) && m2_aligned(target, 8), M2_ERR_ALIGN, "%s: logits or targets are not aligned to their type", name);
  return M2_OK;
}

}  // namespace lp
}  // namespace m2

extern "C" int m2_token_logprobs_fwd(const m2_token_logprobs_args* args, void* stream) {
  using namespace m2::lp;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_token_logprobs_fwd: args is NULL");
  const m2_token_logprobs_args& g = *args;
  if (int rc = check("m2_token_logprobs_fwd", g.logits, g.ld, g.group, g.ld_group, g.targets, g.rows, g.vocab, g.top, g.dtype)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.logprob && g.entropy && (g.top == 0 || (g.top_logprob && g.top_id)), M2_ERR_ARG, "m2_token_logprobs_fwd: an output is NULL");
  Args a;
  a.x = {g.logits, g.ld, g.ld_group, (unsigned)g.group}; a.target = (const long long*)g.targets; a.n = g.rows; a.vocab = g.vocab; a.top = g.top; a.ignore = g.ignore_index;
  a.logprob = g.logprob; a.entropy = g.entropy; a.stats = g.stats; a.top_lp = g.top_logprob; a.top_id = (long long*)g.top_id;
  // a row is shared by the blocks of a cluster where the rows alone do not fill the GPU, each block with 4096 logits at least
  a.split = 1;
  while (a.split < MAX_SPLIT && g.rows * a.split < 2LL * m2_sm_count() && g.vocab / (a.split * 2) >= 4096) a.split *= 2;
  const cudaStream_t st = (cudaStream_t)stream;
  return g.dtype == M2_F32 ? launch_forward<float>(a, st) : launch_forward<__nv_bfloat16>(a, st);
}

extern "C" int m2_token_logprobs_bwd(const m2_token_logprobs_bwd_args* args, void* stream) {
  using namespace m2::lp;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_token_logprobs_bwd: args is NULL");
  const m2_token_logprobs_bwd_args& g = *args;
  if (int rc = check("m2_token_logprobs_bwd", g.logits, g.ld, g.group, g.ld_group, g.targets, g.rows, g.vocab, g.top, g.dtype)) return rc;
  if (g.rows == 0) return M2_OK;
  M2_REQUIRE(g.stats && g.entropy && g.d_logits && (g.top == 0 || g.top_id), M2_ERR_ARG, "m2_token_logprobs_bwd: a result of the forward pass or d_logits is NULL");
  M2_REQUIRE((g.ldd >= g.vocab || g.rows == 1) && m2_aligned(g.d_logits, g.dtype == M2_F32 ? 4 : 2), M2_ERR_ARG,
             "m2_token_logprobs_bwd: rows of d_logits overlap or are not aligned to their type");
  BwdArgs a;
  a.x = {g.logits, g.ld, g.ld_group, (unsigned)g.group}; a.target = (const long long*)g.targets; a.n = g.rows; a.vocab = g.vocab; a.top = g.top; a.ignore = g.ignore_index;
  a.stats = g.stats; a.entropy = g.entropy; a.top_id = (const long long*)g.top_id; a.g_lp = g.d_logprob; a.g_h = g.d_entropy;
  a.g_top = g.top ? g.d_top_logprob : nullptr; a.dx = g.d_logits; a.ldd = g.ldd;
  const int per = THREADS * BWD_PIECES * (g.dtype == M2_F32 ? 4 : 8);
  const int slices = (g.vocab + per - 1) / per;
  M2_REQUIRE(g.rows * slices <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_token_logprobs_bwd: %lld rows of %d logits are more than the grid takes", g.rows, g.vocab);
  const cudaStream_t st = (cudaStream_t)stream;
  if (g.dtype == M2_F32) backward_kernel<float><<<(unsigned)(g.rows * slices), THREADS, 0, st>>>(a, slices);
  else backward_kernel<__nv_bfloat16><<<(unsigned)(g.rows * slices), THREADS, 0, st>>>(a, slices);
  M2_LAUNCH_CHECK("m2_token_logprobs_bwd");
  ++m2_launch_count();
  return M2_OK;
}
