// Dropout from a counter-based generator: y = kept x / (1 - p) (+ residual); the mask is computed anew wherever it is needed and never stored.
//
// Philox 4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): the key is the seed, the
// counter the number of a group of eight elements and the number of the call; each of the four words serves two elements, 16 bits each.  An element is
// kept if its 16 bits are not below p 2^16, so that p is a multiple of 2^-16 and 1 / (1 - p) is that p's.
// The reference drops out with torch's nn.Dropout (bert/src/bert_layers.py:487, 505).
// Bound: memory; ten rounds of two products, some 190 instructions in all, for eight elements.  Measured: 16 x 2048 x 1536 bf16 with a residual 57 us
// (302 MB, 5.3 TB/s), its gradient 42 (201 MB).  Two groups a thread and many short blocks took 70 and 51.
#include "common.cuh"

namespace m2 {
namespace drop {

constexpr int THREADS = 256;
constexpr int AN_SM = 5;                 // blocks of an SM

struct Args {
  const void *x, *residual;
  void* y;
  long long n, groups;
  unsigned threshold; float scale;
  const unsigned long long* seed;        // seed and number of the call, on the device, or these:
  unsigned long long key, call;
  int vec;
};

__device__ __forceinline__ uint4 philox(unsigned long long counter, unsigned long long call, unsigned long long key) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)call, c3 = (uint32_t)(call >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p = (unsigned long long)c0 * 0xD2511F53u, q = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

template <typename T> struct Eight {     // elements as they lie in memory
  static constexpr int E = lp::Piece<T>::N, P = 8 / E;
  uint4 v[P];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float w[E];
      lp::Piece<T>::get(v[i], w);
#pragma unroll
      for (int j = 0; j < E; ++j) f[i * E + j] = w[j];
    }
  }
  static __device__ __forceinline__ void put(T* p, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float w[E];
#pragma unroll
      for (int j = 0; j < E; ++j) w[j] = f[i * E + j];
      reinterpret_cast<uint4*>(p)[i] = lp::Piece<T>::put(w);
    }
  }
};

// y of a group from its numbers
template <bool RES> __device__ __forceinline__ void apply(const uint4& w, unsigned threshold, float scale, float (&f)[8], const float (&r)[8]) {
  const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = j & 1 ? bits[j / 2] >> 16 : bits[j / 2] & 0xffffu;
    const float v = b >= threshold ? f[j] * scale : 0.f;
    f[j] = RES ? v + r[j] : v;
  }
}

// A thread takes one group after another; the next group's elements are under way while this one's numbers are made.
template <typename T, bool RES>
__global__ void __launch_bounds__(THREADS, AN_SM)
dropout_kernel(const Args a) {
  pdl_wait();
  const unsigned long long key = a.seed ? a.seed[0] : a.key, call = a.seed ? a.seed[1] : a.call;
  const long long step = (long long)gridDim.x * THREADS, whole = a.vec ? a.n / 8 : 0;     // whole groups on 16 bytes
  const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  long long g = blockIdx.x * (long long)THREADS + threadIdx.x;
  Eight<T> next, next_r;
  if (g < whole) {
    next.load(x + g * 8);
    if constexpr (RES) next_r.load(res + g * 8);
  }
  for (; g < whole; g += step) {
    const Eight<T> now = next, now_r = next_r;
    if (g + step < whole) {
      next.load(x + (g + step) * 8);
      if constexpr (RES) next_r.load(res + (g + step) * 8);
    }
    const uint4 w = philox((unsigned long long)g, call, key);
    float f[8], r[8];
    now.get(f);
    if constexpr (RES) now_r.get(r);
    apply<RES>(w, a.threshold, a.scale, f, r);
    Eight<T>::put(y + g * 8, f);
  }
  for (; g < a.groups; g += step) {        // one by one: the last group, or all where a tensor is not on 16 bytes
    const uint4 w = philox((unsigned long long)g, call, key);
    float f[8], r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = g * 8 + j < a.n ? lp::load1(x + g * 8 + j) : 0.f;
      if constexpr (RES) r[j] = g * 8 + j < a.n ? lp::load1(res + g * 8 + j) : 0.f;
    }
    apply<RES>(w, a.threshold, a.scale, f, r);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (g * 8 + j < a.n) st_from_float(y + g * 8 + j, f[j]);
  }
}

}  // namespace drop
}  // namespace m2

extern "C" int m2_dropout(const m2_dropout_args* args, void* stream) {
  using namespace m2::drop;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_dropout: args is NULL");
  const m2_dropout_args& g = *args;
  M2_REQUIRE(g.n >= 0 && g.threshold >= 0 && g.threshold <= 65536, M2_ERR_ARG, "m2_dropout: %lld values, threshold %d of 65536", g.n, g.threshold);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "m2_dropout: tensors are float32 or bf16");
  if (g.n == 0) return M2_OK;
  M2_REQUIRE(g.x && g.y, M2_ERR_ARG, "m2_dropout: x or y is NULL");
  const int size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.x, size) && m2_aligned(g.y, size) && m2_aligned(g.residual, size) && m2_aligned(g.seed, 8), M2_ERR_ALIGN,
             "m2_dropout: a tensor is not aligned to its type");
  Args a = {g.x, g.residual, g.y, g.n, (g.n + 7) / 8, (unsigned)g.threshold, g.threshold < 65536 ? 65536.f / (65536 - g.threshold) : 0.f,
            (const unsigned long long*)g.seed, g.key, g.call, m2_aligned(g.x, 16) && m2_aligned(g.y, 16) && m2_aligned(g.residual, 16)};
  const long long need = (a.groups + THREADS - 1) / THREADS, most = (long long)AN_SM * m2_sm_count(), blocks = need < most ? need : most;
  const cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return m2_launch("m2_dropout", g.n, kernel, dim3((unsigned)blocks), THREADS, 0, st, a); };
  if (g.dtype == M2_F32) return g.residual ? go(dropout_kernel<float, true>) : go(dropout_kernel<float, false>);
  return g.residual ? go(dropout_kernel<__nv_bfloat16, true>) : go(dropout_kernel<__nv_bfloat16, false>);
}
