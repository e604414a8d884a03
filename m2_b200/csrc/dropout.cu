// Dropout from a counter-based generator: y = kept x / (1 - p) (+ residual); the mask is computed anew wherever it is needed and never stored.
//
// Philox 4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): the key is the seed, the
// counter the number of a group of eight elements and the number of the call; each of the four words serves two elements, 16 bits each.  An element is
// kept if its 16 bits are not below p 2^16, so that p is a multiple of 2^-16 and 1 / (1 - p) is that p's.
// The reference drops out with torch's nn.Dropout (bert/src/bert_layers.py:487, 505).
// Bound: memory; ten rounds of two products for eight elements.
#include "common.cuh"

namespace m2 {
namespace drop {

constexpr int THREADS = 256;
constexpr int UNROLL = 2;                // groups of eight of a thread

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

template <typename T> __device__ __forceinline__ void get8(const T* p, int valid, bool vec, float (&f)[8]) {
  constexpr int E = lp::Piece<T>::N;
  if (vec && valid >= 8) {
#pragma unroll
    for (int i = 0; i < 8; i += E) {
      float v[E];
      lp::Piece<T>::get(__ldcs(reinterpret_cast<const uint4*>(p + i)), v);
#pragma unroll
      for (int j = 0; j < E; ++j) f[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < valid ? lp::load1(p + j) : 0.f;
  }
}

template <typename T, bool RES>
__global__ void __launch_bounds__(THREADS)
dropout_kernel(const Args a) {
  constexpr int E = lp::Piece<T>::N;
  pdl_wait();
  const unsigned long long key = a.seed ? a.seed[0] : a.key, call = a.seed ? a.seed[1] : a.call;
  const long long first = blockIdx.x * (long long)(THREADS * UNROLL) + threadIdx.x;
  const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  float f[UNROLL][8], r[UNROLL][8];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const long long g = first + u * THREADS;
    const int valid = g < a.groups ? (int)min(8LL, a.n - g * 8) : 0;
    get8<T>(x + g * 8, valid, a.vec, f[u]);
    if constexpr (RES) get8<T>(res + g * 8, valid, a.vec, r[u]);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const long long g = first + u * THREADS;
    if (g >= a.groups) return;
    const int valid = (int)min(8LL, a.n - g * 8);
    const uint4 w = philox((unsigned long long)g, call, key);
    const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = j & 1 ? bits[j / 2] >> 16 : bits[j / 2] & 0xffffu;
      const float v = b >= a.threshold ? f[u][j] * a.scale : 0.f;
      f[u][j] = RES ? v + r[u][j] : v;
    }
    T* to = y + g * 8;
    if (a.vec && valid == 8) {
#pragma unroll
      for (int i = 0; i < 8; i += E) {
        float v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = f[u][i + j];
        __stcs(reinterpret_cast<uint4*>(to + i), lp::Piece<T>::put(v));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < valid) st_from_float(to + j, f[u][j]);
    }
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
  const long long blocks = (a.groups + THREADS * UNROLL - 1) / (THREADS * UNROLL);
  M2_REQUIRE(blocks <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_dropout: %lld values are more than the grid takes", g.n);
  const cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return m2_launch("m2_dropout", g.n, kernel, dim3((unsigned)blocks), THREADS, 0, st, a); };
  if (g.dtype == M2_F32) return g.residual ? go(dropout_kernel<float, true>) : go(dropout_kernel<float, false>);
  return g.residual ? go(dropout_kernel<__nv_bfloat16, true>) : go(dropout_kernel<__nv_bfloat16, false>);
}
