// Linear attention with a decay for each head, beside the long convolutions of m2_longconv_fwd (the reference mixes sequences with
// convolutions alone, bert/src/mm/monarch_mixer_sequence_mixer.py:100-154; this mixer's state has a fixed size):
//     S_t = l S_{t-1} + k_t v_t^T,        o_t = scale q_t^T S_t,        l = exp(log_decay[head])
// Chunks of C tokens: with T the state in front of a chunk and i, j counted inside it
//     o_i = scale ( sum_{j <= i} l^(i-j) (q_i . k_j) v_j + l^(i+1) q_i^T T ),      T' = l^C T + sum_j l^(C-1-j) k_j v_j^T.
// The gradients are the same scan with other roles (G: the gradient of the state, which runs backwards in time):
//     dq = scan(do, v, k) from T^T,     dk = reversed scan(v, do, q),     dv = reversed scan(k, q, do).
// Going backwards the given state G_end meets the last token undecayed, so there the first chunk's l^(i+1) and l^C are l^i and
// l^(C-1), and the gradient of the initial state is l times what is left at the front.
#include "common.cuh"

namespace m2 {
namespace la {

constexpr int C = 64;                    // tokens of a chunk
constexpr int DVT = 64;                  // columns of v that a block keeps
constexpr int MAX_D = 128;

struct Operand { const void* p; long long sb, st, sh; int div; };        // element (b, t, head / div, i)
struct Scan {
  Operand q, k, v;
  void* o; long long o_sb, o_st, o_sh;
  int o_f32;                             // o is float32 whatever the inputs are
  int batch, len, heads, dk, dv;
  const float* log_decay;
  const long long* lengths;              // NULL: all of `len`
  float scale;                           // of o
  int reverse;
  const float* init; float init_scale;   // NULL: zero
  float* final; float final_scale;       // NULL: not wanted; reversed scans multiply it by l too
  long long s_b, s_h, s_i, s_j;          // strides of init and final: row i of k, column j of v
  float* segments;                       // (batch * heads, n_seg, dk, dv): every segment's own sum, where n_seg > 1
  int n_seg, seg_chunks;
  int sums_only;                         // first of the two launches over segments
  int wide, o_wide;                      // rows of q, k and v (of o) start on 16-byte boundaries and are whole 16-byte pieces
};

__device__ __forceinline__ float power(float ld, int n) { return n == 0 ? 1.f : expf(ld * n); }
// l^n - 1: a state is carried as T + (l^n - 1) T, so that the factor's own rounding does not add up over the chunks of a long memory
__device__ __forceinline__ float power_m1(float ld, int n) { return n == 0 ? 0.f : expm1f(ld * n); }

__device__ __forceinline__ int seq_length(const Scan& a, int b) {
  if (!a.lengths) return a.len;
  const long long n = a.lengths[b];
  return n < 0 ? 0 : n > a.len ? a.len : (int)n;
}

// ---- float32: products on CUDA cores ---------------------------------------------------------------------------------------------------
// 256 threads as 16 x 16, each with 4 x 4 outputs of a 64 x 64 product; operands lie in shared memory with the summed index outside
// (two 16-byte loads for 16 products).
constexpr int LD = 68;                   // row pitch of the tiles: 16-byte rows, spread over the banks

__device__ __forceinline__ void mac(float (&acc)[4][4], const float4& a, const float4& b) {
  const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
}
__device__ __forceinline__ float4 f4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__global__ void __launch_bounds__(256)
scan_f32_kernel(const Scan a) {
  extern __shared__ float sm[];
  const int dkp = (a.dk + 15) / 16 * 16;
  float* qt = sm;                        // [dkp][LD]  (k index, token)
  float* kt = qt + dkp * LD;             // [dkp][LD]
  float* vs = kt + dkp * LD;             // [C][LD]    (token, column)
  float* pt = vs + C * LD;               // [C][LD]    (j, i)
  float* st = pt + C * LD;               // [dkp][LD]  (k index, column)
  float* pw = st + dkp * LD;             // [C + 1]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int bh = blockIdx.z, b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y, col0 = blockIdx.x * DVT;
  const int cols = min(DVT, a.dv - col0);
  const int n = seq_length(a, b);
  const float ld = a.log_decay[h];
  const float* q = static_cast<const float*>(a.q.p) + b * a.q.sb + (long long)(h / a.q.div) * a.q.sh;
  const float* k = static_cast<const float*>(a.k.p) + b * a.k.sb + (long long)(h / a.k.div) * a.k.sh;
  const float* v = static_cast<const float*>(a.v.p) + b * a.v.sb + (long long)(h / a.v.div) * a.v.sh + col0;
  const int seg_len = a.seg_chunks * C;
  const int at0 = min(seg * seg_len, a.len), at1 = min(at0 + seg_len, a.len);       // places of this segment, in scan order
  const bool last = n <= at1 && (n > at0 || (n == 0 && seg == 0));                  // holds the last token
  if (a.sums_only && (n <= at1 || seg == a.n_seg - 1)) return;                      // nobody reads the last segment's sum
  for (int i = tid; i <= C; i += 256) pw[i] = power(ld, i);
  const int first = a.reverse && a.init ? 1 : 0;                                    // the given state is one step younger
  float* own = a.segments ? a.segments + ((long long)bh * a.n_seg + seg) * a.dk * a.dv : nullptr;
  // the state in front of this segment
  if (!a.sums_only) {
    const float carry = power_m1(ld, seg_len), carry0 = power_m1(ld, seg_len - first);
    for (int e = tid; e < dkp * DVT; e += 256) {
      const int i = e / DVT, j = e - i * DVT;
      float s = 0.f;
      if (i < a.dk && j < cols && (n > at0 || last)) {
        if (a.init) s = a.init_scale * a.init[b * a.s_b + h * a.s_h + i * a.s_i + (col0 + j) * a.s_j];
        const float* p = a.segments + ((long long)bh * a.n_seg * a.dk + i) * a.dv + col0 + j;
        for (int r = 0; r < seg; ++r) s = fmaf(s, r ? carry : carry0, s) + p[(long long)r * a.dk * a.dv];
      }
      st[i * LD + j] = s;
    }
  } else {
    for (int e = tid; e < dkp * DVT; e += 256) st[e / DVT * LD + e % DVT] = 0.f;
  }
  for (int at = at0; at < min(at1, n); at += C) {
    const int m = min(C, n - at);                                                   // tokens of this chunk
    const int young = at == 0 ? first : 0;
    __syncthreads();
    for (int e = tid; e < dkp * C; e += 256) {                                      // tokens by the lane: no bank conflicts
      const int i = e / C, t = e - i * C;
      float x = 0.f, y = 0.f;
      if (t < m && i < a.dk) {
        const long long tok = a.reverse ? n - 1 - at - t : at + t;
        y = __ldg(k + tok * a.k.st + i);
        if (!a.sums_only) x = __ldg(q + tok * a.q.st + i);
      }
      qt[i * LD + t] = x;
      kt[i * LD + t] = y;
    }
    for (int e = tid; e < C * DVT; e += 256) {
      const int t = e / DVT, j = e - t * DVT;
      const long long tok = a.reverse ? n - 1 - at - t : at + t;
      vs[t * LD + j] = t < m && j < cols ? __ldg(v + tok * a.v.st + j) : 0.f;
    }
    __syncthreads();
    if (!a.sums_only) {
      float acc[4][4] = {};
      for (int i = 0; i < dkp; ++i) mac(acc, f4(kt + i * LD + ty * 4), f4(qt + i * LD + tx * 4));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float w[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) { const int gap = tx * 4 + y - (ty * 4 + x); w[y] = gap >= 0 ? acc[x][y] * pw[gap] : 0.f; }
        *reinterpret_cast<float4*>(pt + (ty * 4 + x) * LD + tx * 4) = make_float4(w[0], w[1], w[2], w[3]);
      }
      __syncthreads();
      float o[4][4] = {};
      for (int i = 0; i < dkp; ++i) mac(o, f4(qt + i * LD + ty * 4), f4(st + i * LD + tx * 4));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float f = pw[ty * 4 + x + 1 - young];
#pragma unroll
        for (int y = 0; y < 4; ++y) o[x][y] *= f;
      }
      const int jn = min(m, ty * 4 + 4);
      for (int j = 0; j < jn; ++j) mac(o, f4(pt + j * LD + ty * 4), f4(vs + j * LD + tx * 4));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = ty * 4 + x;
        if (t >= m) continue;
        const long long tok = a.reverse ? n - 1 - at - t : at + t;
        const long long to = b * a.o_sb + tok * a.o_st + h * a.o_sh + col0 + tx * 4;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if (tx * 4 + y >= cols) continue;
          static_cast<float*>(a.o)[to + y] = a.scale * o[x][y];
        }
      }
      __syncthreads();                                                              // st is read by all
    }
    const float keep = power_m1(ld, m - young);
    for (int i0 = ty * 4; i0 < dkp; i0 += 64) {
      float s[4][4] = {};
      for (int j = 0; j < m; ++j) {
        const float f = pw[m - 1 - j];
        const float4 kk = make_float4(f * kt[i0 * LD + j], f * kt[(i0 + 1) * LD + j], f * kt[(i0 + 2) * LD + j], f * kt[(i0 + 3) * LD + j]);
        mac(s, kk, f4(vs + j * LD + tx * 4));
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float* p = st + (i0 + x) * LD + tx * 4;
#pragma unroll
        for (int y = 0; y < 4; ++y) p[y] = fmaf(p[y], keep, p[y]) + s[x][y];
      }
    }
  }
  __syncthreads();
  if (a.sums_only) {
    for (int e = tid; e < a.dk * cols; e += 256) own[e / cols * a.dv + col0 + e % cols] = st[e / cols * LD + e % cols];
    return;
  }
  if (a.final && last) {
    const float f = a.final_scale * (a.reverse ? power(ld, n == 0 && a.init ? 0 : 1) : 1.f);
    for (int e = tid; e < a.dk * cols; e += 256) {
      const int i = e / cols, j = e - i * cols;
      a.final[b * a.s_b + h * a.s_h + i * a.s_i + (col0 + j) * a.s_j] = f * st[i * LD + j];
    }
  }
  // rows behind the last token are zero
  const int dead0 = max(at0, n);
  for (long long e = tid; e < (long long)(at1 - dead0) * cols; e += 256) {
    static_cast<float*>(a.o)[b * a.o_sb + (dead0 + e / cols) * a.o_st + h * a.o_sh + col0 + e % cols] = 0.f;
  }
}

// ---- bf16: products on the tensor cores ------------------------------------------------------------------------------------------------
// A block of 4 warps keeps the columns [col0, col0 + 64) of one (sequence, head) and walks over the chunks; warp w has rows
// 16 w .. 16 w + 15 of a chunk and rows w DK / 4 .. of the state, whose float32 values stay in its registers.  q, k and v tiles
// arrive by cp.async one chunk ahead.  A chunk's weights P = (q k^T) decay never leave the registers: the accumulators of q k^T are
// the operand of P v.  Every warp needs the whole state as an operand: it goes through shared memory as bf16, into the other one of
// two buffers, so that a chunk has a single block barrier.
//
// Why mma.sync: the scan is bound by its bytes.  A token and head of 64 + 64 channels moves 512 bytes, 11.6 ns of an SM's share of
// 6.5 TB/s, and takes 26 kFLOP (mean), 7 ns at the 555 TFLOP/s that mma.sync reaches on a B200; tiles of 64 tokens whose products
// feed each other through registers fit it, where tcgen05 would take every product through tensor and shared memory.
//
// The state is a sum over thousands of tokens, so nothing of it is rounded to bf16: l^(C-1-j) k_j goes into its product as two or
// (where the state is returned) three bf16 parts, 16 or 24 bits, and every chunk's sum starts from zero and is added in float32, as
// tensor cores cut their sums instead of rounding them.
constexpr int QK_LD(int dk) { return dk * 2; }             // bytes of a tile's row

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ float lo_of(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_of(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait0() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Byte of (row, 16-byte piece) of a tile: pieces are permuted inside 128 bytes, so that 8 rows of one piece lie in different banks.
template <int LDB> __device__ __forceinline__ int at_piece(int row, int piece) { return row * LDB + ((piece ^ (row & 7)) << 4); }

// C rows of up to LDB / 2 channels; rows from m on and channels from d on are zero.  Row r is token t0 + r dir.
template <int LDB> __device__ __forceinline__ void load_tile(char* tile, const __nv_bfloat16* p, long long st, long long t0, int dir, int m, int d, bool wide) {
  constexpr int PIECES = LDB / 16;
  for (int e = threadIdx.x; e < C * PIECES; e += 128) {
    const int r = e / PIECES, c = e - r * PIECES;
    const bool on = r < m && c * 8 < d;
    const __nv_bfloat16* src = p + (t0 + (long long)(on ? r : 0) * dir) * st + (on ? c * 8 : 0);
    char* dst = tile + at_piece<LDB>(r, c);
    if (wide) {
      cp16(saddr(dst), src, on);
    } else {
      uint32_t w[4] = {};
      if (on) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c * 8 + i < d) w[i >> 1] |= (uint32_t)__bfloat16_as_ushort(src[i]) << (16 * (i & 1));
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <int DK> struct MmaSmem {
  static constexpr int TILE = C * DK * 2, VT = C * DVT * 2, STAGE = 2 * TILE + VT, STATE = DK * DVT * 2;
  static constexpr int BYTES = 2 * STAGE + 2 * STATE + (C + 8) * 4;
};

template <int DK, int PARTS>
__global__ void __launch_bounds__(128)
scan_mma_kernel(const Scan a) {
  extern __shared__ __align__(128) char smem[];
  typedef MmaSmem<DK> L;
  constexpr int LK = DK * 2, LV = DVT * 2, MT = DK / 64, KS = DK / 16, NT = DVT / 8;
  float* pw = reinterpret_cast<float*>(smem + 2 * L::STAGE + 2 * L::STATE);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int bh = blockIdx.z, b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y, col0 = blockIdx.x * DVT;
  const int cols = min(DVT, a.dv - col0);
  const int n = seq_length(a, b);
  const float ld = a.log_decay[h];
  typedef __nv_bfloat16 T;
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.sb + (long long)(h / a.q.div) * a.q.sh;
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.sb + (long long)(h / a.k.div) * a.k.sh;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.sb + (long long)(h / a.v.div) * a.v.sh + col0;
  const int seg_len = a.seg_chunks * C;
  const int at0 = min(seg * seg_len, a.len), at1 = min(at0 + seg_len, a.len);       // places of this segment, in scan order
  const bool last = n <= at1 && (n > at0 || (n == 0 && seg == 0));                  // holds the last token
  if (a.sums_only && (n <= at1 || seg == a.n_seg - 1)) return;                      // nobody reads the last segment's sum
  const int first = a.reverse && a.init ? 1 : 0;                                    // the given state is one step younger
  const int end = min(at1, n), dir = a.reverse ? -1 : 1;
  auto token = [&](int at) { return (long long)(a.reverse ? n - 1 - at : at); };
  auto fetch = [&](int at, int stage) {
    char* s = smem + stage * L::STAGE;
    const int m = min(C, end - at);
    if (!a.sums_only) load_tile<LK>(s, q, a.q.st, token(at), dir, m, a.dk, a.wide);
    load_tile<LK>(s + L::TILE, k, a.k.st, token(at), dir, m, a.dk, a.wide);
    load_tile<LV>(s + 2 * L::TILE, v, a.v.st, token(at), dir, m, cols, a.wide);
    cp_commit();
  };
  if (at0 < end) fetch(at0, 0);
  for (int i = tid; i <= C; i += 128) pw[i] = power(ld, i);
  // the state in front of this segment: (mt, nt, e) is row (w MT + mt) 16 + g + 8 (e >> 1), column nt 8 + 2 t4 + (e & 1)
  float s[MT][NT][4];
  {
    const float carry = power_m1(ld, seg_len), carry0 = power_m1(ld, seg_len - first);
    const bool any = !a.sums_only && (n > at0 || last);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = (w * MT + mt) * 16 + g + 8 * (e >> 1), j = nt * 8 + 2 * t4 + (e & 1);
          float x = 0.f;
          if (any && i < a.dk && j < cols) {
            if (a.init) x = a.init_scale * a.init[b * a.s_b + h * a.s_h + i * a.s_i + (col0 + j) * a.s_j];
            const float* p = a.segments + ((long long)bh * a.n_seg * a.dk + i) * a.dv + col0 + j;
            for (int r = 0; r < seg; ++r) x = fmaf(x, r ? carry : carry0, x) + p[(long long)r * a.dk * a.dv];
          }
          s[mt][nt][e] = x;
        }
  }
  char* state = smem + 2 * L::STAGE;
  auto write_state = [&](char* to) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = (w * MT + mt) * 16 + g + 8 * e;
          *reinterpret_cast<uint32_t*>(to + at_piece<LV>(i, nt) + 4 * t4) = pack2(s[mt][nt][2 * e], s[mt][nt][2 * e + 1]);
        }
  };
  if (!a.sums_only) write_state(state);
  __syncthreads();                                                                  // pw
  // decays of this thread's weights: inside the diagonal 16 x 16 block, and l^(i-j+15) for the blocks before it
  float near[2][4], far[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int gap = g + 8 * (e >> 1) - (x * 8 + 2 * t4 + (e & 1));
      near[x][e] = gap >= 0 ? pw[gap] : 0.f;
      far[x][e] = pw[gap + 15];
    }
  int stage = 0;
  for (int at = at0; at < end; at += C, stage ^= 1) {
    const int m = min(C, end - at);
    const int young = at == 0 ? first : 0;
    cp_wait0();
    __syncthreads();
    if (at + C < end) fetch(at + C, stage ^ 1);
    char* qs = smem + stage * L::STAGE;
    const uint32_t q_at = saddr(qs), k_at = saddr(qs + L::TILE), v_at = saddr(qs + 2 * L::TILE), s_at = saddr(state + stage * L::STATE);
    const int r8 = lane & 7, half = (lane >> 3) & 1, quad = lane >> 4;
    if (!a.sums_only) {
      uint32_t qf[KS][4];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) ldsm(qf[ks], q_at + at_piece<LK>(w * 16 + (lane & 15), ks * 2 + quad));
      float o[NT][4] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          uint32_t f[4];
          ldsm_t(f, s_at + at_piece<LV>(ks * 16 + r8 + 8 * half, np * 2 + quad));
          mma(o[2 * np], qf[ks], f[0], f[1]);
          mma(o[2 * np + 1], qf[ks], f[2], f[3]);
        }
      const float d0 = pw[w * 16 + g + 1 - young], d1 = pw[w * 16 + g + 9 - young];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) { o[nt][0] *= d0; o[nt][1] *= d0; o[nt][2] *= d1; o[nt][3] *= d1; }
      for (int jb = 0; jb <= w; ++jb) {                                             // 16 tokens of k and v at a time
        float p[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t f[4];
          ldsm(f, k_at + at_piece<LK>(jb * 16 + r8 + 8 * quad, ks * 2 + half));
          mma(p[0], qf[ks], f[0], f[1]);
          mma(p[1], qf[ks], f[2], f[3]);
        }
        if (jb == w) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[x][e] = near[x][e] == 0.f ? 0.f : p[x][e] * near[x][e];
        } else {
          const float f = pw[16 * (w - jb) - 15];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[x][e] *= f * far[x][e];
        }
        const uint32_t pf[4] = {pack2(p[0][0], p[0][1]), pack2(p[0][2], p[0][3]), pack2(p[1][0], p[1][1]), pack2(p[1][2], p[1][3])};
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          uint32_t f[4];
          ldsm_t(f, v_at + at_piece<LV>(jb * 16 + r8 + 8 * half, np * 2 + quad));
          mma(o[2 * np], pf, f[0], f[1]);
          mma(o[2 * np + 1], pf, f[2], f[3]);
        }
      }
      if (a.o_f32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = w * 16 + g + 8 * (e >> 1);
          if (r >= m) continue;
          float* to = static_cast<float*>(a.o) + b * a.o_sb + token(at + r) * a.o_st + h * a.o_sh + col0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int j = nt * 8 + 2 * t4 + (e & 1);
            if (j < cols) to[j] = a.scale * o[nt][e];
          }
        }
      } else {                                                                      // through this warp's own rows of the q tile
        __syncwarp();
        const float c = a.scale;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          *reinterpret_cast<uint32_t*>(qs + at_piece<LK>(w * 16 + g, nt) + 4 * t4) = pack2(c * o[nt][0], c * o[nt][1]);
          *reinterpret_cast<uint32_t*>(qs + at_piece<LK>(w * 16 + g + 8, nt) + 4 * t4) = pack2(c * o[nt][2], c * o[nt][3]);
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = w * 16 + x * 4 + (lane >> 3), c8 = lane & 7;
          if (r >= m || c8 * 8 >= cols) continue;
          const uint4 u = *reinterpret_cast<const uint4*>(qs + at_piece<LK>(r, c8));
          T* to = static_cast<T*>(a.o) + b * a.o_sb + token(at + r) * a.o_st + h * a.o_sh + col0 + c8 * 8;
          if (a.o_wide) {
            *reinterpret_cast<uint4*>(to) = u;
          } else {
            const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c8 * 8 + i < cols) to[i] = __ushort_as_bfloat16((unsigned short)(ww[i >> 1] >> (16 * (i & 1))));
          }
        }
      }
    }
    // state: k^T (v weighted by age), the weight on k's fragment
    float acc[MT][NT][4] = {};
#pragma unroll
    for (int ks = 0; ks < C / 16; ++ks) {
      uint32_t kf[MT][PARTS][4];
      float wt[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) wt[x] = pw[max(0, m - 1 - (ks * 16 + 2 * t4 + (x & 1) + 8 * (x >> 1)))];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t f[4];
        ldsm_t(f, k_at + at_piece<LK>(ks * 16 + r8 + 8 * quad, (w * MT + mt) * 2 + half));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float lo = lo_of(f[x]) * wt[2 * (x >> 1)], hi = hi_of(f[x]) * wt[2 * (x >> 1) + 1];
#pragma unroll
          for (int y = 0; y < PARTS; ++y) {
            const uint32_t u = pack2(lo, hi);
            kf[mt][y][x] = u;
            lo -= lo_of(u);
            hi -= hi_of(u);
          }
        }
      }
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        uint32_t f[4];
        ldsm_t(f, v_at + at_piece<LV>(ks * 16 + r8 + 8 * half, np * 2 + quad));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int y = PARTS - 1; y >= 0; --y) {
            mma(acc[mt][2 * np], kf[mt][y], f[0], f[1]);
            mma(acc[mt][2 * np + 1], kf[mt][y], f[2], f[3]);
          }
      }
    }
    const float keep = power_m1(ld, m - young);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][nt][e] = fmaf(s[mt][nt][e], keep, s[mt][nt][e]) + acc[mt][nt][e];
    if (!a.sums_only && at + C < end) write_state(state + (stage ^ 1) * L::STATE);
  }
  const float f = a.sums_only ? 1.f : a.final_scale * (a.reverse ? power(ld, n == 0 && a.init ? 0 : 1) : 1.f);
  float* to = a.sums_only ? a.segments + ((long long)bh * a.n_seg + seg) * a.dk * a.dv : a.final && last ? a.final + b * a.s_b + h * a.s_h : nullptr;
  const long long s_i = a.sums_only ? a.dv : a.s_i, s_j = a.sums_only ? 1 : a.s_j;
  if (to) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = (w * MT + mt) * 16 + g + 8 * (e >> 1), j = nt * 8 + 2 * t4 + (e & 1);
          if (i < a.dk && j < cols) to[i * s_i + (col0 + j) * s_j] = f * s[mt][nt][e];
        }
  }
  if (a.sums_only) return;
  const int dead0 = max(at0, n);                                                    // rows behind the last token are zero
  for (long long e = tid; e < (long long)(at1 - dead0) * cols; e += 128) {
    const long long to = b * a.o_sb + (dead0 + e / cols) * a.o_st + h * a.o_sh + col0 + e % cols;
    if (a.o_f32) static_cast<float*>(a.o)[to] = 0.f; else static_cast<T*>(a.o)[to] = __float2bfloat16_rn(0.f);
  }
}

// Gradients of shared heads: out[b, t, h, i] = sum over the group's heads, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
group_sum_kernel(const float* part, T* out, long long rows, int kv_heads, int group, int d) {
  const long long total = rows * kv_heads * d;
  for (long long e = blockIdx.x * 256LL + threadIdx.x; e < total; e += gridDim.x * 256LL) {
    const long long head = e / d;        // (row, kv head)
    const float* p = part + head * group * d + (e - head * d);
    float s = 0.f;
    for (int g = 0; g < group; ++g) s += p[(long long)g * d];
    st_from_float(out + e, s);
  }
}

// ---- one token ---------------------------------------------------------------------------------------------------------------------------
// A block per (sequence, head): 16 column quads x 16 row groups of threads walk over the state once, reading and writing it, while
// q^T S is summed.  Bound by the state's bytes.
template <typename T>
__global__ void __launch_bounds__(256)
step_kernel(const m2_linear_attention_step_args a) {
  __shared__ float red[16][DVT + 4];
  __shared__ float qs[MAX_D], ks[MAX_D];
  const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads, col0 = blockIdx.y * DVT;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int cols = min(DVT, a.dv - col0), kvh = h / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh;
  const T* k = static_cast<const T*>(a.k) + b * a.k_sb + kvh * a.k_sh;
  const T* v = static_cast<const T*>(a.v) + b * a.v_sb + kvh * a.v_sh + col0;
  for (int i = tid; i < a.dk; i += 256) { qs[i] = ld_as_float(q + i); ks[i] = ld_as_float(k + i); }
  const float keep = power(a.log_decay[h], 1);
  float vv[4], o[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) vv[j] = tx * 4 + j < cols ? ld_as_float(v + tx * 4 + j) : 0.f;
  __syncthreads();
  float* s = a.state + b * a.s_b + h * a.s_h + col0 + tx * 4;
  const bool wide = a.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0 && a.s_b % 4 == 0 && a.s_h % 4 == 0;
  if (wide) {
    if (tx * 4 < cols) {
#pragma unroll 4
      for (int i = ty; i < a.dk; i += 16) {
        float4* p = reinterpret_cast<float4*>(s + (long long)i * a.dv);
        float4 u = *p;
        const float kk = ks[i], qq = qs[i];
        u.x = fmaf(keep, u.x, kk * vv[0]); u.y = fmaf(keep, u.y, kk * vv[1]); u.z = fmaf(keep, u.z, kk * vv[2]); u.w = fmaf(keep, u.w, kk * vv[3]);
        *p = u;
        o[0] = fmaf(qq, u.x, o[0]); o[1] = fmaf(qq, u.y, o[1]); o[2] = fmaf(qq, u.z, o[2]); o[3] = fmaf(qq, u.w, o[3]);
      }
    }
  } else {
    for (int i = ty; i < a.dk; i += 16)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (tx * 4 + j < cols) {
          float* p = s + (long long)i * a.dv + j;
          const float u = fmaf(keep, *p, ks[i] * vv[j]);
          *p = u;
          o[j] = fmaf(qs[i], u, o[j]);
        }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) red[ty][tx * 4 + j] = o[j];
  __syncthreads();
  if (tid < cols) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) t += red[r][tid];
    st_from_float(static_cast<T*>(a.o) + ((long long)b * a.heads + h) * a.dv + col0 + tid, a.scale * t);
  }
}

// Segments: where the blocks of all (sequence, head) pairs do not fill the GPU, a long axis is cut; every segment's own sum is made
// first (reading k and v once more) and the segments then run side by side.
static void segments_of(int batch, int heads, int dv, int len, int* n_seg, int* seg_chunks) {
  const long long blocks = (long long)batch * heads * ((dv + DVT - 1) / DVT), want = 2LL * m2_sm_count();
  const int chunks = (len + C - 1) / C;
  long long seg = (want + blocks - 1) / blocks;
  if (seg > chunks / 4) seg = chunks / 4;               // four chunks at least
  if (seg < 1) seg = 1;
  *seg_chunks = chunks ? (int)((chunks + seg - 1) / seg) : 1;
  *n_seg = chunks ? (chunks + *seg_chunks - 1) / *seg_chunks : 1;
}
static long long segment_floats(int batch, int heads, int dk, int dv, int len) {
  int n, c;
  segments_of(batch, heads, dv, len, &n, &c);
  return n > 1 ? (long long)batch * heads * n * dk * dv : 0;
}

// Rows in 16-byte pieces: cp.async copies them, and reads no more than them.
static bool in_pieces(const void* p, long long sb, long long st, long long sh, int d) {
  return m2_aligned(p, 16) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0 && d % 8 == 0;
}

template <int DK, int PARTS> static int launch_mma(const char* name, const Scan& a, dim3 grid, cudaStream_t st) {
  M2_SMEM_ONCE((scan_mma_kernel<DK, PARTS>), MmaSmem<DK>::BYTES);
  scan_mma_kernel<DK, PARTS><<<grid, 128, MmaSmem<DK>::BYTES, st>>>(a);
  M2_LAUNCH_CHECK(name);
  return M2_OK;
}

static int run_scan(const char* name, Scan a, int dtype, float* segments, cudaStream_t st) {
  segments_of(a.batch, a.heads, a.dv, a.len, &a.n_seg, &a.seg_chunks);
  a.segments = a.n_seg > 1 ? segments : nullptr;
  const dim3 grid((a.dv + DVT - 1) / DVT, a.n_seg, a.batch * a.heads);
  a.wide = in_pieces(a.q.p, a.q.sb, a.q.st, a.q.sh, a.dk) && in_pieces(a.k.p, a.k.sb, a.k.st, a.k.sh, a.dk) && in_pieces(a.v.p, a.v.sb, a.v.st, a.v.sh, a.dv);
  a.o_wide = in_pieces(a.o, a.o_sb, a.o_st, a.o_sh, a.dv);
  if (dtype == M2_BF16) {
    for (a.sums_only = a.n_seg > 1; a.sums_only >= 0; --a.sums_only) {
      const int rc = a.dk <= 64 ? (a.final ? launch_mma<64, 3>(name, a, grid, st) : launch_mma<64, 2>(name, a, grid, st))
                                : (a.final ? launch_mma<128, 3>(name, a, grid, st) : launch_mma<128, 2>(name, a, grid, st));
      if (rc) return rc;
    }
    return M2_OK;
  }
  const int dkp = (a.dk + 15) / 16 * 16;
  const size_t smem = ((size_t)(3 * dkp + 2 * C) * LD + C + 4) * sizeof(float);
  constexpr size_t most = ((size_t)(3 * MAX_D + 2 * C) * LD + C + 4) * sizeof(float);
  M2_SMEM_ONCE(scan_f32_kernel, most);
  for (a.sums_only = a.n_seg > 1; a.sums_only >= 0; --a.sums_only) {
    scan_f32_kernel<<<grid, 256, smem, st>>>(a);
    M2_LAUNCH_CHECK(name);
  }
  return M2_OK;
}

static int check(const char* name, int batch, int len, int heads, int kv_heads, int dk, int dv, int dtype, float scale) {
  M2_REQUIRE(batch >= 0 && len >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, M2_ERR_ARG, "%s: batch %d, %d steps, %d heads on %d key heads", name,
             batch, len, heads, kv_heads);
  M2_REQUIRE(dk >= 1 && dv >= 1 && dk <= MAX_D && dv <= MAX_D, M2_ERR_UNSUPPORTED, "%s: heads of 1 to %d channels, got %d and %d", name, MAX_D, dk, dv);
  M2_REQUIRE((long long)batch * heads <= 65535, M2_ERR_UNSUPPORTED, "%s: batch * heads up to 65535, got %d * %d", name, batch, heads);
  M2_REQUIRE(len <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: up to %d steps, got %d", name, 1 << 24, len);
  M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: q, k and v are float32 or bf16", name);
  M2_REQUIRE(scale != 0.f && scale - scale == 0.f, M2_ERR_ARG, "%s: scale %g", name, scale);
  return M2_OK;
}

static int check_operands(const char* name, const m2_linear_attention_args& g) {
  const size_t size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(g.log_decay && (g.seq_len == 0 || (g.q && g.k && g.v)), M2_ERR_ARG, "%s: q, k, v or log_decay is NULL", name);
  M2_REQUIRE(m2_aligned(g.q, size) && m2_aligned(g.k, size) && m2_aligned(g.v, size) && m2_aligned(g.lengths, 8), M2_ERR_ALIGN,
             "%s: a tensor is not aligned to its type", name);
  return M2_OK;
}

static Scan base_of(const m2_linear_attention_args& g) {
  Scan s = {};
  s.batch = g.batch; s.len = g.seq_len; s.heads = g.heads;
  s.log_decay = g.log_decay; s.lengths = (const long long*)g.lengths;
  return s;
}

}  // namespace la
}  // namespace m2

extern "C" long long m2_linear_attention_workspace(int batch, int seq_len, int heads, int kv_heads, int dk, int dv, int backward) {
  using namespace m2::la;
  if (batch < 1 || seq_len < 1 || heads < 1 || kv_heads < 1 || dk < 1 || dv < 1) return 0;
  long long floats = segment_floats(batch, heads, dk, dv, seq_len);
  if (backward) {
    const long long other = segment_floats(batch, heads, dv, dk, seq_len);
    floats = floats > other ? floats : other;
    if (heads != kv_heads) floats += (long long)batch * seq_len * heads * (dk + dv);
  }
  return floats * (long long)sizeof(float);
}

extern "C" int m2_linear_attention_fwd(const m2_linear_attention_args* args, void* stream) {
  using namespace m2::la;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_linear_attention_fwd: args is NULL");
  const m2_linear_attention_args& g = *args;
  if (int rc = check("m2_linear_attention_fwd", g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, g.scale)) return rc;
  if (g.batch == 0) return M2_OK;
  if (int rc = check_operands("m2_linear_attention_fwd", g)) return rc;
  M2_REQUIRE(g.o || g.seq_len == 0, M2_ERR_ARG, "m2_linear_attention_fwd: o is NULL");
  M2_REQUIRE(g.workspace || m2_linear_attention_workspace(g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, 0) == 0, M2_ERR_ARG,
             "m2_linear_attention_fwd: this shape needs a workspace");
  const int group = g.heads / g.kv_heads;
  const long long row = (long long)g.heads * g.dv;
  Scan s = base_of(g);
  s.q = {g.q, g.q_sb, g.q_st, g.q_sh, 1};
  s.k = {g.k, g.k_sb, g.k_st, g.k_sh, group};
  s.v = {g.v, g.v_sb, g.v_st, g.v_sh, group};
  s.o = g.o; s.o_sb = row * g.seq_len; s.o_st = row; s.o_sh = g.dv;
  s.dk = g.dk; s.dv = g.dv; s.scale = g.scale;
  s.init = g.state_in; s.init_scale = 1.f; s.final = g.state_out; s.final_scale = 1.f;
  s.s_j = 1; s.s_i = g.dv; s.s_h = (long long)g.dk * g.dv; s.s_b = s.s_h * g.heads;
  return run_scan("m2_linear_attention_fwd", s, g.dtype, g.workspace, (cudaStream_t)stream);
}

extern "C" int m2_linear_attention_bwd(const m2_linear_attention_args* args, const m2_linear_attention_grads* grads, void* stream) {
  using namespace m2::la;
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_linear_attention_bwd: args or grads is NULL");
  const m2_linear_attention_args& g = *args;
  const m2_linear_attention_grads& d = *grads;
  if (int rc = check("m2_linear_attention_bwd", g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, g.scale)) return rc;
  if (g.batch == 0) return M2_OK;
  if (int rc = check_operands("m2_linear_attention_bwd", g)) return rc;
  M2_REQUIRE(g.seq_len == 0 || (d.d_o && d.d_q && d.d_k && d.d_v), M2_ERR_ARG, "m2_linear_attention_bwd: d_o, d_q, d_k or d_v is NULL");
  M2_REQUIRE(m2_aligned(d.d_o, g.dtype == M2_F32 ? 4 : 2), M2_ERR_ALIGN, "m2_linear_attention_bwd: d_o is not aligned to its type");
  M2_REQUIRE(g.workspace || m2_linear_attention_workspace(g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, 1) == 0, M2_ERR_ARG,
             "m2_linear_attention_bwd: this shape needs a workspace");
  const int group = g.heads / g.kv_heads;
  const cudaStream_t st = (cudaStream_t)stream;
  const long long tokens = (long long)g.batch * g.seq_len;
  float* segments = g.workspace;
  float* part_k = nullptr;
  float* part_v = nullptr;
  if (group > 1) {                       // one gradient per head first, then their sums
    part_k = g.workspace;
    part_v = part_k + tokens * g.heads * g.dk;
    segments = part_v + tokens * g.heads * g.dv;
  }
  const Operand q = {g.q, g.q_sb, g.q_st, g.q_sh, 1}, k = {g.k, g.k_sb, g.k_st, g.k_sh, group}, v = {g.v, g.v_sb, g.v_st, g.v_sh, group};
  const Operand u = {d.d_o, d.o_sb, d.o_st, d.o_sh, 1};
  const long long s_h = (long long)g.dk * g.dv, s_b = s_h * g.heads;
  const long long row_k = (long long)g.heads * g.dk, row_v = (long long)g.heads * g.dv;
  Scan s = base_of(g);                   // dq = scan(do, v, k) from the transposed initial state
  s.q = u; s.k = v; s.v = k;
  s.o = d.d_q; s.o_sb = row_k * g.seq_len; s.o_st = row_k; s.o_sh = g.dk;
  s.dk = g.dv; s.dv = g.dk; s.scale = g.scale;
  s.init = g.state_in; s.init_scale = 1.f;
  s.s_b = s_b; s.s_h = s_h; s.s_i = 1; s.s_j = g.dv;
  if (int rc = run_scan("m2_linear_attention_bwd (d_q)", s, g.dtype, segments, st)) return rc;
  s = base_of(g);                        // dk = reversed scan(v, do, q)
  s.q = v; s.k = u; s.v = q; s.reverse = 1;
  s.o = group > 1 ? (void*)part_k : d.d_k; s.o_f32 = group > 1; s.o_sb = row_k * g.seq_len; s.o_st = row_k; s.o_sh = g.dk;
  s.dk = g.dv; s.dv = g.dk; s.scale = g.scale;
  s.init = d.d_state_out; s.init_scale = 1.f / g.scale;
  s.s_b = s_b; s.s_h = s_h; s.s_i = 1; s.s_j = g.dv;
  if (int rc = run_scan("m2_linear_attention_bwd (d_k)", s, g.dtype, segments, st)) return rc;
  s = base_of(g);                        // dv = reversed scan(k, q, do), and what is left of the state is the initial state's gradient
  s.q = k; s.k = q; s.v = u; s.reverse = 1;
  s.o = group > 1 ? (void*)part_v : d.d_v; s.o_f32 = group > 1; s.o_sb = row_v * g.seq_len; s.o_st = row_v; s.o_sh = g.dv;
  s.dk = g.dk; s.dv = g.dv; s.scale = g.scale;
  s.init = d.d_state_out; s.init_scale = 1.f / g.scale; s.final = d.d_state_in; s.final_scale = g.scale;
  s.s_b = s_b; s.s_h = s_h; s.s_i = g.dv; s.s_j = 1;
  if (int rc = run_scan("m2_linear_attention_bwd (d_v)", s, g.dtype, segments, st)) return rc;
  if (group > 1 && tokens > 0) {
    for (int w = 0; w < 2; ++w) {
      const float* part = w ? part_v : part_k;
      void* out = w ? d.d_v : d.d_k;
      const int width = w ? g.dv : g.dk;
      const long long blocks = (tokens * g.kv_heads * width + 255) / 256;
      const int grid = (int)(blocks < 16LL * m2_sm_count() ? blocks : 16LL * m2_sm_count());
      if (g.dtype == M2_F32) group_sum_kernel<float><<<grid, 256, 0, st>>>(part, static_cast<float*>(out), tokens, g.kv_heads, group, width);
      else group_sum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(part, static_cast<__nv_bfloat16*>(out), tokens, g.kv_heads, group, width);
    }
    M2_LAUNCH_CHECK("m2_linear_attention_bwd (shared heads)");
  }
  return M2_OK;
}

extern "C" int m2_linear_attention_step(const m2_linear_attention_step_args* args, void* stream) {
  using namespace m2::la;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_linear_attention_step: args is NULL");
  const m2_linear_attention_step_args& g = *args;
  if (int rc = check("m2_linear_attention_step", g.batch, 1, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, g.scale)) return rc;
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.q && g.k && g.v && g.log_decay && g.state && g.o, M2_ERR_ARG, "m2_linear_attention_step: a pointer is NULL");
  const size_t size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(m2_aligned(g.q, size) && m2_aligned(g.k, size) && m2_aligned(g.v, size) && m2_aligned(g.o, size) && m2_aligned(g.state, 4), M2_ERR_ALIGN,
             "m2_linear_attention_step: a tensor is not aligned to its type");
  const dim3 grid(g.batch * g.heads, (g.dv + DVT - 1) / DVT);
  const cudaStream_t st = (cudaStream_t)stream;
  if (g.dtype == M2_F32) step_kernel<float><<<grid, 256, 0, st>>>(g);
  else step_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(g);
  M2_LAUNCH_CHECK("m2_linear_attention_step");
  return M2_OK;
}
