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

// Scans that run side by side in one launch (the three of a gradient): blockIdx.x counts the 64-column tiles of all of them, and those of
// one (sequence, head) after the other
struct Scans { Scan s[3]; int tiles[3]; };
template <bool MANY> __device__ __forceinline__ const Scan& pick_scan(const Scans& p, int& tile, int& bh) {
  const int all = p.tiles[0] + (MANY ? p.tiles[1] + p.tiles[2] : 0);
  // divisions by constants, which stay in uniform registers as the block index does
  const unsigned x = blockIdx.x;
  bh = all == 1 ? x : all == 2 ? x / 2 : all == 3 ? x / 3 : all == 4 ? x / 4 : all == 5 ? x / 5 : x / 6;
  tile = x - bh * all;
  int r = 0;
  if (MANY)
    while (r < 2 && tile >= p.tiles[r]) tile -= p.tiles[r++];
  return p.s[MANY ? r : 0];
}

__device__ __forceinline__ float power(float ld, int n) { return n == 0 ? 1.f : expf(ld * n); }
// l^n - 1: a state is carried as T + (l^n - 1) T, so that the factor's own rounding does not add up over the chunks of a long memory
__device__ __forceinline__ float power_m1(float ld, int n) { return n == 0 ? 0.f : expm1f(ld * n); }

// Where the state in front of a segment lies: what join_segments left, or (uncut) the given state; NULL: zero.  Behind a cut the given
// state is read by join_segments alone: it may be the memory that the last segment's state goes to.
struct Front {
  const float* p; long long s_i, s_j; float f;
  __device__ __forceinline__ Front(const Scan& a, int bh, int b, int h, int seg, int col0) {
    const bool cut = a.segments != nullptr;
    p = a.sums_only ? nullptr : cut ? a.segments + ((long long)bh * a.n_seg + seg) * a.dk * a.dv : a.init;
    s_i = cut ? a.dv : a.s_i;
    s_j = cut ? 1 : a.s_j;
    f = cut ? 1.f : a.init_scale;
    if (p) p += (cut ? 0 : b * a.s_b + h * a.s_h) + col0 * s_j;
  }
  __device__ __forceinline__ float operator()(int i, int j) const { return f * p[i * s_i + j * s_j]; }
};

__device__ __forceinline__ int seq_length(const Scan& a, int b) {
  if (!a.lengths) return a.len;
  const long long n = a.lengths[b];
  return n < 0 ? 0 : n > a.len ? a.len : (int)n;
}

// ---- float32: products on CUDA cores ---------------------------------------------------------------------------------------------------
// 256 threads as 16 x 16, each with 4 x 4 outputs of a 64 x 64 product; operands lie in shared memory with the summed index outside
// (two 16-byte loads for 16 products).  Bound by its instructions: 3.6 k FMAs and 1.9 k others a warp and chunk; 4 x 509 tokens of 12
// heads of 64, cut into four segments: 67 us (sums 23, scan 47 under a profiler).  Tensor cores would take six products of bf16 parts
// for each of these.
constexpr int LD = 68;                   // row pitch of the tiles: 16-byte rows, spread over the banks

__device__ __forceinline__ void mac(float (&acc)[4][4], const float4& a, const float4& b) {
  const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
}
__device__ __forceinline__ float4 f4(const float* p) { return *reinterpret_cast<const float4*>(p); }

template <bool MANY>
__global__ void __launch_bounds__(256)
scan_f32_kernel(const __grid_constant__ Scans scans) {
  extern __shared__ float sm[];
  int tile, bh;
  const Scan& a = pick_scan<MANY>(scans, tile, bh);
  pdl_wait();
  const int dkp = (a.dk + 15) / 16 * 16;
  float* qt = sm;                        // [dkp][LD]  (k index, token)
  float* kt = qt + dkp * LD;             // [dkp][LD]
  float* vs = kt + dkp * LD;             // [C][LD]    (token, column)
  float* pt = vs + C * LD;               // [C][LD]    (j, i)
  float* st = pt + C * LD;               // [dkp][LD]  (k index, column)
  float* pw = st + dkp * LD;             // [C + 1]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y, col0 = tile * DVT;
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
  const Front front(a, bh, b, h, seg, col0);
  for (int e = tid; e < dkp * DVT; e += 256) {
    const int i = e / DVT, j = e - i * DVT;
    st[i * LD + j] = front.p && i < a.dk && j < cols && (n > at0 || last) ? front(i, j) : 0.f;
  }
  for (int at = at0; at < min(at1, n); at += C) {
    const int m = min(C, n - at);                                                   // tokens of this chunk
    const int young = at == 0 ? first : 0;
    __syncthreads();
    if (a.wide) {                        // 16-byte pieces; a warp takes 8 tokens x 4 pieces, so that few lanes of a store share a bank
      const int lane = tid & 31;
#pragma unroll 4
      for (int e = tid >> 5; e < dkp / 2; e += 8) {
        const int t = (e & 7) * 8 + (lane & 7), i = (e >> 3) * 16 + (lane >> 3) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
        if (t < m && i < a.dk) {
          const long long tok = a.reverse ? n - 1 - at - t : at + t;
          y = __ldg(reinterpret_cast<const float4*>(k + tok * a.k.st + i));
          if (!a.sums_only) x = __ldg(reinterpret_cast<const float4*>(q + tok * a.q.st + i));
        }
        float* xs = qt + i * LD + t;
        float* ys = kt + i * LD + t;
        xs[0] = x.x; xs[LD] = x.y; xs[2 * LD] = x.z; xs[3 * LD] = x.w;
        ys[0] = y.x; ys[LD] = y.y; ys[2 * LD] = y.z; ys[3 * LD] = y.w;
      }
#pragma unroll
      for (int e = tid; e < C * DVT / 4; e += 256) {
        const int t = e / (DVT / 4), j = e % (DVT / 4) * 4;
        const long long tok = a.reverse ? n - 1 - at - t : at + t;
        *reinterpret_cast<float4*>(vs + t * LD + j) =
            t < m && j < cols ? __ldg(reinterpret_cast<const float4*>(v + tok * a.v.st + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    } else {
      for (int e = tid; e < dkp * C; e += 256) {                                    // tokens by the lane: no bank conflicts
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
    }
    __syncthreads();
    if (!a.sums_only) {
      float acc[4][4] = {};
#pragma unroll 8
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
      if (front.p || at > at0) {         // else the state is zero
#pragma unroll 8
        for (int i = 0; i < dkp; ++i) mac(o, f4(qt + i * LD + ty * 4), f4(st + i * LD + tx * 4));
      }
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
        float* op = static_cast<float*>(a.o) + to;
        if (a.o_wide) {
          if (tx * 4 < cols) *reinterpret_cast<float4*>(op) = make_float4(a.scale * o[x][0], a.scale * o[x][1], a.scale * o[x][2], a.scale * o[x][3]);
          continue;
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (tx * 4 + y < cols) op[y] = a.scale * o[x][y];
      }
      __syncthreads();                                                              // st and vs are read by all
    }
    for (int e = tid; e < C * DVT / 4; e += 256) {                                  // v by its age, l^(m-1-j)
      const int t = e / (DVT / 4), j = e % (DVT / 4) * 4;
      float4* p = reinterpret_cast<float4*>(vs + t * LD + j);
      const float f = pw[max(0, m - 1 - t)];
      const float4 u = *p;
      *p = make_float4(f * u.x, f * u.y, f * u.z, f * u.w);
    }
    __syncthreads();
    const float keep = power_m1(ld, m - young);
    for (int i0 = ty * 4; i0 < dkp; i0 += 64) {
      float s[4][4] = {};
      for (int j = 0; j < m; j += 4) {   // tokens behind the last one are zero in v
        float4 kk[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) kk[x] = f4(kt + (i0 + x) * LD + j);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          auto of = [&](const float4& u) { return y == 0 ? u.x : y == 1 ? u.y : y == 2 ? u.z : u.w; };
          mac(s, make_float4(of(kk[0]), of(kk[1]), of(kk[2]), of(kk[3])), f4(vs + (j + y) * LD + tx * 4));
        }
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
// the operand of P v.  Every warp needs the whole state as an operand: it goes through shared memory, written behind a barrier that
// all pass when they have read the one before.
//
// Nothing but o is rounded to bf16.  P and the state's copy that q meets are two bf16 parts of 8 bits each, 16 bits (one part each:
// o was 1.41 times as far from 64 bits as its own rounding takes it; 32 x 2048 tokens of 12 heads of 64 took 144 us, not 176, and
// 16 x 2048 of 12 heads of 128 262 and 535 back, not 320 and 676).  The state itself is a sum over thousands of tokens:
// l^(C-1-j) k_j goes into its product as three parts, all 24 bits of it, and every chunk's sum starts from zero and is added in
// float32, as tensor cores cut their sums instead of rounding them.  A gradient's state that goes nowhere but into those copies of
// 16 bits has two parts.  Forward there are always three: o has the same bits whether or not the state is asked for.
//
// Bound: a token and head of 64 + 64 channels moves 512 bytes, 64 of them 0.74 us of an SM's share of 6.5 TB/s; the products take
// 0.89 us (gradients 0.76) at the 555 TFLOP/s that mma.sync reaches on a B200.  What costs is the rest: loops are kept rolled, as a
// chunk unrolled (2.2 k instructions a warp) does not fit the SM's instruction cache and waited for it more than for anything else.
// The same scan on tcgen05 (chunks of 128, P and the state's parts through shared memory, five block barriers a chunk) took longer.
// Measured: 32 x 2048 tokens, 12 heads of 64: 176 us, 2.3 TB/s, the tensor pipe 55 % busy, 1.3 k instructions a warp and chunk, which
// 12 warps an SM issue at 41 % of its rate (registers and shared memory admit no more); 16 x 2048, 12 heads of 128: 320 us, the pipe
// 60 % busy, and its three scans back 676 us in one launch.  Heads of 65 to 127 channels do the work of 128: 80 take 322 us.
__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void stsm(uint32_t a, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ float lo_of(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_of(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
// The upper 8 bits of two values, as bf16, and what is left of them
__device__ __forceinline__ uint32_t cut_off(f32x2& z) {
  float l, g;
  f2_unpack(z, l, g);
  const uint32_t u = __float_as_uint(l), w = __float_as_uint(g);
  z = f2_fma(f2_pack(__uint_as_float(u & 0xffff0000u), __uint_as_float(w & 0xffff0000u)), f2_splat(-1.f), z);
  return __byte_perm(u, w, 0x7632);
}
__device__ __forceinline__ uint32_t pack_up(f32x2 z) {
  float l, g;
  f2_unpack(z, l, g);
  return pack2(l, g);
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait0() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Tiles are rows of 64 channels, 128 bytes, in 16-byte pieces; pieces are permuted so that 8 rows of one piece lie in different
// banks.  128 channels are two tiles.
constexpr int SUB = C * 128;
__device__ __forceinline__ uint32_t at_piece(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// What a thread copies of one operand: piece c of rows r0, r0 + 16, r0 + 32, r0 + 48 of every chunk
struct Copy {
  const __nv_bfloat16* p;                // of row r0 of the chunk at hand
  long long row16;                       // elements from one of its rows to the next; 4 of them from chunk to chunk
  int d;                                 // channels of the operand from this piece on
  __device__ __forceinline__ Copy(const void* base, long long at, long long st, int dir, int channels) {
    const int c = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    p = static_cast<const __nv_bfloat16*>(base) + at + (long long)r0 * dir * st + c * 8;
    row16 = 16 * dir * st;
    d = channels - c * 8;
  }
  // into the tile(s) at `tile`; rows from m on and channels beyond the operand's become zero
  template <int SUBS> __device__ __forceinline__ void load(uint32_t tile, int m, bool wide) {
    const int c = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    const uint32_t dst = tile + at_piece(r0, c);
    const __nv_bfloat16* src = p;
    if (wide) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + s * SUB + i * 2048), "l"(src + s * 64),
                       "r"(r0 + 16 * i < m && s * 64 < d ? 16 : 0) : "memory");
        src += row16;
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
#pragma unroll 1
        for (int s = 0; s < SUBS; ++s) {
          uint32_t w[4] = {};
          if (r0 + 16 * i < m) {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (s * 64 + x < d) w[x >> 1] |= (uint32_t)__bfloat16_as_ushort(src[s * 64 + x]) << (16 * (x & 1));
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + s * SUB + i * 2048), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        src += row16;
      }
    }
    p += 4 * row16;
  }
};

template <int DK, bool SUMS> struct MmaSmem {
  static constexpr int TILE = DK / 64 * SUB, K = SUMS ? 0 : TILE, STAGE = K + TILE + SUB, STATE = SUMS ? 0 : DK * 128;      // K: k behind q
  static constexpr int OFF_S = 2 * STAGE, OFF_T = OFF_S + 2 * STATE, BYTES = OFF_T + 256 * 4;
};

// SUMS: a segment's own sum alone, the first of the launches over segments
template <int DK, int PARTS, bool MANY, bool SUMS>
__global__ void __launch_bounds__(128, (DK == 64 ? 3 : 2) + SUMS)
scan_mma_kernel(const __grid_constant__ Scans scans) {
  extern __shared__ __align__(128) char smem[];
  int tile, bh;
  const Scan& a = pick_scan<MANY>(scans, tile, bh);
  pdl_wait();
  typedef MmaSmem<DK, SUMS> L;
  typedef __nv_bfloat16 T;
  constexpr int MT = DK / 64, NT = DVT / 8;
  float* pz = reinterpret_cast<float*>(smem + L::OFF_T) + 64;                       // pz[n] = scale l^n for n = 0 .. 63, 0 below
  float* pr = pz + 64;                                                              // pr[x] = l^(63-x), 0 beyond (and behind it for 64 more)
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int seg = blockIdx.y, col0 = tile * DVT;
  const int cols = min(DVT, a.dv - col0);
  const int n = seq_length(a, b);
  const float ld = a.log_decay[h];
  const int seg_len = a.seg_chunks * C;
  const int at0 = min(seg * seg_len, a.len), at1 = min(at0 + seg_len, a.len);       // places of this segment, in scan order
  const bool last = n <= at1 && (n > at0 || (n == 0 && seg == 0));                  // holds the last token
  if (SUMS && (n <= at1 || seg == a.n_seg - 1)) return;                      // nobody reads the last segment's sum
  const int first = a.reverse && a.init ? 1 : 0;                                    // the given state is one step younger
  const int end = min(at1, n), dir = a.reverse ? -1 : 1;
  const long long tok0 = a.reverse ? n - 1 - at0 : at0;                             // token at place at0
  Copy cq(a.q.p, b * a.q.sb + (long long)(h / a.q.div) * a.q.sh + tok0 * a.q.st, a.q.st, dir, a.dk);
  Copy ck(a.k.p, b * a.k.sb + (long long)(h / a.k.div) * a.k.sh + tok0 * a.k.st, a.k.st, dir, a.dk);
  Copy cv(a.v.p, b * a.v.sb + (long long)(h / a.v.div) * a.v.sh + tok0 * a.v.st + col0, a.v.st, dir, cols);
  const uint32_t base = saddr(smem);
  auto fetch = [&](uint32_t to, int m) {
    if (!SUMS) cq.load<DK / 64>(to, m, a.wide);
    ck.load<DK / 64>(to + L::K, m, a.wide);
    cv.load<1>(to + L::K + L::TILE, m, a.wide);
    cp_commit();
  };
  if (at0 < end) fetch(base, end - at0);
  for (int i = tid; i < 256; i += 128) pz[i - 64] = i < 64 ? 0.f : i < 128 ? a.scale * power(ld, i - 64) : i < 192 ? power(ld, 191 - i) : 0.f;
  // the state in front of this segment: (mt, nt, e) is row (w MT + mt) 16 + g + 8 (e >> 1), column nt 8 + 2 t4 + (e & 1)
  float s[MT][NT][4] = {};
  const Front front(a, bh, b, h, seg, col0);
  if (front.p && (n > at0 || last)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = (w * MT + mt) * 16 + g + 8 * (e >> 1), j = nt * 8 + 2 * t4 + (e & 1);
          const bool in = i < a.dk && j < cols;
          const float x = front(in ? i : 0, in ? j : 0);          // no branch around the load: all are under way at once
          s[mt][nt][e] = in ? x : 0.f;
        }
  }
  // offsets of this lane's rows for ldmatrix and stmatrix; a step of 16 channels is an exclusive or with 32 (tiles start on
  // 128-byte boundaries, so that it is one of the whole address too)
  const int r8 = lane & 7, half = (lane >> 3) & 1, quad = lane >> 4;
  const uint32_t off_a = (r8 + 8 * half) * 128 + ((quad ^ r8) << 4);                // 16 rows, two pieces: A, and B from rows of k
  const uint32_t off_b = (r8 + 8 * quad) * 128 + ((half ^ r8) << 4);                // the other order
  auto write_state = [&]() {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f32x2 z = f2_pack(s[mt][2 * np + (x >> 1)][2 * (x & 1)], s[mt][2 * np + (x >> 1)][2 * (x & 1) + 1]);
          hi[x] = cut_off(z);
          lo[x] = pack_up(z);
        }
        const uint32_t to = (base + L::OFF_S + off_a + (w * MT + mt) * 2048) ^ (np << 5);
        stsm(to, hi[0], hi[1], hi[2], hi[3]);
        stsm(to + L::STATE, lo[0], lo[1], lo[2], lo[3]);
      }
  };
  if (!SUMS) write_state();
  uint32_t stage = 0;                    // bytes to the buffer at hand
  // o: rows 4 x + lane / 8 of this warp's 16, 16-byte piece lane & 7
  const int o_row = w * 16 + (lane >> 3), o_c = lane & 7;
  T* o_at = static_cast<T*>(a.o) + b * a.o_sb + (tok0 + (long long)o_row * dir) * a.o_st + h * a.o_sh + col0 + o_c * 8;
  const long long o_step = 4LL * dir * a.o_st;
  float d0 = 0.f, d1 = 0.f;              // what the state fades by on the way to rows g and g + 8 of this warp's, with the output's scale
  f32x2 keep = f2_splat(0.f);            // and through a chunk, less 1
  for (int at = at0; at < end; at += C) {
    const int m = min(C, end - at);
    if (at == at0 || at == C || m < C) { // else as in the chunk before
      const int young = at == 0 ? first : 0;
      d0 = a.scale * power(ld, w * 16 + g + 1 - young);
      d1 = a.scale * power(ld, w * 16 + g + 9 - young);
      keep = f2_splat(power_m1(ld, m - young));
    }
    cp_wait0();
    __syncthreads();
    if (at + C < end) fetch(base + (L::STAGE - stage), end - at - C);
    const uint32_t qs = base + stage, ks_ = qs + L::K, vs = ks_ + L::TILE, ss = base + L::OFF_S;
    if (!SUMS) {
      const uint32_t q_a = qs + w * 2048 + off_a;
      uint32_t qf[MT][4][4];
      float o[NT][4] = {};
#pragma unroll
      for (int x = 0; x < MT; ++x) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) ldsm(qf[x][ks], (q_a + x * SUB) ^ (ks << 5));
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
#pragma unroll
            for (int y = 1; y >= 0; --y) {
              uint32_t f[4];
              ldsm_t(f, ((ss + off_a + (x * 4 + ks) * 2048) ^ (np << 5)) + y * L::STATE);
              mma(o[2 * np], qf[x][ks], f[0], f[1]);
              mma(o[2 * np + 1], qf[x][ks], f[2], f[3]);
            }
          }
      }
      __syncthreads();                   // the state has been read by all, and may be written anew
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f2_unpack(f2_mul(f2_pack(o[nt][0], o[nt][1]), f2_splat(d0)), o[nt][0], o[nt][1]);
        f2_unpack(f2_mul(f2_pack(o[nt][2], o[nt][3]), f2_splat(d1)), o[nt][2], o[nt][3]);
      }
#pragma unroll 1
      for (int jb = 0; jb <= w; ++jb) {                                             // 16 tokens of k and v at a time
        const uint32_t k_b = ks_ + off_b + jb * 2048, v_a = vs + off_a + jb * 2048;
        float p[2][4] = {}, p2[2][4] = {};                                          // two chains of half the length
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            uint32_t f[4];
            ldsm(f, (k_b + x * SUB) ^ (ks << 5));
            mma(ks & 1 ? p2[0] : p[0], qf[x][ks], f[0], f[1]);
            mma(ks & 1 ? p2[1] : p[1], qf[x][ks], f[2], f[3]);
          }
        const float* f = pz + (16 * (w - jb) + g - 2 * t4);                         // l^(i - j): 0 above the diagonal
        const int gap = 16 * (w - jb) + g - 2 * t4;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int off = 8 * (e >> 1) - 8 * x - (e & 1);
            p[x][e] = gap + off >= 0 ? (p[x][e] + p2[x][e]) * f[off] : 0.f;
          }
        uint32_t pf[2][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f32x2 z = f2_pack(p[x >> 1][2 * (x & 1)], p[x >> 1][2 * (x & 1) + 1]);
          pf[0][x] = cut_off(z);
          pf[1][x] = pack_up(z);
        }
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          uint32_t v[4];
          ldsm_t(v, v_a ^ (np << 5));
#pragma unroll
          for (int y = 1; y >= 0; --y) {
            mma(o[2 * np], pf[y], v[0], v[1]);
            mma(o[2 * np + 1], pf[y], v[2], v[3]);
          }
        }
      }
      if (a.o_f32) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = w * 16 + g + 8 * e;
          if (r >= m) continue;
          float* to = static_cast<float*>(a.o) + b * a.o_sb + (tok0 + (long long)(at - at0 + r) * dir) * a.o_st + h * a.o_sh + col0 + 2 * t4;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (a.o_wide) {
              if (nt * 8 < cols) *reinterpret_cast<float2*>(to + nt * 8) = make_float2(o[nt][2 * e], o[nt][2 * e + 1]);
            } else {
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if (nt * 8 + 2 * t4 + x < cols) to[nt * 8 + x] = o[nt][2 * e + x];
            }
          }
        }
      } else {                                                                      // through this warp's own rows of the q tile
        __syncwarp();
#pragma unroll
        for (int np = 0; np < NT / 2; ++np)
          stsm(q_a ^ (np << 5), pack2(o[2 * np][0], o[2 * np][1]), pack2(o[2 * np][2], o[2 * np][3]),
               pack2(o[2 * np + 1][0], o[2 * np + 1][1]), pack2(o[2 * np + 1][2], o[2 * np + 1][3]));
        __syncwarp();
        T* to = o_at;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = o_row + 4 * x;
          uint4 u;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(qs + at_piece(r, o_c)) : "memory");
          if (r < m && o_c * 8 < cols) {
            if (a.o_wide) {
              *reinterpret_cast<uint4*>(to) = u;
            } else {
              const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (o_c * 8 + i < cols) to[i] = __ushort_as_bfloat16((unsigned short)(ww[i >> 1] >> (16 * (i & 1))));
            }
          }
          to += o_step;
        }
        o_at += 16 * o_step;
      }
    }
    // state: k^T (v weighted by age), the weight on k's fragment
    float acc[MT][NT][4] = {};
    const float* wt = pr + (C - m) + 2 * t4;
    uint32_t k_b = ks_ + off_b, v_a = vs + off_a;
#pragma unroll 1
    for (int ks = 0; ks < C / 16; ++ks) {
      uint32_t kf[MT][PARTS][4];
      const f32x2 w0 = f2_pack(wt[0], wt[1]), w1 = f2_pack(wt[8], wt[9]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t f[4];
        const int c16 = w * MT + mt;                                                // channels 16 c16 ..
        ldsm_t(f, (k_b + (c16 >> 2) * SUB) ^ ((c16 & 3) << 5));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f32x2 z = f2_mul(f2_pack(lo_of(f[x]), hi_of(f[x])), x < 2 ? w0 : w1);
#pragma unroll
          for (int y = 0; y < PARTS - 1; ++y) kf[mt][y][x] = cut_off(z);
          kf[mt][PARTS - 1][x] = pack_up(z);
        }
      }
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        uint32_t f[4];
        ldsm_t(f, v_a ^ (np << 5));
#pragma unroll
        for (int y = PARTS - 1; y >= 0; --y)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma(acc[mt][2 * np], kf[mt][y], f[0], f[1]);
            mma(acc[mt][2 * np + 1], kf[mt][y], f[2], f[3]);
          }
      }
      wt += 16;
      k_b += 2048;
      v_a += 2048;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const f32x2 z = f2_pack(s[mt][nt][e], s[mt][nt][e + 1]);
          f2_unpack(f2_add(f2_fma(z, keep, z), f2_pack(acc[mt][nt][e], acc[mt][nt][e + 1])), s[mt][nt][e], s[mt][nt][e + 1]);
        }
    stage = L::STAGE - stage;
    if (!SUMS && at + C < end) write_state();
  }
  const float f = SUMS ? 1.f : a.final_scale * (a.reverse ? power(ld, n == 0 && a.init ? 0 : 1) : 1.f);
  float* to = SUMS ? a.segments + ((long long)bh * a.n_seg + seg) * a.dk * a.dv : a.final && last ? a.final + b * a.s_b + h * a.s_h : nullptr;
  const long long s_i = SUMS ? a.dv : a.s_i, s_j = SUMS ? 1 : a.s_j;
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
  if (SUMS) return;
  const int dead0 = max(at0, n);                                                    // rows behind the last token are zero
  for (long long e = tid; e < (long long)(at1 - dead0) * cols; e += 128) {
    const long long to = b * a.o_sb + (dead0 + e / cols) * a.o_st + h * a.o_sh + col0 + e % cols;
    if (a.o_f32) static_cast<float*>(a.o)[to] = 0.f; else static_cast<T*>(a.o)[to] = __float2bfloat16_rn(0.f);
  }
}

// The segments' own sums become the states in front of them, in place: a thread walks over the segments of one element.  (Sums of
// segments that reach beyond the last token were not written; they reach only segments that have no tokens.)
__global__ void __launch_bounds__(256)
join_segments(const __grid_constant__ Scans scans) {
  const Scan& a = scans.s[blockIdx.z];
  pdl_wait();
  const int size = a.dk * a.dv, parts = (size + 255) / 256;
  const int bh = blockIdx.x / parts, b = bh / a.heads, h = bh - b * a.heads, e = (blockIdx.x - bh * parts) * 256 + threadIdx.x;
  if (e >= size) return;
  float* p = a.segments + (long long)bh * a.n_seg * size + e;
  const float ld = a.log_decay[h], later = power_m1(ld, a.seg_chunks * C);
  float carry = power_m1(ld, a.seg_chunks * C - (a.reverse && a.init ? 1 : 0));
  float x = a.init ? a.init_scale * a.init[b * a.s_b + h * a.s_h + e / a.dv * a.s_i + e % a.dv * a.s_j] : 0.f;
  for (int r0 = 0; r0 < a.n_seg; r0 += 8) {
    float y[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) y[r] = r0 + r < a.n_seg - 1 ? p[(long long)(r0 + r) * size] : 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r0 + r >= a.n_seg) break;
      p[(long long)(r0 + r) * size] = x;
      x = fmaf(x, carry, x) + y[r];
      carry = later;
    }
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
// q^T S is summed.  Bound by the state's bytes: 256 sequences of 12 heads of 128 x 128 72 us, 5.7 TB/s, 0.87 of the measured copy rate;
// one sequence 2.6 us, a launch.
template <typename T>
__global__ void __launch_bounds__(256)
step_kernel(const m2_linear_attention_step_args a) {
  __shared__ float red[16][DVT + 4];
  __shared__ float qs[MAX_D], ks[MAX_D];
  pdl_wait();
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

// Segments: where the blocks of all (sequence, head) pairs and 64-column tiles do not fill the GPU, a long axis is cut; every
// segment's own sum is made first (reading k and v once more) and the segments then run side by side.
// A cut costs half as much again, so there is one only where all blocks still run at once: an SM holds three of them, two with
// more than 64 channels, and of float32 two with up to 96 channels and one with more (cut for two of those: 4096 float32 tokens of 4
// heads of 128 150 us, gradients 400; for one 144 and 368).
static size_t f32_smem(int dk) { return ((size_t)(3 * ((dk + 15) / 16 * 16) + 2 * C) * LD + C + 4) * sizeof(float); }
static int blocks_an_sm(int dtype, int dk) {             // dk: of the launch's widest keys
  if (dtype == M2_BF16) return dk <= 64 ? 3 : 2;
  return 2 * (f32_smem(dk) + 1024) <= 228 * 1024 ? 2 : 1;       // a block's own 1 KB beside; registers admit two
}
static void segments_of(int batch, int heads, int tiles, int len, int an_sm, int* n_seg, int* seg_chunks) {
  const long long blocks = (long long)batch * heads * tiles;
  const int chunks = (len + C - 1) / C;
  long long seg = (long long)an_sm * m2_sm_count() / blocks;
  if (seg > chunks / 2) seg = chunks / 2;               // two chunks at least
  if (seg < 1) seg = 1;
  *seg_chunks = chunks ? (int)((chunks + seg - 1) / seg) : 1;
  *n_seg = chunks ? (chunks + *seg_chunks - 1) / *seg_chunks : 1;
}
static int tiles_of(int dv) { return (dv + DVT - 1) / DVT; }
// of `scans` scans side by side, each with a state of dk x dv or dv x dk
static long long segment_floats(int batch, int heads, int dk, int dv, int tiles, int scans, int len, int dtype) {
  int n, c;
  segments_of(batch, heads, tiles, len, blocks_an_sm(dtype, scans == 1 || dk > dv ? dk : dv), &n, &c);
  return n > 1 ? (long long)scans * batch * heads * n * dk * dv : 0;
}

// Rows in 16-byte pieces, which are read whole and nothing beside them
static bool in_pieces(const void* p, long long sb, long long st, long long sh, int d, int dtype) {
  const int piece = dtype == M2_F32 ? 4 : 8;
  return m2_aligned(p, 16) && sb % piece == 0 && st % piece == 0 && sh % piece == 0 && d % piece == 0;
}

static long long elements(const Scans& p) { return (long long)p.s[0].batch * p.s[0].len * p.s[0].heads * (p.s[0].dk > p.s[0].dv ? p.s[0].dk : p.s[0].dv); }

template <int DK, int PARTS, bool MANY, bool SUMS> static int launch_mma(const char* name, const Scans& p, dim3 grid, cudaStream_t st) {
  constexpr int bytes = MmaSmem<DK, SUMS>::BYTES;
  M2_SMEM_ONCE((scan_mma_kernel<DK, PARTS, MANY, SUMS>), bytes);
  return m2_launch(name, elements(p), scan_mma_kernel<DK, PARTS, MANY, SUMS>, grid, 128, bytes, st, p);
}
template <int DK, int PARTS> static int launch_mma_of(const char* name, const Scans& p, bool many, bool sums, dim3 grid, cudaStream_t st) {
  if (many) return sums ? launch_mma<DK, PARTS, true, true>(name, p, grid, st) : launch_mma<DK, PARTS, true, false>(name, p, grid, st);
  return sums ? launch_mma<DK, PARTS, false, true>(name, p, grid, st) : launch_mma<DK, PARTS, false, false>(name, p, grid, st);
}
template <bool MANY> static int launch_f32(const char* name, const Scans& p, int dk, dim3 grid, cudaStream_t st) {
  M2_SMEM_ONCE(scan_f32_kernel<MANY>, f32_smem(MAX_D));
  return m2_launch(name, elements(p), scan_f32_kernel<MANY>, grid, 256, f32_smem(dk), st, p);
}

// `count` scans over the same (sequence, head) pairs: one launch for those whose keys have up to 64 channels and one for the others
// (float32: one for all), each behind one of the segments' sums where the axis is cut.
// `whole`: weighted keys keep all their bits though no state is returned.
static int run_scans(const char* name, Scan* list, int count, int dtype, float* segments, bool whole, cudaStream_t st) {
  int tiles = 0, widest = 0, n_seg, seg_chunks;
  for (int i = 0; i < count; ++i) {
    tiles += tiles_of(list[i].dv);
    widest = list[i].dk > widest ? list[i].dk : widest;
  }
  segments_of(list[0].batch, list[0].heads, tiles, list[0].len, blocks_an_sm(dtype, widest), &n_seg, &seg_chunks);
  for (int i = 0; i < count; ++i) {
    Scan& a = list[i];
    a.n_seg = n_seg;
    a.seg_chunks = seg_chunks;
    a.segments = n_seg > 1 ? segments + (long long)i * a.batch * a.heads * n_seg * a.dk * a.dv : nullptr;
    a.wide = in_pieces(a.q.p, a.q.sb, a.q.st, a.q.sh, a.dk, dtype) && in_pieces(a.k.p, a.k.sb, a.k.st, a.k.sh, a.dk, dtype) && in_pieces(a.v.p, a.v.sb, a.v.st, a.v.sh, a.dv, dtype);
    a.o_wide = in_pieces(a.o, a.o_sb, a.o_st, a.o_sh, a.dv, M2_BF16);
  }
  for (int large = 0; large < 2; ++large) {
    Scans p = {};
    int n = 0, dk = 0;
    unsigned x = 0;
    bool parts3 = whole;
    for (int i = 0; i < count; ++i) {
      if (dtype == M2_BF16 ? (list[i].dk > 64) != (large == 1) : large == 1) continue;
      p.s[n] = list[i];
      p.tiles[n] = tiles_of(list[i].dv);
      x += p.tiles[n++];
      dk = list[i].dk > dk ? list[i].dk : dk;
      parts3 |= list[i].final != nullptr;
    }
    if (n == 0) continue;
    const unsigned pairs = (unsigned)list[0].batch * list[0].heads;
    const dim3 grid(x * pairs, n_seg);
    for (int sums = n_seg > 1; sums >= 0; --sums) {
      for (int i = 0; i < n; ++i) p.s[i].sums_only = sums;
      const int rc = dtype != M2_BF16 ? (n > 1 ? launch_f32<true>(name, p, dk, grid, st) : launch_f32<false>(name, p, dk, grid, st))
                     : large  ? (parts3 ? launch_mma_of<128, 3>(name, p, n > 1, sums, grid, st) : launch_mma_of<128, 2>(name, p, n > 1, sums, grid, st))
                     : parts3 ? launch_mma_of<64, 3>(name, p, n > 1, sums, grid, st)
                              : launch_mma_of<64, 2>(name, p, n > 1, sums, grid, st);
      if (rc) return rc;
      if (sums) {
        if (int e = m2_launch(name, elements(p), join_segments, dim3((p.s[0].dk * p.s[0].dv + 255) / 256 * pairs, 1, n), 256, 0, st, p)) return e;
      }
    }
  }
  return M2_OK;
}

static int check(const char* name, int batch, int len, int heads, int kv_heads, int dk, int dv, int dtype, float scale) {
  M2_REQUIRE(batch >= 0 && len >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, M2_ERR_ARG, "%s: batch %d, %d steps, %d heads on %d key heads", name,
             batch, len, heads, kv_heads);
  M2_REQUIRE(dk >= 1 && dv >= 1 && dk <= MAX_D && dv <= MAX_D, M2_ERR_UNSUPPORTED, "%s: heads of 1 to %d channels, got %d and %d", name, MAX_D, dk, dv);
  M2_REQUIRE((long long)batch * heads <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: batch * heads up to %d, got %d * %d", name, 1 << 24, batch, heads);
  M2_REQUIRE(len <= 1 << 24, M2_ERR_UNSUPPORTED, "%s: up to %d steps, got %d", name, 1 << 24, len);
  M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: q, k and v are float32 or bf16", name);
  M2_REQUIRE(scale != 0.f && scale - scale == 0.f && 1.f / scale - 1.f / scale == 0.f, M2_ERR_ARG, "%s: scale %g", name, scale);
  return M2_OK;
}

static int check_operands(const char* name, const m2_linear_attention_args& g) {
  const size_t size = g.dtype == M2_F32 ? 4 : 2;
  M2_REQUIRE(g.log_decay && (g.seq_len == 0 || (g.q && g.k && g.v)), M2_ERR_ARG, "%s: q, k, v or log_decay is NULL", name);
  M2_REQUIRE(m2_aligned(g.q, size) && m2_aligned(g.k, size) && m2_aligned(g.v, size) && m2_aligned(g.lengths, 8), M2_ERR_ALIGN,
             "%s: a tensor is not aligned to its type", name);
  return M2_OK;
}

// The plan of the launch is made for the current device, as the size is that was asked for: a plan for more multiprocessors than the
// workspace was made for would write behind it.
static int check_workspace(const char* name, const m2_linear_attention_args& g, int backward) {
  const long long need = m2_linear_attention_workspace(g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, backward);
  M2_REQUIRE(need == 0 || (g.workspace && g.workspace_bytes >= need), M2_ERR_ARG, "%s: a workspace of %lld bytes, on this device the shape needs %lld", name,
             g.workspace ? g.workspace_bytes : 0, need);
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

extern "C" long long m2_linear_attention_workspace(int batch, int seq_len, int heads, int kv_heads, int dk, int dv, m2_dtype dtype, int backward) {
  using namespace m2::la;
  if (batch < 1 || seq_len < 1 || heads < 1 || kv_heads < 1 || dk < 1 || dv < 1) return 0;
  long long floats = segment_floats(batch, heads, dk, dv, tiles_of(dv), 1, seq_len, dtype);
  if (backward) {
    floats = segment_floats(batch, heads, dk, dv, 2 * tiles_of(dk) + tiles_of(dv), 3, seq_len, dtype);
    if (heads != kv_heads) floats += (long long)batch * seq_len * heads * (dk + dv);
  }
  return floats * (long long)sizeof(float);
}

extern "C" int m2_linear_attention_fwd(const m2_linear_attention_args* args, void* stream) {
  using namespace m2::la;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_linear_attention_fwd: args is NULL");
  const m2_linear_attention_args& g = *args;
  if (int rc = check("m2_linear_attention_fwd", g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, g.scale)) return rc;
  if (g.batch == 0) return M2_OK;
  if (int rc = check_operands("m2_linear_attention_fwd", g)) return rc;
  M2_REQUIRE(g.o || g.seq_len == 0, M2_ERR_ARG, "m2_linear_attention_fwd: o is NULL");
  if (int rc = check_workspace("m2_linear_attention_fwd", g, 0)) return rc;
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
  return run_scans("m2_linear_attention_fwd", &s, 1, g.dtype, g.workspace, true, (cudaStream_t)stream);
}

extern "C" int m2_linear_attention_bwd(const m2_linear_attention_args* args, const m2_linear_attention_grads* grads, void* stream) {
  using namespace m2::la;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr && grads != nullptr, M2_ERR_ARG, "m2_linear_attention_bwd: args or grads is NULL");
  const m2_linear_attention_args& g = *args;
  const m2_linear_attention_grads& d = *grads;
  if (int rc = check("m2_linear_attention_bwd", g.batch, g.seq_len, g.heads, g.kv_heads, g.dk, g.dv, g.dtype, g.scale)) return rc;
  if (g.batch == 0) return M2_OK;
  if (int rc = check_operands("m2_linear_attention_bwd", g)) return rc;
  M2_REQUIRE(g.seq_len == 0 || (d.d_o && d.d_q && d.d_k && d.d_v), M2_ERR_ARG, "m2_linear_attention_bwd: d_o, d_q, d_k or d_v is NULL");
  M2_REQUIRE(m2_aligned(d.d_o, g.dtype == M2_F32 ? 4 : 2), M2_ERR_ALIGN, "m2_linear_attention_bwd: d_o is not aligned to its type");
  if (int rc = check_workspace("m2_linear_attention_bwd", g, 1)) return rc;
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
  Scan list[3];
  Scan& x = list[0] = base_of(g);        // dq = scan(do, v, k) from the transposed initial state
  x.q = u; x.k = v; x.v = k;
  x.o = d.d_q; x.o_sb = row_k * g.seq_len; x.o_st = row_k; x.o_sh = g.dk;
  x.dk = g.dv; x.dv = g.dk; x.scale = g.scale;
  x.init = g.state_in; x.init_scale = 1.f;
  x.s_b = s_b; x.s_h = s_h; x.s_i = 1; x.s_j = g.dv;
  Scan& y = list[1] = base_of(g);        // dk = reversed scan(v, do, q)
  y.q = v; y.k = u; y.v = q; y.reverse = 1;
  y.o = group > 1 ? (void*)part_k : d.d_k; y.o_f32 = group > 1; y.o_sb = row_k * g.seq_len; y.o_st = row_k; y.o_sh = g.dk;
  y.dk = g.dv; y.dv = g.dk; y.scale = g.scale;
  y.init = d.d_state_out; y.init_scale = 1.f / g.scale;
  y.s_b = s_b; y.s_h = s_h; y.s_i = 1; y.s_j = g.dv;
  Scan& z = list[2] = base_of(g);        // dv = reversed scan(k, q, do), and what is left of the state is the initial state's gradient
  z.q = k; z.k = q; z.v = u; z.reverse = 1;
  z.o = group > 1 ? (void*)part_v : d.d_v; z.o_f32 = group > 1; z.o_sb = row_v * g.seq_len; z.o_st = row_v; z.o_sh = g.dv;
  z.dk = g.dk; z.dv = g.dv; z.scale = g.scale;
  z.init = d.d_state_out; z.init_scale = 1.f / g.scale; z.final = d.d_state_in; z.final_scale = g.scale;
  z.s_b = s_b; z.s_h = s_h; z.s_i = g.dv; z.s_j = 1;
  if (int rc = run_scans("m2_linear_attention_bwd", list, 3, g.dtype, segments, false, st)) return rc;
  if (group > 1 && tokens > 0) {
    for (int w = 0; w < 2; ++w) {
      const float* part = w ? part_v : part_k;
      void* out = w ? d.d_v : d.d_k;
      const int width = w ? g.dv : g.dk;
      const long long blocks = (tokens * g.kv_heads * width + 255) / 256;
      const int grid = (int)(blocks < 16LL * m2_sm_count() ? blocks : 16LL * m2_sm_count());
      if (g.dtype == M2_F32) group_sum_kernel<float><<<grid, 256, 0, st>>>(part, static_cast<float*>(out), tokens, g.kv_heads, group, width);
      else group_sum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(part, static_cast<__nv_bfloat16*>(out), tokens, g.kv_heads, group, width);
      ++m2_launch_count();
    }
    M2_LAUNCH_CHECK("m2_linear_attention_bwd (shared heads)");
  }
  return M2_OK;
}

extern "C" int m2_linear_attention_step(const m2_linear_attention_step_args* args, void* stream) {
  using namespace m2::la;
  m2_launch_count() = 0;
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
  const long long states = (long long)g.batch * g.heads * g.dk * g.dv;
  return g.dtype == M2_F32 ? m2_launch("m2_linear_attention_step", states, step_kernel<float>, grid, 256, 0, st, g)
                           : m2_launch("m2_linear_attention_step", states, step_kernel<__nv_bfloat16>, grid, 256, 0, st, g);
}
