// One step of a beam search: the best of all (beam, token) pairs of each text by the beam's score plus log softmax(logits)[token], and the
// states of the chosen beams moved to their new places.  Stands behind the decoder, beside m2_token_logprobs_fwd (the reference has no generation:
// bert/src/bert_layers.py, BertForMaskedLM, ends in a loss).
//
// Selection in two kernels.  The first reads each beam's logits once (a cluster of blocks a row where there are few rows): maximum, sum of
// exponentials, and its `keep` best tokens, found without sorting as in token_logprobs.cu.  The second, a warp a text, merges the beams' sorted lists: a
// lane a beam, the best head `keep` times.  Scores are compared in 64 bits.  Their sums of exponentials are within 5 2^-24 (3e-7) of themselves, however many logits there
// are and however they lie: each exponential within 2 2^-24 (what its argument's subtraction rounds off is put back), those of 16 bytes added in float32 as a
// tree, and from there on in 64 bits, without being scaled again by float32 factors on the way.  So the order is that of exact scores but for gaps below that.
// States: a thread owns a few bytes of the rows of all beams of one text; it reads the rows that its beams come from before it writes any,
// so that nothing waits and no second buffer is needed.  Rows that stay are neither read nor written.
// Measured: selection for one text of four beams 17 us, for 32 of eight beams (float32, 31 MB) 27; states of 12 layers of the latter (256 rows of 58 KB a layer,
// some 227 of which are replaced, by 75 different ones: 212 MB) 40 us, 5.3 TB/s.
#include "common.cuh"

namespace m2 {
namespace beam {

using lp::Piece;
constexpr int THREADS = lp::THREADS;
constexpr int MAX_BEAMS = 32;
constexpr int MAX_KEEP = lp::MAX_TOP;

struct Args {
  const void* x; long long x_sb, x_sk;
  int batch, beams, vocab, keep, list, split;     // list: tokens of a beam that are looked at, min(keep, vocab)
  const float* scores;
  const unsigned char* finished;
  long long end_id;                               // -1: none
  float* row_max; double* row_sum;                // (batch * beams): sums of exponentials of differences to a logit that is the largest but for 32
  unsigned long long* best;                       // (batch * beams, list)
  float* score;
  long long *beam, *token;
  unsigned char* done;
};

// exp(v - m) for v - m < 64: 2^i 2^f with the powers of ln 2 for 2^f, |f| <= 1/2, cut where the next is below 1e-8; 0 below exp(-87), NaN stays NaN
__device__ __forceinline__ float exp_near(float v, float m) {
  const float d = v - m;
  // the sum of two numbers exactly (D. E. Knuth): back is v as d has it, and what d lost is v - back less m - (back - d)
  const float back = d + m, lost = (v - back) - (m - (back - d));
  const float i = rintf(d * lp::LOG2E);
  const float f = fmaf(d, lp::LOG2E, -i) + fmaf(d, 1.92596299e-8f, lost * lp::LOG2E);       // LOG2E and what float32 leaves of it
  float p = 1.52527338e-5f;
  p = fmaf(p, f, 1.54035304e-4f);
  p = fmaf(p, f, 1.33335581e-3f);
  p = fmaf(p, f, 9.61812911e-3f);
  p = fmaf(p, f, 5.55041087e-2f);
  p = fmaf(p, f, 2.40226507e-1f);
  p = fmaf(p, f, 6.93147181e-1f);
  p = fmaf(p, f, 1.f);
  return d < -87.f ? 0.f : __int_as_float(__float_as_int(p) + ((int)i << 23));
}

struct Sum { float m; double s; };
// s of m becomes that of a larger maximum
__device__ __forceinline__ double at_maximum(Sum a, float m) { return a.m < m ? a.s * exp((double)a.m - (double)m) : a.s; }

struct Shared {
  lp::Shared top;
  Sum warp[lp::WARPS], mine;
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 6)
rows_kernel(const Args a) {
  constexpr int N = Piece<T>::N;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, split = a.split;
  pdl_wait();
  const long long row = blockIdx.x / split;
  if (a.finished && a.finished[row]) return;      // the whole cluster
  const uint32_t part = split > 1 ? lp::cta_rank() : 0;
  const T* x = static_cast<const T*>(a.x) + row / a.beams * a.x_sb + row % a.beams * a.x_sk;
  const int per = ((a.vocab + split - 1) / split + 63) / 64 * 64;
  const int lo = min((int)part * per, a.vocab), hi = min(lo + per, a.vocab);
  const lp::Span<T> sp(x, lo, hi);
  // exponentials of differences to m, which stays while no logit is more than RISE above it; vmax is the largest logit.  A NaN or +inf makes s NaN.
  constexpr float RISE = 32.f;
  float m = lp::LOWEST, vmax = lp::LOWEST;
  double s = 0.0;
  auto look = [&](float big) {
    if (big > vmax) vmax = big;
    if (big > m + RISE) { s = at_maximum({m, s}, big); m = big; }
  };
  sp.ends([&](float v, int) { look(v); s += exp_near(v, m); });
  const uint4* body = reinterpret_cast<const uint4*>(x + sp.body());
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
        look(lp::largest(now[j], f));
#pragma unroll
        for (int q = 0; q < N; ++q) f[q] = exp_near(f[q], m);
#pragma unroll
        for (int w = N / 2; w > 0; w /= 2)
#pragma unroll
          for (int q = 0; q < w; ++q) f[q] += f[q + w];
        s += f[0];
      }
      now[j] = next[j];
    }
  }
  const bool nan = s != s;
  Sum st = {m, s};
  auto warp_sum = [&](int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    s = at_maximum(st, m);
    for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    st = {m, s};
  };
  warp_sum(32);
  if (lane == 0) sh.warp[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st = lane < lp::WARPS ? sh.warp[lane] : Sum{lp::LOWEST, 0.0};
    m = st.m;
    warp_sum(32);
    if (lane == 0) sh.mine = st;
  }
  lp::select_top<T>(sh.top, sp, a.list, vmax, nan);
  if (split > 1) lp::cluster_barrier(); else __syncthreads();
  if (part == 0) {
    if (warp == 0) {
      st = lane < split ? *lp::in_cta(&sh.mine, lane) : Sum{lp::LOWEST, 0.0};
      m = st.m;
      warp_sum(32);
      if (lane == 0) {
        a.row_max[row] = st.m;
        a.row_sum[row] = st.s;
      }
    }
    if (split == 1) {
      if (tid < a.list) a.best[row * a.list + tid] = sh.top.best[tid];
    } else {
      const int n = split * a.list;
      for (int c = tid; c < n; c += THREADS) sh.top.cand[c] = lp::in_cta(sh.top.best, c / a.list)[c % a.list];
      __syncthreads();
      for (int c = tid; c < n; c += THREADS) {
        const unsigned long long q = sh.top.cand[c];
        int above = 0;
        for (int o = 0; o < n; ++o) above += sh.top.cand[o] > q;
        if (q != 0 && above < a.list) a.best[row * a.list + above] = q;
      }
    }
  }
  if (split > 1) lp::cluster_barrier();           // the other blocks' memory was read
}

// A double as a number of 64 bits with the same order, NaN above all
__device__ __forceinline__ unsigned long long order_of(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
constexpr unsigned long long MINUS_INF = ~0xfff0000000000000ull;                  // order_of(-inf)
__device__ __forceinline__ double value_of(unsigned long long u) {
  if (u == ~0ull) return __longlong_as_double(0x7fffffffffffffffll);
  return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
}

__global__ void __launch_bounds__(32)
merge_kernel(const Args a) {
  pdl_wait();
  const int k = threadIdx.x;
  const long long b = blockIdx.x, row = b * a.beams + k;
  const bool live = k < a.beams, ended = live && a.finished && a.finished[row];
  const double base = live ? (double)a.scores[row] : 0.0;
  float m = 0.f;
  double log_s = 0.0;
  bool none = false;
  if (live && !ended) {
    m = a.row_max[row];
    const double s = a.row_sum[row];
    none = s == 0.0;                              // every logit is -inf
    log_s = log(s);
  }
  int at = 0;                                     // the next of the beam's list
  const int count = !live ? 0 : ended ? 1 : a.list;
  unsigned long long head = 0, key = 0;           // its token, its score; 0: the list has ended
  auto load = [&] {
    key = 0;
    if (at >= count) return;
    if (ended) { key = order_of(base); return; }
    head = a.best[row * a.list + at];
    const double v = none ? -(double)__int_as_float(0x7f800000) : base + (((double)lp::key_value(head) - (double)m) - log_s);
    key = order_of(v);
  };
  load();
  for (int r = 0; r < a.keep; ++r) {
    const unsigned hi = __reduce_max_sync(~0u, (unsigned)(key >> 32));
    const bool top = (unsigned)(key >> 32) == hi;
    const unsigned lo = __reduce_max_sync(~0u, top ? (unsigned)key : 0u);
    const unsigned who = __ballot_sync(~0u, top && (unsigned)key == lo);
    const int winner = __ffs(who) - 1;
    const unsigned long long best = (unsigned long long)hi << 32 | lo;
    const long long out = b * a.keep + r;
    if (best <= MINUS_INF) {                      // nothing is left that has a score
      if (k == 0) {
        const long long t = a.end_id >= 0 ? a.end_id : 0;
        a.score[out] = -__int_as_float(0x7f800000);
        a.beam[out] = 0;
        a.token[out] = t;
        if (a.done) a.done[out] = a.end_id >= 0 || (a.finished && a.finished[b * a.beams]);
      }
      continue;
    }
    if (k == winner) {
      const long long t = ended ? a.end_id : (long long)lp::key_id(head);
      a.score[out] = ended ? a.scores[row] : (float)value_of(key);
      a.beam[out] = k;
      a.token[out] = t;
      if (a.done) a.done[out] = ended || t == a.end_id;
      ++at;
      load();
    }
  }
}

// ---- states ------------------------------------------------------------------------------------------------------------
constexpr int MAX_STATES = 96;           // tensors of one launch
struct Moves {
  int batch, beams, count;
  const long long* from;                 // (batch, beams)
  struct { char* p; long long stride; unsigned units, first; } t[MAX_STATES];     // units of a row; the tensor's first block
};

template <typename U, int K>
__global__ void __launch_bounds__(256)
reorder_kernel(const __grid_constant__ Moves m, unsigned blocks) {
  __shared__ int s_from[K];
  pdl_wait();
  const unsigned text = blockIdx.x / blocks, block = blockIdx.x % blocks;
  if (threadIdx.x < K) {
    int f = threadIdx.x;
    if (f < m.beams) {
      const long long v = m.from[(long long)text * m.beams + f];
      if (v < 0 || v >= m.beams) atomicOr(&m2_dev_status_word, lp::ST_BAD_TARGET);
      f = (int)(v < 0 ? 0 : v >= m.beams ? m.beams - 1 : v);
    }
    s_from[threadIdx.x] = f;
  }
  int i = 0;
  while (i + 1 < m.count && m.t[i + 1].first <= block) ++i;
  __syncthreads();
  const unsigned at = (block - m.t[i].first) * 256 + threadIdx.x;
  if (at >= m.t[i].units) return;
  char* base = m.t[i].p + text * (long long)m.beams * m.t[i].stride + at * (long long)sizeof(U);
  U v[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (s_from[k] != k) v[k] = *reinterpret_cast<const U*>(base + s_from[k] * m.t[i].stride);
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (s_from[k] != k) *reinterpret_cast<U*>(base + k * m.t[i].stride) = v[k];
}

template <typename U> static int reorder(Moves& m, unsigned blocks, long long bytes, cudaStream_t st) {
  M2_REQUIRE((long long)blocks * m.batch <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_reorder_states: %d texts of %u blocks are more than the grid takes", m.batch, blocks);
  auto go = [&](auto kernel) { return m2_launch("m2_reorder_states", bytes / 4, kernel, dim3(blocks * (unsigned)m.batch), 256, 0, st, m, blocks); };
  if (m.beams <= 4) return go(reorder_kernel<U, 4>);
  if (m.beams <= 8) return go(reorder_kernel<U, 8>);
  if (m.beams <= 16) return go(reorder_kernel<U, 16>);
  return go(reorder_kernel<U, 32>);
}

static long long up16(long long n) { return (n + 15) / 16 * 16; }

}  // namespace beam
}  // namespace m2

extern "C" long long m2_beam_select_workspace(int batch, int beams, int vocab, int keep) {
  using namespace m2::beam;
  if (batch <= 0 || beams <= 0 || vocab <= 0 || keep <= 0) return 0;
  const long long rows = (long long)batch * beams;
  return up16(rows * 8) + up16(rows * 4) + rows * 8 * (keep < vocab ? keep : vocab);
}

extern "C" int m2_beam_select(const m2_beam_select_args* args, void* stream) {
  using namespace m2::beam;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_beam_select: args is NULL");
  const m2_beam_select_args& g = *args;
  M2_REQUIRE(g.batch >= 0 && g.beams >= 1 && g.beams <= MAX_BEAMS && g.vocab >= 1, M2_ERR_ARG, "m2_beam_select: %d texts of %d beams (1 .. %d), %d logits",
             g.batch, g.beams, MAX_BEAMS, g.vocab);
  M2_REQUIRE(g.keep >= 1 && g.keep <= MAX_KEEP, M2_ERR_ARG, "m2_beam_select: %d kept (1 .. %d)", g.keep, MAX_KEEP);
  M2_REQUIRE(g.dtype == M2_F32 || g.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "m2_beam_select: logits are float32 or bf16");
  M2_REQUIRE(g.vocab <= 1 << 28 && (long long)g.batch * g.beams <= 1 << 27, M2_ERR_UNSUPPORTED, "m2_beam_select: %d x %d rows of %d logits are more than the grid takes",
             g.batch, g.beams, g.vocab);
  M2_REQUIRE(!g.finished || g.end_id >= 0, M2_ERR_ARG, "m2_beam_select: finished beams need an end_id");
  if (g.batch == 0) return M2_OK;
  M2_REQUIRE(g.logits && g.scores && g.score && g.beam && g.token, M2_ERR_ARG, "m2_beam_select: a tensor is NULL");
  M2_REQUIRE(m2_aligned(g.logits, g.dtype == M2_F32 ? 4 : 2) && m2_aligned(g.scores, 4) && m2_aligned(g.workspace, 16), M2_ERR_ALIGN,
             "m2_beam_select: logits or scores are not aligned to their type, or the workspace not to 16 bytes");
  const long long need = m2_beam_select_workspace(g.batch, g.beams, g.vocab, g.keep), rows = (long long)g.batch * g.beams;
  M2_REQUIRE(g.workspace && g.workspace_bytes >= need, M2_ERR_ARG, "m2_beam_select: the workspace has %lld bytes of %lld", g.workspace ? g.workspace_bytes : 0, need);
  char* w = static_cast<char*>(g.workspace);
  Args a = {g.logits, g.x_sb, g.x_sk, g.batch, g.beams, g.vocab, g.keep, g.keep < g.vocab ? g.keep : g.vocab, 1, g.scores, (const unsigned char*)g.finished, g.end_id,
            reinterpret_cast<float*>(w + up16(rows * 8)), reinterpret_cast<double*>(w), reinterpret_cast<unsigned long long*>(w + up16(rows * 8) + up16(rows * 4)),
            g.score, (long long*)g.beam, (long long*)g.token, (unsigned char*)g.done};
  // a row is shared by the blocks of a cluster where the rows alone do not fill the GPU, each block with 2048 logits at least (one text of four beams, 30528
  // logits: 13 us with slices of 2048, 15 with 4096); shared further than to two blocks an SM, 256 rows took 30 us instead of 22
  while (a.split < m2::lp::MAX_SPLIT && rows * a.split < 2LL * m2_sm_count() && g.vocab / (a.split * 2) >= 2048) a.split *= 2;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * a.split));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  const cudaError_t e = g.dtype == M2_F32 ? cudaLaunchKernelEx(&cfg, rows_kernel<float>, a) : cudaLaunchKernelEx(&cfg, rows_kernel<__nv_bfloat16>, a);
  if (e != cudaSuccess) return m2_set_error(M2_ERR_CUDA, "launch of m2_beam_select failed: %s", cudaGetErrorString(e));
  ++m2_launch_count();
  return m2_launch("m2_beam_select", 0, merge_kernel, dim3((unsigned)g.batch), 32, 0, st, a);
}

extern "C" int m2_reorder_states(const m2_reorder_states_args* args, void* stream) {
  using namespace m2::beam;
  m2_launch_count() = 0;
  M2_REQUIRE(args != nullptr, M2_ERR_ARG, "m2_reorder_states: args is NULL");
  const m2_reorder_states_args& g = *args;
  M2_REQUIRE(g.batch >= 0 && g.beams >= 1 && g.beams <= MAX_BEAMS && g.count >= 0, M2_ERR_ARG, "m2_reorder_states: %d texts of %d beams (1 .. %d), %d tensors",
             g.batch, g.beams, MAX_BEAMS, g.count);
  if (g.batch == 0 || g.count == 0) return M2_OK;
  M2_REQUIRE(g.beam && g.states && m2_aligned(g.beam, 8), M2_ERR_ARG, "m2_reorder_states: beam or states is NULL");
  const cudaStream_t st = (cudaStream_t)stream;
  auto unit_of = [](const m2_beam_state& s) {
    const unsigned long long all = reinterpret_cast<uintptr_t>(s.p) | (unsigned long long)s.row_bytes | (unsigned long long)s.stride_bytes;
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
  };
  for (int i = 0; i < g.count; ++i) {
    const m2_beam_state& s = g.states[i];
    M2_REQUIRE(s.row_bytes >= 0 && (s.row_bytes == 0 || s.p) && ((long long)g.batch * g.beams == 1 || s.stride_bytes >= s.row_bytes), M2_ERR_ARG,
               "m2_reorder_states: tensor %d has rows of %lld bytes, %lld apart", i, s.row_bytes, s.stride_bytes);
    M2_REQUIRE(s.row_bytes / unit_of(s) <= 0x7fffff00LL, M2_ERR_UNSUPPORTED, "m2_reorder_states: tensor %d has rows of %lld bytes", i, s.row_bytes);
  }
  for (int unit : {16, 4, 1}) {
    for (int i = 0; i < g.count;) {
      Moves m;
      m.batch = g.batch; m.beams = g.beams; m.count = 0; m.from = (const long long*)g.beam;
      long long blocks = 0, bytes = 0;
      for (; i < g.count && m.count < MAX_STATES; ++i) {
        const m2_beam_state& s = g.states[i];
        if (s.row_bytes == 0 || unit_of(s) != unit) continue;
        const long long units = s.row_bytes / unit;
        m.t[m.count++] = {static_cast<char*>(s.p), s.stride_bytes, (unsigned)units, (unsigned)blocks};
        blocks += (units + 255) / 256;
        bytes += s.row_bytes * g.batch * g.beams;
        M2_REQUIRE(blocks <= 0x7fffffffLL, M2_ERR_UNSUPPORTED, "m2_reorder_states: the rows are more than the grid takes");
      }
      if (m.count == 0) continue;
      const int rc = unit == 16 ? reorder<uint4>(m, (unsigned)blocks, bytes, st) : unit == 4 ? reorder<uint32_t>(m, (unsigned)blocks, bytes, st)
                                                                                             : reorder<unsigned char>(m, (unsigned)blocks, bytes, st);
      if (rc) return rc;
    }
  }
  return M2_OK;
}
