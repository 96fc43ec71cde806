// Log probabilities of given labels under a softmax over each row of logits, with the row's entropy and
// its best alternatives, and their gradient.
//
//   m = max x, S = sum exp(x - m), A = sum exp(x - m) (x - m)      (terms with exp(x - m) = 0 add 0)
//   logp = x_t - m - log S,   H = log S - A / S
//   dx_j = p_j (-(g_logp + sum_k g_k) - g_H (log p_j + H)) + [j = t] g_logp + sum_k [j = id_k] g_k
//
// Logits of -inf are masked labels: they have probability 0 and are never an alternative.  A row with
// nothing but masked labels has log probability -inf, entropy 0 and gradient 0; a row that holds a NaN or
// +inf has NaN results.  A negative label says unlabelled (logp 0, whatever the row holds), a label past
// the last one gives NaN and reads nothing.  A row whose incoming gradients are all zero gets zeros.
//
// stats[r] = (m, S); S = 0 marks a row of masked labels only (a real one is at least 1), NaN a bad row.  The
// gradient takes p = exp(x - m) / S from S itself: log S, rounded to fp32, would put its rounding (6 of p's own
// for a row of 32001 equal logits) on every p of the row alike.
//
// The running maximum starts at -FLT_MAX, so that x - m is -inf and never NaN for a masked label, and
// x - m is clamped at D_MIN, where exp is 0 in fp32 already: 0 * D_MIN is 0 in A.  S = 0 then says that
// nothing was there.  The maximum keeps NaN (max.NaN), so m tells a bad row without a test per element.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <type_traits>

#include "rowtype.cuh"

namespace tts {

namespace cg = cooperative_groups;

constexpr int TOP_MAX = 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float F_LOWEST = -3.402823466e38f;
constexpr float D_MIN = -500.f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x: at most 2^-22 off relative to the result, results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Part of a row's softmax: the sums are relative to m.
struct Soft {
  float m, S, A;
  __device__ __forceinline__ void init() { m = F_LOWEST, S = 0.f, A = 0.f; }
  // The sums relative to m2 >= m (or NaN).
  __device__ __forceinline__ void rebase(float m2) {
    const float d = fmaxf(m - m2, D_MIN), c = exp2_fast(d * LOG2E);
    A = c * fmaf(d, S, A);
    S *= c;
    m = m2;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = fmaxf(x - m, D_MIN), e = exp2_fast(d * LOG2E);
    S += e;
    A = fmaf(e, d, A);
  }
  // Over lanes that differ in the bits below `width` (a power of two).
  __device__ __forceinline__ void reduce(int width) {
    float m2 = m;
    for (int d = width / 2; d > 0; d >>= 1) m2 = max_nan(m2, __shfl_xor_sync(0xffffffffu, m2, d));
    rebase(m2);
    for (int d = width / 2; d > 0; d >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, d);
      A += __shfl_xor_sync(0xffffffffu, A, d);
    }
  }
  __device__ __forceinline__ bool bad() const { return !(m < CUDART_INF_F); }
};

// A whole row's sums by one thread: four of each in turn, which keeps the additions' roundings of a long row
// down by as much and the chains of dependent additions short.
struct Soft4 {
  float m, S[4], A[4];
  __device__ __forceinline__ void init() {
    m = F_LOWEST;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] = A[i] = 0.f;
  }
  __device__ __forceinline__ void add(float x, int i) {
    const float d = fmaxf(x - m, D_MIN), e = exp2_fast(d * LOG2E);
    S[i] += e;
    A[i] = fmaf(e, d, A[i]);
  }
  __device__ __forceinline__ Soft total() const {
    return Soft{m, (S[0] + S[1]) + (S[2] + S[3]), (A[0] + A[1]) + (A[2] + A[3])};
  }
};

struct ScoreArgs {
  const void* labels;
  float* logp;
  float* entropy;
  float* top_logp;
  long long* top_ids;
  float2* stats;
  long long C;
  int labels64, top;
};

// A row's results but the alternatives; x is the row (global or shared memory).  Returns (m, log S).
template <class T>
__device__ __forceinline__ float2 write_scores(const ScoreArgs& a, long long r, const Soft& s, const T* x, long long t) {
  const bool bad = s.bad(), empty = !bad && s.S == 0.f;
  const float nan = CUDART_NAN_F;
  const float m = bad ? nan : (empty ? 0.f : s.m), logS = bad ? nan : (empty ? -CUDART_INF_F : logf(s.S));
  float lp = 0.f;
  if (t >= a.C)
    lp = nan;
  else if (t >= 0)
    lp = empty ? -CUDART_INF_F : (to_f32(x[t]) - m) - logS;
  a.logp[r] = lp;
  a.entropy[r] = bad ? nan : (empty ? 0.f : logS - s.A / s.S);
  if (a.stats) a.stats[r] = make_float2(m, bad ? nan : s.S);
  return make_float2(m, logS);
}

// Alternative k of row r: id -1 where there is none.
__device__ __forceinline__ void write_top(const ScoreArgs& a, long long r, int k, float v, long long id, float2 st) {
  a.top_ids[r * a.top + k] = id;
  a.top_logp[r * a.top + k] = st.y != st.y ? CUDART_NAN_F : (id < 0 ? -CUDART_INF_F : (v - st.x) - st.y);
}

// ---- many labels: rows in units of 16 bytes --------------------------------------------------------
template <class T>
using Vec16 = Unit<T, 16>;
// A row of C elements as `head` single ones up to the first 16-byte boundary, nv vectors and a tail.
template <class T>
struct RowSplit {
  int head, tail;
  long long nv;
  __device__ __forceinline__ RowSplit(const T* x, long long C) {
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15u);
    const long long h = off ? (16 - off) / (int)sizeof(T) : 0;
    head = (int)(h < C ? h : C);
    nv = (C - head) / Vec16<T>::E;
    tail = (int)(C - head - nv * Vec16<T>::E);
  }
};

// ---- one block (or a cluster of blocks) per row: many labels -------------------------------------
// TH threads: 256, or 128 for rows of up to BLOCK_FEW labels, where the steps behind the pass cost more than
// the pass and more rows at once hide them (6434 x 12487 bf16: 61 instead of 82 us).
constexpr long long BLOCK_FEW = 16384;
constexpr int SB_CAND = 256;      // candidates for the alternatives held in shared memory
constexpr int SB_CLUSTER = 8;

struct BlockTop {
  float v[TOP_MAX];
  long long id[TOP_MAX];
  int n;
};

// Whether (v, id) comes before (w, jd): the larger value, among equal ones the lower id.
__device__ __forceinline__ bool before(float v, long long id, float w, long long jd) {
  return v > w || (v == w && id < jd);
}

// The `top` best labels of the block's part of the row, best first.  Threads form 32 groups; the k-th
// largest of the 32 groups' maxima is a bound that at least k elements reach and few more (about 1.4 k
// for distinct random values), and only threads whose own maximum reaches it hold any: their elements
// alone are read again.  More candidates than fit (long runs of equal values): one pass for each
// alternative.
template <class T, int TH>
__device__ void block_top(const T* x, const RowSplit<T>& rs, long long lo, long long hi, bool ends, float tmax, int top,
                          BlockTop* out) {
  constexpr int N = Vec16<T>::E;
  __shared__ float s_g[32];
  __shared__ float s_T;
  __shared__ int s_nq, s_nc;
  __shared__ unsigned char s_q[TH];
  __shared__ float s_v[SB_CAND];
  __shared__ long long s_id[SB_CAND];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  float g = tmax;
  constexpr int GROUP = TH / 32;
#pragma unroll
  for (int d = GROUP / 2; d > 0; d >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
  if (lane % GROUP == 0) s_g[tid / GROUP] = g;
  if (tid == 0) s_nq = s_nc = 0;
  __syncthreads();
  if (wid == 0) {
    const float mine = s_g[lane];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) rank += before(s_g[i], i, mine, lane);
    if (rank == top - 1) s_T = mine;
  }
  __syncthreads();
  const float T0 = s_T;
  if (tmax >= T0) s_q[atomicAdd(&s_nq, 1)] = (unsigned char)tid;
  __syncthreads();
  auto consider = [&](float v, long long id) {
    if (v >= T0) {
      const int c = atomicAdd(&s_nc, 1);
      if (c < SB_CAND) {
        s_v[c] = v;
        s_id[c] = id;
      }
    }
  };
  const int rounds = (int)((hi - lo + TH - 1) / TH);
  const long long work = (long long)s_nq * rounds;
  const uint4* xv = reinterpret_cast<const uint4*>(x + rs.head);
  for (long long p = tid; p < work; p += TH) {
    const int q = (int)(p / rounds);
    const long long v = lo + s_q[q] + (p - (long long)q * rounds) * TH;
    if (v >= hi) continue;
    float w[N];
    Vec16<T>(__ldg(xv + v)).get(w);
#pragma unroll
    for (int e = 0; e < N; ++e) consider(w[e], rs.head + v * N + e);
  }
  const long long t0 = rs.head + rs.nv * N;
  if (ends && tid < rs.head) consider(to_f32(x[tid]), tid);
  if (ends && tid < rs.tail) consider(to_f32(x[t0 + tid]), t0 + tid);
  __syncthreads();
  const int nc = s_nc;
  if (nc <= SB_CAND) {
    for (int c = tid; c < nc; c += TH) {
      const float v = s_v[c];
      const long long id = s_id[c];
      int rank = 0;
      for (int i = 0; i < nc; ++i) rank += before(s_v[i], s_id[i], v, id);
      if (rank < top) {
        out->v[rank] = v;
        out->id[rank] = id;
      }
    }
    if (tid == 0) out->n = nc < top ? nc : top;
    __syncthreads();
    return;
  }
  float pv = CUDART_INF_F;
  long long pid = -1;
  int k = 0;
  for (; k < top; ++k) {
    float bv = -CUDART_INF_F;
    long long bi = -1;
    auto look = [&](float v, long long id) {
      if (before(pv, pid, v, id) && v > bv) bv = v, bi = id;
    };
    if (ends && tid < rs.head) look(to_f32(x[tid]), tid);
    for (long long v = lo + tid; v < hi; v += TH) {
      float w[N];
      Vec16<T>(__ldg(xv + v)).get(w);
#pragma unroll
      for (int e = 0; e < N; ++e) look(w[e], rs.head + v * N + e);
    }
    if (ends && tid < rs.tail) look(to_f32(x[t0 + tid]), t0 + tid);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, d);
      const long long oi = __shfl_xor_sync(0xffffffffu, bi, d);
      if (oi >= 0 && (bi < 0 || before(ov, oi, bv, bi))) bv = ov, bi = oi;
    }
    __syncthreads();
    if (lane == 0) s_v[wid] = bv, s_id[wid] = bi;
    __syncthreads();
    bv = s_v[0], bi = s_id[0];
    for (int w = 1; w < TH / 32; ++w)
      if (s_id[w] >= 0 && (bi < 0 || before(s_v[w], s_id[w], bv, bi))) bv = s_v[w], bi = s_id[w];
    if (bi < 0) break;
    if (tid == 0) out->v[k] = bv, out->id[k] = bi;
    pv = bv;
    pid = bi;
  }
  if (tid == 0) out->n = k;
  __syncthreads();
}

// One pass over the row with each thread's own running maximum and sums (UNROLL vectors in flight), then
// one merge; the blocks of a cluster take a part of the row each and the first one merges theirs through
// distributed shared memory.
template <class T, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) k_scores_block(const T* __restrict__ logits, long long stride, int cs,
                                                                ScoreArgs a) {
  constexpr int N = Vec16<T>::E, UNROLL = 4;
  constexpr int WARPS = TH / 32;
  __shared__ Soft s_soft[WARPS > SB_CLUSTER ? WARPS : SB_CLUSTER];
  __shared__ Soft s_all;
  __shared__ BlockTop s_top;
  __shared__ BlockTop s_tops[SB_CLUSTER];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const long long r = blockIdx.x / cs;
  const int rank = blockIdx.x % cs;
  const T* x = logits + r * stride;
  const RowSplit<T> rs(x, a.C);
  const long long lo = rs.nv * rank / cs, hi = rs.nv * (rank + 1) / cs;
  const uint4* xv = reinterpret_cast<const uint4*>(x + rs.head);
  const long long label = load_index(a.labels, a.labels64, r);
  Soft s;
  s.init();
  if (rank == 0) {
    float h = -CUDART_INF_F, t = -CUDART_INF_F;
    if (tid < rs.head) h = to_f32(x[tid]);
    if (tid < rs.tail) t = to_f32(x[rs.head + rs.nv * N + tid]);
    s.m = max_nan(s.m, max_nan(h, t));
    s.add(h);
    s.add(t);
  }
  auto take = [&](const Vec16<T>(&w)[UNROLL], int n) {
    float m = s.m;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (u < n) {
        float f[N];
        w[u].get(f);
#pragma unroll
        for (int e = 0; e < N; ++e) m = max_nan(m, f[e]);
      }
    if (!(m == s.m)) s.rebase(m);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (u < n) {
        float f[N];
        w[u].get(f);
#pragma unroll
        for (int e = 0; e < N; ++e) s.add(f[e]);
      }
  };
  constexpr int STEP = UNROLL * TH;
  const uint4* at = xv + lo + tid;
  int left = (int)(hi - lo) - tid;      // vectors from this thread's next one on, its own every TH-th of them
  Vec16<T> w[UNROLL], next[UNROLL];
  if (left > (UNROLL - 1) * TH) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) next[u].w = __ldg(at + u * TH);
    while (left > STEP + (UNROLL - 1) * TH) {
      // the next vectors are on their way while these are worked on
      at += STEP;
      left -= STEP;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        w[u] = next[u];
        next[u].w = __ldg(at + u * TH);
      }
      take(w, UNROLL);
    }
    take(next, UNROLL);
    at += STEP;
    left -= STEP;
  }
  if (left > 0) {
    const int n = (left + TH - 1) / TH;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (u < n) w[u].w = __ldg(at + u * TH);
    take(w, n);
  }
  const float tmax = s.m;
  s.reduce(32);
  if (lane == 0) s_soft[wid] = s;
  if (tid == 0) s_top.n = 0;
  __syncthreads();
  s = s_soft[lane % WARPS];
  s.reduce(WARPS);
  if (tid == 0) s_all = s;
  if (a.top > 0 && !s.bad()) block_top<T, TH>(x, rs, lo, hi, rank == 0, tmax, a.top, &s_top);
  if (cs == 1) {
    if (tid == 0) {
      const float2 st = write_scores(a, r, s, x, label);
      s_all.m = st.x, s_all.S = st.y;
    }
    if (a.top > 0) {
      __syncthreads();
      if (tid < a.top)
        write_top(a, r, tid, s_top.v[tid], tid < s_top.n ? s_top.id[tid] : -1, make_float2(s_all.m, s_all.S));
    }
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (rank == 0) {
    // every block's part here, then the best of all their bests by counting how many come before each
    if (wid == 0) {
      Soft o;
      o.init();
      if (lane < cs) o = *cluster.map_shared_rank(&s_all, lane);
      o.reduce(32);
      if (lane == 0) {
        const float2 st = write_scores(a, r, o, x, label);
        s_soft[0].m = st.x, s_soft[0].S = st.y;
      }
    }
    const int b = tid / TOP_MAX, k = tid % TOP_MAX;
    if (a.top > 0 && b < cs) {
      const BlockTop* t = cluster.map_shared_rank(&s_top, b);
      const int n = t->n;
      s_tops[b].v[k] = k < n ? t->v[k] : -CUDART_INF_F;
      s_tops[b].id[k] = k < n ? t->id[k] : -1;
      if (k == 0) s_tops[b].n = n;
    }
    __syncthreads();
    const float2 st = make_float2(s_soft[0].m, s_soft[0].S);
    int all = 0;
    if (a.top > 0 && st.y == st.y)
      for (int q = 0; q < cs; ++q) all += s_tops[q].n;
    if (a.top > 0 && b < cs && k < s_tops[b].n && st.y == st.y) {
      const float v = s_tops[b].v[k];
      const long long id = s_tops[b].id[k];
      int place = k;
      for (int q = 0; q < cs; ++q)
        if (q != b)
          for (int i = 0; i < s_tops[q].n; ++i) place += before(s_tops[q].v[i], s_tops[q].id[i], v, id);
      if (place < a.top) write_top(a, r, place, v, id, st);
    }
    if (tid < a.top && tid >= all) write_top(a, r, tid, -CUDART_INF_F, -1, st);
  }
  cluster.sync();
}

// ---- one thread per row: few labels ----------------------------------------------------------------
// A block's rows are one contiguous run of bytes: one bulk copy brings it into shared memory and, for the
// gradient, one takes it back out, so the memory sees nothing but full lines whatever the row size.  A thread
// then owns a row and nothing is shuffled.  Threads walk their rows in 4-byte words (two 16-bit logits) where
// rows are whole words; with an even number of words to a row each thread starts one word further, so that
// the warp's accesses fall into different banks.
template <bool TURN>
struct TileWalk {
  int n, at;        // units of a row; the next one
  __device__ __forceinline__ TileWalk(int n_) : n(n_), at(TURN ? (int)threadIdx.x % n_ : 0) {}
  __device__ __forceinline__ int next(int i) {
    if (!TURN) return i;
    const int j = at;
    at = at + 1 == n ? 0 : at + 1;
    return j;
  }
};

// The best K labels of a row in registers, best first.  A label passes down the places to the first that it
// comes before and takes it.  Walks in the order of the ids (TURN false) need no look at the ids: an equal value
// found later never comes before.
template <int K, bool TURN>
struct Best {
  float v[K > 0 ? K : 1];
  int id[K > 0 ? K : 1];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = -CUDART_INF_F, id[k] = -1;
  }
  // (a masked label never comes before the -inf of an empty place)
  __device__ __forceinline__ void add(float x, int j) {
    bool first = false;      // once it has a place, all behind move down by one
#pragma unroll
    for (int k = 0; k < K; ++k) {
      first = first || x > v[k] || (TURN && x == v[k] && j < id[k]);
      const float w = v[k];
      const int i = id[k];
      v[k] = first ? x : w;
      id[k] = first ? j : i;
      x = first ? w : x;
      j = first ? i : j;
    }
  }
};

// Copies rows [r0, r0 + n) into s (16-byte pieces by the bulk copy, the few bytes behind them by threads);
// false when the copy did not arrive (recorded in the status word): the results are then NaN and their ids -1,
// not what the memory held.
template <class T>
__device__ __forceinline__ bool load_tile(const T* logits, long long first, int count, T* s, uint64_t* bar) {
  const unsigned bytes = (unsigned)count * (unsigned)sizeof(T), whole = bytes & ~15u;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    if (whole > 0) {
      mbar_expect_tx(bar, whole);
      bulk_g2s(s, logits + first, whole, bar);
    }
  }
  for (int i = (int)(whole / sizeof(T)) + threadIdx.x; i < count; i += blockDim.x) s[i] = logits[first + i];
  __syncthreads();
  return whole == 0 || mbar_wait_bounded(bar, 0);
}

__device__ __forceinline__ void write_lost(const ScoreArgs& a, long long r) {
  a.logp[r] = a.entropy[r] = CUDART_NAN_F;
  if (a.stats) a.stats[r] = make_float2(CUDART_NAN_F, CUDART_NAN_F);
  for (int k = 0; k < a.top; ++k) write_top(a, r, k, 0.f, -1, make_float2(CUDART_NAN_F, CUDART_NAN_F));
}

constexpr int TILE_BEST = 4;      // alternatives kept in registers (K of them; K = 0: none or more than these)

template <class T, int VB, bool TURN, int K>
__global__ void __launch_bounds__(128) k_scores_tile(const T* __restrict__ logits, long long P, ScoreArgs a) {
  using U = Unit<T, VB>;
  extern __shared__ __align__(16) char smem[];
  __shared__ __align__(8) uint64_t bar;
  const int C = (int)a.C, units = C / U::E;
  const long long r0 = (long long)blockIdx.x * blockDim.x;
  const int rows = (int)(P - r0 < blockDim.x ? P - r0 : blockDim.x);
  T* s = reinterpret_cast<T*>(smem);
  const long long r = r0 + threadIdx.x;
  const long long label = threadIdx.x < rows ? load_index(a.labels, a.labels64, r) : -1;
  const bool arrived = load_tile(logits, r0 * C, rows * C, s, &bar);
  if (threadIdx.x >= rows) return;
  if (!arrived) {
    write_lost(a, r);
    return;
  }
  T* x = s + threadIdx.x * C;
  typename U::W* xu = reinterpret_cast<typename U::W*>(x);
  Soft4 sums;
  sums.init();
  Best<K, TURN> best;
  best.init();
  TileWalk<TURN> w(units);
#pragma unroll 4
  for (int i = 0; i < units; ++i) {
    const int j = w.next(i);
    float v[U::E];
    U(xu[j]).get(v);
#pragma unroll
    for (int e = 0; e < U::E; ++e) {
      sums.m = max_nan(sums.m, v[e]);
      best.add(v[e], j * U::E + e);
    }
  }
  constexpr int PER = 4 / U::E;
  int i = 0;
#pragma unroll 2
  for (; i + PER <= units; i += PER) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      float v[U::E];
      U(xu[w.next(i + q)]).get(v);
#pragma unroll
      for (int e = 0; e < U::E; ++e) sums.add(v[e], q * U::E + e);
    }
  }
  for (; i < units; ++i) {
    float v[U::E];
    U(xu[w.next(i)]).get(v);
#pragma unroll
    for (int e = 0; e < U::E; ++e) sums.add(v[e], e);
  }
  const Soft f = sums.total();
  const float2 st = write_scores(a, r, f, x, label);
  if constexpr (K > 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) write_top(a, r, k, best.v[k], f.bad() ? -1 : best.id[k], st);
  } else {
    // the best label left, taken out of the tile after each round
    for (int k = 0; k < a.top; ++k) {
      float bv = -CUDART_INF_F;
      int bi = -1;
      if (!f.bad())
#pragma unroll 4
        for (int i = 0; i < units; ++i) {
          const int j = w.next(i);
          float v[U::E];
          U(xu[j]).get(v);
#pragma unroll
          for (int e = 0; e < U::E; ++e) {
            const int id = j * U::E + e;
            if (v[e] > bv || (TURN && v[e] == bv && id < bi)) bv = v[e], bi = id;
          }
        }
      if (bi >= 0) x[bi] = from_f32<T>(-CUDART_INF_F);
      write_top(a, r, k, bv, bi, st);
    }
  }
}

// ---- one warp per row: rows of up to 512 labels that no tile takes -------------------------------------
// The row stays in registers, SLOTS logits a lane (twice as many labels: 73 us for 40000 x 1000 fp32, 58 by the
// kernel for longer rows; for 300 such rows 4.5 and 5.5, in bf16 6.4 and 5.3; 39 and 42 for 40000 x 500).  The
// k-th largest of the lanes' maxima is a bound that at least k logits reach and few more; those are gathered, a
// lane for each, and placed by counting how many come before.  More than 32 of them (equal values): one round
// over the registers for each alternative.
constexpr long long WARP_ROW_MAX = 512;

// Unsigned numbers in the order of the floats (no NaN; -0 counts as 0).
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The k-th largest of the lanes' numbers.
__device__ __forceinline__ float kth_of_lanes(float mine, int k) {
  unsigned key = order_key(mine), kth = 0;
  for (int i = 0; i < k; ++i) {
    kth = __reduce_max_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == __ffs(__ballot_sync(0xffffffffu, key == kth)) - 1) key = 0;
  }
  return order_value(kth);
}
// Writes the row's alternatives from n <= 32 candidates that hold them, a lane for each.
__device__ __forceinline__ void place_candidates(const ScoreArgs& a, long long r, int n, const float* v, const int* id,
                                                 float2 st) {
  const int lane = threadIdx.x & 31;
  if (lane < n) {
    int place = 0;
    for (int i = 0; i < n; ++i) place += before(v[i], id[i], v[lane], id[lane]);
    if (place < a.top) write_top(a, r, place, v[lane], id[lane], st);
  }
  if (lane >= n && lane < a.top) write_top(a, r, lane, 0.f, -1, st);
}
// The best of the lanes' labels, in all of them.
__device__ __forceinline__ void best_of_lanes(float& v, int& id) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, d);
    const int oi = __shfl_xor_sync(0xffffffffu, id, d);
    if (before(ov, oi, v, id)) v = ov, id = oi;
  }
}

template <class T, int SLOTS>
__global__ void __launch_bounds__(256) k_scores_warp(const T* __restrict__ logits, long long P, long long stride,
                                                     ScoreArgs a) {
  __shared__ float s_v[8][32];
  __shared__ int s_id[8][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long r = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (r >= P) return;
  const T* x = logits + r * stride;
  const int C = (int)a.C;
  const long long label = load_index(a.labels, a.labels64, r);
  float v[SLOTS];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) v[i] = i * 32 + lane < C ? to_f32(x[i * 32 + lane]) : -CUDART_INF_F;
  Soft s;
  s.init();
  float most = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) most = max_nan(most, v[i]);
  s.m = max_nan(s.m, most);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s.m = max_nan(s.m, __shfl_xor_sync(0xffffffffu, s.m, d));
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
    if (i * 32 < C) s.add(v[i]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, d);
    s.A += __shfl_xor_sync(0xffffffffu, s.A, d);
  }
  float2 st;
  if (lane == 0) st = write_scores(a, r, s, x, label);
  if (a.top == 0) return;
  st.x = __shfl_sync(0xffffffffu, st.x, 0);
  st.y = __shfl_sync(0xffffffffu, st.y, 0);
  if (s.bad()) {
    if (lane < a.top) write_top(a, r, lane, 0.f, -1, st);
    return;
  }
  const float bound = kth_of_lanes(most, a.top);
  int n = 0;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const bool c = v[i] >= bound && v[i] > -CUDART_INF_F;
    const unsigned b = __ballot_sync(0xffffffffu, c);
    if (b) {
      const int at = n + __popc(b & ((1u << lane) - 1));
      if (c && at < 32) {
        s_v[wid][at] = v[i];
        s_id[wid][at] = i * 32 + lane;
      }
      n += __popc(b);
    }
  }
  __syncwarp();
  if (n <= 32) {
    place_candidates(a, r, n, s_v[wid], s_id[wid], st);
    return;
  }
  float pv = CUDART_INF_F;
  int pid = -1;
  for (int k = 0; k < a.top; ++k) {
    float bv = -CUDART_INF_F;
    int bi = C;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (before(pv, pid, v[i], i * 32 + lane) && v[i] > bv) bv = v[i], bi = i * 32 + lane;
    best_of_lanes(bv, bi);
    if (lane == 0) write_top(a, r, k, bv, bi < C ? bi : -1, st);
    pv = bv;
    pid = bi;
  }
}

// Longer rows of a warp stay in memory: one pass with each lane's own running sums, then the lanes whose maximum
// reaches the bound read theirs again (from a cache, mostly) for the candidates.
// Rows of up to 1024 labels, and of up to 4096 where there are enough to keep the SMs busy; others take a block each
// (20000 x 1100 fp16 top 8: 34 us, 99 by blocks; 4000 x 8000 fp32: 47 and 35; 1200 x 2000 fp32: 9 and 8).
constexpr long long WARP_LONG_FEW = 1024;
constexpr long long WARP_LONG_MAX = 4096;
constexpr long long WARP_LONG_ROWS = 148 * 12;
static bool warp_rows(long long P, long long C) { return C <= WARP_LONG_FEW || (C <= WARP_LONG_MAX && P >= WARP_LONG_ROWS); }

template <class T>
__global__ void __launch_bounds__(256, 4) k_scores_warp_long(const T* __restrict__ logits, long long P, long long stride,
                                                             ScoreArgs a) {
  constexpr int N = Vec16<T>::E, UNROLL = 4;
  __shared__ float s_v[8][32];
  __shared__ int s_id[8][32], s_n[8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long r = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (r >= P) return;
  const T* x = logits + r * stride;
  const RowSplit<T> rs(x, a.C);
  const int nv = (int)rs.nv, t0 = rs.head + nv * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + rs.head);
  const long long label = load_index(a.labels, a.labels64, r);
  const float h = lane < rs.head ? to_f32(x[lane]) : -CUDART_INF_F;
  const float t = lane < rs.tail ? to_f32(x[t0 + lane]) : -CUDART_INF_F;
  Soft s;
  s.init();
  s.m = max_nan(s.m, max_nan(h, t));
  s.add(h);
  s.add(t);
  for (int v0 = lane; v0 < nv; v0 += 32 * UNROLL) {
    Vec16<T> w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + 32 * u < nv) w[u].w = __ldg(xv + v0 + 32 * u);
    float m = s.m;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + 32 * u < nv) {
        float f[N];
        w[u].get(f);
#pragma unroll
        for (int e = 0; e < N; ++e) m = max_nan(m, f[e]);
      }
    if (!(m == s.m)) s.rebase(m);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + 32 * u < nv) {
        float f[N];
        w[u].get(f);
#pragma unroll
        for (int e = 0; e < N; ++e) s.add(f[e]);
      }
  }
  const float most = s.m;
  s.reduce(32);
  float2 st;
  if (lane == 0) st = write_scores(a, r, s, x, label);
  if (a.top == 0) return;
  st.x = __shfl_sync(0xffffffffu, st.x, 0);
  st.y = __shfl_sync(0xffffffffu, st.y, 0);
  if (s.bad()) {
    if (lane < a.top) write_top(a, r, lane, 0.f, -1, st);
    return;
  }
  const float bound = kth_of_lanes(most, a.top);
  if (lane == 0) s_n[wid] = 0;
  __syncwarp();
  auto each = [&](auto look) {
    if (lane < rs.head) look(h, lane);
#pragma unroll 2
    for (int v = lane; v < nv; v += 32) {
      float f[N];
      Vec16<T>(__ldg(xv + v)).get(f);
#pragma unroll
      for (int e = 0; e < N; ++e) look(f[e], rs.head + v * N + e);
    }
    if (lane < rs.tail) look(t, t0 + lane);
  };
  // (the bound is at least the lowest number: masked labels are below)
  if (most >= bound)
    each([&](float v, int id) {
      if (v >= bound) {
        const int at = atomicAdd(&s_n[wid], 1);
        if (at < 32) {
          s_v[wid][at] = v;
          s_id[wid][at] = id;
        }
      }
    });
  __syncwarp();
  const int n = s_n[wid];
  if (n <= 32) {
    place_candidates(a, r, n, s_v[wid], s_id[wid], st);
    return;
  }
  float pv = CUDART_INF_F;
  int pid = -1;
  for (int k = 0; k < a.top; ++k) {
    float bv = -CUDART_INF_F;
    int bi = (int)a.C;
    each([&](float v, int id) {
      if (before(pv, pid, v, id) && v > bv) bv = v, bi = id;
    });
    best_of_lanes(bv, bi);
    if (lane == 0) write_top(a, r, k, bv, bi < a.C ? bi : -1, st);
    pv = bv;
    pid = bi;
  }
}

// ---- the gradient -----------------------------------------------------------------------------------
struct GradArgs {
  const void* labels;
  const float2* stats;
  const float* entropy;
  const long long* top_ids;
  const float* g_logp;
  const float* g_entropy;
  const float* g_top;
  long long C;
  int labels64, top;
};

// With d = x - m:  dx = p (alpha - g_H d),  p = exp(d) / S,  alpha = -total - g_H (H - log S); alpha and g_H are
// held divided by S.
struct RowGrad {
  float m, alpha, gh, gl;
  long long t;
  bool zero;      // nothing comes in: zeros, whatever the row holds
  bool empty;     // masked labels only: zeros
  // What alternative k adds to the total: its gradient if there is one.  A row that holds a NaN or +inf has none,
  // but NaN log probabilities in their place: a gradient that comes in for one is lost in the NaN.
  static __device__ __forceinline__ float top_term(const GradArgs& a, long long r, int k, bool bad) {
    const float g = a.g_top[r * a.top + k];
    return a.top_ids[r * a.top + k] >= 0 ? g : (bad && g != 0.f ? CUDART_NAN_F : 0.f);
  }
  // By one thread, or by a warp that asks together (the alternatives' gradients a lane each).
  template <bool WARP>
  __device__ __forceinline__ RowGrad(const GradArgs& a, long long r, std::bool_constant<WARP>) {
    const float2 st = a.stats[r];
    const float H = a.entropy[r], S = st.y;
    const bool bad = S != S;
    gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    t = load_index(a.labels, a.labels64, r);
    gl = a.g_logp ? a.g_logp[r] : 0.f;
    float of_tops = 0.f;
    if (a.g_top) {
      if constexpr (WARP) {
        const int lane = threadIdx.x & 31;
        if (lane < a.top) of_tops = top_term(a, r, lane, bad);
#pragma unroll
        for (int d = TOP_MAX / 2; d > 0; d >>= 1) of_tops += __shfl_xor_sync(0xffffffffu, of_tops, d);
        of_tops = __shfl_sync(0xffffffffu, of_tops, 0);
      } else {
        for (int k = 0; k < a.top; ++k) of_tops += top_term(a, r, k, bad);
      }
    }
    if (t < 0) gl = 0.f;
    if (t >= a.C && gl != 0.f) gl = CUDART_NAN_F;
    const float total = gl + of_tops;
    m = st.x;
    zero = total == 0.f && gh == 0.f;
    empty = S == 0.f;
    const float over = __frcp_rn(S);
    alpha = bad ? CUDART_NAN_F : (gh != 0.f ? -total - gh * (H - logf(S)) : -total) * over;
    gh *= over;
    if (empty) gl = 0.f;
    if (zero || empty) m = 0.f, alpha = 0.f, gh = 0.f;
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float d = fmaxf(x - m, D_MIN);
    return exp2_fast(d * LOG2E) * fmaf(-gh, d, alpha);
  }
  // The gradient at label j, which the given label or alternatives hit.
  __device__ __forceinline__ float special(const GradArgs& a, long long r, long long j, float x) const {
    float g = zero || empty ? 0.f : (*this)(x);
    if (j == t) g += gl;
    if (a.g_top && !empty)
      for (int k = 0; k < a.top; ++k)
        if (a.top_ids[r * a.top + k] == j) g += a.g_top[r * a.top + k];
    return g;
  }
};

constexpr int GB_THREADS = 256;
constexpr int GB_UNROLL = 4;
constexpr long long GB_STEP = (long long)GB_THREADS * GB_UNROLL;

// Blocks of one row each (blockIdx.x: row, blockIdx.y: a part of `steps` steps of its vectors, the next step's
// on their way while this one's are worked on); the labels whose gradient has a term of its own are stored
// last, behind a barrier.
template <class T, bool SAME>
__global__ void __launch_bounds__(GB_THREADS) k_scores_grad_block(const T* __restrict__ logits, long long stride, int steps,
                                                                  GradArgs a, T* __restrict__ glogits) {
  constexpr int N = Vec16<T>::E;
  const long long r = blockIdx.x;
  const T* x = logits + r * stride;
  T* gx = glogits + r * a.C;
  const RowSplit<T> rs(gx, a.C);
  const long long lo = blockIdx.y * steps * GB_STEP, hi = lo + steps * GB_STEP < rs.nv ? lo + steps * GB_STEP : rs.nv;
  const long long j0 = blockIdx.y == 0 ? 0 : rs.head + lo * N;
  const long long j1 = blockIdx.y == gridDim.y - 1 ? a.C : rs.head + hi * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + rs.head);
  uint4* gv = reinterpret_cast<uint4*>(gx + rs.head);
  Vec16<T> next[GB_UNROLL];
  auto fetch = [&](long long v0) {
#pragma unroll
    for (int u = 0; u < GB_UNROLL; ++u) {
      const long long v = v0 + u * GB_THREADS;
      if (v < hi) {
        if constexpr (SAME) {
          next[u].w = __ldcs(xv + v);
        } else {
          float f[N];
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] = to_f32(x[rs.head + v * N + e]);
          next[u].set(f);
        }
      }
    }
  };
  // the first step's vectors and the row's numbers are on their way together
  fetch(lo + threadIdx.x);
  const RowGrad g(a, r, std::true_type());
  const bool none = g.zero || g.empty;
  for (long long v0 = lo + threadIdx.x; v0 < hi; v0 += GB_STEP) {
    Vec16<T> w[GB_UNROLL];
#pragma unroll
    for (int u = 0; u < GB_UNROLL; ++u) w[u] = next[u];
    if (!none) fetch(v0 + GB_STEP);
#pragma unroll
    for (int u = 0; u < GB_UNROLL; ++u) {
      const long long v = v0 + u * GB_THREADS;
      if (v < hi) {
        float f[N];
        w[u].get(f);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = none ? 0.f : g(f[e]);
        w[u].set(f);
        __stcs(gv + v, w[u].w);
      }
    }
  }
  if (blockIdx.y == 0 && threadIdx.x < rs.head)
    gx[threadIdx.x] = from_f32<T>(none ? 0.f : g(to_f32(x[threadIdx.x])));
  if (blockIdx.y == gridDim.y - 1 && threadIdx.x < rs.tail) {
    const long long j = a.C - rs.tail + threadIdx.x;
    gx[j] = from_f32<T>(none ? 0.f : g(to_f32(x[j])));
  }
  __syncthreads();
  if (threadIdx.x <= (a.g_top ? a.top : 0)) {
    const long long j = threadIdx.x == 0 ? g.t : a.top_ids[r * a.top + threadIdx.x - 1];
    if (j >= j0 && j < j1) gx[j] = from_f32<T>(g.special(a, r, j, to_f32(x[j])));
  }
}

// A warp for each row, in 16-byte units where the logits' line up with the gradient's.
template <class T, bool SAME>
__global__ void __launch_bounds__(256) k_scores_grad_warp(const T* __restrict__ logits, long long P, long long stride,
                                                          GradArgs a, T* __restrict__ glogits) {
  constexpr int N = Vec16<T>::E, UNROLL = 4;
  const int lane = threadIdx.x & 31;
  const long long r = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (r >= P) return;
  const T* x = logits + r * stride;
  T* gx = glogits + r * a.C;
  const int C = (int)a.C;
  const RowGrad g(a, r, std::true_type());
  const bool none = g.zero || g.empty;
  if constexpr (SAME) {
    const RowSplit<T> rs(gx, C);
    const int nv = (int)rs.nv, t0 = rs.head + nv * N;
    const uint4* xv = reinterpret_cast<const uint4*>(x + rs.head);
    uint4* gv = reinterpret_cast<uint4*>(gx + rs.head);
    for (int v0 = lane; v0 < nv; v0 += 32 * UNROLL) {
      Vec16<T> w[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (v0 + 32 * u < nv && !none) w[u].w = __ldg(xv + v0 + 32 * u);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (v0 + 32 * u < nv) {
          float f[N];
          w[u].get(f);
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] = none ? 0.f : g(f[e]);
          w[u].set(f);
          gv[v0 + 32 * u] = w[u].w;
        }
    }
    if (lane < rs.head) gx[lane] = from_f32<T>(none ? 0.f : g(to_f32(x[lane])));
    if (lane < rs.tail) gx[t0 + lane] = from_f32<T>(none ? 0.f : g(to_f32(x[t0 + lane])));
  } else {
    for (int j = lane; j < C; j += 32) gx[j] = from_f32<T>(none ? 0.f : g(to_f32(x[j])));
  }
  __syncwarp();
  if (lane <= (a.g_top ? a.top : 0)) {
    const long long j = lane == 0 ? g.t : a.top_ids[r * a.top + lane - 1];
    if (j >= 0 && j < C) gx[j] = from_f32<T>(g.special(a, r, j, to_f32(x[j])));
  }
}

template <class T, int VB, bool TURN>
__global__ void __launch_bounds__(128) k_scores_grad_tile(const T* __restrict__ logits, long long P, GradArgs a,
                                                          T* __restrict__ glogits) {
  using U = Unit<T, VB>;
  extern __shared__ __align__(16) char smem[];
  __shared__ __align__(8) uint64_t bar;
  const int C = (int)a.C, units = C / U::E;
  const long long r0 = (long long)blockIdx.x * blockDim.x;
  const int rows = (int)(P - r0 < blockDim.x ? P - r0 : blockDim.x);
  T* s = reinterpret_cast<T*>(smem);
  const long long r = r0 + threadIdx.x;
  const long long mine = threadIdx.x < rows ? r : r0;
  const RowGrad g(a, mine, std::false_type());
  const bool arrived = load_tile(logits, r0 * C, rows * C, s, &bar);
  if (arrived && threadIdx.x < rows) {
    T* x = s + threadIdx.x * C;
    typename U::W* xu = reinterpret_cast<typename U::W*>(x);
    const bool none = g.zero || g.empty;
    // the labels with a term of their own, before their logits are overwritten
    const int extra = a.g_top ? a.top : 0;
    const float at_label = g.t >= 0 && g.t < C ? g.special(a, r, g.t, to_f32(x[g.t])) : 0.f;
    float own[TOP_MAX];
    for (int k = 0; k < extra; ++k) {
      const long long j = a.top_ids[r * a.top + k];
      own[k] = j >= 0 && j < C ? g.special(a, r, j, to_f32(x[j])) : 0.f;
    }
    TileWalk<TURN> w(units);
    if (none) {
      U zero;
      float v[U::E];
#pragma unroll
      for (int e = 0; e < U::E; ++e) v[e] = 0.f;
      zero.set(v);
      for (int i = 0; i < units; ++i) xu[w.next(i)] = zero.w;
    } else {
#pragma unroll 4
      for (int i = 0; i < units; ++i) {
        const int j = w.next(i);
        U u(xu[j]);
        float v[U::E];
        u.get(v);
#pragma unroll
        for (int e = 0; e < U::E; ++e) v[e] = g(v[e]);
        u.set(v);
        xu[j] = u.w;
      }
    }
    if (g.t >= 0 && g.t < C) x[g.t] = from_f32<T>(at_label);
    for (int k = 0; k < extra; ++k) {
      const long long j = a.top_ids[r * a.top + k];
      if (j >= 0 && j < C) x[j] = from_f32<T>(own[k]);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  const int count = rows * C;
  if (!__syncthreads_and(arrived)) {
    for (int i = threadIdx.x; i < count; i += blockDim.x) glogits[r0 * C + i] = from_f32<T>(CUDART_NAN_F);
    return;
  }
  const unsigned whole = ((unsigned)count * (unsigned)sizeof(T)) & ~15u;
  if (threadIdx.x == 0 && whole > 0) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(glogits + r0 * C), "r"(smem_u32(s)),
                 "r"(whole)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  for (int i = (int)(whole / sizeof(T)) + threadIdx.x; i < count; i += blockDim.x) glogits[r0 * C + i] = s[i];
}

// Calls f with the unit size and whether the walk turns, for rows of C elements of T.
template <class T, class F>
static int with_tile(long long C, F f) {
  using B4 = std::integral_constant<int, 4>;
  using BT = std::integral_constant<int, (int)sizeof(T)>;
  if (C * sizeof(T) % 8 == 0) return f(B4(), std::true_type());
  if (C * sizeof(T) % 4 == 0) return f(B4(), std::false_type());
  return f(BT(), std::false_type());
}

// Rows of up to TILE_ROW_BYTES that lie one behind the other from a 16-byte boundary on take a thread each, from
// TILE_ROWS rows on: fewer leave SMs idle that a warp for each row keeps busy (13938 x 60 fp16 top 4: 12 us by
// tiles, 10 by warps).
constexpr long long TILE_ROW_BYTES = 512;
constexpr long long TILE_ROWS = 148 * 256;
static bool tile_rows(long long P, long long C, size_t elem, long long stride, const void* x, const void* gx) {
  return P >= TILE_ROWS && C * (long long)elem <= TILE_ROW_BYTES && stride == C && aligned16(x) && aligned16(gx);
}
static int tile_threads(long long C, size_t elem) { return C * (long long)elem <= 128 ? 128 : 64; }

static int check_labels(long long P, long long C, int type, int top) {
  TTS_REQUIRE(type >= TTS_ROW_F32 && type <= TTS_ROW_F16, "unknown row type");
  TTS_REQUIRE(P >= 0 && P < (1ll << 31), "the number of rows must be below 2^31");
  TTS_REQUIRE(C >= 1 && C <= (1ll << 27), "the number of labels must be 1 to 2^27");
  TTS_REQUIRE(top >= 0 && top <= TOP_MAX, "top must be 0 to 16");
  return TTS_OK;
}

template <class T>
static int launch_scores_block(const T* x, long long P, long long stride, const ScoreArgs& a, cudaStream_t st) {
  // few rows: a cluster of blocks for each, as long as that fills the SMs and leaves every block 2048 labels
  int cs = 1;
  while (cs < SB_CLUSTER && P * cs * 2 <= 148 * 4 && a.C / (cs * 2) >= 2048) cs *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(P * cs));
  const bool few = a.C <= BLOCK_FEW && cs == 1;
  cfg.blockDim = dim3(few ? 128 : 256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cs > 1 ? 1 : 0;
  const cudaError_t rc = few ? cudaLaunchKernelEx(&cfg, k_scores_block<T, 128>, x, stride, cs, a)
                             : cudaLaunchKernelEx(&cfg, k_scores_block<T, 256>, x, stride, cs, a);
  if (rc != cudaSuccess) return check_launch("label_log_probs (block per row)");
  return TTS_OK;
}

}  // namespace tts

using namespace tts;

extern "C" int tts_label_log_probs(const void* logits, long long P, long long C, long long row_stride, int type,
                                   const void* labels, int labels64, int top, float* logp, float* entropy,
                                   float* top_logp, int64_t* top_ids, float* stats, void* stream) {
  if (int rc = check_labels(P, C, type, top)) return rc;
  if (P == 0) return TTS_OK;
  TTS_REQUIRE(logits && labels && logp && entropy && (top == 0 || (top_logp && top_ids)),
              "null label_log_probs argument");
  TTS_REQUIRE(aligned_to(row_elem(type), {logits}) && aligned_to(labels64 ? 8 : 4, {labels}) &&
                  aligned_to(4, {logp, entropy, top_logp}) && aligned_to(8, {top_ids, stats}),
              "logits, labels and results must be aligned to their elements, stats to 8 bytes");
  const ScoreArgs a{labels, logp, entropy, top_logp, reinterpret_cast<long long*>(top_ids), reinterpret_cast<float2*>(stats),
                    C, labels64, top};
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    const T* x = static_cast<const T*>(logits);
    if (tile_rows(P, C, sizeof(T), row_stride, x, nullptr)) {
      const int n = tile_threads(C, sizeof(T));
      const size_t bytes = (size_t)n * C * sizeof(T);
      const unsigned grid = (unsigned)((P + n - 1) / n);
      with_tile<T>(C, [&](auto vb, auto turn) {
        constexpr int VB = decltype(vb)::value;
        constexpr bool TURN = decltype(turn)::value;
        const auto launch = [&](auto k) {
          k_scores_tile<T, VB, TURN, decltype(k)::value><<<grid, n, bytes, as_stream(stream)>>>(x, P, a);
        };
        switch (top <= TILE_BEST ? top : 0) {
          case 1: launch(std::integral_constant<int, 1>()); break;
          case 2: launch(std::integral_constant<int, 2>()); break;
          case 3: launch(std::integral_constant<int, 3>()); break;
          case 4: launch(std::integral_constant<int, 4>()); break;
          default: launch(std::integral_constant<int, 0>()); break;
        }
        return TTS_OK;
      });
    } else if (C <= WARP_ROW_MAX) {
      const unsigned grid = (unsigned)((P + 7) / 8);
      if (C <= 256)
        k_scores_warp<T, 8><<<grid, 256, 0, as_stream(stream)>>>(x, P, row_stride, a);
      else
        k_scores_warp<T, 16><<<grid, 256, 0, as_stream(stream)>>>(x, P, row_stride, a);
    } else if (warp_rows(P, C)) {
      k_scores_warp_long<T><<<(unsigned)((P + 7) / 8), 256, 0, as_stream(stream)>>>(x, P, row_stride, a);
    } else if (int rc = launch_scores_block<T>(x, P, row_stride, a, as_stream(stream))) {
      return rc;
    }
    return check_launch("label_log_probs");
  });
}

extern "C" int tts_label_log_probs_bwd(const void* logits, long long P, long long C, long long row_stride, int type,
                                       const void* labels, int labels64, int top, const float* stats,
                                       const float* entropy, const int64_t* top_ids, const float* g_logp,
                                       const float* g_entropy, const float* g_top, void* glogits, void* stream) {
  if (int rc = check_labels(P, C, type, top)) return rc;
  if (P == 0) return TTS_OK;
  TTS_REQUIRE(logits && labels && stats && entropy && glogits && (!g_top || top == 0 || top_ids),
              "null label_log_probs_bwd argument");
  TTS_REQUIRE(aligned_to(row_elem(type), {logits, glogits}) && aligned_to(labels64 ? 8 : 4, {labels}) &&
                  aligned_to(4, {entropy, g_logp, g_entropy, g_top}) && aligned_to(8, {top_ids, stats}),
              "logits, labels and gradients must be aligned to their elements, stats to 8 bytes");
  TTS_REQUIRE(!rows_overlap(logits, P, C, row_stride, row_elem(type), glogits, P * C * (long long)row_elem(type)),
              "the gradient must not overlap the logits");
  const GradArgs a{labels, reinterpret_cast<const float2*>(stats), entropy, reinterpret_cast<const long long*>(top_ids),
                   g_logp, g_entropy, top > 0 ? g_top : nullptr, C, labels64, top};
  cudaStream_t st = as_stream(stream);
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    const T* x = static_cast<const T*>(logits);
    T* gx = static_cast<T*>(glogits);
    if (tile_rows(P, C, sizeof(T), row_stride, x, gx)) {
      const int n = tile_threads(C, sizeof(T));
      const size_t bytes = (size_t)n * C * sizeof(T);
      const unsigned grid = (unsigned)((P + n - 1) / n);
      with_tile<T>(C, [&](auto vb, auto turn) {
        k_scores_grad_tile<T, decltype(vb)::value, decltype(turn)::value><<<grid, n, bytes, st>>>(x, P, a, gx);
        return TTS_OK;
      });
    } else {
      // the logits' 16-byte vectors line up with the gradient's when both start on the same offset in every row
      const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(gx)) & 15u) == 0 &&
                        (row_stride - C) * (long long)sizeof(T) % 16 == 0;
      if (warp_rows(P, C)) {
        const unsigned grid = (unsigned)((P + 7) / 8);
        if (same)
          k_scores_grad_warp<T, true><<<grid, 256, 0, st>>>(x, P, row_stride, a, gx);
        else
          k_scores_grad_warp<T, false><<<grid, 256, 0, st>>>(x, P, row_stride, a, gx);
        return check_launch("label_log_probs_bwd");
      }
      // a few steps to a block where that leaves blocks enough for the SMs
      const long long parts = (C / Vec16<T>::E + GB_STEP - 1) / GB_STEP;
      int steps = 1;
      while (steps < 8 && steps < parts && P * parts / (steps * 2) >= 148 * 16) steps *= 2;
      const dim3 grid((unsigned)P, (unsigned)((parts + steps - 1) / steps));
      if (same)
        k_scores_grad_block<T, true><<<grid, GB_THREADS, 0, st>>>(x, row_stride, steps, a, gx);
      else
        k_scores_grad_block<T, false><<<grid, GB_THREADS, 0, st>>>(x, row_stride, steps, a, gx);
    }
    return check_launch("label_log_probs_bwd");
  });
}
