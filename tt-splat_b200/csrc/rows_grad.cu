// The gradient of the row lookup over its uses in row order:
//
//   gtable_v = sum over the uses n of row v, ascending, of f_n gout_n,   gweight_n = scale <gout_n, table_v>
//
// A group of lanes takes a chunk of L consecutive sorted uses, so that rows with many uses and rows with few
// cost the same.  It keeps the running row in fp32 registers and writes it when the row changes.  A row
// belongs to the chunk in which it begins, which follows it into the next chunk; the next one skips that
// part.  Only a row that goes on behind the next chunk too is split: every chunk leaves its part of it as a
// partial sum, and a second kernel adds the parts in order.  A block brings its chunks' (row, use) pairs and
// factors into shared memory first, so that nothing but gradient rows is waited for afterwards; they are read
// once, in units of up to 16 bytes, several uses in flight.
#include <algorithm>

#include "rows.cuh"

namespace tts {

constexpr int GT = 256;

// Blocks to an SM for rows of per_lane units of vb bytes to a lane, with or without the weights' gradient, which
// also holds the table's row: as many as the registers allow without spills (320000
// lookups of 45 fp16 with weights: 27 us at two, 39 at three).
constexpr int grad_blocks(int per_lane, int vb, bool weights) {
  const int words = per_lane * (vb < 4 ? 1 : vb / 4) * (weights ? 2 : 1);
  return words <= 4 ? 3 : (words <= (weights ? 16 : 8) ? 2 : 1);
}

// Uses of a chunk: the waves of blocks that make it nearest to L_MEAN, and then what fills them, in whole steps
// of 8 (320000 lookups of 45 fp32: 33 us in one wave, 41 at 64 uses and 1.1 waves).  At most 8 for each lane of a
// group, which bounds a block's uses by BLOCK_USES.
constexpr int L_MIN = 8, L_MEAN = 96, L_MAX = 128;
constexpr int BLOCK_USES = 8 * GT;
static int chunk_len(long long N, int lanes, int blocks) {
  const long long wave = 148ll * blocks * (GT / lanes), most = std::min(8 * lanes, L_MAX);
  const long long waves = std::max({1ll, (N + wave * L_MEAN / 2) / (wave * L_MEAN), (N + wave * most - 1) / (wave * most)});
  const long long l = ((N + waves * wave - 1) / (waves * wave) + 7) / 8 * 8;
  return (int)std::min(most, std::max<long long>(L_MIN, l));
}
static long long chunks_of(long long N, int l) { return (N + l - 1) / l; }

struct GradShape {
  long long units;        // of a row
  int lanes, per_lane;    // of a group; lanes * per_lane units a column part
  int parts;              // column parts
};
// Small units are packed 2 to 4 to a lane, so that a warp's steps serve two rows or four (without weights, 300000
// lookups of 63 fp32: 31 us, 44 by one unit a lane in two column parts; with them, 320000 of 31: 27 and 34, 700000
// of 9: 37 and 43; fewer lanes yet lose).  Large ones take one a lane, in column parts where that is not enough
// (134k lookups of 328 fp32: 52 us, 64 with 4 units a lane), unless the weights' sums need the row in one warp.
static GradShape grad_shape(long long C, int elem, int vb, bool weights) {
  GradShape g;
  g.units = C * elem / vb;
  g.lanes = 1;
  while (g.lanes < 32 && g.lanes < g.units) g.lanes *= 2;
  g.per_lane = 1;
  if (vb == 16 && weights && g.units > 32) {
    g.per_lane = g.units <= 64 ? 2 : 4;
  } else if (vb < 16 && g.units > 8) {
    g.lanes = g.units <= 24 ? 8 : (g.units <= 64 ? 16 : 32);
    const long long per = (g.units + g.lanes - 1) / g.lanes;
    g.per_lane = per < 4 ? (int)per : 4;
  }
  g.parts = (int)((g.units + g.lanes * g.per_lane - 1) / (g.lanes * g.per_lane));
  return g;
}

struct RowsGradArgs {
  RowUses u;
  const uint2* s;
  const unsigned* n;
  uint8_t* used;
  long long C, table_stride, gout_stride, chunks;
  int L, lanes, units, unit;
  float* gweight;
  float* partial;        // [2 * chunks][C]: the chunk's part of a split row begun before it; of one begun in it
};

// What a chunk has to do with the rows at its ends; key(i) is the row of sorted use i, R outside 0 .. N - 1.
struct ChunkEnds {
  long long i0, i1;
  unsigned first, last;
  bool skip;       // its first row belongs to the chunk before
  bool open;       // its first row is split and began before it
  bool split;      // its last row is split and goes on behind it
  bool follow;     // its last row goes on in the next chunk and ends there
  template <class K>
  __device__ __forceinline__ ChunkEnds(long long chunk, long long N, long long L, unsigned R, K key) {
    i0 = chunk * L;
    i1 = i0 + L < N ? i0 + L : N;
    first = key(i0);
    last = key(i1 - 1);
    const unsigned after = key(i1);
    const bool begun = first < R && key(i0 - 1) == first;           // the first row began before the chunk,
    const bool through = begun && last == first && after == first;  // and goes on behind it
    const bool longer = begun && key(i0 - L - 1) == first;          // or began before the last one already
    open = begun && (through || longer);
    skip = begun && !open;
    const bool on = last < R && after == last;
    split = on && (through || key(i1 + L) == last);
    follow = on && !split;
  }
};

// Sums v[0 .. 7] over the group's lanes (8 or more, named by mask): each step adds and halves what a lane holds,
// 7 shuffles and the plain steps behind them instead of 8 for each value.  Returns the sum of value j in the
// lanes whose top three bits (of their number in the group) spell j.
__device__ __forceinline__ float sum8(float (&v)[8], int gl, int lanes, unsigned mask) {
  int d = lanes / 2;
#pragma unroll
  for (int n = 4; n > 0; n >>= 1, d >>= 1) {
    const bool up = gl & d;
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float send = up ? v[j] : v[j + n];
      const float keep = up ? v[j + n] : v[j];
      v[j] = keep + __shfl_xor_sync(mask, send, d);
    }
  }
  for (; d > 0; d >>= 1) v[0] += __shfl_xor_sync(mask, v[0], d);
  return v[0];
}

// The same for groups of 1, 2 or 4 lanes, which end with 8 / lanes sums each, in v[0 ...]: those of the values from
// gl * 8 / lanes on (2M weighted lookups of 3 fp32: 65 us, 99 by a sum over the group for each value).
__device__ __forceinline__ void sum8_narrow(float (&v)[8], int gl, int lanes, unsigned mask) {
  int d = lanes / 2;
#pragma unroll
  for (int n = 4; n > 1; n >>= 1, d >>= 1)
    if (d > 0) {
      const bool up = gl & d;
#pragma unroll
      for (int j = 0; j < n; ++j) {
        const float send = up ? v[j] : v[j + n];
        const float keep = up ? v[j + n] : v[j];
        v[j] = keep + __shfl_xor_sync(mask, send, d);
      }
    }
}

template <class T, int VB, int PL, bool GW>
__global__ void __launch_bounds__(GT, grad_blocks(PL, VB, GW))
    k_rows_grad(RowsGradArgs a, const T* __restrict__ table, const T* __restrict__ gout, T* __restrict__ gtable) {
  using U = Unit<T, VB>;
  using W = typename U::W;
  constexpr int E = U::E, UN = PL * VB > (GW ? 16 : 32) ? 4 : 8;
  constexpr int SPAN = BLOCK_USES + 2 * L_MAX + 2;
  __shared__ unsigned s_key[SPAN], s_use[SPAN];
  __shared__ float s_f[SPAN];
  const long long N = *a.n;
  const unsigned R = (unsigned)a.u.R;
  // the block's uses, and as many beside them as a chunk looks at
  const int groups = GT / a.lanes, first = a.L + 1, behind = first + groups * a.L;
  const long long at = (long long)blockIdx.x * groups * a.L - first;
  for (int k = threadIdx.x; k < behind + first; k += GT) {
    const long long i = at + k;
    uint2 p = make_uint2(R, 0);
    float f = 0.f;
    if (i >= 0 && i < N) {
      p = __ldg(a.s + i);
      f = factor_of(a.u, p.y);
    }
    s_key[k] = p.x;
    s_use[k] = p.y;
    s_f[k] = f;
  }
  __syncthreads();
  if (a.used && blockIdx.y == 0)
    for (int k = first + threadIdx.x; k < behind; k += GT)
      if (s_key[k] < R && s_key[k] != s_key[k - 1]) a.used[s_key[k]] = 1;
  const int group = threadIdx.x / a.lanes, gl = threadIdx.x % a.lanes;
  const long long chunk = (long long)blockIdx.x * groups + group;
  if (chunk * a.L >= N) return;
  const ChunkEnds c(chunk, N, a.L, R, [&](long long i) { return s_key[i - at]; });
  // the chunk's uses, without those of a first row that it skips, with those of a last row that it follows
  auto first_at_least = [&](int lo, int hi, unsigned v) {
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_key[mid] < v)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo;
  };
  int j = (int)(c.i0 - at), end = (int)(c.i1 - at);
  if (c.skip) j = first_at_least(j, end, c.first + 1);
  if (c.follow) end = first_at_least(end, end + a.L, c.last + 1);
  const int u0 = blockIdx.y * a.lanes * PL + gl;
  bool col[PL];
#pragma unroll
  for (int k = 0; k < PL; ++k) col[k] = u0 + k * a.lanes < a.units;
  const unsigned mask = a.lanes == 32 ? 0xffffffffu : ((1u << a.lanes) - 1) << ((threadIdx.x & 31) / a.lanes * a.lanes);
  const char* gbase = reinterpret_cast<const char*>(gout) + (long long)u0 * VB;
  const char* tbase = reinterpret_cast<const char*>(table) + (long long)u0 * VB;
  const unsigned gstep = (unsigned)(a.gout_stride * sizeof(T)), tstep = (unsigned)(a.table_stride * sizeof(T));
  constexpr unsigned NOTHING = 0xffffffffu;
  unsigned cur = NOTHING;
  float acc[PL][E], row[GW ? PL : 1][E];
  auto flush = [&](bool split) {
    const bool open = c.open && cur == c.first;
    if (open || split) {
      float* p = a.partial + (2 * chunk + (open ? 0 : 1)) * a.C + (long long)u0 * E;
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (col[k])
#pragma unroll
          for (int e = 0; e < E; ++e) p[k * a.lanes * E + e] = acc[k][e];
    } else {
      W* g = reinterpret_cast<W*>(gtable + (long long)cur * a.C) + u0;
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (col[k]) {
          U x;
          x.set(acc[k]);
          g[k * a.lanes] = x.w;
        }
    }
  };
  // (units past the row's end stay zero)
  U g[UN][PL], t[GW ? UN : 1][GW ? PL : 1];
  float zero[E];
#pragma unroll
  for (int e = 0; e < E; ++e) zero[e] = 0.f;
#pragma unroll
  for (int q = 0; q < UN; ++q)
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      g[q][k].set(zero);
      if constexpr (GW) t[q][k].set(zero);
    }
  // UN uses at once, n of them (all in every step but the last)
  auto step = [&](auto full, int n) {
    constexpr bool ALL = decltype(full)::value;
    unsigned key[UN];
#pragma unroll
    for (int q = 0; q < UN; ++q)
      if (ALL || q < n) {
        key[q] = s_key[j + q];
        const W* src = reinterpret_cast<const W*>(gbase + (unsigned long long)s_use[j + q] * gstep);
#pragma unroll
        for (int k = 0; k < PL; ++k)
          if (col[k]) g[q][k].w = __ldg(src + k * a.lanes);
        if constexpr (GW) {
          if (key[q] != (q == 0 ? cur : key[q > 0 ? q - 1 : 0])) {
            const W* tr = reinterpret_cast<const W*>(tbase + (unsigned long long)key[q] * tstep);
#pragma unroll
            for (int k = 0; k < PL; ++k)
              if (col[k]) t[q][k].w = __ldg(tr + k * a.lanes);
          }
        }
      }
    float dot[UN];
#pragma unroll
    for (int q = 0; q < UN; ++q) {
      dot[q] = 0.f;
      if (ALL || q < n) {
        if (key[q] != cur) {
          if (cur != NOTHING) flush(false);
          cur = key[q];
#pragma unroll
          for (int k = 0; k < PL; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[k][e] = 0.f;
          if constexpr (GW)
#pragma unroll
            for (int k = 0; k < PL; ++k) t[q][k].get(row[k]);
        }
        const float f = s_f[j + q];
#pragma unroll
        for (int k = 0; k < PL; ++k) {
          float x[E];
          g[q][k].get(x);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            acc[k][e] = fmaf(f, x[e], acc[k][e]);
            if constexpr (GW) dot[q] = fmaf(x[e], row[k][e], dot[q]);
          }
        }
      }
    }
    if constexpr (GW) {
      if constexpr (UN == 8) {
        if (a.lanes >= 8) {
          const float sum = sum8(dot, gl, a.lanes, mask);
          const int q = gl / (a.lanes / 8);
          if (gl % (a.lanes / 8) == 0 && (ALL || q < n)) a.gweight[s_use[j + q]] = a.u.scale * sum;
        } else {
          sum8_narrow(dot, gl, a.lanes, mask);
          const int held = 8 / a.lanes, q = gl * held;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < held && (ALL || q + i < n)) a.gweight[s_use[j + q + i]] = a.u.scale * dot[i];
        }
      } else {
#pragma unroll
        for (int q = 0; q < UN; ++q) {
          for (int d = a.lanes / 2; d > 0; d >>= 1) dot[q] += __shfl_xor_sync(mask, dot[q], d);
          if (gl == 0 && (ALL || q < n)) a.gweight[s_use[j + q]] = a.u.scale * dot[q];
        }
      }
    }
  };
  for (; j + UN <= end; j += UN) step(std::true_type(), UN);
  if (j < end) step(std::false_type(), end - j);
  if (cur != NOTHING) flush(c.split);
}

// Split rows: the chunk in which a row begins adds its parts, its own and then those of the chunks behind, a
// lane for each column.  Rows over more than JOIN_MANY chunks are left to the whole block: its warps (and, for
// narrow rows, lanes) take every so many-th part each, joined in a fixed order.
constexpr int JOIN_MANY = 32;
constexpr int JOIN_WARPS = GT / 32;

struct JoinItem {
  long long chunk, last;
  unsigned row;
};

// The first sorted use behind row v, which use `from` still belongs to: the warp's lanes look at 32 places at a
// time, `step` apart, first outwards and then inwards.
__device__ __forceinline__ long long past_row(const uint2* __restrict__ s, long long N, unsigned v, long long from,
                                              long long step) {
  const int lane = threadIdx.x & 31;
  long long lo = from;
  while (true) {
    const long long p = lo + step * (lane + 1) - 1;
    const int k = __popc(__ballot_sync(0xffffffffu, p < N && __ldg(&s[p < N ? p : 0].x) == v));
    lo += step * k;
    if (k == 32)
      step *= 32;
    else if (step == 1)
      return lo;
    else
      step = (step + 31) / 32;
  }
}

// Column p of the parts of chunks from, from + step, ... below to.
__device__ __forceinline__ float add_parts(const float* p, long long C, long long from, long long to, int step) {
  float acc = 0.f;
  long long i = from;
  for (; i + 7ll * step < to; i += 8ll * step) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __ldg(p + 2 * (i + (long long)k * step) * C);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc += x[k];
  }
  for (; i < to; i += step) acc += __ldg(p + 2 * i * C);
  return acc;
}

// Zeros for the rows without a use, a group of lanes for each; the bits of 0 are the same in every type.
template <class W>
__device__ __forceinline__ void zero_rows(const RowsGradArgs& a, void* gtable, long long block, long long blocks) {
  constexpr int UN = 4;
  const int gl = threadIdx.x % a.lanes;
  const long long groups = blocks * GT / a.lanes;
  W* g = static_cast<W*>(gtable);
  W z;
  memset(&z, 0, sizeof z);
  for (long long v = (block * GT + threadIdx.x) / a.lanes; v < a.u.R; v += UN * groups) {
    bool hit[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) hit[i] = v + i * groups < a.u.R && !__ldg(a.used + v + i * groups);
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (hit[i])
        for (long long k = gl; k < a.units; k += a.lanes) g[(v + i * groups) * a.units + k] = z;
  }
}

// A lane tests a chunk for a split row that begins in it; the warp then adds what the lanes found, one row after
// the other.  The blocks behind these write the rows that nothing looks up.
constexpr int JOIN_TEST = 8;        // chunks of a warp

template <class T>
__global__ void __launch_bounds__(GT, 5) k_rows_join(RowsGradArgs a, int lanes, unsigned test_blocks, unsigned parts,
                                                     T* __restrict__ gtable) {
  __shared__ JoinItem s_many[JOIN_TEST * JOIN_WARPS];
  __shared__ int s_n;
  __shared__ float s_sum[JOIN_WARPS][32];
  const long long N = *a.n, C = a.C, L = a.L;
  const unsigned R = (unsigned)a.u.R;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  // test_blocks blocks for each of the column parts, then those for the unused rows
  const unsigned join_blocks = test_blocks * parts, block = blockIdx.x % test_blocks, part = blockIdx.x / test_blocks;
  if (blockIdx.x >= join_blocks) {
    if (a.unit == 16)
      zero_rows<uint4>(a, gtable, blockIdx.x - join_blocks, gridDim.x - join_blocks);
    else if (a.unit == 4)
      zero_rows<unsigned>(a, gtable, blockIdx.x - join_blocks, gridDim.x - join_blocks);
    else
      zero_rows<unsigned short>(a, gtable, blockIdx.x - join_blocks, gridDim.x - join_blocks);
    return;
  }
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  const long long chunk = ((long long)block * JOIN_WARPS + wid) * JOIN_TEST + lane;
  JoinItem it{0, 0, 0};
  bool found = false;
  if (lane < JOIN_TEST && chunk * L < N) {
    const ChunkEnds c(chunk, N, L, R, [&](long long i) { return i >= 0 && i < N ? __ldg(&a.s[i].x) : R; });
    found = c.split && !(c.open && c.last == c.first);
    it = JoinItem{chunk, c.i1 + L, c.last};      // (the last use: not before there)
  }
  const int nq = 32 / lanes, q = lane / lanes, gl = lane % lanes;
  const long long c0 = (long long)part * lanes, cstep = (long long)parts * lanes;
  unsigned todo = __ballot_sync(0xffffffffu, found);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    JoinItem f{__shfl_sync(0xffffffffu, it.chunk, src), __shfl_sync(0xffffffffu, it.last, src),
               __shfl_sync(0xffffffffu, it.row, src)};
    f.last = (past_row(a.s, N, f.row, f.last, L) - 1) / L;
    if (f.last - f.chunk > JOIN_MANY) {
      if (lane == 0) s_many[atomicAdd(&s_n, 1)] = f;
      continue;
    }
    for (long long b = c0; b < C; b += cstep) {
      const long long col = b + gl;
      float sum = 0.f;
      if (col < C) sum = add_parts(a.partial + col, C, f.chunk + 1 + q, f.last + 1, nq);
      for (int d = 16; d >= lanes; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (q == 0 && col < C)
        gtable[(long long)f.row * C + col] = from_f32<T>(a.partial[(2 * f.chunk + 1) * C + col] + sum);
    }
  }
  __syncthreads();
  const int n = s_n;
  for (int m = 0; m < n; ++m) {
    const JoinItem f = s_many[m];
    for (long long b = c0; b < C; b += cstep) {
      const long long col = b + gl;
      float sum = 0.f;
      if (col < C) sum = add_parts(a.partial + col, C, f.chunk + 1 + wid * nq + q, f.last + 1, nq * JOIN_WARPS);
      for (int d = 16; d >= lanes; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      s_sum[wid][lane] = sum;
      __syncthreads();
      if (wid == 0 && q == 0 && col < C) {
        sum = a.partial[(2 * f.chunk + 1) * C + col];
        for (int w = 0; w < JOIN_WARPS; ++w) sum += s_sum[w][lane];
        gtable[(long long)f.row * C + col] = from_f32<T>(sum);
      }
      __syncthreads();
    }
  }
}

size_t grad_space(long long N, long long C) {
  // for the most chunks of any kernel that may run
  long long chunks = 0;
  for (int lanes = 1; lanes <= 32; lanes *= 2)
    if (lanes == 32 || lanes * 16 >= C)
      for (int blocks = 1; blocks <= 3; ++blocks) chunks = std::max(chunks, chunks_of(N, chunk_len(N, lanes, blocks)));
  return align256((size_t)chunks * 2 * (size_t)C * sizeof(float));
}

template <class T>
static int grad_unit(const void* table, long long table_stride, long long C, const void* gout, long long gout_stride,
                     const void* gtable) {
  return unit_bytes<T>({table, gout, gtable}, {C, table ? table_stride : 0, gout_stride});
}
static int grad_unit(int type, const void* table, long long ts, long long C, const void* gout, long long gs,
                     const void* gtable) {
  return with_row_type(type, [&](auto t) { return grad_unit<decltype(t)>(table, ts, C, gout, gs, gtable); });
}

bool grad_takes_weights(const void* table, long long table_stride, int type, long long C, const void* gout,
                        long long gout_stride, const void* gtable) {
  const int vb = grad_unit(type, table, table_stride, C, gout, gout_stride, gtable);
  return grad_shape(C, (int)row_elem(type), vb, true).parts == 1;
}

int rows_grad(const RowUses& u, const SortSpace& s, const void* table, long long table_stride, int type,
              long long C, const void* gout, long long gout_stride, void* gtable, float* gweight, float* partial,
              cudaStream_t st) {
  const void* t = gweight ? table : nullptr;
  const int vb = grad_unit(type, t, table_stride, C, gout, gout_stride, gtable);
  const GradShape g = grad_shape(C, (int)row_elem(type), vb, gweight != nullptr);
  RowsGradArgs a;
  a.u = u;
  a.s = s.sorted;
  a.n = s.n;
  a.used = s.used;
  a.C = C;
  a.table_stride = table_stride;
  a.gout_stride = gout_stride;
  a.L = chunk_len(u.N, g.lanes, grad_blocks(g.per_lane, vb, gweight != nullptr));
  a.chunks = chunks_of(u.N, a.L);
  a.lanes = g.lanes;
  a.units = (int)g.units;
  a.unit = vb;
  a.gweight = gweight;
  a.partial = partial;
  const int per_block = GT / g.lanes;
  const dim3 grid((unsigned)((a.chunks + per_block - 1) / per_block), (unsigned)g.parts);
  return with_unit(type, vb, [&](auto e, auto b) {
    using T = decltype(e);
    constexpr int VB = decltype(b)::value;
    const T* tb = static_cast<const T*>(t);
    const T* go = static_cast<const T*>(gout);
    T* gt = static_cast<T*>(gtable);
    const auto launch = [&](auto per_lane, auto weights) {
      k_rows_grad<T, VB, decltype(per_lane)::value, decltype(weights)::value><<<grid, GT, 0, st>>>(a, tb, go, gt);
    };
    const auto with_weights = [&](auto per_lane) {
      if (gweight)
        launch(per_lane, std::true_type());
      else if constexpr (VB < 16 || decltype(per_lane)::value == 1)
        launch(per_lane, std::false_type());
    };
    if (g.per_lane == 1)
      with_weights(std::integral_constant<int, 1>());
    else if (g.per_lane == 2)
      with_weights(std::integral_constant<int, 2>());
    else if (g.per_lane == 4)
      with_weights(std::integral_constant<int, 4>());
    else if constexpr (VB < 16)
      with_weights(std::integral_constant<int, 3>());
    if (a.chunks > 2 || a.used) {      // (a split row covers a chunk whole)
      int lanes = 1;
      while (lanes < 32 && lanes < C) lanes *= 2;
      const long long cols = (C + lanes - 1) / lanes, per = JOIN_TEST * JOIN_WARPS;
      const unsigned tests = (unsigned)((a.chunks + per - 1) / per), jp = (unsigned)(cols < 32 ? cols : 32);
      const long long zero = a.used ? (u.R * g.lanes + 4 * GT - 1) / (4 * GT) : 0;
      k_rows_join<T><<<tests * jp + (unsigned)(zero < 148 * 8 ? zero : 148 * 8), GT, 0, st>>>(a, lanes, tests, jp, gt);
    }
    return check_launch("row gradient");
  });
}

}  // namespace tts
