// The gradient of the row lookup over its uses in row order:
//
//   gtable_v = sum over the uses n of row v, ascending, of f_n gout_n,   gweight_n = scale <gout_n, table_v>
//
// A group of lanes takes a chunk of L consecutive sorted uses, so that rows with many uses and rows with few
// cost the same.  It keeps the running row in fp32 registers and writes it when the row changes.  A row
// belongs to the chunk in which it begins, which follows it into the next chunk; the next one skips that
// part.  Only a row that goes on behind the next chunk too is split: every chunk leaves its part of it as a
// partial sum, and a second kernel adds the parts in order.  Gradient rows are read once, in units of up to
// 16 bytes, several uses in flight, the next uses' (row, use) pairs one step ahead.
#include "rows.cuh"

namespace tts {

constexpr int GT = 256;

// Uses of a chunk: few where there are few, so that they still spread over the SMs.
static int chunk_len(long long N) { return N <= (1 << 14) ? 8 : (N <= (1 << 17) ? 16 : (N <= (1 << 20) ? 32 : 64)); }
static long long chunks_of(long long N) { return (N + chunk_len(N) - 1) / chunk_len(N); }

struct GradShape {
  long long units;        // of a row
  int lanes, per_lane;    // of a group; lanes * per_lane units a column part
  int parts;              // column parts
};
static GradShape grad_shape(long long C, int elem, int vb) {
  GradShape g;
  g.units = C * elem / vb;
  g.lanes = 1;
  while (g.lanes < 32 && g.lanes < g.units) g.lanes *= 2;
  g.per_lane = g.units <= 32 ? 1 : (g.units <= 64 ? 2 : 4);
  g.parts = (int)((g.units + g.lanes * g.per_lane - 1) / (g.lanes * g.per_lane));
  return g;
}

struct GradArgs {
  RowUses u;
  const uint2* s;
  const uint8_t* used;
  long long C, table_stride, gout_stride, chunks, group_blocks;
  int L, lanes, units;
  float* gweight;
  float* partial;        // [2 * chunks][C]: the chunk's part of a split row begun before it; of one begun in it
};

// What a chunk has to do with the rows at its ends.
struct ChunkEnds {
  long long i0, i1;
  unsigned first, last;
  bool skip;       // its first row belongs to the chunk before
  bool open;       // its first row is split and began before it
  bool split;      // its last row is split and goes on behind it
  bool follow;     // its last row goes on in the next chunk and ends there
  __device__ __forceinline__ ChunkEnds(const GradArgs& a, long long chunk) {
    const long long N = a.u.N, L = a.L;
    const unsigned R = (unsigned)a.u.R;
    i0 = chunk * L;
    i1 = i0 + L < N ? i0 + L : N;
    first = __ldg(&a.s[i0].x);
    last = __ldg(&a.s[i1 - 1].x);
    const unsigned before = i0 > 0 ? __ldg(&a.s[i0 - 1].x) : R, far = i0 > L ? __ldg(&a.s[i0 - L - 1].x) : R;
    const unsigned after = i1 < N ? __ldg(&a.s[i1].x) : R, farther = i1 + L < N ? __ldg(&a.s[i1 + L].x) : R;
    const bool begun = first < R && before == first;             // the first row began before the chunk,
    const bool through = begun && last == first && after == first;  // and goes on behind it
    const bool longer = begun && far == first;                   // or began before the last one already
    open = begun && (through || longer);
    skip = begun && !open;
    const bool on = last < R && after == last;
    split = on && (through || farther == last);
    follow = on && !split;
  }
};

template <class T, int VB, int PL, bool GW>
__global__ void __launch_bounds__(GT) k_rows_grad(GradArgs a, const T* __restrict__ table, const T* __restrict__ gout,
                                                  T* __restrict__ gtable) {
  using U = Unit<T, VB>;
  using W = typename U::W;
  constexpr int E = U::E, UN = PL == 1 ? 8 : 4;
  const int gl = threadIdx.x % a.lanes;
  const int u0 = blockIdx.y * a.lanes * PL + gl;
  if (blockIdx.x >= a.group_blocks) {
    // rows that nothing looks up
    const long long row = ((long long)(blockIdx.x - a.group_blocks) * GT + threadIdx.x) / a.lanes;
    if (row < a.u.R && !__ldg(a.used + row)) {
      W* g = reinterpret_cast<W*>(gtable + row * a.C);
      U z;
#pragma unroll
      for (int e = 0; e < E; ++e) z.t[e] = from_f32<T>(0.f);
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (u0 + k * a.lanes < a.units) g[u0 + k * a.lanes] = z.w;
    }
    return;
  }
  const long long chunk = ((long long)blockIdx.x * GT + threadIdx.x) / a.lanes;
  const long long N = a.u.N;
  const unsigned R = (unsigned)a.u.R;
  const bool live = chunk < a.chunks;
  const ChunkEnds c(a, live ? chunk : 0);
  unsigned cur = c.first;
  bool open = c.open;
  float acc[PL * E], row[GW ? PL * E : 1];
  auto start = [&](unsigned v) {
    cur = v;
#pragma unroll
    for (int k = 0; k < PL * E; ++k) acc[k] = 0.f;
    if constexpr (GW) {
      const W* t = reinterpret_cast<const W*>(table + (long long)v * a.table_stride);
#pragma unroll
      for (int k = 0; k < PL; ++k) {
        U x;
        const bool in = v < R && u0 + k * a.lanes < a.units;
        if (in) x.w = __ldg(t + u0 + k * a.lanes);
#pragma unroll
        for (int e = 0; e < E; ++e) row[k * E + e] = in ? to_f32(x.t[e]) : 0.f;
      }
    }
  };
  auto flush = [&](bool split) {
    if (cur >= R || (c.skip && cur == c.first)) return;
    if (open || split) {
      float* p = a.partial + (2 * chunk + (open ? 0 : 1)) * a.C;
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (u0 + k * a.lanes < a.units)
#pragma unroll
          for (int e = 0; e < E; ++e) p[(u0 + k * a.lanes) * E + e] = acc[k * E + e];
    } else {
      W* g = reinterpret_cast<W*>(gtable + (long long)cur * a.C);
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (u0 + k * a.lanes < a.units) {
          U x;
#pragma unroll
          for (int e = 0; e < E; ++e) x.t[e] = from_f32<T>(acc[k * E + e]);
          g[u0 + k * a.lanes] = x.w;
        }
    }
  };
  // uses of the chunk, and behind it those of a last row that it follows
  const uint2 none = make_uint2(0xffffffffu, 0xffffffffu);
  auto use = [&](long long i) {
    if (!live || i >= N || (i >= c.i1 && !c.follow)) return none;
    const uint2 p = __ldg(a.s + i);
    return i < c.i1 || p.x == c.last ? p : none;
  };
  uint2 next[UN];
#pragma unroll
  for (int j = 0; j < UN; ++j) next[j] = use(c.i0 + j);
  start(cur);
  // every group of a warp takes the same steps (the weights' sums shuffle)
  for (long long i = c.i0;; i += UN) {
    uint2 p[UN];
    float f[UN];
    U g[UN][PL];
#pragma unroll
    for (int j = 0; j < UN; ++j) p[j] = next[j];
    if (!__any_sync(0xffffffffu, p[0].y != none.y)) break;
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      // (a place past the end only after a wait of the sort that ran out)
      const bool in = p[j].x < R && p[j].y < N && !(c.skip && p[j].x == c.first);
      f[j] = in ? factor_of(a.u, p[j].y) : 0.f;
      const W* src = reinterpret_cast<const W*>(gout + (long long)p[j].y * a.gout_stride);
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (in && u0 + k * a.lanes < a.units) g[j][k].w = __ldg(src + u0 + k * a.lanes);
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) next[j] = use(i + UN + j);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const bool here = p[j].y < N, in = here && p[j].x < R && !(c.skip && p[j].x == c.first);
      if (here && p[j].x != cur) {
        flush(false);
        open = false;
        start(p[j].x);
      }
      float dot = 0.f;
      if (in)
#pragma unroll
        for (int k = 0; k < PL; ++k)
          if (u0 + k * a.lanes < a.units)
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float x = to_f32(g[j][k].t[e]);
              acc[k * E + e] = fmaf(f[j], x, acc[k * E + e]);
              if constexpr (GW) dot = fmaf(x, row[k * E + e], dot);
            }
      if constexpr (GW) {
        for (int d = a.lanes / 2; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (here && gl == 0 && (in || p[j].x >= R)) a.gweight[p[j].y] = in ? a.u.scale * dot : 0.f;
      }
    }
  }
  if (live) flush(c.split);
}

// Split rows: the chunk in which a row begins adds its parts, its own and then those of the chunks behind, a
// lane for each column.  Rows over more than JOIN_MANY chunks are left to the whole block: its warps (and, for
// narrow rows, lanes) take every so many-th part each, joined in a fixed order.
constexpr int JOIN_MANY = 64;
constexpr int JOIN_WARPS = GT / 32;

struct JoinItem {
  long long chunk, last;
  unsigned row;
};

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

template <class T>
__global__ void __launch_bounds__(GT) k_rows_join(GradArgs a, int lanes, T* __restrict__ gtable) {
  __shared__ JoinItem s_many[GT];
  __shared__ int s_n;
  __shared__ float s_sum[JOIN_WARPS][32];
  const long long N = a.u.N, C = a.C, L = a.L;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, gl = threadIdx.x % lanes;
  const long long chunk = ((long long)blockIdx.x * GT + threadIdx.x) / lanes;
  const long long c0 = (long long)blockIdx.y * lanes, cstep = (long long)gridDim.y * lanes;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  if (chunk < a.chunks) {
    const ChunkEnds c(a, chunk);
    if (c.split && !(c.open && c.last == c.first)) {
      // the row's last use
      long long lo = c.i1 + L, hi = N;
      for (long long w = L; lo < N; w *= 2) {      // behind a few chunks for most rows
        const long long at = lo + w < N ? lo + w : N;
        if (at == N || a.s[at].x > c.last) {
          hi = at;
          break;
        }
        lo = at + 1;
      }
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (a.s[mid].x <= c.last)
          lo = mid + 1;
        else
          hi = mid;
      }
      const long long last = (lo - 1) / L;
      if (last - chunk > JOIN_MANY) {
        if (gl == 0) s_many[atomicAdd(&s_n, 1)] = JoinItem{chunk, last, c.last};
      } else {
        for (long long b = c0 + gl; b < C; b += cstep)
          gtable[(long long)c.last * C + b] =
              from_f32<T>(a.partial[(2 * chunk + 1) * C + b] + add_parts(a.partial + b, C, chunk + 1, last + 1, 1));
      }
    }
  }
  __syncthreads();
  const int nq = 32 / lanes, q = lane / lanes, n = s_n;
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

size_t grad_space(long long N, long long C) { return align256((size_t)chunks_of(N) * 2 * (size_t)C * sizeof(float)); }

template <class T>
static int grad_unit(const void* table, long long table_stride, long long C, const void* gout, long long gout_stride,
                     const void* gtable) {
  return unit_bytes<T>({table, gout, gtable}, {C, table ? table_stride : 0, gout_stride});
}
static int grad_unit(int type, const void* table, long long ts, long long C, const void* gout, long long gs,
                     const void* gtable) {
  return with_row_type(type, [&](auto t) { return grad_unit<decltype(t)>(table, ts, C, gout, gs, gtable); });
}
static int elem_bytes(int type) { return type == TTS_ROW_F32 ? 4 : 2; }

bool grad_takes_weights(const void* table, long long table_stride, int type, long long C, const void* gout,
                        long long gout_stride, const void* gtable) {
  return grad_shape(C, elem_bytes(type), grad_unit(type, table, table_stride, C, gout, gout_stride, gtable)).parts == 1;
}

int rows_grad(const RowUses& u, const uint2* sorted, const uint8_t* used, const void* table, long long table_stride, int type,
              long long C, const void* gout, long long gout_stride, void* gtable, float* gweight, float* partial,
              cudaStream_t st) {
  const void* t = gweight ? table : nullptr;
  const int vb = grad_unit(type, t, table_stride, C, gout, gout_stride, gtable);
  GradShape g = grad_shape(C, elem_bytes(type), vb);
  // few chunks of wide rows: one unit a lane, more column parts
  if (!gweight && g.per_lane > 1 && chunks_of(u.N) * g.lanes < 148 * 512) {
    g.per_lane = 1;
    g.parts = (int)((g.units + g.lanes - 1) / g.lanes);
    if (g.parts > 65535) g = grad_shape(C, elem_bytes(type), vb);
  }
  GradArgs a;
  a.u = u;
  a.s = sorted;
  a.used = used;
  a.C = C;
  a.table_stride = table_stride;
  a.gout_stride = gout_stride;
  a.chunks = chunks_of(u.N);
  a.L = chunk_len(u.N);
  a.lanes = g.lanes;
  a.units = (int)g.units;
  a.gweight = gweight;
  a.partial = partial;
  const int per_block = GT / g.lanes;
  a.group_blocks = (a.chunks + per_block - 1) / per_block;
  const long long zero_blocks = used ? (u.R + per_block - 1) / per_block : 0;
  const dim3 grid((unsigned)(a.group_blocks + zero_blocks), (unsigned)g.parts);
  return with_unit(type, vb, [&](auto e, auto b) {
    using T = decltype(e);
    constexpr int VB = decltype(b)::value;
    const T* tb = static_cast<const T*>(t);
    const T* go = static_cast<const T*>(gout);
    T* gt = static_cast<T*>(gtable);
    if (gweight) {
      if (g.per_lane == 1)
        k_rows_grad<T, VB, 1, true><<<grid, GT, 0, st>>>(a, tb, go, gt);
      else if (g.per_lane == 2)
        k_rows_grad<T, VB, 2, true><<<grid, GT, 0, st>>>(a, tb, go, gt);
      else
        k_rows_grad<T, VB, 4, true><<<grid, GT, 0, st>>>(a, tb, go, gt);
    } else {
      if (g.per_lane == 1)
        k_rows_grad<T, VB, 1, false><<<grid, GT, 0, st>>>(a, tb, go, gt);
      else if (g.per_lane == 2)
        k_rows_grad<T, VB, 2, false><<<grid, GT, 0, st>>>(a, tb, go, gt);
      else
        k_rows_grad<T, VB, 4, false><<<grid, GT, 0, st>>>(a, tb, go, gt);
    }
    if (a.chunks > 2) {      // a split row covers a chunk whole
      int lanes = 1;
      while (lanes < 32 && lanes < C) lanes *= 2;
      const long long cols = (C + lanes - 1) / lanes;
      const dim3 jg((unsigned)((a.chunks * lanes + GT - 1) / GT), (unsigned)(cols < 32 ? cols : 32));
      k_rows_join<T><<<jg, GT, 0, st>>>(a, lanes, gt);
    }
    return check_launch("row gradient");
  });
}

}  // namespace tts
