// The gradient of the row lookup over its uses in row order:
//
//   gtable_v = sum over the uses n of row v, ascending, of f_n gout_n,   gweight_n = scale <gout_n, table_v>
//
// A group of lanes takes L consecutive sorted uses, so rows with many uses and rows with few cost the same.
// It keeps the running row in fp32 registers and writes it when the row changes.  A row that begins before
// the group's uses or goes on behind them is left as a partial sum, and a second kernel adds a row's partial
// sums in order.  Gradient rows are read once, in units of up to 16 bytes, several uses in flight.
#include "rows.cuh"

namespace tts {

constexpr int GT = 256;
constexpr int CHUNK_MIN = 32;

// Uses per group; the partial sums take 2 rows of C floats for each.
static long long chunk_len(long long N) { return N <= (1 << 19) ? CHUNK_MIN : (N <= (1 << 22) ? 2 * CHUNK_MIN : 4 * CHUNK_MIN); }
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
  float* partial;        // [2 * chunks][C]: the chunk's first row, begun before it; its last, which goes on
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
  const long long i0 = live ? chunk * a.L : N, i1 = i0 + a.L < N ? i0 + a.L : N;
  unsigned cur = live ? a.s[i0].x : R;
  bool open = live && i0 > 0 && a.s[i0 - 1].x == cur;      // the running row began in an earlier chunk
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
  auto flush = [&](bool goes_on) {
    if (cur >= R) return;
    if (open || goes_on) {
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
  if (!GW && cur >= R) return;
  start(cur);
  // every group of a warp takes the same steps (the weights' sums shuffle)
  for (long long s = 0; s < a.L; s += UN) {
    uint2 p[UN];
    float f[UN];
    U g[UN][PL];
#pragma unroll
    for (int j = 0; j < UN; ++j) p[j] = i0 + s + j < i1 ? __ldg(a.s + i0 + s + j) : make_uint2(0xffffffffu, 0);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const bool in = p[j].x < R;
      f[j] = in ? factor_of(a.u, p[j].y) : 0.f;
      const W* src = reinterpret_cast<const W*>(gout + (long long)p[j].y * a.gout_stride);
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (in && u0 + k * a.lanes < a.units) g[j][k].w = __ldg(src + u0 + k * a.lanes);
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const bool here = i0 + s + j < i1, in = p[j].x < R;
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
        if (here && gl == 0) a.gweight[p[j].y] = in ? a.u.scale * dot : 0.f;
      }
    }
  }
  if (live) flush(i1 < N && a.s[i1].x == cur);
}

// Rows over several chunks: the chunk in which a row begins owns it.  A lane tests a chunk; the warp adds the
// partial sums of each row found, lanes over columns (narrow rows: lanes over columns and sums, joined in a
// fixed order), or, for many sums, the warps of the block take a part each.
constexpr int FIX_MANY = 64;
constexpr int FIX_WARPS = GT / 32;
constexpr int FIX_PARTS = 32;       // column parts of a block's grid row

struct FixItem {
  long long chunk, last;
  unsigned row;
};

// Column c of the sums partial(first), first + 1, ... behind the owner's own, by lanes `q` of `nq`.
__device__ __forceinline__ float add_partials(const float* p, long long C, long long from, long long to, int step) {
  float acc = 0.f;
  long long i = from;
  for (; i + 3 * step < to; i += 4 * step) {
    const float a = p[2 * i * C], b = p[2 * (i + step) * C], c = p[2 * (i + 2 * step) * C], d = p[2 * (i + 3 * step) * C];
    acc += a;
    acc += b;
    acc += c;
    acc += d;
  }
  for (; i < to; i += step) acc += p[2 * i * C];
  return acc;
}

template <class T>
__global__ void __launch_bounds__(GT) k_rows_join(GradArgs a, T* __restrict__ gtable) {
  __shared__ FixItem s_many[GT];
  __shared__ int s_n;
  __shared__ float s_sum[FIX_WARPS][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long N = a.u.N, C = a.C;
  const int cols = C < 32 ? (C <= 1 ? 1 : C <= 2 ? 2 : C <= 4 ? 4 : C <= 8 ? 8 : C <= 16 ? 16 : 32) : 32;
  const int nq = 32 / cols, q = lane / cols, cl = lane % cols;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  const long long chunk = (long long)blockIdx.x * GT + threadIdx.x;
  FixItem it{0, 0, 0};
  bool found = false;
  if (chunk < a.chunks && (chunk + 1) * a.L < N) {
    const long long i0 = chunk * a.L, i1 = i0 + a.L;
    const unsigned v = a.s[i1 - 1].x;
    if (v < (unsigned)a.u.R && a.s[i1].x == v && !(i0 > 0 && a.s[i0].x == v && a.s[i0 - 1].x == v)) {
      // the last use of row v
      long long lo = i1, hi = N;
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (a.s[mid].x <= v)
          lo = mid + 1;
        else
          hi = mid;
      }
      it = FixItem{chunk, (lo - 1) / a.L, v};
      found = true;
      if (it.last - it.chunk > FIX_MANY) {
        s_many[atomicAdd(&s_n, 1)] = it;
        found = false;
      }
    }
  }
  unsigned todo = __ballot_sync(0xffffffffu, found);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const long long c0 = __shfl_sync(0xffffffffu, it.chunk, src), c1 = __shfl_sync(0xffffffffu, it.last, src);
    const unsigned v = __shfl_sync(0xffffffffu, it.row, src);
    for (long long b = (long long)blockIdx.y * cols; b < C; b += (long long)gridDim.y * cols) {
      const long long c = b + cl;
      float sum = 0.f;
      if (c < C) sum = add_partials(a.partial + c, C, c0 + 1 + q, c1 + 1, nq);
      for (int d = 16; d >= cols; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (c < C && q == 0) gtable[(long long)v * C + c] = from_f32<T>(a.partial[(2 * c0 + 1) * C + c] + sum);
    }
  }
  __syncthreads();
  for (int m = 0; m < s_n; ++m) {
    const FixItem f = s_many[m];
    for (long long b = (long long)blockIdx.y * cols; b < C; b += (long long)gridDim.y * cols) {
      const long long c = b + cl;
      float sum = 0.f;
      if (c < C) sum = add_partials(a.partial + c, C, f.chunk + 1 + wid * nq + q, f.last + 1, nq * FIX_WARPS);
      for (int d = 16; d >= cols; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      s_sum[wid][lane] = sum;
      __syncthreads();
      if (wid == 0 && q == 0 && c < C) {
        sum = a.partial[(2 * f.chunk + 1) * C + c];
        for (int w = 0; w < FIX_WARPS; ++w) sum += s_sum[w][lane];
        gtable[(long long)f.row * C + c] = from_f32<T>(sum);
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
  const GradShape g = grad_shape(C, elem_bytes(type), vb);
  GradArgs a;
  a.u = u;
  a.s = sorted;
  a.used = used;
  a.C = C;
  a.table_stride = table_stride;
  a.gout_stride = gout_stride;
  a.chunks = chunks_of(u.N);
  a.L = (int)chunk_len(u.N);
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
    if (a.chunks > 1) {
      const long long cols = (C + 31) / 32;
      const dim3 jg((unsigned)((a.chunks + GT - 1) / GT), (unsigned)(cols < FIX_PARTS ? cols : FIX_PARTS));
      k_rows_join<T><<<jg, GT, 0, st>>>(a, gt);
    }
    return check_launch("row gradient");
  });
}

}  // namespace tts
