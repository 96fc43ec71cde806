// Table rows looked up through slot tables, and the gradient of the lookup.
//
//   out_n      = f_n table[idx_n],  f_n = scale weight_n     (0 where nothing is looked up)
//   gtable_v   = sum over the n with idx_n = v, ascending n, of f_n gout_n
//   gweight_n  = scale <gout_n, table[idx_n]>
//
// The gradient sorts the uses by row, so that a row's uses lie together in ascending order, and adds them
// up in that order: no atomics on floats, the same bits on every run.
#include "rows.cuh"

namespace tts {

// A block copies whole rows (or a part of one long row): the rows' addresses and factors go through shared
// memory once, then the block's output is one run of units, spread evenly over its threads whatever the row
// width, 4 loads of a thread in flight.  Unit e of the run lies in row e / units: the quotient by
// multiplication, (e * magic) >> 32 with magic = ceil(2^32 / units), exact for e and units up to 2^16.  (A
// group of lanes for each row, without shared memory or division, took 61 instead of 24 us for 320000 rows of
// 45 fp32: the indices of its rows are waited for by every lane.)
constexpr int GATHER_THREADS = 256;
constexpr int GATHER_UNITS = 2048;      // units of a block: 8 a thread

template <class T, int VB>
__global__ void __launch_bounds__(GATHER_THREADS, 8) k_gather_rows(RowUses u, const T* __restrict__ table, long long stride,
                                                                   long long units, int rows, unsigned magic,
                                                                   T* __restrict__ out) {
  using U = Unit<T, VB>;
  using W = typename U::W;
  __shared__ const W* s_row[GATHER_THREADS];
  __shared__ float s_f[GATHER_THREADS];
  const long long n0 = (long long)blockIdx.x * rows, part = (long long)blockIdx.y * GATHER_UNITS;
  const int n = (int)(u.N - n0 < rows ? u.N - n0 : rows);
  if (threadIdx.x < n) {
    const long long v = row_of(u, n0 + threadIdx.x);
    const float f = factor_of(u, n0 + threadIdx.x);
    const bool in = v >= 0 && v < u.R;
    s_row[threadIdx.x] = in ? reinterpret_cast<const W*>(table + v * stride) + part : nullptr;
    s_f[threadIdx.x] = in ? f : (v < 0 ? 0.f : __int_as_float(0x7fc00000));
  }
  __syncthreads();
  const unsigned w = rows == 1 ? (unsigned)(units - part < GATHER_UNITS ? units - part : GATHER_UNITS) : (unsigned)units;
  const unsigned total = n * w;
  W* dst = reinterpret_cast<W*>(out) + n0 * units + part;
  constexpr int UN = 4;
  for (unsigned e0 = threadIdx.x; e0 < total; e0 += UN * GATHER_THREADS) {
    U x[UN];
    float f[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const unsigned e = e0 + i * GATHER_THREADS;
      if (e < total) {
        const unsigned r = rows == 1 ? 0u : (magic ? __umulhi(e, magic) : e);      // (magic 0: one unit a row)
        const W* src = s_row[r];
        f[i] = s_f[r];
        memset(&x[i].w, 0, sizeof(W));
        if (src) x[i].w = __ldg(src + (e - r * w));
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const unsigned e = e0 + i * GATHER_THREADS;
      if (e < total) {
        float v[U::E];
        x[i].get(v);
#pragma unroll
        for (int k = 0; k < U::E; ++k) v[k] *= f[i];
        x[i].set(v);
        dst[e] = x[i].w;
      }
    }
  }
}

// Many rows that are no whole number of 16-byte units (320000 rows of 45 fp32: 19.5 us, 24 by the kernel above,
// which takes few rows and long ones): a thread reads the units of 16 consecutive output bytes,
// which may lie in two rows or more, and stores them at once.  A block's rows are a multiple of 16 / SB, so
// its output starts on a 16-byte boundary.
template <class T, int SB>
__global__ void __launch_bounds__(GATHER_THREADS) k_gather_packed(RowUses u, const T* __restrict__ table, long long stride,
                                                                  unsigned units, int rows, unsigned magic,
                                                                  T* __restrict__ out) {
  using U = Unit<T, SB>;
  using W = typename U::W;
  constexpr int NU = 16 / SB, UN = 2;
  __shared__ const W* s_row[GATHER_THREADS];
  __shared__ float s_f[GATHER_THREADS];
  const long long n0 = (long long)blockIdx.x * rows;
  const int n = (int)(u.N - n0 < rows ? u.N - n0 : rows);
  if (threadIdx.x < n) {
    const long long v = row_of(u, n0 + threadIdx.x);
    const float f = factor_of(u, n0 + threadIdx.x);
    const bool in = v >= 0 && v < u.R;
    s_row[threadIdx.x] = in ? reinterpret_cast<const W*>(table + v * stride) : nullptr;
    s_f[threadIdx.x] = in ? f : (v < 0 ? 0.f : __int_as_float(0x7fc00000));
  }
  __syncthreads();
  const unsigned total = n * units, whole = total / NU;
  char* dst = reinterpret_cast<char*>(out) + n0 * units * SB;
  for (unsigned q0 = threadIdx.x; q0 < whole; q0 += UN * GATHER_THREADS) {
    U x[UN][NU];
    float f[UN][NU];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const unsigned q = q0 + i * GATHER_THREADS;
      if (q < whole) {
        unsigned r = magic ? __umulhi(q * NU, magic) : q * NU, c = q * NU - r * units;
        const W* src = s_row[r];
        float g = s_f[r];
#pragma unroll
        for (int k = 0; k < NU; ++k) {
          f[i][k] = g;
          x[i][k].w = src ? __ldg(src + c) : W(0);
          if (++c == units && k + 1 < NU) {
            c = 0;
            src = s_row[++r];
            g = s_f[r];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const unsigned q = q0 + i * GATHER_THREADS;
      if (q < whole) {
        W y[NU];
#pragma unroll
        for (int k = 0; k < NU; ++k) {
          float v[U::E];
          x[i][k].get(v);
#pragma unroll
          for (int e = 0; e < U::E; ++e) v[e] *= f[i][k];
          x[i][k].set(v);
          y[k] = x[i][k].w;
        }
        uint4 z;
        memcpy(&z, y, 16);
        *reinterpret_cast<uint4*>(dst + (long long)q * 16) = z;
      }
    }
  }
  if (threadIdx.x < total - whole * NU) {
    const unsigned e = whole * NU + threadIdx.x, r = magic ? __umulhi(e, magic) : e;
    U x;
    x.w = s_row[r] ? __ldg(s_row[r] + (e - r * units)) : W(0);
    float v[U::E];
    x.get(v);
#pragma unroll
    for (int k = 0; k < U::E; ++k) v[k] *= s_f[r];
    x.set(v);
    reinterpret_cast<W*>(dst)[e] = x.w;
  }
}

// Weights' gradients of rows too wide for the sums' registers, or wanted alone: a warp for each use.
template <class T, int VB>
__global__ void __launch_bounds__(256) k_weight_grad(RowUses u, const T* __restrict__ table, long long stride, long long units,
                                                     const T* __restrict__ gout, long long gstride,
                                                     float* __restrict__ gweight) {
  using U = Unit<T, VB>;
  using W = typename U::W;
  const int lane = threadIdx.x & 31;
  const long long n = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (n >= u.N) return;
  const long long v = row_of(u, n);
  float acc = 0.f;
  if (v >= 0 && v < u.R) {
    const W* a = reinterpret_cast<const W*>(gout + n * gstride);
    const W* b = reinterpret_cast<const W*>(table + v * stride);
#pragma unroll 4
    for (long long i = lane; i < units; i += 32) {
      float x[U::E], y[U::E];
      U(__ldg(a + i)).get(x);
      U(__ldg(b + i)).get(y);
#pragma unroll
      for (int k = 0; k < U::E; ++k) acc = fmaf(x[k], y[k], acc);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
  if (lane == 0) gweight[n] = u.scale * acc;
}

static int check_rows(long long R, long long C, int type, long long N, long long stride) {
  TTS_REQUIRE(type >= TTS_ROW_F32 && type <= TTS_ROW_F16, "unknown row type");
  TTS_REQUIRE(N >= 0 && N < (1ll << 30), "the number of lookups must be below 2^30");
  TTS_REQUIRE(R >= 0 && R < (1ll << 31) - 1, "the number of table rows must be below 2^31 - 1");
  TTS_REQUIRE(C >= 0 && C <= (1ll << 22), "the row width must be at most 2^22");
  TTS_REQUIRE(stride >= 0 && stride < (1ll << 30), "the distance between rows must be below 2^30");
  return TTS_OK;
}
static int check_alignment(int type, const void* idx, int idx64, std::initializer_list<const void*> rows,
                           std::initializer_list<const void*> floats) {
  TTS_REQUIRE(aligned_to(row_elem(type), rows) && aligned_to(4, floats) && aligned_to(idx64 ? 8 : 4, {idx}),
              "rows, indices and weights must be aligned to their elements");
  return TTS_OK;
}

}  // namespace tts

using namespace tts;

extern "C" int tts_gather_rows(const void* table, long long R, long long C, long long table_stride, int type,
                               const void* idx, int idx64, const uint8_t* valid, const float* weight, float scale,
                               long long N, void* out, void* stream) {
  if (int rc = check_rows(R, C, type, N, table_stride)) return rc;
  if (N == 0 || C == 0) return TTS_OK;
  TTS_REQUIRE((table || R == 0) && idx && out, "null gather_rows argument");
  if (int rc = check_alignment(type, idx, idx64, {table, out}, {weight})) return rc;
  TTS_REQUIRE(!rows_overlap(table, R, C, table_stride, row_elem(type), out, N * C * (long long)row_elem(type)),
              "the output must not overlap the table");
  const RowUses u{idx, valid, weight, scale, idx64, N, R};
  const int vb = with_row_type(type, [&](auto t) { return unit_bytes<decltype(t)>({table, out}, {C, table_stride}); });
  const long long units = C * (long long)row_elem(type) / vb;
  long long rows = GATHER_UNITS / units;
  rows = rows < 1 ? 1 : (rows > GATHER_THREADS ? GATHER_THREADS : rows);
  const int step = 16 / vb;
  if (vb < 16 && rows >= step && aligned16(out) && N * units >= 148ll * 4 * GATHER_UNITS) {
    rows -= rows % step;
    const unsigned magic = units == 1 ? 0u : (unsigned)(((1ull << 32) + units - 1) / units);
    const unsigned blocks = (unsigned)((N + rows - 1) / rows);
    return with_unit(type, vb, [&](auto t, auto b) {
      using T = decltype(t);
      constexpr int VB = decltype(b)::value;
      if constexpr (VB < 16)
        k_gather_packed<T, VB><<<blocks, GATHER_THREADS, 0, as_stream(stream)>>>(
            u, static_cast<const T*>(table), table_stride, (unsigned)units, (int)rows, magic, static_cast<T*>(out));
      return check_launch("gather_rows");
    });
  }
  const unsigned magic = units == 1 ? 0u : (unsigned)(((1ull << 32) + units - 1) / units);
  const dim3 grid((unsigned)((N + rows - 1) / rows), (unsigned)((units + GATHER_UNITS - 1) / GATHER_UNITS));
  return with_unit(type, vb, [&](auto t, auto b) {
    using T = decltype(t);
    k_gather_rows<T, decltype(b)::value><<<grid, GATHER_THREADS, 0, as_stream(stream)>>>(
        u, static_cast<const T*>(table), table_stride, units, (int)rows, magic, static_cast<T*>(out));
    return check_launch("gather_rows");
  });
}

extern "C" size_t tts_gather_rows_bwd_workspace_bytes(long long N, long long R, long long C) {
  if (N < 0 || R < 0 || C < 0) return 0;
  return sort_space(N, R, nullptr, nullptr) + grad_space(N, C) + 256;
}

extern "C" int tts_gather_rows_bwd(const void* table, long long R, long long C, long long table_stride, int type,
                                   const void* idx, int idx64, const uint8_t* valid, const float* weight, float scale,
                                   long long N, const void* gout, long long gout_stride, void* gtable, float* gweight,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_rows(R, C, type, N, table_stride)) return rc;
  if (int rc = check_rows(R, C, type, N, gout_stride)) return rc;
  TTS_REQUIRE(N == 0 || (idx && (gout || C == 0)), "null gather_rows_bwd argument");
  TTS_REQUIRE(!gweight || table || R == 0 || C == 0, "the weight gradient needs the table");
  if (int rc = check_alignment(type, idx, idx64, {table, gout, gtable}, {weight, gweight})) return rc;
  if (R == 0 || C == 0) gtable = nullptr;      // nothing to write
  if (gtable && workspace_bytes < tts_gather_rows_bwd_workspace_bytes(N, R, C))
    return fail(TTS_ERR_CAPACITY, "gather_rows_bwd workspace too small");
  TTS_REQUIRE(!gtable || workspace, "null gather_rows_bwd workspace");
  TTS_REQUIRE(!rows_overlap(table, R, C, table_stride, row_elem(type), gtable, R * C * (long long)row_elem(type)) &&
                  !rows_overlap(gout, N, C, gout_stride, row_elem(type), gtable, R * C * (long long)row_elem(type)),
              "the table's gradient must not overlap the table or the incoming gradient");
  cudaStream_t st = as_stream(stream);
  const RowUses u{idx, valid, weight, scale, idx64, N, R};
  const bool fused = gtable && gweight && grad_takes_weights(table, table_stride, type, C, gout, gout_stride, gtable);
  if (gtable && N == 0) {
    if (cudaMemsetAsync(gtable, 0, (size_t)R * C * row_elem(type), st) != cudaSuccess) return check_launch("memset of the gradient");
  } else if (gtable) {
    char* w = reinterpret_cast<char*>(align256(reinterpret_cast<size_t>(workspace)));
    SortSpace s;
    const size_t at = sort_space(N, R, w, &s);
    if (int rc = sort_uses(u, s, gtable, (size_t)R * C * row_elem(type), fused ? gweight : nullptr, st)) return rc;
    if (int rc = rows_grad(u, s, table, table_stride, type, C, gout, gout_stride, gtable,
                           fused ? gweight : nullptr, reinterpret_cast<float*>(w + at), st))
      return rc;
  }
  if (gweight && !fused && N > 0) {
    const int vb = with_row_type(type, [&](auto t) {
      return unit_bytes<decltype(t)>({table, gout}, {C, table_stride, gout_stride});
    });
    const long long units = C * (long long)row_elem(type) / vb;
    return with_unit(type, vb, [&](auto t, auto b) {
      using T = decltype(t);
      k_weight_grad<T, decltype(b)::value><<<(unsigned)((N + 7) / 8), 256, 0, st>>>(u, static_cast<const T*>(table), table_stride, units,
                                                                          static_cast<const T*>(gout), gout_stride, gweight);
      return check_launch("weight gradient");
    });
  }
  return TTS_OK;
}
