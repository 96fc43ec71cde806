// Table rows looked up through slot tables, and the gradient of the lookup.
//
//   out_n      = f_n table[idx_n],  f_n = scale weight_n     (0 where nothing is looked up)
//   gtable_v   = sum over the n with idx_n = v, ascending n, of f_n gout_n
//   gweight_n  = scale <gout_n, table[idx_n]>
//
// The gradient sorts the uses by row (stable LSD radix sort of (row, use) pairs), so a row's uses lie
// together in ascending order and are added up in that order: no atomics on floats, the same bits on
// every run.
#include "rowtype.cuh"

namespace tts {

constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ITEMS = 16;                            // entries per thread
constexpr int SORT_TILE = SORT_THREADS * SORT_ITEMS;      // entries per block
constexpr int DIGIT_BITS = 8;
constexpr int DIGITS = 1 << DIGIT_BITS;

// The row that use n looks up: -1 for an unused slot, R for one out of range.
__device__ __forceinline__ long long row_of(const void* idx, int idx64, const uint8_t* valid, long long R, long long n) {
  if (valid && !__ldg(valid + n)) return -1;
  const long long v = load_index(idx, idx64, n);
  return v < 0 ? -1 : (v < R ? v : R);
}

template <class T>
__global__ void __launch_bounds__(256) k_gather_rows(const T* __restrict__ table, long long R, int C, long long stride,
                                                     const void* __restrict__ idx, int idx64,
                                                     const uint8_t* __restrict__ valid,
                                                     const float* __restrict__ weight, float scale, long long N,
                                                     T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long n = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; n < N; n += warps) {
    const long long v = row_of(idx, idx64, valid, R, n);
    T* o = out + n * C;
    if (v < 0 || v >= R) {
      const T fill = from_f32<T>(v < 0 ? 0.f : __int_as_float(0x7fc00000));
      for (int c = lane; c < C; c += 32) o[c] = fill;
      continue;
    }
    const float f = weight ? scale * __ldg(weight + n) : scale;
    const T* t = table + v * stride;
    for (int c = lane; c < C; c += 32) o[c] = from_f32<T>(f * to_f32(t[c]));
  }
}

// ---- the uses in row order: stable LSD radix sort, 8 bits a pass -------------------------------
// Unused and out-of-range slots take the key R, behind every row.  The first pass reads the indices
// themselves.
struct SortIn {
  const void* idx;
  const uint8_t* valid;
  const uint2* pairs;      // (key, use) of the pass before, or NULL
  long long R, N;
  int idx64, shift;
};

__device__ __forceinline__ uint2 sort_entry(const SortIn& a, long long n) {
  if (a.pairs) return a.pairs[n];
  const long long v = row_of(a.idx, a.idx64, a.valid, a.R, n);
  return make_uint2((unsigned)(v < 0 ? a.R : v), (unsigned)n);
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(SortIn a, unsigned* __restrict__ counts, int tiles) {
  __shared__ unsigned h[DIGITS];
  for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) h[d] = 0;
  __syncthreads();
  const long long base = (long long)blockIdx.x * SORT_TILE;
  for (int i = threadIdx.x; i < SORT_TILE && base + i < a.N; i += SORT_THREADS)
    atomicAdd(&h[(sort_entry(a, base + i).x >> a.shift) & (DIGITS - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) counts[(long long)d * tiles + blockIdx.x] = h[d];
}

// Exclusive scan of counts[DIGITS][tiles] in place, one block.
__global__ void __launch_bounds__(1024) k_sort_scan(unsigned* __restrict__ counts, long long n) {
  __shared__ unsigned s_w[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  unsigned run = 0;
  for (long long b = 0; b < n; b += 1024) {
    const long long i = b + threadIdx.x;
    const unsigned x = i < n ? counts[i] : 0u;
    unsigned s = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    if (lane == 31) s_w[wid] = s;
    __syncthreads();
    unsigned before = 0, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < wid) before += s_w[w];
      all += s_w[w];
    }
    if (i < n) counts[i] = run + before + s - x;
    run += all;
    __syncthreads();
  }
}

// Each warp takes consecutive entries, 32 at a time; an entry's place among equal digits is the count
// of the lanes before it plus the warp's count so far, so equal digits keep their order.
__global__ void __launch_bounds__(SORT_THREADS) k_sort_scatter(SortIn a, const unsigned* __restrict__ counts, int tiles,
                                                               uint2* __restrict__ dst) {
  __shared__ unsigned h[SORT_WARPS][DIGITS];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < SORT_WARPS * DIGITS; i += SORT_THREADS) (&h[0][0])[i] = 0;
  __syncthreads();
  const long long base = (long long)blockIdx.x * SORT_TILE + wid * (32 * SORT_ITEMS);
  uint2 e[SORT_ITEMS];
  unsigned rank[SORT_ITEMS];
#pragma unroll
  for (int i = 0; i < SORT_ITEMS; ++i) {
    const long long n = base + i * 32 + lane;
    const bool in = n < a.N;
    e[i] = in ? sort_entry(a, n) : make_uint2(0, 0);
    const unsigned d = in ? (e[i].x >> a.shift) & (DIGITS - 1) : DIGITS;
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    rank[i] = 0;
    if (in) rank[i] = h[wid][d] + __popc(peers & ((1u << lane) - 1));
    __syncwarp();
    if (in && lane == 31 - __clz(peers)) h[wid][d] = rank[i] + 1;
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < DIGITS; d += SORT_THREADS) {
    unsigned run = counts[(long long)d * tiles + blockIdx.x];
    for (int w = 0; w < SORT_WARPS; ++w) {
      const unsigned c = h[w][d];
      h[w][d] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SORT_ITEMS; ++i)
    if (base + i * 32 + lane < a.N) dst[h[wid][(e[i].x >> a.shift) & (DIGITS - 1)] + rank[i]] = e[i];
}

// First sorted entry whose key is at least v.
__device__ __forceinline__ long long lower_bound(const uint2* __restrict__ s, long long N, unsigned v) {
  long long lo = 0, hi = N;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (s[mid].x < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

template <class T>
__global__ void __launch_bounds__(256) k_rows_grad(const uint2* __restrict__ s, long long N, long long R, int C,
                                                   const float* __restrict__ weight, float scale,
                                                   const T* __restrict__ gout, long long gstride,
                                                   T* __restrict__ gtable) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long v = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; v < R; v += warps) {
    const long long lo = lower_bound(s, N, (unsigned)v), hi = lower_bound(s, N, (unsigned)v + 1);
    for (int c = lane; c < C; c += 32) {
      float acc = 0.f;
      for (long long i = lo; i < hi; ++i) {
        const unsigned n = s[i].y;
        acc = fmaf(weight ? scale * weight[n] : scale, to_f32(gout[n * gstride + c]), acc);
      }
      gtable[v * C + c] = from_f32<T>(acc);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_weight_grad(const T* __restrict__ table, long long R, int C, long long stride,
                                                     const void* __restrict__ idx, int idx64,
                                                     const uint8_t* __restrict__ valid, float scale, long long N,
                                                     const T* __restrict__ gout, long long gstride,
                                                     float* __restrict__ gweight) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long n = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; n < N; n += warps) {
    const long long v = row_of(idx, idx64, valid, R, n);
    float acc = 0.f;
    if (v >= 0 && v < R)
      for (int c = lane; c < C; c += 32) acc = fmaf(to_f32(gout[n * gstride + c]), to_f32(table[v * stride + c]), acc);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
    if (lane == 0) gweight[n] = scale * acc;
  }
}

static long long sort_tiles(long long N) { return (N + SORT_TILE - 1) / SORT_TILE; }
static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
static unsigned warp_grid(long long items) {
  long long b = (items + 7) / 8;
  return (unsigned)(b < 148 * 64 ? b : 148 * 64);
}
static int check_rows(long long R, long long C, int type, long long N) {
  TTS_REQUIRE(type >= TTS_ROW_F32 && type <= TTS_ROW_F16, "unknown row type");
  TTS_REQUIRE(N >= 0 && N < (1ll << 31), "the number of lookups must be below 2^31");
  TTS_REQUIRE(R >= 0 && R < (1ll << 31) - 1, "the number of table rows must be below 2^31 - 1");
  TTS_REQUIRE(C >= 0 && C < (1ll << 31), "the row width must be below 2^31");
  return TTS_OK;
}

}  // namespace tts

using namespace tts;

extern "C" int tts_gather_rows(const void* table, long long R, long long C, long long table_stride, int type,
                               const void* idx, int idx64, const uint8_t* valid, const float* weight, float scale,
                               long long N, void* out, void* stream) {
  if (int rc = check_rows(R, C, type, N)) return rc;
  if (N == 0 || C == 0) return TTS_OK;
  TTS_REQUIRE((table || R == 0) && idx && out, "null gather_rows argument");
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    k_gather_rows<T><<<warp_grid(N), 256, 0, as_stream(stream)>>>(static_cast<const T*>(table), R, (int)C, table_stride, idx,
                                                                  idx64, valid, weight, scale, N, static_cast<T*>(out));
    return check_launch("gather_rows");
  });
}

extern "C" size_t tts_gather_rows_bwd_workspace_bytes(long long N, long long R, long long C) {
  if (N < 0 || R < 0 || C < 0) return 0;
  return 2 * align256((size_t)N * sizeof(uint2)) + align256((size_t)sort_tiles(N) * DIGITS * sizeof(unsigned)) + 256;
}

extern "C" int tts_gather_rows_bwd(const void* table, long long R, long long C, long long table_stride, int type,
                                   const void* idx, int idx64, const uint8_t* valid, const float* weight, float scale,
                                   long long N, const void* gout, long long gout_stride, void* gtable, float* gweight,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_rows(R, C, type, N)) return rc;
  TTS_REQUIRE(N == 0 || (idx && (gout || C == 0)), "null gather_rows_bwd argument");
  TTS_REQUIRE(!gweight || table || R == 0 || C == 0, "the weight gradient needs the table");
  if (!gtable && !gweight) return TTS_OK;
  if (gtable && workspace_bytes < tts_gather_rows_bwd_workspace_bytes(N, R, C))
    return fail(TTS_ERR_CAPACITY, "gather_rows_bwd workspace too small");
  cudaStream_t st = as_stream(stream);
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    if (gtable && R > 0 && C > 0) {
      char* w = static_cast<char*>(workspace);
      uint2* buf[2] = {reinterpret_cast<uint2*>(w), reinterpret_cast<uint2*>(w + align256((size_t)N * sizeof(uint2)))};
      unsigned* counts = reinterpret_cast<unsigned*>(w + 2 * align256((size_t)N * sizeof(uint2)));
      const int tiles = (int)sort_tiles(N);
      SortIn a{idx, valid, nullptr, R, N, idx64, 0};
      int cur = 0;
      if (N > 0)
        for (a.shift = 0; a.shift == 0 || (R >> a.shift) > 0; a.shift += DIGIT_BITS) {
          k_sort_count<<<tiles, SORT_THREADS, 0, st>>>(a, counts, tiles);
          k_sort_scan<<<1, 1024, 0, st>>>(counts, (long long)tiles * DIGITS);
          k_sort_scatter<<<tiles, SORT_THREADS, 0, st>>>(a, counts, tiles, buf[cur]);
          a.pairs = buf[cur];
          cur ^= 1;
        }
      k_rows_grad<T><<<warp_grid(R), 256, 0, st>>>(a.pairs, N, R, (int)C, weight, scale, static_cast<const T*>(gout),
                                                   gout_stride, static_cast<T*>(gtable));
    }
    if (gweight && N > 0)
      k_weight_grad<T><<<warp_grid(N), 256, 0, st>>>(static_cast<const T*>(table), R, (int)C, table_stride, idx, idx64,
                                                     valid, scale, N, static_cast<const T*>(gout), gout_stride, gweight);
    return check_launch("gather_rows_bwd");
  });
}
