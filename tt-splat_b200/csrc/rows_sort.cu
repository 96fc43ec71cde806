// Stable sort of the uses of a table's rows by row: LSD radix sort of (row, use) pairs.  Unused and
// out-of-range slots are left out on the way.
//
// A use's place in a pass is the count of smaller digits everywhere, of equal digits in the tiles before its
// own, and of equal digits before it in the tile.  A pass is three launches: the tiles' digit counts; their
// running sums over the tiles, digit by digit; and the move, in which a tile ranks its uses (ballots inside a
// warp, the warps' counts in shared memory), orders them in shared memory and writes every digit's run.  No
// block waits for another.  For 2M uses of 1M rows the sort takes 70 us; with one launch per pass, in which a
// tile adds up what the tiles before it publish, it took 85 us: at 1024 digits the polling costs more than the
// counts.  Tiles of 2048 uses: 4096 and 8192 leave SMs idle (move 47 instead of 41 us at 2M uses, 9 instead of
// 7 us at 100k).  The moves are bound by the ballots (13 cycles a bit and warp).
//
// Digits have 6 to 10 bits and the passes share the bits evenly: 2 passes up to 2^20 rows.
#include <type_traits>

#include "rows.cuh"

namespace tts {

constexpr int ST = 256;                       // threads of a tile
constexpr int SW = ST / 32;
constexpr int SI = 8;                         // uses per thread
constexpr int TILE = ST * SI;
constexpr int MIN_BITS = 6, MAX_BITS = 10;
constexpr int MAX_DIGITS = 1 << MAX_BITS;

struct Digits {
  int bits, passes;
  __host__ __device__ int shift(int p) const { return p * bits; }
};
static Digits digits_for(long long R, int max_bits) {
  int b = 1;
  while (((R - 1) >> b) > 0) ++b;             // keys are 0 .. R - 1
  Digits d;
  d.passes = (b + max_bits - 1) / max_bits;
  d.bits = (b + d.passes - 1) / d.passes;
  if (d.bits < MIN_BITS) d.bits = MIN_BITS;
  return d;
}

// The row of use n, R where there is none.
__device__ __forceinline__ unsigned key_of(const RowUses& u, long long n) {
  const long long v = row_of(u, n);
  return (unsigned)(v < 0 ? u.R : v);
}

// Lanes of the warp with the same digit as this one (ballots over its bits); lanes that are not `in`
// match nobody.
template <int BITS>
__device__ __forceinline__ unsigned same_digit(unsigned d, bool in) {
  unsigned m = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, (d >> b) & 1u);
    m &= ((d >> b) & 1u) ? set : ~set;
  }
  return m;
}

// What a pass reads: the indices themselves in the first (every use, R where there is no row), the pairs of
// the pass before in the others (*n of them).
struct PassIn {
  RowUses u;
  const uint2* src;
  const unsigned* n;
  int shift;
  __device__ __forceinline__ long long count() const { return src ? (long long)*n : u.N; }
  __device__ __forceinline__ uint2 get(long long i, long long N) const {
    if (i >= N) return make_uint2((unsigned)u.R, 0);
    return src ? src[i] : make_uint2(key_of(u, i), (unsigned)i);
  }
};

// Exclusive sum over the block's threads of x (all of ST threads take part).
__device__ __forceinline__ unsigned block_before(unsigned x, unsigned* s_scan) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  unsigned incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) s_scan[wid] = incl;
  __syncthreads();
  unsigned run = incl - x;
#pragma unroll
  for (int w = 0; w < SW; ++w)
    if (w < wid) run += s_scan[w];
  return run;
}

// counts[tile][digit].  The first pass also clears the rows' flags and the weights' gradients of uses without
// a row.
__global__ void __launch_bounds__(ST) k_sort_count(PassIn in, int digits, unsigned* __restrict__ counts,
                                                   uint8_t* __restrict__ used, float* __restrict__ gweight) {
  __shared__ unsigned h[MAX_DIGITS];
  for (int i = threadIdx.x; i < digits; i += ST) h[i] = 0;
  __syncthreads();
  const long long base = (long long)blockIdx.x * TILE, N = in.count();
  unsigned k[SI];
#pragma unroll
  for (int i = 0; i < SI; ++i) k[i] = in.get(base + i * ST + threadIdx.x, N).x;
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    if (k[i] < (unsigned)in.u.R)
      atomicAdd(&h[(k[i] >> in.shift) & (digits - 1)], 1u);
    else if (gweight && base + i * ST + threadIdx.x < N)
      gweight[base + i * ST + threadIdx.x] = 0.f;
  }
  if (used) {
    const long long step = (long long)gridDim.x * ST, words = in.u.R / 16;
    const long long t = (long long)blockIdx.x * ST + threadIdx.x;
    for (long long i = t; i < words; i += step) reinterpret_cast<uint4*>(used)[i] = make_uint4(0, 0, 0, 0);
    if (t < in.u.R - words * 16) used[words * 16 + t] = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += ST) counts[(long long)blockIdx.x * digits + i] = h[i];
}

// Running sums of the counts over the tiles (exclusive, in place) and the digits' totals.  A block takes 8
// digits (32 bytes of a tile's counts) and its 128 groups of 8 lanes consecutive parts of the tiles, so that
// a thread has few loads to wait for.
constexpr int SCAN_DIGITS = 8;
constexpr int SCAN_WARPS = 32;
constexpr int SCAN_PARTS = SCAN_WARPS * 32 / SCAN_DIGITS;
__global__ void __launch_bounds__(32 * SCAN_WARPS) k_sort_scan(unsigned* __restrict__ counts, long long tiles, int digits,
                                                               unsigned* __restrict__ totals) {
  __shared__ unsigned s_warp[SCAN_WARPS][SCAN_DIGITS];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int dl = lane % SCAN_DIGITS, d = blockIdx.x * SCAN_DIGITS + dl, part = threadIdx.x / SCAN_DIGITS;
  const long long t0 = tiles * part / SCAN_PARTS, t1 = tiles * (part + 1) / SCAN_PARTS;
  unsigned sum = 0;
#pragma unroll 8
  for (long long t = t0; t < t1; ++t) sum += counts[t * digits + d];
  unsigned incl = sum;
#pragma unroll
  for (int o = SCAN_DIGITS; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane >= 32 - SCAN_DIGITS) s_warp[wid][dl] = incl;
  __syncthreads();
  unsigned run = incl - sum;
#pragma unroll
  for (int w = 0; w < SCAN_WARPS; ++w)
    if (w < wid) run += s_warp[w][dl];
  if (part == SCAN_PARTS - 1) totals[d] = run + sum;
  for (long long t = t0; t < t1; t += 8) {
    unsigned c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = t + i < t1 ? counts[(t + i) * digits + d] : 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (t + i < t1) counts[(t + i) * digits + d] = run;
      run += c[i];
    }
  }
}

template <int BITS>
__global__ void __launch_bounds__(ST, 4) k_sort_move(PassIn in, const unsigned* __restrict__ counts,
                                                  const unsigned* __restrict__ totals, unsigned* __restrict__ n_used,
                                                  uint2* __restrict__ dst) {
  constexpr int D = 1 << BITS, PER = D > ST ? D / ST : 1;
  // the warps' digit counts, then (every place known) the tile's uses in order
  __shared__ __align__(16) union {
    unsigned short warp[SW][D];
    uint2 e[TILE];
  } s;
  __shared__ unsigned s_start[D];      // where a digit begins in the tile
  __shared__ unsigned s_to[D];         // and its uses' places in dst, less that
  __shared__ unsigned s_scan[SW];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const unsigned R = (unsigned)in.u.R;
  for (int i = tid; i < SW * D / 8; i += ST) reinterpret_cast<uint4*>(s.warp)[i] = make_uint4(0, 0, 0, 0);
  const long long N = in.count(), base = (long long)blockIdx.x * TILE + wid * (32 * SI);
  uint2 e[SI];
  unsigned short rank[SI];
#pragma unroll
  for (int i = 0; i < SI; ++i) e[i] = in.get(base + i * 32 + lane, N);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const bool here = e[i].x < R;
    const unsigned d = here ? (e[i].x >> in.shift) & (D - 1) : 0u;
    const unsigned peers = same_digit<BITS>(d, here);
    rank[i] = (unsigned short)(s.warp[wid][d] + __popc(peers & ((1u << lane) - 1)));
    __syncwarp();
    if (here && (peers >> lane) == 1u) s.warp[wid][d] = (unsigned short)(rank[i] + 1);
    __syncwarp();
  }
  __syncthreads();
  // per digit: the warps' counts become those of the warps before; then the digits' starts, in the tile and
  // in the whole
  unsigned here[PER], all[PER], h = 0, a = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int d = tid * PER + q;
    here[q] = all[q] = 0;
    if (d < D) {
#pragma unroll
      for (int w = 0; w < SW; ++w) {
        const unsigned c = s.warp[w][d];
        s.warp[w][d] = (unsigned short)here[q];
        here[q] += c;
      }
      all[q] = totals[d];
    }
    h += here[q];
    a += all[q];
  }
  unsigned start = block_before(h, s_scan), to = block_before(a, s_scan);
  if (n_used && blockIdx.x == 0 && tid == ST - 1) *n_used = to + a;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int d = tid * PER + q;
    if (d < D) {
      s_start[d] = start;
      s_to[d] = to + counts[(long long)blockIdx.x * D + d] - start;
    }
    start += here[q];
    to += all[q];
  }
  __syncthreads();
  unsigned at[SI];
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const unsigned d = (e[i].x >> in.shift) & (D - 1);
    at[i] = e[i].x < R ? s_start[d] + s.warp[wid][d] + rank[i] : 0xffffffffu;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SI; ++i)
    if (at[i] != 0xffffffffu) s.e[at[i]] = e[i];
  // the last digit's end
  if (tid == ST - 1) s_scan[0] = start;
  __syncthreads();
  const int n = (int)s_scan[0];
  for (int i = tid; i < n; i += ST) {
    const uint2 x = s.e[i];
    dst[s_to[(x.x >> in.shift) & (D - 1)] + i] = x;
  }
}

// ---- one block: up to SORT_SMALL uses in shared memory --------------------------------------------
// The other blocks of the launch clear the gradient meanwhile: the sort leaves the memory idle.
constexpr int SS_THREADS = 1024;
constexpr int SS_WARPS = SS_THREADS / 32;
constexpr int SS_ITEMS = (int)SORT_SMALL / SS_THREADS;
constexpr int SS_BITS = 8;
constexpr int SS_DIGITS = 1 << SS_BITS;
constexpr size_t SS_SMEM = SORT_SMALL * sizeof(uint2) + SS_WARPS * SS_DIGITS * sizeof(unsigned short) + 2 * SS_DIGITS * sizeof(unsigned);

__device__ void sort_small(const RowUses& u, Digits dg, uint2* sorted, unsigned* n_used, float* gweight) {
  extern __shared__ __align__(16) char smem[];
  uint2* s_e = reinterpret_cast<uint2*>(smem);
  unsigned short(*s_warp)[SS_DIGITS] = reinterpret_cast<unsigned short(*)[SS_DIGITS]>(smem + SORT_SMALL * sizeof(uint2));
  unsigned* s_base = reinterpret_cast<unsigned*>(&s_warp[SS_WARPS][0]);
  unsigned* s_scan = s_base + SS_DIGITS;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const unsigned R = (unsigned)u.R;
  const int N = (int)u.N, D = 1 << dg.bits;
  // the warps share the entries evenly, in order
  const int steps = (N + SS_THREADS - 1) / SS_THREADS;
  const int base = wid * steps * 32 + lane;
  uint2 e[SS_ITEMS];
#pragma unroll
  for (int i = 0; i < SS_ITEMS; ++i) {
    const int n = base + i * 32;
    e[i] = make_uint2(R, 0);
    if (i < steps && n < N) {
      e[i] = make_uint2(key_of(u, n), (unsigned)n);
      if (gweight && e[i].x == R) gweight[n] = 0.f;
    }
  }
  for (int p = 0; p < dg.passes; ++p) {
    const int shift = dg.shift(p);
    for (int i = tid; i < SS_WARPS * D; i += SS_THREADS) s_warp[i / D][i % D] = 0;
    __syncthreads();
    unsigned short rank[SS_ITEMS];
#pragma unroll
    for (int i = 0; i < SS_ITEMS; ++i)
      if (i < steps) {
        const bool in = e[i].x < R;
        const unsigned d = (e[i].x >> shift) & (D - 1);
        const unsigned peers = same_digit<SS_BITS>(d, in);
        rank[i] = (unsigned short)(s_warp[wid][d] + __popc(peers & ((1u << lane) - 1)));
        __syncwarp();
        if (in && (peers >> lane) == 1u) s_warp[wid][d] = (unsigned short)(rank[i] + 1);
        __syncwarp();
      }
    __syncthreads();
    // digit d's counts, warp by warp: a thread for each digit, then a scan over the digits
    unsigned count = 0;
    if (tid < D)
#pragma unroll 8
      for (int w = 0; w < SS_WARPS; ++w) {
        const unsigned c = s_warp[w][tid];
        s_warp[w][tid] = (unsigned short)count;
        count += c;
      }
    unsigned incl = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[wid] = incl;
    __syncthreads();
    if (tid < D) {
      unsigned run = incl - count;
      for (int w = 0; w < wid; ++w) run += s_scan[w];
      s_base[tid] = run;
      if (tid == D - 1) s_scan[SS_WARPS] = run + count;
    }
    __syncthreads();
    const int n_left = (int)s_scan[SS_WARPS];
    if (tid == 0 && p == 0) *n_used = n_left;
#pragma unroll
    for (int i = 0; i < SS_ITEMS; ++i)
      if (e[i].x < R) {
        const unsigned d = (e[i].x >> shift) & (D - 1);
        const unsigned at = s_base[d] + s_warp[wid][d] + rank[i];
        if (p + 1 < dg.passes)
          s_e[at] = e[i];
        else
          sorted[at] = e[i];
      }
    __syncthreads();
    if (p + 1 < dg.passes)
#pragma unroll
      for (int i = 0; i < SS_ITEMS; ++i)
        e[i] = i < steps && base + i * 32 < n_left ? s_e[base + i * 32] : make_uint2(R, 0);
  }
}

__global__ void __launch_bounds__(SS_THREADS) k_sort_small(RowUses u, Digits dg, uint2* __restrict__ sorted,
                                                           unsigned* __restrict__ n_used, char* __restrict__ clear,
                                                           size_t bytes, float* __restrict__ gweight) {
  if (blockIdx.x == 0) {
    sort_small(u, dg, sorted, n_used, gweight);
    return;
  }
  // whole 16-byte words first, then the bytes around them
  const size_t head = (16 - (reinterpret_cast<uintptr_t>(clear) & 15u)) & 15u;
  const size_t lead = head < bytes ? head : bytes, words = (bytes - lead) / 16, rest = bytes - lead - words * 16;
  uint4* w = reinterpret_cast<uint4*>(clear + lead);
  const size_t step = (size_t)(gridDim.x - 1) * SS_THREADS;
  for (size_t i = (size_t)(blockIdx.x - 1) * SS_THREADS + threadIdx.x; i < words; i += step) w[i] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == 1) {
    if (threadIdx.x < lead) clear[threadIdx.x] = 0;
    if (threadIdx.x < rest) clear[lead + words * 16 + threadIdx.x] = 0;
  }
}

static long long tiles_of(long long N) { return (N + TILE - 1) / TILE; }

size_t sort_space(long long N, long long R, void* base, SortSpace* s) {
  char* p = static_cast<char*>(base);
  SortSpace t;
  t.n = reinterpret_cast<unsigned*>(p);
  p += 256;
  t.sorted = reinterpret_cast<uint2*>(p);
  p += align256((size_t)N * sizeof(uint2));
  t.other = nullptr;
  t.counts = nullptr;
  t.totals = nullptr;
  t.used = nullptr;
  if (N > SORT_SMALL) {
    const Digits dg = digits_for(R, MAX_BITS);
    t.other = reinterpret_cast<uint2*>(p);
    p += align256((size_t)N * sizeof(uint2));
    t.counts = reinterpret_cast<unsigned*>(p);
    p += align256((size_t)tiles_of(N) * (1 << dg.bits) * sizeof(unsigned));
    t.totals = reinterpret_cast<unsigned*>(p);
    p += align256((size_t)MAX_DIGITS * sizeof(unsigned));
    if (N > R / FEW_USES) {
      t.used = reinterpret_cast<uint8_t*>(p);
      p += align256((size_t)R);
    }
  }
  if (s) *s = t;
  return (size_t)(p - static_cast<char*>(base));
}

int sort_uses(const RowUses& u, const SortSpace& s, void* clear, size_t clear_bytes, float* gweight, cudaStream_t st) {
  if (u.N <= SORT_SMALL) {
    const Digits dg = digits_for(u.R, SS_BITS);
    static std::atomic<unsigned long long> done{0};
    once_per_device(done, [] { cudaFuncSetAttribute(k_sort_small, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SS_SMEM); });
    const size_t per = (size_t)SS_THREADS * 16 * 8;
    size_t blocks = (clear_bytes + per - 1) / per;
    if (blocks > 148 * 2 - 1) blocks = 148 * 2 - 1;
    k_sort_small<<<(unsigned)blocks + 1, SS_THREADS, SS_SMEM, st>>>(u, dg, s.sorted, s.n, static_cast<char*>(clear), clear_bytes,
                                                                    gweight);
    return check_launch("sort of the uses");
  }
  if (!s.used && cudaMemsetAsync(clear, 0, clear_bytes, st) != cudaSuccess) return check_launch("memset of the gradient");
  const Digits dg = digits_for(u.R, MAX_BITS);
  const unsigned tiles = (unsigned)tiles_of(u.N);
  const int D = 1 << dg.bits;
  for (int p = 0; p < dg.passes; ++p) {
    // the last pass writes `sorted`, the ones before alternate so that none reads what it writes
    const bool to_sorted = (dg.passes - 1 - p) % 2 == 0;
    const PassIn in{u, p == 0 ? nullptr : (to_sorted ? s.other : s.sorted), s.n, dg.shift(p)};
    uint2* dst = to_sorted ? s.sorted : s.other;
    k_sort_count<<<tiles, ST, 0, st>>>(in, D, s.counts, p == 0 ? s.used : nullptr, p == 0 ? gweight : nullptr);
    k_sort_scan<<<D / SCAN_DIGITS, 32 * SCAN_WARPS, 0, st>>>(s.counts, tiles, D, s.totals);
    const auto move = [&](auto bits) {
      k_sort_move<decltype(bits)::value><<<tiles, ST, 0, st>>>(in, s.counts, s.totals, p == 0 ? s.n : nullptr, dst);
    };
    switch (dg.bits) {
      case 6: move(std::integral_constant<int, 6>()); break;
      case 7: move(std::integral_constant<int, 7>()); break;
      case 8: move(std::integral_constant<int, 8>()); break;
      case 9: move(std::integral_constant<int, 9>()); break;
      default: move(std::integral_constant<int, 10>()); break;
    }
  }
  return check_launch("sort of the uses");
}

}  // namespace tts
