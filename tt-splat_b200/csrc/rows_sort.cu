// Stable sort of the uses of a table's rows by row: LSD radix sort of (row, use) pairs.
//
// A use's place in a pass is the count of smaller digits everywhere, of equal digits in the tiles before
// its own, and of equal digits before it in the tile.  The first comes from one counting kernel over the
// indices (all passes at once), the last from ballots inside a warp and the warps' counts in shared memory.
// The middle one is passed from tile to tile in the same launch: a tile publishes its counts, then adds up
// those of the tiles before it, from the nearest back, until it meets one that has its own sum already.
// Tiles are numbered by a ticket, so every tile that is waited for has started; the wait has a limit all
// the same.  Each pass therefore reads and writes the pairs once.
//
// Digits have up to 10 bits and the passes share the bits evenly: 2 passes up to 2^20 rows.
#include "rows.cuh"

namespace tts {

constexpr int ST = 512;                       // threads of a tile
constexpr int SW = ST / 32;
constexpr int SI = 16;                        // entries per thread
constexpr int TILE = ST * SI;
constexpr int MAX_BITS = 10;
constexpr int MAX_DIGITS = 1 << MAX_BITS;
constexpr int MAX_PASSES = 4;
constexpr int BACK = 8;                       // earlier tiles that a wait looks at in one go
constexpr int PER = MAX_DIGITS / ST;          // neighbouring digits of a thread, their states one word pair
static_assert(PER == 2, "a thread's digits are one 8-byte word of states and one 4-byte word of counts");
constexpr int STATUS_SORT_TIMEOUT = 16;
// tile states: what is published, in the top two bits of a word whose rest is the count (N < 2^30)
constexpr unsigned HAVE_COUNT = 1u << 30, HAVE_SUM = 2u << 30, VALUE = (1u << 30) - 1;

struct Digits {
  int bits, passes;
  __host__ __device__ int shift(int p) const { return p * bits; }
};
static Digits digits_for(long long R, int max_bits) {
  int b = 1;
  while ((R >> b) > 0) ++b;                   // keys are 0 .. R
  Digits d;
  d.passes = (b + max_bits - 1) / max_bits;
  d.bits = (b + d.passes - 1) / d.passes;
  return d;
}

__device__ __forceinline__ unsigned key_of(const RowUses& u, long long n) {
  const long long v = row_of(u, n);
  return (unsigned)(v < 0 ? u.R : v);
}

// Lanes of the warp with the same digit as this one (ballots over its bits); lanes that are not `in`
// match nobody.
__device__ __forceinline__ unsigned same_digit(unsigned d, int bits, bool in) {
  unsigned m = __ballot_sync(0xffffffffu, in);
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, (d >> b) & 1u);
    m &= ((d >> b) & 1u) ? set : ~set;
  }
  return m;
}

// Digit counts of every pass.  One block per SM, so that few blocks add their counts to the same words.
constexpr int DT = 1024;
__global__ void __launch_bounds__(DT) k_sort_digits(RowUses u, Digits dg, unsigned* __restrict__ counts) {
  __shared__ unsigned h[MAX_PASSES * MAX_DIGITS];
  constexpr int UN = 4;
  const int D = 1 << dg.bits, all = dg.passes * D;
  for (int i = threadIdx.x; i < all; i += DT) h[i] = 0;
  __syncthreads();
  const long long step = (long long)gridDim.x * DT;
  for (long long n0 = (long long)blockIdx.x * DT + threadIdx.x; n0 < u.N; n0 += UN * step) {
    unsigned k[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) k[i] = n0 + i * step < u.N ? key_of(u, n0 + i * step) : 0u;
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (n0 + i * step >= u.N) break;
      for (int p = 0; p < dg.passes; ++p) atomicAdd(&h[p * D + ((k[i] >> dg.shift(p)) & (D - 1))], 1u);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < all; i += DT)
    if (h[i]) atomicAdd(counts + i, h[i]);
}

__device__ __forceinline__ uint2 load_state(const unsigned* p) {
  uint2 v;
  asm volatile("ld.relaxed.gpu.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_state(unsigned* p, uint2 v) {
  asm volatile("st.relaxed.gpu.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}
// The published words of both digits, which arrive each by itself: ready when both are there.
__device__ __forceinline__ bool ready(uint2 s) { return (s.x >> 30) != 0 && (s.y >> 30) != 0; }

__global__ void __launch_bounds__(ST) k_sort_pass(RowUses u, const uint2* __restrict__ src, Digits dg, int pass,
                                                  const unsigned* __restrict__ counts, unsigned* __restrict__ ticket,
                                                  unsigned* __restrict__ states, uint2* __restrict__ dst) {
  __shared__ __align__(16) unsigned short s_warp[SW][MAX_DIGITS];     // counts of each warp, then of the warps before it
  __shared__ unsigned s_base[MAX_DIGITS];               // where the tile's first entry of a digit goes
  __shared__ unsigned s_scan[SW];
  __shared__ unsigned s_tile;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int D = 1 << dg.bits, shift = dg.shift(pass);
  if (tid == 0) s_tile = atomicAdd(ticket, 1u);
  for (int i = tid; i < SW * MAX_DIGITS / 8; i += ST) reinterpret_cast<uint4*>(s_warp)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const unsigned tile = s_tile;
  const long long base = (long long)tile * TILE + wid * (32 * SI);
  uint2 e[SI];
  unsigned short rank[SI];
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const long long n = base + i * 32 + lane;
    e[i] = make_uint2(0, 0);
    if (n < u.N) e[i] = src ? src[n] : make_uint2(key_of(u, n), (unsigned)n);
  }
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const bool in = base + i * 32 + lane < u.N;
    const unsigned d = (e[i].x >> shift) & (D - 1);
    const unsigned peers = same_digit(d, dg.bits, in);
    const unsigned first = s_warp[wid][d];
    rank[i] = (unsigned short)(first + __popc(peers & ((1u << lane) - 1)));
    __syncwarp();
    if (in && (peers >> lane) == 1u) s_warp[wid][d] = (unsigned short)(rank[i] + 1);
    __syncwarp();
  }
  __syncthreads();
  // the tile's counts (two digits to a word), published before anything is waited for
  const int d0 = tid * PER;
  uint2 count = make_uint2(0, 0);
  if (d0 < D) {
    unsigned run = 0;
#pragma unroll
    for (int w = 0; w < SW; ++w) {
      unsigned* p = reinterpret_cast<unsigned*>(&s_warp[w][d0]);
      const unsigned c = *p;
      *p = run;
      run += c;
    }
    count = make_uint2(run & 0xffffu, run >> 16);
    if (tile > 0) store_state(states + (long long)tile * D + d0, make_uint2(HAVE_COUNT | count.x, HAVE_COUNT | count.y));
  }
  uint2 before = make_uint2(0, 0);
  if (tile == 0) {
    // the first tile starts each digit behind the smaller ones
    uint2 c = make_uint2(0, 0);
    if (d0 < D) c = make_uint2(counts[d0], counts[d0 + 1]);
    unsigned incl = c.x + c.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[wid] = incl;
    __syncthreads();
    before.x = incl - c.x - c.y;
    for (int w = 0; w < wid; ++w) before.x += s_scan[w];
    before.y = before.x + c.x;
  } else if (d0 < D) {
    long long t = (long long)tile - 1;
    int tries = 0;
    bool done = false;
    while (!done && tries < (1 << 20)) {
      // a few tiles at once, the nearest first; stop at one that has not published yet
      uint2 s[BACK];
#pragma unroll
      for (int j = 0; j < BACK; ++j) s[j] = t - j >= 0 ? load_state(states + (t - j) * D + d0) : make_uint2(0, 0);
      bool go = true;
      int seen = 0;
#pragma unroll
      for (int j = 0; j < BACK; ++j) {
        go = go && !done && ready(s[j]);
        if (go) {
          // a sum counts where both words hold one; a tile that is just turning its counts into sums is read
          // again in the next round
          const bool sx = (s[j].x & HAVE_SUM) != 0, sy = (s[j].y & HAVE_SUM) != 0;
          if (sx != sy) {
            go = false;
          } else {
            before.x += s[j].x & VALUE;
            before.y += s[j].y & VALUE;
            ++seen;
            done = sx;
          }
        }
      }
      t -= seen;
      if (seen == 0) ++tries;
    }
    if (!done) {
      atomicOr(&g_status, STATUS_SORT_TIMEOUT);
      before = make_uint2(VALUE, VALUE);
    }
  }
  if (d0 < D) {
    store_state(states + (long long)tile * D + d0,
                make_uint2(HAVE_SUM | ((before.x + count.x) & VALUE), HAVE_SUM | ((before.y + count.y) & VALUE)));
    s_base[d0] = before.x;
    s_base[d0 + 1] = before.y;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SI; ++i)
    if (base + i * 32 + lane < u.N) {
      const unsigned d = (e[i].x >> shift) & (D - 1);
      const long long at = (long long)s_base[d] + s_warp[wid][d] + rank[i];
      if (at < u.N) dst[at] = e[i];           // never past the end, after a wait that ran out either
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

__device__ void sort_small(const RowUses& u, Digits dg, uint2* sorted) {
  extern __shared__ __align__(16) char smem[];
  uint2* s_e = reinterpret_cast<uint2*>(smem);
  unsigned short(*s_warp)[SS_DIGITS] = reinterpret_cast<unsigned short(*)[SS_DIGITS]>(smem + SORT_SMALL * sizeof(uint2));
  unsigned* s_base = reinterpret_cast<unsigned*>(&s_warp[SS_WARPS][0]);
  unsigned* s_scan = s_base + SS_DIGITS;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int N = (int)u.N, D = 1 << dg.bits;
  // the warps share the entries evenly, in order
  const int steps = (N + SS_THREADS - 1) / SS_THREADS;
  const int base = wid * steps * 32 + lane;
  uint2 e[SS_ITEMS];
#pragma unroll
  for (int i = 0; i < SS_ITEMS; ++i) {
    const int n = base + i * 32;
    e[i] = make_uint2(0, 0);
    if (i < steps && n < N) e[i] = make_uint2(key_of(u, n), (unsigned)n);
  }
  for (int p = 0; p < dg.passes; ++p) {
    const int shift = dg.shift(p);
    for (int i = tid; i < SS_WARPS * D; i += SS_THREADS) s_warp[i / D][i % D] = 0;
    __syncthreads();
    unsigned short rank[SS_ITEMS];
#pragma unroll
    for (int i = 0; i < SS_ITEMS; ++i)
      if (i < steps) {
        const bool in = base + i * 32 < N;
        const unsigned d = (e[i].x >> shift) & (D - 1);
        const unsigned peers = same_digit(d, dg.bits, in);
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
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SS_ITEMS; ++i)
      if (i < steps && base + i * 32 < N) {
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
        if (i < steps && base + i * 32 < N) e[i] = s_e[base + i * 32];
  }
}

__global__ void __launch_bounds__(SS_THREADS) k_sort_small(RowUses u, Digits dg, uint2* __restrict__ sorted,
                                                           char* __restrict__ clear, size_t bytes) {
  if (blockIdx.x == 0) {
    sort_small(u, dg, sorted);
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
  t.sorted = reinterpret_cast<uint2*>(p);
  p += align256((size_t)N * sizeof(uint2));
  t.other = nullptr;
  t.zeroed = nullptr;
  t.zeroed_bytes = 0;
  t.used = nullptr;
  if (N > SORT_SMALL) {
    const Digits dg = digits_for(R, MAX_BITS);
    t.other = reinterpret_cast<uint2*>(p);
    p += align256((size_t)N * sizeof(uint2));
    t.zeroed = p;
    p += align256((size_t)(MAX_PASSES + (size_t)dg.passes * (1 << dg.bits)) * sizeof(unsigned));
    p += align256((size_t)dg.passes * tiles_of(N) * (1 << dg.bits) * sizeof(unsigned));
    t.used = reinterpret_cast<uint8_t*>(p);
    p += align256((size_t)R);
    t.zeroed_bytes = (size_t)(p - t.zeroed);
  }
  if (s) *s = t;
  return (size_t)(p - static_cast<char*>(base));
}

int sort_uses(const RowUses& u, const SortSpace& s, void* clear, size_t clear_bytes, cudaStream_t st) {
  if (u.N <= SORT_SMALL) {
    const Digits dg = digits_for(u.R, SS_BITS);
    static std::atomic<unsigned long long> done{0};
    once_per_device(done, [] { cudaFuncSetAttribute(k_sort_small, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SS_SMEM); });
    const size_t per = (size_t)SS_THREADS * 16 * 8;
    size_t blocks = (clear_bytes + per - 1) / per;
    if (blocks > 148 * 2 - 1) blocks = 148 * 2 - 1;
    k_sort_small<<<(unsigned)blocks + 1, SS_THREADS, SS_SMEM, st>>>(u, dg, s.sorted, static_cast<char*>(clear), clear_bytes);
    return check_launch("sort of the uses");
  }
  const Digits dg = digits_for(u.R, MAX_BITS);
  const long long tiles = tiles_of(u.N);
  const int D = 1 << dg.bits;
  if (cudaMemsetAsync(s.zeroed, 0, s.zeroed_bytes, st) != cudaSuccess) return check_launch("memset of the sort's state");
  unsigned* tickets = reinterpret_cast<unsigned*>(s.zeroed);
  unsigned* counts = tickets + MAX_PASSES;
  unsigned* states = reinterpret_cast<unsigned*>(s.zeroed + align256((size_t)(MAX_PASSES + (size_t)dg.passes * D) * sizeof(unsigned)));
  long long blocks = (u.N + DT - 1) / DT;
  if (blocks > 148) blocks = 148;
  k_sort_digits<<<(unsigned)blocks, DT, 0, st>>>(u, dg, counts);
  for (int p = 0; p < dg.passes; ++p) {
    // the last pass writes `sorted`, the ones before alternate so that none reads what it writes
    const bool to_sorted = (dg.passes - 1 - p) % 2 == 0;
    const uint2* src = p == 0 ? nullptr : (to_sorted ? s.other : s.sorted);
    k_sort_pass<<<(unsigned)tiles, ST, 0, st>>>(u, src, dg, p, counts + p * D, tickets + p, states + (size_t)p * tiles * D,
                                                to_sorted ? s.sorted : s.other);
  }
  return check_launch("sort of the uses");
}

}  // namespace tts
