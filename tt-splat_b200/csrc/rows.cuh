// The row lookup's pieces: the sort of the uses by row (rows_sort.cu), the sums over it (rows_grad.cu) and
// the lookup itself with the entry points (rows.cu).
#pragma once
#include <initializer_list>
#include <type_traits>

#include "rowtype.cuh"

namespace tts {

// The table slots as given, and how many rows there are.
struct RowUses {
  const void* idx;
  const uint8_t* valid;
  const float* weight;
  float scale;
  int idx64;
  long long N, R;
};

// The row that use n looks up: -1 for an unused slot, R for one out of range.
__device__ __forceinline__ long long row_of(const RowUses& u, long long n) {
  const long long v = load_index(u.idx, u.idx64, n);
  const bool ok = !u.valid || __ldg(u.valid + n);      // both on their way before either is looked at
  return !ok || v < 0 ? -1 : (v < u.R ? v : u.R);
}
__device__ __forceinline__ float factor_of(const RowUses& u, long long n) {
  return u.weight ? u.scale * __ldg(u.weight + n) : u.scale;
}

// Rows are read and written in the largest unit that divides their size, their distance and their address.
template <class T>
inline int unit_bytes(std::initializer_list<const void*> ptrs, std::initializer_list<long long> sizes) {
  unsigned long long bits = 0;
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  for (long long s : sizes) bits |= (unsigned long long)s * sizeof(T);
  return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 2);
}

// Calls f with a value of the element type and the unit size as an integral constant.
template <class F>
inline int with_unit(int type, int vb, F f) {
  using B16 = std::integral_constant<int, 16>;
  using B4 = std::integral_constant<int, 4>;
  using B2 = std::integral_constant<int, 2>;
  if (type == TTS_ROW_F32) return vb == 16 ? f(float(), B16()) : f(float(), B4());
  if (type == TTS_ROW_BF16)
    return vb == 16 ? f(__nv_bfloat16(), B16()) : (vb == 4 ? f(__nv_bfloat16(), B4()) : f(__nv_bfloat16(), B2()));
  return vb == 16 ? f(__half(), B16()) : (vb == 4 ? f(__half(), B4()) : f(__half(), B2()));
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// ---- the uses in row order ---------------------------------------------------------------------
// Entries (row, use) sorted by row, equal rows in the order of their uses; unused and out-of-range slots are
// left out.
constexpr long long SORT_SMALL = 8192;      // uses up to which one block sorts them in shared memory
constexpr long long FEW_USES = 4;            // rows for a use from which on the gradient is cleared as a whole

struct SortSpace {
  unsigned* n;         // entries in `sorted`
  uint2* sorted;       // [N] the result
  uint2* other;        // [N] the pass before the last (large sorts, as the rest)
  unsigned* counts;    // digit counts of each tile
  unsigned* totals;    // digit counts
  uint8_t* used;       // [R] flags for the rows that are looked up, cleared; NULL with few uses for the rows
};

size_t sort_space(long long N, long long R, void* base, SortSpace* s);
// Launches the sort, which also clears the weights' gradients (or NULL) of slots that look nothing up.  Up to
// SORT_SMALL uses, and where most rows have none, it clears the `clear_bytes` at `clear` (the whole gradient);
// else the `used` flags, for the caller to find the rows without a use.
int sort_uses(const RowUses& u, const SortSpace& s, void* clear, size_t clear_bytes, float* gweight, cudaStream_t st);

// ---- the sums over the sorted uses ---------------------------------------------------------------
size_t grad_space(long long N, long long C);
int rows_grad(const RowUses& u, const SortSpace& s, const void* table, long long table_stride, int type,
              long long C, const void* gout, long long gout_stride, void* gtable, float* gweight, float* partial,
              cudaStream_t st);
// Whether rows_grad can write the weights' gradient on its way (a row fits a warp's registers).
bool grad_takes_weights(const void* table, long long table_stride, int type, long long C, const void* gout,
                        long long gout_stride, const void* gtable);

}  // namespace tts
