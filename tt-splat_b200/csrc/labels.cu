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
// stats[r] = (m, log S); log S = -inf marks a row of masked labels only (a real one is at least 0).
#include <math_constants.h>

#include "rowtype.cuh"

namespace tts {

constexpr int TOP_MAX = 16;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

template <class T>
__global__ void __launch_bounds__(256) k_label_scores(const T* __restrict__ logits, long long P, long long C,
                                                      long long stride, const void* __restrict__ labels, int labels64,
                                                      int top, float* __restrict__ logp, float* __restrict__ entropy,
                                                      float* __restrict__ top_logp, long long* __restrict__ top_ids,
                                                      float2* __restrict__ stats) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long r = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < P; r += warps) {
    const T* x = logits + r * stride;
    float m = -CUDART_INF_F;
    bool bad = false;
    for (long long j = lane; j < C; j += 32) {
      const float v = to_f32(x[j]);
      bad |= !(v < CUDART_INF_F);
      m = fmaxf(m, v);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    bad = __any_sync(0xffffffffu, bad);
    const bool empty = !bad && m == -CUDART_INF_F;
    float S = 0.f, A = 0.f;
    if (!bad && !empty)
      for (long long j = lane; j < C; j += 32) {
        const float d = to_f32(x[j]) - m, e = expf(d);
        S += e;
        if (e > 0.f) A = fmaf(e, d, A);
      }
    S = warp_sum(S);
    A = warp_sum(A);
    const float nan = CUDART_NAN_F;
    const float logS = bad ? nan : (empty ? -CUDART_INF_F : logf(S));
    const float base = bad ? nan : (empty ? 0.f : m);
    if (lane == 0) {
      const long long t = load_index(labels, labels64, r);
      float lp = 0.f;
      if (t >= C)
        lp = nan;
      else if (t >= 0)
        lp = bad ? nan : (empty ? -CUDART_INF_F : (to_f32(x[t]) - base) - logS);
      logp[r] = lp;
      entropy[r] = bad ? nan : (empty ? 0.f : logS - A / S);
      if (stats) stats[r] = make_float2(base, logS);
    }
    // the k-th best is the best of those behind the (k-1)-th in the order (value down, id up)
    float pv = CUDART_INF_F;
    long long pi = -1;
    for (int k = 0; k < top; ++k) {
      float bv = -CUDART_INF_F;
      long long bi = C;
      if (!bad)
        for (long long j = lane; j < C; j += 32) {
          const float v = to_f32(x[j]);
          if ((v < pv || (v == pv && j > pi)) && v > bv) {
            bv = v;
            bi = j;
          }
        }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, d);
        const long long oi = __shfl_xor_sync(0xffffffffu, bi, d);
        if (ov > bv || (ov == bv && oi < bi)) {
          bv = ov;
          bi = oi;
        }
      }
      if (lane == 0) {
        top_ids[r * top + k] = bi < C ? bi : -1;
        top_logp[r * top + k] = bad ? nan : (bi < C ? (bv - base) - logS : -CUDART_INF_F);
      }
      pv = bv;
      pi = bi;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_label_scores_bwd(const T* __restrict__ logits, long long P, long long C,
                                                          long long stride, const void* __restrict__ labels, int labels64,
                                                          int top, const float2* __restrict__ stats,
                                                          const float* __restrict__ entropy,
                                                          const long long* __restrict__ top_ids,
                                                          const float* __restrict__ g_logp,
                                                          const float* __restrict__ g_entropy,
                                                          const float* __restrict__ g_top, T* __restrict__ glogits) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long r = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < P; r += warps) {
    const T* x = logits + r * stride;
    T* gx = glogits + r * C;
    const float2 st = stats[r];
    const float H = entropy[r], gh = g_entropy ? g_entropy[r] : 0.f;
    const long long t = load_index(labels, labels64, r);
    float gl = 0.f;
    if (g_logp && t >= 0) gl = t < C ? g_logp[r] : CUDART_NAN_F;
    float total = gl;
    if (g_top)
      for (int k = 0; k < top; ++k)
        if (top_ids[r * top + k] >= 0) total += g_top[r * top + k];
    const bool zero = st.y == -CUDART_INF_F, plain = total == 0.f && gh == 0.f;
    for (long long j = lane; j < C; j += 32) {
      float g = 0.f;
      if (!plain) {
        const float lp = (to_f32(x[j]) - st.x) - st.y, p = expf(lp);
        g = p == 0.f ? 0.f : p * (-total - gh * (lp + H));
      }
      if (j == t) g += gl;
      if (g_top)
        for (int k = 0; k < top; ++k)
          if (top_ids[r * top + k] == j) g += g_top[r * top + k];
      gx[j] = from_f32<T>(zero ? 0.f : g);
    }
  }
}

static unsigned warp_grid(long long items) {
  long long b = (items + 7) / 8;
  return (unsigned)(b < 148 * 64 ? b : 148 * 64);
}
static int check_labels(long long P, long long C, int type, int top) {
  TTS_REQUIRE(type >= TTS_ROW_F32 && type <= TTS_ROW_F16, "unknown row type");
  TTS_REQUIRE(P >= 0 && P < (1ll << 31), "the number of rows must be below 2^31");
  TTS_REQUIRE(C >= 1 && C < (1ll << 31), "the number of labels must be at least 1 and below 2^31");
  TTS_REQUIRE(top >= 0 && top <= TOP_MAX, "top must be 0 to 16");
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
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    k_label_scores<T><<<warp_grid(P), 256, 0, as_stream(stream)>>>(
        static_cast<const T*>(logits), P, C, row_stride, labels, labels64, top, logp, entropy, top_logp,
        reinterpret_cast<long long*>(top_ids), reinterpret_cast<float2*>(stats));
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
  return with_row_type(type, [&](auto t) {
    using T = decltype(t);
    k_label_scores_bwd<T><<<warp_grid(P), 256, 0, as_stream(stream)>>>(
        static_cast<const T*>(logits), P, C, row_stride, labels, labels64, top, reinterpret_cast<const float2*>(stats),
        entropy, reinterpret_cast<const long long*>(top_ids), g_logp, g_entropy, g_top, static_cast<T*>(glogits));
    return check_launch("label_log_probs_bwd");
  });
}
