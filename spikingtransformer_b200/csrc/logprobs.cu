// Log probabilities of given tokens, entropy and top alternatives of the
// T-averaged logits, and their gradient.
//
//   z = mean over t of logits[t]            (rounded once to fp32)
//   L = log sum_j exp z_j,  p_j = exp(z_j - L)
//   logp = z_y - L,  H = -sum_j p_j log p_j,  top: the K largest z_j, ties to the lower j, as z_j - L
//   dz_j = g_logp (1[j = y] - p_j) + sum_k g_top_k (1[j = idx_k] - p_j) - g_H p_j (log p_j + H)
//   dlogits[t] = dz / T
//
// Everything runs in powers of two against an integer reference
// c = rint(max_j z_j * log2 e):  t_j = z_j log2 e - c is one fused multiply-add
// whose only errors are its own rounding and that of the constant, and a change
// of c scales sums by an exact power of two.  With S = sum 2^t_j and
// A = sum t_j 2^t_j:  logp = ln 2 (t_y - log2 S),  H = ln 2 (log2 S - A / S).
// Where the maximum is beyond 2^20 (a row barred with the type's lowest value),
// c would be coarser than 1, so the maximum itself is taken off first:
// t_j = (z_j - off) log2 e.  t is held at -200 or above, where 2^t is 0 already,
// so that a barred symbol (z = -inf) adds 0 and not 0 * inf; the maximum passes
// a NaN on.
#include "common.cuh"

namespace spk {
namespace lpk {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float exp2_approx(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// What t_j is measured from: t_j = (z_j - off) log2 e - c, one of the two 0.
struct Ref {
  float off, c;
};
constexpr float kFar = 1048576.0f;
__device__ __forceinline__ Ref ref_of(float m) {
  return fabsf(m) <= kFar ? Ref{0.0f, rintf(m * kLog2e)} : Ref{m, 0.0f};
}
__device__ __forceinline__ float log2_from(float z, Ref f) { return fmaf(z - f.off, kLog2e, -f.c); }
__device__ __forceinline__ float rel_log2(float z, Ref f) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC3480000;" : "=f"(r) : "f"(log2_from(z, f)));  // -200
  return r;
}
// order of the alternatives as an unsigned number: larger logit first, -0 and +0
// alike, NaN below -inf; 0 is no alternative at all
__device__ __forceinline__ uint32_t order_bits(float z) {
  const uint32_t u = __float_as_uint(z + 0.0f);
  if (z != z) return 1u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  if (k <= 1u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// The mean over the T steps, rounded once: the sum's rounding errors are
// collected (two-sum) and go into the quotient's remainder, so that near ties
// keep the order that the exact means have.
template <int DT, typename In = typename Elem<DT>::T>
__device__ __forceinline__ float mean_over_t(const In* x, int64_t st, int T, float inv_t) {
  float s = Elem<DT>::load(x);
  if (T == 1) return s;
  float err = 0.0f;
  for (int t = 1; t < T; ++t) {
    const float v = Elem<DT>::load(x + t * st);
    const float n = __fadd_rn(s, v);
    const float b = __fsub_rn(n, s);
    err = __fadd_rn(err, __fadd_rn(__fsub_rn(s, __fsub_rn(n, b)), __fsub_rn(v, b)));
    s = n;
  }
  if (!(fabsf(s) < INFINITY)) {  // an infinity or NaN, or steps whose sum alone is too large
    double d = 0.0;
    for (int t = 0; t < T; ++t) d += (double)Elem<DT>::load(x + t * st);
    return (float)(d / (double)T);
  }
  const float q = __fmul_rn(s, inv_t);
  return fmaf(__fadd_rn(fmaf(-q, (float)T, s), err), inv_t, q);
}

constexpr int kThreads = 128;

template <typename Op>
__device__ __forceinline__ float block_all(float v, Op op) {
  __shared__ float red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = op(v, red[i]);
  return v;
}

// largest key of the block below `limit`
__device__ __forceinline__ unsigned long long block_max64(unsigned long long v) {
  __shared__ unsigned long long red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = red[i] > v ? red[i] : v;
  return v;
}

template <int DT, typename In = typename Elem<DT>::T>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const In* __restrict__ logits, int T, int64_t rows, int V,
                                                       int64_t st, int64_t sr, const int64_t* __restrict__ tokens,
                                                       int64_t ignore, int K, float* logp, float* entropy,
                                                       float* top_logp, int64_t* top_idx, float* stats, int* bad) {
  const float inv_t = 1.0f / (float)T;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t y = tokens[r];
    const bool in = y >= 0 && y < V;
    if (y == ignore || !in) {
      if (threadIdx.x == 0) {
        if (y != ignore) atomicExch(bad, 1);
        logp[r] = entropy[r] = 0.0f;
        reinterpret_cast<float4*>(stats)[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      for (int k = threadIdx.x; k < K; k += kThreads) {
        top_logp[r * K + k] = 0.0f;
        top_idx[r * K + k] = -1;
      }
      continue;
    }
    const In* x = logits + r * sr;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < V; j += kThreads) m = fmaxf(m, mean_over_t<DT>(x + j, st, T, inv_t));
    m = block_all(m, [](float a, float b) { return fmaxf(a, b); });
    const Ref f = ref_of(m);
    float S = 0.0f, A = 0.0f;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float t = rel_log2(mean_over_t<DT>(x + j, st, T, inv_t), f);
      const float e = exp2_approx(t);
      S += e;
      A = fmaf(e, t, A);
    }
    auto add = [](float a, float b) { return a + b; };
    S = block_all(S, add);
    A = block_all(A, add);
    const float l2s = log2f(S);
    const float H = kLn2 * (l2s - A / S);
    if (threadIdx.x == 0) {
      logp[r] = kLn2 * (log2_from(mean_over_t<DT>(x + y, st, T, inv_t), f) - l2s);
      entropy[r] = H;
      reinterpret_cast<float4*>(stats)[r] = make_float4(f.off, f.c, S, H);
    }
    unsigned long long limit = ~0ull;
    for (int k = 0; k < K; ++k) {
      unsigned long long best = 0;
      for (int j = threadIdx.x; j < V; j += kThreads) {
        const unsigned long long key =
            ((unsigned long long)order_bits(mean_over_t<DT>(x + j, st, T, inv_t)) << 32) | (uint32_t)~j;
        if (key < limit && key > best) best = key;
      }
      limit = block_max64(best);
      if (threadIdx.x == 0) {
        top_idx[r * K + k] = (int64_t)(~(uint32_t)limit);
        top_logp[r * K + k] = kLn2 * (log2_from(order_value((uint32_t)(limit >> 32)), f) - l2s);
      }
    }
  }
}

template <int DT, typename In = typename Elem<DT>::T>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const In* __restrict__ logits, int T, int64_t rows, int V,
                                                       int64_t st, int64_t sr, const int64_t* __restrict__ tokens,
                                                       int64_t ignore, int K, const int64_t* __restrict__ top_idx,
                                                       const float* __restrict__ stats, const float* g_logp,
                                                       const float* g_entropy, const float* g_top, In* grad) {
  const float inv_t = 1.0f / (float)T;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t y = tokens[r];
    const bool used = y != ignore && y >= 0 && y < V;
    const In* x = logits + r * sr;
    const float4 sv = reinterpret_cast<const float4*>(stats)[r];
    const Ref f = {sv.x, sv.y};
    const float S = sv.z, H = sv.w;
    const float gl = g_logp ? g_logp[r] : 0.0f, gh = g_entropy ? g_entropy[r] : 0.0f;
    float G = gl;
    for (int k = 0; g_top && k < K; ++k) G += g_top[r * K + k];
    const float inv_s = 1.0f / S;
    const float a = -gh * kLn2 * inv_s, b = (-G - gh * (H - kLn2 * log2f(S))) * inv_s;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      float d = 0.0f;
      if (used) {
        const float t = rel_log2(mean_over_t<DT>(x + j, st, T, inv_t), f);
        d = exp2_approx(t) * fmaf(a, t, b);
        if (j == y) d += gl;
        for (int k = 0; g_top && k < K; ++k)
          if (top_idx[r * K + k] == j) d += g_top[r * K + k];
        d *= inv_t;
      }
      for (int t = 0; t < T; ++t) grad[((int64_t)t * rows + r) * V + j] = Elem<DT>::make(d);
    }
  }
}

inline bool float_type(int dt) { return dt == SPK_F32 || dt == SPK_F16 || dt == SPK_BF16; }

}  // namespace lpk
}  // namespace spk

#define SPK_LP_SIZES()                                                                                              \
  SPK_REQUIRE(float_type(dtype), SPK_ERR_INVALID, "logits must be fp32, fp16 or bf16");                            \
  SPK_REQUIRE(T >= 1 && T <= 64 && rows >= 1 && rows < (1ll << 31) && V >= 1 && V < (1ll << 30), SPK_ERR_SHAPE,     \
              "unsupported sizes T=%lld rows=%lld V=%lld", (long long)T, (long long)rows, (long long)V);            \
  SPK_REQUIRE((T == 1 || step_stride >= 0) && (rows == 1 || row_stride >= 0), SPK_ERR_SHAPE, "negative stride");    \
  SPK_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= V, SPK_ERR_SHAPE, "top_k=%lld: at most %d and V",          \
              (long long)top_k, kMaxTop)

extern "C" {

int64_t spk_token_logprobs_workspace_bytes(int64_t, int64_t, int64_t, int64_t) { return 16; }

int spk_token_logprobs_fwd(const void* logits, int dtype, int64_t T, int64_t rows, int64_t V, int64_t step_stride,
                           int64_t row_stride, const int64_t* tokens, int64_t ignore_index, int64_t top_k, float* logp,
                           float* entropy, float* top_logp, int64_t* top_idx, float* stats, int* bad_token,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace spk;
  using namespace spk::lpk;
  SPK_REQUIRE(logits && tokens && logp && entropy && stats && bad_token, SPK_ERR_INVALID, "null pointer argument");
  SPK_LP_SIZES();
  SPK_REQUIRE(top_k == 0 || (top_logp && top_idx), SPK_ERR_INVALID, "null top_logp or top_idx");
  SPK_REQUIRE(aligned(stats, 16), SPK_ERR_ALIGN, "stats must be 16-byte aligned");
  SPK_REQUIRE(workspace && workspace_bytes >= spk_token_logprobs_workspace_bytes(T, rows, V, top_k), SPK_ERR_INVALID,
              "workspace smaller than spk_token_logprobs_workspace_bytes()");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaMemsetAsync(bad_token, 0, sizeof(int), s);
  const int64_t cap = (int64_t)num_sms() * 16;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
#define LAUNCH(DT)                                                                                                  \
  fwd_kernel<DT><<<grid, kThreads, 0, s>>>(reinterpret_cast<const Elem<DT>::T*>(logits), (int)T, rows, (int)V,      \
                                           step_stride, row_stride, tokens, ignore_index, (int)top_k, logp, entropy, \
                                           top_logp, top_idx, stats, bad_token)
  if (dtype == SPK_F32) LAUNCH(SPK_F32);
  else if (dtype == SPK_F16) LAUNCH(SPK_F16);
  else LAUNCH(SPK_BF16);
#undef LAUNCH
  return check_launch("token_logprobs_fwd");
}

int spk_token_logprobs_bwd(const void* logits, int dtype, int64_t T, int64_t rows, int64_t V, int64_t step_stride,
                           int64_t row_stride, const int64_t* tokens, int64_t ignore_index, int64_t top_k,
                           const int64_t* top_idx, const float* stats, const float* g_logp, const float* g_entropy,
                           const float* g_top, void* grad, void* stream) {
  using namespace spk;
  using namespace spk::lpk;
  SPK_REQUIRE(logits && tokens && stats && grad, SPK_ERR_INVALID, "null pointer argument");
  SPK_LP_SIZES();
  SPK_REQUIRE(!g_top || top_idx, SPK_ERR_INVALID, "null top_idx");
  SPK_REQUIRE(aligned(stats, 16), SPK_ERR_ALIGN, "stats must be 16-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t cap = (int64_t)num_sms() * 16;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
#define LAUNCH(DT)                                                                                               \
  bwd_kernel<DT><<<grid, kThreads, 0, s>>>(reinterpret_cast<const Elem<DT>::T*>(logits), (int)T, rows, (int)V,   \
                                           step_stride, row_stride, tokens, ignore_index, (int)top_k, top_idx,   \
                                           stats, g_logp, g_entropy, g_top, reinterpret_cast<Elem<DT>::T*>(grad))
  if (dtype == SPK_F32) LAUNCH(SPK_F32);
  else if (dtype == SPK_F16) LAUNCH(SPK_F16);
  else LAUNCH(SPK_BF16);
#undef LAUNCH
  return check_launch("token_logprobs_bwd");
}

}  // extern "C"
