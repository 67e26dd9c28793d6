// LayerNorm over the last dimension, forward and backward (no LIF behind it:
// ln_lif.cu has the fused form for T <= 4).
//
//   y = h * w + b,  h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   g_b = sum_rows g,  g_w = sum_rows g * h
//   g_x = rstd * (a - mean(a) - h * mean(a * h)),  a = g * w
//
// The variance is the mean of (x - mean)^2, a second sweep over the row, so a
// large common offset costs no digits.  All sums are fp32.
#include "common.cuh"

namespace spk {
namespace lnk {

__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
  if (dt == SPK_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == SPK_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_any(void* p, int dt, int64_t i, float v) {
  if (dt == SPK_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == SPK_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

constexpr int kThreads = 128;

// sum over the block; every thread gets it
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

__global__ void __launch_bounds__(kThreads) fwd_kernel(const void* x, int xdt, int64_t ld, const void* w, int wdt,
                                                       const void* b, int bdt, float eps, int64_t rows, int D,
                                                       void* y, int ydt, float* stats) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    float s = 0.0f;
    for (int i = threadIdx.x; i < D; i += kThreads) s += ld_any(x, xdt, r * ld + i);
    const float mean = block_sum(s) / (float)D;
    float q = 0.0f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float c = ld_any(x, xdt, r * ld + i) - mean;
      q += c * c;
    }
    const float rstd = 1.0f / sqrtf(block_sum(q) / (float)D + eps);
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float h = (ld_any(x, xdt, r * ld + i) - mean) * rstd;
      st_any(y, ydt, r * (int64_t)D + i, h * (w ? ld_any(w, wdt, i) : 1.0f) + (b ? ld_any(b, bdt, i) : 0.0f));
    }
    if (stats && threadIdx.x == 0) {
      stats[2 * r] = mean;
      stats[2 * r + 1] = rstd;
    }
  }
}

__global__ void __launch_bounds__(kThreads) bwd_x_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                         const float* stats, const void* w, int wdt, int64_t rows,
                                                         int D, void* gx) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[2 * r], rstd = stats[2 * r + 1];
    float sa = 0.0f, sh = 0.0f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float a = ld_any(g, gdt, r * (int64_t)D + i) * (w ? ld_any(w, wdt, i) : 1.0f);
      sa += a;
      sh += a * ((ld_any(x, xdt, r * ld + i) - mean) * rstd);
    }
    const float ma = block_sum(sa) / (float)D, mh = block_sum(sh) / (float)D;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float a = ld_any(g, gdt, r * (int64_t)D + i) * (w ? ld_any(w, wdt, i) : 1.0f);
      const float h = (ld_any(x, xdt, r * ld + i) - mean) * rstd;
      st_any(gx, xdt, r * (int64_t)D + i, rstd * (a - ma - h * mh));
    }
  }
}

// part[chunk][2][D]: (sum g * h, sum g) over a chunk of the rows; a thread per column
__global__ void __launch_bounds__(kThreads) bwd_w_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                         const float* stats, int64_t rows, int D, float* part) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= D) return;
  float sw = 0.0f, sb = 0.0f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float gv = ld_any(g, gdt, r * (int64_t)D + i);
    sw += gv * ((ld_any(x, xdt, r * ld + i) - stats[2 * r]) * stats[2 * r + 1]);
    sb += gv;
  }
  part[(int64_t)blockIdx.y * 2 * D + i] = sw;
  part[((int64_t)blockIdx.y * 2 + 1) * D + i] = sb;
}

__global__ void __launch_bounds__(kThreads) bwd_join_kernel(const float* part, int chunks, int D, void* gw, int wdt,
                                                            void* gb, int bdt) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= D) return;
  float sw = 0.0f, sb = 0.0f;
  for (int c = 0; c < chunks; ++c) {
    sw += part[(int64_t)c * 2 * D + i];
    sb += part[((int64_t)c * 2 + 1) * D + i];
  }
  if (gw) st_any(gw, wdt, i, sw);
  if (gb) st_any(gb, bdt, i, sb);
}

inline int64_t chunks_of(int64_t rows) { return rows < 256 ? (rows < 1 ? 1 : rows) : 256; }
inline bool float_type(int dt) { return dt == SPK_F32 || dt == SPK_F16 || dt == SPK_BF16; }

}  // namespace lnk
}  // namespace spk

extern "C" {

int spk_layer_norm_fwd(const void* x, int x_dtype, int64_t ld, const void* w, int w_dtype, const void* b, int b_dtype,
                       float eps, int64_t rows, int64_t D, void* y, int y_dtype, float* stats, void* stream) {
  using namespace spk;
  using namespace spk::lnk;
  SPK_REQUIRE(x && y, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(x_dtype) && float_type(y_dtype) && (!w || float_type(w_dtype)) && (!b || float_type(b_dtype)),
              SPK_ERR_INVALID, "layer_norm takes fp32, fp16 and bf16");
  SPK_REQUIRE(rows >= 1 && D >= 1 && D <= (1 << 20) && ld >= D && rows < (1ll << 40), SPK_ERR_SHAPE,
              "unsupported sizes rows=%lld D=%lld row stride %lld", (long long)rows, (long long)D, (long long)ld);
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  const int64_t cap = (int64_t)num_sms() * 16;
  fwd_kernel<<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      x, x_dtype, ld, w, w_dtype, b, b_dtype, eps, rows, (int)D, y, y_dtype, stats);
  return check_launch("layer_norm_fwd");
}

int64_t spk_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D) {
  return spk::lnk::chunks_of(rows) * 2 * D * (int64_t)sizeof(float);
}

int spk_layer_norm_bwd(const void* g, int g_dtype, const void* x, int x_dtype, int64_t ld, const float* stats,
                       const void* w, int w_dtype, int64_t rows, int64_t D, void* gx, void* gw, void* gb, int b_dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace spk;
  using namespace spk::lnk;
  SPK_REQUIRE(g && x && stats, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(x_dtype) && float_type(g_dtype) && (!(w || gw) || float_type(w_dtype)) &&
                  (!gb || float_type(b_dtype)),
              SPK_ERR_INVALID, "layer_norm takes fp32, fp16 and bf16");
  SPK_REQUIRE(rows >= 1 && D >= 1 && D <= (1 << 20) && ld >= D && rows < (1ll << 40), SPK_ERR_SHAPE,
              "unsupported sizes rows=%lld D=%lld row stride %lld", (long long)rows, (long long)D, (long long)ld);
  SPK_REQUIRE(!(gw || gb) || (workspace && workspace_bytes >= spk_layer_norm_bwd_workspace_bytes(rows, D)),
              SPK_ERR_INVALID, "workspace smaller than spk_layer_norm_bwd_workspace_bytes()");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (gx) {
    const int64_t cap = (int64_t)num_sms() * 16;
    bwd_x_kernel<<<(unsigned)(rows < cap ? rows : cap), kThreads, 0, st>>>(g, g_dtype, x, x_dtype, ld, stats, w,
                                                                         w_dtype, rows, (int)D, gx);
  }
  if (gw || gb) {
    const int chunks = (int)chunks_of(rows);
    float* part = reinterpret_cast<float*>(workspace);
    const unsigned cols = (unsigned)((D + kThreads - 1) / kThreads);
    bwd_w_kernel<<<dim3(cols, (unsigned)chunks), kThreads, 0, st>>>(g, g_dtype, x, x_dtype, ld, stats, rows, (int)D,
                                                                   part);
    bwd_join_kernel<<<cols, kThreads, 0, st>>>(part, chunks, (int)D, gw, w_dtype, gb, b_dtype);
  }
  return check_launch("layer_norm_bwd");
}

}  // extern "C"
