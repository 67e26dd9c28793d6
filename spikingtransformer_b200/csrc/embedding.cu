// Scaled token embedding and its gradient.
//
//   out[i] = scale * W[tok[i]]                     (rounded once)
//   g_W[v] = scale * sum over i with tok[i] = v, in ascending i, of g[i]
//
// Tokens outside [0, V) read as a row of zeros, take no gradient and raise the
// caller's flag.
#include "common.cuh"

namespace spk {
namespace embg {

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

__global__ void __launch_bounds__(256) gather_kernel(const int64_t* __restrict__ tokens, const void* w, int wdt,
                                                     int64_t ldw, float scale, int64_t n, int64_t V, int D, void* out,
                                                     int odt, int* bad) {
  const int64_t total = n * D;
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t i = e / D, d = e - i * D;
    const int64_t t = tokens[i];
    const bool ok = t >= 0 && t < V;
    if (!ok && d == 0) atomicExch(bad, 1);
    st_any(out, odt, e, ok ? ld_any(w, wdt, t * ldw + d) * scale : 0.0f);
  }
}

// a block per vocabulary row: reads every token, adds the rows of its own
__global__ void __launch_bounds__(128) scatter_kernel(const int64_t* __restrict__ tokens, const void* g, int gdt,
                                                      float scale, int64_t padding_idx, int64_t n, int64_t V, int D,
                                                      void* gw, int wdt) {
  __shared__ int hit[128];
  for (int64_t v = blockIdx.x; v < V; v += gridDim.x) {
    for (int d0 = 0; d0 < D; d0 += 512) {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int64_t i0 = 0; i0 < n && v != padding_idx; i0 += 128) {
        const int64_t i = i0 + threadIdx.x;
        hit[threadIdx.x] = i < n && tokens[i] == v;
        if (__syncthreads_or(hit[threadIdx.x])) {
          for (int j = 0; j < 128; ++j)
            if (hit[j])
              for (int k = 0; k < 4; ++k) {
                const int d = d0 + threadIdx.x + 128 * k;
                if (d < D) acc[k] += ld_any(g, gdt, (i0 + j) * D + d);
              }
        }
        __syncthreads();
      }
      for (int k = 0; k < 4; ++k) {
        const int d = d0 + threadIdx.x + 128 * k;
        if (d < D) st_any(gw, wdt, v * D + d, acc[k] * scale);
      }
    }
  }
}

inline bool float_type(int dt) { return dt == SPK_F32 || dt == SPK_F16 || dt == SPK_BF16; }

}  // namespace embg
}  // namespace spk

extern "C" {

int spk_embedding_fwd(const int64_t* tokens, const void* weight, int w_dtype, int64_t ldw, float scale, int64_t n,
                      int64_t V, int64_t D, void* out, int out_dtype, int* bad_token, void* stream) {
  using namespace spk;
  using namespace spk::embg;
  SPK_REQUIRE(tokens && weight && out && bad_token, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(w_dtype) && float_type(out_dtype), SPK_ERR_INVALID, "embedding takes fp32, fp16 and bf16");
  SPK_REQUIRE(n >= 1 && V >= 1 && D >= 1 && D <= (1 << 20) && ldw >= D && n < (1ll << 31) && V < (1ll << 31),
              SPK_ERR_SHAPE, "unsupported sizes n=%lld V=%lld D=%lld row stride %lld", (long long)n, (long long)V,
              (long long)D, (long long)ldw);
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaMemsetAsync(bad_token, 0, sizeof(int), st);
  int64_t grid = (n * D + 255) / 256;
  const int64_t cap = (int64_t)num_sms() * 16;
  if (grid > cap) grid = cap;
  gather_kernel<<<(unsigned)grid, 256, 0, st>>>(tokens, weight, w_dtype, ldw, scale, n, V, (int)D, out, out_dtype,
                                               bad_token);
  return check_launch("embedding_fwd");
}

int64_t spk_embedding_bwd_workspace_bytes(int64_t, int64_t, int64_t) { return 16; }

int spk_embedding_bwd(const int64_t* tokens, const void* g, int g_dtype, float scale, int64_t padding_idx, int64_t n,
                      int64_t V, int64_t D, void* gw, int w_dtype, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  using namespace spk;
  using namespace spk::embg;
  SPK_REQUIRE(tokens && g && gw, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(w_dtype) && float_type(g_dtype), SPK_ERR_INVALID, "embedding takes fp32, fp16 and bf16");
  SPK_REQUIRE(n >= 1 && V >= 1 && D >= 1 && D <= (1 << 20) && n < (1ll << 31) && V < (1ll << 31), SPK_ERR_SHAPE,
              "unsupported sizes n=%lld V=%lld D=%lld", (long long)n, (long long)V, (long long)D);
  SPK_REQUIRE(workspace && workspace_bytes >= spk_embedding_bwd_workspace_bytes(n, V, D), SPK_ERR_INVALID,
              "workspace smaller than spk_embedding_bwd_workspace_bytes()");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  const int64_t cap = (int64_t)num_sms() * 16;
  scatter_kernel<<<(unsigned)(V < cap ? V : cap), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      tokens, g, g_dtype, scale, padding_idx, n, V, (int)D, gw, w_dtype);
  return check_launch("embedding_bwd");
}

}  // extern "C"
