// Vectors of fp32, fp16 or bf16 elements in fp32 registers, for the row-wise
// kernels: one access of N elements (N * element size <= 16 bytes, aligned to
// itself), converted on the way.
#pragma once

#include "common.cuh"

namespace spk {

template <int BYTES> struct Word;
template <> struct Word<2> { using T = uint16_t; };
template <> struct Word<4> { using T = uint32_t; };
template <> struct Word<8> { using T = uint2; };
template <> struct Word<16> { using T = uint4; };

template <int DT, int N>
struct Vec {
  using E = typename Elem<DT>::T;
  using W = typename Word<N * (int)sizeof(E)>::T;
  union U {
    W w;
    E e[N];
    __device__ U() {}
  };
  // unpacks in place; bf16 is the upper half of an fp32
  __device__ static void unpack(const W& w, float (&v)[N]) {
    U u;
    u.w = w;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Elem<DT>::load(&u.e[i]);
  }
  __device__ static W pack(const float (&v)[N]) {
    U u;
#pragma unroll
    for (int i = 0; i < N; ++i) u.e[i] = Elem<DT>::make(v[i]);
    return u.w;
  }
  __device__ static W raw(const E* p) { return *reinterpret_cast<const W*>(p); }
  __device__ static void load(const E* p, float (&v)[N]) { unpack(raw(p), v); }
  __device__ static void store(E* p, const float (&v)[N]) { *reinterpret_cast<W*>(p) = pack(v); }
};

// one element of a type known at run time (parameters, a few values a block)
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

// Whether a token lies outside [0, V) and is not `ignore`, by one block: the only
// writer of *bad, so nothing has to clear it first.  For up to kScanTokens tokens
// (a few microseconds beside the other blocks); more are marked by the blocks
// that meet them, after a memset: 64 to 4096 tokens looked up 8 us against 10, 16384 12
// against 14, 131072 43 against 41.  Returns whether there is one.
constexpr int64_t kScanTokens = 16384;
__device__ __forceinline__ bool scan_tokens(const int64_t* __restrict__ tokens, int64_t n, int64_t V, int64_t ignore,
                                            int* bad) {
  int any = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t t = __ldg(tokens + i);
    any |= t != ignore && (t < 0 || t >= V);
  }
  any = __syncthreads_or(any);
  if (threadIdx.x == 0) *bad = any;
  return any;
}

inline bool float_type(int dt) { return dt == SPK_F32 || dt == SPK_F16 || dt == SPK_BF16; }

}  // namespace spk
