// Scaled token embedding and its gradient.
//
//   out[i] = scale * W[tok[i]]                     (rounded once)
//   g_W[v] = scale * sum over i with tok[i] = v, in ascending i, of g[i]
//
// Tokens outside [0, V) read as a row of zeros, take no gradient and raise the
// caller's flag.
//
// The gradient runs in three launches, without atomics, so equal inputs give
// equal bits:
//   sort    one cluster of blocks sorts the positions by token (stable, radix);
//           the other blocks of the launch meanwhile fill g_W with zeros.
//   sum     a warp adds the rows of g of one chunk of the sorted positions, a
//           tile of columns at a time.  A token whose positions all lie in the
//           chunk is written out; a token that reaches over the chunk's ends
//           leaves its part in a workspace.
//   join    adds the parts of the tokens that reach over chunks, in order.
// A chunk costs the same whatever its tokens are, so a token that fills half the
// batch (padding, a space) is spread over the machine like any other.
#include "vec.cuh"

namespace spk {
namespace embg {

// ---------------------------------------------------------------- forward

// A thread per vector of VEC elements, four in flight.
template <int WDT, int ODT, int VEC>
__global__ void __launch_bounds__(256) gather_kernel(const int64_t* __restrict__ tokens,
                                                     const typename Elem<WDT>::T* __restrict__ w, int64_t ldw,
                                                     float scale, int64_t n, int64_t V, int D,
                                                     typename Elem<ODT>::T* __restrict__ out, int* bad) {
  const unsigned per_row = (unsigned)(D / VEC);
  const int64_t total = n * per_row;
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t e0 = blockIdx.x * (int64_t)256 + threadIdx.x; e0 < total; e0 += 4 * stride) {
    typename Vec<WDT, VEC>::W x[4];
    int64_t tok[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t e = e0 + k * stride;
      tok[k] = -1;
      if (e < total) {
        const int64_t i = total < (1ll << 32) ? (int64_t)((unsigned)e / per_row) : e / per_row;
        const unsigned d = (unsigned)(e - i * per_row);
        tok[k] = __ldg(tokens + i);
        if (tok[k] < 0 || tok[k] >= V) {
          tok[k] = -1;
          if (d == 0) atomicExch(bad, 1);
        } else {
          x[k] = Vec<WDT, VEC>::raw(w + tok[k] * ldw + (int64_t)d * VEC);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t e = e0 + k * stride;
      if (e >= total) break;
      float v[VEC];
      if (tok[k] >= 0) Vec<WDT, VEC>::unpack(x[k], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = tok[k] >= 0 ? v[j] * scale : 0.0f;
      Vec<ODT, VEC>::store(out + e * VEC, v);
    }
  }
}

// ---------------------------------------------------------------- backward: sort

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigit = 10;

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Cluster 0 sorts, the others clear gw.  A pass of the radix sort over a digit
// of `bits` bits: every warp owns a run of consecutive positions and counts its
// digits (lanes of equal digit found by match); the counts are summed over the
// warps of a block, over the blocks of the cluster and over the digits, which
// gives every (warp, digit) its place; the warp then writes its items there in
// order.  Positions without a gradient get the key V and end up last.
__global__ void __launch_bounds__(kSortThreads) sort_clear_kernel(const int64_t* tokens, int64_t n, int64_t V,
                                                                  int64_t padding_idx, int bits, int passes,
                                                                  uint32_t* key0, uint32_t* pos0, uint32_t* key1,
                                                                  uint32_t* pos1, void* gw, int64_t gw_bytes) {
  extern __shared__ uint32_t sm[];
  const uint32_t ncta = cluster_size(), rank = cluster_ctarank(), cl = cluster_id_x();
  if (cl > 0) {
    const int64_t stride = (int64_t)(cluster_count_x() - 1) * ncta * kSortThreads;
    const int64_t me = ((int64_t)(cl - 1) * ncta + rank) * kSortThreads + threadIdx.x;
    if ((reinterpret_cast<uintptr_t>(gw) & 15) == 0) {
      const int64_t n16 = gw_bytes / 16;
      for (int64_t i = me; i < n16; i += stride) reinterpret_cast<uint4*>(gw)[i] = make_uint4(0, 0, 0, 0);
      for (int64_t i = n16 * 8 + me; i < gw_bytes / 2; i += stride) reinterpret_cast<uint16_t*>(gw)[i] = 0;
    } else {
      for (int64_t i = me; i < gw_bytes / 2; i += stride) reinterpret_cast<uint16_t*>(gw)[i] = 0;
    }
    return;
  }
  const int bins = 1 << bits;
  uint32_t* count = sm;                         // [warps][bins]
  uint32_t* total = sm + kSortWarps * bins;     // [bins], read by the cluster's other blocks
  uint32_t* base = total + bins;                // [bins]
  __shared__ uint32_t wsum[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t per_warp = ((n + (int64_t)ncta * kSortWarps - 1) / ((int64_t)ncta * kSortWarps) + 31) / 32 * 32;
  const int64_t lo = ((int64_t)rank * kSortWarps + warp) * per_warp;
  const int64_t hi = lo + per_warp < n ? lo + per_warp : n;
  uint32_t* mine = count + warp * bins;
  for (int p = 0; p < passes; ++p) {
    const uint32_t *kin = (p & 1) ? key0 : key1, *pin = (p & 1) ? pos0 : pos1;
    uint32_t *kout = (p & 1) ? key1 : key0, *pout = (p & 1) ? pos1 : pos0;
    const int shift = p * bits;
    auto key_at = [&](int64_t i) -> uint32_t {
      if (p > 0) return __ldcg(kin + i);
      const int64_t t = __ldg(tokens + i);
      return t >= 0 && t < V && t != padding_idx ? (uint32_t)t : (uint32_t)V;
    };
    for (int i = lane; i < bins; i += 32) mine[i] = 0;
    __syncwarp();
    for (int64_t i0 = lo; i0 < hi; i0 += 32) {
      const int64_t i = i0 + lane;
      const uint32_t d = i < hi ? (key_at(i) >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (i < hi && (same >> lane) == 1u) mine[d] += __popc(same);  // the highest lane of its digit
      __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
      uint32_t s = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w * bins + d];
        count[w * bins + d] = s;
        s += c;
      }
      total[d] = s;
    }
    cluster_sync_all();
    // bins <= threads: one digit a thread; an exclusive sum over the digits of the cluster's counts
    const int d = threadIdx.x;
    uint32_t all = 0, before = 0;
    if (d < bins) {
      for (uint32_t r = 0; r < ncta; ++r) {
        const uint32_t c = ld_cluster_u32(mapa_shared(smem_u32(total + d), r));
        if (r < rank) before += c;
        all += c;
      }
    }
    uint32_t inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    uint32_t off = 0;
    for (int w = 0; w < warp; ++w) off += wsum[w];
    if (d < bins) base[d] = off + inc - all + before;
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 32) {
      const int64_t i = i0 + lane;
      const bool in = i < hi;
      const uint32_t k = in ? key_at(i) : 0u;
      const uint32_t dd = in ? (k >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, dd);
      uint32_t at = 0;
      if (in) at = base[dd] + mine[dd] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (in) {
        kout[at] = k;
        pout[at] = p > 0 ? __ldcg(pin + i) : (uint32_t)i;
        if ((same >> lane) == 1u) mine[dd] += __popc(same);
      }
      __syncwarp();
    }
    cluster_sync_all();  // the items are written and nobody reads `total` any more
  }
}

// ---------------------------------------------------------------- backward: sum and join

// rows of g that a warp has in flight
constexpr int kDeep = 8;

// A warp per (chunk of sorted positions, tile of 32 * VEC columns).
template <int GDT, int WDT, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos,
                                                  const typename Elem<GDT>::T* __restrict__ g, float scale, int64_t n,
                                                  uint32_t V, int D, int chunk, int tiles, int64_t chunks,
                                                  typename Elem<WDT>::T* __restrict__ gw, float* __restrict__ part) {
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
  if (item >= chunks * tiles) return;
  const int64_t c = item / tiles;
  const int col = (int)(item - c * tiles) * 32 * VEC + lane * VEC;
  const bool on = col < D;
  const int64_t lo = c * chunk, hi = lo + chunk < n ? lo + chunk : n;
  const uint32_t before = lo > 0 ? key[lo - 1] : 0xffffffffu;
  const uint32_t after = hi < n ? key[hi] : 0xffffffffu;
  uint32_t cur = key[lo];
  bool first = true;  // the chunk's first token is being added
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  auto flush = [&](bool last) {
    if (cur >= V) return;
    const bool head = first && cur == before;
    const bool tail = last && cur == after;
    if (!on) return;
    if (head || tail) {
      // [chunk][0]: the part of a token that comes from the chunk before (and may go on),
      // [chunk][1]: of one that begins here and goes on
      float* q = part + (c * 2 + (head ? 0 : 1)) * D + col;
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[j] = acc[j];
    } else {
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = acc[j] * scale;
      Vec<WDT, VEC>::store(gw + (int64_t)cur * D + col, v);
    }
  };
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int m = hi - i0 < 32 ? (int)(hi - i0) : 32;
    const uint32_t k = lane < m ? key[i0 + lane] : 0xffffffffu;
    const uint32_t q = lane < m ? pos[i0 + lane] : 0u;
    for (int j0 = 0; j0 < m; j0 += kDeep) {
      typename Vec<GDT, VEC>::W x[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const uint32_t kj = __shfl_sync(0xffffffffu, k, j0 + j), qj = __shfl_sync(0xffffffffu, q, j0 + j);
        if (on && kj < V) x[j] = Vec<GDT, VEC>::raw(g + (int64_t)qj * D + col);
      }
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        if (j0 + j >= m) break;
        const uint32_t kj = __shfl_sync(0xffffffffu, k, j0 + j);
        if (kj != cur) {
          flush(false);
          cur = kj;
          first = false;
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        }
        if (on && kj < V) {
          float v[VEC];
          Vec<GDT, VEC>::unpack(x[j], v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += v[i];
        }
      }
    }
  }
  flush(true);
}

// A block per (chunk, 32 columns): where the chunk's last token begins in it and
// goes on, adds the token's parts.  The parts are cut into one run a warp; the
// warps' sums are added in order.
template <int WDT>
__global__ void __launch_bounds__(256) join_kernel(const uint32_t* __restrict__ key, float scale, int64_t n, uint32_t V,
                                                   int D, int chunk, int64_t chunks,
                                                   typename Elem<WDT>::T* __restrict__ gw,
                                                   const float* __restrict__ part) {
  __shared__ float red[8][32];
  const int64_t c = blockIdx.x;
  const int64_t lo = c * chunk, hi = lo + chunk;
  if (hi >= n) return;
  const uint32_t k = key[hi - 1];
  if (k >= V || key[hi] != k) return;                  // nothing goes on
  if (lo > 0 && key[lo] == k && key[lo - 1] == k) return;  // it began before
  int64_t a = c + 1, b = chunks;                        // chunks (c, a) begin with k
  while (a < b) {
    const int64_t mid = (a + b) / 2;
    if (key[mid * chunk] == k) a = mid + 1;
    else b = mid;
  }
  const int64_t m = a - c;  // parts: [c][1], [c + 1][0], ..., [a - 1][0]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.y * 32 + lane;
  float s = 0.0f;
  if (col < D) {
    const int64_t p0 = m * warp / 8, p1 = m * (warp + 1) / 8;
#pragma unroll 8
    for (int64_t p = p0; p < p1; ++p) s += part[((c + p) * 2 + (p == 0 ? 1 : 0)) * D + col];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < D) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[w][lane];
    gw[(int64_t)k * D + col] = Elem<WDT>::make(s * scale);
  }
}

// positions of a chunk: enough chunks to fill the machine with small batches, few parts with large ones
inline int chunk_of(int64_t n) { return n <= (1 << 14) ? 16 : n <= (1 << 20) ? 64 : 512; }
inline int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

struct Plan {
  int bits, passes, chunk;
  int64_t chunks, items;  // items: bytes of one key or position array
  Plan(int64_t n, int64_t V) {
    int b = 1;
    while ((V >> b) != 0) ++b;  // keys 0 .. V
    passes = (b + kMaxDigit - 1) / kMaxDigit;
    bits = (b + passes - 1) / passes;
    chunk = chunk_of(n);
    chunks = (n + chunk - 1) / chunk;
    items = align16(4 * n);
  }
};

template <int GDT, int WDT, int VEC>
void launch_sum(const Plan& pl, const uint32_t* key, const uint32_t* pos, const void* g, float scale, int64_t n,
                int64_t V, int D, void* gw, float* part, cudaStream_t st) {
  const int tiles = (D + 32 * VEC - 1) / (32 * VEC);
  const int64_t blocks = (pl.chunks * tiles + 7) / 8;
  sum_kernel<GDT, WDT, VEC><<<(unsigned)blocks, 256, 0, st>>>(
      key, pos, reinterpret_cast<const typename Elem<GDT>::T*>(g), scale, n, (uint32_t)V, D, pl.chunk, tiles,
      pl.chunks, reinterpret_cast<typename Elem<WDT>::T*>(gw), part);
}

template <int GDT, int WDT>
void launch_bwd(const Plan& pl, const uint32_t* key, const uint32_t* pos, const void* g, float scale, int64_t n,
                int64_t V, int D, void* gw, float* part, cudaStream_t st) {
  constexpr int kWide = GDT == SPK_F32 || WDT == SPK_F32 ? 4 : 8;  // the wider type's access is 16 bytes
  const int ge = dtype_size(GDT), we = dtype_size(WDT);
  if (D % kWide == 0 && aligned(g, kWide * ge) && aligned(gw, kWide * we))
    launch_sum<GDT, WDT, kWide>(pl, key, pos, g, scale, n, V, D, gw, part, st);
  else
    launch_sum<GDT, WDT, 1>(pl, key, pos, g, scale, n, V, D, gw, part, st);
  if (pl.chunks > 1)
    join_kernel<WDT><<<dim3((unsigned)(pl.chunks - 1), (unsigned)((D + 31) / 32)), 256, 0, st>>>(
        key, scale, n, (uint32_t)V, D, pl.chunk, pl.chunks, reinterpret_cast<typename Elem<WDT>::T*>(gw), part);
}

template <int WDT, int ODT>
void launch_gather(const int64_t* tokens, const void* w, int64_t ldw, float scale, int64_t n, int64_t V, int D,
                   void* out, int* bad, cudaStream_t st) {
  constexpr int kWide = WDT == SPK_F32 || ODT == SPK_F32 ? 4 : 8;
  const bool wide = D % kWide == 0 && ldw % kWide == 0 && aligned(w, kWide * dtype_size(WDT)) &&
                    aligned(out, kWide * dtype_size(ODT));
  int64_t grid = (n * (D / (wide ? kWide : 1)) + 1023) / 1024;
  const int64_t cap = (int64_t)num_sms() * 8;
  if (grid > cap) grid = cap;
  if (grid < 1) grid = 1;
  auto* wp = reinterpret_cast<const typename Elem<WDT>::T*>(w);
  auto* op = reinterpret_cast<typename Elem<ODT>::T*>(out);
  if (wide) gather_kernel<WDT, ODT, kWide><<<(unsigned)grid, 256, 0, st>>>(tokens, wp, ldw, scale, n, V, D, op, bad);
  else gather_kernel<WDT, ODT, 1><<<(unsigned)grid, 256, 0, st>>>(tokens, wp, ldw, scale, n, V, D, op, bad);
}

#define SPK_EMB_TYPES(A, B, CALL)                                                  \
  do {                                                                             \
    if (A == SPK_F32 && B == SPK_F32) { CALL(SPK_F32, SPK_F32); }                  \
    else if (A == SPK_F32 && B == SPK_F16) { CALL(SPK_F32, SPK_F16); }             \
    else if (A == SPK_F32 && B == SPK_BF16) { CALL(SPK_F32, SPK_BF16); }           \
    else if (A == SPK_F16 && B == SPK_F32) { CALL(SPK_F16, SPK_F32); }             \
    else if (A == SPK_F16 && B == SPK_F16) { CALL(SPK_F16, SPK_F16); }             \
    else if (A == SPK_F16 && B == SPK_BF16) { CALL(SPK_F16, SPK_BF16); }           \
    else if (A == SPK_BF16 && B == SPK_F32) { CALL(SPK_BF16, SPK_F32); }           \
    else if (A == SPK_BF16 && B == SPK_F16) { CALL(SPK_BF16, SPK_F16); }           \
    else { CALL(SPK_BF16, SPK_BF16); }                                             \
  } while (0)

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
#define CALL(W, O) launch_gather<W, O>(tokens, weight, ldw, scale, n, V, (int)D, out, bad_token, st)
  SPK_EMB_TYPES(w_dtype, out_dtype, CALL);
#undef CALL
  return check_launch("embedding_fwd");
}

int64_t spk_embedding_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  using namespace spk::embg;
  if (n < 1 || V < 1 || D < 1) return 16;
  const Plan pl(n, V);
  return 4 * pl.items + pl.chunks * 2 * D * (int64_t)sizeof(float);
}

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
  SPK_REQUIRE(aligned(workspace, 16), SPK_ERR_ALIGN, "workspace must be 16-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Plan pl(n, V);
  char* ws = reinterpret_cast<char*>(workspace);
  uint32_t* key0 = reinterpret_cast<uint32_t*>(ws);
  uint32_t* pos0 = reinterpret_cast<uint32_t*>(ws + pl.items);
  uint32_t* key1 = reinterpret_cast<uint32_t*>(ws + 2 * pl.items);
  uint32_t* pos1 = reinterpret_cast<uint32_t*>(ws + 3 * pl.items);
  float* part = reinterpret_cast<float*>(ws + 4 * pl.items);
  const int64_t gw_bytes = V * D * dtype_size(w_dtype);

  const int csize = n <= 4096 ? 1 : 8;
  int64_t fill = (gw_bytes + (int64_t)csize * (64 << 10) - 1) / ((int64_t)csize * (64 << 10));
  const int64_t most = num_sms() / csize;
  if (fill > most) fill = most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((1 + fill) * csize));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = (size_t)((kSortWarps + 2) << pl.bits) * 4;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)csize, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaFuncSetAttribute(sort_clear_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)((kSortWarps + 2) << kMaxDigit) * 4);
  if (e == cudaSuccess)
    e = cudaLaunchKernelEx(&cfg, sort_clear_kernel, tokens, n, V, padding_idx, pl.bits, pl.passes, key0, pos0, key1,
                           pos1, gw, gw_bytes);
  if (e != cudaSuccess) return fail(SPK_ERR_LAUNCH, "embedding_bwd: %s", cudaGetErrorString(e));
  const uint32_t* key = pl.passes & 1 ? key0 : key1;
  const uint32_t* pos = pl.passes & 1 ? pos0 : pos1;
#define CALL(G, W) launch_bwd<G, W>(pl, key, pos, g, scale, n, V, (int)D, gw, part, st)
  SPK_EMB_TYPES(g_dtype, w_dtype, CALL);
#undef CALL
  return check_launch("embedding_bwd");
}

}  // extern "C"
