// LayerNorm over the last dimension, forward and backward (no LIF behind it:
// ln_lif.cu has the fused form for T <= 4).
//
//   y = h * w + b,  h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   g_b = sum_rows g,  g_w = sum_rows g * h
//   g_x = rstd * (a - mean(a) - h * mean(a * h)),  a = g * w
//
// The variance is the mean of (x - mean)^2, a second sweep over the row in
// registers, so a large common offset costs no digits.  All sums are fp32 in a
// fixed order.
//
// Bound by HBM.  A row lives in the registers of 1 to 16 warps (a group), read
// once and written once; a lane owns the same columns of every row, so w and b
// (and, in the backward, the column sums of g_w and g_b) stay in registers too.
// Groups walk over the rows and have the next row's loads on their way while
// they reduce the present one.  A group of one warp needs shuffles only; a wider
// one meets at a named barrier.  The fewest warps are taken that hold the row
// in kNvFwd (kNvBwd) vectors a lane: the backward keeps five values a column
// instead of three.
#include "vec.cuh"

namespace spk {
namespace lnk {

constexpr int kWarps = 8;         // warps of a block (16 where a group is)
constexpr int kMaxGroup = 16;     // warps of a group

// Sums over a group of `wpr` warps.  `turn` alternates between two slots of
// shared memory, so that one barrier a sum is enough.
struct GroupSum {
  float2* slot;  // [2][kMaxGroup] of this group
  int wpr, warp, lane, bar, turn;
  __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (wpr == 1) return v;
    float2* s = slot + turn * kMaxGroup;
    turn ^= 1;
    if (lane == 0) s[warp] = v;
    named_bar_sync(bar, wpr * 32);
    v = lane < wpr ? s[lane] : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int o = kMaxGroup / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return make_float2(__shfl_sync(0xffffffffu, v.x, 0), __shfl_sync(0xffffffffu, v.y, 0));
  }
  __device__ __forceinline__ float operator()(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (wpr == 1) return x;
    float2* s = slot + turn * kMaxGroup;
    turn ^= 1;
    if (lane == 0) s[warp].x = x;
    named_bar_sync(bar, wpr * 32);
    x = lane < wpr ? s[lane].x : 0.0f;
#pragma unroll
    for (int o = kMaxGroup / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return __shfl_sync(0xffffffffu, x, 0);
  }
};

// where the calling thread stands: its group among all groups, and its column of vector i
struct Place {
  int lane, group, in_group;  // group of the block, warp of the group
  int64_t first, step;        // rows of the group: first, first + step, ...
  __device__ __forceinline__ Place(int wpr) {
    const int warp = threadIdx.x >> 5, groups = (blockDim.x >> 5) / wpr;
    lane = threadIdx.x & 31;
    group = warp / wpr;
    in_group = warp - group * wpr;
    first = (int64_t)blockIdx.x * groups + group;
    step = (int64_t)gridDim.x * groups;
  }
};

template <int DT, int VEC, int NV>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* row, int col, int stride, int D,
                                         typename Vec<DT, VEC>::W (&w)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (col + i * stride < D) w[i] = Vec<DT, VEC>::raw(row + col + i * stride);
}

template <int VEC>
__device__ __forceinline__ void store_as(void* y, int ydt, int64_t at, const float (&v)[VEC]) {
  if (ydt == SPK_F32) Vec<SPK_F32, VEC>::store(reinterpret_cast<float*>(y) + at, v);
  else if (ydt == SPK_F16) Vec<SPK_F16, VEC>::store(reinterpret_cast<__half*>(y) + at, v);
  else Vec<SPK_BF16, VEC>::store(reinterpret_cast<__nv_bfloat16*>(y) + at, v);
}

template <int XDT, int VEC, int NV>
__global__ void __launch_bounds__(32 * kMaxGroup) fwd_kernel(const typename Elem<XDT>::T* __restrict__ x, int64_t ld,
                                                             const void* w, int wdt, const void* b, int bdt, float eps,
                                                             int64_t rows, int D, int wpr, void* __restrict__ y,
                                                             int ydt, float2* __restrict__ stats) {
  __shared__ float2 slots[kWarps][2 * kMaxGroup];
  const Place pl(wpr);
  GroupSum sum{slots[pl.group], wpr, pl.in_group, pl.lane, pl.group + 1, 0};
  const int stride = 32 * VEC * wpr, col = (pl.in_group * 32 + pl.lane) * VEC;
  using W = typename Vec<XDT, VEC>::W;
  W next[NV];
  if (pl.first < rows) load_row<XDT, VEC, NV>(x + pl.first * ld, col, stride, D, next);
  float wv[NV * VEC], bv[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = col + i * stride + j;
      wv[i * VEC + j] = w && c < D ? ld_any(w, wdt, c) : 1.0f;
      bv[i * VEC + j] = b && c < D ? ld_any(b, bdt, c) : 0.0f;
    }
  const float inv_d = 1.0f / (float)D;
  for (int64_t r = pl.first; r < rows; r += pl.step) {
    W now[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) now[i] = next[i];
    if (r + pl.step < rows) load_row<XDT, VEC, NV>(x + (r + pl.step) * ld, col, stride, D, next);
    float v[NV][VEC], s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col + i * stride < D) {
        Vec<XDT, VEC>::unpack(now[i], v[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[i][j];
      }
    }
    const float mean = sum(s) * inv_d;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col + i * stride < D)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] -= mean;
          q = fmaf(v[i][j], v[i][j], q);
        }
    const float rstd = 1.0f / sqrtf(fmaf(sum(q), inv_d, eps));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col + i * stride < D) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = fmaf(v[i][j] * rstd, wv[i * VEC + j], bv[i * VEC + j]);
        store_as<VEC>(y, ydt, r * D + col + i * stride, o);
      }
    if (stats && pl.in_group == 0 && pl.lane == 0) stats[r] = make_float2(mean, rstd);
  }
}

// part[block][2][D]: (sum g * h, sum g) over the block's rows
template <int GDT, int XDT, int VEC, int NV>
__global__ void __launch_bounds__(32 * kMaxGroup) bwd_kernel(const typename Elem<GDT>::T* __restrict__ g,
                                                             const typename Elem<XDT>::T* __restrict__ x, int64_t ld,
                                                             const float2* __restrict__ stats, const void* w, int wdt,
                                                             int64_t rows, int D, int wpr,
                                                             typename Elem<XDT>::T* __restrict__ gx,
                                                             float* __restrict__ part) {
  extern __shared__ float cols[];  // [2][D] where a block has several groups
  __shared__ float2 slots[kWarps][2 * kMaxGroup];
  pdl_trigger();
  const Place pl(wpr);
  GroupSum sum{slots[pl.group], wpr, pl.in_group, pl.lane, pl.group + 1, 0};
  const int stride = 32 * VEC * wpr, col = (pl.in_group * 32 + pl.lane) * VEC;
  typename Vec<XDT, VEC>::W nx[NV];
  typename Vec<GDT, VEC>::W ng[NV];
  float2 ns = make_float2(0.0f, 0.0f);
  if (pl.first < rows) {
    load_row<XDT, VEC, NV>(x + pl.first * ld, col, stride, D, nx);
    load_row<GDT, VEC, NV>(g + pl.first * D, col, stride, D, ng);
    ns = stats[pl.first];
  }
  float wv[NV][VEC], sw[NV][VEC], sb[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = col + i * stride + j;
      wv[i][j] = w && c < D ? ld_any(w, wdt, c) : 1.0f;
      sw[i][j] = sb[i][j] = 0.0f;
    }
  const float inv_d = 1.0f / (float)D;
  for (int64_t r = pl.first; r < rows; r += pl.step) {
    float h[NV][VEC], a[NV][VEC];
    const float mean = ns.x, rstd = ns.y;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col + i * stride < D) {
        Vec<XDT, VEC>::unpack(nx[i], h[i]);
        Vec<GDT, VEC>::unpack(ng[i], a[i]);
      }
    if (r + pl.step < rows) {
      load_row<XDT, VEC, NV>(x + (r + pl.step) * ld, col, stride, D, nx);
      load_row<GDT, VEC, NV>(g + (r + pl.step) * D, col, stride, D, ng);
      ns = stats[r + pl.step];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col + i * stride < D)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[i][j] = (h[i][j] - mean) * rstd;
          sw[i][j] = fmaf(a[i][j], h[i][j], sw[i][j]);
          sb[i][j] += a[i][j];
          a[i][j] *= wv[i][j];
          s.x += a[i][j];
          s.y = fmaf(a[i][j], h[i][j], s.y);
        }
    if (gx) {
      s = sum(s);
      const float ma = s.x * inv_d, mh = s.y * inv_d;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (col + i * stride < D) {
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = rstd * (a[i][j] - ma - h[i][j] * mh);
          Vec<XDT, VEC>::store(gx + r * D + col + i * stride, o);
        }
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * D;
  const int groups = (blockDim.x >> 5) / wpr;
  for (int k = 0; k < groups; ++k) {  // the groups in turn, the last one to global memory
    if (pl.group == k)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (col + i * stride < D)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = col + i * stride + j;
            if (k > 0) {
              sw[i][j] += cols[c];
              sb[i][j] += cols[D + c];
            }
            float* to = k + 1 < groups ? cols : out;
            to[c] = sw[i][j];
            to[D + c] = sb[i][j];
          }
    if (k + 1 < groups) __syncthreads();
  }
}

// g_w and g_b from the blocks' parts: 32 columns a block, the parts cut over its warps
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ part, int parts, int D, void* gw, int wdt,
                                                    void* gb, int bdt) {
  __shared__ float red[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;  // of [2 D]
  float s = 0.0f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) s += part[(int64_t)p * 2 * D + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  s = red[lane][warp];  // lane's part of column `warp`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int k = blockIdx.x * 32 + warp;
  if (lane == 0 && k < 2 * D) {
    if (k < D) {
      if (gw) st_any(gw, wdt, k, s);
    } else if (gb) {
      st_any(gb, bdt, k - D, s);
    }
  }
}

// ---------------------------------------------------------------- rows too long for the registers
// A block a row (or a column strip), reading the row again for every sweep.

constexpr int kLong = 512;

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float red[kLong / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kLong / 32; ++i) s += red[i];
  return s;
}

__global__ void __launch_bounds__(kLong) long_fwd_kernel(const void* x, int xdt, int64_t ld, const void* w, int wdt,
                                                         const void* b, int bdt, float eps, int64_t rows, int D,
                                                         void* y, int ydt, float2* stats) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    float s = 0.0f;
    for (int i = threadIdx.x; i < D; i += kLong) s += ld_any(x, xdt, r * ld + i);
    const float mean = block_sum(s) / (float)D;
    float q = 0.0f;
    for (int i = threadIdx.x; i < D; i += kLong) {
      const float c = ld_any(x, xdt, r * ld + i) - mean;
      q = fmaf(c, c, q);
    }
    const float rstd = 1.0f / sqrtf(block_sum(q) / (float)D + eps);
    for (int i = threadIdx.x; i < D; i += kLong) {
      const float h = (ld_any(x, xdt, r * ld + i) - mean) * rstd;
      st_any(y, ydt, r * D + i, fmaf(h, w ? ld_any(w, wdt, i) : 1.0f, b ? ld_any(b, bdt, i) : 0.0f));
    }
    if (stats && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
  }
}

__global__ void __launch_bounds__(kLong) long_bwd_x_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                           const float2* stats, const void* w, int wdt, int64_t rows,
                                                           int D, void* gx) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[r].x, rstd = stats[r].y;
    float sa = 0.0f, sh = 0.0f;
    for (int i = threadIdx.x; i < D; i += kLong) {
      const float a = ld_any(g, gdt, r * D + i) * (w ? ld_any(w, wdt, i) : 1.0f);
      sa += a;
      sh = fmaf(a, (ld_any(x, xdt, r * ld + i) - mean) * rstd, sh);
    }
    const float ma = block_sum(sa) / (float)D, mh = block_sum(sh) / (float)D;
    for (int i = threadIdx.x; i < D; i += kLong) {
      const float a = ld_any(g, gdt, r * D + i) * (w ? ld_any(w, wdt, i) : 1.0f);
      const float h = (ld_any(x, xdt, r * ld + i) - mean) * rstd;
      st_any(gx, xdt, r * D + i, rstd * (a - ma - h * mh));
    }
  }
}

__global__ void __launch_bounds__(kLong) long_bwd_w_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                           const float2* stats, int64_t rows, int D, float* part) {
  pdl_trigger();
  const int i = blockIdx.x * kLong + threadIdx.x;
  if (i >= D) return;
  float sw = 0.0f, sb = 0.0f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float gv = ld_any(g, gdt, r * D + i);
    sw = fmaf(gv, (ld_any(x, xdt, r * ld + i) - stats[r].x) * stats[r].y, sw);
    sb += gv;
  }
  part[(int64_t)blockIdx.y * 2 * D + i] = sw;
  part[((int64_t)blockIdx.y * 2 + 1) * D + i] = sb;
}

// ---------------------------------------------------------------- which kernel, how many blocks

// vectors (single elements) a lane holds at most, forward and backward
constexpr int kNvFwd = 6, kNvBwd = 4, kNv1Fwd = 24, kNv1Bwd = 16;

struct Shape {
  int vec, nv, wpr;  // nv = 0: the row does not fit the registers
  Shape(int64_t D, bool wide, int most4, int most1) {
    vec = wide ? 4 : 1;
    const int most = wide ? most4 : most1;
    const int64_t vecs = (D + vec - 1) / vec;
    for (wpr = 1; wpr < kMaxGroup && vecs > 32ll * wpr * most; wpr *= 2) {}
    const int64_t n = (vecs + 32 * wpr - 1) / (32 * wpr);
    nv = n > most ? 0 : (int)n;
  }
  int threads() const { return 32 * (wpr > kWarps ? wpr : kWarps); }
  int groups() const { return wpr > kWarps ? 1 : kWarps / wpr; }
};

inline unsigned blocks_of(int64_t rows, const Shape& s, int per_sm) {
  const int64_t need = (rows + s.groups() - 1) / s.groups(), cap = (int64_t)num_sms() * per_sm * kWarps * 32 / s.threads();
  return (unsigned)(need < cap ? need : cap);
}

constexpr int kFwdPerSm = 4, kBwdPerSm = 2, kLongChunks = 64;

// parts of the backward's column sums, whatever its kernel
inline int64_t max_parts(int64_t rows) {
  const int64_t cap = (int64_t)num_sms() * kBwdPerSm;
  return rows < cap ? rows : cap > kLongChunks ? cap : kLongChunks;
}

template <int XDT, int VEC, int NV>
void launch_fwd(const void* x, int64_t ld, const void* w, int wdt, const void* b, int bdt, float eps, int64_t rows,
                int64_t D, const Shape& s, void* y, int ydt, float* stats, cudaStream_t st) {
  fwd_kernel<XDT, VEC, NV><<<blocks_of(rows, s, kFwdPerSm), s.threads(), 0, st>>>(
      reinterpret_cast<const typename Elem<XDT>::T*>(x), ld, w, wdt, b, bdt, eps, rows, (int)D, s.wpr, y, ydt,
      reinterpret_cast<float2*>(stats));
}

template <int GDT, int XDT, int VEC, int NV>
int launch_bwd(const void* g, const void* x, int64_t ld, const float* stats, const void* w, int wdt, int64_t rows,
               int64_t D, const Shape& s, void* gx, float* part, cudaStream_t st) {
  const unsigned blocks = blocks_of(rows, s, kBwdPerSm);
  const size_t smem = part && s.groups() > 1 ? (size_t)(2 * D) * sizeof(float) : 0;
  bwd_kernel<GDT, XDT, VEC, NV><<<blocks, s.threads(), smem, st>>>(
      reinterpret_cast<const typename Elem<GDT>::T*>(g), reinterpret_cast<const typename Elem<XDT>::T*>(x), ld,
      reinterpret_cast<const float2*>(stats), w, wdt, rows, (int)D, s.wpr,
      reinterpret_cast<typename Elem<XDT>::T*>(gx), part);
  return (int)blocks;
}

template <int XDT>
bool dispatch_fwd(const void* x, int64_t ld, const void* w, int wdt, const void* b, int bdt, float eps, int64_t rows,
                  int64_t D, const Shape& s, void* y, int ydt, float* stats, cudaStream_t st) {
#define GO(VEC, NV) (launch_fwd<XDT, VEC, NV>(x, ld, w, wdt, b, bdt, eps, rows, D, s, y, ydt, stats, st), true)
  if (s.nv == 0) return false;
  if (s.vec == 4) {
    switch (s.nv) {
      case 1: return GO(4, 1);
      case 2: return GO(4, 2);
      case 3: return GO(4, 3);
      case 4: return GO(4, 4);
      default: return GO(4, 6);
    }
  }
  return s.nv <= 6 ? GO(1, 6) : s.nv <= 12 ? GO(1, 12) : GO(1, 24);
#undef GO
}

template <int GDT, int XDT>
int dispatch_bwd(const void* g, const void* x, int64_t ld, const float* stats, const void* w, int wdt, int64_t rows,
                 int64_t D, const Shape& s, void* gx, float* part, cudaStream_t st) {
#define GO(VEC, NV) launch_bwd<GDT, XDT, VEC, NV>(g, x, ld, stats, w, wdt, rows, D, s, gx, part, st)
  if (s.vec == 4) {
    switch (s.nv) {
      case 1: return GO(4, 1);
      case 2: return GO(4, 2);
      case 3: return GO(4, 3);
      default: return GO(4, 4);
    }
  }
  return s.nv <= 4 ? GO(1, 4) : s.nv <= 10 ? GO(1, 10) : GO(1, 16);
#undef GO
}

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
  SPK_REQUIRE(aligned(stats, 8), SPK_ERR_ALIGN, "stats must be 8-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = D % 4 == 0 && ld % 4 == 0 && aligned(x, 4 * dtype_size(x_dtype)) && aligned(y, 4 * dtype_size(y_dtype));
  const Shape s(D, wide, kNvFwd, kNv1Fwd);
  auto go = x_dtype == SPK_F32 ? dispatch_fwd<SPK_F32> : x_dtype == SPK_F16 ? dispatch_fwd<SPK_F16> : dispatch_fwd<SPK_BF16>;
  if (!go(x, ld, w, w_dtype, b, b_dtype, eps, rows, D, s, y, y_dtype, stats, st)) {
    const int64_t cap = (int64_t)num_sms() * 4;
    long_fwd_kernel<<<(unsigned)(rows < cap ? rows : cap), kLong, 0, st>>>(x, x_dtype, ld, w, w_dtype, b, b_dtype, eps,
                                                                          rows, (int)D, y, y_dtype,
                                                                          reinterpret_cast<float2*>(stats));
  }
  return check_launch("layer_norm_fwd");
}

int64_t spk_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D) {
  return rows < 1 || D < 1 ? 16 : spk::lnk::max_parts(rows) * 2 * D * (int64_t)sizeof(float);
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
  SPK_REQUIRE(aligned(stats, 8) && aligned(workspace, 4), SPK_ERR_ALIGN, "stats or workspace misaligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  if (!gx && !gw && !gb) return SPK_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  float* part = gw || gb ? reinterpret_cast<float*>(workspace) : nullptr;
  const bool wide = D % 4 == 0 && ld % 4 == 0 && aligned(x, 4 * dtype_size(x_dtype)) &&
                    aligned(g, 4 * dtype_size(g_dtype)) && aligned(gx, 4 * dtype_size(x_dtype));
  const Shape s(D, wide, kNvBwd, kNv1Bwd);
  int parts;
  if (s.nv > 0) {
#define GO(G, X) dispatch_bwd<G, X>(g, x, ld, stats, w, w_dtype, rows, D, s, gx, part, st)
#define GOX(G) (x_dtype == SPK_F32 ? GO(G, SPK_F32) : x_dtype == SPK_F16 ? GO(G, SPK_F16) : GO(G, SPK_BF16))
    parts = g_dtype == SPK_F32 ? GOX(SPK_F32) : g_dtype == SPK_F16 ? GOX(SPK_F16) : GOX(SPK_BF16);
#undef GOX
#undef GO
  } else {
    const float2* sv = reinterpret_cast<const float2*>(stats);
    const int64_t cap = (int64_t)num_sms() * 4;
    if (gx)
      long_bwd_x_kernel<<<(unsigned)(rows < cap ? rows : cap), kLong, 0, st>>>(g, g_dtype, x, x_dtype, ld, sv, w, w_dtype,
                                                                              rows, (int)D, gx);
    parts = (int)(rows < kLongChunks ? rows : kLongChunks);
    if (part)
      long_bwd_w_kernel<<<dim3((unsigned)((D + kLong - 1) / kLong), (unsigned)parts), kLong, 0, st>>>(
          g, g_dtype, x, x_dtype, ld, sv, rows, (int)D, part);
  }
  if (part) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((2 * D + 31) / 32));
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    add_pdl_attr(cfg, at);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel, (const float*)part, parts, (int)D, gw, w_dtype, gb,
                                             b_dtype);
    if (e != cudaSuccess) return fail(SPK_ERR_LAUNCH, "layer_norm_bwd: %s", cudaGetErrorString(e));
  }
  return check_launch("layer_norm_bwd");
}

}  // extern "C"
