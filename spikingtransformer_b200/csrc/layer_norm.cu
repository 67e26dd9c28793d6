// LayerNorm over the last dimension, forward and backward (no LIF behind it:
// ln_lif.cu has the fused form for T <= 4).
//
//   y = h * w + b,  h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   g_b = sum_rows g,  g_w = sum_rows g * h
//   g_x = rstd * (a - mean(a) - h * mean(a * h)),  a = g * w
//
// The variance is the mean of (x - mean)^2, a second sweep over the row in
// registers, so a large common offset does not cancel in it as it would in
// mean(x^2) - mean^2.  The mean itself is an fp32 sum: its error, some 2^-24 of
// |mean|, moves a whole row of h by that over the standard deviation (by up to
// 1e-4 with 384 values about 1000 of deviation 1.5).  All sums are fp32 in a fixed
// order.
//
// Bound by HBM.  A row lives in the registers of a group of 8 lanes to 16 warps,
// read once and written once; a lane owns the same columns of every row, so w and b
// (and, in the backward, the column sums of g_w and g_b) stay in registers too.
// Groups walk over the rows.  Rows that can be read in vectors of four are copied
// asynchronously, up to four rows ahead, into a ring in shared memory: a lane
// reads back only what it copied itself, so the ring needs no barrier.  Other
// rows go element by element through registers, one row ahead.  A group within
// a warp needs shuffles only; a wider one meets at a named barrier.  The fewest
// warps are taken that hold the row in kNvFwd (kNvBwd) vectors a lane: the
// backward keeps five values a column instead of three.  Rows of up to 16
// vectors share a warp: with a warp each, 262144 rows of 64 bf16 took 41 us
// forward and 57 us backward instead of 25 and 41.  Columns past the end
// hold zeros, and the arithmetic runs on pairs (fp32x2) without asking where
// they are: with a branch for them a row took three times the instructions, and
// 65536 x 1536 bf16 forward and backward 351 us instead of 193.
#include "vec.cuh"

namespace spk {
namespace lnk {

constexpr int kWarps = 8;         // warps of a block (16 where a group is)
constexpr int kMaxGroup = 16;     // warps of a group

// Sums over a group of `wpr` warps.  `turn` alternates between two slots of
// shared memory, so that one barrier a sum is enough.
struct GroupSum {
  float2* slot;  // [2][kMaxGroup] of this group
  int wpr, warp, lane, bar, turn, lpr;  // lpr: lanes of a group within a warp
  __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      if (o < lpr) {
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
    for (int o = 1; o < 32; o <<= 1)
      if (o < lpr) x += __shfl_xor_sync(0xffffffffu, x, o);
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

// Where the calling thread stands: its group, the rows that the group walks over
// (first, first + step, ...), how many they are, and its lane in its warp's part
// of the group.  wpr: warps of a group, lpr: lanes where several share a warp.
// The lanes of a warp take turns together: `turns` is the most of its groups.
struct Place {
  int lane, group, in_group, count, turns;
  int64_t first, step;
  __device__ __forceinline__ Place(int wpr, int lpr, int64_t rows) {
    const int warp = threadIdx.x >> 5, per_warp = 32 / lpr, groups = (blockDim.x >> 5) / wpr * per_warp;
    lane = (threadIdx.x & 31) & (lpr - 1);
    in_group = wpr > 1 ? warp % wpr : 0;
    group = wpr > 1 ? warp / wpr : warp * per_warp + (threadIdx.x & 31) / lpr;
    first = (int64_t)blockIdx.x * groups + group;
    step = (int64_t)gridDim.x * groups;
    count = first < rows ? (int)((rows - first + step - 1) / step) : 0;
    turns = __shfl_sync(0xffffffffu, count, 0);  // the warp's first group has the lowest row
  }
};

// A lane's values of a row as pairs: vector i of four is pairs 2 i and 2 i + 1,
// single elements 2 i and 2 i + 1 are pair i.
template <int DT, int VEC, int NV>
struct Pairs {
  static constexpr int P = NV * VEC / 2;
  using E = typename Elem<DT>::T;
  using W = typename Vec<DT, VEC>::W;
  static_assert(VEC == 4 || (VEC == 1 && NV % 2 == 0), "vectors of four, or an even number of elements");
  __device__ static __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (DT == SPK_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  __device__ static __forceinline__ uint32_t pack2(float2 v) {
    if constexpr (DT == SPK_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ void unpack(const W (&w)[NV], float2 (&v)[P]) {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float lo[1], hi[1];
        Vec<DT, 1>::unpack(w[2 * i], lo);
        Vec<DT, 1>::unpack(w[2 * i + 1], hi);
        v[i] = make_float2(lo[0], hi[0]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (DT == SPK_F32) {
          v[2 * i] = make_float2(__uint_as_float(w[i].x), __uint_as_float(w[i].y));
          v[2 * i + 1] = make_float2(__uint_as_float(w[i].z), __uint_as_float(w[i].w));
        } else {
          v[2 * i] = unpack2(w[i].x);
          v[2 * i + 1] = unpack2(w[i].y);
        }
      }
    }
  }
  // the values to a row, from column `col` of D
  __device__ static __forceinline__ void store(E* row, int col, int D, const float2 (&v)[P]) {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (col + i * 32 < D) row[i * 32] = Elem<DT>::make(i & 1 ? v[i / 2].y : v[i / 2].x);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        W w;
        if constexpr (DT == SPK_F32) {
          w.x = __float_as_uint(v[2 * i].x);
          w.y = __float_as_uint(v[2 * i].y);
          w.z = __float_as_uint(v[2 * i + 1].x);
          w.w = __float_as_uint(v[2 * i + 1].y);
        } else {
          w.x = pack2(v[2 * i]);
          w.y = pack2(v[2 * i + 1]);
        }
        if (col + i * 128 < D) *reinterpret_cast<W*>(row + i * 128) = w;
      }
    }
  }
};

// A lane's vectors of the coming rows, zeros past column D and past the last
// row.  VEC > 1: `S` rows in a ring in shared memory; VEC = 1: the next row in
// registers.
template <int DT, int VEC, int NV, int S>
struct Rows {
  using E = typename Elem<DT>::T;
  using W = typename Vec<DT, VEC>::W;
  using PR = Pairs<DT, VEC, NV>;
  static constexpr int kBytes = VEC > 1 ? S * NV * (int)sizeof(W) : 0;  // of shared memory a thread
  W next[VEC > 1 ? 1 : NV];
  uint32_t mine, at;  // the lane's part of the ring [S][NV][32], and the slot's offset in it
  const E* src;       // the lane's first column of the next row to fetch
  int64_t hop;
  int left, col, D;   // rows to fetch
  __device__ __forceinline__ Rows(void* ring, const E* base, int64_t ld, const Place& pl, int c, int cols)
      : mine(0), at(0), src(base + (pl.count > 0 ? pl.first * ld : 0) + (c < cols ? c : 0)), hop(pl.step * ld), left(pl.count), col(c), D(cols) {
    if constexpr (VEC > 1)
      mine = smem_u32(ring) + (threadIdx.x >> 5) * 32 * kBytes + (threadIdx.x & 31) * (int)sizeof(W);
    else
#pragma unroll
      for (int i = 0; i < NV; ++i) next[i] = 0;
  }
  __device__ __forceinline__ void fetch() {
    const bool in = left > 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool on = in && col + i * 32 * VEC < D;
      if constexpr (VEC > 1) {
        // no bytes to copy: zeros are written, the address is not read
        const uint32_t to = mine + at + i * 32 * (int)sizeof(W);
        const int bytes = on ? (int)sizeof(W) : 0;
        if constexpr (sizeof(W) == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src + (on ? i * 32 * VEC : 0)),
                       "r"(bytes)
                       : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(src + (on ? i * 32 * VEC : 0)),
                       "r"(bytes)
                       : "memory");
      } else if (on) {
        next[i] = Vec<DT, VEC>::raw(src + i * 32);
      }
    }
    if (--left > 0) src += hop;
    at = at + NV * 32 * (int)sizeof(W) == (uint32_t)(kBytes * 32) ? 0 : at + NV * 32 * (int)sizeof(W);
  }
  // the oldest row
  __device__ __forceinline__ void take(float2 (&v)[PR::P]) {
    if constexpr (VEC > 1) {
      W w[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t from = mine + at + i * 32 * (int)sizeof(W);
        if constexpr (sizeof(W) == 16)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                       : "r"(from)
                       : "memory");
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[i].x), "=r"(w[i].y) : "r"(from) : "memory");
      }
      PR::unpack(w, v);
    } else {
      PR::unpack(next, v);
    }
  }
};
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// column of the lane's value that is half `hi` of pair p
template <int VEC>
__device__ __forceinline__ int pair_col(int col, int p, int hi) {
  return VEC == 4 ? col + (p >> 1) * 128 + (p & 1) * 2 + hi : col + (2 * p + hi) * 32;
}

// the lane's columns of a parameter, `other` where there is none, zeros past column D
template <int VEC, int P>
__device__ __forceinline__ void load_param(const void* w, int wdt, int col, int D, float other, float2 (&v)[P]) {
  auto go = [&](auto at) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c0 = pair_col<VEC>(col, p, 0), c1 = pair_col<VEC>(col, p, 1);
      v[p] = make_float2(c0 < D ? at(c0) : 0.0f, c1 < D ? at(c1) : 0.0f);
    }
  };
  if (!w) go([&](int) { return other; });
  else if (wdt == SPK_F32) go([&](int c) { return __ldg(reinterpret_cast<const float*>(w) + c); });
  else if (wdt == SPK_F16) go([&](int c) { return __half2float(reinterpret_cast<const __half*>(w)[c]); });
  else go([&](int c) { return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[c]); });
}

// rows ahead: as many as 48 KB (forward) or 96 KB (backward) of shared memory hold for 256 threads, at most 4
constexpr int ahead(int bytes_a_row, int most) {
  return most / bytes_a_row > 4 ? 4 : most / bytes_a_row < 2 ? 2 : most / bytes_a_row;
}

template <int XDT, int VEC, int NV>
struct Fwd {
  static constexpr int S = VEC > 1 ? ahead(NV * VEC * (int)sizeof(typename Elem<XDT>::T), 192) : 1;
  using X = Rows<XDT, VEC, NV, S>;
};
template <int GDT, int XDT, int VEC, int NV>
struct Bwd {
  static constexpr int S =
      VEC > 1 ? ahead(NV * VEC * (int)(sizeof(typename Elem<XDT>::T) + sizeof(typename Elem<GDT>::T)), 384) : 1;
  using X = Rows<XDT, VEC, NV, S>;
  using G = Rows<GDT, VEC, NV, S>;
};

// 262144 x 384 bf16: 76 us, 5.3 TB/s (0.82 of a plain copy); 65536 x 1536: 77 us.
template <int XDT, int VEC, int NV>
__global__ void __launch_bounds__(NV == 8 ? 32 * kWarps : 32 * kMaxGroup) fwd_kernel(const typename Elem<XDT>::T* __restrict__ x, int64_t ld,
                                                             const void* w, int wdt, const void* b, int bdt, float eps,
                                                             int64_t rows, int D, int wpr, int lpr, void* __restrict__ y,
                                                             int ydt, float2* __restrict__ stats) {
  extern __shared__ uint4 ring[];
  __shared__ float2 slots[kWarps][2 * kMaxGroup];  // of groups of several warps
  constexpr int S = Fwd<XDT, VEC, NV>::S, P = NV * VEC / 2;
  const Place pl(wpr, lpr, rows);
  GroupSum sum{slots[wpr > 1 ? pl.group : 0], wpr, pl.in_group, pl.lane, pl.group + 1, 0, lpr};
  const int col = (pl.in_group * 32 * NV + pl.lane) * VEC;
  typename Fwd<XDT, VEC, NV>::X in(ring, x, ld, pl, col, D);
#pragma unroll
  for (int k = 0; k < S; ++k) {
    in.fetch();
    commit_copies();
  }
  float2 wv[P], bv[P];
  load_param<VEC, P>(w, wdt, col, D, 1.0f, wv);
  load_param<VEC, P>(b, bdt, col, D, 0.0f, bv);
  const float inv_d = 1.0f / (float)D;
  int64_t at = pl.first * D + col;  // of y
  const int64_t hop = pl.step * D;
  float2* st = stats ? stats + pl.first : nullptr;
  for (int n = 0; n < pl.turns; ++n, at += hop) {
    const bool here = n < pl.count;  // not behind the last row
    float2 v[P];
    wait_copies<S - 1>();
    in.take(v);
    float2 s2 = v[0];
#pragma unroll
    for (int p = 1; p < P; ++p) s2 = add2(s2, v[p]);
    const float part = s2.x + s2.y;
    in.fetch();
    commit_copies();
    const float mean = sum(part) * inv_d;
    const float2 shift = make_float2(-mean, -mean);
    float2 q2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      v[p] = add2(v[p], shift);
      if (pair_col<VEC>(col, p, 0) >= D) v[p].x = 0.0f;
      if (pair_col<VEC>(col, p, 1) >= D) v[p].y = 0.0f;
      q2 = fma2(v[p], v[p], q2);
    }
    const float rstd = rsqrtf(fmaf(sum(q2.x + q2.y), inv_d, eps));
    const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
    for (int p = 0; p < P; ++p) v[p] = fma2(mul2(v[p], r2), wv[p], bv[p]);
    const int end = here ? D : 0;
    if (ydt == SPK_F32) Pairs<SPK_F32, VEC, NV>::store(reinterpret_cast<float*>(y) + at, col, end, v);
    else if (ydt == SPK_F16) Pairs<SPK_F16, VEC, NV>::store(reinterpret_cast<__half*>(y) + at, col, end, v);
    else Pairs<SPK_BF16, VEC, NV>::store(reinterpret_cast<__nv_bfloat16*>(y) + at, col, end, v);
    if (stats) {
      if (here && pl.in_group == 0 && pl.lane == 0) *st = make_float2(mean, rstd);
      st += pl.step;
    }
  }
  wait_copies<0>();
}

// part[block][2][D]: (sum g * h, sum g) over the block's rows.  65536 x 1536 bf16:
// 107 us, 5.6 TB/s.
template <int GDT, int XDT, int VEC, int NV>
__global__ void __launch_bounds__(32 * kMaxGroup) bwd_kernel(const typename Elem<GDT>::T* __restrict__ g,
                                                             const typename Elem<XDT>::T* __restrict__ x, int64_t ld,
                                                             const float2* __restrict__ stats, const void* w, int wdt,
                                                             int64_t rows, int D, int wpr, int lpr,
                                                             typename Elem<XDT>::T* __restrict__ gx,
                                                             float* __restrict__ part) {
  extern __shared__ uint4 ring[];  // the rows ahead; at the end [groups][2][D] column sums
  __shared__ float2 slots[kWarps][2 * kMaxGroup];
  using T = Bwd<GDT, XDT, VEC, NV>;
  constexpr int S = T::S, P = NV * VEC / 2;
  pdl_trigger();
  const Place pl(wpr, lpr, rows);
  GroupSum sum{slots[wpr > 1 ? pl.group : 0], wpr, pl.in_group, pl.lane, pl.group + 1, 0, lpr};
  const int col = (pl.in_group * 32 * NV + pl.lane) * VEC;
  typename T::X xin(ring, x, ld, pl, col, D);
  typename T::G gin(reinterpret_cast<char*>(ring) + T::X::kBytes * (int)blockDim.x, g, D, pl, col, D);
#pragma unroll
  for (int k = 0; k < S; ++k) {
    xin.fetch();
    gin.fetch();
    commit_copies();
  }
  // statistics of the present row and the next one
  const float2* st = stats + pl.first;
  float2 st0 = pl.count > 0 ? *st : make_float2(0.0f, 0.0f), st1 = st0;
  if (pl.count > 1) st1 = *(st += pl.step);
  float2 wv[P], sw[P], sb[P];
  load_param<VEC, P>(w, wdt, col, D, 1.0f, wv);
#pragma unroll
  for (int p = 0; p < P; ++p) sw[p] = sb[p] = make_float2(0.0f, 0.0f);
  const float inv_d = 1.0f / (float)D;
  int64_t at = pl.first * D + col;  // of gx
  const int64_t hop = pl.step * D;
  for (int n = 0; n < pl.turns; ++n, at += hop) {
    const bool here = n < pl.count;  // behind the last row x and g are zeros
    float2 h[P], a[P];
    const float2 shift = make_float2(-st0.x, -st0.x), r2 = make_float2(st0.y, st0.y);
    st0 = n + 1 < pl.count ? st1 : make_float2(0.0f, 0.0f);
    if (n + 2 < pl.count) st1 = *(st += pl.step);
    wait_copies<S - 1>();
    xin.take(h);
    gin.take(a);
    float2 sa = make_float2(0.0f, 0.0f), sh = sa;
#pragma unroll
    for (int p = 0; p < P; ++p) {  // past column D a is 0, and h counts nowhere
      h[p] = mul2(add2(h[p], shift), r2);
      sw[p] = fma2(a[p], h[p], sw[p]);
      sb[p] = add2(sb[p], a[p]);
      a[p] = mul2(a[p], wv[p]);
      sa = add2(sa, a[p]);
      sh = fma2(a[p], h[p], sh);
    }
    const float2 both = make_float2(sa.x + sa.y, sh.x + sh.y);
    xin.fetch();
    gin.fetch();
    commit_copies();
    if (gx) {
      const float2 s = sum(both);
      const float ma = s.x * inv_d, mh = s.y * inv_d;
      const float2 ma2 = make_float2(-ma, -ma), mh2 = make_float2(-mh, -mh);
#pragma unroll
      for (int p = 0; p < P; ++p) a[p] = mul2(r2, fma2(h[p], mh2, add2(a[p], ma2)));
      Pairs<XDT, VEC, NV>::store(gx + at, col, here ? D : 0, a);
    }
  }
  wait_copies<0>();
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * D;
  const int groups = (blockDim.x >> 5) / wpr * (32 / lpr);
  float* cols = groups > 1 ? reinterpret_cast<float*>(ring) + (int64_t)pl.group * 2 * D : out;
  __syncthreads();  // nobody reads rows from the ring any more
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int c = pair_col<VEC>(col, p, hi);
      if (c < D) {
        cols[c] = hi ? sw[p].y : sw[p].x;
        cols[D + c] = hi ? sb[p].y : sb[p].x;
      }
    }
  if (groups == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) {
    float s = 0.0f;
    for (int k = 0; k < groups; ++k) s += reinterpret_cast<float*>(ring)[k * 2 * D + c];
    out[c] = s;
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

// VEC = 4 or 1 elements of a type known at run time (aligned to themselves)
template <int VEC>
__device__ __forceinline__ void ld_long(const void* p, int dt, int64_t i, float (&v)[VEC]) {
  if (dt == SPK_F32) Vec<SPK_F32, VEC>::load(reinterpret_cast<const float*>(p) + i, v);
  else if (dt == SPK_F16) Vec<SPK_F16, VEC>::load(reinterpret_cast<const __half*>(p) + i, v);
  else Vec<SPK_BF16, VEC>::load(reinterpret_cast<const __nv_bfloat16*>(p) + i, v);
}
template <int VEC>
__device__ __forceinline__ void st_long(void* p, int dt, int64_t i, const float (&v)[VEC]) {
  if (dt == SPK_F32) Vec<SPK_F32, VEC>::store(reinterpret_cast<float*>(p) + i, v);
  else if (dt == SPK_F16) Vec<SPK_F16, VEC>::store(reinterpret_cast<__half*>(p) + i, v);
  else Vec<SPK_BF16, VEC>::store(reinterpret_cast<__nv_bfloat16*>(p) + i, v);
}

// 1024 x 20000 bf16: 51 us (74 us by single elements); the backward 119 us (242).
template <int VEC>
__global__ void __launch_bounds__(kLong) long_fwd_kernel(const void* x, int xdt, int64_t ld, const void* w, int wdt,
                                                         const void* b, int bdt, float eps, int64_t rows, int D,
                                                         void* y, int ydt, float2* stats) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    float v[VEC], s = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x * VEC; i < D; i += kLong * VEC) {
      ld_long<VEC>(x, xdt, r * ld + i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[j];
    }
    const float mean = block_sum(s) / (float)D;
    float q = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x * VEC; i < D; i += kLong * VEC) {
      ld_long<VEC>(x, xdt, r * ld + i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) q = fmaf(v[j] - mean, v[j] - mean, q);
    }
    const float rstd = 1.0f / sqrtf(block_sum(q) / (float)D + eps);
#pragma unroll 2
    for (int i = threadIdx.x * VEC; i < D; i += kLong * VEC) {
      ld_long<VEC>(x, xdt, r * ld + i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        v[j] = fmaf((v[j] - mean) * rstd, w ? ld_any(w, wdt, i + j) : 1.0f, b ? ld_any(b, bdt, i + j) : 0.0f);
      st_long<VEC>(y, ydt, r * D + i, v);
    }
    if (stats && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
  }
}

template <int VEC>
__global__ void __launch_bounds__(kLong) long_bwd_x_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                           const float2* stats, const void* w, int wdt, int64_t rows,
                                                           int D, void* gx) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = stats[r].x, rstd = stats[r].y;
    float v[VEC], a[VEC], sa = 0.0f, sh = 0.0f;
#pragma unroll 2
    for (int i = threadIdx.x * VEC; i < D; i += kLong * VEC) {
      ld_long<VEC>(g, gdt, r * D + i, a);
      ld_long<VEC>(x, xdt, r * ld + i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float t = a[j] * (w ? ld_any(w, wdt, i + j) : 1.0f);
        sa += t;
        sh = fmaf(t, (v[j] - mean) * rstd, sh);
      }
    }
    const float ma = block_sum(sa) / (float)D, mh = block_sum(sh) / (float)D;
#pragma unroll 2
    for (int i = threadIdx.x * VEC; i < D; i += kLong * VEC) {
      ld_long<VEC>(g, gdt, r * D + i, a);
      ld_long<VEC>(x, xdt, r * ld + i, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        a[j] = rstd * (a[j] * (w ? ld_any(w, wdt, i + j) : 1.0f) - ma - (v[j] - mean) * rstd * mh);
      st_long<VEC>(gx, xdt, r * D + i, a);
    }
  }
}

template <int VEC>
__global__ void __launch_bounds__(kLong) long_bwd_w_kernel(const void* g, int gdt, const void* x, int xdt, int64_t ld,
                                                           const float2* stats, int64_t rows, int D, float* part) {
  pdl_trigger();
  const int i = (blockIdx.x * kLong + threadIdx.x) * VEC;
  if (i >= D) return;
  float sw[VEC], sb[VEC], v[VEC], a[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sw[j] = sb[j] = 0.0f;
#pragma unroll 4
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    ld_long<VEC>(g, gdt, r * D + i, a);
    ld_long<VEC>(x, xdt, r * ld + i, v);
    const float2 st = stats[r];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sw[j] = fmaf(a[j], (v[j] - st.x) * st.y, sw[j]);
      sb[j] += a[j];
    }
  }
  float* to = part + (int64_t)blockIdx.y * 2 * D + i;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    to[j] = sw[j];
    to[D + j] = sb[j];
  }
}

// ---------------------------------------------------------------- which kernel, how many blocks

// Vectors (single elements) that a lane holds at most, forward and backward: the
// more, the fewer warps meet for a row (65536 x 1536 bf16 forward: 80 us with 6
// vectors and 2 warps, 94 us with 3 and 4; 65536 x 1024: 57 us with 8 and one
// warp, 68 us with 4 and 2; backward 80 us with 4 and 2, 107 us with 2 and 4).
// The `Last` number where 16 warps are needed.
constexpr int kNvFwd = 8, kNvFwdLast = 6, kNvBwd = 4, kNvBwdLast = 4;
constexpr int kNv1Fwd = 12, kNv1FwdLast = 24, kNv1Bwd = 10, kNv1BwdLast = 16;

struct Shape {
  int vec, nv, wpr, lpr = 32;  // nv = 0: the row does not fit the registers
  Shape(int64_t D, bool wide, int most4, int last4, int most1, int last1) {
    vec = wide ? 4 : 1;
    const int most = wide ? most4 : most1;
    const int64_t vecs = (D + vec - 1) / vec;
    for (wpr = 1; wpr < kMaxGroup && vecs > 32ll * wpr * most; wpr *= 2) {}
    const int64_t n = (vecs + 32 * wpr - 1) / (32 * wpr);
    nv = n > (wide ? (wpr > kWarps ? last4 : most4) : last1) ? 0 : (int)n;
    if (wide && vecs <= 16) lpr = vecs <= 8 ? 8 : 16;
  }
  int threads() const { return 32 * (wpr > kWarps ? wpr : kWarps); }
  int groups() const { return wpr > kWarps ? 1 : kWarps / wpr * (32 / lpr); }
};

// Blocks an SM that leave column sums to be joined, and parts of a long row's columns.
// Backward with 1 / 2 / 3 / 4 blocks: 65536 x 1536 bf16 160 / 119 / 119 / 119 us, 65536 x 64
// 27 / 21 / 19 / 19, 16384 x 512 fp32 29 in all.  With 16 / 64 / 256 parts: 1024 x 20000 bf16
// 145 / 119 / 123, 4096 x 16384 473 / 356 / 322, 64 x 20000 37 / 41 / 41.
constexpr int kBwdPerSm = 3, kLongChunks = 64;

// Blocks of a kernel that walks over the rows: what the machine holds at once.
// The answer for the last (device, threads, shared memory) is kept: asking takes
// as long as a launch.
struct Resident {
  int dev = -1, threads = 0, per_sm = 1;
  size_t smem = 0;
};
template <typename K>
unsigned blocks_of(K kernel, Resident& last, int64_t rows, const Shape& s, size_t smem, int most) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (last.dev != dev || last.threads != s.threads() || last.smem != smem) {
    int per_sm = 1;
    // 48 KB without asking, the kernel's static arrays included; the same limit in every call,
    // since another thread may be asking for another size
    if (smem > (40u << 10)) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 << 10);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, s.threads(), smem) != cudaSuccess || per_sm < 1)
      per_sm = 1;
    last.dev = dev;
    last.threads = s.threads();
    last.smem = smem;
    last.per_sm = per_sm;
  }
  const int64_t per_sm = last.per_sm > most ? most : last.per_sm;
  const int64_t need = (rows + s.groups() - 1) / s.groups(), cap = (int64_t)num_sms() * per_sm;
  return (unsigned)(need < cap ? need : cap);
}

// parts of the backward's column sums, whatever its kernel
inline int64_t max_parts(int64_t rows) {
  const int64_t cap = (int64_t)num_sms() * kBwdPerSm;
  return rows < cap ? rows : cap > kLongChunks ? cap : kLongChunks;
}

template <int XDT, int VEC, int NV>
void launch_fwd(const void* x, int64_t ld, const void* w, int wdt, const void* b, int bdt, float eps, int64_t rows,
                int64_t D, const Shape& s, void* y, int ydt, float* stats, cudaStream_t st) {
  const size_t smem = (size_t)Fwd<XDT, VEC, NV>::X::kBytes * s.threads();
  static thread_local Resident last;
  const unsigned blocks = blocks_of(fwd_kernel<XDT, VEC, NV>, last, rows, s, smem, 8);
  fwd_kernel<XDT, VEC, NV><<<blocks, s.threads(), smem, st>>>(reinterpret_cast<const typename Elem<XDT>::T*>(x), ld, w,
                                                             wdt, b, bdt, eps, rows, (int)D, s.wpr, s.lpr, y, ydt,
                                                             reinterpret_cast<float2*>(stats));
}

template <int GDT, int XDT, int VEC, int NV>
int launch_bwd(const void* g, const void* x, int64_t ld, const float* stats, const void* w, int wdt, int64_t rows,
               int64_t D, const Shape& s, void* gx, float* part, cudaStream_t st) {
  using T = Bwd<GDT, XDT, VEC, NV>;
  size_t smem = (size_t)(T::X::kBytes + T::G::kBytes) * s.threads();
  const size_t sums = part && s.groups() > 1 ? (size_t)s.groups() * 2 * D * sizeof(float) : 0;
  if (sums > smem) smem = sums;
  static thread_local Resident last;
  const unsigned blocks = blocks_of(bwd_kernel<GDT, XDT, VEC, NV>, last, rows, s, smem, kBwdPerSm);
  bwd_kernel<GDT, XDT, VEC, NV><<<blocks, s.threads(), smem, st>>>(
      reinterpret_cast<const typename Elem<GDT>::T*>(g), reinterpret_cast<const typename Elem<XDT>::T*>(x), ld,
      reinterpret_cast<const float2*>(stats), w, wdt, rows, (int)D, s.wpr, s.lpr,
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
      case 5:
      case 6: return GO(4, 6);
      default: return GO(4, 8);
    }
  }
  return s.nv <= 4 ? GO(1, 4) : s.nv <= 6 ? GO(1, 6) : s.nv <= 10 ? GO(1, 10) : s.nv <= 12 ? GO(1, 12) : GO(1, 24);
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
  return s.nv <= 4 ? GO(1, 4) : s.nv <= 6 ? GO(1, 6) : s.nv <= 10 ? GO(1, 10) : GO(1, 16);
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
  const Shape s(D, wide, kNvFwd, kNvFwdLast, kNv1Fwd, kNv1FwdLast);
  auto go = x_dtype == SPK_F32 ? dispatch_fwd<SPK_F32> : x_dtype == SPK_F16 ? dispatch_fwd<SPK_F16> : dispatch_fwd<SPK_BF16>;
  if (!go(x, ld, w, w_dtype, b, b_dtype, eps, rows, D, s, y, y_dtype, stats, st)) {
    const int64_t cap = (int64_t)num_sms() * 4;
    auto kernel = wide ? long_fwd_kernel<4> : long_fwd_kernel<1>;
    kernel<<<(unsigned)(rows < cap ? rows : cap), kLong, 0, st>>>(x, x_dtype, ld, w, w_dtype, b, b_dtype, eps, rows,
                                                                 (int)D, y, y_dtype, reinterpret_cast<float2*>(stats));
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
  const Shape s(D, wide, kNvBwd, kNvBwdLast, kNv1Bwd, kNv1BwdLast);
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
    auto of_x = wide ? long_bwd_x_kernel<4> : long_bwd_x_kernel<1>;
    auto of_w = wide ? long_bwd_w_kernel<4> : long_bwd_w_kernel<1>;
    if (gx)
      of_x<<<(unsigned)(rows < cap ? rows : cap), kLong, 0, st>>>(g, g_dtype, x, x_dtype, ld, sv, w, w_dtype, rows,
                                                                 (int)D, gx);
    parts = (int)(rows < kLongChunks ? rows : kLongChunks);
    if (part)
      of_w<<<dim3((unsigned)((D + kLong * s.vec - 1) / (kLong * s.vec)), (unsigned)parts), kLong, 0, st>>>(
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
