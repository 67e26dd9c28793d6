// Scaled token embedding and its gradient.
//
//   out[i] = scale * W[tok[i]]                     (rounded once)
//   g_W[v] = scale * sum over i with tok[i] = v, in ascending i, of g[i]
//
// Tokens outside [0, V) read as a row of zeros, take no gradient and raise the
// caller's flag, and a second one that no call clears (a word of the host's memory,
// so that the host can look at it without waiting).
//
// The gradient needs the positions sorted by token (stable, radix).  One cluster
// of blocks does that; a forward whose gradient will be wanted launches it just
// before the gather, which runs beside it, so that the sort costs little.  The
// gradient itself is two launches, without atomics, so equal inputs give equal
// bits:
//   sum     a warp adds the rows of g of one chunk of the sorted positions, a
//           tile of columns at a time.  A token whose positions all lie in the
//           chunk is written out; a token that reaches over the chunk's ends
//           leaves its part in a workspace.  Further blocks write zeros to the
//           rows of tokens that do not occur.
//   join    adds the parts of the tokens that reach over chunks, in order.
// A chunk costs the same whatever its tokens are, so a token that fills half the
// batch (padding, a space) is spread over the machine like any other.
#include <atomic>
#include <cstdlib>

#include "vec.cuh"

namespace spk {
namespace embg {

// ---------------------------------------------------------------- forward

// rows that a warp has in flight
constexpr int kDeep = 8;

// Columns of a lane in a tile: one vector, or kSingle single elements 32 apart.
constexpr int kSingle = 4;
constexpr int cols_of(int vec) { return vec > 1 ? vec : kSingle; }
template <int VEC>
struct Columns {
  static constexpr int N = cols_of(VEC);
  int base, D;
  __device__ __forceinline__ Columns(int64_t tile, int lane, int d)
      : base((int)tile * 32 * N + lane * (VEC > 1 ? VEC : 1)), D(d) {}
  __device__ __forceinline__ int at(int i) const { return VEC > 1 ? base + i : base + 32 * i; }
  __device__ __forceinline__ bool any() const { return base < D; }
  __device__ __forceinline__ bool on(int i) const { return VEC > 1 ? base < D : at(i) < D; }
};
// a lane's values of a row as they lie in memory
template <int DT, int VEC>
struct Raw {
  using E = typename Elem<DT>::T;
  using C = Columns<VEC>;
  typename Vec<DT, VEC>::W w[VEC > 1 ? 1 : kSingle];
  __device__ __forceinline__ void load(const E* row, const C& c) {
    if constexpr (VEC > 1) {
      w[0] = Vec<DT, VEC>::raw(row + c.base);
    } else {
#pragma unroll
      for (int i = 0; i < kSingle; ++i)
        if (c.on(i)) w[i] = Vec<DT, 1>::raw(row + c.at(i));
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[C::N]) const {
    if constexpr (VEC > 1) {
      Vec<DT, VEC>::unpack(w[0], v);
    } else {
#pragma unroll
      for (int i = 0; i < kSingle; ++i) {
        float one[1];
        Vec<DT, 1>::unpack(w[i], one);
        v[i] = one[0];
      }
    }
  }
  __device__ __forceinline__ static void store(E* row, const C& c, const float (&v)[C::N]) {
    if constexpr (VEC > 1) {
      Vec<DT, VEC>::store(row + c.base, v);
    } else {
#pragma unroll
      for (int i = 0; i < kSingle; ++i)
        if (c.on(i)) row[c.at(i)] = Elem<DT>::make(v[i]);
    }
  }
};

// A warp per (kDeep tokens, tile of columns): the tokens are read together, then
// their rows, then written.  Bound by HBM: 131072 tokens of a long-tailed
// distribution over 65536 rows of 1024 bf16 (348 MB) take 63 us, 5.5 TB/s.
template <int WDT, int ODT, int VEC>
__global__ void __launch_bounds__(256, 4) gather_kernel(const int64_t* __restrict__ tokens,
                                                     const typename Elem<WDT>::T* __restrict__ w, int64_t ldw,
                                                     float scale, int64_t n, int64_t V, int D, int tiles,
                                                     typename Elem<ODT>::T* __restrict__ out, int* bad, int* ever,
                                                     int extra, int scan_bad, int after_sort) {
  if (extra && blockIdx.x == 0) {  // the first block, so that it is not the last to end
    if (scan_bad && scan_tokens(tokens, n, V, 0, bad) && ever && threadIdx.x == 0) *ever = 1;
    // The sort before this kernel may still be running: this block does not end before it, so
    // whoever comes after this kernel finds the sort done.
    if (after_sort) pdl_wait();
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t item = ((int64_t)blockIdx.x - extra) * 8 + (threadIdx.x >> 5);
  const int64_t group = item / tiles;
  const Columns<VEC> col(item - group * tiles, lane, D);
  const int64_t i0 = group * kDeep;
  if (i0 >= n) return;
  int64_t tok = -1;
  if (lane < kDeep && i0 + lane < n) {
    tok = __ldg(tokens + i0 + lane);
    if (tok < 0 || tok >= V) {
      tok = -1;
      if (!scan_bad) {
        atomicExch(bad, 1);
        if (ever) *reinterpret_cast<volatile int*>(ever) = 1;
      }
    }
  }
  Raw<WDT, VEC> x[kDeep];
  unsigned in = 0;  // rows that are inside the vocabulary
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    const int64_t t = __shfl_sync(0xffffffffu, tok, k);
    if (t >= 0 && col.any()) {
      in |= 1u << k;
      x[k].load(w + t * ldw, col);
    }
  }
  if (!col.any()) return;
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    if (i0 + k >= n) break;
    float v[Columns<VEC>::N];
    x[k].unpack(v);
#pragma unroll
    for (int j = 0; j < Columns<VEC>::N; ++j) v[j] = (in >> k) & 1u ? v[j] * scale : 0.0f;
    Raw<ODT, VEC>::store(out + (i0 + k) * D, col, v);
  }
}

// ---------------------------------------------------------------- backward: sort

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigit = 10;
constexpr int kBatch = 8;  // items of a lane that are loaded together

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

// Lanes whose digit equals the caller's: one vote a bit (the sort of 131072 keys of
// 17 bits takes 43 us so, 50 us with a match instruction).
__device__ __forceinline__ uint32_t same_digit(uint32_t d, int bits, bool in) {
  uint32_t same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < kMaxDigit; ++b) {
    if (b >= bits) break;
    const bool one = (d >> b) & 1u;
    const uint32_t v = __ballot_sync(0xffffffffu, one);
    same &= one ? v : ~v;
  }
  return same;
}

// One cluster.  A pass of the radix sort over a digit of `bits` bits: every warp
// owns a run of consecutive positions and counts its digits; the counts are
// summed over the warps of a block, over the blocks of the cluster and over the
// digits, which gives every (warp, digit) its place; the warp then writes its
// items there in order.  Positions without a gradient get the key V and end up
// last.  131072 tokens of 17 bits: 43 us, much of it the scattered writes.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const int64_t* tokens, int64_t n, int64_t V,
                                                            int64_t padding_idx, int bits, int passes, uint2* item0,
                                                            uint2* item1) {
  extern __shared__ uint32_t sm[];
  pdl_trigger();
  const uint32_t ncta = cluster_size(), rank = cluster_ctarank();
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
    const uint2* in_items = (p & 1) ? item0 : item1;
    uint2* out_items = (p & 1) ? item1 : item0;
    const int shift = p * bits;
    auto item_at = [&](int64_t i) -> uint2 {  // (key, position)
      if (p > 0) return __ldcg(in_items + i);
      const int64_t t = __ldg(tokens + i);
      return make_uint2(t >= 0 && t < V && t != padding_idx ? (uint32_t)t : (uint32_t)V, (uint32_t)i);
    };
    for (int i = lane; i < bins; i += 32) mine[i] = 0;
    __syncwarp();
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * kBatch) {
      uint32_t k[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) k[b] = i0 + b * 32 + lane < hi ? item_at(i0 + b * 32 + lane).x : 0u;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (i0 + b * 32 >= hi) break;
        const bool in = i0 + b * 32 + lane < hi;
        const uint32_t d = (k[b] >> shift) & (bins - 1);
        const uint32_t same = same_digit(d, bits, in);
        if (in && (same >> lane) == 1u) mine[d] += __popc(same);  // the highest lane of its digit
        __syncwarp();
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
      uint32_t c[kSortWarps], s = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c[w] = count[w * bins + d];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        count[w * bins + d] = s;
        s += c[w];
      }
      total[d] = s;
    }
    cluster_sync_all();
    // bins <= threads: one digit a thread; an exclusive sum over the digits of the cluster's counts
    const int d = threadIdx.x;
    uint32_t all = 0, before = 0;
    if (d < bins) {
#pragma unroll 8
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
    uint32_t off = lane < warp ? wsum[lane] : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) off += __shfl_xor_sync(0xffffffffu, off, o);
    if (d < bins) base[d] = off + inc - all + before;
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * kBatch) {
      uint2 k[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        k[b] = i0 + b * 32 + lane < hi ? item_at(i0 + b * 32 + lane) : make_uint2(0u, 0u);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (i0 + b * 32 >= hi) break;
        const bool in = i0 + b * 32 + lane < hi;
        const uint32_t dd = (k[b].x >> shift) & (bins - 1);
        const uint32_t same = same_digit(dd, bits, in);
        uint32_t at = 0;
        if (in) at = base[dd] + mine[dd] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (in) {
          out_items[at] = k[b];
          if ((same >> lane) == 1u) mine[dd] += __popc(same);
        }
        __syncwarp();
      }
    }
    cluster_sync_all();  // the items are written and nobody reads `total` any more
  }
}

// ---------------------------------------------------------------- backward: sum and join

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes_is_16) {
  if (bytes_is_16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// zeros to those of 32 rows whose token does not occur (a search of the sorted keys a lane)
template <int WDT, int VEC>
__device__ __forceinline__ void clear_rows(const uint2* __restrict__ items, int64_t n, uint32_t V, int D, int64_t group,
                                           int lane, typename Elem<WDT>::T* __restrict__ gw) {
  const int64_t row = group * 32 + lane;
  int64_t a = 0, b = n;  // the first item with a key of at least `row`
  while (a < b) {
    const int64_t mid = (a + b) / 2;
    if (items[mid].x < row) a = mid + 1;
    else b = mid;
  }
  uint32_t absent = __ballot_sync(0xffffffffu, row < V && (a >= n || items[a].x != row));
  float zero[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) zero[i] = 0.0f;
  for (; absent; absent &= absent - 1) {
    typename Elem<WDT>::T* to = gw + (group * 32 + __ffs(absent) - 1) * D;
    for (int c = lane * VEC; c < D; c += 32 * VEC) Vec<WDT, VEC>::store(to + c, zero);
  }
}

// A warp per (chunk of sorted positions, tile of columns).  With
// VEC > 1 a lane's vectors of the next kRing rows are on their way into a
// ring of its own in shared memory (a lane reads back only what it copied
// itself, so the ring needs no barrier); single elements, which asynchronous
// copies cannot move in two bytes, go through registers.  Bound by HBM: the
// 131072 rows of 1024 bf16 and the 65536 rows of the gradient (403 MB with the
// zeros) take 70 us; with rows in registers instead of the ring 103 us.
constexpr int kRing = 16;
constexpr int kStep = 4;  // rows of one copy group

template <int GDT, int WDT, int VEC>
__global__ void __launch_bounds__(256) sum_kernel(const uint2* __restrict__ items,
                                                  const typename Elem<GDT>::T* __restrict__ g, float scale, int64_t n,
                                                  uint32_t V, int D, int chunk, int tiles, int64_t chunks,
                                                  int64_t sum_blocks, typename Elem<WDT>::T* __restrict__ gw,
                                                  float* __restrict__ part) {
  using W = typename Vec<GDT, VEC>::W;
  extern __shared__ uint4 ring_mem[];
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  if (blockIdx.x >= sum_blocks) {
    clear_rows<WDT, VEC>(items, n, V, D, ((int64_t)blockIdx.x - sum_blocks) * 8 + (threadIdx.x >> 5), lane, gw);
    return;
  }
  const int64_t item = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
  if (item >= chunks * tiles) return;
  const int64_t c = item / tiles;
  constexpr int N = Columns<VEC>::N;
  const Columns<VEC> col(item - c * tiles, lane, D);
  const bool on = col.any();
  const int64_t lo = c * chunk, hi = lo + chunk < n ? lo + chunk : n;
  const int m = (int)(hi - lo);
  const uint32_t before = lo > 0 ? items[lo - 1].x : 0xffffffffu;
  const uint32_t after = hi < n ? items[hi].x : 0xffffffffu;
  uint32_t cur = items[lo].x;
  bool first = true;  // the chunk's first token is being added
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.0f;
  // the sum so far belongs to token `cur`: to the gradient, or to the parts
  auto flush = [&](bool last) {
    if (cur >= V || !on) return;
    const bool head = first && cur == before;
    const bool tail = last && cur == after;
    if (head || tail) {
      // [chunk][0]: the part of a token that comes from the chunk before (and may go on),
      // [chunk][1]: of one that begins here and goes on
      float* q = part + (c * 2 + (head ? 0 : 1)) * D;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (col.on(j)) q[col.at(j)] = acc[j];
    } else {
      float v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = acc[j] * scale;
      Raw<WDT, VEC>::store(gw + (int64_t)cur * D, col, v);
    }
  };
  auto take = [&](uint32_t k, const Raw<GDT, VEC>& x) {
    if (k != cur) {
      flush(false);
      cur = k;
      first = false;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.0f;
    }
    if (k < V) {
      float v[N];
      x.unpack(v);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[i];
    }
  };
  // the items of the group of 32 that is added, and of the next one
  auto group_of = [&](int j) { return j + lane < m ? items[lo + j + lane] : make_uint2(0xffffffffu, 0u); };
  uint2 a = group_of(0);
  if constexpr (VEC > 1) {
    uint2 b = group_of(32);
    W* ring = reinterpret_cast<W*>(ring_mem) + (threadIdx.x >> 5) * kRing * 32 + lane;
    const uint32_t ring_at = smem_u32(ring);
    auto issue = [&](int j) {  // rows [j, j + kStep), at most 32 + the group of `a` away
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int r = (j + i) & 31;
        const bool in_b = ((j + i) >> 5) != 0;
        const uint32_t k = __shfl_sync(0xffffffffu, in_b ? b.x : a.x, r);
        const uint32_t q = __shfl_sync(0xffffffffu, in_b ? b.y : a.y, r);
        if (on && k < V)
          copy_async(ring_at + ((j + i) & (kRing - 1)) * 32 * (int)sizeof(W), g + (int64_t)q * D + col.base,
                     sizeof(W) == 16);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int j = 0; j < kRing; j += kStep) issue(j);
    for (int j0 = 0; j0 < m; j0 += 32) {
#pragma unroll
      for (int j = 0; j < 32; j += kStep) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing / kStep - 1) : "memory");
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const uint32_t k = __shfl_sync(0xffffffffu, a.x, j + i);
          if (j0 + j + i < m) {
            Raw<GDT, VEC> x;
            x.w[0] = ring[((j + i) & (kRing - 1)) * 32];
            take(k, x);
          }
        }
        issue(j + kRing);
      }
      a = b;
      b = group_of(j0 + 64);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    for (int j0 = 0; j0 < m; j0 += 32) {
      for (int j = 0; j < 32 && j0 + j < m; j += kDeep) {
        Raw<GDT, VEC> x[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
          const uint32_t k = __shfl_sync(0xffffffffu, a.x, j + i), q = __shfl_sync(0xffffffffu, a.y, j + i);
          if (on && k < V) x[i].load(g + (int64_t)q * D, col);
        }
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
          const uint32_t k = __shfl_sync(0xffffffffu, a.x, j + i);
          if (j0 + j + i < m) take(k, x[i]);
        }
      }
      a = group_of(j0 + 32);
    }
  }
  flush(true);
}

// A block per chunk: where the chunk's last token begins in it and goes on, adds
// the token's parts.  Few parts: a thread adds them, four columns each.  Many:
// they are cut into one run a warp, and the warps' sums are added in order.  The
// border does not matter much: with 4 / 16 / 64 parts the gradient of 131072 tokens takes
// 133 / 133 / 131 us (V 65536, D 1024 bf16), 119 in all (one token, D 1024 bf16) and 98 /
// 98 / 96 (V 256, D 384 fp32), that of 20000 tokens of D 512 41 / 41 / 43.
constexpr int kFewParts = 16;

template <int WDT, int VEC>
__global__ void __launch_bounds__(256) join_kernel(const uint2* __restrict__ items, float scale, int64_t n, uint32_t V,
                                                   int D, int chunk, int64_t chunks,
                                                   typename Elem<WDT>::T* __restrict__ gw,
                                                   const float* __restrict__ part) {
  __shared__ float red[8][32 * VEC];
  pdl_wait();
  const int64_t c = blockIdx.x;
  const int64_t lo = c * chunk, hi = lo + chunk;
  const uint32_t k = items[hi - 1].x;
  if (k >= V || items[hi].x != k) return;                      // nothing goes on
  if (lo > 0 && items[lo].x == k && items[lo - 1].x == k) return;  // it began before
  int64_t a = c + 1, step = 1;  // chunks (c, a) begin with k: doubling steps, then halving ones
  while (a + step < chunks && items[(a + step) * chunk].x == k) {
    a += step;
    step *= 2;
  }
  for (; step > 0; step /= 2)
    if (a + step < chunks && items[(a + step) * chunk].x == k) a += step;
  const int64_t m = a + 1 - c;  // parts: [c][1], [c + 1][0], ..., [a][0]
  const float* first = part + (c * 2 + 1) * D;
  const float* rest = part + c * 2 * D;  // part p > 0 at rest + 2 p D
  auto add = [&](int64_t p0, int64_t p1, int col, float (&s)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = 0.0f;
#pragma unroll 8
    for (int64_t p = p0; p < p1; ++p) {
      float v[VEC];
      Vec<SPK_F32, VEC>::load((p == 0 ? first : rest + 2 * p * D) + col, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += v[j];
    }
  };
  auto put = [&](int col, float (&s)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] *= scale;
    Vec<WDT, VEC>::store(gw + (int64_t)k * D + col, s);
  };
  float s[VEC];
  if (m <= kFewParts) {
    for (int col = (blockIdx.y * 256 + threadIdx.x) * VEC; col < D; col += gridDim.y * 256 * VEC) {
      add(0, m, col, s);
      put(col, s);
    }
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int col0 = blockIdx.y * 32 * VEC; col0 < D; col0 += gridDim.y * 32 * VEC) {
    const int col = col0 + lane * VEC;
    if (col < D) {
      add(m * warp / 8, m * (warp + 1) / 8, col, s);
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[warp][lane * VEC + j] = s[j];
    }
    __syncthreads();
    if (warp == 0 && col < D) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s[j] = 0.0f;
        for (int w = 0; w < 8; ++w) s[j] += red[w][lane * VEC + j];
      }
      put(col, s);
    }
    __syncthreads();
  }
}

inline int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

// Chunks: one for every warp that the machine holds (24 an SM) where there are
// positions enough, of 16 to 1024 positions.  The gradient with 12 / 24 / 48 warps an
// SM, us: 131072 tokens, V 65536, D 1024 bf16 145 / 135 / 150; one token 131072 times
// 113 / 121 / 186; V 256, D 384 fp32 88 / 98 / 113; 4096 tokens alike.  Chunks of at
// most 256 / 1024 / 4096: 2^20 tokens of D 128 397 / 381 / 381, fewer tokens alike.
struct Plan {
  int bits, passes, chunk, tiles;
  int64_t chunks, items;  // items: bytes of one of the two arrays of (key, position)
  Plan(int64_t n, int64_t V, int64_t D, int cols) {  // cols: columns of a lane in a tile
    int b = 1;
    while ((V >> b) != 0) ++b;  // keys 0 .. V
    passes = (b + kMaxDigit - 1) / kMaxDigit;
    bits = (b + passes - 1) / passes;
    tiles = (int)((D + 32 * cols - 1) / (32 * cols));
    const int64_t warps = (int64_t)num_sms() * 24;
    int64_t ch = ((n * tiles + warps - 1) / warps + 15) / 16 * 16;
    chunk = (int)(ch < 16 ? 16 : ch > 1024 ? 1024 : ch);
    chunks = (n + chunk - 1) / chunk;
    items = align16(8 * n);
  }
};

template <int GDT, int WDT, int VEC>
int launch_bwd(const Plan& pl, const uint2* items, const void* g, float scale, int64_t n, int64_t V, int D, void* gw,
               float* part, cudaStream_t st) {
  auto* out = reinterpret_cast<typename Elem<WDT>::T*>(gw);
  const int64_t blocks = (pl.chunks * pl.tiles + 7) / 8;
  const int smem = VEC > 1 ? 8 * kRing * 32 * (int)sizeof(typename Vec<GDT, VEC>::W) : 0;
  if (smem > 48 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(sum_kernel<GDT, WDT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               smem);
    if (e != cudaSuccess) return fail(SPK_ERR_LAUNCH, "embedding_bwd: %s", cudaGetErrorString(e));
  }
  const int64_t clear = (V + 255) / 256;  // 32 rows a warp
  sum_kernel<GDT, WDT, VEC><<<(unsigned)(blocks + clear), 256, smem, st>>>(
      items, reinterpret_cast<const typename Elem<GDT>::T*>(g), scale, n, (uint32_t)V, D, pl.chunk, pl.tiles, pl.chunks,
      blocks, out, part);
  if (pl.chunks > 1) {
    cudaLaunchConfig_t cfg = {};
    // a few blocks a chunk: a token of many parts has its columns spread over them (1 / 4 blocks,
    // the gradient of one token 131072 times, D 1024: 199 / 121 us; 20000 tokens, D 512 49 / 43;
    // D 384 98 / 90 with 131072 tokens, 29 / 31 with 4096; D 128 379 / 393 with 2^20)
    cfg.gridDim = dim3((unsigned)(pl.chunks - 1), D >= 512 ? 4 : 1);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    add_pdl_attr(cfg, at);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<WDT, VEC == 1 ? 1 : 4>, items, scale, n, (uint32_t)V, D,
                                             pl.chunk, pl.chunks, out, (const float*)part);
    if (e != cudaSuccess) return fail(SPK_ERR_LAUNCH, "embedding_bwd: %s", cudaGetErrorString(e));
  }
  return check_launch("embedding_bwd");
}

// elements of an access: 16 bytes of the wider type where the layout allows, else one
inline int bwd_vec(const void* g, int g_dtype, const void* gw, int w_dtype, int64_t D) {
  const int v = g_dtype == SPK_F32 || w_dtype == SPK_F32 ? 4 : 8;
  return D % v == 0 && aligned(g, v * dtype_size(g_dtype)) && aligned(gw, v * dtype_size(w_dtype)) ? v : 1;
}

// The most blocks of a cluster of the sort that the current device can hold: 16 (not
// portable) where a partition or another program's claim leaves room for them, else 8.
// Asked once a device.  SPK_SORT_CLUSTER=8 leaves the 16 out (for tests).
inline int largest_cluster() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
  int most = known[dev].load(std::memory_order_relaxed);
  if (most) return most;
  const char* env = getenv("SPK_SORT_CLUSTER");
  most = env && atoi(env) == 8 ? 8 : 16;
  if (most == 16) {
    constexpr int kSmem = ((kSortWarps + 2) << kMaxDigit) * 4;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {16, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
        cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, (const void*)sort_kernel, &cfg) != cudaSuccess || clusters < 1) {
      cudaGetLastError();  // the answer is no, and no error of the call's
      most = 8;
    }
  }
  known[dev].store(most, std::memory_order_relaxed);
  return most;
}

// The items in order: in plan, or in plan + its second half.
int launch_sort(const Plan& pl, const int64_t* tokens, int64_t n, int64_t V, int64_t padding_idx, void* plan,
                cudaStream_t st) {
  uint2* item0 = reinterpret_cast<uint2*>(plan);
  uint2* item1 = reinterpret_cast<uint2*>(reinterpret_cast<char*>(plan) + pl.items);
  // Lookup and gradient of n tokens, V 256, D 384 fp32, us with 1 / 8 / 16 blocks: 256 tokens
  // 19 / 21 / 23, 2048 25 / 25 / 25, 4096 29 / 25 / 27, 16384 58 / 35 / 33, 32768 92 / 43 / 39,
  // 131072 311 / 115 / 98; V 65536, D 32: 256 25 / 27 / 27, 4096 41 / 31 / 33, 32768 145 / 51 / 45.
  const int csize = n <= 4096 ? 1 : n <= 32768 ? 8 : largest_cluster();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)csize);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = (size_t)((kSortWarps + 2) << pl.bits) * 4;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)csize, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaSuccess;
  if (cfg.dynamicSmemBytes > (40u << 10))  // the most of any call: another thread may be setting it too
    e = cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)((kSortWarps + 2) << kMaxDigit) * 4);
  if (e == cudaSuccess && csize > 8) e = cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaLaunchKernelEx(&cfg, sort_kernel, tokens, n, V, padding_idx, pl.bits, pl.passes, item0, item1);
  return e == cudaSuccess ? SPK_OK : fail(SPK_ERR_LAUNCH, "embedding sort: %s", cudaGetErrorString(e));
}
inline const uint2* sorted_items(const Plan& pl, const void* plan) {
  return reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(plan) + (pl.passes & 1 ? 0 : pl.items));
}

template <int WDT, int ODT>
int launch_gather(const int64_t* tokens, const void* w, int64_t ldw, float scale, int64_t n, int64_t V, int D,
                  void* out, int* bad, int* ever, bool after_sort, cudaStream_t st) {
  constexpr int kWide = WDT == SPK_F32 || ODT == SPK_F32 ? 4 : 8;
  const bool wide = D % kWide == 0 && ldw % kWide == 0 && aligned(w, kWide * dtype_size(WDT)) &&
                    aligned(out, kWide * dtype_size(ODT));
  const int cols = 32 * cols_of(wide ? kWide : 1), tiles = (D + cols - 1) / cols;
  const int scan = n <= kScanTokens ? 1 : 0, extra = scan || after_sort ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((n + kDeep - 1) / kDeep * tiles + 7) / 8 + extra));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (after_sort) add_pdl_attr(cfg, at);  // beside the sort, whose results it does not read
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, wide ? gather_kernel<WDT, ODT, kWide> : gather_kernel<WDT, ODT, 1>, tokens,
      reinterpret_cast<const typename Elem<WDT>::T*>(w), ldw, scale, n, V, D, tiles,
      reinterpret_cast<typename Elem<ODT>::T*>(out), bad, ever, extra, scan, after_sort ? 1 : 0);
  return e == cudaSuccess ? check_launch("embedding_fwd") : fail(SPK_ERR_LAUNCH, "embedding_fwd: %s", cudaGetErrorString(e));
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

int64_t spk_embedding_plan_bytes(int64_t n) { return n < 1 ? 16 : 2 * spk::embg::align16(8 * n); }

int spk_embedding_fwd(const int64_t* tokens, const void* weight, int w_dtype, int64_t ldw, float scale, int64_t n,
                      int64_t V, int64_t D, void* out, int out_dtype, int* bad_token, int64_t padding_idx, void* plan,
                      int64_t plan_bytes, void* stream) {
  return spk_embedding_fwd_watched(tokens, weight, w_dtype, ldw, scale, n, V, D, out, out_dtype, bad_token, nullptr,
                                   padding_idx, plan, plan_bytes, stream);
}

int spk_embedding_fwd_watched(const int64_t* tokens, const void* weight, int w_dtype, int64_t ldw, float scale,
                              int64_t n, int64_t V, int64_t D, void* out, int out_dtype, int* bad_token, int* bad_ever,
                              int64_t padding_idx, void* plan, int64_t plan_bytes, void* stream) {
  using namespace spk;
  using namespace spk::embg;
  SPK_REQUIRE(tokens && weight && out && bad_token, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(w_dtype) && float_type(out_dtype), SPK_ERR_INVALID, "embedding takes fp32, fp16 and bf16");
  SPK_REQUIRE(n >= 1 && V >= 1 && D >= 1 && D <= (1 << 20) && ldw >= D && n < (1ll << 31) && V < (1ll << 31),
              SPK_ERR_SHAPE, "unsupported sizes n=%lld V=%lld D=%lld row stride %lld", (long long)n, (long long)V,
              (long long)D, (long long)ldw);
  SPK_REQUIRE(!plan || plan_bytes >= spk_embedding_plan_bytes(n), SPK_ERR_INVALID,
              "plan smaller than spk_embedding_plan_bytes()");
  SPK_REQUIRE(aligned(plan, 16) && aligned(bad_ever, 4), SPK_ERR_ALIGN,
              "plan must be 16-byte aligned, bad_ever 4-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (n > kScanTokens) cudaMemsetAsync(bad_token, 0, sizeof(int), st);
  if (plan) {
    rc = launch_sort(Plan(n, V, D, 8), tokens, n, V, padding_idx, plan, st);
    if (rc != SPK_OK) return rc;
  }
#define CALL(W, O) return launch_gather<W, O>(tokens, weight, ldw, scale, n, V, (int)D, out, bad_token, bad_ever, plan != nullptr, st)
  SPK_EMB_TYPES(w_dtype, out_dtype, CALL);
#undef CALL
}

int64_t spk_embedding_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  using namespace spk::embg;
  if (n < 1 || V < 1 || D < 1) return 16;
  const Plan pl(n, V, D, 8);  // the widest tiles make the most chunks
  return pl.chunks * 2 * D * (int64_t)sizeof(float);
}

int spk_embedding_bwd(const int64_t* tokens, const void* g, int g_dtype, float scale, int64_t padding_idx, int64_t n,
                      int64_t V, int64_t D, void* gw, int w_dtype, void* plan, int64_t plan_bytes, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  using namespace spk;
  using namespace spk::embg;
  SPK_REQUIRE(g && gw && plan, SPK_ERR_INVALID, "null pointer argument");
  SPK_REQUIRE(float_type(w_dtype) && float_type(g_dtype), SPK_ERR_INVALID, "embedding takes fp32, fp16 and bf16");
  SPK_REQUIRE(n >= 1 && V >= 1 && D >= 1 && D <= (1 << 20) && n < (1ll << 31) && V < (1ll << 31), SPK_ERR_SHAPE,
              "unsupported sizes n=%lld V=%lld D=%lld", (long long)n, (long long)V, (long long)D);
  SPK_REQUIRE(plan_bytes >= spk_embedding_plan_bytes(n), SPK_ERR_INVALID,
              "plan smaller than spk_embedding_plan_bytes()");
  SPK_REQUIRE(workspace && workspace_bytes >= spk_embedding_bwd_workspace_bytes(n, V, D), SPK_ERR_INVALID,
              "workspace smaller than spk_embedding_bwd_workspace_bytes()");
  SPK_REQUIRE(aligned(workspace, 16) && aligned(plan, 16), SPK_ERR_ALIGN, "plan and workspace must be 16-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int vec = bwd_vec(g, g_dtype, gw, w_dtype, D);
  const Plan pl(n, V, D, cols_of(vec));
  if (tokens) {
    rc = launch_sort(pl, tokens, n, V, padding_idx, plan, st);
    if (rc != SPK_OK) return rc;
  }
  const uint2* items = sorted_items(pl, plan);
  float* part = reinterpret_cast<float*>(workspace);
#define CALL(G, W)                                                                                        \
  constexpr int kWide = G == SPK_F32 || W == SPK_F32 ? 4 : 8;                                             \
  return vec == kWide ? launch_bwd<G, W, kWide>(pl, items, g, scale, n, V, (int)D, gw, part, st)          \
                      : launch_bwd<G, W, 1>(pl, items, g, scale, n, V, (int)D, gw, part, st)
  SPK_EMB_TYPES(g_dtype, w_dtype, CALL);
#undef CALL
}

}  // extern "C"
