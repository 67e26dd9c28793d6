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
// of c scales sums by a power of two.  With S = sum 2^t_j and
// A = sum t_j 2^t_j:  logp = ln 2 (t_y - log2 S),  H = ln 2 (log2 S - A / S).
// t_y and log2 S of a likely symbol are small, so logp and H near 0 are right to a
// few 2^-24 (not to so much of themselves); they are held at their side of 0.
// Where the maximum is beyond 2^20 (a row barred with the type's lowest value),
// c would be coarser than 1, so the maximum itself is taken off first:
// t_j = (z_j - off) log2 e.  t is held at -200 or above, where 2^t is 0 already,
// so that a barred symbol (z = -inf) adds 0 and not 0 * inf; the maximum passes
// a NaN on.
//
// Bound by HBM: the logits are read once in each direction, with no maximum
// known beforehand.  A thread keeps (m, S, A) of the values that it has seen
// against the reference of its own m and rescales when a tile raises it; the
// states of lanes, warps and blocks are joined in the same way.  Short rows, and
// longer ones where there are many, belong to a warp, others to a block of 8
// warps; where the rows are too few to fill the machine a row is cut over several
// blocks and a second kernel joins them.  Logits come in tiles of 16-byte vectors by
// asynchronous copies, kStages ahead, into a ring of the thread's own (no
// barrier); a stage is one step t of one tile.  A row that does not begin on 16
// bytes has its first and last values taken one by one.
#include "vec.cuh"

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
  if (m == -INFINITY) return Ref{0.0f, 0.0f};  // nothing but barred values so far
  return fabsf(m) <= kFar ? Ref{0.0f, rintf(m * kLog2e)} : Ref{m, 0.0f};
}
__device__ __forceinline__ float log2_from(float z, Ref f) { return fmaf(z - f.off, kLog2e, -f.c); }
__device__ __forceinline__ float not_below(float t) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC3480000;" : "=f"(r) : "f"(t));  // -200
  return r;
}

// The values seen so far: their maximum, S and A against ref_of(m).
struct State {
  float m, S, A;
  Ref f;
  __device__ __forceinline__ State(float max = -INFINITY, float s = 0.0f, float a = 0.0f)
      : m(max), S(s), A(a), f(ref_of(max)) {}
  __device__ __forceinline__ void move_to(float nm) {
    const Ref a = f, b = ref_of(nm);
    // never above 0; held so where there is nothing yet (m = -inf, S = A = 0)
    const float d = fminf(fmaxf((a.c - b.c) + (a.off - b.off) * kLog2e, -200.0f), 0.0f);
    const float k = m == -INFINITY ? 0.0f : exp2_approx(d);
    A = k * fmaf(d, S, A);
    S *= k;
    m = nm;
    f = b;
  }
  __device__ __forceinline__ void join_warp() {
    float nm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, o));
    if (nm > m) move_to(nm);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, o);
      A += __shfl_xor_sync(0xffffffffu, A, o);
    }
  }
};

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


// ---------------------------------------------------------------- the mean over the steps

// s + v with the rounding error of the sum added to err (two-sum)
__device__ __forceinline__ void add_exactly(float& s, float& err, float v) {
  const float n = __fadd_rn(s, v);
  const float b = __fsub_rn(n, s);
  err = __fadd_rn(err, __fadd_rn(__fsub_rn(s, __fsub_rn(n, b)), __fsub_rn(v, b)));
  s = n;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, make_float2(-1.0f, -1.0f), a); }
__device__ __forceinline__ void add_exactly(float2& s, float2& err, float2 v) {
  const float2 n = add2(s, v);
  const float2 b = sub2(n, s);
  err = add2(err, add2(sub2(s, sub2(n, b)), sub2(v, b)));
  s = n;
}

// An infinity or NaN among the steps behind the first, or steps whose sum alone is too large.
template <int DT>
__device__ __noinline__ float mean_of_extremes(const typename Elem<DT>::T* x, int64_t st, int T) {
  double d = 0.0;
  for (int t = 0; t < T; ++t) d += (double)Elem<DT>::load(x + t * st);
  return (float)(d / (double)T);
}

// (s + err) / T rounded once: the quotient's remainder takes the errors in, so
// that near ties keep the order that the exact means have.  With a T that is no
// power of two 1 / T is rounded, which may push a quotient that lies half way
// between two numbers to the odd one: the remainder of the result then is half a
// step of it, exactly, and the even neighbour is taken.
__device__ __forceinline__ bool power_of_two(int T) { return (T & (T - 1)) == 0; }
__device__ __forceinline__ float quotient(float s, float err, int T, float inv_t) {
  const float steps = (float)T, q = __fmul_rn(s, inv_t);
  float z = fmaf(__fadd_rn(fmaf(-q, steps, s), err), inv_t, q);
  if (!power_of_two(T)) {
    const float rest = __fadd_rn(fmaf(-z, steps, s), err);
    const uint32_t bits = __float_as_uint(z), exponent = bits & 0x7f800000u;
    // half a step of z, T times; 0 where a step is below the normal numbers
    const float half = exponent > (24u << 23) ? __uint_as_float(exponent - (24u << 23)) * steps : 0.0f;
    if ((bits & 1u) && fabsf(rest) == half && half > 0.0f)
      z = __uint_as_float((rest > 0.0f) == (z > 0.0f) ? bits + 1u : bits - 1u);
  }
  return z;
}

// x: the value's first step
template <int DT>
__device__ __forceinline__ float mean_of(float s, float err, const typename Elem<DT>::T* x, int64_t st, int T,
                                         float inv_t) {
  if (!(fabsf(s) < INFINITY)) {
    // a first step that is an infinity (a barred symbol) or NaN: its sum is the mean, and its
    // other steps are not read again (4 x 16384 x 256 fp32 with 30 % barred: 35 us, 59 with
    // all steps read again, 27 with none barred)
    return fabsf(Elem<DT>::load(x)) < INFINITY ? mean_of_extremes<DT>(x, st, T) : s;
  }
  return quotient(s, err, T, inv_t);
}

// z_j of one value
template <int DT>
__device__ __forceinline__ float mean_over_t(const typename Elem<DT>::T* x, int64_t st, int T, float inv_t) {
  float s = Elem<DT>::load(x);
  if (T == 1) return s;
  float err = 0.0f;
  for (int t = 1; t < T; ++t) add_exactly(s, err, Elem<DT>::load(x + t * st));
  return mean_of<DT>(s, err, x, st, T, inv_t);
}

// ---------------------------------------------------------------- tiles of a row

constexpr int kStages = 4;

struct Logits {  // element (t, r, v) at base + t st + r sr + v
  const void* base;
  int T, V;
  int64_t rows, st, sr;
  float inv_t;
};

// A tile's values as words (a 16-bit value alone is a word's lower half), and as pairs of fp32.
template <int DT>
__device__ __forceinline__ uint32_t one_word(const typename Elem<DT>::T* p) {
  if constexpr (DT == SPK_F32) return __float_as_uint(*p);
  else return *reinterpret_cast<const uint16_t*>(p);
}
template <int DT>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {  // two 16-bit values
  if constexpr (DT == SPK_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT, int VEC, int WORDS, int P>
__device__ __forceinline__ void unpack_words(const uint32_t (&w)[WORDS], float2 (&z)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if constexpr (DT == SPK_F32) z[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (VEC > 1) z[i] = unpack_pair<DT>(w[i]);
    else z[i] = make_float2(unpack_pair<DT>(w[2 * i]).x, unpack_pair<DT>(w[2 * i + 1]).x);
  }
}
// a value's bits where there is none: -inf, in both halves of a word of two
template <int DT>
__device__ __forceinline__ constexpr uint32_t no_value() {
  return DT == SPK_F32 ? 0xff800000u : DT == SPK_BF16 ? 0xff80ff80u : 0xfc00fc00u;
}

// Values [lo, hi) of a row in tiles of GT threads x U vectors of VEC; thread
// tid's vector u of a tile begins at lo + ((tile U + u) GT + tid) VEC.
template <int DT, int VEC, int U, int GT>
struct Tiles {
  using E = typename Elem<DT>::T;
  using W = typename Vec<DT, VEC>::W;
  static constexpr int N = U * VEC, kSpan = GT * U * VEC;
  static constexpr int kWords = VEC > 1 ? U * 4 : U;
  static constexpr int kBytes = VEC > 1 ? kStages * U * 16 : 0;  // of shared memory a thread
  static_assert(VEC == 1 || sizeof(W) == 16, "16-byte vectors");
  static_assert(N % 2 == 0, "pairs");
  const E* row;
  int64_t st;
  int T, lo, hi, tid;
  int ft, fj;         // the stage to fetch: step, and the thread's first value in the tile
  const E* fp;
  uint32_t ring, at;  // the thread's ring [kStages][U][256], the slot's offset
  __device__ __forceinline__ Tiles(void* smem, const E* r, int64_t step, int steps, int l, int h, int thread)
      : row(r), st(step), T(steps), lo(l), hi(h), tid(thread), ft(0), fj(l + thread * VEC), fp(r), ring(0), at(0) {
    if constexpr (VEC > 1) {
      ring = smem_u32(smem) + threadIdx.x * 16;
#pragma unroll
      for (int k = 0; k < kStages; ++k) fetch();
    }
  }
  __device__ __forceinline__ int first(int tile) const { return lo + tile * kSpan + tid * VEC; }
  __device__ __forceinline__ void fetch() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = fj + u * GT * VEC;
      if (j < hi)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + at + u * 256 * 16), "l"(fp + j) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    at = at + U * 256 * 16 == kStages * U * 256 * 16 ? 0 : at + U * 256 * 16;
    if (++ft == T) {
      ft = 0;
      fj += kSpan;
      fp = row;
    } else {
      fp += st;
    }
  }
  // the words of one step of the tile whose first value of this thread is j0, in the order of
  // the stages; `none` where there is no value
  __device__ __forceinline__ void take(int j0, uint32_t none, uint32_t (&w)[kWords], int t) {
    if constexpr (VEC > 1) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      from_ring(at, w);
      blank(j0, none, w);
      fetch();
    } else {
      from_row(j0, t, none, w);
    }
  }
  __device__ __forceinline__ void from_ring(uint32_t slot, uint32_t (&w)[kWords]) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * u]), "=r"(w[4 * u + 1]), "=r"(w[4 * u + 2]), "=r"(w[4 * u + 3])
                   : "r"(ring + slot + u * 256 * 16)
                   : "memory");
  }
  __device__ __forceinline__ void blank(int j0, uint32_t none, uint32_t (&w)[kWords]) const {
    if (j0 + (U - 1) * GT * VEC >= hi)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j0 + u * GT * VEC >= hi) w[4 * u] = w[4 * u + 1] = w[4 * u + 2] = w[4 * u + 3] = none;
  }
  __device__ __forceinline__ void from_row(int j0, int t, uint32_t none, uint32_t (&w)[kWords]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * GT * VEC;
      if constexpr (VEC > 1) {
        uint4 v = make_uint4(none, none, none, none);
        if (j < hi) v = *reinterpret_cast<const uint4*>(row + t * st + j);
        w[4 * u] = v.x;
        w[4 * u + 1] = v.y;
        w[4 * u + 2] = v.z;
        w[4 * u + 3] = v.w;
      } else {
        w[u] = none;
        if (j < hi) w[u] = one_word<DT>(row + t * st + j);
      }
    }
  }
  // z of a tile, -inf where there is no value; get(t, none, w): the words of step t
  template <typename G>
  __device__ __forceinline__ void mean(int j0, float inv_t, G get, float2 (&z)[N / 2]) const {
    uint32_t w[kWords];
    if (T == 1) {
      get(0, no_value<DT>(), w);
      unpack_words<DT, VEC>(w, z);
      return;
    }
    float2 err[N / 2];
    get(0, 0u, w);
    unpack_words<DT, VEC>(w, z);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) err[i] = make_float2(0.0f, 0.0f);
    for (int t = 1; t < T; ++t) {
      float2 v[N / 2];
      get(t, 0u, w);
      unpack_words<DT, VEC>(w, v);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) add_exactly(z[i], err[i], v[i]);
    }
    float2 odd = make_float2(0.0f, 0.0f);  // NaN if a sum is not finite
#pragma unroll
    for (int i = 0; i < N / 2; ++i) odd = fma2(z[i], odd, odd);
    if (odd.x + odd.y == 0.0f) {
      if (power_of_two(T)) {  // s / T is exact
        const float2 r2 = make_float2(inv_t, inv_t);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) z[i] = fma2(err[i], r2, mul2(z[i], r2));
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          z[i] = make_float2(quotient(z[i].x, err[i].x, T, inv_t), quotient(z[i].y, err[i].y, T, inv_t));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = j0 + place(i);
        if (j < hi) {
          float& v = i & 1 ? z[i / 2].y : z[i / 2].x;
          v = mean_of<DT>(v, i & 1 ? err[i / 2].y : err[i / 2].x, row + j, st, T, inv_t);
        }
      }
    }
    if (j0 + place(N - 1) >= hi)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (j0 + place(i) >= hi) (i & 1 ? z[i / 2].y : z[i / 2].x) = -INFINITY;
  }
  __device__ __forceinline__ void mean(int j0, float inv_t, float2 (&z)[N / 2]) {
    mean(j0, inv_t, [&](int t, uint32_t none, uint32_t (&w)[kWords]) { take(j0, none, w, t); }, z);
  }
  // The thread's values once more, when all have been taken: put(index) of those at or above
  // `least`, or of all.  kAgain stages are read together; what is put is rare, and read singly.
  static constexpr int kAgain = GT == 32 ? 1 : kWords >= 16 ? 2 : 4;
  __device__ static __forceinline__ uint32_t at_least(const float2 (&z)[N / 2], float least, bool all) {
    uint32_t who = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (all || (i & 1 ? z[i / 2].y : z[i / 2].x) >= least) who |= 1u << i;
    return who;
  }
  template <typename F>
  __device__ __forceinline__ void again(float inv_t, float least, bool all, F put) const {
    const int n = tiles();
    const bool kept = VEC > 1 && n * T <= kStages;  // the whole row is in the ring still
    auto stage = [&](int tile, int t, uint32_t none, uint32_t (&w)[kWords]) {
      if (kept) {
        from_ring((tile * T + t) * U * 256 * 16, w);
        blank(first(tile), none, w);
      } else {
        from_row(first(tile), t, none, w);
      }
    };
    auto wanted = [&](const float2 (&z)[N / 2]) { return at_least(z, least, all); };
    auto put_all = [&](int tile, uint32_t who) {
      for (; who; who &= who - 1) {
        const int j = first(tile) + place(__ffs(who) - 1);
        if (j < hi) put(j);
      }
    };
    if (T == 1) {
      for (int k = 0; k < n; k += kAgain) {
        uint32_t w[kAgain][kWords], who[kAgain], any = 0;
#pragma unroll
        for (int q = 0; q < kAgain; ++q)
          if (k + q < n) stage(k + q, 0, no_value<DT>(), w[q]);
#pragma unroll
        for (int q = 0; q < kAgain; ++q) {
          float2 z[N / 2];
          unpack_words<DT, VEC>(w[q], z);
          who[q] = k + q < n ? wanted(z) : 0;
          any |= who[q];
        }
        if (any)
#pragma unroll 1
          for (int q = 0; q < kAgain; ++q) {
            uint32_t mine = who[0];
#pragma unroll
            for (int i = 1; i < kAgain; ++i) mine = q == i ? who[i] : mine;
            put_all(k + q, mine);
          }
      }
      return;
    }
    for (int k = 0; k < n; ++k) {
      float2 z[N / 2];
      mean(first(k), inv_t, [&](int t, uint32_t none, uint32_t (&v)[kWords]) { stage(k, t, none, v); }, z);
      put_all(k, wanted(z));
    }
  }
  // value i's place after the thread's first value of the tile
  __device__ static __forceinline__ constexpr int place(int i) { return (i / VEC) * GT * VEC + i % VEC; }
  __device__ __forceinline__ int tiles() const { return hi > lo ? (hi - lo + kSpan - 1) / kSpan : 0; }
};

// values before the first 16-byte boundary of a row, with 16-byte vectors
template <int DT, int VEC>
__device__ __forceinline__ int head_of(const typename Elem<DT>::T* row, int V) {
  if constexpr (VEC == 1) return 0;
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(typename Elem<DT>::T);
  return h < V ? h : V;
}

// values [lo, hi) of split `s` of `splits`, of the vectors between head and tail
template <int VEC>
__device__ __forceinline__ void range_of(int V, int head, int split, int splits, int& lo, int& hi) {
  const int vecs = (V - head) / VEC;
  const int each = ((vecs + splits - 1) / splits + 31) / 32 * 32;
  const int a = split * each < vecs ? split * each : vecs, b = a + each < vecs ? a + each : vecs;
  lo = head + a * VEC;
  hi = head + b * VEC;
}

// ---------------------------------------------------------------- alternatives

// The K best keys (order bits, ~index) of a row, after its one pass: every thread
// knows the maximum of its values.  The K-th largest of 32 maxima (of a lane, or
// of 8 threads of a block) is a floor: K values at least lie at or above it, and
// few more.  Only the threads whose maximum reaches it look at their values again
// (in the ring, or by then in L2) and put the keys above the floor into shared
// memory, where the K best are ranked.  More keys than it holds (ties, or rows
// without 32 numbers, where there is no floor): the K-th of those gathered is the
// next floor, and the threads look again; every turn leaves out kGather - K keys
// for good.  A floor among the keys of -inf and NaN is no bound on values (a NaN
// compares with none), so every value is offered again and the keys are compared.
// The K best do not depend on the order in which the keys came.
template <int GT>
struct Gather {
  static constexpr int kGather = GT == 32 ? 128 : 512;
  unsigned long long key[kGather], best[kMaxTop];
  uint32_t group[32];
  int count;
  __device__ __forceinline__ static void sync() {
    if constexpr (GT == 32) __syncwarp();
    else __syncthreads();
  }
  // order bits of the K-th largest of 32 group maxima; most: the thread's
  __device__ __forceinline__ uint32_t kth_group(uint32_t most, int K, int tid) {
    const int lane = tid & 31;
    if constexpr (GT > 32) {
#pragma unroll
      for (int o = GT / 64; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (tid % (GT / 32) == 0) group[tid / (GT / 32)] = most;
      sync();
      most = group[lane];
    }
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)  // a bitonic sort, falling
#pragma unroll
      for (int step = size / 2; step > 0; step /= 2) {
        const uint32_t o = __shfl_xor_sync(0xffffffffu, most, step);
        const bool larger = ((lane & step) == 0) == ((lane & size) == 0 || size == 32);
        most = larger ? max(most, o) : min(most, o);
      }
    return __shfl_sync(0xffffffffu, most, K - 1);
  }
  // the K best of the n keys into best[], falling, zeros where there are fewer
  __device__ __forceinline__ void rank(int n, int K, int tid) {
    if (tid < kMaxTop) best[tid] = 0;
    sync();
    for (int i = tid; i < n; i += GT) {
      const unsigned long long k = key[i];
      int above = 0;
#pragma unroll 4
      for (int o = 0; o < n; ++o) above += key[o] > k;
      if (above < K) best[above] = k;
    }
    sync();
  }
  // offers(least, all, put): put(value, index) of the thread's values at or above least, or of all
  template <typename F>
  __device__ __forceinline__ void select(float most, int K, int tid, F offers) {
    const uint32_t mine = order_bits(most), kth = kth_group(mine, K, tid);
    // -inf stands for a thread without a number too: no floor
    unsigned long long floor = kth > 0x007fffffu ? ((unsigned long long)kth << 32) - 1 : 0;
    for (;;) {
      if (tid == 0) count = 0;
      sync();
      const uint32_t least = (uint32_t)((floor + 1) >> 32);
      const bool all = least <= 0x007fffffu;  // -inf, NaN, or no floor
      if (all || mine >= (uint32_t)(floor >> 32))
        offers(order_value(least), all, [&](float v, int j) {
          const uint32_t bits = order_bits(v);
          const unsigned long long k = ((unsigned long long)bits << 32) | (uint32_t)~j;
          if (k > floor) {
            const int at = atomicAdd(&count, 1);
            if (at < kGather) key[at] = k;
          }
        });
      sync();
      const int n = count;
      rank(n < kGather ? n : kGather, K, tid);
      if (n <= kGather) return;
      floor = best[K - 1] - 1;
    }
  }
};

// The K best of up to 32 falling lists of 64-bit keys in shared memory (lane l
// walks list l): lane k gets the k-th.
__device__ __forceinline__ unsigned long long best_of_lists(const unsigned long long* list, int lists, int stride, int K,
                                                            int lane) {
  unsigned long long mine = 0;
  int at = 0;
  for (int n = 0; n < K; ++n) {
    const unsigned long long head = lane < lists && at < K ? list[lane * stride + at] : 0ull;
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32) == hi ? (uint32_t)head : 0u);
    const unsigned long long top = ((unsigned long long)hi << 32) | lo;
    if (lane == n) mine = top;
    if (head == top) ++at;
  }
  return mine;
}

template <int P>
__device__ __forceinline__ void add_terms(State& s, const float2 (&z)[P], float c);
// a tile into the thread's state
template <int P>
__device__ __forceinline__ void absorb(State& s, const float2 (&z)[P], float most) {
  if (most > s.m) s.move_to(most);
  const Ref f = s.f;
  if (f.off != 0.0f) {
    float2 d[P];
#pragma unroll
    for (int i = 0; i < P; ++i) d[i] = add2(z[i], make_float2(-f.off, -f.off));
    add_terms(s, d, 0.0f);
  } else {
    add_terms(s, z, f.c);
  }
}
template <int P>
__device__ __forceinline__ void add_terms(State& s, const float2 (&z)[P], float c) {
  float2 S2 = make_float2(0.0f, 0.0f), A2 = S2;
  const float2 l2 = make_float2(kLog2e, kLog2e), c2 = make_float2(-c, -c);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float2 t = fma2(z[i], l2, c2);
    t = make_float2(not_below(t.x), not_below(t.y));
    const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
    S2 = add2(S2, e);
    A2 = fma2(e, t, A2);
  }
  s.S += S2.x + S2.y;
  s.A += A2.x + A2.y;
}

// The same for 16-bit logits of one step, in pairs before they are unpacked: the
// maximum, and instead of holding t at -200 the logits at a finite value whose
// 2^t is 0 too (-1e30, and fp16's lowest), half an instruction each.  A
// maximum beyond kFar, or near fp16's lowest, takes the way above.
template <int DT, int WORDS>
__device__ __forceinline__ float most_of(const uint32_t (&w)[WORDS]) {
  uint32_t m = w[0];
#pragma unroll
  for (int i = 1; i < WORDS; ++i) {
    if constexpr (DT == SPK_BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[i]));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[i]));
  }
  const float2 v = unpack_pair<DT>(m);
  return fmaxf(v.x, v.y);
}
template <int DT, int WORDS>
__device__ __forceinline__ void absorb_words(State& s, const uint32_t (&w)[WORDS], float most) {
  if (most > s.m) s.move_to(most);
  const Ref f = s.f;
  if (f.off != 0.0f || s.m < -32768.0f) {
    float2 z[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) z[i] = unpack_pair<DT>(w[i]);
    absorb(s, z, most);
    return;
  }
  float2 S2 = make_float2(0.0f, 0.0f), A2 = S2;
  const float2 l2 = make_float2(kLog2e, kLog2e), c2 = make_float2(-f.c, -f.c);
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    uint32_t v;
    if constexpr (DT == SPK_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(w[i]), "r"(0xf149f149u));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(v) : "r"(w[i]), "r"(0xfbfffbffu));
    const float2 t = fma2(unpack_pair<DT>(v), l2, c2);
    const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
    S2 = add2(S2, e);
    A2 = fma2(e, t, A2);
  }
  s.S += S2.x + S2.y;
  s.A += A2.x + A2.y;
}

template <int P>
__device__ __forceinline__ float most_of(const float2 (&z)[P]) {
  float m = fmaxf(z[0].x, z[0].y);
#pragma unroll
  for (int i = 1; i < P; ++i) m = fmaxf(m, fmaxf(z[i].x, z[i].y));
  return m;
}

struct Out {
  float *logp, *entropy, *top_logp;
  int64_t* top_idx;
  float4* stats;
};

// a log probability: the rounded difference of two numbers may come out above 0 (and an
// entropy below it); a NaN passes
__device__ __forceinline__ float at_most_0(float v) { return v > 0.0f ? 0.0f : v; }

// the row's results from its state and list (one warp).  The gradient gets the
// entropy as it came out: where one symbol has all of the probability its error and
// that of log p cancel in log p + H.
template <int DT>
__device__ __forceinline__ void write_row(const Logits& x, const typename Elem<DT>::T* row, int64_t r, int64_t y,
                                          State s, unsigned long long key, int K, int lane, const Out& o) {
  const Ref f = s.f;
  const float l2s = log2f(s.S), H = kLn2 * (l2s - s.A / s.S);
  if (lane == 0) {
    o.logp[r] = at_most_0(kLn2 * (log2_from(mean_over_t<DT>(row + y, x.st, x.T, x.inv_t), f) - l2s));
    o.entropy[r] = H < 0.0f ? 0.0f : H;
    if (o.stats) o.stats[r] = make_float4(f.off, f.c, s.S, H);
  }
  if (lane < K) {
    o.top_idx[r * K + lane] = (int64_t)(~(uint32_t)key);
    // a row without a distribution has none for the alternatives either
    o.top_logp[r * K + lane] = at_most_0(kLn2 * (log2_from(order_value((uint32_t)(key >> 32)), f) - l2s));
  }
}

__device__ __forceinline__ void write_unused(int64_t r, int K, int lane, const Out& o) {
  if (lane == 0) {
    o.logp[r] = o.entropy[r] = 0.0f;
    if (o.stats) o.stats[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  if (lane < K) {
    o.top_logp[r * K + lane] = 0.0f;
    o.top_idx[r * K + lane] = -1;
  }
}

// Values of a row that one warp takes, where there are rows for 16 warps on every
// SM, and for 64: fewer threads share what a row costs beside its values (4096 x
// 1000 fp32 of 4 steps 27 us, by blocks 37; 16384 x 1000 bf16 25, by blocks 82;
// 16384 x 8192 78, by blocks 111).
constexpr int kWarpRow = 1024, kManyRow = 8192;

// Without alternatives bound by instructions more than by HBM: 8192 x 65536 bf16
// (1.07 GB) take 213 us, 0.78 of a plain copy's rate, at 80 % of the issue slots;
// with 5 alternatives 389 us, with 32 537 us.  16384 x 256 fp32 of 4 steps: 27 us,
// with 5 alternatives 37 us, bound by latency (half of the issue slots, 43 and 33 %
// of the warps: a warp waits for its one row's copies and reductions).
// GT = 32: a warp a row.  GT = 256: a block a (row, split); with several splits
// the state and list go to part / keys.
template <int DT, int VEC, int U, int GT, bool TOP>
__global__ void __launch_bounds__(256, TOP ? 3 : 4) fwd_kernel(Logits x, const int64_t* __restrict__ tokens, int64_t ignore, int K,
                                                  int splits, Out o, float4* part, unsigned long long* keys, int* bad,
                                                  int scan_bad) {
  using E = typename Elem<DT>::T;
  extern __shared__ uint4 ring[];
  if (scan_bad && blockIdx.x == 0) {  // the first block, so that it is not the last to end
    scan_tokens(tokens, x.rows, x.V, ignore, bad);
    return;
  }
  const int64_t block = (int64_t)blockIdx.x - scan_bad;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = GT == 32 ? block * 8 + warp : block;
  const int64_t r = GT == 32 ? unit : unit / splits;
  const int split = GT == 32 ? 0 : (int)(unit - r * splits);
  if (r >= x.rows) return;
  const int64_t y = __ldg(tokens + r);
  const E* row = reinterpret_cast<const E*>(x.base) + r * x.sr;
  const int head = head_of<DT, VEC>(row, x.V), tail = (x.V - head) % VEC;
  int lo, hi;
  range_of<VEC>(x.V, head, split, splits, lo, hi);
  const int tid = GT == 32 ? lane : (int)threadIdx.x;
  Tiles<DT, VEC, U, GT> tl(ring, row, x.st, x.T, lo, hi, tid);  // the first copies go out before the token is here
  if (y == ignore || y < 0 || y >= x.V) {
    if constexpr (VEC > 1) asm volatile("cp.async.wait_all;" ::: "memory");
    if (split == 0 && (GT == 32 || warp == 0)) {
      write_unused(r, K, lane, o);
      if (!scan_bad && y != ignore && lane == 0) atomicExch(bad, 1);
    }
    return;
  }
  State s;
  const int tiles = tl.tiles();
  using TL = Tiles<DT, VEC, U, GT>;
  constexpr int N = TL::N;
  float2 z[N / 2];
  for (int k = 0; k < tiles; ++k) {
    const int j0 = tl.first(k);
    if constexpr (VEC > 1 && DT != SPK_F32)
      if (x.T == 1) {
        uint32_t w[TL::kWords];
        tl.take(j0, no_value<DT>(), w, 0);
        if constexpr (TOP && GT == 32) unpack_words<DT, VEC>(w, z);
        absorb_words<DT>(s, w, most_of<DT>(w));
        continue;
      }
    tl.mean(j0, x.inv_t, z);
    absorb(s, z, most_of(z));
  }
  if constexpr (VEC > 1) asm volatile("cp.async.wait_all;" ::: "memory");
  // the values beside the vectors
  const int edge = VEC == 1 || split > 0 ? -1 : tid < head ? tid : tid >= GT - tail ? x.V - (GT - tid) : -1;
  float beside = -INFINITY;
  if (edge >= 0) {
    beside = mean_over_t<DT>(row + edge, x.st, x.T, x.inv_t);
    float2 z[1] = {make_float2(beside, -INFINITY)};
    absorb(s, z, fmaxf(beside, -INFINITY));
  }
  __shared__ Gather<GT> mem[TOP ? 256 / GT : 1];
  Gather<GT>& top = mem[TOP && GT == 32 ? warp : 0];
  if constexpr (TOP)
    top.select(s.m, K, tid, [&](float least, bool all, auto put) {
      if (GT == 32 && tiles == 1) {  // a short row's values are here still
        for (uint32_t who = TL::at_least(z, least, all); who; who &= who - 1) {
          const int at = __ffs(who) - 1, j = tl.first(0) + TL::place(at);
          float v = z[0].x;
#pragma unroll
          for (int i = 1; i < N; ++i) v = at == i ? (i & 1 ? z[i / 2].y : z[i / 2].x) : v;
          if (j < hi) put(v, j);
        }
      } else {
        tl.again(x.inv_t, least, all, [&](int j) { put(mean_over_t<DT>(row + j, x.st, x.T, x.inv_t), j); });
      }
      if (edge >= 0) put(beside, edge);
    });
  s.join_warp();
  if constexpr (GT > 32) {
    __shared__ float ws[8][3];
    if (lane == 0) {
      ws[warp][0] = s.m;
      ws[warp][1] = s.S;
      ws[warp][2] = s.A;
    }
    __syncthreads();
    if (warp > 0) return;
    s = lane < 8 ? State(ws[lane][0], ws[lane][1], ws[lane][2]) : State();
    s.join_warp();
  }
  const unsigned long long key = TOP && lane < K ? top.best[lane] : 0ull;
  if (GT > 32 && splits > 1) {
    if (lane == 0) part[unit] = make_float4(s.m, s.S, s.A, 0.0f);
    if (lane < K) keys[unit * K + lane] = key;
    return;
  }
  write_row<DT>(x, row, r, y, s, key, K, lane, o);
}

// a block of one warp a row: the splits' states and lists
template <int DT>
__global__ void __launch_bounds__(32) join_kernel(Logits x, const int64_t* __restrict__ tokens, int64_t ignore, int K,
                                                  int splits, Out o, const float4* part, const unsigned long long* keys) {
  __shared__ unsigned long long list[32 * kMaxTop];
  const int lane = threadIdx.x;
  const int64_t r = blockIdx.x, y = tokens[r];
  pdl_wait();
  if (y == ignore || y < 0 || y >= x.V) return;
  State s;
  if (lane < splits) {
    const float4 p = part[r * splits + lane];
    s = State(p.x, p.y, p.z);
  }
#pragma unroll 8
  for (int i = lane; i < splits * K; i += 32) list[i] = keys[r * splits * K + i];
  __syncwarp();
  s.join_warp();
  const unsigned long long key = K > 0 ? best_of_lists(list, splits, K, K, lane) : 0ull;
  write_row<DT>(x, reinterpret_cast<const typename Elem<DT>::T*>(x.base) + r * x.sr, r, y, s, key, K, lane, o);
}

// ---------------------------------------------------------------- backward

struct Grads {
  const float *logp, *entropy, *top;
  const int64_t* top_idx;
  const float4* stats;
};

// dz_j = 2^t_j (a t_j + b), and g_logp, g_top added at their symbols.  Bound by
// HBM: 8192 x 65536 bf16, read and written, take 320 us, 6.7 TB/s.
template <int DT, int VEC, int U, int GT>
__global__ void __launch_bounds__(256) bwd_kernel(Logits x, const int64_t* __restrict__ tokens, int64_t ignore, int K,
                                                  int splits, Grads g, typename Elem<DT>::T* __restrict__ grad) {
  using E = typename Elem<DT>::T;
  using TL = Tiles<DT, VEC, U, GT>;
  extern __shared__ uint4 ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = GT == 32 ? (int64_t)blockIdx.x * 8 + warp : (int64_t)blockIdx.x;
  const int64_t r = GT == 32 ? unit : unit / splits;
  const int split = GT == 32 ? 0 : (int)(unit - r * splits);
  if (r >= x.rows) return;
  const int64_t y = __ldg(tokens + r);
  const bool used = y != ignore && y >= 0 && y < x.V;
  const E* row = reinterpret_cast<const E*>(x.base) + r * x.sr;
  E* out = grad + r * x.V;
  const int64_t ot = x.rows * x.V;  // step stride of the gradient
  const int head = head_of<DT, VEC>(row, x.V), tail = (x.V - head) % VEC;
  int lo, hi;
  range_of<VEC>(x.V, head, split, splits, lo, hi);
  const int tid = GT == 32 ? lane : (int)threadIdx.x;
  const int edge = VEC == 1 || split > 0 ? -1 : tid < head ? tid : tid >= GT - tail ? x.V - (GT - tid) : -1;
  if (!used) {
    float zero[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero[i] = 0.0f;
    for (int t = 0; t < x.T; ++t) {
      for (int j = lo + tid * VEC; j < hi; j += GT * VEC) Vec<DT, VEC>::store(out + t * ot + j, zero);
      if (edge >= 0) out[t * ot + edge] = Elem<DT>::make(0.0f);
    }
    return;
  }
  TL tl(ring, row, x.st, x.T, lo, hi, tid);
  const float4 sv = g.stats[r];
  const Ref f = {sv.x, sv.y};
  const float gl = g.logp ? g.logp[r] : 0.0f, gh = g.entropy ? g.entropy[r] : 0.0f;
  float G = gl;
  if (g.top)
    for (int k = 0; k < K; ++k) G += g.top[r * K + k];
  const float scale = x.inv_t / sv.z;  // 1 / (T S)
  const float a = -gh * kLn2 * scale, b = -(G + gh * (sv.w - kLn2 * log2f(sv.z))) * scale;
  const float2 l2 = make_float2(kLog2e, kLog2e), c2 = make_float2(-f.c, -f.c), a2 = make_float2(a, a),
               b2 = make_float2(b, b);
  auto at_one = [&](float z) {
    const float t = not_below(log2_from(z, f));
    return exp2_approx(t) * fmaf(a, t, b);
  };
  const int tiles = tl.tiles();
  for (int k = 0; k < tiles; ++k) {
    const int j0 = tl.first(k);
    float2 z[TL::N / 2];
    tl.mean(j0, x.inv_t, z);
    if (f.off != 0.0f)
#pragma unroll
      for (int i = 0; i < TL::N / 2; ++i) z[i] = add2(z[i], make_float2(-f.off, -f.off));
#pragma unroll
    for (int i = 0; i < TL::N / 2; ++i) {
      float2 t = fma2(z[i], l2, c2);
      t = make_float2(not_below(t.x), not_below(t.y));
      z[i] = mul2(make_float2(exp2_approx(t.x), exp2_approx(t.y)), fma2(a2, t, b2));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * GT * VEC;
      if (j < hi) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = (u * VEC + i) & 1 ? z[(u * VEC + i) / 2].y : z[(u * VEC + i) / 2].x;
        const typename Vec<DT, VEC>::W w = Vec<DT, VEC>::pack(v);
        for (int t = 0; t < x.T; ++t) *reinterpret_cast<typename Vec<DT, VEC>::W*>(out + t * ot + j) = w;
      }
    }
  }
  if constexpr (VEC > 1) asm volatile("cp.async.wait_all;" ::: "memory");
  if (edge >= 0) {
    const E d = Elem<DT>::make(at_one(mean_over_t<DT>(row + edge, x.st, x.T, x.inv_t)));
    for (int t = 0; t < x.T; ++t) out[t * ot + edge] = d;
  }
  // the named symbols once more, by one warp after the others' writes: lane k the k-th
  // alternative, then the token where it is none of them
  if constexpr (GT > 32) __syncthreads();
  else __syncwarp();
  if (GT > 32 && warp > 0) return;
  auto mine = [&](int64_t j) {  // of this block's share of the row, and a symbol at all
    return (j >= lo && j < hi) ||
           (split == 0 && VEC > 1 && ((j >= 0 && j < head) || (j >= x.V - tail && j < x.V)));
  };
  auto put = [&](int64_t j, float add) {
    const E d = Elem<DT>::make(fmaf(add, x.inv_t, at_one(mean_over_t<DT>(row + j, x.st, x.T, x.inv_t))));
    for (int t = 0; t < x.T; ++t) out[t * ot + j] = d;
  };
  bool is_top = false;
  if (g.top && lane < K) {
    const int64_t j = g.top_idx[r * K + lane];
    is_top = j == y;
    if (mine(j)) put(j, g.top[r * K + lane] + (is_top ? gl : 0.0f));
  }
  is_top = __any_sync(0xffffffffu, is_top);
  if (lane == 0 && !is_top && mine(y)) put(y, gl);
}

// ---------------------------------------------------------------- host

// Blocks that a row is cut over, so that there are two for every SM: 1 x 65536 bf16
// 10 us and with 8 alternatives 14 us, in one block 12 and 21; 32 x 65536 12 and
// 18, uncut 12 and 21.
inline int splits_of(int64_t rows, int64_t V) {
  if (V <= kWarpRow * 4 || rows >= 2 * (int64_t)num_sms()) return 1;
  int64_t s = (2 * (int64_t)num_sms() + rows - 1) / rows;
  const int64_t most = V / 2048;
  if (s > most) s = most;
  return (int)(s > 32 ? 32 : s < 1 ? 1 : s);
}
inline bool warp_rows(int64_t rows, int64_t V) {
  return V <= 256 || (V <= kWarpRow && rows >= 16 * (int64_t)num_sms()) ||
         (V <= kManyRow && rows >= 64 * (int64_t)num_sms());
}

// 48 KB of dynamic shared memory without asking, the kernel's static arrays included
template <typename K>
bool ask_smem(K kernel, int bytes) {
  return bytes <= (40 << 10) ||
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

template <int DT, int VEC, int U, int GT>
int launch_fwd(const Logits& x, const int64_t* tokens, int64_t ignore, int K, int splits, const Out& o, float4* part,
               unsigned long long* keys, int* bad, cudaStream_t st) {
  const int64_t units = GT == 32 ? (x.rows + 7) / 8 : x.rows * splits;
  const bool scan = x.rows <= kScanTokens;
  if (!scan) cudaMemsetAsync(bad, 0, sizeof(int), st);
  constexpr int smem = Tiles<DT, VEC, U, GT>::kBytes * 256;
  auto kernel = K > 0 ? fwd_kernel<DT, VEC, U, GT, true> : fwd_kernel<DT, VEC, U, GT, false>;
  if (!ask_smem(kernel, smem)) return check_launch("token_logprobs_fwd");
  kernel<<<(unsigned)(units + (scan ? 1 : 0)), 256, smem, st>>>(x, tokens, ignore, K, splits, o, part, keys, bad,
                                                                scan ? 1 : 0);
  if (splits > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)x.rows);
    cfg.blockDim = dim3(32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    add_pdl_attr(cfg, at);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<DT>, x, tokens, ignore, K, splits, o, (const float4*)part,
                                             (const unsigned long long*)keys);
    if (e != cudaSuccess) return fail(SPK_ERR_LAUNCH, "token_logprobs_fwd: %s", cudaGetErrorString(e));
  }
  return check_launch("token_logprobs_fwd");
}

template <int DT>
int dispatch_fwd(bool wide, const Logits& x, const int64_t* tokens, int64_t ignore, int K, int splits, const Out& o,
                 float4* part, unsigned long long* keys, int* bad, cudaStream_t st) {
  constexpr int kWide = 16 / (int)sizeof(typename Elem<DT>::T);
#define GO(VEC, U, GT) launch_fwd<DT, VEC, U, GT>(x, tokens, ignore, K, splits, o, part, keys, bad, st)
  if (warp_rows(x.rows, x.V)) return wide ? GO(kWide, 8 / kWide, 32) : GO(1, 8, 32);
  // Shorter tiles: fewer threads without a value.  Shorter / longer, us: 10 x 1003 x 1000 fp32
  // 21 / 35 (with 5 alternatives 37 / 55), 4096 x 2048 bf16 25 / 29 (51 / 53), 4096 x 4096 31 / 29
  // (59 / 55), 2048 x 8192 23 / 21 (41 / 37).
  if (x.V <= 4096) return wide ? GO(kWide, 1, 256) : GO(1, 4, 256);
  return wide ? GO(kWide, 16 / kWide, 256) : GO(1, 8, 256);
#undef GO
}

template <int DT, int VEC, int U, int GT>
int launch_bwd(const Logits& x, const int64_t* tokens, int64_t ignore, int K, int splits, const Grads& g, void* grad,
               cudaStream_t st) {
  const int64_t units = GT == 32 ? (x.rows + 7) / 8 : x.rows * splits;
  constexpr int smem = Tiles<DT, VEC, U, GT>::kBytes * 256;
  if (!ask_smem(bwd_kernel<DT, VEC, U, GT>, smem)) return check_launch("token_logprobs_bwd");
  bwd_kernel<DT, VEC, U, GT><<<(unsigned)units, 256, smem, st>>>(x, tokens, ignore, K, splits, g,
                                                                reinterpret_cast<typename Elem<DT>::T*>(grad));
  return check_launch("token_logprobs_bwd");
}

template <int DT>
int dispatch_bwd(bool wide, const Logits& x, const int64_t* tokens, int64_t ignore, int K, int splits, const Grads& g,
                 void* grad, cudaStream_t st) {
  constexpr int kWide = 16 / (int)sizeof(typename Elem<DT>::T);
#define GO(VEC, U, GT) launch_bwd<DT, VEC, U, GT>(x, tokens, ignore, K, splits, g, grad, st)
  if (warp_rows(x.rows, x.V)) return wide ? GO(kWide, 8 / kWide, 32) : GO(1, 8, 32);
  // forward and backward with shorter / longer tiles, us: 10 x 1003 x 1000 fp32 37 / 64, 4096 x
  // 4096 bf16 53 / 62, 2048 x 8192 41 / 43
  if (x.V <= 4096) return wide ? GO(kWide, 1, 256) : GO(1, 4, 256);
  return wide ? GO(kWide, 16 / kWide, 256) : GO(1, 8, 256);
#undef GO
}

}  // namespace lpk
}  // namespace spk

#define SPK_LP_SIZES()                                                                                              \
  SPK_REQUIRE(float_type(dtype), SPK_ERR_INVALID, "logits must be fp32, fp16 or bf16");                            \
  SPK_REQUIRE(T >= 1 && T <= 64 && rows >= 1 && rows < (1ll << 31) - 8 && V >= 1 && V < (1ll << 30), SPK_ERR_SHAPE,     \
              "unsupported sizes T=%lld rows=%lld V=%lld", (long long)T, (long long)rows, (long long)V);            \
  SPK_REQUIRE((T == 1 || step_stride >= 0) && (rows == 1 || row_stride >= 0), SPK_ERR_SHAPE, "negative stride");    \
  SPK_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= V, SPK_ERR_SHAPE, "top_k=%lld: at most %d and V",          \
              (long long)top_k, kMaxTop);                                                                           \
  SPK_REQUIRE(aligned(stats, 16), SPK_ERR_ALIGN, "stats must be 16-byte aligned")

extern "C" {

int64_t spk_token_logprobs_workspace_bytes(int64_t, int64_t rows, int64_t V, int64_t top_k) {
  if (rows < 1 || V < 1 || top_k < 0) return 0;
  const int64_t s = spk::lpk::splits_of(rows, V);
  return s > 1 ? rows * s * (16 + 8 * top_k) : 0;
}

int spk_token_logprobs_fwd(const void* logits, int dtype, int64_t T, int64_t rows, int64_t V, int64_t step_stride,
                           int64_t row_stride, const int64_t* tokens, int64_t ignore_index, int64_t top_k, float* logp,
                           float* entropy, float* top_logp, int64_t* top_idx, float* stats, int* bad_token,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace spk;
  using namespace spk::lpk;
  SPK_REQUIRE(logits && tokens && logp && entropy && bad_token, SPK_ERR_INVALID, "null pointer argument");
  SPK_LP_SIZES();
  SPK_REQUIRE(top_k == 0 || (top_logp && top_idx), SPK_ERR_INVALID, "null top_logp or top_idx");
  const int64_t need = spk_token_logprobs_workspace_bytes(T, rows, V, top_k);
  SPK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SPK_ERR_INVALID,
              "workspace smaller than spk_token_logprobs_workspace_bytes()");
  SPK_REQUIRE(aligned(workspace, 16), SPK_ERR_ALIGN, "workspace must be 16-byte aligned");
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Logits x = {logits, (int)T, (int)V, rows, step_stride, row_stride, 1.0f / (float)T};
  const Out o = {logp, entropy, top_logp, top_idx, reinterpret_cast<float4*>(stats)};
  const int splits = splits_of(rows, V), K = (int)top_k;
  float4* part = reinterpret_cast<float4*>(workspace);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(part + rows * splits);
  // the steps of a value lie alike to 16 bytes
  const bool wide = aligned(logits, dtype_size(dtype)) && (T == 1 || step_stride * dtype_size(dtype) % 16 == 0);
  auto go = dtype == SPK_F32 ? dispatch_fwd<SPK_F32> : dtype == SPK_F16 ? dispatch_fwd<SPK_F16> : dispatch_fwd<SPK_BF16>;
  return go(wide, x, tokens, ignore_index, K, splits, o, part, keys, bad_token, s);
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
  int rc = check_stream_device(stream);
  if (rc != SPK_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Logits x = {logits, (int)T, (int)V, rows, step_stride, row_stride, 1.0f / (float)T};
  const Grads g = {g_logp, g_entropy, g_top, top_idx, reinterpret_cast<const float4*>(stats)};
  const int64_t e = dtype_size(dtype);
  // the steps of a value, and its gradient's, lie alike to 16 bytes
  const bool wide = aligned(logits, (int)e) && (T == 1 || (step_stride * e % 16 == 0 && rows * V * e % 16 == 0)) &&
                    (rows == 1 || (row_stride - V) * e % 16 == 0) &&
                    (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad)) % 16 == 0;
  auto go = dtype == SPK_F32 ? dispatch_bwd<SPK_F32> : dtype == SPK_F16 ? dispatch_bwd<SPK_F16> : dispatch_bwd<SPK_BF16>;
  return go(wide, x, tokens, ignore_index, (int)top_k, splits_of(rows, V), g, grad, s);
}

}  // extern "C"
