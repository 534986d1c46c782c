// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
// With y = (x - max x) log2(e) / tau, S = sum 2^y and A = sum 2^y y:
// log p(t) = (x_t - max x) / tau - ln2 log2 S, H = ln2 (log2 S - A / S). The maximum is
// taken off before the product, which would overflow for logits at the type's lowest value.
//
// The logits are read once: a thread keeps a maximum and both sums of its own, moved to a
// new maximum chunk by chunk. The alternatives come along: a CTA keeps a list of candidates
// and a threshold that at least top_k logits reach, and an ordinary chunk costs each warp a
// vote that nothing reaches it. Few rows are split over the CTAs of a cluster, which join
// through shared memory; there is no workspace and no atomic on global memory.
//
// One read of the logits is the least there is; instructions bound it, 8.5 a logit without
// alternatives and 12.3 with 20 (of 16 bits: unpacking, four halves of packed operations, 2^y,
// a maximum; the look at the few chunks of a warp that hold candidates). 2048 x 151936 bf16, top
// 20: 144 us, 4.3 TB/s, 66% of a copy's rate, with 8 CTAs of 128 threads an SM, whose first
// chunks and list cuts overlap better than those of 4 of 256 (156 us); 1776 rows without
// alternatives 92 us, 5.8 TB/s, 89%. 16 x 50257 fp16, top 5, split over clusters: 9.3 us.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace dropkv {
namespace {

constexpr int LP_NT = 128;
constexpr int LP_WARPS = LP_NT / 32;
constexpr int LP_CTAS = 8;                      // CTAs an SM holds
constexpr int LP_MAX_K = 64;
constexpr int LP_CAP = 1024;                    // candidates
constexpr int LP_MAX_S = 8;                     // CTAs of a cluster, at most
constexpr int LP_GROUPS = 64;                   // groups of threads
constexpr int LP_GT = LP_NT / LP_GROUPS;        // threads of a group
static_assert(LP_GROUPS >= LP_MAX_K && LP_NT == LP_GT * LP_GROUPS && 32 % LP_GT == 0, "the top_k-th of the groups' best");

// Order of the alternatives: larger logits first (NaN above all), then lower index. 0 is
// below every logit's key.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
  const uint32_t k = x != x ? 0xffffffffu : ordered_key(x);
  return ((uint64_t)k << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(uint64_t key) { return key_to_float((uint32_t)(key >> 32)); }

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The two halves of a cluster barrier. Nothing is handed over between them: no release is needed.
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// What a thread, a CTA or a row knows: maximum, S and A against it.
struct LpSums {
  float m, s, t;
};
// Both sums moved to the maximum of two parts; an empty part has m = -inf and sums of 0.
__device__ __forceinline__ void lp_move(LpSums& a, float m, float c) {
  if (a.m == m) return;                 // (-inf too)
  if (a.m != -INFINITY || a.s != 0.f) {  // a part of NaN alone has m = -inf as well: it stays NaN
    const float d = (a.m - m) * c, f = lp_ex2(d);
    a.t = f == 0.f ? 0.f : f * fmaf(d, a.s, a.t);  // (d times s may overflow then)
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b, float c) {
  const float m = fmaxf(a.m, b.m);
  lp_move(a, m, c);
  lp_move(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}

struct LpSmem {
  uint64_t list[LP_CAP];
  uint64_t lists[LP_MAX_S * LP_MAX_K];  // in a cluster's first CTA: every CTA's best
  LpSums parts[LP_MAX_S];               // and sums
  uint64_t tops[LP_NT];
  uint32_t groups[LP_GROUPS];           // the best value of each group of threads, as an ordered key
  uint32_t level;                       // the top_k-th of them
  uint64_t edge;                        // the top_k-th best key of the threads
  LpSums warps[LP_WARPS];
  int count;
};

// The first n entries of `list` sorted, the best k of them kept: an entry's place is the
// number of entries above it. A thread has one entry; a longer list goes through LP_NT entries
// at a time, the best so far among them. All threads; returns the number kept.
__device__ __forceinline__ int lp_keep_best(uint64_t* list, int n, int k) {
  const int tid = threadIdx.x;
  int done = min(n, LP_NT), m = done;  // entries seen, entries in the round
  while (true) {
    __syncthreads();
    uint64_t mine = 0;
    int rank = LP_CAP;
    if (tid - (tid & 31) < m) {  // (warps without an entry have nothing to count)
      if (tid < m) mine = list[tid];
      rank = 0;
      int e = 0;
#pragma unroll 2
      for (; e + 4 <= m; e += 4) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list + e), y = *reinterpret_cast<const ulonglong2*>(list + e + 2);
        rank += (x.x > mine) + (x.y > mine) + (y.x > mine) + (y.y > mine);
      }
      for (; e < m; ++e) rank += list[e] > mine;
    }
    __syncthreads();
    if (tid < m && rank < k) list[rank] = mine;
    m = min(m, k);
    if (done >= n) break;
    const int more = min(n - done, LP_NT - m);
    uint64_t x = 0;
    if (tid < more) x = list[done + tid];
    __syncthreads();
    if (tid < more) list[m + tid] = x;
    done += more;
    m += more;
  }
  __syncthreads();
  return m;
}

// Two floats in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t lp_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void lp_unpair(uint64_t r, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t lp_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <typename T>
struct LpVec;  // 16 bytes of logits
template <>
struct LpVec<float> {
  static constexpr int N = 4, U = 4;  // logits of a vector, vectors of a thread and chunk
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8, U = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
};
template <>
struct LpVec<__half> {
  static constexpr int N = 8, U = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
};

// The largest logit of a vector, NaN if one is.
__device__ __forceinline__ float lp_top(const uint4& v, float) {
  return lp_max_nan(lp_max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), lp_max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float lp_top(const uint4& v, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return lp_max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float lp_top(const uint4& v, __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return lp_max_nan(__low2float(m), __high2float(m));
}

// A bit for each logit of U vectors that is not below x (x is a logit's value: it converts
// exactly), and the logit a bit stands for. 16-bit types: even logits have the low half.
template <int U>
__device__ __forceinline__ uint32_t lp_reach(const uint4* v, float x, float) {
  uint32_t bits = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= __uint_as_float(w[i]) < x ? 0u : 1u << (4 * u + i);
  }
  return bits;
}
template <int U, typename T2>
__device__ __forceinline__ uint32_t lp_reach2(const uint4* v, T2 x) {
  uint32_t below = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) below |= __hlt2_mask(reinterpret_cast<const T2&>(w[i]), x) & (0x00010001u << (4 * u + i));
  }
  return ~below;
}
template <int U>
__device__ __forceinline__ uint32_t lp_reach(const uint4* v, float x, __nv_bfloat16) {
  return lp_reach2<U>(v, __float2bfloat162_rn(x));
}
template <int U>
__device__ __forceinline__ uint32_t lp_reach(const uint4* v, float x, __half) {
  return lp_reach2<U>(v, __float2half2_rn(x));
}
__device__ __forceinline__ int lp_place(int bit, float) { return bit; }
__device__ __forceinline__ int lp_place(int bit, __nv_bfloat16) { return 2 * (bit & 15) + (bit >> 4); }
__device__ __forceinline__ int lp_place(int bit, __half) { return 2 * (bit & 15) + (bit >> 4); }

// and its value: registers have no index, but a tree of selects
template <int U>
__device__ __forceinline__ uint32_t lp_word(const uint4* v, int i) {
  static_assert(U == 4, "16 words");
  uint32_t w[8];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    w[2 * u] = i & 1 ? v[u].y : v[u].x;
    w[2 * u + 1] = i & 1 ? v[u].w : v[u].z;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) w[u] = i & 2 ? w[2 * u + 1] : w[2 * u];
  return i & 8 ? (i & 4 ? w[3] : w[2]) : (i & 4 ? w[1] : w[0]);
}
template <int U>
__device__ __forceinline__ float lp_pick(const uint4* v, int bit, float) { return __uint_as_float(lp_word<U>(v, bit)); }
template <int U>
__device__ __forceinline__ float lp_pick(const uint4* v, int bit, __nv_bfloat16) {
  const uint32_t w = lp_word<U>(v, bit & 15);
  return __uint_as_float(bit & 16 ? w & 0xffff0000u : w << 16);
}
template <int U>
__device__ __forceinline__ float lp_pick(const uint4* v, int bit, __half) {
  const uint32_t w = lp_word<U>(v, bit & 15);
  return __half2float(__ushort_as_half((unsigned short)(bit & 16 ? w >> 16 : w)));
}

template <typename T>
__device__ __forceinline__ uint4 lp_lowest();
template <>
__device__ __forceinline__ uint4 lp_lowest<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <>
__device__ __forceinline__ uint4 lp_lowest<__nv_bfloat16>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
template <>
__device__ __forceinline__ uint4 lp_lowest<__half>() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }

// The alternatives found so far: at least top_k logits reach the threshold (0: none yet), and
// every logit read that does is among the list's first `kept`.
struct LpCandidates {
  uint64_t floor_key;
  int kept;
};
__device__ __forceinline__ float lp_floor_value(uint64_t key) {  // what a logit has to reach
  return key ? lp_value(key) : __int_as_float(0xff800000);
}

// The logits of the chunk that reach the threshold go to the list, while there is room; all are
// counted. A bit for each of a thread's logits first, then the few that are set.
template <typename T>
__device__ __forceinline__ void lp_collect(LpSmem& sm, uint64_t floor_key, const uint4* cur, int V, int v0, int v_end, float mx) {
  constexpr int N = LpVec<T>::N, U = LpVec<T>::U;
  const float fv = lp_floor_value(floor_key);
  if (!__any_sync(0xffffffffu, !(mx < fv))) return;
  for (uint32_t bits = lp_reach<U>(cur, fv, T()); bits; bits &= bits - 1) {
    const int b = __ffs(bits) - 1, q = lp_place(b, T()), v = v0 + (q / N) * LP_NT + (int)threadIdx.x;
    const int64_t e = (int64_t)v * N + q % N;
    if (v >= v_end || e >= V) continue;
    const uint64_t key = lp_key(lp_pick<U>(cur, b, T()), (int)e);
    if (key < floor_key) continue;
    const int at = atomicAdd(&sm.count, 1);
    if (at < LP_CAP) sm.list[at] = key;
  }
  __syncwarp();
}
// The list of n entries cut to the best top_k, and the threshold moved up to the last of them.
// All threads; ends without a barrier.
__device__ __forceinline__ void lp_cut(LpSmem& sm, LpCandidates& cand, int n, int k) {
  cand.kept = lp_keep_best(sm.list, n, k);
  if (cand.kept == k && sm.list[k - 1] > cand.floor_key) cand.floor_key = sm.list[k - 1];
  if (threadIdx.x == 0) sm.count = cand.kept;
}

// A chunk whose candidates may be many: the threshold is raised from the chunk itself first.
template <typename T>
__device__ __forceinline__ void lp_top_chunk(LpSmem& sm, LpCandidates& cand, const uint4* cur, const T* x0, int V, int v0, int v_end,
                                             float mx, int k) {
  const int tid = threadIdx.x;
  // The k-th of the best of 64 groups of threads is a threshold that k logits reach, and
  // few more. A group's threads share out the groups to compare theirs with. (Padding
  // counts as -inf, which every logit reaches.)
  uint32_t best = mx != mx ? 0xffffffffu : ordered_key(mx);
#pragma unroll
  for (int o = 1; o < LP_GT; o *= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (tid % LP_GT == 0) sm.groups[tid / LP_GT] = best;
  __syncthreads();
  int over = 0, same = 0;
#pragma unroll
  for (int q = 0; q < LP_GROUPS / LP_GT; q += 4) {
    const uint4 g = *reinterpret_cast<const uint4*>(&sm.groups[(tid % LP_GT) * (LP_GROUPS / LP_GT) + q]);
    over += (g.x > best) + (g.y > best) + (g.z > best) + (g.w > best);
    same += (g.x == best) + (g.y == best) + (g.z == best) + (g.w == best);
  }
#pragma unroll
  for (int o = 1; o < LP_GT; o *= 2) {
    over += __shfl_xor_sync(0xffffffffu, over, o);
    same += __shfl_xor_sync(0xffffffffu, same, o);
  }
  if (over < k && over + same >= k) sm.level = best;  // (all that write it have one value)
  __syncthreads();
  const uint64_t least = (uint64_t)sm.level << 32;  // the lowest key of that value
  if (least > cand.floor_key) cand.floor_key = least;
  lp_collect<T>(sm, cand.floor_key, cur, V, v0, v_end, mx);
  __syncthreads();
  if (sm.count > LP_CAP) {
    // Too many (logits in an order that defeats the groups). With the list as it was before this
    // chunk, cut to k, each thread's first vector is taken, then its second, and so on: the exact
    // k-th of the threads' best keys is a threshold that all but k threads stay below, and
    // whatever these hold in a vector fits. (The logits are read again: registers have no index.)
    constexpr int N = LpVec<T>::N, U = LpVec<T>::U;
    static_assert(LP_CAP >= LP_MAX_K * (1 + N), "a list and a vector of k threads");
    __syncthreads();
    lp_cut(sm, cand, cand.kept, k);
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * LP_NT + tid;
      auto key = [&](int i) -> uint64_t {  // 0: not to be taken
        const int64_t e = (int64_t)v * N + i;
        const uint64_t q = v < v_end && e < V ? lp_key(to_f(x0[e]), (int)e) : 0;
        return q >= cand.floor_key ? q : 0;
      };
      uint64_t top = 0;
#pragma unroll 1
      for (int i = 0; i < N; ++i) top = max(top, key(i));
      sm.tops[tid] = top;
      if (tid == 0) sm.edge = 0;
      __syncthreads();
      int r = 0;
      for (int e = 0; e < LP_NT; ++e) r += sm.tops[e] > top;
      if (r == k - 1 && top) sm.edge = top;
      __syncthreads();
      if (sm.edge > cand.floor_key) cand.floor_key = sm.edge;
#pragma unroll 1
      for (int i = 0; i < N; ++i)
        if (const uint64_t q = key(i)) sm.list[atomicAdd(&sm.count, 1)] = q;
      __syncthreads();
      const int n = sm.count;
      __syncthreads();
      if (n > cand.kept) lp_cut(sm, cand, n, k);
      __syncthreads();
    }
  }
  const int n = sm.count;
  __syncthreads();
  if (n > cand.kept) lp_cut(sm, cand, n, k);
  __syncthreads();  // the list and its length are as the next chunk finds them
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_NT, LP_CTAS) logprobs_kernel(Logprobs a, int vecs_per_cta, int row0, int last) {
  constexpr int N = LpVec<T>::N, U = LpVec<T>::U;
  extern __shared__ __align__(16) uint8_t raw[];
  LpSmem& sm = *reinterpret_cast<LpSmem*>(raw);
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int64_t row = row0 + blockIdx.x / split;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Shared memory of another CTA may be written once that CTA is known to have begun: each says so
  // here, and waits for the others just before its first such write.
  if (split > 1) lp_cluster_arrive();
  if (!last) pdl_launch_dependents();
  const T* x0 = static_cast<const T*>(a.logits) + row * a.row_stride;
  // The row in vectors of 16 bytes from its first logit on, whatever its address: a thread's
  // logits, and so the order of every sum, do not depend on it. Loads are aligned; where the
  // row is not, a vector is put together from a thread's load and its neighbour's. What a
  // load would cover outside the row is not read.
  const int lead = (int)((reinterpret_cast<uintptr_t>(x0) % 16) / sizeof(T));  // elements of the first load before the row
  const int vecs = (int)(((int64_t)a.V + N - 1) / N);
  const int v_begin = part * vecs_per_cta, v_end = min(vecs, v_begin + vecs_per_cta);
  const float c = a.scale_log2;
  auto aligned = [&](int v) -> uint4 {
    const int64_t e = (int64_t)v * N - lead;
    if (e >= 0 && e + N <= a.V) return *reinterpret_cast<const uint4*>(x0 + e);
    uint4 r = lp_lowest<T>();
    T* p = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (e + i >= 0 && e + i < a.V) p[i] = x0[e + i];
    return r;
  };
  // a thread's loads of the chunk at v0; most chunks lie inside the row and the CTA's share
  const int v_load = v_end + (lead != 0);  // loads end one later where vectors are put together
  const int v_inner = min(v_load, (int)(((int64_t)a.V + lead) / N));
  auto load = [&](int v0, uint4* x) {
    if (v0 + U * LP_NT <= v_inner && (lead == 0 || v0 > 0)) {
      const uint4* p = reinterpret_cast<const uint4*>(x0 - lead) + v0 + tid;
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = p[u * LP_NT];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * LP_NT + tid;
        x[u] = v < v_load ? aligned(v) : lp_lowest<T>();
      }
    }
  };
  // vector v of the row from the aligned load of the same number and the next one (whole warps)
  auto shifted = [&](const uint4& own, int v) -> uint4 {
    uint4 give = own;
    if (lane == 0) give = v + 32 <= v_end ? aligned(v + 32) : lp_lowest<T>();  // what lane 31 wants
    const int from = (lane + 1) & 31;
    uint32_t w[8] = {own.x, own.y, own.z, own.w, __shfl_sync(0xffffffffu, give.x, from), __shfl_sync(0xffffffffu, give.y, from),
                     __shfl_sync(0xffffffffu, give.z, from), __shfl_sync(0xffffffffu, give.w, from)};
    const int bytes = lead * (int)sizeof(T);
    if (bytes & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (bytes & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = 8 * (bytes & 3);
    return v < v_end ? make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                                  __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits))
                     : lp_lowest<T>();
  };
  LpSums own{-INFINITY, 0.f, 0.f};
  LpCandidates cand{0, 0};
  if (TOP && tid == 0) sm.count = 0;  // (the first chunk begins with a barrier)
  uint4 next[U];
  load(v_begin, next);
  int chunk = 0;
  for (int v0 = v_begin; v0 < v_end; v0 += U * LP_NT, ++chunk) {
    uint4 cur[U];
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = next[u];
    load(v0 + U * LP_NT, next);
    if (lead) {
#pragma unroll
      for (int u = 0; u < U; ++u) cur[u] = shifted(cur[u], v0 + u * LP_NT + tid);
    }
    float mx = lp_top(cur[0], T());
#pragma unroll
    for (int u = 1; u < U; ++u) mx = lp_max_nan(mx, lp_top(cur[u], T()));
    if (mx > own.m) lp_move(own, mx, c);
    const float m = own.m == -INFINITY ? 0.f : own.m;
    const uint64_t less2 = lp_pair(-m, -m), c2 = lp_pair(c, c);
    uint64_t s2 = 0, t2 = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      LpVec<T>::get(cur[u], x);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        uint64_t y2 = lp_mul2(lp_add2(lp_pair(x[i], x[i + 1]), less2), c2);
        float y0, y1;
        lp_unpair(y2, y0, y1);
        const uint64_t e2 = lp_pair(lp_ex2(y0), lp_ex2(y1));
        s2 = lp_add2(s2, e2);
        t2 = lp_fma2(e2, lp_pair(fmaxf(y0, -4096.f), fmaxf(y1, -4096.f)), t2);  // 2^-inf is 0, and 0 its share
      }
    }
    float s0, s1, t0, t1;
    lp_unpair(s2, s0, s1);
    lp_unpair(t2, t0, t1);
    own.s += s0 + s1;
    own.t += t0 + t1;
    if (TOP) {
      if (chunk == 0) {
        lp_top_chunk<T>(sm, cand, cur, x0, a.V, v0, v_end, mx, a.top_k);
      } else {
        // no barrier in an ordinary chunk: warps add what reaches the threshold, and now and
        // then the list is cut and the threshold moves up to it (after 2, 6, 18 and 66 chunks:
        // 2048 x 151936 in 143 us; after 4, 16 and 64: 147; 8, 32 and 128: 154)
        lp_collect<T>(sm, cand.floor_key, cur, a.V, v0, v_end, mx);
        if (chunk == 1 || chunk == 5 || chunk == 17 || chunk == 65) {
          __syncthreads();
          const int n = sm.count;
          if (n > cand.kept && n <= LP_CAP) lp_cut(sm, cand, n, a.top_k);
          __syncthreads();
        }
      }
    }
  }
  if (TOP) {
    __syncthreads();
    cand.kept = sm.count;
    if (sm.count > LP_CAP) {
      // More candidates than the list holds (logits that rise along the row, say): once more over
      // the CTA's share for the alternatives alone, with a threshold of its own for every chunk
      __syncthreads();
      cand = LpCandidates{0, 0};
      if (tid == 0) sm.count = 0;
      __syncthreads();
      for (int v0 = v_begin; v0 < v_end; v0 += U * LP_NT) {
        uint4 cur[U];
        load(v0, cur);
        if (lead) {
#pragma unroll
          for (int u = 0; u < U; ++u) cur[u] = shifted(cur[u], v0 + u * LP_NT + tid);
        }
        float mx = lp_top(cur[0], T());
#pragma unroll
        for (int u = 1; u < U; ++u) mx = lp_max_nan(mx, lp_top(cur[u], T()));
        lp_top_chunk<T>(sm, cand, cur, x0, a.V, v0, v_end, mx, a.top_k);
      }
    }
  }
  // ---- the CTA's sums and best, then the row's ------------------------------------
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums b;
    b.m = __shfl_xor_sync(0xffffffffu, own.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, own.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, own.t, o);
    own = lp_join(own, b, c);
  }
  if (lane == 0) sm.warps[warp] = own;
  __syncthreads();
  own = sm.warps[0];
#pragma unroll
  for (int w = 1; w < LP_WARPS; ++w) own = lp_join(own, sm.warps[w], c);
  if (TOP) cand.kept = lp_keep_best(sm.list, cand.kept, a.top_k);
  if (split > 1) {
    lp_cluster_wait();
    LpSmem* first = cluster.map_shared_rank(&sm, 0);
    if (tid == 0) first->parts[part] = own;
    if (TOP)
      for (int i = tid; i < a.top_k; i += LP_NT) first->lists[part * a.top_k + i] = i < cand.kept ? sm.list[i] : 0;
    cluster.sync();
    if (last) pdl_wait();  // (below, for the others)
    if (part != 0) return;
    own = sm.parts[0];
    for (int p = 1; p < split; ++p) own = lp_join(own, sm.parts[p], c);
    if (TOP) {
      for (int i = tid; i < split * a.top_k; i += LP_NT) sm.list[i] = sm.lists[i];
      lp_keep_best(sm.list, split * a.top_k, a.top_k);
    }
  }
  // The second launch of a call ends after the first: what comes after on the stream takes
  // its end for the end of both.
  if (last && split == 1) pdl_wait();
  const float ls = log2f(own.s), ln2 = 0.69314718055994531f;
  auto logprob = [&](float v) { return fmaf(v - own.m, a.inv_temperature, -ln2 * ls); };
  if (tid == 0) a.entropy[row] = ln2 * (ls - own.t / own.s);
  for (int i = tid; i < a.C; i += LP_NT) {
    const int64_t at = a.tokens[row * a.C + i];
    a.logprob[row * a.C + i] = at >= 0 && at < a.V ? logprob(to_f(x0[at])) : -INFINITY;
  }
  if (TOP && tid < a.top_k) {
    const uint64_t key = sm.list[tid];
    a.top_tokens[row * a.top_k + tid] = (int)~(uint32_t)key;
    a.top_logprobs[row * a.top_k + tid] = logprob(lp_value(key));
  }
}

// Rows [row0, row0 + rows), each by a cluster of `split` CTAs; beside the launch before this
// one, if it is the second of a call.
template <typename T, bool TOP>
int lp_rows(const Logprobs& a, int64_t row0, int64_t rows, int split, bool second, cudaStream_t st) {
  constexpr int N = LpVec<T>::N;
  const int per = (int)((((int64_t)a.V + N - 1) / N + split - 1) / split);
  auto kern = logprobs_kernel<T, TOP>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = second ? 2 : 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(rows * split));
  cfg.blockDim = dim3(LP_NT);
  cfg.dynamicSmemBytes = sizeof(LpSmem);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, per, (int)row0, (int)second);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  return check_launch("token_logprobs");
}

template <typename T, bool TOP>
int lp_launch(const Logprobs& a, cudaStream_t st) {
  // Whole waves of CTAs take a row each; the rows that are left are split over clusters so
  // that their wave is full and short. They go in a launch of their own, which starts as
  // the first one's CTAs leave (2048 x 151936 bf16, top 20: 178 -> 162 us, with the CTAs of 256 threads of then).
  const int64_t slots = (int64_t)LP_CTAS * num_sms_current_device();
  if (a.N > 0x7fffffff - slots) return fail(DROPKV_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  const int64_t whole = a.N / slots * slots;
  if (whole) {
    const int rc = lp_rows<T, TOP>(a, 0, whole, 1, false, st);
    if (rc || whole == a.N) return rc;
  }
  // CTAs a row: by the waves of CTAs and what one costs, its chunks and what its start and end
  // take, about 8 chunks with alternatives and 2 without. A CTA takes one chunk at least.
  constexpr int N = LpVec<T>::N, U = LpVec<T>::U;
  const int64_t vecs = ((int64_t)a.V + N - 1) / N, rest = a.N - whole;
  int split = 1;
  double best = 1e30;
  for (int s = 1; s <= LP_MAX_S; s *= 2) {
    const int64_t share = (vecs + s - 1) / s;
    if (s > 1 && share < U * LP_NT) break;
    const double cost = (double)((rest * s + slots - 1) / slots) * ((double)share / (U * LP_NT) + (TOP ? 8 : 2));
    if (cost < best) best = cost, split = s;
  }
  return lp_rows<T, TOP>(a, whole, rest, split, whole > 0, st);
}

}  // namespace

size_t token_logprobs_workspace_size(int64_t N, int V, int top_k) {
  (void)N, (void)V, (void)top_k;
  return 0;
}

int launch_token_logprobs(const Logprobs& a, int dtype, void* ws, cudaStream_t st) {
  (void)ws;
  if (dtype == DROPKV_DTYPE_BF16)
    return a.top_k ? lp_launch<__nv_bfloat16, true>(a, st) : lp_launch<__nv_bfloat16, false>(a, st);
  if (dtype == DROPKV_DTYPE_F16) return a.top_k ? lp_launch<__half, true>(a, st) : lp_launch<__half, false>(a, st);
  return a.top_k ? lp_launch<float, true>(a, st) : lp_launch<float, false>(a, st);
}

}  // namespace dropkv
