// Verification of drafted tokens against the target's probabilities, by given random numbers.
//
// With p_i = softmax(target_i / tau), q_i = softmax(draft_i / tau) (without draft logits: all of it at
// the drafted token), token x_i is accepted while u_i q_i(x_i) < p_i(x_i), in order. At the first
// one rejected, n, the token after the accepted ones is drawn from max(p_n - q_n, 0), else, after the
// last drafted one, from p_n: the first t whose cumulative sum passes u_T times the whole.
//
// Two launches. The first takes every row once, in chunks: a maximum and a sum of exponentials in
// fp32 (HBM bounds it). The second has a cluster of CTAs for each sequence: it joins the
// chunks, decides, and draws. A token is found by a sum over a whole vocabulary, among steps of which many are
// smaller than fp32's error in it: 150 thousand words would answer another token in a hundredth of
// the draws. So the drawing's exponentials and sums are in 64 bits, of the one row that is drawn
// from; and where fp32 cannot tell whether a token is accepted, its rows' sums are taken
// in 64 bits too.
//
// Measured: 64 drafts of up to 7 tokens over 151936 words in bf16, 292 MB: 118 us, of which the first launch takes 55 (81% of a
// copy's rate) and the second 66; 4 of 5 tokens over 50257 words 20, 16 of 4 over 32000 without draft logits 14, most of it the
// second one's chain (join, sums shared over the cluster, a second look where q has a row, the search).
// 2^x in 64 bits: a table of 2^(j / 2048), made by each CTA, and three terms of the exponential's series for what is left of x.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace dropkv {
namespace {

namespace cg = cooperative_groups;

constexpr int VF_NT = 256;        // threads of a chunk's CTA
constexpr int VF_AHEAD = 4;       // vectors of a thread on their way
constexpr int VD_SEGS = 256;      // segments of a row, at most
constexpr int VF_MAX_T = 256;
// fp32's sums and exponentials are off by less than this in the logarithm of a ratio (sums of positive terms over 256 threads and
// up to 32 chunks: 2^-17 at most; 2^x within 2^-22, of exponents off by 2^-23 of themselves).
constexpr float kVfUnsure = 4e-5f;
// Log of a probability under what 64 bits hold: that is 0, and a token with p of 0 is not accepted, whatever q says.
constexpr double kVfLeast = -745.0;

struct VfArgs {
  const char* target;  // [B, T + 1, V], strides in elements
  int64_t t_sb, t_si;
  const char* draft;  // [B, T, V] or nullptr
  int64_t d_sb, d_si;
  const int64_t* tokens;   // [B, T]
  const float* uniforms;   // [B, T + 1]
  int B, T, V, S, chunk;   // S chunks of a row
  float c;                 // log2(e) / tau
  double c64;
  float2* part;            // [rows][S]: maximum, sum of 2^((x - maximum) c)
  int64_t* accepted;
  int64_t* next_token;
  float* prob;             // [B, T]
};

__device__ __forceinline__ float vf_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t vf_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void vf_unpair(uint64_t r, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ float vf_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t vf_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t vf_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <typename T>
struct VfVec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Rows: b's T + 1 of the target, then b's T of the draft.
template <typename T>
__device__ __forceinline__ const T* vf_row(const VfArgs& a, int b, int i, bool draft) {
  return draft ? reinterpret_cast<const T*>(a.draft) + b * a.d_sb + i * a.d_si
               : reinterpret_cast<const T*>(a.target) + b * a.t_sb + i * a.t_si;
}
__device__ __forceinline__ int64_t vf_index(const VfArgs& a, int b, int i, bool draft) {
  return draft ? (int64_t)a.B * (a.T + 1) + (int64_t)b * a.T + i : (int64_t)b * (a.T + 1) + i;
}

// A chunk of a row: elements [e0, e1), the whole vectors of 16 bytes between them by all threads, the ends by some. Each thread
// has a reference (near its maximum) and a sum of its own. (Differences first, then the product: exponents are off by little of
// themselves, however far from zero the logits are.)
template <typename T>
__global__ void __launch_bounds__(VF_NT, 6) verify_rows_kernel(const __grid_constant__ VfArgs a) {
  constexpr int N = VfVec<T>::N;
  __shared__ float ms[VF_NT / 32], ss[VF_NT / 32];
  const int64_t row = blockIdx.x / a.S;
  const int part = blockIdx.x % a.S, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t targets = (int64_t)a.B * (a.T + 1);
  const bool draft = row >= targets;
  const int64_t r = draft ? row - targets : row;
  const int per = draft ? a.T : a.T + 1;
  const T* x = vf_row<T>(a, (int)(r / per), (int)(r % per), draft);
  const int e0 = part * a.chunk, e1 = min(e0 + a.chunk, a.V);
  pdl_launch_dependents();
  pdl_wait();
  float m = -INFINITY, base = 0.f, s = 0.f;
  auto raise = [&](float top) {  // (a reference that is a little low does as well: weights up to 2^16)
    if ((top - m) * a.c > 16.f || m == -INFINITY) {
      s *= m == -INFINITY ? 1.f : vf_ex2((m - top) * a.c);
      m = top;
      base = top == -INFINITY ? 0.f : top;
    }
  };
  const T* p = x + e0;
  const int n = e1 - e0;
  const int head = n <= 0 ? 0 : min(n, (int)((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
  const int vecs = (n - head) / N, tail = n - head - vecs * N;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head) + tid;
  const uint64_t c2 = vf_pair(a.c, a.c);
  auto take = [&](const uint4& w) {
    const T* t = reinterpret_cast<const T*>(&w);
    float y[N], top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = to_f(t[e]);
#pragma unroll
    for (int e = 0; e < N; e += 2) top = vf_max3(top, y[e], y[e + 1]);
    raise(top);
    const uint64_t base2 = vf_pair(-base, -base);
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float f, g;
      vf_unpair(vf_mul2(vf_add2(vf_pair(y[e], y[e + 1]), base2), c2), f, g);
      sum = vf_add2(sum, vf_pair(vf_ex2(f), vf_ex2(g)));
    }
    float f, g;
    vf_unpair(sum, f, g);
    s += f + g;
  };
  constexpr int STEP = VF_NT * VF_AHEAD;
  uint4 w[VF_AHEAD];
  int v = tid;
  for (; v + STEP - VF_NT < vecs; v += STEP) {
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u) w[u] = __ldcs(pv + (v - tid) + u * VF_NT);
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u) take(w[u]);
  }
  for (; v < vecs; v += VF_NT) take(__ldcs(pv + (v - tid)));
  if (tid < head + tail) {
    const float y = to_f(p[tid < head ? tid : n - tail + (tid - head)]);
    raise(y);
    s += vf_ex2((y - base) * a.c);
  }
  auto join = [&](float om, float os) {
    const float mn = fmaxf(m, om);
    if (mn == -INFINITY) {
      s += os;  // (NaN stays)
      return;
    }
    s = s * (m == mn ? 1.f : vf_ex2((m - mn) * a.c)) + os * (om == mn ? 1.f : vf_ex2((om - mn) * a.c));
    m = mn;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    join(om, os);
  }
  if (lane == 0) ms[warp] = m, ss[warp] = s;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < VF_NT / 32; ++w) join(ms[w], ss[w]);
    a.part[row * a.S + part] = make_float2(m, s);
  }
}

constexpr int VD_TABLE = 2048;  // steps of 2^x's table: 2^x = 2^(k / 2048) 2^r, |r| <= 2^-12, whose series' fourth term is 4e-17

enum { VD_ACCEPT = 0, VD_REJECT, VD_UNSURE, VD_END, VD_NONE };

template <int WARPS>
struct VdSmem {
  double table[VD_TABLE];
  double root[96];          // 2^(i / 32), 2^(i / 2048)
  double all[3][VD_SEGS + VD_SEGS / 8];  // all segments' sums, as vd_at says: of p's row, of q's, of what is drawn from them
  double sub[WARPS + WARPS / 8];      // of parts of the segment, likewise
  float mp[VF_MAX_T + 1], mq[VF_MAX_T + 1];
  int8_t what[VF_MAX_T];    // of a drafted token
};

// Log of a probability: of a word's logit over the largest, and the sum of the row's weights.
__device__ __forceinline__ double vf_log(double over, double sum) {
  const double l = over - log(sum);
  return l < kVfLeast ? -INFINITY : l;
}

// Where value i of a list of 256 lies: eight a lane then meet all banks.
__device__ __forceinline__ int vd_at(int i) { return i + (i >> 3); }

// Of n values, at most 256, a lane has eight: their sum, and which is the first to pass `least` by what is summed up to it
// from `start` (the last with any weight, where rounding lets none); `before`: the sum before that one. All lanes get the same.
__device__ __forceinline__ double vd_sum(const double* v, int n, int lane) {
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += 32 * k + lane < n ? v[vd_at(32 * k + lane)] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ int vd_find(const double* v, int n, int lane, double start, double least, double* before) {
  double mine[8], own = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    mine[k] = 8 * lane + k < n ? v[vd_at(8 * lane + k)] : 0.0;
    if (mine[k] > 0.0) last = 8 * lane + k;
    own += mine[k];
  }
  double upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double z = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += z;
  }
  double run = start + (upto - own), at_run = run, last_run = run;
  int at = -1;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (8 * lane + k == last) last_run = run;
    if (at < 0 && mine[k] > 0.0 && run + mine[k] > least) {
      at = 8 * lane + k;
      at_run = run;
    }
    run += mine[k];
  }
  const unsigned past = __ballot_sync(0xffffffffu, at >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
  const int from = past ? __ffs(past) - 1 : 31 - __clz(some | 1u);
  *before = __shfl_sync(0xffffffffu, past ? at_run : last_run, from);
  return max(__shfl_sync(0xffffffffu, past ? at : last, from), 0);
}

// A cluster has a sequence; a warp a segment of the vocabulary, VD_SEGS of them in order. Half of its time is
// 64-bit arithmetic: ten operations for an exponential, two to four of them a word, and the tenth took 3.2 us of the large batch's 66
// when it was added. The rest is the rows' second reading, from L2, the tables, and the waits at the cluster's barriers.
template <typename T, int VD_WARPS>
__global__ void __launch_bounds__(32 * VD_WARPS, 32 / VD_WARPS) verify_draw_kernel(const __grid_constant__ VfArgs a) {
  constexpr int VD_NT = 32 * VD_WARPS;
  __shared__ VdSmem<VD_WARPS> sm;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / ctas, segs = ctas * VD_WARPS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster.barrier_arrive();  // (waited for before the first write to another CTA: it has begun)
  if (tid < 96) sm.root[tid] = exp2(tid < 32 ? tid / 32.0 : (tid - 32) / 2048.0);
  __syncthreads();
  for (int i = tid; i < VD_TABLE; i += VD_NT) sm.table[i] = sm.root[i >> 6] * sm.root[32 + (i & 63)];
  constexpr double LN2 = 0.69314718055994530942;
  // weight of a word: 2^((x - m) c). (Beyond `floor_` below the largest nothing is left to count.)
  const float floor_ = (float)(-1000.0 / a.c64);
  auto weight = [&](float x, float m) -> double {
    const double shift = 6755399441055744.0 / VD_TABLE;  // 1.5 * 2^52 / 2048: sums with it are multiples of 1 / 2048
    const double d = (double)x - m, t = fma(d, a.c64, shift), r = fma(d, a.c64, -(t - shift));
    const int k = __double2loint(t);
    const double z = sm.table[k & (VD_TABLE - 1)] * fma(r, fma(r, fma(r, LN2 * LN2 * LN2 / 6, LN2 * LN2 / 2), LN2), 1.0);
    const double w = __hiloint2double(__double2hiint(z) + (k >> 11) * (1 << 20), __double2loint(z));
    return x - m > floor_ ? w : 0.0;
  };
  pdl_wait();
  __syncthreads();
  // ---- the rows' maxima and sums, and what becomes of the drafted tokens ---------
  const double per = a.c64 * LN2;  // 1 / tau
  for (int i = warp; i <= a.T; i += VD_WARPS) {
    float tops[2] = {0.f, 0.f}, sums[2] = {1.f, 1.f};
    const bool two = a.draft && i < a.T;
    float2 w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w[k] = lane < a.S && (k == 0 || two) ? a.part[vf_index(a, b, i, k) * a.S + lane] : make_float2(-INFINITY, 0.f);
    int64_t x = -1;
    float xp = 0.f, xq = 0.f, u = 0.f;
    if (lane == 0 && i < a.T) {  // (beside the chunks')
      x = a.tokens[(int64_t)b * a.T + i];
      u = a.uniforms[(int64_t)b * (a.T + 1) + i];
      if (x >= 0 && x < a.V) {
        xp = to_f(vf_row<T>(a, b, i, false)[x]);
        if (two) xq = to_f(vf_row<T>(a, b, i, true)[x]);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k && !two) break;
      float m = w[k].x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float s = w[k].x == -INFINITY ? w[k].y : w[k].y * vf_ex2((w[k].x - m) * a.c);
      if (m == INFINITY) s = NAN;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      tops[k] = m;
      sums[k] = s > 0.f && s <= 3.4e38f ? s : NAN;  // (a sum of 0: nothing but -inf)
    }
    if (lane == 0) {
      sm.mp[i] = isnan(sums[0]) ? NAN : tops[0];
      sm.mq[i] = isnan(sums[1]) ? NAN : tops[1];
      if (i < a.T) {
        int what = VD_END;
        float prob = 0.f;
        if (x >= 0 && x < a.V) {
          const double dp = ((double)xp - tops[0]) * per, dq = two ? ((double)xq - tops[1]) * per : 0.0;
          if (isnan(sums[0]) || isnan(sums[1])) {
            what = VD_NONE;
            prob = NAN;
          } else if (dp > -700.0 && dq > -700.0) {  // p / q, without a logarithm (in 64 bits one takes longer than a row's sums)
            const double d = dp - dq;
            const float hi = fminf((float)d, 80.f), e = expf(hi);
            const float ratio = hi == 80.f ? INFINITY : fmaf(e, (float)(d - hi), e) * (sums[1] / sums[0]);
            prob = fminf(ratio, 1.f);
            what = u < ratio ? VD_ACCEPT : VD_REJECT;
            // where fp32 cannot tell; where its range ends, too
            if (ratio < INFINITY && (fabsf(u - ratio) <= kVfUnsure * fmaxf(u, ratio) || fmaxf(u, ratio) < 1e-29f)) what = VD_UNSURE;
          } else {
            const double lp = vf_log(dp, sums[0]), lq = two ? vf_log(dq, sums[1]) : 0.0;
            const double d = lp == -INFINITY ? -INFINITY : lp - lq, lu = log((double)u);
            prob = d >= 0.0 ? 1.f : (float)exp(d);
            what = lu < d ? VD_ACCEPT : VD_REJECT;
            if (fabs(lu - d) < kVfUnsure) what = VD_UNSURE;
          }
        }
        sm.what[i] = (int8_t)what;
        if (rank == 0) a.prob[(int64_t)b * a.T + i] = prob;
      }
    }
  }
  __syncthreads();
  const int seg = (a.V + segs - 1) / segs, lo = min(a.V, (rank * VD_WARPS + warp) * seg), hi = min(a.V, lo + seg);
  // sum of f(e, x_e, y_e) over elements [at, end), by the lanes of a warp
  auto walk = [&](const T* x, const T* y, int at, int end, auto f) {
    constexpr int AHEAD = 8;
    double sums[4] = {0.0, 0.0, 0.0, 0.0};  // (chains of additions side by side)
    auto batch = [&](int e, auto whole) {
      T u[AHEAD], v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (!decltype(whole)::value && e + 32 * k >= end) continue;
        u[k] = x[e + 32 * k];
        if (y) v[k] = y[e + 32 * k];
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (decltype(whole)::value || e + 32 * k < end) sums[k & 3] += f(e + 32 * k, to_f(u[k]), y ? to_f(v[k]) : 0.f);
    };
    int e = at + lane;
    for (; e + 32 * (AHEAD - 1) < end; e += 32 * AHEAD) batch(e, std::true_type());
    batch(e, std::false_type());
    double s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  // A warp's sum of its segment, to every CTA.
  auto share = [&](int which, double s) {
    if (lane < ctas) cluster.map_shared_rank(&sm, lane)->all[which][vd_at(rank * VD_WARPS + warp)] = s;
  };
  // sums of weights of p's row, a word left out, and, unless it is NULL, of q's over the whole vocabulary
  auto sum_rows = [&](const T* x, float mx, int out, const T* y, float my, double* zx, double* zy) {
    double sx = 0.0, sy = 0.0;
    if (VD_WARPS == 16) {  // few words a lane: both rows' on their way at once
      constexpr int AHEAD = 4;
      for (int e0 = lo + lane; e0 < hi; e0 += 32 * AHEAD) {
        T u[AHEAD], v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (e0 + 32 * k >= hi) continue;
          u[k] = x[e0 + 32 * k];
          if (y) v[k] = y[e0 + 32 * k];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (e0 + 32 * k >= hi) continue;
          sx += e0 + 32 * k == out ? 0.0 : weight(to_f(u[k]), mx);
          if (y) sy += weight(to_f(v[k]), my);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sx += __shfl_xor_sync(0xffffffffu, sx, o);
        sy += __shfl_xor_sync(0xffffffffu, sy, o);
      }
    } else {
      sx = walk(x, static_cast<const T*>(nullptr), lo, hi, [&](int e, float u, float) { return e == out ? 0.0 : weight(u, mx); });
      if (y) sy = walk(y, static_cast<const T*>(nullptr), lo, hi, [&](int, float u, float) { return weight(u, my); });
    }
    share(0, sx);
    if (y) share(1, sy);
    cluster.sync();
    *zx = vd_sum(sm.all[0], segs, lane);
    *zy = y ? vd_sum(sm.all[1], segs, lane) : 1.0;
  };
  cluster.barrier_wait();
  // ---- which are accepted ----------------------------------------------------------
  int n = 0, what = VD_END;
  double zp, zq;
  for (; n < a.T; ++n) {
    what = sm.what[n];
    if (what == VD_UNSURE) {  // (the same in every thread of the cluster)
      const int64_t x = a.tokens[(int64_t)b * a.T + n];
      const T *xp = vf_row<T>(a, b, n, false), *xq = a.draft ? vf_row<T>(a, b, n, true) : nullptr;
      sum_rows(xp, sm.mp[n], -1, xq, sm.mq[n], &zp, &zq);
      cluster.sync();  // (all have read these sums before they change)
      const double lp = vf_log(((double)to_f(xp[x]) - sm.mp[n]) * per, zp);
      const double lq = xq ? vf_log(((double)to_f(xq[x]) - sm.mq[n]) * per, zq) : 0.0;
      const bool taken = lp > -INFINITY && log((double)a.uniforms[(int64_t)b * (a.T + 1) + n]) < lp - lq;
      what = taken ? VD_ACCEPT : VD_REJECT;
    }
    if (what != VD_ACCEPT) break;
  }
  const bool rejected = n < a.T && what == VD_REJECT;
  const T *xp = vf_row<T>(a, b, n, false), *xq = rejected && a.draft ? vf_row<T>(a, b, n, true) : nullptr;
  const float mp = sm.mp[n], mq = xq ? sm.mq[n] : 0.f;
  if ((n < a.T && what == VD_NONE) || isnan(mp) || isnan(mq)) {
    if (rank == 0 && tid == 0) {
      a.accepted[b] = n;
      a.next_token[b] = -1;
    }
    return;  // (all of the cluster)
  }
  // ---- the token after them --------------------------------------------------------
  // Drawn from p its weights do as they are, but for the drafted token's where q is 1 at it: the sums are there. From
  // max(p - q, 0), a second look at both rows, by now in L2.
  const int out = rejected && !a.draft ? (int)a.tokens[(int64_t)b * a.T + n] : -1;
  sum_rows(xp, mp, out, xq, mq, &zp, &zq);
  const double iq = zp / zq;  // (in units of p's weights)
  bool both = xq != nullptr;
  auto term = [&](int e, float u, float v) -> double {
    const double w = weight(u, mp);
    if (both) return fmax(fma(-iq, weight(v, mq), w), 0.0);
    return e == out ? 0.0 : w;
  };
  auto sum_terms = [&](int at, int end) { return walk(xp, both ? xq : static_cast<const T*>(nullptr), at, end, term); };
  const double* drawn = sm.all[0];
  double whole = zp;
  if (both) {
    share(2, sum_terms(lo, hi));
    cluster.sync();
    drawn = sm.all[2];
    whole = vd_sum(drawn, segs, lane);
  }
  if (!(whole > 0.0)) {  // p nowhere above q (they are equal, and a rounding rejected): p itself
    if (!both) {
      if (rank == 0 && tid == 0) {
        a.accepted[b] = n;
        a.next_token[b] = out;
      }
      return;
    }
    both = false;
    drawn = sm.all[0];
    whole = zp;
  }
  const double least = (double)a.uniforms[(int64_t)b * (a.T + 1) + a.T] * whole;
  double before, start;
  const int at_seg = vd_find(drawn, segs, lane, 0.0, least, &before);
  if (at_seg / VD_WARPS != rank) return;  // (what others write to a CTA they have written before the last barrier that all passed)
  // this CTA's warps take parts of the segment, then one its elements
  const int s0 = min(a.V, at_seg * seg), s1 = min(a.V, s0 + seg), part = (s1 - s0 + VD_WARPS - 1) / VD_WARPS;
  const double mine = sum_terms(min(s1, s0 + warp * part), min(s1, s0 + (warp + 1) * part));
  if (lane == 0) sm.sub[vd_at(warp)] = mine;
  __syncthreads();
  const int at_part = vd_find(sm.sub, VD_WARPS, lane, before, least, &start);
  if (warp == at_part) {
    int pick = -1, highest = -1;  // the last element with any weight
    double run = start;
    const int w0 = min(s1, s0 + warp * part), w1 = min(s1, w0 + part);
    for (int e0 = w0; e0 < w1 && pick < 0; e0 += 32) {
      const int e = e0 + lane;
      double w = 0.0;
      if (e < w1) w = term(e, to_f(xp[e]), both ? to_f(xq[e]) : -INFINITY);
      const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
      double sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double z = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += z;
      }
      const unsigned past = __ballot_sync(0xffffffffu, w > 0.0 && run + sum > least);
      if (past) pick = e0 + __ffs(past) - 1;
      if (some) highest = e0 + 31 - __clz(some);
      run += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
      a.accepted[b] = n;
      a.next_token[b] = pick >= 0 ? pick : highest;
    }
  }
}

int vf_chunks(int64_t rows, int V) {
  const int64_t want = (8 * (int64_t)num_sms_current_device() + rows - 1) / rows;
  // chunks of 4096 words at least: shorter ones start more CTAs than there is work for (of 2048 words: 50257 words 21.3 us, not 19.6)
  const int64_t most = std::max<int64_t>(1, V / 4096), least = (V + 65535) / 65536;
  return (int)std::min<int64_t>(32, std::max(std::min(want, most), least));
}

template <typename T>
int vf_launch(const VfArgs& a, int64_t rows, cudaStream_t st) {
  if (rows * a.S > 0x7fffffff || (int64_t)a.B * 16 > 0x7fffffff)
    return fail(DROPKV_ERR_UNSUPPORTED, "verify_draft: %lld rows are too many", (long long)rows);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(rows * a.S));
  cfg.blockDim = dim3(VF_NT);
  cudaError_t e = cudaLaunchKernelEx(&cfg, verify_rows_kernel<T>, a);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "verify_draft launch: %s", cudaGetErrorString(e));
  int rc = check_launch("verify_rows");
  if (rc) return rc;
  // Few sequences: 16 CTAs of 16 warps each, all there are. Many: as many CTAs of eight warps as fit at once, four an SM.
  const int sms = num_sms_current_device();
  const bool few = (int64_t)a.B * 8 <= sms;
  int ctas = few ? 16 : 8;
  while (ctas > 1 && (int64_t)a.B * ctas > (few ? sms : 4 * sms)) ctas /= 2;
  auto kern = few ? verify_draw_kernel<T, 16> : verify_draw_kernel<T, 8>;
  static DeviceOnce done;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done.done(dev)) {
    if (cudaFuncSetAttribute(verify_draw_kernel<T, 16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "cannot allow clusters of 16");
    done.mark(dev);
  }
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(a.B * ctas);
  cfg.blockDim = dim3(few ? 512 : 256);
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "verify_draft launch: %s", cudaGetErrorString(e));
  return check_launch("verify_draw");
}

}  // namespace

size_t verify_draft_workspace_size(int B, int T, int V, bool draft) {
  const int64_t rows = (int64_t)B * (T + 1) + (draft ? (int64_t)B * T : 0);
  return align_up((size_t)rows * vf_chunks(rows, V) * sizeof(float2), 256);
}

int launch_verify_draft(const VerifyDraft& q, int dtype, void* ws, cudaStream_t st) {
  VfArgs a;
  const int64_t rows = (int64_t)q.B * (q.T + 1) + (q.draft ? (int64_t)q.B * q.T : 0);
  a.target = static_cast<const char*>(q.target), a.t_sb = q.t_sb, a.t_si = q.t_si;
  a.draft = static_cast<const char*>(q.draft), a.d_sb = q.d_sb, a.d_si = q.d_si;
  a.tokens = q.tokens, a.uniforms = q.uniforms;
  a.B = q.B, a.T = q.T, a.V = q.V;
  a.S = vf_chunks(rows, q.V);
  a.chunk = (q.V + a.S - 1) / a.S;
  a.c64 = 1.4426950408889634 / q.temperature;
  a.c = (float)a.c64;
  a.part = static_cast<float2*>(ws);
  a.accepted = q.accepted, a.next_token = q.next_token, a.prob = q.prob;
  if (dtype == DROPKV_DTYPE_BF16) return vf_launch<__nv_bfloat16>(a, rows, st);
  return dtype == DROPKV_DTYPE_F16 ? vf_launch<__half>(a, rows, st) : vf_launch<float>(a, rows, st);
}

}  // namespace dropkv
