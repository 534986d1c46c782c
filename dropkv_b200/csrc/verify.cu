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
// 2^x in 64 bits: x = k / 64 + r, a table of 2^(j / 64) and the exponential's series in r ln 2 (|r| <= 2^-7: five terms leave
// 4e-14 of the value).
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.cuh"

namespace dropkv {
namespace {

namespace cg = cooperative_groups;

constexpr int VF_NT = 256;        // threads of a chunk's CTA
constexpr int VF_AHEAD = 4;       // vectors of a thread on their way
constexpr int VD_WARPS = 16, VD_NT = 32 * VD_WARPS;
constexpr int VD_CTAS = 8;        // of a cluster
constexpr int VD_SEGS = VD_CTAS * VD_WARPS;
constexpr int VF_MAX_T = 256;
// fp32's sums and exponentials are off by less than this in the logarithm of a ratio (sums of positive terms over 256 threads and
// up to 32 chunks: 2^-17 at most; 2^x within 2^-22).
constexpr double kVfUnsure = 4e-5;
constexpr double kVfLeast = -745.0;  // log of a probability under what 64 bits hold

struct VfArgs {
  const char* target;  // [B, T + 1, V], strides in elements
  int64_t t_sb, t_si;
  const char* draft;  // [B, T, V] or nullptr
  int64_t d_sb, d_si;
  const int64_t* tokens;   // [B, T]
  const float* uniforms;   // [B, T + 1]
  int B, T, V, S, chunk;   // S chunks of a row
  float c, c_lo;           // log2(e) / tau in two parts, both positive: -inf times them stays -inf
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
// has a maximum and a sum of its own. (Differences first, then the product in two parts: exponents are off by little of
// themselves, however far from zero the logits are.)
template <typename T>
__global__ void __launch_bounds__(VF_NT) verify_rows_kernel(const __grid_constant__ VfArgs a) {
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
  auto add = [&](const float* y, int n) {  // n elements
    float top = y[0];
#pragma unroll
    for (int e = 1; e < n; ++e) top = fmaxf(top, y[e]);
    if (top > m) {
      s *= m == -INFINITY ? 0.f : vf_ex2((m - top) * a.c);
      m = base = top;
    }
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float d = y[e] - base;
      s += vf_ex2(fmaf(d, a.c_lo, d * a.c));
    }
  };
  const T* p = x + e0;
  const int n = e1 - e0;
  const int head = n <= 0 ? 0 : min(n, (int)((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
  const int vecs = (n - head) / N, tail = n - head - vecs * N;
  for (int v0 = tid; v0 < vecs; v0 += VF_NT * VF_AHEAD) {
    uint4 w[VF_AHEAD];
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u)
      if (v0 + u * VF_NT < vecs) w[u] = __ldcs(reinterpret_cast<const uint4*>(p + head) + v0 + u * VF_NT);
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u) {
      if (v0 + u * VF_NT >= vecs) continue;
      const T* t = reinterpret_cast<const T*>(&w[u]);
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = to_f(t[e]);
      add(y, N);
    }
  }
  if (tid < head + tail) {
    const float y = to_f(p[tid < head ? tid : n - tail + (tid - head)]);
    add(&y, 1);
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

struct VdSmem {
  double table[64];
  double seg[2][VD_WARPS];             // sums of this CTA's segments: of p's row, of q's
  double all[2][VD_SEGS];              // of all
  double sub[VD_WARPS];
  double ratio[VF_MAX_T];              // log(p_i(x_i) / q_i(x_i)), +-inf; NaN where a row is none
  float mp[VF_MAX_T + 1], mq[VF_MAX_T + 1];
  int found;
};

// A cluster has a sequence; a warp a segment of the vocabulary, VD_SEGS of them in order.
template <typename T>
__global__ void __launch_bounds__(VD_NT) verify_draw_kernel(const __grid_constant__ VfArgs a) {
  __shared__ VdSmem sm;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / VD_CTAS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 64) sm.table[tid] = exp2(tid / 64.0);
  const double ln2 = 0.69314718055994530942;
  // 2^y for y <= 0; NaN stays
  auto pow2 = [&](double y) -> double {
    const double shift = 6755399441055744.0 / 64;  // 1.5 * 2^52 / 64: sums with it are multiples of 1 / 64
    const double t = y + shift;
    const int k = __double2loint(t);
    const double r = (y - (t - shift)) * ln2;
    const double f = fma(r, fma(r, fma(r, fma(r, 1.0 / 24, 1.0 / 6), 0.5), 1.0), 1.0);
    const double z = sm.table[k & 63] * f;
    // (under 2^-1000 nothing is left to count)
    const double scaled = __hiloint2double(__double2hiint(z) + (k >> 6) * (1 << 20), __double2loint(z));
    return y >= -1000.0 ? scaled : (y < -1000.0 ? 0.0 : y);
  };
  pdl_wait();
  __syncthreads();
  // ---- the rows' maxima and sums, and the drafted tokens' ratios -----------------
  for (int i = warp; i <= a.T; i += VD_WARPS) {
    double lse[2] = {0.0, 0.0};
    float tops[2] = {0.f, 0.f};
    const bool two = a.draft && i < a.T;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k && !two) break;
      const float2 w = lane < a.S ? a.part[vf_index(a, b, i, k) * a.S + lane] : make_float2(-INFINITY, 0.f);
      float m = w.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      float s = w.x == -INFINITY ? w.y : w.y * vf_ex2((w.x - m) * a.c);
      if (m == INFINITY) s = NAN;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      tops[k] = m;
      lse[k] = s > 0.f && s <= 3.4e38f ? log((double)s) : NAN;  // (a sum of 0: nothing but -inf)
    }
    if (lane == 0) {
      sm.mp[i] = isnan(lse[0]) ? NAN : tops[0];
      sm.mq[i] = isnan(lse[1]) ? NAN : tops[1];
      if (i < a.T) {
        const int64_t x = a.tokens[(int64_t)b * a.T + i];
        double d = 0.0;
        float prob = 0.f;
        if (x >= 0 && x < a.V) {
          const double per = a.c64 * ln2;  // 1 / tau
          double lp = ((double)to_f(vf_row<T>(a, b, i, false)[x]) - tops[0]) * per - lse[0];
          double lq = two ? ((double)to_f(vf_row<T>(a, b, i, true)[x]) - tops[1]) * per - lse[1] : 0.0;
          // what 64 bits hold no number for is 0: a token with p of 0 is not accepted, whatever q says
          if (lp < kVfLeast) lp = -INFINITY;
          if (lq < kVfLeast) lq = -INFINITY;
          d = lp == -INFINITY && !isnan(lq) ? -INFINITY : lp - lq;
          prob = d >= 0.0 ? 1.f : (float)exp(d);
          if (isnan(d)) prob = NAN;
        }
        sm.ratio[i] = d;
        if (rank == 0) a.prob[(int64_t)b * a.T + i] = prob;
      }
    }
  }
  __syncthreads();
  const int seg = (a.V + VD_SEGS - 1) / VD_SEGS, lo = min(a.V, (rank * VD_WARPS + warp) * seg), hi = min(a.V, lo + seg);
  // sums over a warp's segment, for all of the cluster: term(e) of each of its elements
  auto over_segments = [&](int which, auto sum_of) -> double {
    const double mine = sum_of(lo, hi);
    if (lane == 0) sm.seg[which][warp] = mine;
    cluster.sync();
    if (tid < VD_SEGS) sm.all[which][tid] = cluster.map_shared_rank(&sm, tid / VD_WARPS)->seg[which][tid % VD_WARPS];
    cluster.sync();  // (who reads a CTA's sums is done with them before they change, or the CTA ends)
    double all = 0.0;
#pragma unroll 4
    for (int i = 0; i < VD_SEGS; ++i) all += sm.all[which][i];
    return all;
  };
  auto warp_sum = [&](double s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  // sum of f(x_e) (and y_e) over elements [at, end) by the lanes of a warp
  auto walk = [&](const T* x, const T* y, int at, int end, auto f) {
    double s = 0.0;
    for (int e = at + lane; e < end; e += 32 * 4) {
      float u[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u[k] = v[k] = -INFINITY;
        if (e + 32 * k < end) {
          u[k] = to_f(x[e + 32 * k]);
          if (y) v[k] = to_f(y[e + 32 * k]);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + 32 * k < end) s += f(e + 32 * k, u[k], v[k]);
    }
    return warp_sum(s);
  };
  auto weight = [&](float x, float m) { return pow2(((double)x - m) * a.c64); };
  auto sum_row = [&](const T* x, float m, int which) {
    return over_segments(which, [&](int at, int end) {
      return walk(x, static_cast<const T*>(nullptr), at, end, [&](int, float u, float) { return weight(u, m); });
    });
  };
  // ---- which are accepted ----------------------------------------------------------
  int n = 0;
  bool rejected = false, none = false;
  for (; n < a.T; ++n) {
    const int64_t x = a.tokens[(int64_t)b * a.T + n];
    if (x < 0 || x >= a.V) break;
    double d = sm.ratio[n];
    if (isnan(d)) {
      none = true;
      break;
    }
    const double lu = log((double)a.uniforms[(int64_t)b * (a.T + 1) + n]);
    if (fabs(lu - d) < kVfUnsure) {  // (the same in every thread of the cluster)
      const T* xp = vf_row<T>(a, b, n, false);
      double lp = ((double)to_f(xp[x]) - sm.mp[n]) * a.c64 * ln2 - log(sum_row(xp, sm.mp[n], 0)), lq = 0.0;
      if (a.draft) {
        const T* xq = vf_row<T>(a, b, n, true);
        lq = ((double)to_f(xq[x]) - sm.mq[n]) * a.c64 * ln2 - log(sum_row(xq, sm.mq[n], 0));
      }
      d = lp - lq;
    }
    if (!(lu < d)) {
      rejected = true;
      break;
    }
  }
  const T* xp = vf_row<T>(a, b, n, false);
  const float mp = sm.mp[n], mq = rejected && a.draft ? sm.mq[n] : 0.f;
  none = none || isnan(mp) || isnan(mq);
  if (none) {
    if (rank == 0 && tid == 0) {
      a.accepted[b] = n;
      a.next_token[b] = -1;
    }
    return;  // (all of the cluster)
  }
  // ---- the token after them --------------------------------------------------------
  const T* xq = rejected && a.draft ? vf_row<T>(a, b, n, true) : nullptr;
  const int64_t out = rejected && !a.draft ? a.tokens[(int64_t)b * a.T + n] : -1;  // q's only word
  double zp = sum_row(xp, mp, 0), zq = 1.0;
  if (xq) zq = sum_row(xq, mq, 1);
  const double ip = 1.0 / zp, iq = 1.0 / zq;
  bool residual = rejected;
  auto term = [&](int e, float u, float v) -> double {
    const double p = weight(u, mp) * ip;
    if (!residual) return p;
    if (!xq) return e == out ? 0.0 : p;
    return fmax(p - weight(v, mq) * iq, 0.0);
  };
  auto sum_terms = [&](int at, int end) { return walk(xp, residual ? xq : static_cast<const T*>(nullptr), at, end, term); };
  double whole = over_segments(0, sum_terms);
  if (residual && !(whole > 0.0)) {  // p nowhere above q (they are equal, and a rounding rejected): p itself
    residual = false;
    whole = over_segments(0, sum_terms);
  }
  const double least = (double)a.uniforms[(int64_t)b * (a.T + 1) + a.T] * whole;
  // the segment whose sum passes it; the last that has any weight, where rounding lets none
  int at_seg = -1, last = 0;
  double before = 0.0, upto = 0.0;
  for (int i = 0; i < VD_SEGS; ++i) {
    const double w = sm.all[0][i];
    if (w > 0.0) last = i;
    if (at_seg < 0 && upto + w > least) {
      at_seg = i;
      before = upto;
    }
    upto += w;
  }
  if (at_seg < 0) {
    at_seg = last;
    before = 0.0;
    for (int i = 0; i < last; ++i) before += sm.all[0][i];
  }
  if (at_seg / VD_WARPS != rank) return;  // (all have read what they read of one another)
  // this CTA's sixteen warps take parts of the segment, then one its elements
  const int s0 = min(a.V, at_seg * seg), s1 = min(a.V, s0 + seg), part = (s1 - s0 + VD_WARPS - 1) / VD_WARPS;
  const int w0 = min(s1, s0 + warp * part), w1 = min(s1, w0 + part);
  const double mine = sum_terms(w0, w1);
  if (lane == 0) sm.sub[warp] = mine;
  if (tid == 0) sm.found = -1;
  __syncthreads();
  int at_part = -1;
  last = 0;
  upto = before;
  double start = before;
  for (int i = 0; i < VD_WARPS; ++i) {
    const double w = sm.sub[i];
    if (w > 0.0) last = i;
    if (at_part < 0 && upto + w > least) {
      at_part = i;
      start = upto;
    }
    upto += w;
  }
  if (at_part < 0) {
    at_part = last;
    start = before;
    for (int i = 0; i < last; ++i) start += sm.sub[i];
  }
  if (warp == at_part) {
    int pick = -1, highest = -1;  // the last element with any weight
    double run = start;
    for (int e0 = w0; e0 < w1 && pick < 0; e0 += 32) {
      const int e = e0 + lane;
      double w = 0.0;
      if (e < w1) w = term(e, to_f(xp[e]), residual && xq ? to_f(xq[e]) : -INFINITY);
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
  const int64_t most = std::max<int64_t>(1, V / 2048), least = (V + 65535) / 65536;
  return (int)std::min<int64_t>(32, std::max(std::min(want, most), least));
}

template <typename T>
int vf_launch(const VfArgs& a, int64_t rows, cudaStream_t st) {
  if (rows * a.S > 0x7fffffff || (int64_t)a.B * VD_CTAS > 0x7fffffff)
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
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = VD_CTAS;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(a.B * VD_CTAS);
  cfg.blockDim = dim3(VD_NT);
  e = cudaLaunchKernelEx(&cfg, verify_draw_kernel<T>, a);
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
  a.c64 = 1.4426950408889634 / (double)q.temperature;
  a.c = (float)a.c64;
  if ((double)a.c > a.c64) a.c = std::nextafter(a.c, 0.f);
  a.c_lo = std::max((float)(a.c64 - (double)a.c), FLT_MIN);
  a.part = static_cast<float2*>(ws);
  a.accepted = q.accepted, a.next_token = q.next_token, a.prob = q.prob;
  if (dtype == DROPKV_DTYPE_BF16) return vf_launch<__nv_bfloat16>(a, rows, st);
  return dtype == DROPKV_DTYPE_F16 ? vf_launch<__half>(a, rows, st) : vf_launch<float>(a, rows, st);
}

}  // namespace dropkv
