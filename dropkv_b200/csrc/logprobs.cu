// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
// With y = (x - max x) log2(e) / tau, S = sum 2^y and A = sum 2^y y:
// log p(t) = (x_t - max x) / tau - ln2 log2 S, H = ln2 (log2 S - A / S). The maximum is taken off
// before the product, which would overflow for logits at the type's lowest value.
#include "common.cuh"

namespace dropkv {
namespace {

constexpr int LP_NT = 512;
constexpr int LP_WARPS = LP_NT / 32;

// Order of the alternatives: larger logits first (NaN above all), then lower index.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
  const uint32_t k = x != x ? 0xffffffffu : ordered_key(x);
  return ((uint64_t)k << 32) | (uint32_t)~i;
}

template <typename T>
__global__ void __launch_bounds__(LP_NT) logprobs_rows_kernel(Logprobs a) {
  __shared__ float rf[LP_WARPS], rg[LP_WARPS];
  __shared__ uint64_t rk[LP_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(a.logits) + blockIdx.x * a.row_stride;
  float m = -INFINITY;
  for (int i = tid; i < a.V; i += LP_NT) m = fmaxf(m, to_f(x[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) rf[warp] = m;
  __syncthreads();
  for (int w = 0; w < LP_WARPS; ++w) m = fmaxf(m, rf[w]);
  __syncthreads();
  float s = 0.f, t = 0.f;
  for (int i = tid; i < a.V; i += LP_NT) {
    const float y = (to_f(x[i]) - m) * a.scale_log2, e = exp2f(y);  // NaN if the maximum is infinite
    s += e;
    t = fmaf(e, y < -1000.f ? 0.f : y, t);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0) rf[warp] = s, rg[warp] = t;
  __syncthreads();
  s = t = 0.f;
  for (int w = 0; w < LP_WARPS; ++w) s += rf[w], t += rg[w];
  const float ls = log2f(s), ln2 = 0.69314718055994531f;
  auto logprob = [&](float v) { return fmaf(v - m, a.inv_temperature, -ln2 * ls); };
  if (tid == 0) a.entropy[blockIdx.x] = ln2 * (ls - t / s);
  for (int c = tid; c < a.C; c += LP_NT) {
    const int64_t at = a.tokens[(int64_t)blockIdx.x * a.C + c];
    a.logprob[(int64_t)blockIdx.x * a.C + c] = at >= 0 && at < a.V ? logprob(to_f(x[at])) : -INFINITY;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    for (int i = tid; i < a.V; i += LP_NT) {
      const uint64_t key = lp_key(to_f(x[i]), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) rk[warp] = best;
    __syncthreads();
    for (int w = 0; w < LP_WARPS; ++w) best = rk[w] > best ? rk[w] : best;
    last = best;
    if (tid == 0) {
      const int i = (int)~(uint32_t)best;
      a.top_tokens[(int64_t)blockIdx.x * a.top_k + k] = i;
      a.top_logprobs[(int64_t)blockIdx.x * a.top_k + k] = logprob(to_f(x[i]));
    }
  }
}

}  // namespace

size_t token_logprobs_workspace_size(int64_t N, int V, int top_k) {
  (void)N, (void)V, (void)top_k;
  return 0;
}

int launch_token_logprobs(const Logprobs& a, int dtype, void* ws, cudaStream_t st) {
  (void)ws;
  if (dtype == DROPKV_DTYPE_BF16)
    logprobs_rows_kernel<__nv_bfloat16><<<(int)a.N, LP_NT, 0, st>>>(a);
  else if (dtype == DROPKV_DTYPE_F16)
    logprobs_rows_kernel<__half><<<(int)a.N, LP_NT, 0, st>>>(a);
  else
    logprobs_rows_kernel<float><<<(int)a.N, LP_NT, 0, st>>>(a);
  return check_launch("token_logprobs");
}

}  // namespace dropkv
