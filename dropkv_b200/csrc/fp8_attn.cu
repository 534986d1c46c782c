// Attention over a paged cache held in 8 bits: for token i of sequence b and query head h,
// O = sum_j softmax_j(scale q . k8_j sk_j) v8_j sv_j over the rows j that it sees, with the
// scales sk and sv of the rows' pages.
#include <algorithm>

#include "fp8_attn.cuh"

namespace dropkv {
namespace {

constexpr int FA_NT = 128;

template <typename T>
__device__ __forceinline__ T fa_from(float x);
template <>
__device__ __forceinline__ __half fa_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 fa_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float fa_widen(uint8_t x) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3))); }

// A CTA has one query row and takes 128 rows of the cache at a time, a thread a row for the
// logits and a column for the output.
template <typename T, int D>
__global__ void __launch_bounds__(FA_NT) attention_fp8_row_kernel(const __grid_constant__ AttnFp8 a) {
  __shared__ float q[D], w[FA_NT], red[FA_NT / 32];
  __shared__ int64_t at[FA_NT];
  __shared__ float sv[FA_NT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const int i = (int)(row % a.T), hq = (int)(row / a.T % a.Hq), b = (int)(row / a.T / a.Hq), h = hq / (a.Hq / a.Hkv);
  if (tid < D) q[tid] = to_f(static_cast<const T*>(a.q)[b * a.q_sb + hq * a.q_sh + i * a.q_ss + tid * a.q_sd]) * a.scale;
  const int len = max(a.cache_lens[b], 0), keys = (int)min((int64_t)len + a.T, (int64_t)a.cap);
  const uint8_t* mr = a.mask ? a.mask + b * a.mask_sb + i * a.mask_sr : nullptr;
  int depth = i;
  if (mr) {
    depth = -1;
    for (int n = 0; n < a.T; ++n) depth += mr[n * a.mask_sc] != 0;
    depth = max(depth, 0);
  }
  const int64_t first = a.window ? (int64_t)len + depth - a.window + 1 : 0;
  auto over_cta = [&](float x, bool sum) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, o);
      x = sum ? x + y : fmaxf(x, y);
    }
    __syncthreads();
    if (lane == 0) red[warp] = x;
    __syncthreads();
    x = red[0];
    for (int k = 1; k < FA_NT / 32; ++k) x = sum ? x + red[k] : fmaxf(x, red[k]);
    return x;
  };
  float m = -INFINITY, l = 0.f, o = 0.f;
  __syncthreads();
  for (int j0 = 0; j0 < keys; j0 += FA_NT) {
    const int j = j0 + tid;
    float s = -INFINITY;
    int64_t v_at = -1;
    if (j < keys) {
      bool see = j < a.sinks || j >= first || (mr && j >= len);
      if (j >= len) see = see && (mr ? mr[(j - len) * a.mask_sc] != 0 : j - len <= i);
      const int page = see ? a.table[(int64_t)b * a.max_blocks + j / a.pool.block] : -1;
      if (page >= 0 && page < a.pool.n_pages) {
        const uint8_t* k = static_cast<const uint8_t*>(a.pool.k) + page * a.pool.k_s0 + h * a.pool.k_sh + (j % a.pool.block) * a.pool.k_st;
        float x = 0.f;
        for (int d = 0; d < D; ++d) x = fmaf(q[d], fa_widen(k[d]), x);
        s = x * a.pool.k_scale[page * a.pool.ks_s0 + h * a.pool.ks_sh];
        v_at = page * a.pool.v_s0 + h * a.pool.v_sh + (j % a.pool.block) * a.pool.v_st;
        sv[tid] = a.pool.v_scale[page * a.pool.vs_s0 + h * a.pool.vs_sh];
      }
    }
    at[tid] = v_at;
    const float mn = fmaxf(m, over_cta(s, false)), ref = mn == -INFINITY ? 0.f : mn;
    const float f = m == mn ? 1.f : expf(m - ref), p = v_at < 0 ? 0.f : expf(s - ref);
    m = mn;
    l = l * f + over_cta(p, true);
    o *= f;
    w[tid] = p;
    __syncthreads();
    if (tid < D) {
      for (int n = 0; n < FA_NT; ++n)
        if (at[n] >= 0) o = fmaf(w[n] * sv[n], fa_widen(static_cast<const uint8_t*>(a.pool.v)[at[n] + tid]), o);
    }
    __syncthreads();
  }
  if (tid < D) static_cast<T*>(a.out)[row * D + tid] = fa_from<T>(l == 0.f ? 0.f : o / l);
}

constexpr int FM_NT = 256;
constexpr int FM_AHEAD = 4;  // partials on their way at once

// Joins the partials of the segments that fell into several CTAs. Grid: (CTAs before it, groups of
// eight rows); a warp has a row, a lane four of its columns. With M the largest of the partials' maxima and
// w_i = l_i 2^(m_i - M), O = sum w_i o_i / sum w_i, in the order of the CTAs. Bound by the
// latency of its loads, from L2.
template <typename T, int D>
__global__ void __launch_bounds__(FM_NT) fp8_merge_kernel(const __grid_constant__ fa::Args A) {
  const int lane = threadIdx.x & 31, row = blockIdx.y * (FM_NT / 32) + (threadIdx.x >> 5);
  // every CTA waits for the kernel before this one, with work or without: what comes after on the
  // stream takes this kernel's end for the end of both
  pdl_wait();
  const int4 seg = A.meta[blockIdx.x];
  const int n = seg.w;
  const int n0 = seg.z * A.npr, rows = (min(n0 + A.npr, A.a.T) - n0) * A.g;
  if (n == 0 || row >= rows) return;
  auto slot = [&](int i) { return 2 * ((int64_t)blockIdx.x + i) + (i == 0 ? 1 : 0); };
  const float* ml = A.part_ml + row;
  const int c = 4 * (lane % (D / 4));
  const float* po = A.part_o + (int64_t)row * D + c;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(ml + slot(i) * 2 * A.rows_pad));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int cnt = min(32, n - i0);
    float w = 0.f;
    if (lane < cnt) {
      const float* pm = ml + slot(i0 + lane) * 2 * A.rows_pad;
      const float m = __ldcg(pm);
      w = __ldcg(pm + A.rows_pad) * (m == top ? 1.f : fa::ex2(m - top));
    }
    for (int i = 0; i < cnt; i += FM_AHEAD) {
      float4 x[FM_AHEAD];
#pragma unroll
      for (int u = 0; u < FM_AHEAD; ++u)
        x[u] = __ldcg(reinterpret_cast<const float4*>(po + slot(i0 + min(i + u, cnt - 1)) * A.rows_pad * D));
#pragma unroll
      for (int u = 0; u < FM_AHEAD; ++u) {
        const float f = __shfl_sync(0xffffffffu, w, min(i + u, 31));
        if (i + u >= cnt) continue;
        sum += f;
        y.x = fmaf(x[u].x, f, y.x), y.y = fmaf(x[u].y, f, y.y), y.z = fmaf(x[u].z, f, y.z), y.w = fmaf(x[u].w, f, y.w);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane < D / 4)
    *reinterpret_cast<uint2*>(static_cast<T*>(A.a.out) + fa::out_row(A, seg.x, seg.y, n0, row) * D + c) =
        make_uint2(fa::Out<T>::pack(y.x * inv, y.y * inv), fa::Out<T>::pack(y.z * inv, y.w * inv));
}

template <typename T, int D>
int fm_launch(const fa::Args& A, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(ctas, (A.rows_pad + FM_NT / 32 - 1) / (FM_NT / 32));
  cfg.blockDim = dim3(FM_NT);
  cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_merge_kernel<T, D>, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 merge launch: %s", cudaGetErrorString(e));
  return check_launch("attention_fp8_merge");
}

}  // namespace

int launch_fp8_merge(const fa::Args& A, int dtype, int ctas, cudaStream_t st) {
  if (dtype == DROPKV_DTYPE_BF16)
    return A.a.D == 128 ? fm_launch<__nv_bfloat16, 128>(A, ctas, st) : fm_launch<__nv_bfloat16, 64>(A, ctas, st);
  return A.a.D == 128 ? fm_launch<__half, 128>(A, ctas, st) : fm_launch<__half, 64>(A, ctas, st);
}

size_t attention_fp8_workspace_size(int B, int Hq, int Hkv, int T, int D, int cap) {
  (void)B, (void)cap;
  const int rows = Hq / Hkv * T;
  return rows <= kFp8DecodeRows ? fp8_decode_plan(rows, D).bytes : 0;
}

int launch_attention_fp8(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  if (a.cap == 0) {  // no rows at all: nothing is seen
    if (cudaMemsetAsync(a.out, 0, (size_t)a.B * a.Hq * a.T * a.D * 2, st) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "attention_fp8: memset failed");
    return DROPKV_OK;
  }
  if ((int64_t)a.Hq / a.Hkv * a.T <= kFp8DecodeRows) return launch_fp8_decode(a, dtype, ws, st);
  const unsigned rows = (unsigned)((int64_t)a.B * a.Hq * a.T);
  if (dtype == DROPKV_DTYPE_BF16) {
    if (a.D == 128)
      attention_fp8_row_kernel<__nv_bfloat16, 128><<<rows, FA_NT, 0, st>>>(a);
    else
      attention_fp8_row_kernel<__nv_bfloat16, 64><<<rows, FA_NT, 0, st>>>(a);
  } else if (a.D == 128) {
    attention_fp8_row_kernel<__half, 128><<<rows, FA_NT, 0, st>>>(a);
  } else {
    attention_fp8_row_kernel<__half, 64><<<rows, FA_NT, 0, st>>>(a);
  }
  return check_launch("attention_fp8");
}

}  // namespace dropkv
