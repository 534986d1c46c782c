// Attention of a tree of drafted tokens over a cache: for sequence b, query head h
// and node i, O = sum_j softmax_j(scale q_i . k_j) v_j over the len_b cached rows
// and the tree's nodes j (rows len_b + j of the cache) that mask[i][j] shows.
#include "common.cuh"

namespace dropkv {
namespace {

constexpr int TA_NT = 128;

// Row `key` of KV head h: in a row buffer, or in the page the table names (nullptr:
// no such page).
template <typename T>
__device__ __forceinline__ const T* ta_row(const TreeAttn& a, const void* base, int64_t s0, int64_t sh, int64_t ss, int b,
                                           int h, int key) {
  const T* p = static_cast<const T*>(base);
  if (!a.table) return p + b * s0 + h * sh + key * ss;
  const int page = a.table[b * (int64_t)a.max_blocks + key / a.block];
  if (page < 0 || page >= a.n_pages) return nullptr;
  return p + page * s0 + h * sh + (key % a.block) * ss;
}

template <typename T>
__device__ __forceinline__ T ta_from(float x);
template <>
__device__ __forceinline__ __half ta_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 ta_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One CTA per (b, query head, node): TA_NT keys at a time, a thread for each key's
// score, then a thread for each column of the output.
template <typename T>
__global__ void __launch_bounds__(TA_NT) tree_attn_rows_kernel(TreeAttn a) {
  __shared__ float q[128], p[TA_NT], red[TA_NT / 32];
  const int tid = threadIdx.x, b = blockIdx.y, hq = blockIdx.x / a.T, i = blockIdx.x % a.T;
  const int h = hq / (a.Hq / a.Hkv);
  const int len = min(max(a.cache_lens[b], 0), a.cap), keys = min((int64_t)len + a.T, (int64_t)a.cap);
  if (tid < a.D) q[tid] = to_f(static_cast<const T*>(a.q)[b * a.q_sb + hq * a.q_sh + i * a.q_ss + tid * a.q_sd]) * a.scale;
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_sb + i * a.mask_sr : nullptr;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int j0 = 0; j0 < keys; j0 += TA_NT) {
    __syncthreads();
    const int j = j0 + tid;
    float s = -INFINITY;
    const T* kr = nullptr;
    if (j < keys && (j < len || (mask ? mask[(j - len) * a.mask_sc] != 0 : j - len <= i)))
      kr = ta_row<T>(a, a.k, a.k_s0, a.k_sh, a.k_ss, b, h, j);
    if (kr) {
      s = 0.f;
      for (int d = 0; d < a.D; ++d) s = fmaf(q[d], to_f(kr[d]), s);
    }
    float mx = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float use = mn == -INFINITY ? 0.f : mn;
    p[tid] = kr ? __expf(s - use) : -1.f;  // -1: not seen
    const float alpha = __expf(m - use);
    m = mn;
    __syncthreads();
    o *= alpha;
    l *= alpha;
    for (int t = 0; t < TA_NT && j0 + t < keys; ++t) {
      const float w = p[t];
      if (w == -1.f) continue;
      l += w;
      if (tid < a.D) o = fmaf(w, to_f(ta_row<T>(a, a.v, a.v_s0, a.v_sh, a.v_ss, b, h, j0 + t)[tid]), o);
    }
  }
  if (tid < a.D)
    static_cast<T*>(a.out)[((b * (int64_t)a.Hq + hq) * a.T + i) * a.D + tid] = ta_from<T>(l == 0.f ? 0.f : o / l);
}

}  // namespace

size_t tree_attention_workspace_size(int B, int Hq, int Hkv, int T, int D, int cap) {
  (void)B, (void)Hq, (void)Hkv, (void)T, (void)D, (void)cap;
  return 0;
}

int launch_tree_attention(const TreeAttn& a, int dtype, void* ws, cudaStream_t st) {
  (void)ws;
  const dim3 grid(a.Hq * a.T, a.B);
  if (dtype == DROPKV_DTYPE_BF16)
    tree_attn_rows_kernel<__nv_bfloat16><<<grid, TA_NT, 0, st>>>(a);
  else
    tree_attn_rows_kernel<__half><<<grid, TA_NT, 0, st>>>(a);
  return check_launch("tree_attention");
}

}  // namespace dropkv
