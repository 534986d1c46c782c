// RMS norm of the heads of queries and keys, the position rotation and the cache
// write in one pass: y = x * rsqrt(mean(x^2) + eps) * w over a head of D, then for
// each of the R / 2 pairs (a, b) of the head's first R elements
// (a c - b s, b c + a s) with c, s = cos, sin[position][pair].
#include "common.cuh"

namespace dropkv {
namespace {

constexpr int QR_NT = 128;

template <typename T>
__device__ __forceinline__ T qr_from(float x);
template <>
__device__ __forceinline__ float qr_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half qr_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 qr_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One warp per row (b, l, head): heads [0, Hq) of Q, [Hq, Hq + Hkv) of K, then V.
template <typename T>
__global__ void __launch_bounds__(QR_NT) qk_rope_rows_kernel(QkRope a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.Hq + a.Hkv + (a.slots ? a.Hkv : 0);
  const int64_t rows = (int64_t)a.B * a.L * heads;
  const int64_t row = (int64_t)blockIdx.x * (QR_NT / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int h = (int)(row % heads);
  const int64_t bl = row / heads;
  const int b = (int)(bl / a.L), l = (int)(bl % a.L);
  const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
  const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
  const T* x = is_q ? static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + l * a.q_sl
               : is_v ? static_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh + l * a.v_sl
                      : static_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh + l * a.k_sl;
  T* page = nullptr;
  if (!is_q && a.slots) {
    const int64_t slot = a.slots[b * (int64_t)a.L + l];
    if (slot >= 0 && slot < (int64_t)a.n_pages * a.block) {
      const int64_t p = slot / a.block, at = slot % a.block;
      page = is_v ? static_cast<T*>(a.v_pages) + p * a.vp_sb + hk * a.vp_sh + at * a.vp_st
                  : static_cast<T*>(a.k_pages) + p * a.kp_sb + hk * a.kp_sh + at * a.kp_st;
    }
  }
  if (is_v) {
    if (page)
      for (int d = lane; d < a.D; d += 32) page[d] = x[d];
    return;
  }
  T* out = is_q ? static_cast<T*>(a.q_out) + ((b * (int64_t)a.Hq + h) * a.L + l) * a.D
                : static_cast<T*>(a.k_out) + ((b * (int64_t)a.Hkv + hk) * a.L + l) * a.D;
  const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
  float inv = 1.f;
  if (w) {
    float ss = 0.f;
    for (int d = lane; d < a.D; d += 32) ss = fmaf(to_f(x[d]), to_f(x[d]), ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    inv = rsqrtf(ss / a.D + a.eps);
  }
  auto normed = [&](int d) { return w ? to_f(x[d]) * inv * to_f(w[d]) : to_f(x[d]); };
  const int64_t pos = a.positions[b * a.pos_sb + l];
  const bool known = pos >= 0 && pos < a.P;  // a position outside the tables gives NaN
  for (int i = lane; i < a.R / 2; i += 32) {
    const float c = known ? a.cos[pos * (a.R / 2) + i] : NAN, s = known ? a.sin[pos * (a.R / 2) + i] : NAN;
    const int lo = a.interleaved ? 2 * i : i, hi = a.interleaved ? 2 * i + 1 : i + a.R / 2;
    const float u = normed(lo), v = normed(hi);
    const T y0 = qr_from<T>(u * c - v * s), y1 = qr_from<T>(v * c + u * s);
    out[lo] = y0;
    out[hi] = y1;
    if (page) page[lo] = y0, page[hi] = y1;
  }
  for (int d = a.R + lane; d < a.D; d += 32) {
    const T y = qr_from<T>(normed(d));
    out[d] = y;
    if (page) page[d] = y;
  }
}

}  // namespace

int launch_qk_norm_rope(const QkRope& a, int dtype, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.L * (a.Hq + a.Hkv + (a.slots ? a.Hkv : 0));
  const int64_t grid = (rows + QR_NT / 32 - 1) / (QR_NT / 32);
  if (grid > 0x7fffffff) return fail(DROPKV_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
  if (dtype == DROPKV_DTYPE_BF16)
    qk_rope_rows_kernel<__nv_bfloat16><<<(int)grid, QR_NT, 0, st>>>(a);
  else if (dtype == DROPKV_DTYPE_F16)
    qk_rope_rows_kernel<__half><<<(int)grid, QR_NT, 0, st>>>(a);
  else
    qk_rope_rows_kernel<float><<<(int)grid, QR_NT, 0, st>>>(a);
  return check_launch("qk_norm_rope");
}

}  // namespace dropkv
