// RMS norm of the heads of queries and keys, the position rotation and the cache
// write in one pass: y = x * rsqrt(mean(x^2) + eps) * w over a head of D, then for
// each of the R / 2 pairs (a, b) of the head's first R elements
// (a c - b s, b c + a s) with c, s = cos, sin[position][pair].
#include <type_traits>

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

// Rows of any size, alignment and stride: one warp per row (b, l, head): heads [0, Hq) of Q, [Hq, Hq + Hkv) of K, then V.
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

// The same with 16-byte vectors: G lanes have a row, each one unit of two vectors -- the
// vectors whose elements rotate together (elements i and i + R / 2; interleaved pairs lie
// within a vector), or two that do not turn. A group of G lanes takes every hpg-th row of one
// token: a lane's cosines and sines, which weigh more than a row (64 bytes of table against 32
// of Q), are fetched once and stay in registers, and QR_BATCH rows are on their way at a time.
constexpr int QR_BATCH = 3;

template <typename T>
struct QrVec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f(p[i]);
  }
  static __device__ __forceinline__ uint4 put(const float* x) {
    uint4 v;
    T* p = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = qr_from<T>(x[i]);
    return v;
  }
};

template <typename T, int G, bool INTERLEAVED>
__global__ void __launch_bounds__(QR_NT) qk_rope_vec_kernel(QkRope a, int tokens, int hpg) {
  constexpr int N = QrVec<T>::N, GROUPS = QR_NT / G;
  const int heads = a.Hq + a.Hkv + (a.slots ? a.Hkv : 0);
  const int64_t gid = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
  const bool idle = gid >= (int64_t)tokens * hpg;  // (shuffles want the whole warp)
  const unsigned bl = idle ? 0u : (unsigned)(gid / (unsigned)hpg);
  const int b = (int)(bl / (unsigned)a.L), l = (int)(bl - (unsigned)b * (unsigned)a.L);
  const int u = threadIdx.x % G, step = hpg;
  const int h0 = idle ? heads : (int)(gid - (int64_t)bl * hpg);
  // this lane's elements: [lo, lo + N) and [hi, hi + N)
  const int turning = a.R / (2 * N);  // units that turn
  const bool turns = u < turning;
  int lo, hi;
  if (INTERLEAVED) {
    lo = 2 * N * u;
    hi = lo + N;
  } else {
    lo = turns ? N * u : a.R + 2 * N * (u - turning);
    hi = turns ? lo + a.R / 2 : lo + N;
  }
  auto row_of = [&](int h) -> const T* {
    if (h < a.Hq) return static_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + l * a.q_sl;
    if (h < a.Hq + a.Hkv) return static_cast<const T*>(a.k) + b * a.k_sb + (h - a.Hq) * a.k_sh + l * a.k_sl;
    return static_cast<const T*>(a.v) + b * a.v_sb + (h - a.Hq - a.Hkv) * a.v_sh + l * a.v_sl;
  };
  const int64_t pos = a.positions[b * a.pos_sb + l];
  int64_t slot = -1;
  if (a.slots) slot = a.slots[bl];
  uint4 va[QR_BATCH], vb[QR_BATCH];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < QR_BATCH; ++i) {
      const int hi_ = h + i * step;
      if (hi_ < heads) {
        const T* x = row_of(hi_);
        va[i] = *reinterpret_cast<const uint4*>(x + lo);
        vb[i] = *reinterpret_cast<const uint4*>(x + hi);
      }
    }
  };
  load(h0);
  // cosines and sines of the lane's N pairs (interleaved: N / 2 of each vector)
  const bool known = pos >= 0 && pos < a.P;  // a position outside the tables gives NaN
  float cs[N], sn[N];
#pragma unroll
  for (int i = 0; i < N; ++i) cs[i] = turns ? NAN : 1.f, sn[i] = turns ? NAN : 0.f;
  if (turns && known) {
    const float* c = a.cos + pos * (a.R / 2) + N * u;
    const float* s = a.sin + pos * (a.R / 2) + N * u;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(c + i), y = *reinterpret_cast<const float4*>(s + i);
      cs[i] = x.x, cs[i + 1] = x.y, cs[i + 2] = x.z, cs[i + 3] = x.w;
      sn[i] = y.x, sn[i + 1] = y.y, sn[i + 2] = y.z, sn[i + 3] = y.w;
    }
  }
  T* kp = nullptr;
  T* vp = nullptr;
  if (slot >= 0 && slot < (int64_t)a.n_pages * a.block) {
    const int64_t page = slot >> 32 ? slot / a.block : (int64_t)((uint32_t)slot / (uint32_t)a.block);
    const int64_t at = slot - page * a.block;
    kp = static_cast<T*>(a.k_pages) + page * a.kp_sb + at * a.kp_st;
    vp = static_cast<T*>(a.v_pages) + page * a.vp_sb + at * a.vp_st;
  }
  const int rounds = (heads + QR_BATCH * step - 1) / (QR_BATCH * step);
  for (int r = 0; r < rounds; ++r) {
    const int h = h0 + r * QR_BATCH * step;
    if (r) load(h);
#pragma unroll
    for (int i = 0; i < QR_BATCH; ++i) {
      const int hh = h + i * step;
      const bool there = hh < heads, is_q = hh < a.Hq, is_v = hh >= a.Hq + a.Hkv;
      float x[N], y[N];
      QrVec<T>::get(va[i], x);
      QrVec<T>::get(vb[i], y);
      if (a.q_weight || a.k_weight) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
        if (there && !is_v && w) {
          const float inv = rsqrtf(ss / a.D + a.eps);
          float wx[N], wy[N];  // (from L1: held in registers they cost occupancy, 24 -> 33 us)
          QrVec<T>::get(*reinterpret_cast<const uint4*>(w + lo), wx);
          QrVec<T>::get(*reinterpret_cast<const uint4*>(w + hi), wy);
#pragma unroll
          for (int e = 0; e < N; ++e) x[e] = x[e] * inv * wx[e], y[e] = y[e] * inv * wy[e];
        }
      }
      if (!there) continue;
      if (is_v) {
        if (vp) {
          T* dst = vp + (hh - a.Hq - a.Hkv) * a.vp_sh;
          *reinterpret_cast<uint4*>(dst + lo) = va[i];
          *reinterpret_cast<uint4*>(dst + hi) = vb[i];
        }
        continue;
      }
      if (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float p = x[e], q = x[e + 1], r = y[e], s = y[e + 1];
          x[e] = p * cs[e / 2] - q * sn[e / 2];
          x[e + 1] = q * cs[e / 2] + p * sn[e / 2];
          y[e] = r * cs[(N + e) / 2] - s * sn[(N + e) / 2];
          y[e + 1] = s * cs[(N + e) / 2] + r * sn[(N + e) / 2];
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float p = x[e], q = y[e];
          x[e] = p * cs[e] - q * sn[e];
          y[e] = q * cs[e] + p * sn[e];
        }
      }
      const uint4 ox = QrVec<T>::put(x), oy = QrVec<T>::put(y);
      T* out = is_q ? static_cast<T*>(a.q_out) + ((b * (int64_t)a.Hq + hh) * a.L + l) * a.D
                    : static_cast<T*>(a.k_out) + ((b * (int64_t)a.Hkv + hh - a.Hq) * a.L + l) * a.D;
      *reinterpret_cast<uint4*>(out + lo) = ox;
      *reinterpret_cast<uint4*>(out + hi) = oy;
      if (!is_q && kp) {
        T* dst = kp + (hh - a.Hq) * a.kp_sh;
        *reinterpret_cast<uint4*>(dst + lo) = ox;
        *reinterpret_cast<uint4*>(dst + hi) = oy;
      }
    }
  }
}

template <typename T>
int qr_launch(const QkRope& a, cudaStream_t st) {
  constexpr int N = QrVec<T>::N;
  const int64_t eb = sizeof(T);
  const int heads = a.Hq + a.Hkv + (a.slots ? a.Hkv : 0);
  // vectors: every row, table row and page row on 16-byte boundaries, a power of two of lanes
  // a row, whole units that turn
  uint64_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.q_out) |
                  reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.q_weight) |
                  reinterpret_cast<uintptr_t>(a.k_weight) |
                  (uint64_t)((a.q_sb | a.q_sh | a.q_sl | a.k_sb | a.k_sh | a.k_sl) * eb) | (uint64_t)(a.D * eb);
  if (a.R) bits |= reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin) | (uint64_t)(a.R / 2 * 4);
  if (a.slots)
    bits |= reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages) |
            (uint64_t)((a.v_sb | a.v_sh | a.v_sl | a.kp_sb | a.kp_sh | a.kp_st | a.vp_sb | a.vp_sh | a.vp_st) * eb);
  const int G = a.D % (2 * N) == 0 ? a.D / (2 * N) : 0;
  const bool lanes = G == 2 || G == 4 || G == 8 || G == 16 || G == 32;
  const int64_t tokens = (int64_t)a.B * a.L;
  if (bits % 16 == 0 && lanes && a.R % (2 * N) == 0 && tokens <= 0x7fffffff) {
    // a group takes QR_BATCH rows of its token where that still fills the device, else one row
    const int few = (heads + QR_BATCH - 1) / QR_BATCH;
    const int64_t want = 4 * (int64_t)num_sms_current_device() * (QR_NT / G);
    const int hpg = tokens * few >= want ? few : heads;
    const int64_t ctas = (tokens * hpg * G + QR_NT - 1) / QR_NT;
    if (ctas > 0x7fffffff) return fail(DROPKV_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
    const dim3 grid((unsigned)ctas);
    auto run = [&](auto g) {
      constexpr int GG = decltype(g)::value;
      if (a.interleaved)
        qk_rope_vec_kernel<T, GG, true><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg);
      else
        qk_rope_vec_kernel<T, GG, false><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg);
    };
    switch (G) {
      case 2: run(std::integral_constant<int, 2>()); break;
      case 4: run(std::integral_constant<int, 4>()); break;
      case 8: run(std::integral_constant<int, 8>()); break;
      case 16: run(std::integral_constant<int, 16>()); break;
      default: run(std::integral_constant<int, 32>()); break;
    }
    return check_launch("qk_norm_rope");
  }
  const int64_t grid = (tokens * heads + QR_NT / 32 - 1) / (QR_NT / 32);
  if (grid > 0x7fffffff) return fail(DROPKV_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
  qk_rope_rows_kernel<T><<<(int)grid, QR_NT, 0, st>>>(a);
  return check_launch("qk_norm_rope");
}

}  // namespace

int launch_qk_norm_rope(const QkRope& a, int dtype, cudaStream_t st) {
  if (dtype == DROPKV_DTYPE_BF16) return qr_launch<__nv_bfloat16>(a, st);
  if (dtype == DROPKV_DTYPE_F16) return qr_launch<__half>(a, st);
  return qr_launch<float>(a, st);
}

}  // namespace dropkv
