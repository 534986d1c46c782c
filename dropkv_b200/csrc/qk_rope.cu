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
//
// HBM bounds long chunks in principle (4 D bytes a row of 16 bits, the tables beside them);
// in fact it is instructions, and the latency of the chains position - table row - rows. So
// arithmetic is done on two floats at once, as many CTAs are resident as registers allow without
// spilling, and a group takes several rounds of rows for one look at the tables. 4096 tokens x 40
// heads of 128, bf16, normed (86 MB with the tables): 19.9 us, 4.3 TB/s (66% of a copy's rate), without
// a norm 15.6 (84%), in a graph over inputs larger than L2; 16384 tokens 72 us (4.7 TB/s). Rows on
// their way x rounds, for 4096 (one set of inputs, in part in L2) and 16384 tokens: 2 x 2 18.8 and 71.7 us, 3 x 1 21.2 and 80.3, 3 x 2 20.7 and 70.5, 2 x 4 20.7 and 67.8;
// 8 CTAs an SM 22.5 us, and the next round's rows loaded ahead 28.9.
constexpr int QR_BATCH = 2, QR_ROUNDS = 2;

// Two floats in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t qr_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void qr_unpair(uint64_t r, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t qr_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t qr_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes of a row as pairs of floats.
template <typename T>
struct QrVec;
template <>
struct QrVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, uint64_t* x) {
    x[0] = qr_pair(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = qr_pair(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 put(const uint64_t* x) {
    float a, b, c, d;
    qr_unpair(x[0], a, b);
    qr_unpair(x[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  }
};
template <>
struct QrVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, uint64_t* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = qr_pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 put(const uint64_t* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      qr_unpair(x[i], a, b);
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[i] = reinterpret_cast<const uint32_t&>(h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct QrVec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, uint64_t* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(reinterpret_cast<const __half2&>(w[i]));
      x[i] = qr_pair(f.x, f.y);
    }
  }
  static __device__ __forceinline__ uint4 put(const uint64_t* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      qr_unpair(x[i], a, b);
      const __half2 h = __floats2half2_rn(a, b);
      w[i] = reinterpret_cast<const uint32_t&>(h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <typename T, int G, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(QR_NT, 7) qk_rope_vec_kernel(QkRope a, int tokens, int hpg) {
  constexpr int N = QrVec<T>::N, GROUPS = QR_NT / G;
  const int heads = a.Hq + a.Hkv + (a.slots ? a.Hkv : 0);
  const int64_t gid = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
  const bool idle = gid >= (int64_t)tokens * hpg;  // (shuffles want the whole warp)
  const unsigned bl = idle ? 0u : (unsigned)(gid / (unsigned)hpg);
  const int b = (int)(bl / (unsigned)a.L), l = (int)(bl - (unsigned)b * (unsigned)a.L);
  const int u = threadIdx.x % G, step = hpg;
  const float inv_d = 1.f / a.D;  // (D is a power of two here)
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
  // cosines and sines of the lane's N pairs; interleaved, N / 2 pairs of each vector: (c, c) and (-s, s)
  const bool known = pos >= 0 && pos < a.P;  // a position outside the tables gives NaN
  uint64_t cs[INTERLEAVED ? N : N / 2], sn[INTERLEAVED ? N : N / 2];
  {
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = s[i] = NAN;
    if (turns && known) {
      const float* pc = a.cos + pos * (a.R / 2) + N * u;
      const float* ps = a.sin + pos * (a.R / 2) + N * u;
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(pc + i), y = *reinterpret_cast<const float4*>(ps + i);
        c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
        s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
      }
    }
    if (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < N; ++i) cs[i] = qr_pair(c[i], c[i]), sn[i] = qr_pair(-s[i], s[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) cs[i] = qr_pair(c[2 * i], c[2 * i + 1]), sn[i] = qr_pair(s[2 * i], s[2 * i + 1]);
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
      uint64_t x[N / 2], y[N / 2];
      QrVec<T>::get(va[i], x);
      QrVec<T>::get(vb[i], y);
      if (NORM) {
        uint64_t ss2 = 0;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) ss2 = qr_fma2(x[e], x[e], qr_fma2(y[e], y[e], ss2));
        float ss, s1;
        qr_unpair(ss2, ss, s1);
        ss += s1;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
        if (there && !is_v && w) {
          const float inv = rsqrtf(ss * inv_d + a.eps);
          const uint64_t inv2 = qr_pair(inv, inv);
          uint64_t wx[N / 2], wy[N / 2];  // (from L1: held in registers they cost occupancy: 33 us where this took 24)
          QrVec<T>::get(*reinterpret_cast<const uint4*>(w + lo), wx);
          QrVec<T>::get(*reinterpret_cast<const uint4*>(w + hi), wy);
#pragma unroll
          for (int e = 0; e < N / 2; ++e) {
            x[e] = qr_mul2(qr_mul2(x[e], inv2), wx[e]);
            y[e] = qr_mul2(qr_mul2(y[e], inv2), wy[e]);
          }
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
      if (!turns) {  // (untouched, not times one: infinities stay)
      } else if (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          float p, q;
          qr_unpair(x[e], p, q);
          x[e] = qr_fma2(qr_pair(q, p), sn[e], qr_mul2(x[e], cs[e]));
          qr_unpair(y[e], p, q);
          y[e] = qr_fma2(qr_pair(q, p), sn[N / 2 + e], qr_mul2(y[e], cs[N / 2 + e]));
        }
      } else {
        const uint64_t minus = qr_pair(-1.f, -1.f);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const uint64_t p = x[e], q = y[e];
          x[e] = qr_fma2(qr_mul2(q, sn[e]), minus, qr_mul2(p, cs[e]));
          y[e] = qr_fma2(p, sn[e], qr_mul2(q, cs[e]));
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
    // a group takes up to QR_ROUNDS batches of its token's rows, fewer where that would leave SMs
    // short of CTAs (3 x 1037 tokens x 18 heads: 9.2 us with all of a batch of three, 6.4 so)
    const int few = (heads + QR_BATCH * QR_ROUNDS - 1) / (QR_BATCH * QR_ROUNDS);
    const int64_t want = 4 * (int64_t)num_sms_current_device() * (QR_NT / G);
    const int64_t fill = (want + tokens - 1) / tokens;
    const int hpg = fill < few ? few : fill < heads ? (int)fill : heads;
    const int64_t ctas = (tokens * hpg * G + QR_NT - 1) / QR_NT;
    if (ctas > 0x7fffffff) return fail(DROPKV_ERR_UNSUPPORTED, "qk_norm_rope: too many rows");
    const dim3 grid((unsigned)ctas);
    auto run = [&](auto g) {
      constexpr int GG = decltype(g)::value;
      const bool norm = a.q_weight || a.k_weight;
      if (a.interleaved)
        norm ? qk_rope_vec_kernel<T, GG, true, true><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg)
             : qk_rope_vec_kernel<T, GG, true, false><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg);
      else
        norm ? qk_rope_vec_kernel<T, GG, false, true><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg)
             : qk_rope_vec_kernel<T, GG, false, false><<<grid, QR_NT, 0, st>>>(a, (int)tokens, hpg);
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
