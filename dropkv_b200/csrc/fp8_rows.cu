// Rows of a paged K/V cache held in 8 bits: quantised as they are written, and read back.
//
// A page of one head has one scale, a power of two s, and a row's value is e4m3 * s. With
// powers of two a value is divided by s and multiplied by it exactly, so the 8 bits' rounding
// (2^-4 of a value, or 2^-10 s below 2^-6 s) is the only one, values read back are exact in
// 16 bits, and a page whose scale grows moves its rows by exponents: only what falls under
// 2^-6 of the new scale is rounded again. e4m3 keeps 15 binades above that, so a finer scale
// would gain nothing but the last binade's end.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"

namespace dropkv {
namespace {

constexpr int F8_KEEP = 4;          // vectors of a run that a thread keeps from the first look at them to the second
constexpr int F8_MAX_BLOCK = 1024;  // rows of a page
constexpr int F8_GAP = 256;         // rows without a slot are looked over within a run up to here: the nodes of a tree

struct F8Rows {      // K's or V's
  const char* x;     // [B, H, N, D] in the row type, byte strides
  int64_t x_sb, x_sh, x_sn;
  uint8_t* p;        // [pages, H, block, D]
  int64_t p_s0, p_sh, p_st;
  float* s;          // [pages, H]
  int64_t s_s0, s_sh;
};

struct F8Run {
  int64_t page;
  int start, stop;  // rows; start < 0: there is none left
};

struct F8StoreArgs {
  F8Rows r[2];
  const int64_t* slots;  // [B, N]
  int64_t n_slots;
  int N, block, D, chunks;
  int lanes, shift;      // vectors of a row, and log2 of that (vector form)
};

__device__ __forceinline__ uint32_t f8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The smallest power of two, 2^-126 at least, that brings a largest value with these bits to at
// most 448 = 1.75 * 2^8.
__device__ __forceinline__ float f8_scale_for(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

template <typename T, int VEC>
struct F8Vec {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void f8_load(const char* p, F8Vec<T, VEC>& x) {
  if (VEC == 1)
    x.v[0] = *reinterpret_cast<const T*>(p);
  else
    *reinterpret_cast<uint4*>(&x) = __ldcs(reinterpret_cast<const uint4*>(p));
}

// The larger of m and the largest magnitude in x, as bits of the row type: of two values in each word's halves for 16-bit
// types (f8_top() gives the larger), of one in fp32.
template <typename T, int VEC>
__device__ __forceinline__ uint32_t f8_largest(const F8Vec<T, VEC>& x, uint32_t m) {
  if (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = max(m, f8_abs_bits(to_f<T>(x.v[e])));
  } else if (VEC == 1) {
    m = __vmaxu2(m, *reinterpret_cast<const uint16_t*>(&x) & 0x7fffu);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) m = __vmaxu2(m, w[e] & 0x7fff7fffu);
  }
  return m;
}
// That magnitude as fp32's bits (the order of a type's bits is that of its magnitudes).
template <typename T>
__device__ __forceinline__ uint32_t f8_top(uint32_t m) {
  if (sizeof(T) == 4) return m;
  const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
  return f8_abs_bits(to_f<T>(*reinterpret_cast<const T*>(&h)));
}
template <typename T, int VEC>
__device__ __forceinline__ uint32_t f8_largest_finite(const F8Vec<T, VEC>& x, uint32_t m) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const uint32_t b = f8_abs_bits(to_f<T>(x.v[e]));
    m = b < 0x7f800000u ? max(m, b) : m;
  }
  return m;
}

// x * inv in 8 bits at p. What is no number, infinities too (e4m3 has none), becomes NaN.
template <typename T, int VEC>
__device__ __forceinline__ void f8_put(uint8_t* p, const F8Vec<T, VEC>& x, float inv, bool odd) {
  float y[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) y[e] = to_f<T>(x.v[e]) * inv;
  if (odd) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (f8_abs_bits(to_f<T>(x.v[e])) >= 0x7f800000u) y[e] = __uint_as_float(0x7fffffffu);
  }
  if (VEC == 1) {
    *p = __nv_cvt_float_to_fp8(y[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[VEC / 4 + (VEC < 4)];
#pragma unroll
    for (int e = 0; e < VEC / 4; ++e) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * e], y[4 * e + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * e + 2], y[4 * e + 3]), __NV_SATFINITE, __NV_E4M3);
      w[e] = lo | hi << 16;
    }
    if (VEC == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[VEC == 8]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// VEC stored values times f (at most 1), rounded to 8 bits again.
template <int VEC>
struct F8Bytes {
  uint32_t w[(VEC + 3) / 4];
};
template <int VEC>
__device__ __forceinline__ void f8_get_bytes(const uint8_t* p, F8Bytes<VEC>& x) {
  if (VEC == 8) {
    const uint2 y = *reinterpret_cast<const uint2*>(p);
    x.w[0] = y.x, x.w[(VEC + 3) / 4 - 1] = y.y;
  } else {
    x.w[0] = VEC == 4 ? *reinterpret_cast<const uint32_t*>(p) : *p;
  }
}
template <int VEC>
__device__ __forceinline__ void f8_rescale(uint8_t* p, const F8Bytes<VEC>& x, float f) {
  uint32_t y[(VEC + 3) / 4];
#pragma unroll
  for (int i = 0; i < (VEC + 3) / 4; ++i) {
    y[i] = 0;
#pragma unroll
    for (int s = 0; s < 32; s += 16) {
      const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)(x.w[i] >> s), __NV_E4M3)));
      y[i] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v.x * f, v.y * f), __NV_SATFINITE, __NV_E4M3) << s;
    }
  }
  if (VEC == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(y[0], y[(VEC + 3) / 4 - 1]);
  else if (VEC == 4)
    *reinterpret_cast<uint32_t*>(p) = y[0];
  else
    *p = (uint8_t)y[0];
}

// Rows to slots. A run is the rows of one sequence that follow one another in one page, fewer
// than F8_GAP rows without a slot between two of them; one CTA takes a run of one head of K or of V, so nothing is
// shared between CTAs and nothing waits. The CTA of a chunk of `block` rows takes the runs
// that begin in it, usually one. First look: the run's largest value, its offsets; then the page's
// scale: s' = need where the run holds the page's first row (what stood there before means
// nothing), else max(s, need), and where it grew the rows that the run does not write follow.
// HBM bounds a long call: rows are read once (a page of up to 16 KB stays in registers
// between the two looks; the rest of a larger one comes from L2), half or a quarter of that is written. 13107 rows x 8 heads x
// 128 in bf16: 19.2 us for 54 MB in and 27 out, 64% of a copy's rate (71% of the issue slots: rounding, a page's barrier).
template <typename T, int NT, int VEC>
__global__ void __launch_bounds__(NT, 1024 / NT) store_rows_fp8_kernel(const __grid_constant__ F8StoreArgs a) {
  constexpr int EB = sizeof(T), WARPS = NT / 32;
  __shared__ uint32_t written[F8_MAX_BLOCK / 32];  // the page's rows that the run writes
  __shared__ uint32_t red[WARPS];
  __shared__ F8Run run;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.chunks, i0 = (blockIdx.x % a.chunks) * a.block, h = blockIdx.y >> 1;
  const F8Rows& R = a.r[blockIdx.y & 1];
  const int64_t* slots = a.slots + (int64_t)b * a.N;
  const int end = min(i0 + a.block, a.N);
  auto page_of = [&](int64_t slot) -> int64_t {
    return slot >> 32 ? slot / a.block : (int64_t)((uint32_t)slot / (uint32_t)a.block);
  };
  auto slot_at = [&](int i) -> int64_t {
    const int64_t s = slots[i];
    return s < a.n_slots ? s : -1;
  };
  for (int i = tid; i < F8_MAX_BLOCK / 32; i += NT) written[i] = 0;
  auto split = [&](int item, int& row, int& col) {
    row = VEC > 1 ? item >> a.shift : item / a.lanes;
    col = VEC > 1 ? item & (a.lanes - 1) : item - row * a.lanes;
  };
  auto over_cta = [&]() {  // the largest of what the warps have left
    uint32_t m = red[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = max(m, red[w]);
    return m;
  };
  // The chunk's rows are on their way with their slots: where the chunk is a page's, from its first row on (a prompt from its
  // start), that is all there is to know. One barrier, no scale to read, no other rows: 43 us of a layer's, by the general way, to 19.
  const char* xb = R.x + b * R.x_sb + h * R.x_sh;
  F8Vec<T, VEC> keep[F8_KEEP];
  const int there = (end - i0) * a.lanes;
  const int64_t s0 = slots[i0];
  bool whole = s0 >= 0 && s0 + a.block <= a.n_slots && there <= F8_KEEP * NT;
  uint32_t chunk_largest = 0;
  {
    int64_t at[F8_KEEP];
#pragma unroll
    for (int u = 0; u < F8_KEEP; ++u) {
      int row, col;
      split(tid + u * NT, row, col);
      if (i0 + row < end) {
        at[u] = slots[i0 + row];
        f8_load<T, VEC>(xb + (i0 + row) * R.x_sn + col * (VEC * EB), keep[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < F8_KEEP; ++u) {
      int row, col;
      split(tid + u * NT, row, col);
      if (i0 + row < end) {
        whole = whole && at[u] == s0 + row;
        chunk_largest = f8_largest<T, VEC>(keep[u], chunk_largest);
      }
    }
  }
  chunk_largest = __reduce_max_sync(0xffffffffu, f8_top<T>(chunk_largest));
  if (lane == 0) red[warp] = chunk_largest;
  const int64_t s0_page = whole ? page_of(s0) : 0;
  if (__syncthreads_and(whole && s0 == s0_page * a.block)) {
    chunk_largest = over_cta();
    if (chunk_largest < 0x7f800000u) {
      const float scale = f8_scale_for(chunk_largest), inv = 1.f / scale;
      uint8_t* pb = R.p + s0_page * R.p_s0 + h * R.p_sh;
#pragma unroll
      for (int u = 0; u < F8_KEEP; ++u) {
        int row, col;
        split(tid + u * NT, row, col);
        if (i0 + row < end) f8_put<T, VEC>(pb + row * R.p_st + col * VEC, keep[u], inv, false);
      }
      if (tid == 0) R.s[s0_page * R.s_s0 + h * R.s_sh] = scale;
      return;
    }
  }
  int64_t s_before = -1, s_first = -1, s_after[4] = {-1, -1, -1, -1};
  if (warp == 0) {
    if (i0 - 1 - lane >= 0) s_before = slot_at(i0 - 1 - lane);
    if (i0 + lane < a.N) s_first = slot_at(i0 + lane);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (warp == 0) s_after[u] = i0 + 32 * (u + 1) + lane < a.N ? slot_at(i0 + 32 * (u + 1) + lane) : -1;
  // The first warp finds the runs that begin in the chunk, one after the other, for all.
  int64_t prev = -1, page = -1;  // of the last row with a slot before a window; of a lane's row in it
  int prev_row = -1, w0 = i0 - 32;
  unsigned some = 0, begins = 0, todo = 0;  // a window's rows with a slot, those that begin a run, those still to be taken
  if (warp == 0) {
    for (int top = i0 - 1; top >= 0 && top > i0 - 1 - F8_GAP; top -= 32) {
      const int64_t s = top == i0 - 1 ? s_before : (top - lane >= 0 ? slot_at(top - lane) : -1);
      const unsigned with = __ballot_sync(0xffffffffu, s >= 0);
      if (with) {
        prev = page_of(__shfl_sync(0xffffffffu, s, __ffs(with) - 1));
        prev_row = top - (__ffs(with) - 1);
        break;
      }
    }
  }
  auto next_run = [&](F8Run* out) {
    while (!todo) {
      w0 += 32;
      if (w0 >= end) {
        if (lane == 0) out->start = -1;
        return;
      }
      const int64_t s = w0 == i0 ? s_first : (w0 + lane < a.N ? slot_at(w0 + lane) : -1);
      page = s >= 0 ? page_of(s) : -1;
      some = __ballot_sync(0xffffffffu, s >= 0);
      const unsigned below = some & ((1u << lane) - 1);
      int64_t left = __shfl_sync(0xffffffffu, page, below ? 31 - __clz(below) : 0);
      if (!below) left = w0 + lane - prev_row <= F8_GAP ? prev : -1;
      begins = __ballot_sync(0xffffffffu, s >= 0 && page != left);
      if (some) {
        prev = __shfl_sync(0xffffffffu, page, 31 - __clz(some));
        prev_row = w0 + 31 - __clz(some);
      }
      todo = end - w0 < 32 ? begins & ((1u << (end - w0)) - 1) : begins;
    }
    const int at = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t mine = __shfl_sync(0xffffffffu, page, at);
    // the run's last row: before the next that begins one, here or in a later window
    const unsigned later = begins & ~((2u << at) - 1);
    int last = w0 + 31 - __clz(later ? some & ((1u << (__ffs(later) - 1)) - 1) : some);
    bool open = !later;
    for (int w = w0 + 32; open && w < a.N && w - last <= F8_GAP; w += 128) {
      int64_t t[4];  // four windows at a time on their way
#pragma unroll
      for (int u = 0; u < 4; ++u)
        t[u] = w == i0 + 32 ? s_after[u] : (w + 32 * u + lane < a.N ? slot_at(w + 32 * u + lane) : -1);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned there = __ballot_sync(0xffffffffu, t[u] >= 0);
        const unsigned same = __ballot_sync(0xffffffffu, t[u] >= 0 && page_of(t[u]) == mine);
        if (!open || !there) continue;
        const unsigned other = there & ~same;
        const unsigned run = other ? same & ((1u << (__ffs(other) - 1)) - 1) : same;
        if (run && w + 32 * u + __ffs(run) - 1 - last <= F8_GAP)
          last = w + 32 * u + 31 - __clz(run);
        else
          open = false;
        if (other) open = false;
      }
    }
    if (lane == 0) *out = F8Run{mine, w0 + at, last + 1};
  };
  for (;;) {
    if (warp == 0) next_run(&run);
    __syncthreads();
    if (run.start < 0) break;
    const int64_t mine = run.page;
    const int start = run.start, stop = run.stop;
    const int64_t first_slot = mine * a.block;
    const float old = R.s[mine * R.s_s0 + h * R.s_sh];
    uint8_t* pb = R.p + mine * R.p_s0 + h * R.p_sh;
    const int items = (stop - start) * a.lanes;
    // first look
    int off[F8_KEEP];
    uint32_t largest = 0;
#pragma unroll
    for (int u = 0; u < F8_KEEP; ++u) {
      const int item = tid + u * NT;
      int row, col;
      split(item, row, col);
      off[u] = -1;
      if (item < items) {
        const int64_t t = slot_at(start + row);
        if (t >= 0) {
          off[u] = (int)(t - first_slot);
          if (start != i0 || start + row >= end) f8_load<T, VEC>(xb + (start + row) * R.x_sn + col * (VEC * EB), keep[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < F8_KEEP; ++u) {
      if (off[u] < 0) continue;
      int row, col;
      split(tid + u * NT, row, col);
      if (col == 0) atomicOr(&written[off[u] >> 5], 1u << (off[u] & 31));
      largest = f8_largest<T, VEC>(keep[u], largest);
    }
    for (int item = tid + F8_KEEP * NT; item < items; item += NT) {
      int row, col;
      split(item, row, col);
      const int64_t t = slot_at(start + row);
      if (t < 0) continue;
      F8Vec<T, VEC> x;
      f8_load<T, VEC>(xb + (start + row) * R.x_sn + col * (VEC * EB), x);
      if (col == 0) atomicOr(&written[(int)(t - first_slot) >> 5], 1u << ((int)(t - first_slot) & 31));
      largest = f8_largest<T, VEC>(x, largest);
    }
    auto largest_of_cta = [&](uint32_t m) {
      m = __reduce_max_sync(0xffffffffu, m);
      __syncthreads();  // (what was there has been read)
      if (lane == 0) red[warp] = m;
      __syncthreads();
      return over_cta();
    };
    largest = largest_of_cta(f8_top<T>(largest));
    const bool odd = largest >= 0x7f800000u;  // some value is no number: the largest of the others counts
    if (odd) {
      largest = 0;
#pragma unroll
      for (int u = 0; u < F8_KEEP; ++u)
        if (off[u] >= 0) largest = f8_largest_finite<T, VEC>(keep[u], largest);
      for (int item = tid + F8_KEEP * NT; item < items; item += NT) {
        int row, col;
        split(item, row, col);
        if (slot_at(start + row) < 0) continue;
        F8Vec<T, VEC> x;
        f8_load<T, VEC>(xb + (start + row) * R.x_sn + col * (VEC * EB), x);
        largest = f8_largest_finite<T, VEC>(x, largest);
      }
      largest = largest_of_cta(largest);
    }
    const float need = f8_scale_for(largest);
    const bool held = !(written[0] & 1) && old >= 0.f && old < __uint_as_float(0x7f800000u);
    const float scale = held ? fmaxf(old, need) : need;
    if (held && scale > old) {  // the rows that the run does not write follow the scale
      const float f = old / scale;
      const int all = a.block * a.lanes;
      for (int e0 = tid; e0 < all; e0 += F8_KEEP * NT) {
        F8Bytes<VEC> x[F8_KEEP];
        uint8_t* p[F8_KEEP];
#pragma unroll
        for (int u = 0; u < F8_KEEP; ++u) {
          int row, col;
          split(e0 + u * NT, row, col);
          p[u] = nullptr;
          if (e0 + u * NT >= all || ((written[row >> 5] >> (row & 31)) & 1)) continue;
          p[u] = pb + row * R.p_st + col * VEC;
          f8_get_bytes<VEC>(p[u], x[u]);
        }
#pragma unroll
        for (int u = 0; u < F8_KEEP; ++u)
          if (p[u]) f8_rescale<VEC>(p[u], x[u], f);
      }
    }
    // second look
    const float inv = 1.f / scale;
#pragma unroll
    for (int u = 0; u < F8_KEEP; ++u) {
      int row, col;
      split(tid + u * NT, row, col);
      if (off[u] >= 0) f8_put<T, VEC>(pb + off[u] * R.p_st + col * VEC, keep[u], inv, odd);
    }
    for (int item = tid + F8_KEEP * NT; item < items; item += NT) {
      int row, col;
      split(item, row, col);
      const int64_t t = slot_at(start + row);
      if (t < 0) continue;
      F8Vec<T, VEC> x;
      f8_load<T, VEC>(xb + (start + row) * R.x_sn + col * (VEC * EB), x);
      f8_put<T, VEC>(pb + (t - first_slot) * R.p_st + col * VEC, x, inv, odd);
    }
    if (tid == 0) R.s[mine * R.s_s0 + h * R.s_sh] = scale;
    __syncthreads();  // `written` and `red` have been read
    for (int i = tid; i < F8_MAX_BLOCK / 32; i += NT) written[i] = 0;
  }
}

// ---------------------------------------------------------------------------
// Reading back
// ---------------------------------------------------------------------------
struct F8LoadArgs {
  F8Rows r[2];
  char* out[2];          // [B, H, N, D] contiguous
  const int64_t* slots;  // [B, N]
  int64_t n_slots;
  unsigned rows;         // B * H * N (vector form)
  int B, H, N, block, D;
};

constexpr int FL_NT = 256;
constexpr int FL_ROWS = 2;

template <typename T>
__device__ __forceinline__ T f8_from(float x);
template <>
__device__ __forceinline__ float f8_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half f8_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 f8_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// LANES threads have a row, 16 bytes of its output each, FL_ROWS rows on their way at once.
// Each value is widened exactly (e4m3 to fp16 to fp32), scaled and rounded once (exact but
// for ranges). HBM bounds it: a byte in, two or four out. 8 x 65536 rows at most x 4 heads x 128 to fp16, 1.4 GB: 214 us, 98% of
// a copy's rate.
template <typename T, int LANES>
__global__ void __launch_bounds__(FL_NT) load_rows_fp8_vec_kernel(const __grid_constant__ F8LoadArgs a) {
  constexpr int RPB = FL_NT / LANES, VEC = 16 / sizeof(T), WORDS = VEC / 4;
  const unsigned r0 = blockIdx.x * (RPB * FL_ROWS) + threadIdx.x / LANES;
  const int c = threadIdx.x % LANES;
  int64_t slot[FL_ROWS];
  unsigned h[FL_ROWS];
#pragma unroll
  for (int i = 0; i < FL_ROWS; ++i) {
    const unsigned r = r0 + i * RPB, bh = r / (unsigned)a.N, n = r - bh * a.N, b = bh / (unsigned)a.H;
    h[i] = bh - b * a.H;
    slot[i] = r < a.rows ? a.slots[(int64_t)b * a.N + n] : -1;
    if (slot[i] >= a.n_slots) slot[i] = -1;
  }
  uint32_t x[2][FL_ROWS][WORDS];
  float s[2][FL_ROWS];
#pragma unroll
  for (int i = 0; i < FL_ROWS; ++i) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      s[kv][i] = 0.f;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) x[kv][i][w] = 0;
    }
    if (slot[i] >= 0) {
      const int64_t page = slot[i] >> 32 ? slot[i] / a.block : (int64_t)((uint32_t)slot[i] / (uint32_t)a.block);
      const int64_t at = slot[i] - page * a.block;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const F8Rows& R = a.r[kv];
        const uint8_t* p = R.p + page * R.p_s0 + h[i] * R.p_sh + at * R.p_st + c * VEC;
        if (WORDS == 2) {
          const uint2 y = *reinterpret_cast<const uint2*>(p);
          x[kv][i][0] = y.x;
          x[kv][i][WORDS - 1] = y.y;
        } else {
          x[kv][i][0] = *reinterpret_cast<const uint32_t*>(p);
        }
        s[kv][i] = R.s[page * R.s_s0 + h[i] * R.s_sh];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FL_ROWS; ++i) {
    const unsigned r = r0 + i * RPB;
    if (r >= a.rows) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      union {
        T t[VEC];
        uint4 q;
      } y;
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const uint16_t two = (uint16_t)(x[kv][i][e / 4] >> (8 * (e & 2)));
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
        y.t[e] = f8_from<T>(f.x * s[kv][i]);
        y.t[e + 1] = f8_from<T>(f.y * s[kv][i]);
      }
      if (slot[i] < 0) y.q = make_uint4(0u, 0u, 0u, 0u);
      __stcs(reinterpret_cast<uint4*>(a.out[kv] + (int64_t)r * (LANES * 16) + c * 16), y.q);
    }
  }
}

// Rows of any size, alignment and number.
template <typename T>
__global__ void __launch_bounds__(FL_NT) load_rows_fp8_kernel(const __grid_constant__ F8LoadArgs a) {
  const int64_t total = (int64_t)a.B * a.H * a.N * a.D;
  for (int64_t e = (int64_t)blockIdx.x * FL_NT + threadIdx.x; e < total; e += (int64_t)gridDim.x * FL_NT) {
    int64_t r = e / a.D;
    const int d = (int)(e - r * a.D);
    const int n = (int)(r % a.N);
    r /= a.N;
    const int h = (int)(r % a.H), b = (int)(r / a.H);
    const int64_t slot = a.slots[(int64_t)b * a.N + n];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float y = 0.f;
      if (slot >= 0 && slot < a.n_slots) {
        const F8Rows& R = a.r[kv];
        const int64_t page = slot / a.block;
        const __half_raw x = __nv_cvt_fp8_to_halfraw(R.p[page * R.p_s0 + h * R.p_sh + (slot - page * a.block) * R.p_st + d], __NV_E4M3);
        y = __half2float(__half(x)) * R.s[page * R.s_s0 + h * R.s_sh];
      }
      reinterpret_cast<T*>(a.out[kv])[e] = f8_from<T>(y);
    }
  }
}

F8Rows f8_rows(const Fp8Pool& p, int kv) {
  F8Rows r = {};
  r.p = static_cast<uint8_t*>(kv ? p.v : p.k);
  r.p_s0 = kv ? p.v_s0 : p.k_s0, r.p_sh = kv ? p.v_sh : p.k_sh, r.p_st = kv ? p.v_st : p.k_st;
  r.s = kv ? p.v_scale : p.k_scale;
  r.s_s0 = kv ? p.vs_s0 : p.ks_s0, r.s_sh = kv ? p.vs_sh : p.ks_sh;
  return r;
}

int f8_log2(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

// Every page row starts on a multiple of `bytes`.
bool f8_pool_aligned(const Fp8Pool& p, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
           (uint64_t)(p.k_s0 | p.k_sh | p.k_st | p.v_s0 | p.v_sh | p.v_st)) % bytes) == 0;
}

template <typename T>
int store_fp8(const StoreRowsFp8& q, cudaStream_t st) {
  constexpr int EB = sizeof(T), VEC = 16 / EB;
  F8StoreArgs a;
  for (int kv = 0; kv < 2; ++kv) {
    a.r[kv] = f8_rows(q.pool, kv);
    a.r[kv].x = static_cast<const char*>(kv ? q.v : q.k);
    a.r[kv].x_sb = (kv ? q.v_sb : q.k_sb) * EB, a.r[kv].x_sh = (kv ? q.v_sh : q.k_sh) * EB;
    a.r[kv].x_sn = (kv ? q.v_sn : q.k_sn) * EB;
  }
  a.slots = q.slots;
  a.n_slots = (int64_t)q.pool.n_pages * q.pool.block;
  a.N = q.N, a.block = q.pool.block, a.D = q.pool.D;
  a.chunks = (int)(((int64_t)q.N + a.block - 1) / a.block);
  uint64_t bits = 0;
  for (int kv = 0; kv < 2; ++kv)
    bits |= reinterpret_cast<uintptr_t>(a.r[kv].x) | (uint64_t)(a.r[kv].x_sb | a.r[kv].x_sh | a.r[kv].x_sn);
  const int lanes = a.D / VEC;
  const bool vec = bits % 16 == 0 && a.D % VEC == 0 && (lanes & (lanes - 1)) == 0 && f8_pool_aligned(q.pool, VEC);
  a.lanes = vec ? lanes : a.D;
  a.shift = vec ? f8_log2(lanes) : 0;
  const int64_t ctas = (int64_t)q.B * a.chunks;
  if (ctas > 0x7fffffff || (int64_t)a.N * a.lanes > 0x7fffffff - 2048 || q.pool.H > 32767)
    return fail(DROPKV_ERR_UNSUPPORTED, "store_rows_fp8: %d x %d rows of %d heads are too many", q.B, q.N, q.pool.H);
  if ((int64_t)a.block * a.lanes > 0x7fffffff - 2048)  // (a page's vectors are counted in 31 bits)
    return fail(DROPKV_ERR_UNSUPPORTED, "store_rows_fp8: pages of %d rows of %d elements are too large", a.block, a.D);
  const dim3 grid((unsigned)ctas, 2 * q.pool.H);
  // a page of up to 4 KB by 64 threads, a larger one by 256: its vectors then stay in registers up to 16 KB
  const bool small = (int64_t)std::min(a.block, a.N) * a.D * EB <= 64 * 16 * F8_KEEP;
  if (vec && small)
    store_rows_fp8_kernel<T, 64, VEC><<<grid, 64, 0, st>>>(a);
  else if (vec)
    store_rows_fp8_kernel<T, 256, VEC><<<grid, 256, 0, st>>>(a);
  else
    store_rows_fp8_kernel<T, 256, 1><<<grid, 256, 0, st>>>(a);
  return check_launch("store_rows_fp8");
}

template <typename T>
int load_fp8(const LoadRowsFp8& q, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  F8LoadArgs a;
  for (int kv = 0; kv < 2; ++kv) a.r[kv] = f8_rows(q.pool, kv);
  a.out[0] = static_cast<char*>(q.k_out);
  a.out[1] = static_cast<char*>(q.v_out);
  a.slots = q.slots;
  a.n_slots = (int64_t)q.pool.n_pages * q.pool.block;
  a.B = q.B, a.H = q.pool.H, a.N = q.N, a.block = q.pool.block, a.D = q.pool.D;
  const int64_t rows = (int64_t)q.B * a.H * q.N;
  a.rows = (unsigned)rows;
  const int lanes = a.D / VEC;
  const bool aligned = f8_pool_aligned(q.pool, VEC) && a.D % VEC == 0 && rows < 0x7fffffff - FL_NT * FL_ROWS &&
                       (reinterpret_cast<uintptr_t>(q.k_out) | reinterpret_cast<uintptr_t>(q.v_out)) % 16 == 0;
  if (aligned && (lanes == 8 || lanes == 16 || lanes == 32)) {
    const int per = FL_NT / lanes * FL_ROWS, ctas = (int)((rows + per - 1) / per);
    if (lanes == 8)
      load_rows_fp8_vec_kernel<T, 8><<<ctas, FL_NT, 0, st>>>(a);
    else if (lanes == 16)
      load_rows_fp8_vec_kernel<T, 16><<<ctas, FL_NT, 0, st>>>(a);
    else
      load_rows_fp8_vec_kernel<T, 32><<<ctas, FL_NT, 0, st>>>(a);
    return check_launch("load_rows_fp8");
  }
  const int64_t want = (rows * a.D + FL_NT - 1) / FL_NT, most = 32 * (int64_t)num_sms_current_device();
  load_rows_fp8_kernel<T><<<(int)std::min(want, most), FL_NT, 0, st>>>(a);
  return check_launch("load_rows_fp8");
}

}  // namespace

int launch_store_rows_fp8(const StoreRowsFp8& q, int dtype, cudaStream_t st) {
  if (q.pool.block > F8_MAX_BLOCK)
    return fail(DROPKV_ERR_UNSUPPORTED, "store_rows_fp8 takes pages of at most %d rows (got %d)", F8_MAX_BLOCK, q.pool.block);
  if (dtype == DROPKV_DTYPE_BF16) return store_fp8<__nv_bfloat16>(q, st);
  return dtype == DROPKV_DTYPE_F16 ? store_fp8<__half>(q, st) : store_fp8<float>(q, st);
}

int launch_load_rows_fp8(const LoadRowsFp8& q, int dtype, cudaStream_t st) {
  if (dtype == DROPKV_DTYPE_BF16) return load_fp8<__nv_bfloat16>(q, st);
  return dtype == DROPKV_DTYPE_F16 ? load_fp8<__half>(q, st) : load_fp8<float>(q, st);
}

}  // namespace dropkv
