// What the two kernels of attention over a cache in 8 bits share (fp8_decode.cu: few query rows,
// fp8_attn.cu: many): which keys a row tile reads, the line of tiles that is cut over the CTAs,
// and the partials that fp8_attn.cu's merge kernel joins.
//
// The M = g T query rows of a KV head are ordered by token, then head of the group, and taken in
// row tiles of `npr` whole tokens. A row tile reads tiles of TK keys: from the first that some
// token's window reaches (0 without one) to the last token's own, and those of the sinks
// before it. All (sequence, row tile, KV head) segments form one line of units, `lead` and then
// one for each tile, that is cut evenly over the CTAs, from the lengths on the device: the host does
// not know them, and no CTA waits for another. A segment that falls into several CTAs leaves a partial
// in each: the output divided by its sum, its maximum and its sum.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace dropkv {
namespace fa {

struct Args {
  AttnFp8 a;
  int g, npr, RT;    // heads of a group, tokens of a row tile, row tiles of a sequence
  int g_mul;         // ceil(2^16 / g)
  int lead;          // units before a segment's tiles: about what a further segment costs a CTA, in tiles
  int rows_pad;      // rows of a partial
  int mask_vec;      // the mask's rows are read 4 bytes at a time
  int q_vec;         // Q's rows are read 16 bytes at a time
  float scale_log2;
  int* status;       // [CTAs]: 0, or which wait gave up
  int4* meta;        // [CTAs]: the split segment that begins in a CTA: b, KV head, row tile, its partials (0: none)
  float* part_o;     // [2 CTAs][rows_pad][D]; many rows: [2 CTAs][D / 4][rows_pad][4]
  float* part_ml;    // [2 CTAs][2][rows_pad]
  float* units;      // [row tiles][128]: what a unit of a row's queries makes of a logit, in base 2 (many rows)
  uint8_t* queries;  // [row tiles][parts][128][D]: 8-bit parts of the queries, as the products read them
  // r / g for a row r of a tile: r (g_mul g - 2^16) < 2^7 2^7 < 2^16
  __device__ __forceinline__ int quot(int r) const { return (r * g_mul) >> 16; }
};

// Keys of a row tile of sequence b.
template <int TK>
struct Keys {
  int len, keys;   // cached rows (past the table, too); cached rows and tokens that fit it
  int n0, n1;      // its tokens
  int lo;          // no token sees a key from the sinks to here
  int ns, w0, n;   // tiles of sinks, the first tile after them, all tiles (one at least)
  __device__ __forceinline__ void set(const Args& A, int b, int rt) {
    const AttnFp8& a = A.a;
    len = max(A.queries ? __ldcg(a.cache_lens + b) : a.cache_lens[b], 0);  // (many rows: read before the wait for the kernel before)
    keys = (int)min((int64_t)len + a.T, (int64_t)a.cap);
    n0 = rt * A.npr;
    n1 = min(n0 + A.npr, a.T);
    const int hi = a.mask ? keys : (int)min((int64_t)len + n1, (int64_t)a.cap);
    lo = a.window ? (int)min(max((int64_t)len + (a.mask ? 0 : n0) - a.window + 1, (int64_t)0), (int64_t)a.cap) : 0;
    w0 = lo / TK;
    ns = a.window ? min((min(a.sinks, hi) + TK - 1) / TK, w0) : 0;
    const int w1 = (hi + TK - 1) / TK;
    n = ns + max(w1 - w0, 0);
    if (n == 0) n = 1, w0 = 0;  // no key is seen: one tile says so
  }
  // first key of tile t
  __device__ __forceinline__ int first(int t) const { return (t < ns ? t : w0 + (t - ns)) * TK; }
  // some token sees some of keys [j, j + count)
  __device__ __forceinline__ bool any(const Args& A, int j, int count) const {
    return j < keys && (j + count > lo || j < A.a.sinks);
  }
  // Every token sees all of keys [j, j + count), their pages given, where j + count <= end and either j >= low
  // or j + count <= sinks.
  __device__ __forceinline__ void all(const Args& A, int* end, int* low) const {
    const AttnFp8& a = A.a;
    *end = a.mask ? min(len, keys) : (int)min((int64_t)len + n0 + 1, (int64_t)keys);
    *low = a.window ? (int)min(max((int64_t)len + (a.mask ? a.T : n1) - a.window, (int64_t)0), (int64_t)a.cap) : 0;
  }
};

// What one token sees of a sequence's keys, its page aside.
struct Sees {
  int lo, hi;  // keys [lo, hi) and those below sinks
  int node;
  // a token that sees nothing
  __device__ __forceinline__ void none() { lo = hi = node = 0; }
  __device__ __forceinline__ void set(const Args& A, int b, int len, int keys, int node_) {
    const AttnFp8& a = A.a;
    node = node_;
    int64_t depth = node;
    if (a.mask && a.window) {
      const uint8_t* row = a.mask + b * a.mask_sb + node * a.mask_sr;
      depth = -1;
      for (int n = 0; n < a.T; ++n) depth += row[n * a.mask_sc] != 0;
      depth = max(depth, (int64_t)0);
    }
    lo = a.window ? (int)min(max((int64_t)len + depth - a.window + 1, (int64_t)0), (int64_t)a.cap) : 0;
    hi = a.mask ? keys : (int)min((int64_t)len + node + 1, (int64_t)keys);
  }
  // bit e: key j0 + e is seen
  template <int COUNT>
  __device__ __forceinline__ uint64_t bits(const Args& A, int b, int len, int j0) const {
    constexpr int count = COUNT;
    static_assert(COUNT <= 64 && COUNT % 8 == 0, "keys");
    const AttnFp8& a = A.a;
    auto below = [&](int n) -> uint64_t { return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1); };
    uint64_t m = below(hi - j0) & below(count);
    const uint64_t near = ~below(lo - j0) | below(a.sinks - j0);
    if (!a.mask || !m) return m & near;
    const uint64_t cached = below(len - j0);
    const uint8_t* row = a.mask + b * a.mask_sb + node * a.mask_sr;
    uint64_t nodes = 0;
    const int n0 = j0 - len;  // the node of bit 0
    if (m & ~cached) {
      // (many loads on their way at once: a truth value at a time takes as many trips to memory)
      if (A.mask_vec) {
        constexpr int WORDS = COUNT / 4 + 1;
        uint32_t x[WORDS];
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          const int n = (n0 & ~3) + 4 * i;
          x[i] = n >= 0 && n < a.T ? *reinterpret_cast<const uint32_t*>(row + n) : 0u;
        }
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {  // four truth values to four bits
          const int at = 4 * i - (n0 & 3);
          const uint64_t four = ((__vcmpne4(x[i], 0u) & 0x01010101u) * 0x10204080u) >> 28;
          nodes |= at < 0 ? four >> -at : (at < 64 ? four << at : 0ull);
        }
      } else {
#pragma unroll 1
        for (int e0 = 0; e0 < count; e0 += 8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int n = n0 + e0 + e;
            if (n >= 0 && n < a.T && row[(int64_t)n * a.mask_sc]) nodes |= 1ull << (e0 + e);
          }
        }
      }
      nodes &= m & ~cached;
    }
    return (m & cached & near) | nodes;
  }
};

// A CTA's part of one segment: tiles [t0, t1) of `tiles`.
template <int TK>
struct Piece {
  int b, h, rt, t0, t1, tiles, rows;
  int parts;  // partials of a split segment that begins here, else 0
  Keys<TK> k;
};

// Where a CTA's share of the line begins: found by one warp, read by all.
struct Start {
  long long w, w1, per;  // units: the share's, and a share's size
  int pair, h, u;        // the (sequence, row tile) pair, the head and the unit in it
};

template <int TK>
__device__ __forceinline__ void find_start(const Args& A, int lane, Start* out) {
  const int pairs = A.a.B * A.RT;
  Keys<TK> k;
  auto units = [&](int p) -> long long {
    if (p >= pairs) return 0;
    k.set(A, p / A.RT, p % A.RT);
    return (long long)(k.n + A.lead) * A.a.Hkv;
  };
  const long long own0 = units(lane);
  long long total = own0;
  for (int p = lane + 32; p < pairs; p += 32) total += units(p);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const long long per = (total + gridDim.x - 1) / gridDim.x;
  const long long w0 = min(total, per * blockIdx.x), w1 = min(total, w0 + per);
  long long before = 0;
  if (w0 < w1) {
    for (int c = 0; c < pairs; c += 32) {
      const long long own = c == 0 ? own0 : units(c + lane);
      long long upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > w0);
      if (past) {
        if (lane == __ffs(past) - 1) {
          const long long rel = w0 - (before + upto - own);
          k.set(A, (c + lane) / A.RT, (c + lane) % A.RT);
          const int each = k.n + A.lead;  // (many heads of a cache near 2^31 rows are more units than 32 bits count)
          out->pair = c + lane;
          out->h = own < 0x80000000ll ? (int)rel / each : (int)(rel / each);
          out->u = (int)(rel - (long long)out->h * each);
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (lane == 0) {
    out->w = w0;
    out->w1 = w1;
    out->per = per;
  }
}

// Steps through a CTA's pieces; every role has one of its own and sees the same.
template <int TK>
struct Walk {
  long long left, per;
  int pair, h, u;
  __device__ __forceinline__ void start(const Start& s) {
    left = s.w1 - s.w, per = s.per, pair = s.pair, h = s.h, u = s.u;
  }
  __device__ __forceinline__ bool next(const Args& A, Piece<TK>& p) {
    while (left > 0) {
      p.b = pair / A.RT;
      p.rt = pair % A.RT;
      p.h = h;
      p.k.set(A, p.b, p.rt);
      p.tiles = p.k.n;
      p.rows = (p.k.n1 - p.k.n0) * A.g;
      const int units = p.tiles + A.lead, u1 = (int)min((long long)units, u + left);
      p.t0 = max(u - A.lead, 0);
      p.t1 = u1 - A.lead;
      left -= u1 - u;
      if (u1 == units) {
        u = 0;
        if (++h == A.a.Hkv) {
          h = 0;
          ++pair;
        }
      } else {
        u = u1;
      }
      if (p.t1 > p.t0) {
        p.parts = p.t0 == 0 && p.t1 < p.tiles ? 1 + (int)((units - u1 + per - 1) / per) : 0;
        return true;
      }
    }
    return false;
  }
};

// A warp's walk in shared memory: the first lane steps, all read. What a loop over tiles does not use of it then
// takes no registers there.
template <int TK>
struct WarpWalk {
  Walk<TK> walk;
  Piece<TK> piece;
  __device__ __forceinline__ bool next(const Args& A, int lane) {
    __syncwarp();
    int more = 0;
    if (lane == 0) more = walk.next(A, piece);
    more = __shfl_sync(0xffffffffu, more, 0);
    __syncwarp();
    return more;
  }
};

// The partial that a CTA writes of a piece: its segment's first part, or a later one.
template <int TK>
__device__ __forceinline__ int64_t slot_of(const Piece<TK>& p) {
  return 2 * (int64_t)blockIdx.x + (p.t0 > 0 ? 0 : 1);
}

// The number of a row tile.
__device__ __forceinline__ int64_t row_tile(const Args& A, int b, int h, int rt) {
  return ((int64_t)b * A.a.Hkv + h) * A.RT + rt;
}

// Row r of a row tile in the output [B, Hq, T, D].
__device__ __forceinline__ int64_t out_row(const Args& A, int b, int h, int n0, int r) {
  const int token = A.quot(r), head = h * A.g + r - token * A.g;
  return ((int64_t)b * A.a.Hq + head) * A.a.T + n0 + token;
}

__device__ __forceinline__ float ex2(float x) {  // 2^x, hardware approximation; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(m - R): what a weight's measure is to that of a weight times a page's scale of V (of a row that has seen nothing: anything
// finite).
__device__ __forceinline__ float share_of(float m, float R) { return ex2(fmaxf(fminf(m - R, 126.f), -126.f)); }

template <typename T>
struct Out;
template <>
struct Out<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Out<__half> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
__device__ __forceinline__ uint32_t pack_half(float x, float y) { return Out<__half>::pack(x, y); }

// Four stored values as two words of two fp16 values, exactly.
__device__ __forceinline__ void widen4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}

// The unit of a row of queries: the power of two (2^-126 at least) that brings its largest element to
// at most 448.
__device__ __forceinline__ float query_unit(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

// Four values in 8 bits; what that leaves of them, times `up`, stays in v.
__device__ __forceinline__ uint32_t split4(float* v, float up) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE, __NV_E4M3);
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)two, __NV_E4M3)));
    v[e] = (v[e] - f.x) * up;
    v[e + 1] = (v[e + 1] - f.y) * up;
    w |= two << (8 * e);
  }
  return w;
}

struct Plan {
  int ctas, rows_pad;
  size_t off_meta, off_o, off_ml, bytes;
};
inline Plan make_plan(int ctas, int rows_pad, int D) {
  Plan p;
  p.ctas = ctas;
  p.rows_pad = rows_pad;
  p.off_meta = align_up((size_t)ctas * 4, 256);
  p.off_o = align_up(p.off_meta + (size_t)ctas * sizeof(int4), 256);
  p.off_ml = p.off_o + (size_t)2 * ctas * rows_pad * D * 4;
  p.bytes = align_up(p.off_ml + (size_t)2 * ctas * 2 * rows_pad * 4, 256);
  return p;
}
inline Args make_args(const AttnFp8& a, const Plan& p, int npr, int lead, void* ws) {
  Args A;
  A.a = a;
  A.g = a.Hq / a.Hkv;
  A.g_mul = (65536 + A.g - 1) / A.g;
  A.npr = npr;
  A.RT = (a.T + npr - 1) / npr;
  A.lead = lead;
  A.rows_pad = p.rows_pad;
  A.q_vec = a.q_sd == 1 && (reinterpret_cast<uintptr_t>(a.q) | (uint64_t)((a.q_sb | a.q_sh | a.q_ss) * 2)) % 16 == 0;
  A.mask_vec = a.mask && a.mask_sc == 1 && a.T % 4 == 0 &&
               (reinterpret_cast<uintptr_t>(a.mask) | (uint64_t)(a.mask_sb | a.mask_sr)) % 4 == 0;
  A.scale_log2 = a.scale * 1.4426950408889634f;
  uint8_t* w = static_cast<uint8_t*>(ws);
  A.status = reinterpret_cast<int*>(w);
  A.meta = reinterpret_cast<int4*>(w + p.off_meta);
  A.part_o = reinterpret_cast<float*>(w + p.off_o);
  A.part_ml = reinterpret_cast<float*>(w + p.off_ml);
  A.units = nullptr;
  A.queries = nullptr;
  return A;
}

}  // namespace fa

// Few query rows of a KV head (g T): fp8_decode.cu takes up to 8, and up to 16 of heads of 64. Its 16 rows take twice the registers of
// 8, and at D = 128 the tiles and their queries no longer fit them: 4 tokens x 4 heads a KV head over 32 sequences of up to 13107
// rows, bf16, take 194 us there and 128 in fp8_attn.cu (one sequence of 13107 rows 28.3 and 25.8, of 819 14.5 and 14.6, a window of
// 1000 58.8 and 58.3); at D = 64, 2 tokens x 7 heads, 30.0 and 39.1 (18.2 and 22.2, 9.6 and 12.4, 14.7 and 23.5).
inline bool fp8_few_rows(int64_t rows, int D) { return rows <= (D == 64 ? 16 : 8); }
fa::Plan fp8_decode_plan(int rows, int D);
int launch_fp8_decode(const AttnFp8& a, int dtype, void* ws, cudaStream_t st);
// Joins the partials of what was just launched with A on `ctas` CTAs.
int launch_fp8_merge(const fa::Args& A, int dtype, int ctas, cudaStream_t st);

}  // namespace dropkv
