// Attention over a cache in 8 bits for few query rows (g T <= 16): single tokens, short drafts.
//
// A key costs 2 D bytes and 4 D M operations, so HBM bounds this by far, and what counts is to
// keep loads on their way and instructions few. Each warp takes 16 keys of a tile at a time, K and V
// straight into registers, the next step's K under way when S is there, its V when P V is; nothing
// is shared between warps until a piece ends. Both products are m16n8k16 MMAs of fp16 (the
// tcgen05 kernel's M = 128 would hold 1 to 16 rows here, and its softmax as many threads):
//   S = Q K^T      A = up to 16 query rows, B = 8 keys;
//   O^T += V^T P^T A = 16 columns of V for 16 keys, B = the weights of 8 rows as they lie in S's
//                  accumulators.
// e4m3 widens to fp16 exactly and two at a time. The order of D within a product is free:
// lane (gid, tig) = (lane / 4, lane % 4) reads bytes [64 i + 16 tig, + 16) of key gid's row of K, and for V
// bytes [D / 8 gid, + D / 8) of keys 2 tig, 2 tig + 1, 2 tig + 8 and 2 tig + 9, whose bytes are
// paired before they are widened. Queries in bf16 are brought to fp16 by a power of two for each
// row (its largest element to 2^14 or so; elements under 2^-28 of it lose bits).
// A page's scale of K multiplies its logits in fp32; that of V, over the largest of the warp so far,
// the weights. Weights are rounded to fp16 for their product (2^-11), sums taken from
// them before that.
#include <algorithm>
#include <type_traits>

#include "fp8_attn.cuh"

namespace dropkv {
namespace {

using namespace fa;

// 8 rows: two CTAs of 8 warps an SM; 16 rows need 64 registers for the output: one of 12 warps
template <bool R16>
struct FdShape {
  static constexpr int WARPS = R16 ? 12 : 8, NT = 32 * WARPS, CTAS = R16 ? 1 : 2;
  static constexpr int TK = 16 * WARPS, ROWS = R16 ? 16 : 8;
};
constexpr int kFdLead = 3;
// A row's reference moves once its maximum has grown by this much (base 2); weights are
// 2^(s - m + bias), so that fp16 holds them from 2^-24 to 2^15.
constexpr float kFdSlack = 8.f, kFdBias = 7.f;

template <int D, bool R16>
constexpr int fd_smem() {
  using S = FdShape<R16>;
  return S::WARPS * S::ROWS * (D + 2) * 4 + (int)sizeof(Start);
}

__device__ __forceinline__ void fd_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D, bool R16>
__global__ void __launch_bounds__(FdShape<R16>::NT, FdShape<R16>::CTAS)
    fp8_decode_kernel(const __grid_constant__ Args A) {
  using S = FdShape<R16>;
  constexpr int NT = S::NT, WARPS = S::WARPS, TK = S::TK, ROWS = S::ROWS, HR = R16 ? 2 : 1;
  constexpr int KV = D / 64;   // 16-byte vectors of K a lane has of a key
  constexpr int VW = D / 32;   // words of V a lane has of a key
  constexpr int VB = 4 * VW;
  extern __shared__ __align__(16) uint8_t sm[];
  float* wo = reinterpret_cast<float*>(sm);         // [WARPS][ROWS][D]
  float* wm = wo + WARPS * ROWS * D;                // [WARPS][ROWS]
  float* wl = wm + WARPS * ROWS;
  Start* start = reinterpret_cast<Start*>(wl + WARPS * ROWS);
  const AttnFp8& a = A.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: the merge may then read this kernel's inputs at once)
  if (warp == 0) find_start<TK>(A, lane, start);
  __syncthreads();
  Walk<TK> walk(*start);
  Piece<TK> p;
  while (walk.next(A, p)) {
    // ---- queries: rows gid and, of 16, gid + 8 ---------------------------------
    uint32_t q[KV * 4][2][HR];  // [k step][k half][row half]
    float qscale[HR];
    Sees sees[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      const int r = gid + 8 * x;
      float v[KV * 16];
      float big = 0.f;
      if (r < p.rows) {
        const int node = p.k.n0 + r / A.g, head = p.h * A.g + r % A.g;
        const T* src = static_cast<const T*>(a.q) + p.b * a.q_sb + head * a.q_sh + node * a.q_ss;
        sees[x].set(A, p.b, p.k.len, p.k.keys, node);
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          if (A.q_vec) {
            T t[16];
            *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(src + 64 * i + 16 * tig);
            *reinterpret_cast<uint4*>(t + 8) = *reinterpret_cast<const uint4*>(src + 64 * i + 16 * tig + 8);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[16 * i + e] = to_f(t[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[16 * i + e] = to_f(src[(64 * i + 16 * tig + e) * a.q_sd]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < KV * 16; ++e) v[e] = 0.f;
        sees[x].none();
      }
      qscale[x] = 1.f;
      if (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int e = 0; e < KV * 16; ++e) big = fmaxf(big, isfinite(v[e]) ? fabsf(v[e]) : 0.f);
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = min(max((int)(__float_as_uint(big) >> 23) - 14, 1), 253);  // 2^(e - 127): the largest over 2^14
        qscale[x] = __uint_as_float((uint32_t)e << 23);
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int i = 0; i < KV * 16; ++i) v[i] *= inv;
      }
      qscale[x] *= A.scale_log2;
#pragma unroll
      for (int s = 0; s < KV * 4; ++s) {
        q[s][0][x] = pack_half(v[4 * s], v[4 * s + 1]);
        q[s][1][x] = pack_half(v[4 * s + 2], v[4 * s + 3]);
      }
    }
    // ---- the warp's steps --------------------------------------------------------
    const uint8_t* kb = static_cast<const uint8_t*>(a.pool.k) + p.h * a.pool.k_sh + 16 * tig;
    const uint8_t* vb = static_cast<const uint8_t*>(a.pool.v) + p.h * a.pool.v_sh + VB * gid;
    const float* ksb = a.pool.k_scale + p.h * a.pool.ks_sh;
    const float* vsb = a.pool.v_scale + p.h * a.pool.vs_sh;
    const int32_t* table = a.table + (int64_t)p.b * a.max_blocks;
    const int block = a.pool.block, lb = __ffs(block) - 1;
    auto key_of = [&](int t) { return p.k.first(t) + 16 * warp; };
    // pages of the halves of a step: -1 where no token sees any of it
    auto pages_of = [&](int t, int* pg) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        pg[x] = -1;
        if (t >= p.t1) continue;
        const int j = key_of(t) + 8 * x;
        if (p.k.any(A, j, 8)) pg[x] = table[j >> lb];
        if (pg[x] >= a.pool.n_pages) pg[x] = -1;
      }
    };
    uint4 k[2][KV];
    uint32_t v[4][VW];
    float ks[2], vs[2];
    auto load_k = [&](int t, const int* pg) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = (key_of(t) + 8 * x + gid) & (block - 1);
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          k[x][i] = make_uint4(0u, 0u, 0u, 0u);
          if (pg[x] >= 0)
            k[x][i] = __ldcs(reinterpret_cast<const uint4*>(kb + pg[x] * a.pool.k_s0 + at * a.pool.k_st + 64 * i));
        }
      }
    };
    auto load_v = [&](int t, const int* pg) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int x = c >> 1, at = (key_of(t) + 8 * x + 2 * tig + (c & 1)) & (block - 1);
        const uint8_t* src = vb + pg[x] * a.pool.v_s0 + at * a.pool.v_st;
#pragma unroll
        for (int w = 0; w < VW; ++w) v[c][w] = 0;
        if (pg[x] >= 0) {
          if (VW == 4) {
            const uint4 y = __ldcs(reinterpret_cast<const uint4*>(src));
            v[c][0] = y.x, v[c][1] = y.y, v[c][VW - 2] = y.z, v[c][VW - 1] = y.w;
          } else {
            const uint2 y = __ldcs(reinterpret_cast<const uint2*>(src));
            v[c][0] = y.x, v[c][1] = y.y;
          }
        }
      }
    };
    float o[HR][VB / 2][4];
    float m[HR], l[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
      for (int t = 0; t < VB / 2; ++t) o[x][t][0] = o[x][t][1] = o[x][t][2] = o[x][t][3] = 0.f;
    }
    float vref = 0.f;  // the output is o * vref
    int pg[2], pg1[2];
    pages_of(p.t0, pg);
    pages_of(p.t0 + 1, pg1);
    load_k(p.t0, pg);
    load_v(p.t0, pg);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      ks[x] = pg[x] >= 0 ? ksb[pg[x] * a.pool.ks_s0] : 0.f;
      vs[x] = pg[x] >= 0 ? vsb[pg[x] * a.pool.vs_s0] : 0.f;
    }
    for (int t = p.t0; t < p.t1; ++t) {
      int pg2[2];
      pages_of(t + 2, pg2);
      const int j0 = key_of(t);
      const bool some = pg[0] >= 0 || pg[1] >= 0;
      float s[2][4];
      if (some) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
          for (int i = 0; i < KV; ++i) {
            const uint32_t w[4] = {k[x][i].x, k[x][i].y, k[x][i].z, k[x][i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int st = 4 * i + e;
              const uint32_t qa[4] = {q[st][0][0], R16 ? q[st][0][HR - 1] : 0u, q[st][1][0], R16 ? q[st][1][HR - 1] : 0u};
              fd_mma(s[x], qa, widen2(w[e] & 0xffffu), widen2(w[e] >> 16));
            }
          }
        }
      }
      const float ks0 = ks[0], ks1 = ks[1], vs0 = vs[0], vs1 = vs[1];
      // the next step's K and scales
      load_k(t + 1, pg1);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        ks[x] = pg1[x] >= 0 ? ksb[pg1[x] * a.pool.ks_s0] : 0.f;
        vs[x] = pg1[x] >= 0 ? vsb[pg1[x] * a.pool.vs_s0] : 0.f;
      }
      if (some) {
        const bool masked = pg[0] < 0 || pg[1] < 0 || !p.k.all(A, j0, 16);
#pragma unroll
        for (int x = 0; x < HR; ++x) {
          const float c0 = fminf(qscale[x] * ks0, 3e38f), c1 = fminf(qscale[x] * ks1, 3e38f);
          s[0][2 * x] *= c0, s[0][2 * x + 1] *= c0;
          s[1][2 * x] *= c1, s[1][2 * x + 1] *= c1;
        }
        if (masked) {
          uint32_t seen = 0, mine[HR];
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            uint32_t b = (uint32_t)sees[x].bits(A, p.b, p.k.len, j0, 16);
            if (pg[0] < 0) b &= 0xff00u;
            if (pg[1] < 0) b &= 0x00ffu;
            mine[x] = b;
            seen |= b;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              if (!((b >> (8 * y + 2 * tig)) & 1)) s[y][2 * x] = -INFINITY;
              if (!((b >> (8 * y + 2 * tig + 1)) & 1)) s[y][2 * x + 1] = -INFINITY;
            }
          }
          // V of keys that no row sees is cleared; NaN of those that some see is taken out, and given to these
          seen = __reduce_or_sync(0xffffffffu, seen);
          uint32_t nan = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool see = (seen >> (8 * (c >> 1) + 2 * tig + (c & 1))) & 1;
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              if (!see) v[c][w] = 0;
              nan |= __vcmpeq4(v[c][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            }
          }
          if (__any_sync(0xffffffffu, nan)) {
#pragma unroll
            for (int e = 0; e < VB; ++e) {
              uint32_t at = 0;  // the keys whose element e of this lane's columns is NaN, over the lanes of the column
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (((v[c][e >> 2] >> (8 * (e & 3))) & 0x7f) == 0x7f) {
                  at |= 1u << (8 * (c >> 1) + 2 * tig + (c & 1));
                  v[c][e >> 2] &= ~(0xffu << (8 * (e & 3)));
                }
              at |= __shfl_xor_sync(0xffffffffu, at, 1);
              at |= __shfl_xor_sync(0xffffffffu, at, 2);
#pragma unroll
              for (int x = 0; x < HR; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {  // rows 8 x + 2 tig + y
                  const uint32_t b = __shfl_sync(0xffffffffu, mine[x], 4 * (2 * tig + y));
                  if (b & at) o[x][e >> 1][2 * (e & 1) + y] = __uint_as_float(0x7fffffffu);
                }
            }
          }
        }
        // the reference moves where some row's maximum has outgrown it
        float top[HR];
        bool over = false;
#pragma unroll
        for (int x = 0; x < HR; ++x) {
          top[x] = fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1]));
          over = over || top[x] > m[x] + kFdSlack;
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
            const float mn = top[x] > m[x] + kFdSlack ? top[x] : m[x];
            const float f = mn == m[x] ? 1.f : ex2(m[x] - mn);
            m[x] = mn;
            l[x] *= f;
            const float f0 = __shfl_sync(0xffffffffu, f, 8 * tig), f1 = __shfl_sync(0xffffffffu, f, 8 * tig + 4);
#pragma unroll
            for (int e = 0; e < VB / 2; ++e) o[x][e][0] *= f0, o[x][e][1] *= f1, o[x][e][2] *= f0, o[x][e][3] *= f1;
          }
        }
        const float vmax = fmaxf(vs0, vs1);
        if (vmax > vref) {  // (the same in every lane)
          const float f = vref / vmax;
#pragma unroll
          for (int x = 0; x < HR; ++x)
#pragma unroll
            for (int e = 0; e < VB / 2; ++e) o[x][e][0] *= f, o[x][e][1] *= f, o[x][e][2] *= f, o[x][e][3] *= f;
          vref = vmax;
        }
        const float inv = 1.f / vref, f0 = vs0 * inv, f1 = vs1 * inv;
        uint32_t b0[HR], b1[HR];
#pragma unroll
        for (int x = 0; x < HR; ++x) {
          const float ref = (m[x] == -INFINITY ? 0.f : m[x]) - kFdBias;
          const float p0 = ex2(s[0][2 * x] - ref), p1 = ex2(s[0][2 * x + 1] - ref);
          const float p2 = ex2(s[1][2 * x] - ref), p3 = ex2(s[1][2 * x + 1] - ref);
          l[x] += (p0 + p1) + (p2 + p3);
          b0[x] = pack_half(p0 * f0, p1 * f0);
          b1[x] = pack_half(p2 * f1, p3 * f1);
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t lo0 = __byte_perm(v[0][w], v[1][w], 0x5140), lo1 = __byte_perm(v[2][w], v[3][w], 0x5140);
          const uint32_t hi0 = __byte_perm(v[0][w], v[1][w], 0x7362), hi1 = __byte_perm(v[2][w], v[3][w], 0x7362);
          const uint32_t va[4] = {widen2(lo0 & 0xffffu), widen2(lo0 >> 16), widen2(lo1 & 0xffffu), widen2(lo1 >> 16)};
          const uint32_t vc[4] = {widen2(hi0 & 0xffffu), widen2(hi0 >> 16), widen2(hi1 & 0xffffu), widen2(hi1 >> 16)};
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            fd_mma(o[x][2 * w], va, b0[x], b1[x]);
            fd_mma(o[x][2 * w + 1], vc, b0[x], b1[x]);
          }
        }
      }
      load_v(t + 1, pg1);
      pg[0] = pg1[0], pg[1] = pg1[1];
      pg1[0] = pg2[0], pg1[1] = pg2[1];
    }
    // ---- the warps' parts, joined --------------------------------------------------
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      const int r = gid + 8 * x;
      if (tig == 0) {
        wm[warp * ROWS + r] = m[x] - kFdBias;
        wl[warp * ROWS + r] = l[x];
      }
      float* o0 = wo + (warp * ROWS + 8 * x + 2 * tig) * D + VB * gid;
#pragma unroll
      for (int e = 0; e < VB / 2; ++e) {
        *reinterpret_cast<float2*>(o0 + 2 * e) = make_float2(o[x][e][0] * vref, o[x][e][2] * vref);
        *reinterpret_cast<float2*>(o0 + D + 2 * e) = make_float2(o[x][e][1] * vref, o[x][e][3] * vref);
      }
    }
    __syncthreads();
    const bool whole = p.t0 == 0 && p.t1 == p.tiles;
    for (int e = tid; e < p.rows * (D / 4); e += NT) {
      const int r = e / (D / 4), c = e % (D / 4) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, wm[w * ROWS + r]);
      float sum = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float mw = wm[w * ROWS + r], f = mw == mx ? 1.f : ex2(mw - mx);
        sum = fmaf(wl[w * ROWS + r], f, sum);
        const float4 z = *reinterpret_cast<const float4*>(wo + (w * ROWS + r) * D + c);
        y.x = fmaf(z.x, f, y.x), y.y = fmaf(z.y, f, y.y), y.z = fmaf(z.z, f, y.z), y.w = fmaf(z.w, f, y.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
      if (whole) {
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + out_row(A, p.b, p.h, p.k.n0, r) * D + c) =
            make_uint2(Out<T>::pack(y.x, y.y), Out<T>::pack(y.z, y.w));
      } else {
        const int64_t slot = slot_of(p);
        *reinterpret_cast<float4*>(A.part_o + (slot * A.rows_pad + r) * D + c) = y;
        if (c == 0) {
          A.part_ml[slot * 2 * A.rows_pad + r] = mx;
          A.part_ml[(slot * 2 + 1) * A.rows_pad + r] = sum;
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) {
    A.meta[blockIdx.x] = walk.meta;
    A.status[blockIdx.x] = 0;
  }
}

template <typename T, int D, bool R16>
int fd_launch(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  using S = FdShape<R16>;
  const Plan plan = fp8_decode_plan(a.Hq / a.Hkv * a.T, D);
  const Args A = make_args(a, plan, a.T, kFdLead, ws);
  auto kern = fp8_decode_kernel<T, D, R16>;
  static DeviceOnce done;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done.done(dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fd_smem<D, R16>()) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "cannot set attention_fp8 shared memory size %d", fd_smem<D, R16>());
    done.mark(dev);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(S::NT);
  cfg.dynamicSmemBytes = fd_smem<D, R16>();
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 launch: %s", cudaGetErrorString(e));
  int rc = check_launch("attention_fp8");
  if (rc || a.cap <= S::TK) return rc;  // a cache of one tile: nothing is split
  return launch_fp8_merge(A, dtype, plan.ctas, st);
}

template <typename T>
int fd_typed(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  if (a.Hq / a.Hkv * a.T > 8)
    return a.D == 128 ? fd_launch<T, 128, true>(a, dtype, ws, st) : fd_launch<T, 64, true>(a, dtype, ws, st);
  return a.D == 128 ? fd_launch<T, 128, false>(a, dtype, ws, st) : fd_launch<T, 64, false>(a, dtype, ws, st);
}

}  // namespace

fa::Plan fp8_decode_plan(int rows, int D) {
  const bool r16 = rows > 8;
  return make_plan(num_sms_current_device() * (r16 ? FdShape<true>::CTAS : FdShape<false>::CTAS), r16 ? 16 : 8, D);
}

int launch_fp8_decode(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  return dtype == DROPKV_DTYPE_BF16 ? fd_typed<__nv_bfloat16>(a, dtype, ws, st) : fd_typed<__half>(a, dtype, ws, st);
}

}  // namespace dropkv
