// Attention of a tree of drafted tokens over a cache: for sequence b, query head h
// and node i, O = sum_j softmax_j(scale q_i . k_j) v_j over the len_b cached rows
// and the tree's nodes j (rows len_b + j of the cache) that mask[i][j] shows.
//
// The M = g T query rows of a KV head read the same keys, so a tile of 128 keys is
// fetched once for up to 256 rows: 4 D bytes and 4 D M operations a key, which HBM
// bounds below about 250 rows and the tensor cores above. Both products run on
// them: S = Q K^T with Q and K in shared memory, O += P V with the weights P left in
// tensor memory, where S was. A warp for K and one for V issue the TMA loads (a box per
// page), one for each softmax group the products, and two groups of four warps do the
// softmax, a thread for each row:
//   * up to 128 rows: both groups have the same rows and take key tiles in turn,
//     each with a maximum, a sum and an output of its own, joined at the end;
//   * above: each group has 128 rows, and both use every key tile.
// Either way one group's softmax runs beside the products of the other.
//
// The keys of all (sequence, KV head, group of 256 rows) segments form one line of
// tiles that is cut evenly over the CTAs, one to an SM, from the lengths on the
// device: a ragged batch is balanced without the host knowing it. A segment that
// falls into several CTAs leaves partials (output, maximum, sum; fp32) in the
// workspace, and a second kernel joins them in the order of the CTAs. No CTA waits
// for another.
//
// Weights are rounded to 16 bits for the second product, as its operands have to be; sums are
// taken from the same weights before they are rounded, and products, sums and the joining
// are in fp32.
//
// What it measured alone: 295K keys in 8 sequences x 4 KV heads x 224 rows of 128, fp16 (135
// GFLOP, 604 MB): 150 us, 900 TFLOP/s (55% of a matrix product's burst rate) and 4.0 TB/s
// (61% of a copy's); with the merge, one after another in a graph, 166 to 178 us, and 200 from
// Python, as the clock falls under load. What bounds
// it is the chain of a group's tile, 3800 cycles: from S to its last weights 2500 (480 for the
// first half's logits and maximum, 1000 a half for weights), 440 until the products are
// issued, 860 until the next S is there; the other group's runs beside it. The tile's four
// products take 2048, its loads 2800 at a copy's rate. 13107 keys x 256 rows x 8 heads, bf16:
// 26 us, of which the tiles are 11; the rest is the start, the first tiles and the partials (20 MB
// out). With the merge 31 us in a graph, 33 over inputs larger than L2.
#include <algorithm>
#include <type_traits>

#include "tc_common.cuh"

namespace dropkv {
namespace {

constexpr int TA_TK = 128;               // keys of a tile
constexpr int TA_ROWS = 256;             // query rows of a segment
constexpr int TA_SM = 128;               // threads of a softmax group, one for each row
constexpr int TA_NT = 2 * TA_SM + 128;   // two softmax groups, a TMA warp for K and for V, an MMA warp for each group
constexpr int TA_WARP_TMA = 8, TA_WARP_MMA = 10;
constexpr uint64_t kTaWaitNs = 1000000000ull;
// The reference a row's weights are taken against is moved only when its maximum has
// grown by this much (base 2): weights then stay below 2^8, and the accumulated
// output, in tensor memory, is hardly ever rescaled.
constexpr float kTaSlack = 8.f;

// Division by a node count from 1 to 256 of numbers below 2^24.
struct TaDiv {
  uint32_t mul, d;
  __device__ __forceinline__ int quot(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, mul); }
};

struct TaArgs {
  TreeAttn a;
  TaDiv by_t;
  int g, M, RT;            // query rows of a KV head: M = g T, in RT segments of 256
  int HR;                  // segments of a sequence: Hkv RT
  int box;                 // rows of a TMA box
  int rows_pad;            // rows of a partial
  float scale_log2;
  int q_tma;               // Q comes by TMA, all rows of a KV head in a box for each slab
  int q_vec;               // else: its rows are read 16 bytes at a time
  int mask_vec;            // the mask's rows are read 4 bytes at a time
  float bias;              // weights are 2^(s - m + bias): fp16 has few bits below 1
  int* status;             // [CTAs]: 0, or which wait gave up
  float* part_o;           // [2 CTAs][D / 4][rows_pad] float4
  float* part_ml;          // [2 CTAs][2][rows_pad]
};

// per softmax group s: Q written, S ready, P ready (keys 0 to 63; and, at + 2, 64 to 127), O ready,
// its turn to issue, every product done, the products of a tile's first half done;
// both MMA warps have seen a piece's Q
enum { B_Q = 0, B_S = 2, B_P = 4, B_O = 8, B_T = 10, B_END = 12, B_H = 14, B_SEEN = 16, B_COUNT = 18 };

template <int D>
struct TaSmem {
  static constexpr int TILE = TA_TK * D * 2;  // K, V or Q tile: D / 64 slabs of 128 rows x 128 B
  static constexpr int SLOTS = D == 128 ? 5 : 10;
  static constexpr int Q = 0;                 // D / 64 slabs of 256 rows x 128 B: the groups' rows one after the other
  static constexpr int RING = 2 * TILE;
  static constexpr int BARS = RING + SLOTS * TILE;        // full[SLOTS], empty[SLOTS], then B_*
  static constexpr int BAD = BARS + (2 * SLOTS + B_COUNT) * 8;  // uint32 [2][8]: nodes with non-finite V
  static constexpr int ML = BAD + 64;                      // float [2][2][128]: the groups' maxima and sums
  static constexpr int MISC = ML + 2048;
  static constexpr int BYTES = MISC + 64;
};
static_assert(TaSmem<128>::BYTES <= 232448, "shared memory");

struct TaMisc {
  int w0, w1, base;  // this CTA's units, and the first unit of sequence b0
  int b0;
  uint32_t tmem;
  int dead;
};

// Keys of sequence b (cached rows and nodes that fit), its cached rows, its tiles.
__device__ __forceinline__ int ta_len(const TreeAttn& a, int b) { return min(max(a.cache_lens[b], 0), a.cap); }
__device__ __forceinline__ int ta_keys(const TreeAttn& a, int len) { return (int)min((int64_t)len + a.T, (int64_t)a.cap); }
__device__ __forceinline__ int ta_tiles(const TreeAttn& a, int b) { return (ta_keys(a, ta_len(a, b)) + TA_TK - 1) / TA_TK; }

// A CTA's part of one segment: tiles [t0, t1) of sequence b, KV head h, row group rt.
struct TaPiece {
  int b, h, rt, t0, t1, tiles, len, keys, rows;
  bool two;    // two groups of rows, else tiles in turn
};

// Steps through a CTA's pieces; every role has one of its own and sees the same. On the line
// each segment takes kTaLead units before its tiles, about what a further piece costs a CTA
// (Q, an output, an empty pipeline): a CTA that ends a segment gets that much less of the next.
constexpr int kTaLead = 4;
struct TaWalk {
  int w, w1, base;  // units
  int b;
  __device__ __forceinline__ bool next(const TaArgs& A, TaPiece& p) {
    const TreeAttn& a = A.a;
    while (w < w1) {
      p.b = b;
      p.len = ta_len(a, b);
      p.keys = ta_keys(a, p.len);
      p.tiles = (p.keys + TA_TK - 1) / TA_TK;
      const int units = p.tiles + kTaLead;
      const int rel = w - base, seg = rel / units, u0 = rel - seg * units;
      const int u1 = min(units, u0 + (w1 - w));
      p.t0 = max(u0 - kTaLead, 0);
      p.t1 = u1 - kTaLead;
      p.h = seg / A.RT;
      p.rt = seg % A.RT;
      p.rows = min(TA_ROWS, A.M - p.rt * TA_ROWS);
      p.two = p.rows > 128;
      w += u1 - u0;
      if (w - base == units * A.HR) {
        base = w;
        ++b;
      }
      if (p.t1 > p.t0) return true;
    }
    return false;
  }
};

template <typename T>
struct TaType;
template <>
struct TaType<__nv_bfloat16> {
  using Two = __nv_bfloat162;
  static __device__ __forceinline__ Two two(float x) { return __float2bfloat162_rn(x); }
  static constexpr uint32_t kInf = 0x7F80u;  // the exponent bits
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct TaType<__half> {
  using Two = __half2;
  static __device__ __forceinline__ Two two(float x) { return __float2half2_rn(x); }
  static constexpr uint32_t kInf = 0x7C00u;
  static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

__device__ __forceinline__ float ta_ex2(float x) {  // 2^x, hardware approximation; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t ta_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void ta_unpair(uint64_t r, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t ta_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t ta_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ta_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What a partial of maximum m weighs under the joint maximum `to`; parts that saw
// nothing (or NaN alone) have -inf, which must not turn into NaN (or hide it).
__device__ __forceinline__ float ta_factor(float m, float to) { return m == to ? 1.f : ta_ex2(m - to); }

// A word with its non-finite halves zeroed.
template <typename T>
__device__ __forceinline__ uint32_t ta_finite(uint32_t x) {
  constexpr uint32_t E = TaType<T>::kInf;
  if ((x & E) == E) x &= 0xFFFF0000u;
  if ((x & (E << 16)) == (E << 16)) x &= 0x0000FFFFu;
  return x;
}

__device__ __forceinline__ void ta_softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(TA_NT, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ CUtensorMap qmap, const __grid_constant__ TaArgs A) {
  using L = TaSmem<D>;
  constexpr int SLABS = D / 64, NS = L::SLOTS;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t sm[];  // swizzled tiles start on multiples of 1024
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::BARS);
  uint64_t* empty = full + NS;
  uint64_t* bars = empty + NS;
  uint32_t* bad = reinterpret_cast<uint32_t*>(sm + L::BAD);
  TaMisc* misc = reinterpret_cast<TaMisc*>(sm + L::MISC);
  volatile int* dead = &misc->dead;
  const TreeAttn& a = A.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tc::smem_addr(sm) % 1024) {  // as declared; nothing may run on any other layout
    pdl_wait();
    pdl_launch_dependents();
    if (tid == 0) A.status[blockIdx.x] = 9;
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 2);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(&bars[B_Q + s], A.q_tma ? 1 : TA_SM / 32);
      tc::mbar_init(&bars[B_S + s], 1);
      tc::mbar_init(&bars[B_P + s], TA_SM / 32);
      tc::mbar_init(&bars[B_P + 2 + s], TA_SM / 32);
      tc::mbar_init(&bars[B_O + s], 1);
      tc::mbar_init(&bars[B_T + s], 1);
      tc::mbar_init(&bars[B_END + s], 1);
      tc::mbar_init(&bars[B_H + s], 1);
    }
    tc::mbar_init(&bars[B_SEEN], 2);
    tc::fence_mbar_init();
    misc->dead = 0;
  }
  if (tid < 16) bad[tid] = 0;
  if (warp == TA_WARP_MMA) {
    tc::tmem_alloc(&misc->tmem, 512);
    tc::tmem_relinquish();
  }
  if (warp == TA_WARP_TMA && lane == 0) {
    tc::tma_prefetch_desc(&kmap);
    tc::tma_prefetch_desc(&vmap);
    if (A.q_tma) tc::tma_prefetch_desc(&qmap);
  }
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: the merge may then read this kernel's inputs at once)
  if (warp == 0) {  // where this CTA's share of the line of tiles starts
    const int own0 = lane < a.B ? ta_tiles(a, lane) + kTaLead : 0;
    int total = own0;
    for (int b = lane + 32; b < a.B; b += 32) total += ta_tiles(a, b) + kTaLead;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int W = total * A.HR, per = (W + (int)gridDim.x - 1) / (int)gridDim.x;
    const int w0 = min((long long)W, (long long)per * blockIdx.x), w1 = min(W, w0 + per);
    if (w0 < w1) {
      int before = 0;
      for (int c = 0; c < a.B; c += 32) {
        const int own = c == 0 ? own0 : (c + lane < a.B ? ta_tiles(a, c + lane) + kTaLead : 0);
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, (before + upto) * A.HR > w0);
        if (past) {
          const int at = __ffs(past) - 1;
          if (lane == at) {
            misc->b0 = c + at;
            misc->base = (before + upto - own) * A.HR;
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) {
      misc->w0 = w0;
      misc->w1 = w1;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = misc->tmem;
  TaWalk walk{misc->w0, misc->w1, misc->base, misc->b0};
  TaPiece p;
  // a wait that gives up marks the CTA dead: every role then ends without waiting
  int code = 0;
  auto wait = [&](uint64_t* bar, uint32_t count, int why) {  // for the count-th completion (from 0)
    if (tc::mbar_try_wait(bar, count & 1)) return true;
    const uint64_t t0 = tc::globaltimer_ns();
    while (!*dead) {
      if (tc::mbar_try_wait(bar, count & 1)) return true;
      if (tc::globaltimer_ns() - t0 > kTaWaitNs) *dead = code = why;
    }
    return false;
  };

  // Load numbers from a piece's first on: K_i is number i (i < lead) or lead + 2 (i - lead) + 1, V_i
  // number lead + 2 i, short of the K loads that do not exist; the order of use, in which K runs one
  // tile ahead of V (two where the groups take tiles in turn). Load number n uses slot n % NS.
  auto k_load = [&](int i, int lead) { return i < lead ? i : 2 * i - lead + 1; };
  auto v_load = [&](int i, int lead, int nt) { return min(lead, nt) + i + min(i, max(nt - lead, 0)); };

  if (warp == TA_WARP_TMA || warp == TA_WARP_TMA + 1) {
    // ======================= TMA producers: K tiles, V tiles ====================
    const bool is_v = __shfl_sync(0xffffffffu, warp, 0) != TA_WARP_TMA;
    const CUtensorMap* map = is_v ? &vmap : &kmap;
    const int boxes = TA_TK / A.box;
    uint32_t base = 0;  // load number of the piece's first
    uint32_t last = 0, any = 0, before = 0;  // `before`: loads of the pieces before the one before
    int nt_before = 0, lead_before = 0, queries = 0;
    while (walk.next(A, p)) {
      const int nt = __shfl_sync(0xffffffffu, p.t1 - p.t0, 0), lead = __shfl_sync(0xffffffffu, p.two ? 1 : 2, 0);
      const int h = __shfl_sync(0xffffffffu, p.h, 0), b = __shfl_sync(0xffffffffu, p.b, 0);
      const int t0 = __shfl_sync(0xffffffffu, p.t0, 0);
      // the page of a lane's box of a tile: -1 past the keys
      auto page_of = [&](int i) {
        const int key = (t0 + i) * TA_TK + lane * A.box;
        return i < nt && lane < boxes && key < p.keys ? a.table[(int64_t)b * a.max_blocks + key / a.block] : -1;
      };
      int page = a.table ? page_of(0) : 0;
      bool ok = true;
      if (A.q_tma && !is_v) {
        // the piece's Q, once the products that read the last one's are done: those with its last
        // K tile (of each group)
        if (base)
          for (int i = max(nt_before - lead_before, 0); i < nt_before; ++i) {
            const uint32_t k = before + k_load(i, lead_before);
            ok = __all_sync(0xffffffffu, ok && wait(&empty[k % NS], k / NS, 12));
          }
        // and once both MMA warps have seen the last one: a warp without work in that piece may
        // still be at the one before, and a barrier two phases on looks as if it had not moved
        if (queries) ok = __all_sync(0xffffffffu, ok && wait(&bars[B_SEEN], queries - 1, 11));
        if (!ok) break;
        if (tc::elect_one()) {
          tc::mbar_arrive_expect_tx(&bars[B_Q], A.M * 128 * SLABS);
#pragma unroll
          for (int s = 0; s < SLABS; ++s)
            tc::tma_load_4d(sm + L::Q + s * (TA_ROWS * 128), &qmap, &bars[B_Q], 64 * s, 0, h * A.g, b);
        }
        __syncwarp();
        ++queries;
      }
      for (int i = 0; i < nt; ++i) {
        const int next = a.table ? page_of(i + 1) : 0;
        const uint32_t k = base + (is_v ? v_load(i, lead, nt) : k_load(i, lead)), slot = k % NS;
        // The load before in this slot may be the other producer's. That it has landed says that the one
        // before it had left; while that is not known, a slot two loads back looks free.
        ok = k < (uint32_t)NS || (wait(&full[slot], k / NS - 1, 13) && wait(&empty[slot], k / NS - 1, 1));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* dst = sm + L::RING + slot * L::TILE;
        if (tc::elect_one()) tc::mbar_arrive_expect_tx(&full[slot], L::TILE);
        __syncwarp();
        const int key0 = (t0 + i) * TA_TK;
        if (!a.table) {
          if (tc::elect_one()) {
#pragma unroll
            for (int s = 0; s < SLABS; ++s)
              tc::tma_load_4d(dst + s * (TA_TK * 128), map, &full[slot], 64 * s, key0, h, b);
          }
          __syncwarp();
        } else {
          // on no page of the pool: out of range, and read as zeros
          const int there = page < 0 || page > a.n_pages ? a.n_pages : page;
          const int row = a.block > TA_TK ? key0 & (a.block - 1) : 0;
          auto issue = [&](auto count) {  // the boxes of a tile, all by one lane
            constexpr int N = decltype(count)::value;
            int at[N];
#pragma unroll
            for (int x = 0; x < N; ++x) at[x] = __shfl_sync(0xffffffffu, there, x);
            if (tc::elect_one()) {
#pragma unroll
              for (int x = 0; x < N; ++x)
#pragma unroll
                for (int s = 0; s < SLABS; ++s)
                  tc::tma_load_4d(dst + s * (TA_TK * 128) + x * (TA_TK / N) * 128, map, &full[slot], 64 * s, row, h, at[x]);
            }
            __syncwarp();
          };
          if (boxes == 1)
            issue(std::integral_constant<int, 1>());
          else if (boxes == 2)
            issue(std::integral_constant<int, 2>());
          else if (boxes == 4)
            issue(std::integral_constant<int, 4>());
          else if (boxes == 8)
            issue(std::integral_constant<int, 8>());
          else
            issue(std::integral_constant<int, 16>());
        }
        last = k, any = 1;
        page = next;
      }
      if (!ok) break;
      before = base;
      nt_before = nt;
      lead_before = lead;
      base += 2 * nt;
    }
    if (*dead && (any || queries)) {  // every issued copy lands before the CTA may exit
      for (uint32_t j = last >= (uint32_t)NS ? last - NS + 1 : 0u; j <= last; ++j)  // (some are the other's, or not issued)
        tc::mbar_wait(&full[j % NS], (j / NS) & 1, kTaWaitNs / 8);
      if (queries) tc::mbar_wait(&bars[B_Q], (queries - 1) & 1, kTaWaitNs);
    }
  } else if (warp >= TA_WARP_MMA) {
    // ======================= MMA issuers ========================================
    // A warp for each softmax group, in turns: while one issues the products of its item (a
    // tile of its group), the other waits for its own data. The products of one group then run
    // beside the softmax of the other. (Without turns the tensor cores served both at once, the
    // groups fell into step and nothing overlapped: 295K keys x 224 rows in 210 us, with turns 180;
    // now 151.)
    // The whole warp runs this and one lane issues, so that counts, addresses and descriptors
    // can stay in uniform registers.
    constexpr uint32_t ID_QK = tc::idesc_f16(BF16, 128, TA_TK, false, false);
    constexpr uint32_t ID_PV = tc::idesc_f16(BF16, 128, D, false, true);
    constexpr uint32_t LBO_V = SLABS == 2 ? TA_TK * 128 : 0;
    const int s = __shfl_sync(0xffffffffu, warp - TA_WARP_MMA, 0);
    const uint32_t ts = __shfl_sync(0xffffffffu, tmem, 0) + s * 128, to = ts + 256;
    const uint32_t ring0 = __shfl_sync(0xffffffffu, tc::smem_addr(sm + L::RING), 0);
    const uint32_t q0 = __shfl_sync(0xffffffffu, tc::smem_addr(sm + L::Q), 0);
    uint32_t base = 0, n_q = 0, n_p = 0, n_t = 0, pieces = 0;
    bool handed = false;  // group 1 issued the last item of the piece before, and handed the turn over
    bool ok = true;
    while (ok && walk.next(A, p)) {
      const int two = __shfl_sync(0xffffffffu, (int)p.two, 0), nt = __shfl_sync(0xffffffffu, p.t1 - p.t0, 0);
      const int lead = two ? 1 : 2, step = lead, first = two ? 0 : s;
      // tiles in turn: by TMA there is one copy of the rows, for both groups
      const uint64_t qd = tc::smem_desc(q0 + (A.q_tma && !two ? 0 : s * (128 * 128)), 16, 1024);
      auto release = [&](uint64_t* bar) {  // two arrivals empty a slot: one of each group, or both of its only one
        tc::mma_commit(bar);
        if (!two) tc::mma_commit(bar);
      };
      auto qk = [&](uint32_t slot, bool shared = false) {
        const uint64_t kd = tc::smem_desc(ring0 + slot * L::TILE, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          tc::mma_f16(ts, tc::desc_add(qd, (kk / 4) * (TA_ROWS * 128) + (kk % 4) * 32),
                      tc::desc_add(kd, (kk / 4) * (TA_TK * 128) + (kk % 4) * 32), ID_QK, kk > 0);
        }
        tc::mma_commit(&bars[B_S + s]);
        if (shared)
          tc::mma_commit(&empty[slot]);  // the other arrival is the other group's
        else
          release(&empty[slot]);
      };
      if (A.q_tma) {  // every piece's Q is waited for, with work in it or without
        ok = __all_sync(0xffffffffu, wait(&bars[B_Q], pieces, 2));
        if (ok && tc::elect_one()) tc::mbar_arrive(&bars[B_SEEN]);
        __syncwarp();
      }
      if (first < nt && ok) {  // the first product, out of turn: nothing is running yet
        const uint32_t at = base + k_load(first, lead), slot = at % NS;
        ok = (A.q_tma || wait(&bars[B_Q + s], n_q++, 2)) && wait(&full[slot], at / NS, 3);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          tc::tc_fence_after();
          if (tc::elect_one()) qk(slot, s == 1 && !two);
          __syncwarp();
        }
      }
      if (!two && s == 0 && nt > 1 && ok) {
        // K_1 is group 1's alone, and the slot it frees takes (of five) V_2, whose landing group 0's
        // softmax waits for where the tile has nodes. All else that lands before V_2 in a slot of it is
        // behind this warp's products by then; K_1 is not, and as long as it is under way the barrier
        // looks as if V_2 had landed. So this warp sees it land, before its slot is free again.
        const uint32_t at = base + k_load(1, lead), slot = at % NS;
        ok = __all_sync(0xffffffffu, wait(&full[slot], at / NS, 3));
        if (ok && tc::elect_one()) tc::mbar_arrive(&empty[slot]);
        __syncwarp();
      }
      for (int i = first; i < nt && ok; i += step) {
        const uint32_t at = base + v_load(i, lead, nt), slot = at % NS;
        const uint32_t kat = base + k_load(i + step, lead), kslot = kat % NS;
        const uint64_t vd = tc::smem_desc(ring0 + slot * L::TILE, LBO_V, 1024);
        const bool more = i + step < nt;
        // the group's turn comes when the other has issued the item before this one. Its own loads
        // are waited for after that: the load before one in its slot may be the other group's, and
        // while that is not there its phase looks like this one's
        if (s == 1 || i > first || handed) ok = wait(&bars[B_T + s], n_t++, 10);
        ok = ok && wait(&full[slot], at / NS, 4) && (!more || wait(&full[kslot], kat / NS, 3));
        for (int half = 0; half < 2 && ok; ++half) {
          ok = __all_sync(0xffffffffu, ok && wait(&bars[B_P + 2 * half + s], n_p, 5));
          if (!ok) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < TA_TK / 32; ++kk)
              tc::mma_f16_tmem_a(to, ts + half * 32 + kk * 8, tc::desc_add(vd, half * (TA_TK * 64) + kk * 2048), ID_PV,
                                 i > first || half > 0 || kk > 0);
            if (half == 0) tc::mma_commit(&bars[B_H + s]);
          }
          __syncwarp();
        }
        if (!ok) break;
        ++n_p;
        if (tc::elect_one()) {
          release(&empty[slot]);
          if (more)
            qk(kslot);
          else
            tc::mma_commit(&bars[B_O + s]);
          // the next item is the other group's; after a piece's last it is group 0's
          if (s == 1 || two || i + 1 < nt) tc::mbar_arrive(&bars[B_T + 1 - s]);
        }
        __syncwarp();
      }
      base += 2 * nt;
      ++pieces;
      handed = two || nt % 2 == 0;
    }
    if (*dead) {  // no product may run on when tensor memory is given back
      if (tc::elect_one()) tc::mma_commit(&bars[B_END + s]);
      __syncwarp();
      tc::mbar_wait(&bars[B_END + s], 0, kTaWaitNs);
    }
  } else {
    // ======================= softmax groups =====================================
    // group s, its TMEM lane (row) and its warp's quarter of the lanes
    const int s = warp >> 2, quad = warp & 3, r = tid & 127;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + lanes + s * 128, to = tmem + lanes + 256;
    float* ml0 = reinterpret_cast<float*>(sm + L::ML);  // [2][128]: maxima, sums
    float* ml1 = ml0 + 256;
    uint32_t n_s = 0, n_o = 0, base = 0;
    bool ok = true;
    for (int piece = 0; walk.next(A, p); ++piece) {
      const int nt = p.t1 - p.t0;
      const bool mine = p.two || s < nt;  // this group has work in the piece
      const int row0 = p.rt * TA_ROWS + (p.two ? s * 128 : 0);  // the group's first row
      const int rows = min(128, A.M - row0);
      const bool live = quad * 32 < rows;  // some row of this warp exists
      uint32_t* bad_now = bad + 8 * (piece & 1);
      float m = -INFINITY, l = 0.f;
      if (mine && !A.q_tma) {
        // Q rows into shared memory, 16 bytes a thread and step: row = head of the group, then
        // node. The loads of four steps are on their way before the first is stored.
        const T* qb = static_cast<const T*>(a.q) + p.b * a.q_sb + (int64_t)p.h * A.g * a.q_sh;
        constexpr int STEP = TA_SM / (D / 8);  // rows a step of the group covers
        const int c = r % (D / 8);             // a thread's column of vectors stays, its row moves on
#pragma unroll 1
        for (int e0 = r / (D / 8); e0 < 128; e0 += 4 * STEP) {  // (rolled: code that runs once is fetched as it runs)
          uint4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int mrow = row0 + min(e0 + i * STEP, rows - 1), head = A.by_t.quot(mrow);
            const T* src = qb + head * a.q_sh + (mrow - head * a.T) * a.q_ss + c * 8 * a.q_sd;
            if (A.q_vec) {
              x[i] = *reinterpret_cast<const uint4*>(src);
            } else {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
              x[i].x = h[0] | (uint32_t)h[a.q_sd] << 16;
              x[i].y = h[2 * a.q_sd] | (uint32_t)h[3 * a.q_sd] << 16;
              x[i].z = h[4 * a.q_sd] | (uint32_t)h[5 * a.q_sd] << 16;
              x[i].w = h[6 * a.q_sd] | (uint32_t)h[7 * a.q_sd] << 16;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = e0 + i * STEP;
            if (row >= rows) x[i] = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(sm + L::Q + (c / 8) * (TA_ROWS * 128) + s * (128 * 128) +
                                      tc::sw128_offset(row, (c % 8) * 8)) = x[i];
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bars[B_Q + s]);
      }
      const int lead = p.two ? 1 : 2, step = lead;
      for (int i = p.two ? 0 : s; i < nt && ok; i += step) {
        const int j0 = (p.t0 + i) * TA_TK;
        // the page of a lane's box of the tile, looked at once S is there
        int page = 0;
        if (a.table) {
          const int key = j0 + lane * A.box;
          if (lane < TA_TK / A.box && key < p.keys) page = a.table[(int64_t)p.b * a.max_blocks + key / a.block];
        }
        const bool tree = j0 + TA_TK > p.len;  // the tile holds nodes, or ends the keys
        uint32_t see[4] = {0u, 0u, 0u, 0u};    // the keys of the tile that this thread's row sees
        if (tree && live) {
          const int mrow = row0 + min(r, rows - 1), node = mrow - A.by_t.quot(mrow) * a.T, fit = p.keys - p.len;
          const uint8_t* mr = a.mask ? a.mask + p.b * a.mask_sb + node * a.mask_sr : nullptr;
          const int n0 = j0 - p.len, q0 = n0 >> 5;  // the tile's first node, and its word of 32 nodes (rounded down)
          uint32_t words[5];                         // words q0 .. q0 + 4 of what the row sees
          if (mr && A.mask_vec) {
            uint32_t x[5][8];
#pragma unroll
            for (int w = 0; w < 5; ++w)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int n = 32 * (q0 + w) + 4 * e;
                x[w][e] = n >= 0 && n < fit ? *reinterpret_cast<const uint32_t*>(mr + n) : 0u;
              }
#pragma unroll
            for (int w = 0; w < 5; ++w) {
              words[w] = 0;
#pragma unroll
              for (int e = 0; e < 8; ++e) {  // four truth values to four bits
                const uint32_t y = __vcmpne4(x[w][e], 0u) & 0x01010101u;
                words[w] |= ((y * 0x10204080u) >> 28) << (4 * e);
              }
            }
          } else {
#pragma unroll
            for (int w = 0; w < 5; ++w) {
              words[w] = 0;
              if (32 * (q0 + w) + 32 <= 0 || 32 * (q0 + w) >= fit) continue;
#pragma unroll 8
              for (int e = 0; e < 32; ++e) {
                const int n = 32 * (q0 + w) + e;
                if (n >= 0 && n < fit && (mr ? mr[n * a.mask_sc] != 0 : n <= node)) words[w] |= 1u << e;
              }
            }
          }
#pragma unroll
          for (int w = 0; w < 5; ++w) {  // every cached row is seen, nothing past the last node that fits
            const int n = 32 * (q0 + w);
            if (n < 0) words[w] = 0xffffffffu;
            if (n + 32 > fit) words[w] &= n >= fit ? 0u : 0xffffffffu >> (32 - (fit - n));
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) see[w] = __funnelshift_r(words[w], words[w + 1], n0 & 31);
        }
        ok = __all_sync(0xffffffffu, wait(&bars[B_S + s], n_s++, 6));
        if (!ok) break;
        uint32_t gone = 0;  // which of the tile's pages are missing: 16 bits, from 8 rows up
        if (a.table) gone = __ballot_sync(0xffffffffu, page < 0 || page >= a.n_pages);
        if (gone) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (!tree) see[w] = 0xffffffffu;
            for (int key = 0; key < 32; key += 8)  // boxes have 8 rows at least
              if ((gone >> ((32 * w + key) / A.box)) & 1) see[w] &= ~(0xffu << key);
          }
        }
        tc::tc_fence_after();
        if (tree) {
          // rows of V that a weight of 0 would not silence: past the keys they are cleared, and
          // non-finite values of a node are taken out here and given to its viewers at the end
          const uint32_t at = base + v_load(i, lead, nt), slot = at % NS;
          ok = __all_sync(0xffffffffu, wait(&full[slot], at / NS, 7));
          if (!ok) break;
          const int key = j0 + r;
          if (key >= p.len) {
            uint8_t* row = sm + L::RING + slot * L::TILE + r * 128;
            auto vec = [&](int c) {  // lanes start at different columns: no bank conflicts
              return reinterpret_cast<uint4*>(row + (c / 8) * (TA_TK * 128) + ((c + r) % 8) * 16);
            };
            constexpr int VECS = SLABS * 8;
            bool off = false;
            if (key >= p.keys) {
#pragma unroll
              for (int c = 0; c < VECS; ++c) *vec(c) = make_uint4(0u, 0u, 0u, 0u);
            } else {
              using T2 = typename TaType<T>::Two;
              T2 z = TaType<T>::two(0.f);  // stays 0 unless some value is infinite or NaN
#pragma unroll
              for (int c = 0; c < VECS; ++c) {
                const uint4 v = *vec(c);
                z = __hfma2(reinterpret_cast<const T2&>(v.x), TaType<T>::two(0.f), z);
                z = __hfma2(reinterpret_cast<const T2&>(v.y), TaType<T>::two(0.f), z);
                z = __hfma2(reinterpret_cast<const T2&>(v.z), TaType<T>::two(0.f), z);
                z = __hfma2(reinterpret_cast<const T2&>(v.w), TaType<T>::two(0.f), z);
              }
              off = __hisnan(z.x) || __hisnan(z.y);
            }
            if (off) {
#pragma unroll 1
              for (int c = 0; c < VECS; ++c) {
                uint4 v = *vec(c);
                v.x = ta_finite<T>(v.x);
                v.y = ta_finite<T>(v.y);
                v.z = ta_finite<T>(v.z);
                v.w = ta_finite<T>(v.w);
                *vec(c) = v;
              }
              atomicOr(&bad_now[(key - p.len) >> 5], 1u << ((key - p.len) & 31));
            }
          }
          tc::fence_proxy_async_smem();
        }
        if (live) {
          const bool masked = tree || gone;
          const bool first = i < step;
          const uint64_t scale2 = ta_pair(A.scale_log2, A.scale_log2);
          // S is read once, a half of 64 keys at a time (128 do not stay in registers): the half's
          // maximum decides whether the row's reference moves, then its weights overwrite it. The
          // first half's products start beside the second half's weights; where the second half
          // moves the reference, which is rare, they are waited for. (A pass for the maximum of all
          // 128, a second one for the weights and a polynomial in place of one ex2 in four took as
          // long for long caches and 2 us more for one layer's: 13107 keys x 256 rows 28.8 us, now
          // 26.5; with that polynomial here 28.8 too.)
          auto weigh = [&](auto hide, int h) {
            float x[64];
            tc::tmem_ld64(ts + 64 * h, x);
            if (decltype(hide)::value) {
#pragma unroll
              for (int e = 0; e < 64; ++e) x[e] = (see[2 * h + e / 32] >> (e & 31)) & 1 ? x[e] : -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 64; e += 2) mx[(e / 2) & 3] = ta_max3(mx[(e / 2) & 3], x[e], x[e + 1]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * A.scale_log2;
            const bool start = first && h == 0;
            if (__any_sync(0xffffffffu, start || top > m + kTaSlack)) {  // some row's reference moves
              if (h == 1) {
                ok = __all_sync(0xffffffffu, wait(&bars[B_H + s], n_s - 1, 7)) && ok;
                tc::tc_fence_after();
              }
              const float mn = start || top > m + kTaSlack ? top : m;
              const float alpha = mn == m ? 1.f : ta_ex2(m - mn);
              m = mn;
              l *= alpha;
              if (!start) {
                float o[16];
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                  tc::tmem_ld16(to + s * 128 + c, o);
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] *= alpha;
                  tc::tmem_st16(to + s * 128 + c, o);
                  tc::tmem_st_wait();
                }
              }
            }
            const float ref = (m == -INFINITY ? 0.f : m) - A.bias;
            const uint64_t ref2 = ta_pair(-ref, -ref);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const uint64_t y = ta_fma2(ta_pair(x[32 * w + e], x[32 * w + e + 1]), scale2, ref2);
                float u, v;
                ta_unpair(y, u, v);
                u = ta_ex2(u), v = ta_ex2(v);
                sum[(e / 2) & 1] = ta_add2(sum[(e / 2) & 1], ta_pair(u, v));
                pk[e / 2] = TaType<T>::pack(u, v);
              }
              tc::tmem_st16(ts + 32 * h + 16 * w, reinterpret_cast<const float*>(pk));
            }
            // (a sum for each half, whether or not a row beside this one moves its reference)
            float s0, s1, s2, s3;
            ta_unpair(sum[0], s0, s1);
            ta_unpair(sum[1], s2, s3);
            l += (s0 + s1) + (s2 + s3);
          };
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (masked)
              weigh(std::true_type(), h);
            else
              weigh(std::false_type(), h);
            tc::tmem_st_wait();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bars[B_P + 2 * h + s]);
          }
        } else {
          __syncwarp();
          if (lane == 0) {
            tc::mbar_arrive(&bars[B_P + s]);
            tc::mbar_arrive(&bars[B_P + 2 + s]);
          }
        }
      }
      base += 2 * nt;
      // ---- the piece's output ---------------------------------------------------
      if (mine && ok) ok = __all_sync(0xffffffffu, wait(&bars[B_O + s], n_o++, 8));
      m -= A.bias;  // the reference the weights were taken against
      float* ml = s ? ml1 : ml0;
      ml[r] = m;
      ml[128 + r] = l;
      ta_softmax_sync();
      tc::tc_fence_after();
      if (tid < 8) bad[8 * ((piece + 1) & 1) + tid] = 0;
      const bool whole = p.t0 == 0 && p.t1 == p.tiles;
      // tiles in turn: each group writes half the columns of the joined rows; else all of its own
      const int part = p.two ? 0 : s, width = p.two ? D : D / 2;
      float f0 = 1.f, f1 = 0.f;  // factors of the two outputs (own rows: of this one alone)
      if (!p.two) {
        m = ml0[r];
        l = ml0[128 + r];
        if (nt > 1) {
          const float m0 = m, m1 = ml1[r];
          m = fmaxf(m0, m1);
          f0 = ta_factor(m0, m);
          f1 = ta_factor(m1, m);
          l = l * f0 + ml1[128 + r] * f1;
        }
      }
      if (live && ok) {
        const bool own = r < rows;
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const int mrow = row0 + r;
        const int64_t out_row = ((int64_t)p.b * a.Hq + p.h * A.g) * a.T + mrow;  // heads of T rows follow one another
        const int slot = 2 * blockIdx.x + (p.t0 > 0 ? 0 : 1);
        const int prow = (p.two ? s * 128 : 0) + r;
        uint32_t any_bad = 0;
        if (p.t1 * TA_TK > p.len) {
#pragma unroll
          for (int i = 0; i < 8; ++i) any_bad |= bad_now[i];
        }
#pragma unroll 1
        for (int c = part * width; c < (part + 1) * width; c += 16) {
          float o[16];
          tc::tmem_ld16(to + (p.two ? s * 128 : 0) + c, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= f0;
          if (!p.two && nt > 1) {
            float o1[16];
            tc::tmem_ld16(to + 128 + c, o1);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(o1[e], f1, o[e]);
          }
          if (any_bad && own) {  // the non-finite values of the nodes this row sees
            const int node = mrow - A.by_t.quot(mrow) * a.T;
#pragma unroll 1
            for (int n = 0; n < a.T; ++n) {
              if (!((bad_now[n >> 5] >> (n & 31)) & 1)) continue;
              if (a.mask ? a.mask[p.b * a.mask_sb + node * a.mask_sr + n * a.mask_sc] == 0 : n > node) continue;
              const int key = p.len + n;
              const T* v = static_cast<const T*>(a.v) + p.h * a.v_sh;
              if (a.table) {
                const int page = a.table[(int64_t)p.b * a.max_blocks + key / a.block];
                v += page * a.v_s0 + (key % a.block) * a.v_ss;  // a page that was read
              } else {
                v += p.b * a.v_s0 + key * a.v_ss;
              }
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float y = to_f(v[c + e]);
                if (!isfinite(y)) o[e] += y;
              }
            }
          }
          if (own && whole) {
            T* dst = static_cast<T*>(a.out) + out_row * D + c;
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              uint4 y;
              y.x = TaType<T>::pack(o[e] * inv, o[e + 1] * inv);
              y.y = TaType<T>::pack(o[e + 2] * inv, o[e + 3] * inv);
              y.z = TaType<T>::pack(o[e + 4] * inv, o[e + 5] * inv);
              y.w = TaType<T>::pack(o[e + 6] * inv, o[e + 7] * inv);
              *reinterpret_cast<uint4*>(dst + e) = y;
            }
          } else if (own) {
            float4* po = reinterpret_cast<float4*>(A.part_o) + (int64_t)slot * (D / 4) * A.rows_pad + prow;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              po[((c + e) / 4) * (int64_t)A.rows_pad] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (own && !whole && part == 0) {
          float* pm = A.part_ml + (int64_t)slot * 2 * A.rows_pad + prow;
          pm[0] = m;
          pm[A.rows_pad] = l;
        }
      }
      tc::tc_fence_before();
      ta_softmax_sync();  // outputs are read: the next piece may overwrite them
      tc::tc_fence_after();
    }
  }
  if (code) *dead = code;
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == TA_WARP_MMA) tc::tmem_dealloc(tmem, 512);
  if (tid == 0) A.status[blockIdx.x] = *dead;
}

constexpr int TM_NT = 256;
constexpr int TM_WARPS = TM_NT / 32;
constexpr int TM_PIECES = 64;  // partials whose factors are held at once
constexpr int TM_AHEAD = 8;    // partials on their way at once

// Joins the partials of the segments that fell into several CTAs. Grid: (segments,
// 32-row blocks x blocks of 32 columns); a thread has a row and four columns. The
// partials lie [column / 4][row], so a warp reads 32 rows of 16 bytes in one piece.
// With m the largest of the partials' maxima, O = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m).
// Bound by the latency of its loads, from L2 mostly (19 partials of 256 rows x 128 x 8 heads,
// 20 MB: about 4 us after the kernel before it, whose end it is launched beside). The eight
// warps share out the partials' maxima and sums, while the first partials come.
template <typename T, int D>
__global__ void __launch_bounds__(TM_NT) tree_attn_merge_kernel(const __grid_constant__ TaArgs A, int ctas) {
  __shared__ int red[2][TM_WARPS];
  __shared__ float fac[TM_PIECES][32], mxs[TM_WARPS][32], sums[TM_WARPS][32];
  const TreeAttn& a = A.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / A.HR, seg = blockIdx.x % A.HR;
  const int rt = seg % A.RT, h = seg / A.RT;
  const int rb = blockIdx.y / (D / 32), cb = blockIdx.y % (D / 32);
  const int row = rb * 32 + lane, mrow = rt * TA_ROWS + row;
  // Every CTA waits for the kernel before this one before it ends, with work or without: what
  // comes after on the stream takes this kernel's end for the end of both.
  if (rt * TA_ROWS + rb * 32 >= A.M) {
    pdl_wait();
    return;
  }
  // the lengths were there before the kernel whose partials these are began: no wait yet
  int before = 0, total = 0;
  for (int i = tid; i < a.B; i += TM_NT) {
    const int t = ta_tiles(a, i) + kTaLead;
    total += t;
    before += i < b ? t : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) red[0][warp] = total, red[1][warp] = before;
  __syncthreads();
  total = before = 0;
#pragma unroll
  for (int w = 0; w < TM_WARPS; ++w) total += red[0][w], before += red[1][w];
  const int per = (total * A.HR + ctas - 1) / ctas, tiles = ta_tiles(a, b);
  const int w0 = before * A.HR + seg * (tiles + kTaLead) + kTaLead, w1 = w0 + tiles;
  const int c0 = w0 / per, n = (w1 - 1) / per - c0 + 1;
  if (n == 1) {  // written by its one CTA
    pdl_wait();
    return;
  }
  // partial i is CTA c0 + i's: the segment is the last piece of the first CTA, the first of the others
  auto slot = [&](int i) { return (int64_t)2 * (c0 + i) + (i == 0 ? 1 : 0); };
  const bool own = row < A.rows_pad && mrow < A.M;
  const float* pml = A.part_ml + row;
  const int q = cb * 8 + warp;  // the thread's group of four columns
  const float4* po = reinterpret_cast<const float4*>(A.part_o) + (int64_t)q * A.rows_pad + row;
  auto load = [&](int i, float4* x) {
#pragma unroll
    for (int u = 0; u < TM_AHEAD; ++u) x[u] = __ldcg(po + slot(min(i + u, n - 1)) * (D / 4) * A.rows_pad);
  };
  pdl_wait();
  float4 x[TM_AHEAD];
  if (own) load(0, x);
  float mine = -INFINITY;
  if (own) {
#pragma unroll 4
    for (int i = warp; i < n; i += TM_WARPS) mine = fmaxf(mine, __ldcg(pml + slot(i) * 2 * A.rows_pad));
  }
  mxs[warp][lane] = mine;
  __syncthreads();
  float m = mxs[0][lane];
#pragma unroll
  for (int w = 1; w < TM_WARPS; ++w) m = fmaxf(m, mxs[w][lane]);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += TM_PIECES) {
    const int cnt = min(TM_PIECES, n - i0);
    if (i0) __syncthreads();  // the factors before have been used
    for (int i = warp; i < cnt; i += TM_WARPS) {
      float f = 0.f;
      if (own) {
        const float* pm = pml + slot(i0 + i) * 2 * A.rows_pad;
        f = ta_factor(__ldcg(pm), m);
        l = fmaf(__ldcg(pm + A.rows_pad), f, l);
      }
      fac[i][lane] = f;
    }
    __syncthreads();
    if (own) {
      for (int i = 0; i < cnt; i += TM_AHEAD) {
        float4 y[TM_AHEAD];
        if (i0 + i + TM_AHEAD < n) load(i0 + i + TM_AHEAD, y);
#pragma unroll
        for (int u = 0; u < TM_AHEAD; ++u) {
          if (i + u < cnt) {
            const float f = fac[i + u][lane];
            o.x = fmaf(x[u].x, f, o.x);
            o.y = fmaf(x[u].y, f, o.y);
            o.z = fmaf(x[u].z, f, o.z);
            o.w = fmaf(x[u].w, f, o.w);
          }
          x[u] = y[u];
        }
      }
    }
  }
  sums[warp][lane] = l;
  __syncthreads();
  if (!own) return;
  l = sums[0][lane];
#pragma unroll
  for (int w = 1; w < TM_WARPS; ++w) l += sums[w][lane];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t out_row = ((int64_t)b * a.Hq + h * A.g) * a.T + mrow;  // heads of T rows follow one another
  uint2 y;
  y.x = TaType<T>::pack(o.x * inv, o.y * inv);
  y.y = TaType<T>::pack(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + out_row * D + 4 * q) = y;
}

struct TaPlan {
  int ctas, rows_pad;
  size_t off_o, off_ml, bytes;
};

TaPlan ta_plan(int Hq, int Hkv, int T, int D) {
  TaPlan p;
  p.ctas = num_sms_current_device();
  p.rows_pad = std::min(TA_ROWS, (Hq / Hkv * T + 31) / 32 * 32);
  p.off_o = align_up((size_t)p.ctas * 4, 256);
  p.off_ml = p.off_o + (size_t)2 * p.ctas * p.rows_pad * D * 4;
  p.bytes = align_up(p.off_ml + (size_t)2 * p.ctas * 2 * p.rows_pad * 4, 256);
  return p;
}

template <typename T, int D>
int ta_launch(const TreeAttn& a, int dtype, void* ws, cudaStream_t st) {
  using L = TaSmem<D>;
  const bool bf16 = dtype == DROPKV_DTYPE_BF16;
  const TaPlan plan = ta_plan(a.Hq, a.Hkv, a.T, D);
  TaArgs A;
  A.a = a;
  A.by_t.d = (uint32_t)a.T;
  A.by_t.mul = a.T == 1 ? 0u : (uint32_t)(((uint64_t(1) << 32) + a.T - 1) / a.T);
  A.g = a.Hq / a.Hkv;
  A.M = A.g * a.T;
  A.RT = (A.M + TA_ROWS - 1) / TA_ROWS;
  A.HR = a.Hkv * A.RT;
  // Keys of the last tile's boxes, units of the line and the end of the last CTA's share are counted in 32 bits.
  if (a.cap > 0x7fffffff - 64 * TA_TK)
    return fail(DROPKV_ERR_UNSUPPORTED, "tree attention: caches of up to %d rows are too long", a.cap);
  const int64_t units = (int64_t)a.B * A.HR * (((int64_t)a.cap + TA_TK - 1) / TA_TK + kTaLead);
  if (units + units / plan.ctas + plan.ctas > 0x7fffffff)
    return fail(DROPKV_ERR_UNSUPPORTED, "tree attention: %d sequences of up to %d rows are too many tiles", a.B, a.cap);
  A.box = a.table ? std::min(a.block, TA_TK) : TA_TK;
  A.rows_pad = plan.rows_pad;
  A.scale_log2 = a.scale * 1.4426950408889634f;
  A.bias = bf16 ? 0.f : 7.f;
  A.mask_vec = a.mask_sc == 1 && a.T % 4 == 0 && (reinterpret_cast<uintptr_t>(a.mask) | (uint64_t)(a.mask_sb | a.mask_sr)) % 4 == 0;
  A.q_vec = a.q_sd == 1 && (reinterpret_cast<uintptr_t>(a.q) | (uint64_t)((a.q_sb | a.q_sh | a.q_ss) * 2)) % 16 == 0;
  A.status = static_cast<int*>(ws);
  A.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + plan.off_o);
  A.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + plan.off_ml);
  const int n0 = a.table ? a.n_pages : a.B, rows = a.table ? a.block : a.cap;
  CUtensorMap km, vm, qm;
  int rc = make_kv_tensor_map_4d(&km, a.k, n0, a.Hkv, rows, D, bf16, a.k_s0, a.k_sh, a.k_ss, A.box);
  if (!rc) rc = make_kv_tensor_map_4d(&vm, a.v, n0, a.Hkv, rows, D, bf16, a.v_s0, a.v_sh, a.v_ss, A.box);
  if (rc) return rc;
  A.q_tma = A.q_vec && A.RT == 1 && make_head_tensor_map(&qm, a.q, a.B, a.Hq, a.T, D, bf16, a.q_sb, a.q_sh, a.q_ss, A.g);
  if (!A.q_tma) qm = km;  // not used
  auto kern = tree_attn_kernel<T, D>;
  auto merge = tree_attn_merge_kernel<T, D>;
  static DeviceOnce done;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done.done(dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "cannot set tree attention shared memory size %d", L::BYTES);
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
  cfg.blockDim = dim3(TA_NT);
  cfg.dynamicSmemBytes = L::BYTES;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, km, vm, qm, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "tree attention launch: %s", cudaGetErrorString(e));
  rc = check_launch("tree_attention");
  if (rc || a.cap <= TA_TK) return rc;  // a cache of one tile: nothing is split
  cfg.gridDim = dim3(a.B * a.Hkv * A.RT, (A.rows_pad / 32) * (D / 32));
  cfg.blockDim = dim3(TM_NT);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, merge, A, plan.ctas);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "tree attention merge launch: %s", cudaGetErrorString(e));
  return check_launch("tree_attention_merge");
}

}  // namespace

size_t tree_attention_workspace_size(int B, int Hq, int Hkv, int T, int D, int cap) {
  (void)B, (void)cap;
  return ta_plan(Hq, Hkv, T, D).bytes;
}

int launch_tree_attention(const TreeAttn& a, int dtype, void* ws, cudaStream_t st) {
  if (a.cap == 0) {  // no rows at all: nothing is seen
    if (cudaMemsetAsync(a.out, 0, (size_t)a.B * a.Hq * a.T * a.D * 2, st) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "tree attention: memset failed");
    return DROPKV_OK;
  }
  if (dtype == DROPKV_DTYPE_BF16)
    return a.D == 128 ? ta_launch<__nv_bfloat16, 128>(a, dtype, ws, st) : ta_launch<__nv_bfloat16, 64>(a, dtype, ws, st);
  return a.D == 128 ? ta_launch<__half, 128>(a, dtype, ws, st) : ta_launch<__half, 64>(a, dtype, ws, st);
}

}  // namespace dropkv
