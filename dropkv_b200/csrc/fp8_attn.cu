// Attention over a paged cache held in 8 bits for many query rows (g T > 8, of heads of 64 g T > 16): drafted trees, prompt chunks; and the
// kernel that joins partials. For token i of sequence b and query head h, O = sum_j softmax_j(scale q . k8_j sk_j)
// v8_j sv_j over the rows j that it sees, with the scales sk and sv of the rows' pages.
//
// A CTA has 128 query rows (whole tokens of a KV head's group) and two CTAs share an SM, so that one's softmax runs
// beside the other's products; keys come in tiles of 64. Both products are tcgen05 MMAs:
//   S = Q K^T  kind::f8f6f4, K's bytes as TMA brings them; queries as sums of 8-bit parts (two of a bf16,
//              three of an fp16), each part a product into the same accumulator: as many operations as in 16 bits
//              (half as many again for fp16), and no tile of K is ever widened;
//   O += P V   kind::f16: weights in fp16 left in tensor memory where S was, V widened to fp16 (exactly) by two
//              warps from one ring of tiles into another. (V as it lies would need weights in 8-bit parts: two roundings
//              and conversions a weight, for a tile's 128 rows, instead of one a byte of V.)
// S has two buffers, and the product of a tile is issued before the weights of the one before it are
// awaited. Warps: four of softmax, a thread for each row; two that widen V; one for TMA (a box a page); one that
// issues products.
// A page's scale of K enters with the exponent's argument, that of V, over the row's largest weight times scale so far, with
// the weights (both for eight keys at a time: pages have eight rows at least). Weights are rounded to fp16 (2^-11),
// sums taken from them before that.
// Measured (in a graph, three launches): 4096 tokens x 32 heads over 13107 rows x 8 heads x 128 before them, bf16, 968 us: 1050
// TFLOP/s, 64% of a large bf16 product's rate (fp16: 1100 us; 16 heads of 64 over 2: 460, a third of it); 64 nodes over 13107 rows 39 us;
// 8 nodes over 819 rows 16. A
// tile takes 1900 cycles with two CTAs an SM: 1400 from its logits to its weights, the rest until the products are issued and
// seen; products alone would take 640 a CTA (at 64 columns the reading of Q from shared memory bounds S's).
#include <algorithm>
#include <type_traits>

#include "fp8_attn.cuh"
#include "tc_common.cuh"

namespace dropkv {
namespace {

using namespace fa;

constexpr int FA_ROWS = 128;  // query rows of a CTA
constexpr int FA_TK = 64;     // keys of a tile
constexpr int FA_HALVES = FA_TK / 8;
constexpr int FA_WARP_V = 4, FA_WARP_TMA = 6, FA_WARP_MMA = 7, FA_NT = 256;
constexpr int FA_CTAS = 2;    // of an SM
constexpr int kFaLead = 6;  // (64 nodes over 13107 rows: 41.6 us at 2, 39.4 at 6, 38.9 at 9, where larger ones lose what that gains)
constexpr uint64_t kFaWaitNs = 1000000000ull;
// A row's reference moves once its maximum has grown by this much (base 2); weights times scales are
// 2^(s + log2 sv - R + bias), so that fp16 holds them from 2^-24 to 2^15.
constexpr float kFaSlack = 8.f, kFaBias = 7.f;
// Where a tile's weights are formed first: a row's sum of them above this moves its reference to the row's maximum
// (64 weights of 2^7 then sum to 2^13 at most).
constexpr float kFaMost = 32768.f;

// A tile whose keys all tokens see, with no page missing and none of zeros in V; and one whose pages have one scale of K and one of V, besides
constexpr int FA_WHOLE = 1, FA_PLAIN = 2;
struct FaKind {
  int kind;
  float vmax;  // the largest scale of V
};

template <int D, int PARTS>
struct FaSmem {
  static constexpr int NS = PARTS == 2 ? 3 : 2;         // slots of K's ring, and of V's
  static constexpr int TILE = FA_TK * D;                // a tile of K or V
  static constexpr int Q = 0;                           // PARTS x [128 rows][D]
  static constexpr int V16 = Q + PARTS * FA_ROWS * D;   // 2 x D / 64 slabs of [64 keys][128 bytes]
  static constexpr int K = V16 + 2 * 2 * TILE;
  static constexpr int V = K + NS * TILE;
  // Tiles whose scales are held: the load of K of tile i waits for the product of tile i - NS, which waits for the weights
  // of tile i - NS - 2, and V's before it for tile i - 1 - NS to be widened; so all are past the tile NS + 2 back.
  static constexpr int SCALES = NS + 2;
  static constexpr int SC = V + NS * TILE;              // float [SCALES][2][8]: -1 and 0 for a missing page
  static constexpr int KIND = SC + SCALES * 2 * FA_HALVES * 4;  // {int, float} [SCALES]: FA_WHOLE, FA_PLAIN; the largest of V's
  static constexpr int WALKS = KIND + SCALES * 8;  // WarpWalk [4], of the softmax warps
  static constexpr int BARS = (WALKS + 4 * (int)sizeof(WarpWalk<FA_TK>) + 7) / 8 * 8;
  static constexpr int B_KF = 0, B_KE = NS, B_VF = 2 * NS, B_VE = 3 * NS, B_S = 4 * NS, B_P = B_S + 2,
                       B_W = B_P + 2, B_O = B_W + 2, B_Q = B_O + 2, B_END = B_Q + 1, BARRIERS = B_END + 1;
  static constexpr int START = BARS + BARRIERS * 8;
  static constexpr int MISC = START + (int)sizeof(Start);  // tensor memory's address, `dead`, bad[2][2]
  static constexpr int BYTES = MISC + 24;
  static_assert(FA_CTAS * (BYTES + 1024) <= 233472, "shared memory");
};

__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The queries of all row tiles in 8-bit parts, laid out as the products read them, and their units. Grid: (row tiles of a
// sequence, SPLIT blocks for each; KV heads; sequences); D / 8 lanes have a row, eight elements each. A row's unit is the power of two that
// brings its largest element to at most 448; the first part is an element's nearest e4m3, each next the nearest e5m2 of what those
// before it left: the parts add up in one accumulator, so they share the unit, and e4m3's grid ends at 2^-9 of it, where a second part
// in e4m3 could leave 2^-10; e5m2's ends at 2^-16. What e4m3 leaves of a bf16 over 2^-6 has three bits, and so has what the second
// leaves of an fp16: those are held exactly. Of smaller elements two parts leave at most 2^-14, three 2^-17.
// In a kernel of its own because a row tile's rows are a long chain for its four softmax warps (3.5 us of a piece's 7 before
// its first product) and a short one for a whole GPU; bound by the chain load, largest element, parts.
constexpr int FQ_NT = 256;

template <typename T, int D, int SPLIT>
__global__ void __launch_bounds__(FQ_NT) fp8_queries_kernel(const __grid_constant__ Args A) {
  constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 2 : 3;
  constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  constexpr int LANES = D / 8, PER = FQ_NT / LANES, TURNS = FA_ROWS / PER / SPLIT;
  const AttnFp8& a = A.a;
  const int rt = blockIdx.x / SPLIT, h = blockIdx.y, b = blockIdx.z;
  const int row0 = blockIdx.x % SPLIT * (TURNS * PER) + threadIdx.x / LANES;
  const int c = threadIdx.x % LANES, n0 = rt * A.npr, rows = (min(n0 + A.npr, a.T) - n0) * A.g;
  const int64_t tile = row_tile(A, b, h, rt);
  uint8_t* out = A.queries + tile * (PARTS * FA_ROWS * D);
  pdl_wait();
  pdl_launch_dependents();
  uint4 x[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int row = row0 + i * PER, token = A.quot(row), head = h * A.g + row - token * A.g;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows) {
      const T* src = static_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh + (n0 + token) * a.q_ss + 8 * c * a.q_sd;
      if (A.q_vec) {
        x[i] = *reinterpret_cast<const uint4*>(src);
      } else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
        x[i].x = s[0] | (uint32_t)s[a.q_sd] << 16;
        x[i].y = s[2 * a.q_sd] | (uint32_t)s[3 * a.q_sd] << 16;
        x[i].z = s[4 * a.q_sd] | (uint32_t)s[5 * a.q_sd] << 16;
        x[i].w = s[6 * a.q_sd] | (uint32_t)s[7 * a.q_sd] << 16;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int row = row0 + i * PER;
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    // the largest magnitude, as bits: two 16-bit values a word
    uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = max(top & 0xffffu, top >> 16);
    const bool odd = top >= kInf;
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T* y = reinterpret_cast<const T*>(&w[e]);
      v[2 * e] = to_f(y[0]);
      v[2 * e + 1] = to_f(y[1]);
    }
    float big = to_f(*reinterpret_cast<const T*>(&top));
    if (__any_sync(0xffffffffu, odd)) {  // a row with what is no number: the largest of the others counts
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, isfinite(v[e]) ? fabsf(v[e]) : 0.f);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (odd) big = most;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = isfinite(v[e]) ? v[e] : __uint_as_float(0x7fffffffu);
    }
    const float one = query_unit(big), inv = __uint_as_float((254u << 23) - __float_as_uint(one));
    if (c == 0) A.units[tile * FA_ROWS + row] = one * A.scale_log2;
    __half2 z[4];  // (parts in fp16, whose 11 bits hold what is left at every step)
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = __floats2half2_rn(v[2 * e] * inv, v[2 * e + 1] * inv);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      uint32_t q8[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_fp8_interpretation_t kind = part ? __NV_E5M2 : __NV_E4M3;
        const uint32_t two = __nv_cvt_halfraw2_to_fp8x2(__half2_raw(z[e]), __NV_SATFINITE, kind);
        q8[e / 2] |= two << (16 * (e & 1));
        if (part + 1 < PARTS) z[e] = __hsub2(z[e], __half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)two, kind)));
      }
      *reinterpret_cast<uint2*>(out + part * (FA_ROWS * D) + tc::swz_offset<D>(row, (c / 2) * 8) + (c & 1) * 8) = make_uint2(q8[0], q8[1]);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(FA_NT, FA_CTAS)
    fp8_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ Args A) {
  constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 2 : 3;
  using L = FaSmem<D, PARTS>;
  constexpr int NS = L::NS, SLABS = D / 64, TK = FA_TK;
  extern __shared__ __align__(1024) uint8_t sm[];  // swizzled tiles start on multiples of 1024
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BARS);
  float* sc = reinterpret_cast<float*>(sm + L::SC);
  FaKind* kinds = reinterpret_cast<FaKind*>(sm + L::KIND);
  Start* start = reinterpret_cast<Start*>(sm + L::START);
  uint32_t* misc = reinterpret_cast<uint32_t*>(sm + L::MISC);
  volatile int* dead = reinterpret_cast<volatile int*>(misc + 1);
  volatile int* bad = reinterpret_cast<volatile int*>(misc + 2);  // [2][2]: a widening warp met NaN in a masked tile
  const AttnFp8& a = A.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tc::smem_addr(sm) % 1024) {  // as declared; nothing may run on any other layout
    pdl_wait();
    pdl_launch_dependents();
    if (tid == 0) {
      A.status[blockIdx.x] = 9;
      A.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      tc::mbar_init(&bars[L::B_KF + i], 1);
      tc::mbar_init(&bars[L::B_KE + i], 1);
      tc::mbar_init(&bars[L::B_VF + i], 1);
      tc::mbar_init(&bars[L::B_VE + i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bars[L::B_S + i], 2);  // the products' end, and the thread that issued them
      tc::mbar_init(&bars[L::B_P + i], 4);
      tc::mbar_init(&bars[L::B_W + i], 2);
      tc::mbar_init(&bars[L::B_O + i], 1);
    }
    tc::mbar_init(&bars[L::B_Q], 1);
    tc::mbar_init(&bars[L::B_END], 1);
    tc::fence_mbar_init();
    *dead = 0;
  }
  if (warp == FA_WARP_MMA) {
    tc::tmem_alloc(misc, 256);
    tc::tmem_relinquish();
  }
  if (warp == FA_WARP_TMA && lane == 0) {
    tc::tma_prefetch_desc(&kmap);
    tc::tma_prefetch_desc(&vmap);
  }
  // Of the kernel before this one only the queries' parts and units are needed, and only who reads them waits for it:
  // it let this one begin once all before it was over.
  if (warp == 0) find_start<TK>(A, lane, start);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *misc;  // S (and P) 2 x 64 columns, O 128
  // a wait that gives up marks the CTA dead: every role then ends without waiting
  auto wait = [&](uint64_t* bar, uint32_t count, int why) {  // for the count-th completion (from 0)
#pragma unroll 1
    for (int i = 0; i < 64; ++i)  // (the timer takes longer to read than most waits last)
      if (tc::mbar_try_wait(bar, count & 1)) return true;
    const uint64_t t0 = tc::globaltimer_ns();
    while (!*dead) {
      if (tc::mbar_try_wait(bar, count & 1)) return true;
      if (tc::globaltimer_ns() - t0 > kFaWaitNs) *dead = why;
    }
    return false;
  };
  // Tile j of the CTA (from 0, over all pieces): K and V in slot j % NS, scales in place j % SCALES (written before
  // K's load is announced), S, P and widened V
  // in buffer j % 2. What waits for what: K's load for the product that had the slot; S(j) for K and for O(j - 2), which has
  // read P in its buffer; P(j) for S(j); widened V(j) for V's load and O(j - 2); O(j) for P(j) and widened V(j).
  // A wait that is not taken for every tile (O's, where a reference moves; widened V's, in masked tiles) begins
  // with the phase before over, which S(j) says, and ends before the next, which needs P(j).
  // The softmax warps hold a tile's logits and need more registers than the others: (168 + 88) x 128 threads are what the
  // block was launched with, 256 x 128.
  if (warp >= FA_WARP_V) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == FA_WARP_TMA) {
    // ======================= TMA producer =======================================
    const int block = a.pool.block, lb = __ffs(block) - 1, box = min(block, TK), boxes = TK / box;
    Walk<TK> walk;
    Piece<TK> p;
    walk.start(*start);
    uint32_t n = 0, slot = 0, turn = 0, place = 0, queries = 0;
    bool ok = true;
    pdl_wait();
    while (ok && walk.next(A, p)) {
      // the piece's queries, once the products that read the last piece's are done: those with its last tile of K
      if (n) ok = __all_sync(0xffffffffu, wait(&bars[L::B_KE + (n - 1) % NS], (n - 1) / NS, 8));
      if (!ok) break;
      if (lane == 0) {
        constexpr uint32_t BYTES = PARTS * FA_ROWS * D;
        tc::mbar_arrive_expect_tx(&bars[L::B_Q], BYTES);
        tc::bulk_load(sm + L::Q, A.queries + row_tile(A, p.b, p.h, p.rt) * BYTES, BYTES, &bars[L::B_Q]);
      }
      __syncwarp();
      ++queries;
      const int32_t* table = a.table + (int64_t)p.b * a.max_blocks;
      const float* ksb = a.pool.k_scale + p.h * a.pool.ks_sh;
      const float* vsb = a.pool.v_scale + p.h * a.pool.vs_sh;
      // a lane has eight keys of a tile: their page, -1 where no token sees any of them
      auto page_of = [&](int t) {
        if (t >= p.t1 || lane >= FA_HALVES) return -1;
        const int j = p.k.first(t) + 8 * lane;
        return p.k.any(A, j, 8) ? table[j >> lb] : -1;
      };
      auto there = [&](int page) { return page >= 0 && page < a.pool.n_pages; };
      int all_end, all_low;
      p.k.all(A, &all_end, &all_low);
      int page = page_of(p.t0), page1 = page_of(p.t0 + 1);
      float ks = there(page) ? ksb[page * a.pool.ks_s0] : -1.f, vs = there(page) ? vsb[page * a.pool.vs_s0] : 0.f;
      for (int t = p.t0; t < p.t1; ++t, ++n) {
        const int page2 = page_of(t + 2);
        const float ks1 = there(page1) ? ksb[page1 * a.pool.ks_s0] : -1.f;
        const float vs1 = there(page1) ? vsb[page1 * a.pool.vs_s0] : 0.f;
        // the page of a lane's box: that of any of its eights that is read, else out of range (zeros)
        int at = there(page) ? page : -1;
        for (int o = 1; o < box / 8; o <<= 1) at = max(at, __shfl_xor_sync(0xffffffffu, at, o));
        at = __shfl_sync(0xffffffffu, at, min(lane, boxes - 1) * (box / 8));
        if (at < 0) at = a.pool.n_pages;
        const int row = p.k.first(t) & (block - 1);  // (of a page larger than a tile; else 0)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* full = &bars[(kv ? L::B_VF : L::B_KF) + slot];
          if (turn) ok = __all_sync(0xffffffffu, wait(&bars[(kv ? L::B_VE : L::B_KE) + slot], turn - 1, 1 + kv));
          if (!ok) break;
          if (lane == 0) tc::mbar_expect_tx(full, L::TILE);
          __syncwarp();
          if (lane < boxes)
            tc::tma_load_4d(sm + (kv ? L::V : L::K) + slot * L::TILE + lane * box * D, kv ? &vmap : &kmap, full, 0, row, p.h, at);
          if (kv == 0) {  // (the scales are on their way as the tile is)
            const float ks0 = __shfl_sync(0xffffffffu, ks, 0), vs0 = __shfl_sync(0xffffffffu, vs, 0);
            const int j0 = p.k.first(t);
            const bool there = __all_sync(0xffffffffu, lane >= FA_HALVES || (ks >= 0.f && vs > 0.f));
            const bool one = __all_sync(0xffffffffu, lane >= FA_HALVES || (ks == ks0 && vs == vs0));
            const bool whole = there && j0 + TK <= all_end && (j0 >= all_low || j0 + TK <= a.sinks);
            const int kind = whole ? (one ? FA_WHOLE | FA_PLAIN : FA_WHOLE) : 0;
            float vmax = vs;
#pragma unroll
            for (int o = FA_HALVES / 2; o > 0; o >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
            if (lane < FA_HALVES) {
              float* s = sc + place * (2 * FA_HALVES) + lane;
              s[0] = ks;
              s[FA_HALVES] = vs;
              if (lane == 0) kinds[place] = FaKind{kind, vmax};
            }
          }
          __syncwarp();  // (who sees K's or V's tile land sees the scales)
          if (lane == 0) tc::mbar_arrive(full);
        }
        if (!ok) break;
        if (++slot == NS) slot = 0, ++turn;
        if (++place == L::SCALES) place = 0;
        page = page1, page1 = page2, ks = ks1, vs = vs1;
      }
    }
    if (*dead) {  // every issued copy lands before the CTA may exit (of the tile that gave up, K may be one)
      if (queries) tc::mbar_wait(&bars[L::B_Q], (queries - 1) & 1, kFaWaitNs / 8);
      for (uint32_t j = n > (uint32_t)NS ? n - NS : 0u; j <= n; ++j)
        for (int kv = 0; kv < 2; ++kv)
          if (j < n || kv == 0) tc::mbar_wait(&bars[(kv ? L::B_VF : L::B_KF) + j % NS], (j / NS) & 1, kFaWaitNs / 8);
    }
  } else if (warp == FA_WARP_MMA) {
    // ======================= MMA issuer =========================================
    // The whole warp runs this and one lane issues, so that counts, addresses and descriptors can stay uniform.
    constexpr uint32_t ID_QK[2] = {tc::idesc_f8(FA_ROWS, TK, false), tc::idesc_f8(FA_ROWS, TK, true)};
    constexpr uint32_t ID_PV = tc::idesc_f16(false, FA_ROWS, D, false, true);
    constexpr uint32_t LAYOUT = tc::layout_for_row_bytes(D);
    constexpr uint32_t LBO_V = SLABS == 2 ? TK * 128 : 0;
    const uint32_t base = __shfl_sync(0xffffffffu, tc::smem_addr(sm), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
    Walk<TK> walk;
    Piece<TK> p;
    walk.start(*start);
    uint32_t j = 0, slot = 0, turn = 0, pieces = 0;
    bool ok = true;
    // O of tile i: the first of a piece begins it
    auto product = [&](uint32_t i, bool first) {
      const uint32_t buf = i & 1;
      ok = __all_sync(0xffffffffu, wait(&bars[L::B_W + buf], i >> 1, 4) && wait(&bars[L::B_P + buf], i >> 1, 3));
      if (!ok) return;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        const uint64_t vd = tc::smem_desc(base + L::V16 + buf * (2 * L::TILE), LBO_V, 1024);
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          tc::mma_f16_tmem_a(tm + 128, tm + buf * 64 + kk * 8, tc::desc_add(vd, kk * 2048), ID_PV, !first || kk > 0);
        tc::mma_commit(&bars[L::B_O + buf]);
      }
      __syncwarp();
    };
    while (ok && walk.next(A, p)) {
      const int nt = __shfl_sync(0xffffffffu, p.t1 - p.t0, 0);
      ok = __all_sync(0xffffffffu, wait(&bars[L::B_Q], pieces++, 5));
      for (int i = 0; i < nt && ok; ++i, ++j) {
        const uint32_t buf = j & 1;
        ok = __all_sync(0xffffffffu, wait(&bars[L::B_KF + slot], turn, 6) && (j < 2 || wait(&bars[L::B_O + buf], (j - 2) >> 1, 7)));
        if (!ok) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
          const uint64_t kd = tc::smem_desc(base + L::K + slot * L::TILE, 16, 8 * D, LAYOUT);
          const uint64_t qd = tc::smem_desc(base + L::Q, 16, 8 * D, LAYOUT);
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
              tc::mma_f8(tm + buf * 64, tc::desc_add(qd, part * (FA_ROWS * D) + kk * 32), tc::desc_add(kd, kk * 32), ID_QK[part > 0],
                         part > 0 || kk > 0);
          tc::mma_commit(&bars[L::B_S + buf]);
          tc::mma_commit(&bars[L::B_KE + slot]);
          tc::mbar_arrive(&bars[L::B_S + buf]);  // (hands on the scales, which came with K)
        }
        __syncwarp();
        if (++slot == NS) slot = 0, ++turn;
        if (i > 0) product(j - 1, i == 1);
      }
      if (ok) product(j - 1, nt == 1);
    }
    if (*dead) {  // no product may run on when tensor memory is given back
      if (tc::elect_one()) tc::mma_commit(&bars[L::B_END]);
      __syncwarp();
      tc::mbar_wait(&bars[L::B_END], 0, kFaWaitNs);
    }
  } else {
    // ======================= V to fp16 ==========================================
    // A thread has a key's row: 16-byte reads and writes of eight rows at a time meet all banks once.
    const int r = tid - FA_WARP_V * 32;
    Walk<TK> walk;
    Piece<TK> p;
    walk.start(*start);
    uint32_t j = 0, slot = 0, turn = 0, place = 0;
    bool ok = true;
    while (ok && walk.next(A, p)) {
      for (int t = p.t0; t < p.t1; ++t, ++j) {
        const uint32_t buf = j & 1;
        ok = __all_sync(0xffffffffu, wait(&bars[L::B_VF + slot], turn, 9) && (j < 2 || wait(&bars[L::B_O + buf], (j - 2) >> 1, 10)));
        if (!ok) break;
        const float* vs = sc + place * (2 * FA_HALVES) + FA_HALVES;
        const bool whole = kinds[place].kind & FA_WHOLE;
        const uint8_t* src = sm + L::V + slot * L::TILE;
        uint8_t* dst = sm + L::V16 + buf * (2 * L::TILE);
        auto widen = [&](auto clean) {
          const bool there = vs[r >> 3] > 0.f && p.k.first(t) + r < p.k.keys;
          uint32_t nan = 0;
#pragma unroll(decltype(clean)::value ? 1 : D / 16)
          for (int c = 0; c < D / 16; ++c) {
            uint4 x = *reinterpret_cast<const uint4*>(src + tc::swz_offset<D>(r, c * 8));
            if (decltype(clean)::value) {
              uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t odd = __vcmpeq4(w[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                if (!there)
                  w[e] = 0;
                else
                  nan |= odd, w[e] &= ~odd;
              }
              x = make_uint4(w[0], w[1], w[2], w[3]);
            }
            uint4 lo, hi;
            widen4(x.x, lo.x, lo.y);
            widen4(x.y, lo.z, lo.w);
            widen4(x.z, hi.x, hi.y);
            widen4(x.w, hi.z, hi.w);
            uint8_t* slab = dst + (c / 4) * (TK * 128);
            *reinterpret_cast<uint4*>(slab + tc::sw128_offset(r, (c % 4) * 16)) = lo;
            *reinterpret_cast<uint4*>(slab + tc::sw128_offset(r, (c % 4) * 16 + 8)) = hi;
          }
          return nan;
        };
        if (whole) {
          widen(std::false_type());
        } else {
          // what a weight of 0 would not silence: rows past the keys are cleared, and NaN is taken out here and given to those
          // who see it at the end
          const int some = __any_sync(0xffffffffu, widen(std::true_type()) != 0);
          if (lane == 0) bad[2 * buf + warp - FA_WARP_V] = some;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&bars[L::B_W + buf]);
          tc::mbar_arrive(&bars[L::B_VE + slot]);
        }
        if (++slot == NS) slot = 0, ++turn;
        if (++place == L::SCALES) place = 0;
      }
    }
  }
  } else {
    // ======================= softmax ============================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lanes = (uint32_t)(warp * 32) << 16, to = tmem + lanes + 128;
    const int r = tid;
    WarpWalk<TK>& ww = reinterpret_cast<WarpWalk<TK>*>(sm + L::WALKS)[warp];
    if (lane == 0) ww.walk.start(*start);
    const Piece<TK>& p = ww.piece;
    uint32_t j = 0, place = 0;
    bool ok = true;
    float unit = 0.f;  // of the row's queries, for logits in base 2
    Sees sees;
    auto begin = [&]() {  // a piece
      if (r < p.rows)
        sees.set(A, p.b, p.k.len, p.k.keys, p.k.n0 + A.quot(r));
      else
        sees.none();
      unit = A.units[row_tile(A, p.b, p.h, p.rt) * FA_ROWS + r];
    };
    int4 split = make_int4(0, 0, 0, 0);  // the split segment that begins in this CTA (its last piece)
    bool more = ww.next(A, lane);
    if (more) begin();
    while (more) {
      const bool live = warp * 32 < p.rows;  // some row of this warp exists
      // m measures the sums; R, also in base 2, the weights that meet V, times their pages' scales, of what the row sees alone.
      // (With one for all rows of a warp, pages of large scales took the bits of rows that do not see them, or give them no weight.)
      float m = -INFINITY, l = 0.f, R = -INFINITY, vinv = 0.f;  // vinv: 2^(m - R); the output is O / vinv
      int any_bad = 0;
      const int t1 = p.t1;
      for (int t = p.t0; t < t1 && ok; ++t, ++j) {
        const uint32_t buf = j & 1, ts = tmem + lanes + buf * 64;
        const bool first = t == p.t0;
        const float* scales = sc + place * (2 * FA_HALVES);
        const FaKind* kind_at = kinds + place;
        if (++place == L::SCALES) place = 0;
        uint64_t sum[2];
        // The references move where some row's largest logit, or that and its scale, has outgrown them.
        auto settle = [&](float top, float wtop, float slack) {
          if (!__any_sync(0xffffffffu, top > m + slack || wtop > R + slack)) return;
          const float mn = top > m + slack ? top : m, Rn = wtop > R + slack ? wtop : R;
          l *= mn == m ? 1.f : ex2(m - mn);
          const float alpha = Rn == R ? 1.f : ex2(R - Rn);
          m = mn, R = Rn;
          vinv = share_of(m, R);
          if (first || !__any_sync(0xffffffffu, alpha != 1.f)) return;
          ok = __all_sync(0xffffffffu, wait(&bars[L::B_O + 1 - buf], (j - 1) >> 1, 13)) && ok;
          tc::tc_fence_after();
          float o[16];
#pragma unroll 1
          for (int e0 = 0; e0 < D; e0 += 16) {
            tc::tmem_ld16(to + e0, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= alpha;
            tc::tmem_st16(to + e0, o);
            tc::tmem_st_wait();
          }
        };
        // (all lanes together from the vote to the stores: those are the whole warp's)
        // weights of 64 logits of one scale: into place, and into the sum before they are rounded
        float share = 1.f;  // of a tile with one scale of V: over the reference
        auto weigh = [&](const float* x, auto plain) {
          // of one scale of V: its share enters with the exponent, and leaves the sum again
          const float ref = (m == -INFINITY ? 0.f : m) - kFaBias - (decltype(plain)::value ? __log2f(share) : 0.f);
          const uint64_t ref2 = pair_of(-ref, -ref);
          uint64_t c2 = 0, f2 = 0;
          if (decltype(plain)::value) {
            const float c = fminf(scales[0] * unit, 3e38f);
            c2 = pair_of(c, c);
          }
          sum[0] = sum[1] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              if (!decltype(plain)::value && e % 8 == 0) {
                const float c = fminf(scales[4 * h + e / 8] * unit, 3e38f), f = fminf(scales[FA_HALVES + 4 * h + e / 8] * vinv, 3e38f);
                c2 = pair_of(c, c);
                f2 = pair_of(f, f);
              }
              float u, v;
              unpair(fma2(pair_of(x[32 * h + e], x[32 * h + e + 1]), c2, ref2), u, v);
              uint64_t w = pair_of(ex2(u), ex2(v));
              sum[(e / 2) & 1] = add2(sum[(e / 2) & 1], w);
              if (!decltype(plain)::value) w = mul2(w, f2);
              unpair(w, u, v);
              pk[e / 2] = pack_half(u, v);
            }
            tc::tmem_st16(ts + 16 * h, reinterpret_cast<const float*>(pk));
          }
        };
        auto largest = [&](const float* x, float& wtop) {
          float top = wtop = -INFINITY;
#pragma unroll
          for (int y = 0; y < FA_HALVES; ++y) {
            const float* z = x + 8 * y;
            const float u = max3(max3(z[0], z[1], z[2]), max3(z[3], z[4], z[5]), fmaxf(z[6], z[7])) * fminf(scales[y] * unit, 3e38f);
            top = fmaxf(top, u);
            wtop = fmaxf(wtop, u + __log2f(scales[FA_HALVES + y]));
          }
          return top;
        };
        ok = __all_sync(0xffffffffu, wait(&bars[L::B_S + buf], j >> 1, 12));
        if (!ok) break;
        if (live) {
          tc::tc_fence_after();
          const int kind = kind_at->kind;
          const float vmax = kind_at->vmax;
          auto total = [&]() {
            float s0, s1, s2, s3;
            unpair(sum[0], s0, s1);
            unpair(sum[1], s2, s3);
            return (s0 + s1) + (s2 + s3);
          };
          if (kind & FA_WHOLE) {  // what most tiles are
            // Weights against the standing references, without a look at the maximum: a sum within fp16's range says that
            // all of them are. (The maximum first: 64 logits' worth of instructions and of latency more a tile.)
            float x[TK];
            tc::tmem_ld64(ts, x);
            bool settled = first;
#pragma unroll 1
            for (;;) {
              if (settled) {
                float wtop;
                const float top = largest(x, wtop);
                settle(top, wtop, 0.f);
              }
              share = m == -INFINITY ? 1.f : vmax * vinv;  // (a row with nothing but NaN has no say)
              float most;  // of the weights times scales, their sum or more
              if (kind & FA_PLAIN && __all_sync(0xffffffffu, share >= 0x1p-40f && share <= 0x1p40f)) {
                weigh(x, std::true_type());
                most = total();
              } else {
                const float up = fmaxf(share, 1.f);
                share = 1.f;
                weigh(x, std::false_type());
                most = total() * up;
              }
              if (settled || !__any_sync(0xffffffffu, most > kFaMost || m == -INFINITY)) break;
              tc::tmem_st_wait();
              settled = true;
            }
          } else {
            // eight keys at a time, S read twice (rolled, as this is what few tiles are)
            const uint64_t see = sees.template bits<TK>(A, p.b, p.k.len, p.k.first(t));
            __syncwarp();
            float top = -INFINITY, wtop = -INFINITY;
            auto eight = [&](int y, float* z) {  // logits
              tc::tmem_ld8(ts + 8 * y, z);
              const float s = scales[y], c = fminf(s * unit, 3e38f);
              const uint32_t bits = s >= 0.f ? (uint32_t)(see >> (8 * y)) : 0u;
#pragma unroll
              for (int e = 0; e < 8; ++e) z[e] = (bits >> e) & 1 ? z[e] * c : -INFINITY;
            };
#pragma unroll 1
            for (int y = 0; y < FA_HALVES; ++y) {
              float z[8];
              eight(y, z);
              const float u = max3(max3(z[0], z[1], z[2]), max3(z[3], z[4], z[5]), fmaxf(z[6], z[7]));
              top = fmaxf(top, u);
              wtop = fmaxf(wtop, u + __log2f(scales[FA_HALVES + y]));
            }
            settle(top, wtop, kFaSlack);
            const float ref = (m == -INFINITY ? 0.f : m) - kFaBias;
            sum[0] = sum[1] = 0;
#pragma unroll 1
            for (int y = 0; y < FA_HALVES; ++y) {
              float z[8];
              eight(y, z);
              const float f = fminf(scales[FA_HALVES + y] * vinv, 3e38f);
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const float u = ex2(z[e] - ref), v = ex2(z[e + 1] - ref);
                sum[(e / 2) & 1] = add2(sum[(e / 2) & 1], pair_of(u, v));
                pk[e / 2] = pack_half(u * f, v * f);
              }
              tc::tmem_st4(ts + 4 * y, pk);  // (S of these columns has been read)
            }
            ok = __all_sync(0xffffffffu, wait(&bars[L::B_W + buf], j >> 1, 14)) && ok;
            any_bad |= bad[2 * buf] | bad[2 * buf + 1];
          }
          l += __fdividef(total(), share);
        }
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bars[L::B_P + buf]);
      }
      // ---- the piece's output; the next one begun first ----------------------
      if (p.parts) split = make_int4(p.b, p.h, p.rt, p.parts);
      const int b = p.b, h = p.h, n0 = p.k.n0, t0 = p.t0;
      const bool whole = t0 == 0 && t1 == p.tiles, own = r < p.rows && ok;
      const int64_t slot = slot_of(p);
      const Sees saw = sees;
      const Keys<TK> keys = p.k;
      more = ww.next(A, lane);
      if (more) begin();
      if (!ok) continue;
      const uint32_t last = j - 1;
      ok = __all_sync(0xffffffffu, wait(&bars[L::B_O + (last & 1)], last >> 1, 15));
      if (!ok) continue;
      tc::tc_fence_after();
      if (live) {
        // (l counts weights, of which a row that sees anything has one of 2^-1 at least)
        const float inv = l == 0.f ? 0.f : 1.f / vinv / l;
        uint32_t nan[D / 32];  // columns whose value is NaN for a row of V that this row sees
#pragma unroll
        for (int w = 0; w < D / 32; ++w) nan[w] = 0;
        if (any_bad && own) {
          const uint8_t* vb = static_cast<const uint8_t*>(a.pool.v) + h * a.pool.v_sh;
          for (int t = t0; t < t1; ++t) {
            const int j0 = keys.first(t);
            uint64_t todo = saw.template bits<TK>(A, b, keys.len, j0);
            while (todo) {
              const int key = j0 + __ffsll((long long)todo) - 1;
              todo &= todo - 1;
              const int page = a.table[(int64_t)b * a.max_blocks + key / a.pool.block];
              if (page < 0 || page >= a.pool.n_pages) continue;
              const uint8_t* v = vb + page * a.pool.v_s0 + (key % a.pool.block) * a.pool.v_st;
#pragma unroll
              for (int w = 0; w < D / 32; ++w)
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const uint32_t y = *reinterpret_cast<const uint32_t*>(v + 32 * w + e);
                  const uint32_t odd = __vcmpeq4(y & 0x7f7f7f7fu, 0x7f7f7f7fu) & 0x01010101u;
                  nan[w] |= ((odd * 0x10204080u) >> 28) << e;
                }
            }
          }
        }
        T* dst = static_cast<T*>(a.out) + out_row(A, b, h, n0, own ? r : 0) * D;
        float4* part = reinterpret_cast<float4*>(A.part_o + slot * A.rows_pad * D) + r;  // (32 rows of a vector, side by side)
#pragma unroll 1
        for (int w = 0; w < D / 32; ++w) {
          float o[32];
          __syncwarp();  // (rows part ways below; the load is the whole warp's)
          tc::tmem_ld32(to + 32 * w, o);
          if (any_bad && nan[w]) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if ((nan[w] >> e) & 1) o[e] = __uint_as_float(0x7fffffffu);
          }
          if (!own) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(dst + 32 * w + e) =
                  make_uint4(Out<T>::pack(o[e], o[e + 1]), Out<T>::pack(o[e + 2], o[e + 3]), Out<T>::pack(o[e + 4], o[e + 5]),
                             Out<T>::pack(o[e + 6], o[e + 7]));
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              part[(8 * w + e / 4) * A.rows_pad] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (own && !whole) {
          A.part_ml[slot * 2 * A.rows_pad + r] = m - kFaBias;
          A.part_ml[(slot * 2 + 1) * A.rows_pad + r] = l;
        }
        tc::tc_fence_before();  // (O is read before the next piece's first weights say so)
      }
    }
    if (tid == 0) A.meta[blockIdx.x] = split;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == FA_WARP_MMA) tc::tmem_dealloc(tmem, 256);
  if (tid == 0) A.status[blockIdx.x] = *dead;
}

constexpr int FM_NT = 256;
constexpr int FM_AHEAD = 8;  // partials on their way at once

// Joins the partials of the segments that fell into several CTAs. Grid: (split segments at most, or, `direct`, where FEW rows
// make few blocks or segments are many, the CTAs that they may begin in; groups of eight rows). With M the largest of the partials' maxima
// and w_i = l_i 2^(m_i - M), O = sum w_i o_i / sum w_i, in the order of the CTAs: a warp takes a row's weights, then a
// thread four columns of a row, as they lie: of FEW rows a row's vectors side by side, else eight rows' of a vector (who
// wrote them had a row a thread). Bound by the latency of its loads, from L2.
template <typename T, int D, bool FEW>
__global__ void __launch_bounds__(FM_NT) fp8_merge_kernel(const __grid_constant__ Args A, int ctas, bool direct) {
  constexpr int ROWS = FM_NT / 32;
  __shared__ int counts[ROWS], found;
  __shared__ float weights[ROWS][33], before_[ROWS];  // of 32 partials; what those before them are scaled by
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (!direct && threadIdx.x == 0) found = -1;
  // every CTA waits for the kernel before this one, with work or without: what comes after on the
  // stream takes this kernel's end for the end of both
  pdl_wait();
  int pick = blockIdx.x;
  if (!direct) {  // the CTA in which the blockIdx.x-th split segment begins
    for (int c0 = 0, before = 0; c0 < ctas; c0 += FM_NT) {
      const int at = c0 + threadIdx.x;
      const bool splits = at < ctas && A.meta[at].w > 0;
      const unsigned some = __ballot_sync(0xffffffffu, splits);
      if (lane == 0) counts[warp] = __popc(some);
      __syncthreads();
      for (int w = 0; w < ROWS; ++w) {
        if (w == warp && splits && before + __popc(some & ((1u << lane) - 1)) == (int)blockIdx.x) found = at;
        before += counts[w];
      }
      __syncthreads();
    }
    pick = found;
    if (pick < 0) return;
  }
  const int4 seg = A.meta[pick];
  if (seg.w == 0) return;
  const int n = seg.w, n0 = seg.z * A.npr, rows = (min(n0 + A.npr, A.a.T) - n0) * A.g, row0 = blockIdx.y * ROWS;
  if (row0 + (FEW ? warp : 0) >= rows) return;
  auto slot = [&](int i) { return 2 * ((int64_t)pick + i) + (i == 0 ? 1 : 0); };
  const float* ml = A.part_ml + row0 + warp;
  const int r = FEW ? warp : threadIdx.x % ROWS, c = FEW ? lane % (D / 4) : min((int)threadIdx.x / ROWS, D / 4 - 1);
  const float4* po = reinterpret_cast<const float4*>(A.part_o) + (FEW ? (row0 + r) * (D / 4) + c : c * A.rows_pad + row0 + r);
  auto sync = [&]() {
    if (FEW)
      __syncwarp();
    else
      __syncthreads();
  };
  float sum = 0.f, top = -INFINITY;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int cnt = min(32, n - i0);
    float4 x[FM_AHEAD];
    auto load = [&](int i, float4* to) {
#pragma unroll
      for (int u = 0; u < FM_AHEAD; ++u) to[u] = __ldcg(po + slot(i0 + min(i + u, cnt - 1)) * A.rows_pad * (D / 4));
    };
    load(0, x);  // (beside the maxima and sums)
    float m = -INFINITY, w = 0.f;
    if (lane < cnt && row0 + warp < rows) {
      const float* pm = ml + slot(i0 + lane) * 2 * A.rows_pad;
      m = __ldcg(pm);
      w = __ldcg(pm + A.rows_pad);
    }
    float mx = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(mx, top);
    if (lane == 0) before_[warp] = top == mx ? 1.f : ex2(top - mx);
    top = mx;
    weights[warp][lane] = w * (m == top ? 1.f : ex2(m - top));
    sync();
    const float f0 = before_[r];
    sum *= f0;
    y.x *= f0, y.y *= f0, y.z *= f0, y.w *= f0;
    for (int i = 0; i < cnt; i += FM_AHEAD) {
      if (i) load(i, x);
#pragma unroll
      for (int u = 0; u < FM_AHEAD; ++u) {
        if (i + u >= cnt) continue;
        const float f = weights[r][i + u];
        sum += f;
        y.x = fmaf(x[u].x, f, y.x), y.y = fmaf(x[u].y, f, y.y), y.z = fmaf(x[u].z, f, y.z), y.w = fmaf(x[u].w, f, y.w);
      }
    }
    sync();
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (row0 + r < rows && (FEW ? lane < D / 4 : threadIdx.x < ROWS * (D / 4)))
    *reinterpret_cast<uint2*>(static_cast<T*>(A.a.out) + out_row(A, seg.x, seg.y, n0, row0 + r) * D + 4 * c) =
        make_uint2(Out<T>::pack(y.x * inv, y.y * inv), Out<T>::pack(y.z * inv, y.w * inv));
}

template <typename T, int D>
int fm_launch(const Args& A, int ctas, cudaStream_t st) {
  const int64_t segments = (int64_t)A.a.B * A.RT * A.a.Hkv;
  const bool few = !A.queries, direct = few || segments >= ctas;  // (a block for each CTA: no list to look through)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(direct ? ctas : segments), (A.rows_pad + FM_NT / 32 - 1) / (FM_NT / 32));
  cfg.blockDim = dim3(FM_NT);
  cudaError_t e = cudaLaunchKernelEx(&cfg, few ? fp8_merge_kernel<T, D, true> : fp8_merge_kernel<T, D, false>, A, ctas, direct);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 merge launch: %s", cudaGetErrorString(e));
  return check_launch("attention_fp8_merge");
}

// What the queries' parts take, after the plan's regions (for fp16, which has more of them; a row's unit in four bytes).
struct FaQueries {
  int64_t tiles;
  size_t off_units, off_parts, bytes;
};
FaQueries fa_queries(const Plan& p, int64_t B, int64_t Hkv, int g, int T, int D) {
  FaQueries q;
  const int npr = FA_ROWS / g;
  q.tiles = B * Hkv * ((T + npr - 1) / npr);
  q.off_units = p.bytes;
  q.off_parts = align_up(q.off_units + (size_t)q.tiles * FA_ROWS * 4, 256);
  q.bytes = q.off_parts + (size_t)q.tiles * 3 * FA_ROWS * D;
  return q;
}

Plan fa_plan(int64_t rows, int D) {
  return make_plan(FA_CTAS * num_sms_current_device(), (int)std::min<int64_t>(FA_ROWS, (rows + 7) / 8 * 8), D);
}

template <typename T, int D>
int fa_launch(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  using L = FaSmem<D, std::is_same<T, __nv_bfloat16>::value ? 2 : 3>;
  const int g = a.Hq / a.Hkv;
  const Plan plan = fa_plan((int64_t)g * a.T, D);
  const FaQueries qs = fa_queries(plan, a.B, a.Hkv, g, a.T, D);
  Args A = make_args(a, plan, FA_ROWS / g, kFaLead, ws);
  A.units = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + qs.off_units);
  A.queries = static_cast<uint8_t*>(ws) + qs.off_parts;
  if (a.B > 65535) return fail(DROPKV_ERR_UNSUPPORTED, "attention_fp8: %d sequences are too many", a.B);
  CUtensorMap km, vm;
  int rc = make_fp8_tensor_maps(&km, &vm, a.pool, std::min(a.pool.block, FA_TK));
  if (rc) return rc;
  auto kern = fp8_attn_kernel<T, D>;
  static DeviceOnce done;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done.done(dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "cannot set attention_fp8 shared memory size %d", L::BYTES);
    // the split of registers between the warps counts on this many at launch: with fewer it would wait forever
    cudaFuncAttributes attrs;
    if (cudaFuncGetAttributes(&attrs, kern) != cudaSuccess || attrs.numRegs * FA_NT < (168 + 88) * 128)
      return fail(DROPKV_ERR_CUDA, "attention_fp8 was compiled for too few registers");
    done.mark(dev);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  constexpr int SPLIT = 4;  // of a tile's rows, while all blocks still run at once
  const bool few = qs.tiles <= num_sms_current_device();
  cfg.gridDim = dim3(few ? A.RT * SPLIT : A.RT, a.Hkv, a.B);
  cfg.blockDim = dim3(FQ_NT);
  cudaError_t e = cudaLaunchKernelEx(&cfg, few ? fp8_queries_kernel<T, D, SPLIT> : fp8_queries_kernel<T, D, 1>, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 queries launch: %s", cudaGetErrorString(e));
  if ((rc = check_launch("attention_fp8_queries"))) return rc;
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(FA_NT);
  cfg.dynamicSmemBytes = L::BYTES;
  e = cudaLaunchKernelEx(&cfg, kern, km, vm, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 launch: %s", cudaGetErrorString(e));
  rc = check_launch("attention_fp8");
  if (rc || a.cap <= FA_TK) return rc;  // a cache of one tile: nothing is split
  return launch_fp8_merge(A, dtype, plan.ctas, st);
}

}  // namespace

int launch_fp8_merge(const fa::Args& A, int dtype, int ctas, cudaStream_t st) {
  if (dtype == DROPKV_DTYPE_BF16)
    return A.a.D == 128 ? fm_launch<__nv_bfloat16, 128>(A, ctas, st) : fm_launch<__nv_bfloat16, 64>(A, ctas, st);
  return A.a.D == 128 ? fm_launch<__half, 128>(A, ctas, st) : fm_launch<__half, 64>(A, ctas, st);
}

size_t attention_fp8_workspace_size(int B, int Hq, int Hkv, int T, int D, int cap) {
  (void)cap;
  const int64_t rows = (int64_t)Hq / Hkv * T;
  return fp8_few_rows(rows, D) ? fp8_decode_plan((int)rows, D).bytes : fa_queries(fa_plan(rows, D), B, Hkv, Hq / Hkv, T, D).bytes;
}

int launch_attention_fp8(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  if (a.cap == 0) {  // no rows at all: nothing is seen
    if (cudaMemsetAsync(a.out, 0, (size_t)a.B * a.Hq * a.T * a.D * 2, st) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "attention_fp8: memset failed");
    return DROPKV_OK;
  }
  if (fp8_few_rows((int64_t)a.Hq / a.Hkv * a.T, a.D)) return launch_fp8_decode(a, dtype, ws, st);
  if (dtype == DROPKV_DTYPE_BF16)
    return a.D == 128 ? fa_launch<__nv_bfloat16, 128>(a, dtype, ws, st) : fa_launch<__nv_bfloat16, 64>(a, dtype, ws, st);
  return a.D == 128 ? fa_launch<__half, 128>(a, dtype, ws, st) : fa_launch<__half, 64>(a, dtype, ws, st);
}

}  // namespace dropkv
