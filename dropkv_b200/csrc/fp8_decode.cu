// Attention over a cache in 8 bits for few query rows (g T <= 8, of heads of 64 g T <= 16): single tokens, short drafts.
//
// A key costs 2 D bytes and 4 D M operations, so HBM bounds this by far, and what counts is to
// keep loads on their way and instructions few. One warp issues TMA loads (a box a page) of K and V
// tiles of 128 keys into a ring of slots; four warps take 32 keys of each tile. Both products are warp
// MMAs fed from registers (tcgen05.mma takes 128 rows, of which 1 to 16 would exist, and as many
// threads would do the softmax):
//   S = Q K^T      m16n8k32 of e4m3: K's bytes as they lie, and queries as sums of 8-bit parts, each
//                  what the one before left, times 16: two parts of a bf16 (the second takes the
//                  MMA's rows 8 to 15 where there are at most 8 queries), three of an fp16;
//   O^T += V^T P^T m16n8k16 of fp16: A = 16 columns of V for 16 keys, widened (exactly, two at a time),
//                  B = the weights of 8 rows as they lie in S's accumulators.
// The order of D and of the keys within a product is free, and chosen so that a quarter warp's 16-byte
// reads of the swizzled tiles meet all banks once (D = 128): lane (gid, tig) = (lane / 4, lane % 4) reads
// chunks 4 i + tig of key fd_key(gid)'s row of K, and for V chunk fd_chunk(gid) of keys
// fd_key(2 tig + {0, 1}) and of those 8 on, whose bytes are paired before they are widened.
// A row's queries are brought to 8 bits' range by a power of two (its largest element to 224 or more;
// what the parts leave is at most 2^-14 of that unit, 2^-18 in fp16). A page's scale of K multiplies its logits in fp32;
// that of V, over the row's largest weight times scale so far, the weights. Weights are rounded to fp16 for their
// product (2^-11), sums taken from them before that.
// Measured (in a graph, the merge with it): 32 sequences of up to 13107 rows x 8 heads x 128 in pages of 64 rows, bf16, 87
// us for 484 MB: 5.6 TB/s, 85% of a copy's rate (pages of 16: 92); 295K rows x 4 heads in pages of 16, fp16, 70 us for 303 MB:
// 66% (bf16 queries and pages of 64: 59). Some 10 us of each are start and end (walk, first tiles, partials, merge).
#include <algorithm>
#include <type_traits>

#include "fp8_attn.cuh"
#include "tc_common.cuh"

namespace dropkv {
namespace {

using namespace fa;

constexpr int FD_WARPS = 4, FD_NT = 32 * FD_WARPS + 32;  // warps that compute; and one that loads
constexpr int FD_TK = 32 * FD_WARPS;                      // keys of a tile
constexpr int FD_HALVES = FD_TK / 8;                      // a page has 8 rows at least
constexpr int FD_CTAS = 2;                                // of an SM
constexpr uint64_t kFdWaitNs = 1000000000ull;

template <int D, bool R16, int PARTS>
struct FdShape {
  static constexpr int ROWS = R16 ? 16 : 8;
  static constexpr int TILE = FD_TK * D, SLOTS = (R16 ? 4 : 5) * (128 / D);
  static constexpr int WO = SLOTS * TILE;                        // float [WARPS][ROWS][D]: the warps' outputs
  static constexpr int WM = WO + FD_WARPS * ROWS * D * 4;        // float [2][WARPS][ROWS]: maxima, sums
  // tiles whose scales are held: before tile i's first load is issued, the slot is free that load 2 i - SLOTS had,
  // so all warps are past the tiles before that
  static constexpr int SCALES = SLOTS / 2 + 1;
  static constexpr int SC = WM + 2 * FD_WARPS * ROWS * 4;        // float [SCALES][2][FD_HALVES]: -1 and 0 for a missing page
  static constexpr int BARS = SC + SCALES * 2 * FD_HALVES * 4;   // full[SLOTS], empty[SLOTS]
  // the queries' operands of S, the same for all warps, lie in shared memory where they are many
  static constexpr bool QS = R16 || PARTS == 3;
  static constexpr int ACCS = R16 ? PARTS : PARTS - 1;  // products of S: one for each part; 8 rows' first two share one
  static constexpr int QO = (BARS + 2 * SLOTS * 8 + 15) / 16 * 16;  // uint4 [ACCS][D / 32][32]
  static constexpr int WALKS = QO + (QS ? ACCS * (D / 32) * 512 : 0);
  // WarpWalk [WARPS + 1] there
  static constexpr int START = WALKS + (FD_WARPS + 1) * (int)sizeof(WarpWalk<FD_TK>);
  static constexpr int BYTES = START + (int)sizeof(Start) + 8;
  static_assert(FD_CTAS * (BYTES + 1024) <= 233472, "shared memory");
};

// 8-bit parts that hold an element of a query
template <typename T>
constexpr int fd_parts() { return std::is_same<T, __nv_bfloat16>::value ? 2 : 3; }

template <int D>
__device__ __forceinline__ int fd_key(int n) { return D == 128 ? ((n & 1) << 2) | (n >> 1) : n; }
template <int D>
__device__ __forceinline__ int fd_chunk(int gid) { return D == 128 ? ((gid & 1) << 2) | (gid >> 1) : gid; }

constexpr int kFdLead = 3;
// A row's reference moves once its maximum has grown by this much (base 2); weights times scales are
// 2^(s + log2 sv - R + bias), so that fp16 holds them from 2^-24 to 2^15.
constexpr float kFdSlack = 8.f, kFdBias = 7.f;

__device__ __forceinline__ void fd_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void fd_mma8(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void fd_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
static_assert(FD_WARPS == 4, "threads of fd_sync");

template <typename T, int D, bool R16>
__global__ void __launch_bounds__(FD_NT, FD_CTAS)
    fp8_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ Args A) {
  constexpr int PARTS = fd_parts<T>();
  using S = FdShape<D, R16, PARTS>;
  constexpr int TK = FD_TK, WARPS = FD_WARPS, ROWS = S::ROWS, HR = R16 ? 2 : 1, NS = S::SLOTS;
  constexpr int ACCS = S::ACCS;
  constexpr int KV = D / 64;   // 16-byte vectors of K a lane has of a key
  constexpr int VW = D / 32;   // words of V a lane has of a key
  constexpr int VB = 4 * VW;
  extern __shared__ __align__(1024) uint8_t sm[];  // swizzled tiles start on multiples of 1024
  float* wo = reinterpret_cast<float*>(sm + S::WO);
  float* wm = reinterpret_cast<float*>(sm + S::WM);
  float* wl = wm + WARPS * ROWS;
  float* sc = reinterpret_cast<float*>(sm + S::SC);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + S::BARS);
  uint64_t* empty = full + NS;
  Start* start = reinterpret_cast<Start*>(sm + S::START);
  volatile int* dead = reinterpret_cast<volatile int*>(start + 1);
  const AttnFp8& a = A.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
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
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], WARPS);
    }
    tc::fence_mbar_init();
    *dead = 0;
  }
  if (warp == WARPS && lane == 0) {
    tc::tma_prefetch_desc(&kmap);
    tc::tma_prefetch_desc(&vmap);
  }
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: the merge may then read this kernel's inputs at once)
  if (warp == 0) find_start<TK>(A, lane, start);
  __syncthreads();
  WarpWalk<TK>& ww = reinterpret_cast<WarpWalk<TK>*>(sm + S::WALKS)[warp];
  if (lane == 0) ww.walk.start(*start);
  const Piece<TK>& p = ww.piece;
  // a wait that gives up marks the CTA dead: every role then ends without waiting
  auto wait = [&](uint64_t* bar, uint32_t count, int why) {  // for the count-th completion (from 0)
    if (tc::mbar_try_wait(bar, count & 1)) return true;
    const uint64_t t0 = tc::globaltimer_ns();
    while (!*dead) {
      if (tc::mbar_try_wait(bar, count & 1)) return true;
      if (tc::globaltimer_ns() - t0 > kFdWaitNs) *dead = why;
    }
    return false;
  };
  // Tile i of the CTA (from 0, over all pieces) is loads 2 i (K) and 2 i + 1 (V); load n uses slot n % NS. Every
  // role waits for every load (or slot) of its own in turn, so a barrier is never two phases ahead of a wait.
  if (warp == WARPS) {
    // ======================= TMA producer =======================================
    const int block = a.pool.block, lb = __ffs(block) - 1, box = min(block, TK), boxes = TK / box;
    uint32_t n = 0;
    bool ok = true;
    while (ok && ww.next(A, lane)) {
      const int32_t* table = a.table + (int64_t)p.b * a.max_blocks;
      const float* ksb = a.pool.k_scale + p.h * a.pool.ks_sh;
      const float* vsb = a.pool.v_scale + p.h * a.pool.vs_sh;
      // a lane has eight keys of a tile: their page, -1 where no token sees any of them
      auto page_of = [&](int t) {
        if (t >= p.t1 || lane >= FD_HALVES) return -1;
        const int j = p.k.first(t) + 8 * lane;
        return p.k.any(A, j, 8) ? table[j >> lb] : -1;
      };
      auto there = [&](int page) { return page >= 0 && page < a.pool.n_pages; };
      int page = page_of(p.t0), page1 = page_of(p.t0 + 1);
      float ks = there(page) ? ksb[page * a.pool.ks_s0] : -1.f, vs = there(page) ? vsb[page * a.pool.vs_s0] : 0.f;
      for (int t = p.t0; t < p.t1; ++t) {
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
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t slot = n % NS;
          if (n >= (uint32_t)NS) ok = __all_sync(0xffffffffu, wait(&empty[slot], n / NS - 1, 1));
          if (!ok) break;
          if (lane == 0) tc::mbar_expect_tx(&full[slot], S::TILE);
          __syncwarp();
          if (lane < boxes)
            tc::tma_load_4d(sm + slot * S::TILE + lane * box * D, kv ? &vmap : &kmap, &full[slot], 0, row, p.h, at);
          if (kv == 0 && lane < FD_HALVES) {  // (on their way as the tile is; who sees K land sees them)
            float* s = sc + (n / 2 % S::SCALES) * (2 * FD_HALVES) + lane;
            s[0] = ks;
            s[FD_HALVES] = vs;
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&full[slot]);
        }
        if (!ok) break;
        page = page1, page1 = page2, ks = ks1, vs = vs1;
      }
    }
    if (*dead && n) {  // every issued copy lands before the CTA may exit
      for (uint32_t j = n > (uint32_t)NS ? n - NS : 0u; j < n; ++j) tc::mbar_wait(&full[j % NS], (j / NS) & 1, kFdWaitNs / 8);
    }
  } else {
  // ======================= the warps that compute =============================
  uint32_t slot = 0, turn = 0, held = 0;  // of the next load: its slot, how often that was filled; of the next tile: its scales
  bool ok = true;
  int4 split = make_int4(0, 0, 0, 0);  // the split segment that begins in this CTA (its last piece)
  // what a lane reads of a tile: K's vectors of its two keys, V's of its four
  uint32_t k_at[KV], v_at[2];
#pragma unroll
  for (int i = 0; i < KV; ++i) k_at[i] = tc::swz_offset<D>(32 * warp + fd_key<D>(gid), (4 * i + tig) * 8);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = 32 * warp + fd_key<D>(2 * tig + c);
    v_at[c] = VW == 4 ? tc::swz_offset<D>(r, fd_chunk<D>(gid) * 8) : tc::swz_offset<D>(r, (gid >> 1) * 8) + (gid & 1) * 8;
  }
  while (ww.next(A, lane)) {
    // ---- queries: rows gid and, of 16, gid + 8 ---------------------------------
    uint32_t q[PARTS][KV * 4][HR];  // four elements a word, as a lane has them of K
    float qscale[HR];
    Sees sees[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      const int r = gid + 8 * x;
      float v[KV * 16];
      float big = 0.f;
      if (r < p.rows) {
        const int token = A.quot(r), node = p.k.n0 + token, head = p.h * A.g + r - token * A.g;
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
#pragma unroll
      for (int e = 0; e < KV * 16; ++e) big = fmaxf(big, isfinite(v[e]) ? fabsf(v[e]) : 0.f);
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const float unit = query_unit(big), inv = 1.f / unit;
      qscale[x] = unit * A.scale_log2;
#pragma unroll
      for (int e = 0; e < KV * 16; ++e) v[e] = isfinite(v[e]) ? v[e] * inv : __uint_as_float(0x7fffffffu);
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int s = 0; s < KV * 4; ++s) q[part][s][x] = split4(v + 4 * s, 16.f);
    }
    // operand A of S for step e of D (two words of a vector) and product j
    auto operand = [&](int j, int e, uint32_t* qa) {
      if (R16) {
        qa[0] = q[j][e][0], qa[1] = q[j][e][HR - 1], qa[2] = q[j][e + 1][0], qa[3] = q[j][e + 1][HR - 1];
      } else if (j == 0) {  // rows 8 to 15 are the second part's
        qa[0] = q[0][e][0], qa[1] = q[1][e][0], qa[2] = q[0][e + 1][0], qa[3] = q[1][e + 1][0];
      } else {
        qa[0] = q[PARTS - 1][e][0], qa[1] = 0u, qa[2] = q[PARTS - 1][e + 1][0], qa[3] = 0u;
      }
    };
    uint4* qo = reinterpret_cast<uint4*>(sm + S::QO) + lane;
    if (S::QS) {  // (all warps are past the piece before: they met at its end)
#pragma unroll
      for (int e = 0; e < 4 * KV; e += 2)
#pragma unroll
        for (int j = 0; j < ACCS; ++j)
          if ((e / 2) % WARPS == warp) {
            uint32_t qa[4];
            operand(j, e, qa);
            qo[(j * 2 * KV + e / 2) * 32] = make_uint4(qa[0], qa[1], qa[2], qa[3]);
          }
      fd_sync();
    }
    // ---- the warp's steps --------------------------------------------------------
    float o[HR][VB / 2][4];
    float m[HR], l[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) {
      m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
      for (int t = 0; t < VB / 2; ++t) o[x][t][0] = o[x][t][1] = o[x][t][2] = o[x][t][3] = 0.f;
    }
    // what a row's weights times scales are measured by, in base 2, and 2^(m - R): the output is o / share
    float R[HR], share[HR];
#pragma unroll
    for (int x = 0; x < HR; ++x) R[x] = -INFINITY, share[x] = 1.f;
    int all_end, all_low;
    p.k.all(A, &all_end, &all_low);
    for (int t = p.t0; t < p.t1; ++t) {
      ok = ok && __all_sync(0xffffffffu, wait(&full[slot], turn, 2));
      if (!ok) break;
      const float4* scales = reinterpret_cast<const float4*>(sc + held * (2 * FD_HALVES)) + warp;
      if (++held == S::SCALES) held = 0;
      float ks[4], vs[4];
      *reinterpret_cast<float4*>(ks) = scales[0];
      *reinterpret_cast<float4*>(vs) = scales[FD_HALVES / 4];
      const int j0 = p.k.first(t) + 32 * warp;
      const bool some = fmaxf(fmaxf(ks[0], ks[1]), fmaxf(ks[2], ks[3])) >= 0.f;
      float s[4][2 * HR];  // of eight keys each: rows gid, then gid + 8
      if (some) {
        const uint8_t* kt = sm + slot * S::TILE;
        constexpr int XS = ACCS < 3 ? 4 : 2;  // eights of keys at once: four chains of products or more
#pragma unroll
        for (int x0 = 0; x0 < 4; x0 += XS) {
          float c[XS][ACCS][4];
          uint4 k[XS][KV];
#pragma unroll
          for (int x = 0; x < XS; ++x) {
#pragma unroll
            for (int i = 0; i < KV; ++i)
              k[x][i] = *reinterpret_cast<const uint4*>(kt + k_at[i] + (x0 + x) * 8 * D);  // (the swizzle repeats after 8 rows)
#pragma unroll
            for (int j = 0; j < ACCS; ++j) c[x][j][0] = c[x][j][1] = c[x][j][2] = c[x][j][3] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 4 * KV; e += 2)
#pragma unroll
            for (int j = 0; j < ACCS; ++j) {
              uint32_t qa[4];
              if (S::QS) {
                const uint4 y = qo[(j * 2 * KV + e / 2) * 32];
                qa[0] = y.x, qa[1] = y.y, qa[2] = y.z, qa[3] = y.w;
              } else {
                operand(j, e, qa);
              }
#pragma unroll
              for (int x = 0; x < XS; ++x) {
                const uint4 kx = k[x][e / 4];
                fd_mma8(c[x][j], qa, e % 4 ? kx.z : kx.x, e % 4 ? kx.w : kx.y);
              }
            }
#pragma unroll
          for (int x = 0; x < XS; ++x)
#pragma unroll
            for (int e = 0; e < 2 * HR; ++e) {
              float z = R16 ? c[x][ACCS > 1 ? 1 : 0][e] : c[x][0][(e + 2) & 3];
              if (PARTS == 3) z = fmaf(c[x][ACCS - 1][e], 0.0625f, z);
              s[x0 + x][e] = fmaf(z, 0.0625f, c[x][0][e]);
            }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[slot]);
      if (++slot == NS) slot = 0, ++turn;
      uint32_t b[4][HR];         // weights of the 16 keys of two eights, for the second product
      uint32_t seen = 0xffffffffu, mine[HR];
      bool masked = false;
      if (some) {
        const float least = fminf(fminf(ks[0], ks[1]), fminf(ks[2], ks[3]));
        masked = !(least >= 0.f) || j0 + 32 > all_end || (j0 < all_low && j0 + 32 > a.sinks);
#pragma unroll
        for (int x = 0; x < HR; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float c = fminf(qscale[x] * ks[y], 3e38f);
            s[y][2 * x] *= c, s[y][2 * x + 1] *= c;
          }
        if (masked) {
          seen = 0;
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            uint32_t see = (uint32_t)sees[x].template bits<32>(A, p.b, p.k.len, j0);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              if (!(ks[y] >= 0.f)) see &= ~(0xffu << (8 * y));
              if (!((see >> (8 * y + fd_key<D>(2 * tig))) & 1)) s[y][2 * x] = -INFINITY;
              if (!((see >> (8 * y + fd_key<D>(2 * tig + 1))) & 1)) s[y][2 * x + 1] = -INFINITY;
            }
            mine[x] = see;
            seen |= see;
          }
          seen = __reduce_or_sync(0xffffffffu, seen);
        }
        // The references move where some row's maximum has outgrown them: m, of the sums, by logits; R, of the weights that
        // meet V, by logits and scales, of what the row sees alone. (With one for all rows, pages of large scales took the bits
        // of rows that do not see them, or give them no weight.)
        const float lv = __log2f(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])));
        float top[HR];
        bool over = false;
#pragma unroll
        for (int x = 0; x < HR; ++x) {
          top[x] = fmaxf(fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1])),
                         fmaxf(fmaxf(s[2][2 * x], s[2][2 * x + 1]), fmaxf(s[3][2 * x], s[3][2 * x + 1])));
          over = over || top[x] > m[x] + kFdSlack || top[x] + lv > R[x] + kFdSlack;
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int x = 0; x < HR; ++x) {
            float wtop = -INFINITY;
#pragma unroll
            for (int y = 0; y < 4; ++y) wtop = fmaxf(wtop, fmaxf(s[y][2 * x], s[y][2 * x + 1]) + __log2f(vs[y]));
#pragma unroll
            for (int i = 1; i < 4; i *= 2) {
              top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], i));
              wtop = fmaxf(wtop, __shfl_xor_sync(0xffffffffu, wtop, i));
            }
            const float mn = top[x] > m[x] + kFdSlack ? top[x] : m[x], Rn = wtop > R[x] + kFdSlack ? wtop : R[x];
            l[x] *= mn == m[x] ? 1.f : ex2(m[x] - mn);
            const float f = Rn == R[x] ? 1.f : ex2(R[x] - Rn);
            m[x] = mn, R[x] = Rn;
            share[x] = share_of(mn, Rn);
            const float f0 = __shfl_sync(0xffffffffu, f, 8 * tig), f1 = __shfl_sync(0xffffffffu, f, 8 * tig + 4);
#pragma unroll
            for (int e = 0; e < VB / 2; ++e) o[x][e][0] *= f0, o[x][e][1] *= f1, o[x][e][2] *= f0, o[x][e][3] *= f1;
          }
        }
#pragma unroll
        for (int x = 0; x < HR; ++x) {
          const float ref = (m[x] == -INFINITY ? 0.f : m[x]) - kFdBias;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float p0 = ex2(s[y][2 * x] - ref), p1 = ex2(s[y][2 * x + 1] - ref), f = fminf(vs[y] * share[x], 3e38f);
            l[x] += p0 + p1;
            b[y][x] = pack_half(p0 * f, p1 * f);
          }
        }
      }
      ok = __all_sync(0xffffffffu, wait(&full[slot], turn, 3));
      if (!ok) break;
      if (some) {
        const uint8_t* vt = sm + slot * S::TILE;
#pragma unroll
        for (int y = 0; y < 4; y += 2) {  // 16 keys
          uint32_t v[4][VW];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint8_t* src = vt + v_at[c & 1] + (y + (c >> 1)) * 8 * D;
            if (VW == 4) {
              const uint4 z = *reinterpret_cast<const uint4*>(src);
              v[c][0] = z.x, v[c][1] = z.y, v[c][VW - 2] = z.z, v[c][VW - 1] = z.w;
            } else {
              const uint2 z = *reinterpret_cast<const uint2*>(src);
              v[c][0] = z.x, v[c][1] = z.y;
            }
          }
          if (masked) {
            // V of keys that no row sees is cleared; NaN of those that some see is taken out, and given to these
            uint32_t nan = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const bool see = (seen >> (8 * (y + (c >> 1)) + fd_key<D>(2 * tig + (c & 1)))) & 1;
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
                    at |= 1u << (8 * (y + (c >> 1)) + fd_key<D>(2 * tig + (c & 1)));
                    v[c][e >> 2] &= ~(0xffu << (8 * (e & 3)));
                  }
                at |= __shfl_xor_sync(0xffffffffu, at, 1);
                at |= __shfl_xor_sync(0xffffffffu, at, 2);
#pragma unroll
                for (int x = 0; x < HR; ++x)
#pragma unroll
                  for (int z = 0; z < 2; ++z) {  // rows 8 x + 2 tig + z
                    const uint32_t see = __shfl_sync(0xffffffffu, mine[x], 4 * (2 * tig + z));
                    if (see & at) o[x][e >> 1][2 * (e & 1) + z] = __uint_as_float(0x7fffffffu);
                  }
              }
            }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t va[4], vc[4];
            widen4(__byte_perm(v[0][w], v[1][w], 0x5140), va[0], va[1]);
            widen4(__byte_perm(v[2][w], v[3][w], 0x5140), va[2], va[3]);
            widen4(__byte_perm(v[0][w], v[1][w], 0x7362), vc[0], vc[1]);
            widen4(__byte_perm(v[2][w], v[3][w], 0x7362), vc[2], vc[3]);
#pragma unroll
            for (int x = 0; x < HR; ++x) {
              fd_mma(o[x][2 * w], va, b[y][x], b[y + 1][x]);
              fd_mma(o[x][2 * w + 1], vc, b[y][x], b[y + 1][x]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[slot]);
      if (++slot == NS) slot = 0, ++turn;
    }
    if (p.parts) split = make_int4(p.b, p.h, p.rt, p.parts);
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
      const float back = 1.f / share[x];
      const float b0 = __shfl_sync(0xffffffffu, back, 8 * tig), b1 = __shfl_sync(0xffffffffu, back, 8 * tig + 4);
      float* o0 = wo + (warp * ROWS + 8 * x + 2 * tig) * D + VB * fd_chunk<D>(gid);
#pragma unroll
      for (int e = 0; e < VB / 2; ++e) {
        *reinterpret_cast<float2*>(o0 + 2 * e) = make_float2(o[x][e][0] * b0, o[x][e][2] * b0);
        *reinterpret_cast<float2*>(o0 + D + 2 * e) = make_float2(o[x][e][1] * b1, o[x][e][3] * b1);
      }
    }
    fd_sync();
    const bool whole = p.t0 == 0 && p.t1 == p.tiles;
    for (int e = tid; ok && e < p.rows * (D / 4); e += 32 * WARPS) {
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
    fd_sync();
  }
  if (tid == 0) A.meta[blockIdx.x] = split;
  }
  __syncthreads();
  if (tid == 0) A.status[blockIdx.x] = *dead;
}

template <typename T, int D, bool R16>
int fd_launch(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  using S = FdShape<D, R16, fd_parts<T>()>;
  const Plan plan = fp8_decode_plan(a.Hq / a.Hkv * a.T, D);
  const Args A = make_args(a, plan, a.T, kFdLead, ws);
  CUtensorMap km, vm;
  int rc = make_fp8_tensor_maps(&km, &vm, a.pool, std::min(a.pool.block, FD_TK));
  if (rc) return rc;
  auto kern = fp8_decode_kernel<T, D, R16>;
  static DeviceOnce done;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done.done(dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES) != cudaSuccess)
      return fail(DROPKV_ERR_CUDA, "cannot set attention_fp8 shared memory size %d", S::BYTES);
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
  cfg.blockDim = dim3(FD_NT);
  cfg.dynamicSmemBytes = S::BYTES;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, km, vm, A);
  if (e != cudaSuccess) return fail(DROPKV_ERR_CUDA, "attention_fp8 launch: %s", cudaGetErrorString(e));
  rc = check_launch("attention_fp8");
  if (rc || a.cap <= FD_TK) return rc;  // a cache of one tile: nothing is split
  return launch_fp8_merge(A, dtype, plan.ctas, st);
}

template <typename T>
int fd_typed(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  if (a.Hq / a.Hkv * a.T > 8) return fd_launch<T, 64, true>(a, dtype, ws, st);  // (heads of 64: fp8_few_rows)
  return a.D == 128 ? fd_launch<T, 128, false>(a, dtype, ws, st) : fd_launch<T, 64, false>(a, dtype, ws, st);
}

}  // namespace

fa::Plan fp8_decode_plan(int rows, int D) {
  return make_plan(num_sms_current_device() * FD_CTAS, rows > 8 ? 16 : 8, D);
}

int launch_fp8_decode(const AttnFp8& a, int dtype, void* ws, cudaStream_t st) {
  return dtype == DROPKV_DTYPE_BF16 ? fd_typed<__nv_bfloat16>(a, dtype, ws, st) : fd_typed<__half>(a, dtype, ws, st);
}

}  // namespace dropkv
