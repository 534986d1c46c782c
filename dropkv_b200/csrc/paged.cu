// Pages of a shared K/V pool for a ragged batch of caches: block tables and slot
// maps from lengths that exist on the device only (an eviction's keep_len, a decode
// loop's counters), and the rows that go to those slots.
#include <algorithm>

#include "common.cuh"

namespace dropkv {
namespace {

constexpr int BT_NT = 256;
constexpr int BT_EACH = 8;                  // slots of a thread
constexpr int BT_TOKENS = BT_EACH * BT_NT;  // slots of a CTA

struct BtArgs {
  const int32_t* lens;
  const int32_t* new_lens;  // nullptr: every token is new
  const int32_t* table_in;  // nullptr: no pages held
  int64_t table_in_stride;
  const int32_t* held_in;
  const int32_t* free_blocks;
  int B, block, n_free, max_blocks, max_new;
  uint32_t by_mul, by_shift;  // division by block
  int32_t* table;
  int32_t* held;
  int64_t* slots;
  int64_t* used;
};

// t / block for t below 2^31, by a multiplication (Granlund and Montgomery): with l = ceil(log2
// block), mul = floor(2^(31 + l) / block) + 1 exceeds 2^(31 + l) / block by at most one part in
// 2^31, which no such t turns into a quotient too large.
__device__ __forceinline__ unsigned bt_quot(const BtArgs& a, unsigned t) {
  return a.block == 1 ? t : __umulhi(t, a.by_mul) >> a.by_shift;
}
__device__ __forceinline__ int bt_len(const BtArgs& a, int b) { return max(a.lens[b], 0); }
__device__ __forceinline__ int bt_held(const BtArgs& a, int b) {
  return a.held_in ? min(max(a.held_in[b], 0), a.max_blocks) : 0;
}
// pages request b still needs
__device__ __forceinline__ int bt_take(const BtArgs& a, int b) {
  const int len = bt_len(a, b), need = len ? (int)bt_quot(a, (unsigned)(len - 1)) + 1 : 0;
  return max(min(need, a.max_blocks) - bt_held(a, b), 0);
}

// CTA (b, y): table row b (y = 0) and the slots [y, y + 1) * BT_TOKENS of request b.
// A request's pages start where those of the requests before it end in the free
// list, so each CTA sums the needs of the requests before its own; no CTA waits
// for another. With need_b = ceil(len_b / block) and take_b = max(need_b - held_b, 0),
// request b gets entries [f, f + take_b) of the free list, f = sum of take over the
// requests before it, and token t of it the slot table[b][t / block] * block + t % block.
// What bounds it: a step's call is its launch and two chains of loads (32 requests: 2.8 us);
// a prefill's is the 8 bytes a token that it writes (128 requests of up to 13107 tokens,
// 13 MB: 5.6 us, 2.4 TB/s, behind the sums and a page's lookup for each token; with a division
// and one lookup after the other 7.2). Slots of a thread 2, 4, 8, 16: 8.4, 6.4, 5.6, 6.0 us.
// The sums are taken again by every CTA because a list of a few hundred lengths is one load a
// thread, less than a second launch or a wait for a first CTA.
__global__ void __launch_bounds__(BT_NT) block_tables_kernel(BtArgs a) {
  __shared__ long long part[BT_NT / 32];
  const int b = blockIdx.x, tid = threadIdx.x;
  long long sum = 0;
  for (int i = tid; i < b; i += BT_NT) sum += bt_take(a, i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((tid & 31) == 0) part[tid >> 5] = sum;
  __syncthreads();
  long long first = 0;
#pragma unroll
  for (int w = 0; w < BT_NT / 32; ++w) first += part[w];
  const int held = bt_held(a, b), take = bt_take(a, b);
  const long long left = a.n_free - first;
  const int got = (int)(left < 0 ? 0 : (left < take ? left : take));
  const int32_t* old = a.table_in ? a.table_in + b * a.table_in_stride : nullptr;
  auto page = [&](int col) -> int {
    if (col < held) return old[col];
    return col < held + got ? a.free_blocks[first + (col - held)] : -1;
  };
  if (blockIdx.y == 0) {
    int32_t* row = a.table + (int64_t)b * a.max_blocks;
    for (int c = tid; c < a.max_blocks; c += BT_NT) row[c] = page(c);
    if (tid == 0) {
      a.held[b] = held + got;
      if (b == a.B - 1) *a.used = first + take;
    }
  }
  const int len = bt_len(a, b), nn = a.new_lens ? min(max(a.new_lens[b], 0), len) : len;
  const int64_t i0 = (int64_t)blockIdx.y * BT_TOKENS + tid;
  int64_t* out = a.slots + (int64_t)b * a.max_new;
  int p[BT_EACH];  // the slots' pages, all on their way before the first is used
  unsigned at[BT_EACH];
#pragma unroll
  for (int e = 0; e < BT_EACH; ++e) {
    const int64_t i = i0 + e * BT_NT;
    p[e] = -1;
    if (i >= nn) continue;
    const unsigned t = (unsigned)(len - nn) + (unsigned)i, col = bt_quot(a, t);
    at[e] = t - col * (unsigned)a.block;
    if (col < (unsigned)a.max_blocks) p[e] = page((int)col);
  }
#pragma unroll
  for (int e = 0; e < BT_EACH; ++e) {
    const int64_t i = i0 + e * BT_NT;
    if (i < a.max_new) out[i] = p[e] >= 0 ? (int64_t)p[e] * a.block + at[e] : -1;
  }
}

constexpr int SR_NT = 256;

struct SrArgs {
  const char* k;  // [B, H, N, row bytes], byte strides
  const char* v;
  int64_t k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  const int64_t* slots;  // [B, N]
  char* kp;              // [pages, H, block, row bytes], byte strides
  char* vp;
  int64_t kp_sb, kp_sh, kp_st, vp_sb, vp_sh, vp_st;
  int64_t n_slots;       // pages * block
  int B, H, N, block, vecs;  // vecs: vectors of a row
};

// Rows of LANES 16-byte vectors: LANES threads have a row, SR_ROWS rows each, whose slots,
// then K and V vectors, are on their way at once. Rows follow one another along a head, so
// reads are one stream and writes come in runs of a page's rows. HBM bounds it: each byte is
// read and written once. One layer's 13107 rows (8 heads of 128, bf16, 107 MB): 18.8 us alone
// (5.7 TB/s, 87% of a copy's rate), 19.3 us in a graph over inputs larger than L2; rows in flight 1,
// 2, 4, 8: 18.7, 18.8, 19.4, 20.4 us alone, and a few hundred rows 1.8, 2.2, 3.0, 4.2 us; 2 for the
// heads of 64, where 1 row is slower (16.8 us against 15.7 over one set of rows, in part in L2).
constexpr int SR_ROWS = 2;

template <int LANES>
__global__ void __launch_bounds__(SR_NT) store_rows_vec_kernel(SrArgs a) {
  constexpr int RPB = SR_NT / LANES;
  const unsigned rows = (unsigned)a.B * a.H * a.N;
  const unsigned r0 = blockIdx.x * (RPB * SR_ROWS) + threadIdx.x / LANES;
  const int c = threadIdx.x % LANES * 16;
  int64_t slot[SR_ROWS];
  int b[SR_ROWS], h[SR_ROWS], n[SR_ROWS];
#pragma unroll
  for (int i = 0; i < SR_ROWS; ++i) {
    const unsigned r = r0 + i * RPB, bh = r / (unsigned)a.N;
    n[i] = (int)(r - bh * a.N);
    b[i] = (int)(bh / (unsigned)a.H);
    h[i] = (int)(bh - (unsigned)b[i] * a.H);
    slot[i] = r < rows ? a.slots[(int64_t)b[i] * a.N + n[i]] : -1;
  }
  uint4 k[SR_ROWS], v[SR_ROWS];
#pragma unroll
  for (int i = 0; i < SR_ROWS; ++i) {
    if (slot[i] >= a.n_slots) slot[i] = -1;
    if (slot[i] >= 0) {
      k[i] = __ldcs(reinterpret_cast<const uint4*>(a.k + b[i] * a.k_sb + h[i] * a.k_sh + n[i] * a.k_sn + c));
      v[i] = __ldcs(reinterpret_cast<const uint4*>(a.v + b[i] * a.v_sb + h[i] * a.v_sh + n[i] * a.v_sn + c));
    }
  }
#pragma unroll
  for (int i = 0; i < SR_ROWS; ++i) {
    if (slot[i] < 0) continue;
    const int64_t page = slot[i] >> 32 ? slot[i] / a.block : (int64_t)((uint32_t)slot[i] / (uint32_t)a.block);
    const int64_t at = slot[i] - page * a.block;
    *reinterpret_cast<uint4*>(a.kp + page * a.kp_sb + h[i] * a.kp_sh + at * a.kp_st + c) = k[i];
    *reinterpret_cast<uint4*>(a.vp + page * a.vp_sb + h[i] * a.vp_sh + at * a.vp_st + c) = v[i];
  }
}

// Rows of any size, alignment and number.
template <typename T>
__global__ void __launch_bounds__(SR_NT) store_rows_kernel(SrArgs a) {
  const int64_t total = (int64_t)a.B * a.H * a.N * a.vecs;
  for (int64_t e = (int64_t)blockIdx.x * SR_NT + threadIdx.x; e < total; e += (int64_t)gridDim.x * SR_NT) {
    const int c = (int)(e % a.vecs);
    int64_t r = e / a.vecs;
    const int n = (int)(r % a.N);
    r /= a.N;
    const int h = (int)(r % a.H), b = (int)(r / a.H);
    const int64_t slot = a.slots[(int64_t)b * a.N + n];
    if (slot < 0 || slot >= a.n_slots) continue;
    const int64_t page = slot / a.block, at = slot % a.block;
    *reinterpret_cast<T*>(a.kp + page * a.kp_sb + h * a.kp_sh + at * a.kp_st + c * (int)sizeof(T)) =
        *reinterpret_cast<const T*>(a.k + b * a.k_sb + h * a.k_sh + n * a.k_sn + c * (int)sizeof(T));
    *reinterpret_cast<T*>(a.vp + page * a.vp_sb + h * a.vp_sh + at * a.vp_st + c * (int)sizeof(T)) =
        *reinterpret_cast<const T*>(a.v + b * a.v_sb + h * a.v_sh + n * a.v_sn + c * (int)sizeof(T));
  }
}

}  // namespace

int launch_block_tables(const int32_t* lens, const int32_t* new_lens, const int32_t* table_in, int64_t table_in_stride,
                        const int32_t* held_in, int B, int block, const int32_t* free_blocks, int n_free,
                        int max_blocks, int max_new, int32_t* table, int32_t* held, int64_t* slots, int64_t* used,
                        cudaStream_t st) {
  int l = 0;
  while ((int64_t(1) << l) < block) ++l;
  const uint32_t by_mul = block == 1 ? 0u : (uint32_t)((uint64_t(1) << (31 + l)) / block + 1);
  BtArgs a{lens, new_lens, table_in, table_in_stride, held_in, free_blocks, B, block, n_free, max_blocks, max_new,
           by_mul, (uint32_t)std::max(l - 1, 0), table, held, slots, used};
  const int ys = (int)(((int64_t)max_new + BT_TOKENS - 1) / BT_TOKENS);
  if (ys > 65535) return fail(DROPKV_ERR_UNSUPPORTED, "block tables: max_new %d exceeds %d", max_new, 65535 * BT_TOKENS);
  block_tables_kernel<<<dim3(B, ys > 0 ? ys : 1), BT_NT, 0, st>>>(a);
  return check_launch("block_tables");
}

int launch_store_rows(const StoreRows& s, cudaStream_t st) {
  SrArgs a;
  const int eb = s.elem_bytes;
  a.k = static_cast<const char*>(s.k);
  a.v = static_cast<const char*>(s.v);
  a.kp = static_cast<char*>(s.k_pages);
  a.vp = static_cast<char*>(s.v_pages);
  a.k_sb = s.k_sb * eb, a.k_sh = s.k_sh * eb, a.k_sn = s.k_sn * eb;
  a.v_sb = s.v_sb * eb, a.v_sh = s.v_sh * eb, a.v_sn = s.v_sn * eb;
  a.kp_sb = s.kp_sb * eb, a.kp_sh = s.kp_sh * eb, a.kp_st = s.kp_st * eb;
  a.vp_sb = s.vp_sb * eb, a.vp_sh = s.vp_sh * eb, a.vp_st = s.vp_st * eb;
  a.slots = s.slots;
  a.n_slots = (int64_t)s.n_pages * s.block;
  a.B = s.B, a.H = s.H, a.N = s.N, a.block = s.block;
  // 16-byte vectors where every address they form is a multiple of 16
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                        reinterpret_cast<uintptr_t>(a.kp) | reinterpret_cast<uintptr_t>(a.vp) |
                        (uint64_t)(a.k_sb | a.k_sh | a.k_sn | a.v_sb | a.v_sh | a.v_sn | a.kp_sb | a.kp_sh | a.kp_st |
                                   a.vp_sb | a.vp_sh | a.vp_st) |
                        (uint64_t)s.D * eb;
  const int w = bits % 16 == 0 ? 16 : eb;
  a.vecs = s.D * eb / w;
  const int64_t total = (int64_t)s.B * s.H * s.N * a.vecs;
  const int64_t want = (total + SR_NT - 1) / SR_NT, most = 32 * (int64_t)num_sms_current_device();
  const int grid = (int)(want < most ? want : most);
  const int64_t rows = (int64_t)s.B * s.H * s.N;
  if (w == 16 && rows < 0x7fffffff - SR_NT * SR_ROWS && (a.vecs == 4 || a.vecs == 8 || a.vecs == 16 || a.vecs == 32)) {
    const int per = SR_NT / a.vecs * SR_ROWS, ctas = (int)((rows + per - 1) / per);
    if (a.vecs == 4)
      store_rows_vec_kernel<4><<<ctas, SR_NT, 0, st>>>(a);
    else if (a.vecs == 8)
      store_rows_vec_kernel<8><<<ctas, SR_NT, 0, st>>>(a);
    else if (a.vecs == 16)
      store_rows_vec_kernel<16><<<ctas, SR_NT, 0, st>>>(a);
    else
      store_rows_vec_kernel<32><<<ctas, SR_NT, 0, st>>>(a);
    return check_launch("store_rows");
  }
  if (w == 16)
    store_rows_kernel<uint4><<<grid, SR_NT, 0, st>>>(a);
  else if (w == 4)
    store_rows_kernel<uint32_t><<<grid, SR_NT, 0, st>>>(a);
  else
    store_rows_kernel<uint16_t><<<grid, SR_NT, 0, st>>>(a);
  return check_launch("store_rows");
}

}  // namespace dropkv
