// Attention over a paged cache with a window and sinks, or with a tree of drafted tokens behind the past, on tcgen05 /
// TMEM / TMA (monofab_masked_attention in monofab.h says what is computed).
//
// o_i = sum_j p_ij v_j / sum_j p_ij over the keys j that row i sees, p_ij = 2^(c s_ij - m_i), s = q k, c = scale log2(e), in one
// pass over the keys in tiles of 128. m_i is a reference that all of a row's weights share: the first maximum, moved only when a later
// one passes it by more than 2^8, and then the sums so far are scaled. Scores, sums and outputs are in 32 bits; a weight is rounded
// once, to the type of V, for the product: its matrix instruction wants both operands alike. Weights of fp16 are 2^7 times as large, so
// that they use the type's range upwards as well (below 2^16) and those far below the reference are not lost: steps of 2^-31 of it.
// All of a row's weights share the rounding of m_i, half a step of it: harmless while 2^8 times that is in the type (c s up to 2^24 in fp16).
//
//   * An item is (request, block of query tokens, KV head); a row of the matrix products is a (token, query head of the group) pair,
//     so a K or V tile is read once for all of them. A CTA has two streams of 128 rows, each with scores S (128 columns of TMEM), the
//     weights P in the place of the scores that they come from (64 columns, the A operand of P V) and an accumulator O (D
//     columns): 512 columns for D = 128. In an item of more rows than one stream takes (a pair) the streams have a block of rows each
//     and share the tiles; else they take alternate tiles of the same rows and are joined at the end.
//   * An item of at most 16 rows (a token and its group) in a batch of such (D = 128) is multiplied the other way round, keys and head
//     dims as the 128 rows and its rows as 16 columns (softmax_few).
//   * Warps: 0 loads K and V through a ring of 32 or 16 KB stages; 1 issues the products; 2 hands out items and loads queries; 4 - 7
//     and 8 - 11 are the streams' softmax, a thread a row. One warp issues both streams' products: it keeps them a step apart, so
//     that one's products run under the other's softmax. (A warp for each: their products run into each other, both streams wait at the
//     same time.)
//   * The work is shared out on the device, from lengths that are read there: tiles and items have a cost (below), every
//     CTA takes an equal part of its sum, and items that a border cuts leave 32-bit rows and (reference, sum) in a workspace,
//     which a second kernel joins in order: the same bits every time. A border near an item's begin is moved there.
//   * An item's tiles are cut from the pages that its rows see, one behind the other: those of the sinks, then those of the window. A
//     tile that all rows of a stream see goes without masks; else a row has the tile's keys as bits: the ranges of the window and the
//     sinks, or the past and the tree's bits, shifted. Pages that no row of the item sees are not loaded, and values that
//     none sees are zeroed in shared memory, so that nothing there can reach a sum.
//
// What bounds it (B200, clocks as they come): contexts of single tokens HBM, 5.7 TB/s of K and V (128 sequences, 843 MB: 147 us);
// prompts and large trees the chain of a stream's tile and the card's power: 3350 cycles, 1900 from S to P (maxima 280, weights 1400) and 1450
// from P to the next S (values 512, scores 512, hand-overs); window prompts 131 us, long trees 425 in short runs and 530 in long ones.
// The loop of tiles is short on purpose: a warp's instructions come from a small cache, and every one that the loop does not need shows
// (masks in the loops of maxima and weights instead of ahead of them: 141 us). Measured and dropped: a row of S in registers (234), two chunks of
// weights in line (134), the next columns' TMEM loads ahead of the weights (177 -> 201 at the time), sixteen warps of softmax (177 -> 206),
// half tiles with two score buffers a stream (177 -> 191; the scores cost half as much again), a warp for each stream's products (177 -> 187),
// weights handed over in two parts (128).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/monofab.h"
#include "kernels.h"
#include "moe_layer.h"
#include "ptx.cuh"

namespace mf {

int encode_map(CUtensorMap* map, int dtype, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
               int swizzle);   // api.cu

namespace {

constexpr int kTile = 128;          // keys of a tile, rows of a stream
constexpr int kThreads = 384;
constexpr int kRecords = 4;
// What work costs, in tiles of an item whose streams take alternate ones (2000 cycles): a tile of a pair, an item beyond its tiles, and the
// least share of a CTA.
constexpr int kPairCost = 2, kItemCost = 2, kMinCost = 2;
static_assert(kMinCost >= kPairCost, "every share that begins inside an item has a tile of it");
constexpr int kSlotRows = 2 * kTile;
constexpr int kMaxRequests = 16384;
constexpr int kFewRows = 16, kFewBytes = 2 * kFewRows * 128;   // kFewBytes: weights of such a stream, two times 64 keys of a row in 128 bytes
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kSlack = 8.f;       // powers of two by which a weight may pass that of its reference
constexpr int kByFma = 8;           // weights of 32 worked out by multiplications

// Where a call that names no status word leaves its bits.
__device__ int g_masked_attention_status;

struct Params {
  CUtensorMap q_map;      // dims (D, hq, tokens), box (64, group, tokens of a stream)
  CUtensorMap q_one_map;  // box (64, group, 1)
  CUtensorMap k_map;      // dims (64, 8, halves x hkv, page / 8, pages), box (64, 8, halves, page / 8, 1)
  CUtensorMap v_map;
  const int32_t *block_table, *q_start, *kv_len, *tree;
  void* out;
  int* status;
  float* ws_o;            // [2 x CTAs][256][D]
  float2* ws_ml;          // [2 x CTAs][256]
  int4* ws_meta;          // [CTAs][2]
  long long out_row, out_head;
  int tokens, requests, hkv, group, page, bt_stride, words, window, sinks;
  int per_stream;         // query tokens of a stream's 128 rows
  float scale_log2;
};

// A bounded wait by the whole warp, which goes on or gives up as one (ptx.cuh); what happens when the phase is not there yet is kept out of
// the callers' code.
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, int* abort_flag) {
  return mbar_wait_warp(bar, parity, abort_flag, kWaitNs);
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_longer(bar, parity, abort_flag);
}

// A request as the device sees it.
struct Request {
  int row0, rows, kv_len;
};
__device__ __forceinline__ Request request_of(const Params& p, int r) {
  Request q;
  q.row0 = max(0, min(p.q_start[r], p.tokens));
  q.rows = max(0, min(p.q_start[r + 1], p.tokens) - q.row0);
  q.kv_len = max(0, p.kv_len[r]);
  return q;
}
__device__ __forceinline__ int blocks_of(const Params& p, int rows) { return (rows + 2 * p.per_stream - 1) / (2 * p.per_stream); }

// The keys that the rows of a block see lie in [0, near) and [lo, hi). An item's tiles are 128 places in a row: first the pages of the
// former, `split` places, then those of the latter; place v is key v below `split` and key v + shift from there on. (Where the two meet
// in a page, and for trees, places are keys.) lo, hi and near are places.
// (Tiles at multiples of 128 keys, the sinks in one of their own: window prompts with 4 sinks 157 us where this took 141.)
struct Span {
  int tokens, pos0, lo, hi, near, split, shift;
  __device__ __forceinline__ int tiles() const { return (hi + kTile - 1) / kTile; }
  __device__ __forceinline__ int tile_cost(const Params& p) const { return tokens > p.per_stream ? kPairCost : 1; }
  __device__ __forceinline__ int cost(const Params& p) const { return tiles() * tile_cost(p) + kItemCost; }
};
__device__ __forceinline__ Span span_of(const Params& p, const Request& q, int block) {
  Span s;
  const int first = block * 2 * p.per_stream;
  s.tokens = min(2 * p.per_stream, q.rows - first);
  s.pos0 = q.kv_len - q.rows + first;
  const int there = min(q.kv_len, p.bt_stride * p.page);
  s.near = s.lo = s.split = s.shift = 0;
  s.hi = there;
  if (p.tree) return s;
  s.hi = max(0, min(there, s.pos0 + s.tokens));
  const int lo = static_cast<int>(max(0ll, static_cast<long long>(s.pos0) - p.window + 1));
  s.near = min(min(p.sinks, s.hi), lo);
  if (lo >= there) {   // no key of the window is there: places are keys, and none of them is past 2^30
    s.lo = s.hi = s.near;
    return s;
  }
  const int split = (s.near + p.page - 1) / p.page * p.page, from = lo / p.page * p.page;
  if (split < from) {
    s.split = split;
    s.shift = from - split;
  }
  s.lo = lo - s.shift;
  s.hi = max(s.near, s.hi - s.shift);
  return s;
}

// A CTA's share of the work begins at tile t of (request, block, head); r == requests: the end.
struct Place {
  int r, b, h, t;
};
__device__ __forceinline__ bool same_item(const Place& a, const Place& b) { return a.r == b.r && a.b == b.b && a.h == b.h; }

// One part of an item, as the roles get it.
struct Record {
  int req, head, row0, tokens, pos0, past, there;   // there: keys in the block table; past: first drafted key
  int lo, hi, near, split, shift;                   // of its Span
  int t0, t1;
  int slot;     // -1: the whole item, else the workspace slot
  int pair;     // two streams of rows; else the streams take alternate tiles. -1: no more items
  int few;      // not a pair, and few enough rows to be the columns of the scores (kFewRows)
};

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kGroupBytes = 1024 * kHalves;   // eight keys of a K or V tile
  static constexpr int kSmem = (2 + kStages) * kTileBytes;
};

struct Shared {
  uint64_t kv_full[10], kv_empty[10], rec_full[kRecords], rec_empty[kRecords];
  uint64_t q_full, q_empty, s_full[2], p_full[2], o_full[2], told[2], x_full, x_done, drain;
  uint32_t tmem_base;
  int abort_flag;
  Place place[2];
  Record rec[kRecords];
  union {
    float2 ml[2][kTile];   // (reference, sum) of the streams' rows
    struct {               // of an item of few rows: of each stream, warp and row, maxima of a tile and sums of the item; references
      float top[2][4][kFewRows], sum[2][4][kFewRows], m[2][kFewRows];
    } few;
  };
};

// Descriptors: Q rows of 128 bytes a half, halves 16 KB apart; K and V tiles in groups of eight keys, the halves of a group
// 1 KB apart (one TMA box of a page delivers both).
__device__ __forceinline__ uint64_t smem_desc(uint32_t low, uint32_t stride) {   // low: address / 16 | leading offset / 16 << 16
  return static_cast<uint64_t>((stride >> 4) | 1u << 14 | 2u << 29) << 32 | low;
}

// D[tmem] (+)= A[tmem] * B[smem]; issued by one thread.
__device__ __forceinline__ void umma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void load_box_3d(void* smem, const void* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               :
               : "r"(smem_u32(smem)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void load_box_5d(void* smem, const void* map, uint64_t* bar, int c2, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %4, %3, %5}], [%2];"
               :
               : "r"(smem_u32(smem)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(c2), "r"(c4)
               : "memory");
}
__device__ __forceinline__ void store_tmem_16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void load_tmem_4(uint32_t at, uint32_t (&v)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void store_tmem_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two 32-bit values as one operand of the packed instructions.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 parts_of(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <class E>
struct Half2;
template <>
struct Half2<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static constexpr float kLift = 0.f;   // weights are 2^kLift times p_ij, sums and outputs alike; bf16 has the exponents of fp32
  // 2^x on [-1/2, 1/2] with the least relative error of its degree, 7.5e-5: a fiftieth of the rounding to bf16 that follows
  static __device__ __forceinline__ Pair power(Pair f) {
    Pair y = pair_of(0.05517166852951f, 0.05517166852951f);
    y = fma2(y, f, pair_of(0.24261112511158f, 0.24261112511158f));
    y = fma2(y, f, pair_of(0.69326096773148f, 0.69326096773148f));
    return fma2(y, f, pair_of(0.99992805719376f, 0.99992805719376f));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Half2<__half> {
  static constexpr uint32_t kFormat = 0;
  static constexpr float kLift = 7.f;   // with kSlack below 2^16
  // one degree more, 2.6e-6, for fp16's smaller rounding
  static __device__ __forceinline__ Pair power(Pair f) {
    Pair y = pair_of(0.00957010220736f, 0.00957010220736f);
    y = fma2(y, f, pair_of(0.05591785907745f, 0.05591785907745f));
    y = fma2(y, f, pair_of(0.24024744331837f, 0.24024744331837f));
    y = fma2(y, f, pair_of(0.69312179088593f, 0.69312179088593f));
    return fma2(y, f, pair_of(0.99999928474426f, 0.99999928474426f));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
static_assert(Half2<__half>::kLift + kSlack < 16.f, "weights are finite in fp16");
template <class E>
__host__ __device__ constexpr uint32_t idesc_of(int n) {   // fp32 accumulators, M = 128
  return (1u << 4) | (Half2<E>::kFormat << 7) | (Half2<E>::kFormat << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// 2^x of two values by multiplications: x = n + f with n whole, 2^f by a polynomial, n added to its exponent. Zero below 2^-126.
template <class E>
__device__ __forceinline__ float2 exp2_by_fma(Pair x) {
  const float2 v = parts_of(x);
  x = pair_of(max_or_nan(v.x, -126.f), max_or_nan(v.y, -126.f));
  const float big = 12582912.f;   // 3 * 2^22: sums with it are rounded to whole numbers
  const Pair t = add2(x, pair_of(big, big));
  const Pair f = fma2(add2(t, pair_of(-big, -big)), pair_of(-1.f, -1.f), x);
  const float2 y = parts_of(Half2<E>::power(f)), n = parts_of(t);
  return make_float2(v.x < -126.f ? 0.f : __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                     v.y < -126.f ? 0.f : __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}

// The weights of 32 scores, packed, and added to `sum`. kByFma of them are worked out by multiplications: the special-function unit
// gives 16 a cycle and SM, as long for a tile as its matrix products. (None: window prompts 136 us; 4: 130.5; 8: 129; 12: 129.)
template <class E>
__device__ __forceinline__ void weigh(const uint32_t (&v)[32], float scale, float shift, Pair& sum, uint32_t (&out)[16]) {
  const Pair scales = pair_of(scale, scale), shifts = pair_of(shift, shift);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const Pair x = fma2(pair_of(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), scales, shifts);
    float2 w;
    if (i * kByFma / 32 != (i + 1) * kByFma / 32) {   // spread over them
      w = exp2_by_fma<E>(x);
    } else {
      const float2 a = parts_of(x);
      w = make_float2(exp2_approx(a.x), exp2_approx(a.y));
    }
    sum = add2(sum, pair_of(w.x, w.y));
    out[i] = Half2<E>::pack(w.x, w.y);
  }
}

// Bits of [lo, hi) in a word.
__device__ __forceinline__ uint32_t bits_of(int lo, int hi) {
  lo = max(lo, 0), hi = min(hi, 32);
  if (lo >= hi) return 0u;
  return (0xffffffffu >> (32 - (hi - lo))) << lo;
}

// ---------------------------------------------------------------------------------------------------- the shares

// Tiles and items of a request as cost, by `lanes` neighbouring lanes.
__device__ __forceinline__ long long request_cost(const Params& p, const Request& q, int lane, int lanes) {
  long long sum = 0;
  const int n = blocks_of(p, q.rows);
  for (int b = lane; b < n; b += lanes) sum += span_of(p, q, b).cost(p);
  for (int bit = lanes / 2; bit >= 1; bit >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, bit);
  return sum * p.hkv;
}

// Place number k of `shares` equal parts of the total cost, by a warp. prefix: inclusive sums over the requests. A place within a
// sixteenth of a share from an item's begin is put there.
__device__ Place place_of(const Params& p, const long long* prefix, long long total, int shares, int k) {
  const int lane = threadIdx.x & 31;
  Place at{p.requests, 0, 0, 0};
  if (k >= shares) return at;
  const long long target = total * k / shares;
  int lo = 0, hi = p.requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (prefix[mid] > target) hi = mid;
    else lo = mid + 1;
  }
  at.r = lo;
  const Request q = request_of(p, lo);
  long long rest = target - (lo ? prefix[lo - 1] : 0);
  const int blocks = blocks_of(p, q.rows);
  int cost = 0;
  for (int b0 = 0; b0 < blocks; b0 += 32) {   // 32 blocks at a time
    const int mine = b0 + lane < blocks ? span_of(p, q, b0 + lane).cost(p) : 0;
    long long sum = static_cast<long long>(mine) * p.hkv;
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > rest);
    if (past) {
      const int l = __ffs(past) - 1;
      cost = __shfl_sync(0xffffffffu, mine, l);
      rest -= __shfl_sync(0xffffffffu, sum, l) - static_cast<long long>(cost) * p.hkv;
      at.b = b0 + l;
      break;
    }
    rest -= __shfl_sync(0xffffffffu, sum, 31);
  }
  at.h = static_cast<int>(rest / cost);
  const int off = static_cast<int>(rest - static_cast<long long>(at.h) * cost);
  const long long near = total / shares / 16;
  if (off <= near) return at;
  if (cost - off > near) {
    at.t = max(0, off - kItemCost) / span_of(p, q, at.b).tile_cost(p);
    return at;
  }
  if (++at.h == p.hkv) {
    at.h = 0;
    if (++at.b == blocks) {
      at.b = 0;
      do ++at.r;
      while (at.r < p.requests && prefix[at.r] == prefix[at.r - 1]);
    }
  }
  return at;
}

// Writes the records of the items from place[0] to place[1], and loads each one's queries once the scores of the one before have read theirs.
template <int D, bool kFew>
__device__ void schedule(const Params& p, Shared& sh, uint8_t* q_mem) {
  using L = Layout<D>;
  const int lane = threadIdx.x & 31;
  uint32_t q_uses = 0;
  Place at = sh.place[0];
  const Place end = sh.place[1];
  int seen_from = -1;
  Request seen{0, 0, 0};
  for (int n = 0;; ++n) {
    Record rec;
    rec.pair = -1;
    if (at.r < p.requests && !(same_item(at, end) && end.t <= at.t)) {
      if (seen_from < 0 || at.r >= seen_from + 32) {   // 32 requests in the lanes
        seen_from = at.r;
        if (at.r + lane < p.requests) seen = request_of(p, at.r + lane);
      }
      Request q;
      const int from = at.r - seen_from;
      q.row0 = __shfl_sync(0xffffffffu, seen.row0, from);
      q.rows = __shfl_sync(0xffffffffu, seen.rows, from);
      q.kv_len = __shfl_sync(0xffffffffu, seen.kv_len, from);
      const int blocks = blocks_of(p, q.rows);
      if (at.b >= blocks) {   // a request without rows, or the end of one
        ++at.r;
        at.b = 0;
        --n;
        continue;
      }
      const Span s = span_of(p, q, at.b);
      const int tiles = s.tiles();
      rec.req = at.r;
      rec.head = at.h;
      rec.row0 = q.row0 + at.b * 2 * p.per_stream;
      rec.tokens = s.tokens;
      rec.pos0 = s.pos0;
      rec.past = q.kv_len - q.rows;
      rec.there = min(q.kv_len, p.bt_stride * p.page);
      rec.lo = s.lo;
      rec.hi = s.hi;
      rec.near = s.near;
      rec.split = s.split;
      rec.shift = s.shift;
      rec.t0 = at.t;
      rec.t1 = same_item(at, end) ? end.t : tiles;
      const int cta = static_cast<int>(blockIdx.x);
      rec.slot = rec.t0 > 0 ? 2 * cta : rec.t1 < tiles ? 2 * cta + 1 : -1;
      rec.pair = s.tokens > p.per_stream;
      rec.few = kFew && s.tokens * p.group <= kFewRows;
      at.t = 0;
      if (same_item(at, end)) at.r = p.requests;   // nothing behind it
      else if (++at.h == p.hkv) {
        at.h = 0;
        ++at.b;
      }
    }
    const int slot = n % kRecords;
    if (n >= kRecords && !wait_for(&sh.rec_empty[slot], (n / kRecords - 1) & 1, &sh.abort_flag)) break;
    if (lane == 0) {
      sh.rec[slot] = rec;
      mbar_arrive(&sh.rec_full[slot]);
    }
    __syncwarp();
    if (rec.pair < 0) break;
    if (rec.t0 == rec.t1) continue;
    if (q_uses > 0 && !wait_for(&sh.q_empty, (q_uses - 1) & 1, &sh.abort_flag)) break;
    ++q_uses;
    if (lane == 0) {
      const bool one = rec.tokens == 1;
      const CUtensorMap* const map = one ? &p.q_one_map : &p.q_map;
      mbar_arrive_expect_tx(&sh.q_full, (1 + rec.pair) * L::kHalves * p.group * (one ? 1 : p.per_stream) * 128);
      for (int s = 0; s <= rec.pair; ++s)
        for (int h = 0; h < L::kHalves; ++h)
          load_box_3d(q_mem + s * L::kTileBytes + h * (kTile * 128), map, &sh.q_full, 64 * h, rec.head * p.group, rec.row0 + s * p.per_stream);
    }
    __syncwarp();
  }
  // however it ended, the last queries have landed before the CTA's memory is given up
  int ignored = 0;
  if (q_uses > 0) wait_for(&sh.q_full, (q_uses - 1) & 1, &ignored);
}

// The records one after the other, by every warp of a role alike. What a warp got is its own until it asks for the next one.
struct Records {
  int n = 0;
  __device__ __forceinline__ const Record* next(Shared& sh) {
    if (n > 0) {
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.rec_empty[(n - 1) % kRecords]);
    }
    const int slot = n % kRecords;
    if (!wait_for(&sh.rec_full[slot], (n / kRecords) & 1, &sh.abort_flag)) return nullptr;
    ++n;
    return sh.rec[slot].pair >= 0 ? &sh.rec[slot] : nullptr;
  }
};

// Stage of the operand ring and its parity.
template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// Values in a tile of keys that no row of the item sees become zeros, by a warp: their weights are, but zero times infinity is none.
// tree: of the item's first token, or NULL. Runs while the tile's weights are worked out, and apart from the loop of tiles, which pays for
// every instruction (window prompts 131 us; in line 133, as two functions around the wait for the values 136).
template <int D>
__device__ __noinline__ void clean_values(const int32_t* tree, int words, int tokens, int past, int near, int lo, int hi, int place0, uint8_t* v) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    const int at = place0 + c, d = at - past;   // d: the drafted token of the first key
    uint32_t seen = bits_of(lo - at, hi - at) | bits_of(0, near - at);
    if (tree && d + 32 > 0) {
      const int w = d >> 5, s = d & 31;   // floor; w >= -1
      uint32_t some = 0;
      for (int t = lane; t < tokens; t += 32) {
        const int32_t* const row = tree + static_cast<size_t>(t) * words;
        const uint32_t a = w >= 0 && w < words ? row[w] : 0u, b = w + 1 < words ? row[w + 1] : 0u;
        some |= __funnelshift_r(a, b, s);
      }
      seen &= __reduce_or_sync(0xffffffffu, some) | bits_of(0, -d);
    }
    if (seen == 0xffffffffu) continue;
    for (int k = lane / 8; k < 32; k += 4) {
      if (seen >> k & 1u) continue;
#pragma unroll
      for (int h = 0; h < Layout<D>::kHalves; ++h)
        *reinterpret_cast<uint4*>(v + ((c + k) >> 3) * Layout<D>::kGroupBytes + h * 1024 + (k & 7) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// ------------------------------------------------------------------------------------------------------ the roles

template <int D>
__device__ void produce(const Params& p, Shared& sh, uint8_t* ring_mem) {
  using L = Layout<D>;
  const int lane = threadIdx.x & 31;
  const int pages = kTile / p.page, page_bytes = p.page * D * 2;
  Ring<L::kStages> ring;
  uint32_t loads = 0;
  Records records;
  auto run = [&] {
    while (const Record* const got = records.next(sh)) {
      const Record rec = *got;   // in registers: the loops below would read it again behind every barrier
      const int n = rec.t1 - rec.t0, lead = rec.pair ? 0 : 1;   // K runs one tile ahead of V where the streams take alternate tiles
      const int32_t* const table = p.block_table + static_cast<size_t>(rec.req) * p.bt_stride;
      int ahead = 0;   // this lane's page of the tile of `step`, and whether some row sees a key of it
      bool there = false;
      auto look_up = [&](int j) {
        const int place = (rec.t0 + j) * kTile + lane * p.page;
        there = lane < pages && (place < rec.near || (place + p.page > rec.lo && place < rec.hi));
        ahead = there ? table[(place < rec.split ? place : place + rec.shift) / p.page] : 0;
      };
      int last_page = 0;
      bool last_there = false;
      auto load = [&](const CUtensorMap* map, int page, bool wanted) {
        if (!wait_for(&sh.kv_empty[ring.stage], ring.phase ^ 1, &sh.abort_flag)) return false;
        const uint32_t which = __ballot_sync(0xffffffffu, wanted);
        if (lane == 0) mbar_arrive_expect_tx(&sh.kv_full[ring.stage], __popc(which) * page_bytes);
        __syncwarp();
        if (wanted) load_box_5d(ring_mem + ring.stage * L::kTileBytes + lane * page_bytes, map, &sh.kv_full[ring.stage], L::kHalves * rec.head, page);
        ring.advance();
        ++loads;
        return true;
      };
      for (int step = 0; step < n + lead; ++step) {
        if (step < n) {
          look_up(step);
          if (!load(&p.k_map, ahead, there)) return;
        }
        if (lead == 0) {
          if (!load(&p.v_map, ahead, there)) return;
        } else {
          if (step > 0 && !load(&p.v_map, last_page, last_there)) return;
          last_page = ahead;
          last_there = there;
        }
      }
    }
  };
  run();
  // however it ended, the last loads have landed before the CTA's memory is given up
  for (uint32_t i = loads > L::kStages ? loads - L::kStages : 0; i < loads; ++i) {
    int ignored = 0;
    wait_for(&sh.kv_full[i % L::kStages], (i / L::kStages) & 1, &ignored);
  }
}

// The products of both streams, by one warp: it keeps them a step apart, so that one stream's products run under the other's softmax.
template <class E, int D, bool kFew>
__device__ void multiply(const Params& p, Shared& sh, uint8_t* q_mem, uint8_t* ring_mem) {
  using L = Layout<D>;
  const int lane = threadIdx.x & 31;
  const bool leader = elect_one();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem_base, 0);
  constexpr uint32_t idesc_s = idesc_of<E>(kTile), idesc_o = idesc_of<E>(D) | (1u << 16);   // V is MN-major
  Ring<L::kStages> ring;
  Records records;
  uint32_t q_count = 0, p_phase = 0;   // p_phase: bit x, the parity of stream x's next weights
  auto wait_stage = [&] { return wait_for(&sh.kv_full[ring.stage], ring.phase, &sh.abort_flag); };
  auto release = [&](int stage) {
    if (leader) umma_commit(&sh.kv_empty[stage]);
  };
  auto scores = [&](int x, int q_tile) {   // S[x] = Q K^T of the ring's stage
    if (!leader) return;
    const uint32_t q = (smem_u32(q_mem) + q_tile * L::kTileBytes) >> 4, k = (smem_u32(ring_mem) + ring.stage * L::kTileBytes) >> 4;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      umma_bf16(tmem + x * 128, smem_desc(q + (i >> 2) * (kTile * 8) + (i & 3) * 2, 1024), smem_desc(k + (i >> 2) * 64 + (i & 3) * 2, L::kGroupBytes), idesc_s,
                i != 0);
    umma_commit(&sh.s_full[x]);
  };
  auto values = [&](int x, int stage, bool accumulate) {   // O[x] (+)= P[x] V
    const uint32_t v = (smem_u32(ring_mem) + stage * L::kTileBytes) >> 4 | 64u << 16;
    if (!wait_for(&sh.p_full[x], p_phase >> x & 1, &sh.abort_flag)) return false;
    p_phase ^= 1u << x;
    tc_fence_after_sync();
    if (leader) {
#pragma unroll
      for (int i = 0; i < kTile / 16; ++i)
        umma_tmem_a(tmem + 256 + x * 128, tmem + x * 128 + 8 * i, smem_desc(v + i * (L::kGroupBytes / 8), L::kGroupBytes), idesc_o, accumulate || i != 0);
    }
    return true;
  };
  auto clean = [&](const Record& rec, int stage, int t) {
    const int place0 = t * kTile, alike = p.tree ? min(rec.hi, rec.past) : rec.hi;
    if (place0 + kTile <= rec.near || (place0 >= rec.lo && place0 + kTile <= alike)) return;
    clean_values<D>(p.tree ? p.tree + static_cast<size_t>(rec.row0) * p.words : nullptr, p.words, rec.tokens, rec.past, rec.near, rec.lo, rec.hi, place0,
                    ring_mem + stage * L::kTileBytes);
  };
  // An item of few rows: S^T[x] = K Q^T and O^T[x] (+)= V^T P^T[x]. Apart from the others, whose loop pays for every instruction.
  auto run_few = [&](const Record& rec, int n) {
    auto scores_few = [&](int x) {
      if (!wait_stage()) return false;
      tc_fence_after_sync();
      if (leader) {
        const uint32_t q = smem_u32(q_mem) >> 4, k = (smem_u32(ring_mem) + ring.stage * L::kTileBytes) >> 4;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          umma_bf16(tmem + x * 128, smem_desc(k + (i >> 2) * 64 + (i & 3) * 2, L::kGroupBytes), smem_desc(q + (i >> 2) * (kTile * 8) + (i & 3) * 2, 1024),
                    idesc_of<E>(kFewRows), i != 0);
        umma_commit(&sh.s_full[x]);
        umma_commit(&sh.kv_empty[ring.stage]);
      }
      ring.advance();
      return true;
    };
    for (int j = 0; j < min(n, 2); ++j)
      if (!scores_few(j)) return false;
    for (int j = 0; j < n; ++j) {
      const int x = j & 1;
      if (!wait_stage()) return false;
      clean(rec, ring.stage, rec.t0 + j);
      if (!wait_for(&sh.p_full[x], p_phase >> x & 1, &sh.abort_flag)) return false;
      p_phase ^= 1u << x;
      tc_fence_after_sync();
      if (leader) {
        const uint32_t v = (smem_u32(ring_mem) + ring.stage * L::kTileBytes) >> 4 | 64u << 16;
        const uint32_t w = smem_u32(q_mem + L::kTileBytes + x * kFewBytes) >> 4;
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i)
          umma_bf16(tmem + 256 + x * 128, smem_desc(v + i * (L::kGroupBytes / 8), L::kGroupBytes), smem_desc(w + (i >> 2) * (kFewRows * 8) + (i & 3) * 2, 1024),
                    idesc_of<E>(kFewRows) | 1u << 15, j > 1 || i != 0);   // V is MN-major
        umma_commit(&sh.kv_empty[ring.stage]);
      }
      ring.advance();
      if (j + 2 < n && !scores_few(x)) return false;
    }
    if (leader) {
      umma_commit(&sh.q_empty);   // not before: the weights lie where a pair's other queries go
      umma_commit(&sh.o_full[0]);
      if (n > 1) umma_commit(&sh.o_full[1]);
    }
    return true;
  };
  auto run = [&] {
    while (const Record* const got = records.next(sh)) {
      const Record rec = *got;   // in registers: the loops below would read it again behind every barrier
      const int n = rec.t1 - rec.t0;
      const bool pair = rec.pair;
      if (n == 0) continue;
      if (!wait_for(&sh.q_full, q_count & 1, &sh.abort_flag)) return;
      ++q_count;
      if constexpr (kFew) {
        if (rec.few) {
          if (!run_few(rec, n)) return;
          continue;
        }
      }
      // The stages come as K 0, V 0, K 1, V 1 ... for a pair, else as K 0, K 1, V 0, K 2, V 1, ... K n - 1, V n - 2, V n - 1.
      for (int j = 0; j < (pair ? 1 : min(n, 2)); ++j) {
        if (!wait_stage()) return;
        tc_fence_after_sync();
        scores(j, 0);
        if (pair) scores(1, 1);
        release(ring.stage);
        ring.advance();
      }
      if (leader && n <= (pair ? 1 : 2)) umma_commit(&sh.q_empty);
      for (int j = 0; j < n; ++j) {
        if (!wait_stage()) return;
        const int v_stage = ring.stage;
        clean(rec, v_stage, rec.t0 + j);
        ring.advance();
        const bool more = pair ? j + 1 < n : j + 2 < n;
        for (int x = pair ? 0 : j & 1; x <= (pair ? 1 : j & 1); ++x) {
          if (!values(x, v_stage, pair ? j > 0 : j > 1)) return;
          if (leader && !pair) umma_commit(&sh.kv_empty[v_stage]);
          if (!more) {
            if (leader && pair) umma_commit(&sh.o_full[x]);
            continue;
          }
          if (x == 0 || !pair) {
            if (!wait_stage()) return;
            tc_fence_after_sync();
          }
          scores(x, pair ? x : 0);
        }
        if (pair) release(v_stage);
        if (more) {
          release(ring.stage);
          if (leader && j + (pair ? 2 : 3) == n) umma_commit(&sh.q_empty);
          ring.advance();
        }
      }
      // Only of streams that have tiles: their softmax holds this warp back. Without, the barrier could be completed twice before
      // its waiters look.
      if (leader && !pair) {
        umma_commit(&sh.o_full[0]);
        if (n > 1) umma_commit(&sh.o_full[1]);
      }
    }
  };
  run();
  // whatever ended the loop: nothing of this warp is in flight when it leaves
  if (leader) umma_commit(&sh.drain);
  int ignored = 0;
  wait_for(&sh.drain, 0, &ignored);
}

// 64 bytes of each lane's row, at `to` (NULL: of none). Four lanes exchange 16-byte pieces, so that they store 64 bytes of one row side
// by side: 32 rows' pieces in one instruction, each in another line, take four times as long.
__device__ __forceinline__ void store_lines(uint32_t (&w)[16], void* to) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {   // transposes 4 x 4 pieces
    const bool hi = lane & bit;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & bit) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t &a = w[4 * i + k], &b = w[4 * (i | bit) + k];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, hi ? a : b, bit);
        if (hi) a = got;
        else b = got;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // w[4 i ..]: of the group's row i
    uint4* const row = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), (lane & 28) + i));
    if (row) row[lane & 3] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

struct Counts {   // phases of the barriers so far: tiles, items with tiles, joined items, tiles of few rows
  uint32_t s = 0, o = 0, x = 0, told = 0;
};

// An item of at most 16 rows: S^T = K Q^T and O^T = V^T P^T, keys and head dims on the 128 lanes and the rows as columns, so that
// neither the products nor the exponentials are of 128 rows. A thread has a key of each tile. A row's reference is known to all of a
// stream's threads and held by lane `row`, too; the weights go to shared memory, as the other operand.
template <class E>
__device__ bool softmax_few(const Params& p, Shared& sh, uint8_t* q_mem, const Record& rec, int wg, Counts& c) {
  constexpr int D = 128, N = kFewRows;
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3, r = quad * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
  const uint32_t tmem_s = sh.tmem_base + wg * 128 + lanes, tmem_o = sh.tmem_base + 256 + lanes;
  uint8_t* const mine = q_mem + Layout<D>::kTileBytes + wg * kFewBytes + (r >> 6) * (kFewRows * 128) + (r & 7) * 2;   // the key's place in row 0
  const int chunk = (r & 63) >> 3;
  const int n = rec.t1 - rec.t0, rows = rec.tokens * p.group;
  const float scale = p.scale_log2;
  float m[N], l[N], held = -INFINITY;   // held: the reference of row `lane`
#pragma unroll
  for (int i = 0; i < N; ++i) m[i] = l[i] = 0.f;
  bool begun = false;
#pragma unroll 1
  for (int j = wg; j < n; j += 2) {
    if (!wait_for(&sh.s_full[wg], c.s & 1, &sh.abort_flag)) return false;
    ++c.s;
    tc_fence_after_sync();
    const int place0 = (rec.t0 + j) * kTile, place = place0 + r, key = place < rec.split ? place : place + rec.shift;
    float s[N];
    {
      uint32_t v[N];
      tmem_ld_32x16(tmem_s, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = __uint_as_float(v[i]) * scale;
    }
    bool full;
    if (p.tree) full = place0 + kTile <= min(rec.past, rec.there);
    else full = place0 + kTile <= rec.near || (place0 + kTile + rec.shift <= min(rec.pos0 + 1, rec.there) &&
                                               static_cast<long long>(place0) + rec.shift >= static_cast<long long>(rec.pos0) + rec.tokens - p.window);
    if (!full) {
      uint32_t seen = 0;   // the rows that see the key
      const uint32_t token = (1u << p.group) - 1u;
      for (int t = 0; t < rec.tokens; ++t) {
        bool sees = key < rec.there;
        if (p.tree) {
          const int d = key - rec.past;
          if (d >= 0) sees = sees && (d >> 5) < p.words && (p.tree[static_cast<size_t>(rec.row0 + t) * p.words + (d >> 5)] >> (d & 31) & 1);
        } else {
          const int pos = rec.pos0 + t;
          sees = sees && key <= pos && (key > static_cast<long long>(pos) - p.window || key < p.sinks);
        }
        if (sees) seen |= token << (t * p.group);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = seen >> i & 1u ? s[i] : -INFINITY;
    }
    float own = -INFINITY;   // the warp's maximum of row `lane`
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float top = warp_max(s[i]);
      if (lane == i) own = top;
    }
    if (lane < N) sh.few.top[wg][quad][lane] = own;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.told[wg]);
    if (!wait_for(&sh.told[wg], c.told & 1, &sh.abort_flag)) return false;
    ++c.told;
    float top = -INFINITY;
    if (lane < rows) top = fmaxf(fmaxf(sh.few.top[wg][0][lane], sh.few.top[wg][1][lane]), fmaxf(sh.few.top[wg][2][lane], sh.few.top[wg][3][lane]));
    const bool grows = begun ? top > held + kSlack : true;
    if (__any_sync(0xffffffffu, lane < rows && grows)) {   // of all four warps alike
      const float moved = grows ? top : held;
      if (begun) {   // S of this tile is there, so P V of the stream's tile before it is, too
        const float alpha = moved > held ? exp2_approx(held - moved) : 1.f;
        uint32_t o[N];
        tmem_ld_32x16(tmem_o + wg * 128, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float a = __shfl_sync(0xffffffffu, alpha, i);
          o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
          l[i] *= a;
        }
        store_tmem_16(tmem_o + wg * 128, o);
        store_tmem_wait();
      }
      held = moved;
      const float shift = held == -INFINITY ? 0.f : held - Half2<E>::kLift;
#pragma unroll
      for (int i = 0; i < N; ++i) m[i] = __shfl_sync(0xffffffffu, shift, i);
    }
    begun = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = exp2_approx(s[i] - m[i]);
      l[i] += w;
      *reinterpret_cast<E*>(mine + i * 128 + ((chunk ^ (i & 7)) << 4)) = static_cast<E>(w);
    }
    fence_proxy_async_smem();
    tc_fence_before_sync();
    mbar_arrive(&sh.p_full[wg]);
  }
  if (n > wg) {   // the stream has tiles
    if (!wait_for(&sh.o_full[wg], c.o & 1, &sh.abort_flag)) return false;
    ++c.o;
    tc_fence_after_sync();
  }
  float sum = 0.f;   // the warp's part of row `lane`'s sum
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = l[i];
#pragma unroll
    for (int bit = 16; bit; bit >>= 1) t += __shfl_xor_sync(0xffffffffu, t, bit);
    if (lane == i) sum = t;
  }
  if (lane < N) sh.few.sum[wg][quad][lane] = sum;
  if (quad == 0 && lane < N) sh.few.m[wg][lane] = held;
  mbar_arrive(&sh.x_full);
  if (!wait_for(&sh.x_full, c.x & 1, &sh.abort_flag)) return false;
  tc_fence_after_sync();
  // of row `lane`: how the streams are joined
  const int at = min(lane, N - 1);
  const float ma = sh.few.m[0][at], mb = sh.few.m[1][at], ref = fmaxf(ma, mb), shift = ref == -INFINITY ? 0.f : ref;
  const float ea = exp2_approx(ma - shift), eb = exp2_approx(mb - shift);
  float sums[2] = {0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    sums[0] += sh.few.sum[0][q][at];
    sums[1] += sh.few.sum[1][q][at];
  }
  const float total = sums[0] * ea + sums[1] * eb;
  const float inv = rec.slot >= 0 ? 1.f : total == 0.f ? 0.f : 1.f / total;
  // where row `lane` goes; the streams' threads store every other row
  const int token = at / p.group, head = rec.head * p.group + at - token * p.group;
  unsigned long long to = 0;
  if (lane < rows)
    to = rec.slot >= 0 ? reinterpret_cast<unsigned long long>(p.ws_o + (static_cast<size_t>(rec.slot) * kSlotRows + lane) * D)
                       : reinterpret_cast<unsigned long long>(static_cast<E*>(p.out) + (rec.row0 + token) * p.out_row + head * p.out_head);
  const float fa = n > 0 ? ea * inv : 0.f, fb = n > 1 ? eb * inv : 0.f;
#pragma unroll 1
  for (int c0 = 0; c0 < rows; c0 += 4) {
    uint32_t a[4], b[4];   // head dim r of four rows, of the two streams
    if (n > 0) load_tmem_4(tmem_o + c0, a);
    if (n > 1) load_tmem_4(tmem_o + 128 + c0, b);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ga = __shfl_sync(0xffffffffu, fa, c0 + i), gb = __shfl_sync(0xffffffffu, fb, c0 + i);
      const unsigned long long row = __shfl_sync(0xffffffffu, to, c0 + i);
      if ((i & 1) == wg && row) {
        float f = n > 0 ? __uint_as_float(a[i]) * ga : 0.f;
        if (n > 1) f = fmaf(__uint_as_float(b[i]), gb, f);
        if (rec.slot >= 0) reinterpret_cast<float*>(row)[r] = f;
        else reinterpret_cast<E*>(row)[r] = static_cast<E>(f);
      }
    }
    __syncwarp();
  }
  if (rec.slot >= 0 && quad == 0 && wg == 0 && lane < rows) p.ws_ml[static_cast<size_t>(rec.slot) * kSlotRows + lane] = make_float2(ref, total);
  tc_fence_before_sync();
  mbar_arrive(&sh.x_done);
  if (!wait_for(&sh.x_done, c.x & 1, &sh.abort_flag)) return false;
  ++c.x;
  return true;
}

template <class E, int D, bool kFew>
__device__ void softmax(const Params& p, Shared& sh, uint8_t* q_mem, int wg) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3, r = quad * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
  const uint32_t tmem_s = sh.tmem_base + wg * 128 + lanes, tmem_o = sh.tmem_base + 256 + lanes;
  const int token_in = r / p.group, head_in = r - token_in * p.group;
  Counts counts;
  Records records;
  const float scale = p.scale_log2;
  while (const Record* const got = records.next(sh)) {
    const Record& rec = *got;
    if constexpr (kFew) {
      if (rec.few) {
        if (!softmax_few<E>(p, sh, q_mem, rec, wg, counts)) return;
        continue;
      }
    }
    const int n = rec.t1 - rec.t0;
    const bool pair = rec.pair;
    const int first = pair ? wg * p.per_stream : 0;                            // first token of the stream in the item
    const int tokens = min(rec.tokens - first, p.per_stream);
    const bool row_ok = r < tokens * p.group;
    const bool works = quad * 32 < tokens * p.group;                           // warp-uniform
    // first places of the tiles that all rows of the stream see: from full_lo to full_hi, or up to full_near
    const int pos_first = rec.pos0 + first;
    const int full_hi = min(p.tree ? rec.past : pos_first + 1, rec.there) - rec.shift - kTile;
    const int full_lo = p.tree ? 0 : static_cast<int>(max(0ll, static_cast<long long>(pos_first + tokens) - p.window)) - rec.shift;
    const int full_near = rec.near - kTile;
    float m = -INFINITY, l = 0.f;
    bool begun = false;
#pragma unroll 1
    for (int j = pair ? 0 : wg; j < n; j += pair ? 1 : 2) {
      if (!wait_for(&sh.s_full[wg], counts.s & 1, &sh.abort_flag)) return;
      ++counts.s;
      tc_fence_after_sync();
      if (!works) {   // no row of this warp exists
        tc_fence_before_sync();
        mbar_arrive(&sh.p_full[wg]);
        continue;
      }
      const int place0 = (rec.t0 + j) * kTile;
      const bool full = place0 <= full_near || (place0 <= full_hi && place0 >= full_lo);
      uint32_t seen[4];   // what the row sees of the tile
      if (!full) {
        if (p.tree) {
          const int32_t* const words = p.tree + static_cast<size_t>(rec.row0 + (row_ok ? first + token_in : 0)) * p.words;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int d = place0 + 32 * c - rec.past;   // the drafted token of the first column; places are keys
            const int w = d >> 5, s = d & 31;         // floor
            const uint32_t a = w >= 0 && w < p.words ? words[w] : 0u, b = w + 1 >= 0 && w + 1 < p.words ? words[w + 1] : 0u;
            seen[c] = (__funnelshift_r(a, b, s) | bits_of(0, -d)) & bits_of(0, rec.there - place0 - 32 * c);
          }
        } else {
          const int pos = pos_first + token_in;
          // as places: the window's keys lie behind the split, where place = key - shift; what is near lies in front of it, or
          // there is no split and the row's own sinks may reach into the window of an earlier one
          const long long origin = static_cast<long long>(place0) + rec.shift;
          const int hi = static_cast<int>(max(0ll, min(min(static_cast<long long>(pos) + 1, static_cast<long long>(rec.there)) - origin, static_cast<long long>(kTile))));
          const int lo = static_cast<int>(max(0ll, min(static_cast<long long>(pos) - p.window + 1 - origin, static_cast<long long>(kTile))));
          const int near = rec.split ? rec.near - place0 : min(p.sinks - place0, rec.shift ? 0 : hi);
#pragma unroll
          for (int c = 0; c < 4; ++c) seen[c] = bits_of(lo - 32 * c, hi - 32 * c) | bits_of(0, near - 32 * c);
        }
      }
      if (!full) {   // what the row does not see is hidden in TMEM, so that the loops below need not know
#pragma unroll 1
        for (int c = 0; c < kTile; c += 32) {
          const uint32_t bits = c < 64 ? (c < 32 ? seen[0] : seen[1]) : (c < 96 ? seen[2] : seen[3]);
          if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;   // a border lies in one or two of the four chunks
          uint32_t v[32];
          tmem_ld_32x32(tmem_s + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = bits >> i & 1u ? v[i] : 0xff800000u;
          store_tmem_16(tmem_s + c, v);
          store_tmem_16(tmem_s + c + 16, v + 16);
        }
        store_tmem_wait();
      }
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < kTile; c += 64) {
        uint32_t v[64];
        tmem_ld_32x32(tmem_s + c, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld_32x32(tmem_s + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_ld_wait();
        float top[4] = {mx, mx, mx, mx};
#pragma unroll
        for (int i = 0; i < 64; i += 2) top[i / 2 & 3] = max3_or_nan(top[i / 2 & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        mx = max3_or_nan(max_or_nan(top[0], top[1]), top[2], top[3]);
      }
      mx *= scale;
      if (!(mx < INFINITY)) l = NAN;   // not left to the weights: those by multiplications make a number of it
      // The point that a row's exponentials refer to moves when its maximum has grown past it by more than kSlack: weights stay
      // below 2^kSlack, and O is rarely rescaled. S of this tile is there, so P V of the stream's tile before it is, too.
      if (!begun) {
        m = mx;
      } else {
        if (!(mx > m + kSlack)) mx = m;
        if (__any_sync(0xffffffffu, mx > m && row_ok)) {
          const float alpha = mx > m ? exp2_approx(m - mx) : 1.f;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld_32x16(tmem_o + wg * 128 + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            store_tmem_16(tmem_o + wg * 128 + c, o);
          }
          l *= alpha;
          m = mx;
        }
      }
      begun = true;
      const float shift = m == -INFINITY ? 0.f : Half2<E>::kLift == 0.f ? -m : Half2<E>::kLift - m;
      Pair sum = 0ull;
#pragma unroll 1
      for (int c = 0; c < kTile; c += 32) {
        uint32_t v[32], w[16];
        tmem_ld_32x32(tmem_s + c, v);
        tmem_ld_wait();
        weigh<E>(v, scale, shift, sum, w);
        store_tmem_16(tmem_s + c / 2, w);
      }
      const float2 sums = parts_of(sum);
      l += sums.x + sums.y;
      store_tmem_wait();
      tc_fence_before_sync();
      mbar_arrive(&sh.p_full[wg]);
    }
    if (n > (pair ? 0 : wg)) {   // the stream has tiles
      if (!wait_for(&sh.o_full[wg], counts.o & 1, &sh.abort_flag)) return;
      ++counts.o;
      tc_fence_after_sync();
    }
    // Rows of the item: of a pair both streams have their own; else the streams' results are joined, each group storing half of
    // the columns.
    E* const out = static_cast<E*>(p.out) + (rec.row0 + first + token_in) * p.out_row + (rec.head * p.group + head_in) * p.out_head;
    const size_t ws_row = rec.slot < 0 ? 0 : static_cast<size_t>(rec.slot) * kSlotRows + (rec.pair ? wg * kTile : 0) + r;
    float wa = 1.f, wb = 0.f, total = l, ref = m;
    int c0 = 0, c1 = D, other = 0;
    if (!rec.pair) {
      sh.ml[wg][r] = make_float2(m, l);
      mbar_arrive(&sh.x_full);
      if (!wait_for(&sh.x_full, counts.x & 1, &sh.abort_flag)) return;
      tc_fence_after_sync();   // the other stream's products are there, too: its threads have waited for them
      const float2 a = sh.ml[0][r], b = sh.ml[1][r];
      ref = fmaxf(a.x, b.x);
      const float at = ref == -INFINITY ? 0.f : ref;
      wa = exp2_approx(a.x - at);
      wb = exp2_approx(b.x - at);
      total = a.y * wa + b.y * wb;
      c0 = wg * (D / 2);
      c1 = c0 + D / 2;
      other = 128;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const uint32_t from = tmem_o + (rec.pair ? wg * 128 : 0);
    if (works) {
#pragma unroll 1
      for (int c = c0; c < c1; c += 32) {
        uint32_t a[32], b[32];
        float f[32];
        if (n > 0) {
          tmem_ld_32x32(from + c, a);
          if (other && n > 1) tmem_ld_32x32(from + other + c, b);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          f[i] = n > 0 ? __uint_as_float(a[i]) * wa : 0.f;
          if (other && n > 1) f[i] += __uint_as_float(b[i]) * wb;
        }
        if (rec.slot >= 0) {
          float* const to = row_ok ? p.ws_o + ws_row * D + c : nullptr;
          uint32_t w[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(f[16 * g + i]);
            store_lines(w, to ? to + 16 * g : nullptr);
          }
        } else {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = Half2<E>::pack(f[2 * i] * inv, f[2 * i + 1] * inv);
          store_lines(w, row_ok ? out + c : nullptr);
        }
        __syncwarp();
      }
      if (rec.slot >= 0 && row_ok && c0 == 0) p.ws_ml[ws_row] = make_float2(ref, total);
    }
    tc_fence_before_sync();
    if (!rec.pair) {   // the accumulators and the exchange are free once both groups have read them
      mbar_arrive(&sh.x_done);
      if (!wait_for(&sh.x_done, counts.x & 1, &sh.abort_flag)) return;
      ++counts.x;
    }
  }
}

template <class E, int D, bool kFew>
__global__ void __launch_bounds__(kThreads, 1) masked_attention_kernel(const __grid_constant__ Params p) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(16) Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_release();
  if (tid == 0) {
    sh.abort_flag = 0;
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    for (int i = 0; i < kRecords; ++i) {
      mbar_init(&sh.rec_full[i], 1);
      mbar_init(&sh.rec_empty[i], 10);   // loads, products and eight warps of softmax
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 128);
      mbar_init(&sh.o_full[i], 1);
      mbar_init(&sh.told[i], 4);
    }
    mbar_init(&sh.x_full, 256);
    mbar_init(&sh.x_done, 256);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  chain_wait();
  // The shares: each CTA adds up what all requests cost and finds where its part begins and ends.
  long long* const prefix = reinterpret_cast<long long*>(smem);
  int lanes = 32;
  while (lanes > 1 && p.requests * lanes > kThreads) lanes /= 2;
  for (int r0 = 0; r0 < p.requests; r0 += kThreads / lanes) {
    const int r = r0 + tid / lanes;
    Request q{0, 0, 0};
    if (r < p.requests) q = request_of(p, r);
    const long long cost = request_cost(p, q, tid % lanes, lanes);
    if (r < p.requests && tid % lanes == 0) prefix[r] = cost;
  }
  __syncthreads();
  if (warp == 0) {
    long long before = 0;
    for (int r0 = 0; r0 < p.requests; r0 += 32) {
      long long sum = r0 + lane < p.requests ? prefix[r0 + lane] : 0;
      for (int d = 1; d < 32; d <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      sum += before;
      if (r0 + lane < p.requests) prefix[r0 + lane] = sum;
      before = __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __syncthreads();
  const long long total = prefix[p.requests - 1];
  const int shares = static_cast<int>(max(min(static_cast<long long>(gridDim.x), total / kMinCost), total > 0 ? 1ll : 0ll));
  const bool mine = static_cast<int>(blockIdx.x) < shares;
  if (warp < 2 && mine) {
    const Place at = place_of(p, prefix, total, shares, blockIdx.x + warp);
    if (lane == 0) sh.place[warp] = at;
  }
  fence_proxy_async_smem();   // the loads write where the sums were
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (tid == 0) {   // for the kernel that joins the parts
    int4 a = make_int4(0, 0, 0, 0), b = a;
    if (mine && sh.place[0].t > 0) {
      const Place at = sh.place[0];
      const Request q = request_of(p, at.r);
      a = make_int4(1, at.r, at.b, at.h);
      b = make_int4(q.row0 + at.b * 2 * p.per_stream, min(2 * p.per_stream, q.rows - at.b * 2 * p.per_stream), 0, 0);
    }
    p.ws_meta[2 * blockIdx.x] = a;
    p.ws_meta[2 * blockIdx.x + 1] = b;
  }
  uint8_t* const ring_mem = smem + 2 * L::kTileBytes;
  if (warp < 4) {
    if (mine) {
      if (warp == 0) produce<D>(p, sh, ring_mem);
      else if (warp == 1) multiply<E, D, kFew>(p, sh, smem, ring_mem);
      else if (warp == 2) schedule<D, kFew>(p, sh, smem);
    }
  } else {
    if (mine) softmax<E, D, kFew>(p, sh, smem, (warp - 4) >> 2);
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (tid == 0 && sh.abort_flag) atomicOr(p.status ? p.status : &g_masked_attention_status, kErrWaitTimeout);
  if (warp == 1) tmem_dealloc(sh.tmem_base, 512);
}

// Joins the parts of the items that lie in several CTAs' shares, in order. Blocks (k, .): of the item inside which CTA k's share begins,
// if it is the first to begin there. What bounds it is latency, so there are two steps of loads: 32 shares' beginnings by the
// lanes of each warp, then four parts of two rows together. (One row after the other, with a chain of
// loads for its parts: 12 us where a batch of trees takes 47.)
template <class E, int D>
__global__ void __launch_bounds__(256) masked_join_kernel(const __grid_constant__ Params p, int ctas) {
  constexpr int kRows = 2, kParts = 4, kOwn = D / 32;   // kOwn: columns of a lane
  using Piece = std::conditional_t<kOwn == 4, float4, float2>;
  chain_release();
  chain_wait();
  const int k = blockIdx.x + 1, lane = threadIdx.x & 31;
  // how the shares of CTAs k - 1, k, k + 1, ... begin
  const int4 before = p.ws_meta[2 * (k - 1)], rows = p.ws_meta[2 * k + 1];
  int4 at_lane = k + lane < ctas ? p.ws_meta[2 * (k + lane)] : make_int4(0, 0, 0, 0);
  const int4 it = make_int4(__shfl_sync(0xffffffffu, at_lane.x, 0), __shfl_sync(0xffffffffu, at_lane.y, 0), __shfl_sync(0xffffffffu, at_lane.z, 0),
                            __shfl_sync(0xffffffffu, at_lane.w, 0));
  auto same = [&](const int4& a) { return a.x && a.y == it.y && a.z == it.z && a.w == it.w; };
  if (!it.x || same(before)) return;
  int parts = 1;   // the tail of CTA k - 1, then the heads of k, k + 1, ...
  for (int from = k;;) {
    const uint32_t others = ~__ballot_sync(0xffffffffu, same(at_lane));
    parts += others ? __ffs(others) - 1 : 32;
    if (others) break;
    from += 32;
    at_lane = from + lane < ctas ? p.ws_meta[2 * (from + lane)] : make_int4(0, 0, 0, 0);
  }
  const int row0 = rows.x, tokens = rows.y;
  const int n = tokens * p.group, warps = gridDim.y * 8;
  const bool pair = tokens > p.per_stream;
  auto slot = [&](int q) { return static_cast<size_t>(q == 0 ? 2 * (k - 1) + 1 : 2 * (k + q - 1)) * kSlotRows; };
  for (int i0 = blockIdx.y * 8 + threadIdx.x / 32; i0 < n; i0 += kRows * warps) {
    int at[kRows];   // places of the rows in a slot
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int i = min(i0 + j * warps, n - 1);
      at[j] = pair && i >= p.per_stream * p.group ? kTile + i - p.per_stream * p.group : i;
    }
    float top[kRows], sum[kRows], o[kRows][kOwn];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      top[j] = -INFINITY;
      sum[j] = 0.f;
#pragma unroll
      for (int d = 0; d < kOwn; ++d) o[j][d] = 0.f;
    }
    for (int q0 = 0; q0 < parts; q0 += kParts) {
      float2 ml[kParts][kRows];
      Piece piece[kParts][kRows];
#pragma unroll
      for (int q = 0; q < kParts; ++q)
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          const size_t row = slot(min(q0 + q, parts - 1)) + at[j];
          ml[q][j] = p.ws_ml[row];
          piece[q][j] = reinterpret_cast<const Piece*>(p.ws_o + row * D)[lane];
        }
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        if (q0 + q >= parts) break;
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          const float ref = fmaxf(top[j], ml[q][j].x), from = ref == -INFINITY ? 0.f : ref;
          const float keep = exp2_approx(top[j] - from), w = exp2_approx(ml[q][j].x - from);
          top[j] = ref;
          sum[j] = sum[j] * keep + ml[q][j].y * w;
#pragma unroll
          for (int d = 0; d < kOwn; ++d) o[j][d] = o[j][d] * keep + reinterpret_cast<const float*>(&piece[q][j])[d] * w;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int i = i0 + j * warps;
      if (i >= n) break;
      const float inv = sum[j] == 0.f ? 0.f : 1.f / sum[j];
      const int token = i / p.group, head = it.w * p.group + i - token * p.group;
      E* const out = static_cast<E*>(p.out) + (row0 + token) * p.out_row + head * p.out_head + lane * kOwn;
      uint32_t w[kOwn / 2];
#pragma unroll
      for (int d = 0; d < kOwn / 2; ++d) w[d] = Half2<E>::pack(o[j][2 * d] * inv, o[j][2 * d + 1] * inv);
      if constexpr (kOwn == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(out) = w[0];
    }
  }
}

struct Grid {
  int ctas;
  size_t o_bytes, ml_bytes, meta_bytes;
};
// One CTA per SM and the workspace of all of them, whatever the call: how much there is to do stands in lengths on the device.
Grid grid_of(int head_dim, int sms) {
  Grid g;
  g.ctas = sms;
  g.o_bytes = static_cast<size_t>(2 * g.ctas) * kSlotRows * head_dim * sizeof(float);
  g.ml_bytes = static_cast<size_t>(2 * g.ctas) * kSlotRows * sizeof(float2);
  g.meta_bytes = static_cast<size_t>(g.ctas) * 2 * sizeof(int4);
  return g;
}

template <class E, int D, bool kFew = false>
cudaError_t launch(const Params& p, const Grid& g, cudaStream_t stream) {
  static PerDeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(masked_attention_kernel<E, D, kFew>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kSmem);
  });
  if (e == cudaSuccess) e = launch_chained(masked_attention_kernel<E, D, kFew>, dim3(g.ctas), dim3(kThreads), Layout<D>::kSmem, stream, p);
  if (e == cudaSuccess && g.ctas > 1) e = launch_chained(masked_join_kernel<E, D>, dim3(g.ctas - 1, 8), dim3(256), 0, stream, p, g.ctas);
  return e;
}

int sm_count(int* sms) {
  int device = 0;
  MF_CUDA(cudaGetDevice(&device));
  MF_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
  return MONOFAB_OK;
}

}  // namespace

}  // namespace mf

using namespace mf;

extern "C" int64_t monofab_masked_attention_ws_bytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(MONOFAB_EINVAL, "masked_attention: head_dim=%d must be 64 or 128", head_dim);
  int sms = 0;
  if (int r = sm_count(&sms)) return r;
  const Grid g = grid_of(head_dim, sms);
  return static_cast<int64_t>(g.o_bytes + g.ml_bytes + g.meta_bytes);
}

extern "C" int monofab_masked_attention(const monofab_masked_attention_args* a, void* stream) {
  if (!a) return fail(MONOFAB_EINVAL, "masked_attention: NULL argument");
  if (a->tokens < 0 || a->requests < 0 || a->n_pages < 1 || a->bt_stride < 1)
    return fail(MONOFAB_EINVAL, "masked_attention: tokens=%d, requests=%d, n_pages=%d, bt_stride=%d", a->tokens, a->requests, a->n_pages, a->bt_stride);
  if (a->requests > kMaxRequests) return fail(MONOFAB_EINVAL, "masked_attention: %d requests, at most %d a call", a->requests, kMaxRequests);
  if (a->hkv < 1 || a->hq < a->hkv || a->hq % a->hkv) return fail(MONOFAB_EINVAL, "masked_attention: hq=%d must be a multiple of hkv=%d", a->hq, a->hkv);
  const int group = a->hq / a->hkv, D = a->head_dim;
  if (group > 128) return fail(MONOFAB_EINVAL, "masked_attention: %d query heads for a KV head, at most 128", group);
  if (D != 64 && D != 128) return fail(MONOFAB_EINVAL, "masked_attention: head_dim=%d must be 64 or 128", D);
  if (a->page_size < 8 || a->page_size > 128 || 128 % a->page_size)
    return fail(MONOFAB_EINVAL, "masked_attention: page_size=%d must be 8, 16, 32, 64 or 128", a->page_size);
  if (static_cast<int64_t>(a->bt_stride) * a->page_size > (1ll << 30))
    return fail(MONOFAB_EINVAL, "masked_attention: block tables of %lld keys, at most 2^30", static_cast<long long>(a->bt_stride) * a->page_size);
  if (!(a->scale > 0.f) || std::isinf(a->scale)) return fail(MONOFAB_EINVAL, "masked_attention: the scale must be positive and finite");
  if (a->tree ? a->words < 1 : a->window < 1 || a->sinks < 0)
    return fail(MONOFAB_EINVAL, "masked_attention: window=%d and sinks=%d, or words=%d of a tree", a->window, a->sinks, a->words);
  if (a->tokens == 0 || a->requests == 0) return MONOFAB_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->block_table || !a->q_start || !a->kv_len || !a->ws)
    return fail(MONOFAB_EINVAL, "masked_attention: NULL argument");
  const uintptr_t at16 = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache) |
                         reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->ws);
  if ((at16 & 15) || ((a->q_row | a->q_head | a->out_row | a->out_head) & 7) || a->q_row < 8 || a->q_head < 8)
    return fail(MONOFAB_EINVAL, "masked_attention: rows and heads of q and out, the caches and the workspace must start at multiples of 16 bytes");
  if (a->ws_bytes < 1) return fail(MONOFAB_EINVAL, "masked_attention: an empty workspace");
  int sms = 0;
  if (int r = sm_count(&sms)) return r;
  const Grid g = grid_of(D, sms);
  if (a->ws_bytes < static_cast<int64_t>(g.o_bytes + g.ml_bytes + g.meta_bytes))
    return fail(MONOFAB_EINVAL, "masked_attention: a workspace of %lld bytes is smaller than monofab_masked_attention_ws_bytes says", static_cast<long long>(a->ws_bytes));
  Params p{};
  p.per_stream = kTile / group;
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->hq), static_cast<uint64_t>(a->tokens)};
    const uint64_t strides[2] = {2 * static_cast<uint64_t>(a->q_head), 2 * static_cast<uint64_t>(a->q_row)};
    uint32_t box[3] = {64, static_cast<uint32_t>(group), static_cast<uint32_t>(p.per_stream)};
    if (int r = encode_map(&p.q_map, 0, a->q, 3, dims, strides, box, 128)) return r;
    box[2] = 1;
    if (int r = encode_map(&p.q_one_map, 0, a->q, 3, dims, strides, box, 128)) return r;
  }
  for (int i = 0; i < 2; ++i) {   // a page's keys of one head, both halves of the head dimension, in groups of eight keys
    const uint64_t halves = D / 64, row = static_cast<uint64_t>(a->hkv) * D * 2;
    const uint64_t dims[5] = {64, 8, halves * a->hkv, static_cast<uint64_t>(a->page_size / 8), static_cast<uint64_t>(a->n_pages)};
    const uint64_t strides[4] = {row, 128, 8 * row, static_cast<uint64_t>(a->page_size) * row};
    const uint32_t box[5] = {64, 8, static_cast<uint32_t>(halves), static_cast<uint32_t>(a->page_size / 8), 1};
    if (int r = encode_map(i ? &p.v_map : &p.k_map, 0, i ? a->v_cache : a->k_cache, 5, dims, strides, box, 128)) return r;
  }
  p.block_table = a->block_table;
  p.q_start = a->q_start;
  p.kv_len = a->kv_len;
  p.tree = a->tree;
  p.out = a->out;
  p.status = a->status;
  p.ws_o = static_cast<float*>(a->ws);
  p.ws_ml = reinterpret_cast<float2*>(static_cast<char*>(a->ws) + g.o_bytes);
  p.ws_meta = reinterpret_cast<int4*>(static_cast<char*>(a->ws) + g.o_bytes + g.ml_bytes);
  p.out_row = a->out_row;
  p.out_head = a->out_head;
  p.tokens = a->tokens;
  p.requests = a->requests;
  p.hkv = a->hkv;
  p.group = group;
  p.page = a->page_size;
  p.bt_stride = a->bt_stride;
  p.words = a->words;
  p.window = a->window;
  p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Batches of single tokens and the like (by the mean of their rows: what the host knows) take the kernel that also has a form for items
  // of few rows. 128 single tokens over 843 MB, long runs: 153 us, without the form 177 (at the card's power limit: 128 rows of products
  // for eight that are there); but its code alone, unused, makes prompts 114 -> 121. The mean is a rough rule: 127 single tokens beside a
  // portion of 512 rows (1.14 GB) take 245 us without the form, 230 with it. Head dimension 64 has no such form: 128 single tokens
  // over 571 MB take 175 us, 3.3 TB/s.
  const bool few = static_cast<int64_t>(a->tokens) * group <= static_cast<int64_t>(a->requests) * kFewRows;
  auto go = [&](auto e) {
    using E = decltype(e);
    return D == 64 ? launch<E, 64>(p, g, st) : few ? launch<E, 128, true>(p, g, st) : launch<E, 128>(p, g, st);
  };
  MF_CUDA(a->fp16 ? go(__half()) : go(__nv_bfloat16()));
  return MONOFAB_OK;
}

extern "C" int monofab_masked_attention_status(int32_t* out) {
  if (!out) return fail(MONOFAB_EINVAL, "masked_attention_status: NULL argument");
  const int zero = 0;
  MF_CUDA(cudaDeviceSynchronize());
  MF_CUDA(cudaMemcpyFromSymbol(out, g_masked_attention_status, sizeof(int)));
  if (*out) MF_CUDA(cudaMemcpyToSymbol(g_masked_attention_status, &zero, sizeof(int)));
  return MONOFAB_OK;
}
