// Operators on a paged KV cache, launched on a stream: the append of new rows (norms of queries and keys for each head
// and the position rotation in the same pass), copies of whole pages in all layers, and the move of accepted drafts'
// rows to the places behind their sequence in all layers.
//
// A cache tensor is [pages][page size][kv heads][head dim], 16-bit values; a slot is page * page size + row in the page.
// All of this is bound by HBM or, for a few rows, by the latency of one launch: every kernel keeps several 16-byte accesses a
// thread in flight and touches each byte of the caches once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "moe_layer.h"

namespace mf {

namespace {

// `each` for every SM of the current device.
cudaError_t resident_blocks(int* blocks, int each) {
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  *blocks = sms * each;
  return e;
}

template <class E>
struct Pack;
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ float2 open(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t close(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pack<__half> {
  static __device__ __forceinline__ float2 open(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t close(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

struct QkRopeParams {
  const uint16_t* qkv;      // [T] rows of (hq + 2 hkv) heads, `ld` values apart
  const int32_t* positions; // [T]
  const int32_t* slots;     // [T]
  const float* cos_sin;     // [max_pos][rot / 2][2]
  const uint16_t *q_norm, *k_norm;   // [D] or null: no norm
  uint16_t* q_out;          // [T] rows of hq heads, `ld_out` values apart
  uint16_t *k_cache, *v_cache;
  long long ld, ld_out, n_slots;
  int T, hq, hkv, rot, max_pos, interleaved;
  float eps;
};

// A lane holds two runs of R dims of a head, `a` and `b`, so that both values of a rotated pair are its own whatever the pairs
// are: of the first rot / 2R lanes, halves: dims R l.. of either half; neighbours: dims 2R l.. and 2R l + R..; both take the R
// (cos, sin) from R l on. The other lanes hold what is not turned, in order. So there is no exchange but the sum of squares. A unit
// is U passes of a warp over the heads of one row (32 / (D / 2R) heads a pass): their loads are issued together, and the row's
// (cos, sin) are read once for all of them.
// Everything is in 32 bits and rounded once, at the store.
// Bound by the loads that are in flight: 8191 rows of 40 heads of 128 (169 MB) take 31.6 us, 5.3 TB/s, with 64 registers and so four
// blocks an SM (72, three blocks: 33.7; eight bytes a lane at a time and rows found by division: 38).
template <int R>
struct Run {   // R values, 2 in a word
  using Vec = std::conditional_t<R == 8, uint4, uint2>;
  uint32_t w[R / 2];
  __device__ __forceinline__ void load(const uint16_t* p) { *reinterpret_cast<Vec*>(w) = *reinterpret_cast<const Vec*>(p); }
  __device__ __forceinline__ void store(uint16_t* p) const { *reinterpret_cast<Vec*>(p) = *reinterpret_cast<const Vec*>(w); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < R / 2; ++i) w[i] = 0;
  }
};
template <class E, int D, int R, int U, bool kNeighbours>
__global__ void __launch_bounds__(256, 4) qk_rope_kernel(const __grid_constant__ QkRopeParams p) {
  constexpr int kLanes = D / (2 * R), kHeads = 32 / kLanes;
  chain_release();
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  const int heads = p.hq + 2 * p.hkv;
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.z + threadIdx.z;   // a warp: (unit, row) = (y, z)
  const int head0 = static_cast<int>(blockIdx.y * blockDim.y + threadIdx.y) * U * kHeads + lane / kLanes;
  chain_wait();
  if (row >= p.T) return;   // the whole warp
  const bool turns = l < p.rot / (2 * R);
  const int da = turns && !kNeighbours ? R * l : 2 * R * l;
  const int db = turns && !kNeighbours ? p.rot / 2 + R * l : 2 * R * l + R;
  const int slot = p.slots[row], position = p.positions[row];   // first: the table waits for it
  const uint16_t* const from = p.qkv + row * p.ld;
  Run<R> a[U], b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int head = head0 + u * kHeads;
    if (head < heads) {
      a[u].load(from + head * D + da);
      b[u].load(from + head * D + db);
    } else {
      a[u].zero();
      b[u].zero();
    }
  }
  float cs[2 * R];   // (cos, sin) of R pairs
#pragma unroll
  for (int i = 0; i < 2 * R; ++i) cs[i] = i & 1 ? 0.f : 1.f;
  if (turns) {
    const int pos = max(0, min(position, p.max_pos - 1));
    const float4* const t = reinterpret_cast<const float4*>(p.cos_sin + (static_cast<long long>(pos) * (p.rot / 2) + R * l) * 2);
#pragma unroll
    for (int i = 0; i < R / 2; ++i) *reinterpret_cast<float4*>(&cs[4 * i]) = t[i];
  }
  const bool stored = slot >= 0 && slot < p.n_slots;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int head = head0 + u * kHeads;
    const bool is_q = head < p.hq, is_k = !is_q && head < p.hq + p.hkv;
    float x[2 * R];
#pragma unroll
    for (int i = 0; i < R / 2; ++i) {
      const float2 ta = Pack<E>::open(a[u].w[i]), tb = Pack<E>::open(b[u].w[i]);
      x[2 * i] = ta.x, x[2 * i + 1] = ta.y, x[R + 2 * i] = tb.x, x[R + 2 * i + 1] = tb.y;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int bit = kLanes / 2; bit >= 1; bit >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, bit);
    if (head >= heads) continue;
    uint16_t* to;
    if (is_q) {
      to = p.q_out + row * p.ld_out + head * D;
    } else {
      if (!stored) continue;
      const int kvh = is_k ? head - p.hq : head - p.hq - p.hkv;
      to = (is_k ? p.k_cache : p.v_cache) + (static_cast<long long>(slot) * p.hkv + kvh) * D;
    }
    if (is_q || is_k) {
      if (const uint16_t* const norm = is_q ? p.q_norm : p.k_norm) {
        const float inv = rsqrtf(ss / D + p.eps);
        Run<R> wa, wb;   // from L1: in registers for q and k heads they would take a third of the warps' places
        wa.load(norm + da);
        wb.load(norm + db);
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          const float2 ta = Pack<E>::open(wa.w[i]), tb = Pack<E>::open(wb.w[i]);
          x[2 * i] *= inv * ta.x, x[2 * i + 1] *= inv * ta.y, x[R + 2 * i] *= inv * tb.x, x[R + 2 * i + 1] *= inv * tb.y;
        }
      }
      if (turns) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const int i0 = kNeighbours ? 2 * j : j, i1 = kNeighbours ? 2 * j + 1 : j + R;
          const float first = x[i0], second = x[i1];
          x[i0] = first * cs[2 * j] - second * cs[2 * j + 1];
          x[i1] = second * cs[2 * j] + first * cs[2 * j + 1];
        }
      }
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        a[u].w[i] = Pack<E>::close(x[2 * i], x[2 * i + 1]);
        b[u].w[i] = Pack<E>::close(x[R + 2 * i], x[R + 2 * i + 1]);
      }
    }
    a[u].store(to + da);
    b[u].store(to + db);
  }
}

template <class E, int D>
cudaError_t launch_qk_rope(const QkRopeParams& p, bool aligned16, cudaStream_t stream) {
  const int heads = p.hq + 2 * p.hkv;
  auto go = [&](auto kernel, int r, int u) {
    const int each = u * (32 / (D / (2 * r)));   // heads of a unit
    const int units = (heads + each - 1) / each, groups = (units + 7) / 8, y = (units + groups - 1) / groups, z = 8 / y;
    return launch_chained(kernel, dim3(static_cast<unsigned>((p.T + z - 1) / z), groups), dim3(32, y, z), 0, stream, p);
  };
  // 16 bytes at a time where the rows and both halves of what is turned start at multiples of them. Two passes a warp (8191 rows of 40
  // heads 31.6 us; one: 36.7), one where that leaves SMs without eight warps (four rows of 20 heads 1.7 us; two: 2.2).
  int warps = 0;
  if (const cudaError_t e = resident_blocks(&warps, 8); e != cudaSuccess) return e;
  constexpr int kHeads = 32 / (D / 16);
  const bool few = static_cast<long long>(p.T) * ((heads + 2 * kHeads - 1) / (2 * kHeads)) < warps;
  auto pick = [&](auto nb) {
    constexpr bool kN = decltype(nb)::value;
    if (!aligned16 || p.rot % 16) return go(qk_rope_kernel<E, D, 4, 2, kN>, 4, 2);
    return few ? go(qk_rope_kernel<E, D, 8, 1, kN>, 8, 1) : go(qk_rope_kernel<E, D, 8, 2, kN>, 8, 2);
  };
  return p.interleaved ? pick(std::true_type()) : pick(std::false_type());
}

// ------------------------------------------------------------------------------------------------- pages and rows

struct PageCopyParams {
  const unsigned long long* tensors;   // [n_tensors] device addresses
  const int32_t *src, *dst;
  int* status;
  int pairs, n_pages;
  long long page_bytes;
};

constexpr int kCopyThreads = 256, kCopyLoads = 4, kCopyBytes = kCopyThreads * kCopyLoads * 16;

// Block (chunk of a page, tensor, pair): 131 pages of 16 KB in 96 tensors take 66 us, 6.2 TB/s. Whether the pair may be copied is looked at first, in every block alike:
// its destination may be no other pair's source or destination, and its source no other pair's destination - copies run side
// by side, and either would make the result depend on their order. A page to itself is nothing to do, and in nobody's way.
// Every block reads both lists for that, which grows with the square of the pairs: 4096 pairs of 16 KB are still at HBM's rate (1946 us,
// 6.6 TB/s), of 16384 the lists take half the time (17.2 ms, 3.0 TB/s), and beside pages of 1 KB those of 4096 do most of the work (0.6 TB/s).
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ PageCopyParams p) {
  chain_release();
  chain_wait();
  const int pair = blockIdx.z;
  const int src = p.src[pair], dst = p.dst[pair];
  bool bad = src < 0 || src >= p.n_pages || dst < 0 || dst >= p.n_pages;
  if (src == dst && !bad) return;
  for (int j = threadIdx.x; j < p.pairs; j += kCopyThreads) {
    if (j == pair) continue;
    const int s = p.src[j], d = p.dst[j];
    bad = bad || (s != d && (s == dst || d == dst || d == src));
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) atomicOr(p.status, kErrBadArgs);
    return;
  }
  const long long at = static_cast<long long>(blockIdx.x) * kCopyBytes + threadIdx.x * 16;
  char* const tensor = reinterpret_cast<char*>(p.tensors[blockIdx.y]);
  const char* const from = tensor + src * p.page_bytes + at;
  char* const to = tensor + dst * p.page_bytes + at;
  uint4 v[kCopyLoads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i)
    if (at + i * (kCopyThreads * 16) < p.page_bytes) v[i] = *reinterpret_cast<const uint4*>(from + i * (kCopyThreads * 16));
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i)
    if (at + i * (kCopyThreads * 16) < p.page_bytes) *reinterpret_cast<uint4*>(to + i * (kCopyThreads * 16)) = v[i];
}

struct AcceptParams {
  const unsigned long long* tensors;
  const int32_t *block_table, *base, *path, *count;
  int* status;
  int n_tensors, requests, most, bt_stride, page, n_pages;
  int lanes;           // 16-byte pieces of a row that a block moves, a power of two
  int pieces;          // of a row
  int per_block;       // tensors of a block
};

constexpr int kAcceptThreads = 256, kAcceptRows = 8;   // rows a thread holds at most

// Block (slice of a row, group of tensors, request): every row that moves is read before the first is written, so a path may lead
// anywhere among the drafts, whatever it overwrites. The slice is as wide as lets the block's threads hold all rows.
// What bounds it is the chain count, path, table, row: it is gone through once for a group of tensors, and the next
// tensor's rows are on their way while the last one's are written. (64 requests, 96 tensors, 4 moved rows of 1 KB each: 15.7 us,
// 3.5 TB/s; a block for each tensor: 42.7. With 38, 63 and 126 registers 6, 4 and 2 blocks of the three forms fit on an SM: these 1280
// blocks of the middle one go through the chain in three rounds.)
template <int kRows>
__global__ void __launch_bounds__(kAcceptThreads) accept_kernel(const __grid_constant__ AcceptParams p) {
  chain_release();
  chain_wait();
  const int r = blockIdx.z;
  const int n = max(0, min(p.count[r], p.most));
  const long long base = p.base[r];
  const int piece = blockIdx.x * p.lanes + threadIdx.x % p.lanes;
  const int row0 = threadIdx.x / p.lanes, step = kAcceptThreads / p.lanes;
  const int32_t* const table = p.block_table + static_cast<long long>(r) * p.bt_stride;
  const long long there = static_cast<long long>(p.bt_stride) * p.page;
  bool bad = false;
  long long from[kRows], to[kRows];   // in a tensor; from < 0: nothing to move
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int row = row0 + i * step;
    from[i] = -1;
    if (row >= n) continue;
    const int taken = p.path[static_cast<long long>(r) * p.most + row];
    const long long src = base + taken, dst = base + row;
    if (taken < 0 || base < 0 || src >= there || dst >= there) {
      bad = true;
      continue;
    }
    const uint32_t a = static_cast<uint32_t>(src), b = static_cast<uint32_t>(dst), page = p.page;
    const int pa = table[a / page], pb = table[b / page];
    if (pa < 0 || pa >= p.n_pages || pb < 0 || pb >= p.n_pages) {
      bad = true;
      continue;
    }
    if (taken == row || piece >= p.pieces) continue;
    from[i] = ((static_cast<long long>(pa) * page + a % page) * p.pieces + piece) * 16;
    to[i] = ((static_cast<long long>(pb) * page + b % page) * p.pieces + piece) * 16;
  }
  if (bad && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(p.status, kErrBadArgs);
  const int t0 = blockIdx.y * p.per_block, t1 = min(t0 + p.per_block, p.n_tensors);
  uint4 v[kRows];
  auto load = [&](int t, uint4(&into)[kRows]) {
    const char* const tensor = reinterpret_cast<const char*>(p.tensors[t]);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (from[i] >= 0) into[i] = *reinterpret_cast<const uint4*>(tensor + from[i]);
  };
  load(t0, v);
  for (int t = t0; t < t1; ++t) {
    uint4 next[kRows];
    if (t + 1 < t1) load(t + 1, next);
    __syncthreads();   // all rows of this tensor have been read
    char* const tensor = reinterpret_cast<char*>(p.tensors[t]);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (from[i] >= 0) *reinterpret_cast<uint4*>(tensor + to[i]) = v[i];
      v[i] = next[i];
    }
  }
}

}  // namespace

}  // namespace mf

using namespace mf;

extern "C" int monofab_qk_rope(const monofab_qk_rope_args* a, void* stream) {
  if (!a) return fail(MONOFAB_EINVAL, "qk_rope: NULL argument");
  const int T = a->T, hq = a->hq, hkv = a->hkv, D = a->head_dim, rot = a->rot;
  if (T < 0) return fail(MONOFAB_EINVAL, "qk_rope: negative T");
  if (D != 64 && D != 128 && D != 256) return fail(MONOFAB_EINVAL, "qk_rope: head_dim=%d must be 64, 128 or 256", D);
  if (hq < 0 || hkv < 0 || hq + hkv < 1 || hq > (1 << 16) || hkv > (1 << 16)) return fail(MONOFAB_EINVAL, "qk_rope: hq=%d, hkv=%d", hq, hkv);
  if (rot < 0 || rot > D || rot % 8) return fail(MONOFAB_EINVAL, "qk_rope: rot=%d must be a multiple of 8 up to head_dim", rot);
  if (T == 0) return MONOFAB_OK;
  if (!a->qkv || !a->positions || !a->slots || (rot && !a->cos_sin) || (hq && !a->q_out) || (hkv && (!a->k_cache || !a->v_cache)))
    return fail(MONOFAB_EINVAL, "qk_rope: NULL argument");
  if (a->max_pos < 1 || a->n_slots < 0) return fail(MONOFAB_EINVAL, "qk_rope: max_pos=%d, n_slots=%lld", a->max_pos, static_cast<long long>(a->n_slots));
  if (!(a->eps >= 0.f)) return fail(MONOFAB_EINVAL, "qk_rope: eps must not be negative");
  const uintptr_t at8 = reinterpret_cast<uintptr_t>(a->qkv) | reinterpret_cast<uintptr_t>(a->q_out) | reinterpret_cast<uintptr_t>(a->k_cache) |
                        reinterpret_cast<uintptr_t>(a->v_cache) | reinterpret_cast<uintptr_t>(a->q_norm) | reinterpret_cast<uintptr_t>(a->k_norm);
  if ((at8 & 7) || (reinterpret_cast<uintptr_t>(a->cos_sin) & 15) || ((a->ld_qkv | a->ld_out) & 3))
    return fail(MONOFAB_EINVAL, "qk_rope: rows must start at multiples of 8 bytes, the table at one of 16");
  QkRopeParams p{};
  p.qkv = static_cast<const uint16_t*>(a->qkv);
  p.positions = a->positions;
  p.slots = a->slots;
  p.cos_sin = a->cos_sin;
  p.q_norm = static_cast<const uint16_t*>(a->q_norm);
  p.k_norm = static_cast<const uint16_t*>(a->k_norm);
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.k_cache = static_cast<uint16_t*>(a->k_cache);
  p.v_cache = static_cast<uint16_t*>(a->v_cache);
  p.ld = a->ld_qkv;
  p.ld_out = a->ld_out;
  p.n_slots = a->n_slots;
  p.T = T;
  p.hq = hq;
  p.hkv = hkv;
  p.rot = rot;
  p.max_pos = a->max_pos;
  p.interleaved = a->interleaved != 0;
  p.eps = a->eps;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = !(at8 & 15) && !((a->ld_qkv | a->ld_out) & 7);
  auto go = [&](auto e) {
    using E = decltype(e);
    return D == 64 ? launch_qk_rope<E, 64>(p, wide, st) : D == 128 ? launch_qk_rope<E, 128>(p, wide, st) : launch_qk_rope<E, 256>(p, wide, st);
  };
  MF_CUDA(a->fp16 ? go(__half()) : go(__nv_bfloat16()));
  return MONOFAB_OK;
}

extern "C" int monofab_page_copy(const uint64_t* tensors, int n_tensors, const int32_t* src, const int32_t* dst, int pairs,
                                 int n_pages, int64_t page_bytes, int32_t* status, void* stream) {
  if (n_tensors < 1 || pairs < 0 || n_pages < 1) return fail(MONOFAB_EINVAL, "page_copy: n_tensors=%d, pairs=%d, n_pages=%d", n_tensors, pairs, n_pages);
  if (page_bytes < 16 || page_bytes % 16) return fail(MONOFAB_EINVAL, "page_copy: page_bytes=%lld must be a multiple of 16", static_cast<long long>(page_bytes));
  if (pairs == 0) return MONOFAB_OK;
  if (!tensors || !src || !dst || !status) return fail(MONOFAB_EINVAL, "page_copy: NULL argument");
  if (pairs > 65535) return fail(MONOFAB_EINVAL, "page_copy: %d pairs, at most 65535 a call", pairs);
  PageCopyParams p{};
  p.tensors = reinterpret_cast<const unsigned long long*>(tensors);
  p.src = src;
  p.dst = dst;
  p.status = status;
  p.pairs = pairs;
  p.n_pages = n_pages;
  p.page_bytes = page_bytes;
  const long long chunks = (page_bytes + kCopyBytes - 1) / kCopyBytes;
  if (chunks > 65535 || n_tensors > 65535) return fail(MONOFAB_EINVAL, "page_copy: pages of %lld bytes in %d tensors", static_cast<long long>(page_bytes), n_tensors);
  MF_CUDA(launch_chained(page_copy_kernel, dim3(static_cast<unsigned>(chunks), n_tensors, pairs),
                         dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), p));
  return MONOFAB_OK;
}

extern "C" int monofab_accept_rows(const uint64_t* tensors, int n_tensors, const int32_t* block_table, int bt_stride,
                                   const int32_t* base, const int32_t* path, const int32_t* count, int requests, int most,
                                   int page_size, int n_pages, int64_t row_bytes, int32_t* status, void* stream) {
  if (n_tensors < 1 || n_tensors > 65535 || requests < 0 || most < 0 || page_size < 1 || n_pages < 1 || bt_stride < 1)
    return fail(MONOFAB_EINVAL, "accept_rows: bad sizes");
  if (row_bytes < 16 || row_bytes % 16 || row_bytes > (1 << 20))
    return fail(MONOFAB_EINVAL, "accept_rows: row_bytes=%lld must be a multiple of 16 up to 2^20", static_cast<long long>(row_bytes));
  if (requests > 65535) return fail(MONOFAB_EINVAL, "accept_rows: %d requests, at most 65535 a call", requests);
  if (most > kAcceptThreads * kAcceptRows) return fail(MONOFAB_EINVAL, "accept_rows: paths of %d rows, at most %d", most, kAcceptThreads * kAcceptRows);
  if (requests == 0 || most == 0) return MONOFAB_OK;
  if (!tensors || !block_table || !base || !path || !count || !status) return fail(MONOFAB_EINVAL, "accept_rows: NULL argument");
  AcceptParams p{};
  p.tensors = reinterpret_cast<const unsigned long long*>(tensors);
  p.block_table = block_table;
  p.base = base;
  p.path = path;
  p.count = count;
  p.status = status;
  p.n_tensors = n_tensors;
  p.requests = requests;
  p.most = most;
  p.bt_stride = bt_stride;
  p.page = page_size;
  p.n_pages = n_pages;
  p.pieces = static_cast<int>(row_bytes / 16);
  p.lanes = 1;
  while (2 * p.lanes <= kAcceptThreads && 2 * p.lanes * most <= kAcceptThreads * kAcceptRows && p.lanes < p.pieces) p.lanes *= 2;
  const int slices = (p.pieces + p.lanes - 1) / p.lanes, rows = (most * p.lanes + kAcceptThreads - 1) / kAcceptThreads;
  // up to 16 tensors a block, as many as leave eight blocks for each SM (not all of them there at once: see the kernel)
  int blocks = 0;
  MF_CUDA(resident_blocks(&blocks, 8));
  const long long all = static_cast<long long>(slices) * n_tensors * requests;
  p.per_block = static_cast<int>(std::max(1ll, std::min(16ll, all / blocks)));
  const dim3 grid(slices, (n_tensors + p.per_block - 1) / p.per_block, requests);
  auto go = [&](auto kernel) { return launch_chained(kernel, grid, dim3(kAcceptThreads), 0, static_cast<cudaStream_t>(stream), p); };
  MF_CUDA(rows <= 2 ? go(accept_kernel<2>) : rows <= 4 ? go(accept_kernel<4>) : go(accept_kernel<kAcceptRows>));
  return MONOFAB_OK;
}
