// Attention over a paged cache with a window and sinks, or with a tree of drafted tokens behind the past.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "masked_attention.h"
#include "moe_layer.h"

namespace mf {

namespace {

template <class E>
__device__ __forceinline__ float to_float(E x) {
  return static_cast<float>(x);
}

// A warp per (row, query head), keys one after the other.
template <class E, int D>
__global__ void __launch_bounds__(256) masked_attention_kernel(const __grid_constant__ MaskedAttnParams p) {
  chain_release();
  chain_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 8 + threadIdx.x / 32;
  const int head = static_cast<int>(item % p.hq);
  const long long row = item / p.hq;
  if (row >= p.tokens) return;
  int lo = 0, hi = p.requests;   // the last request that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.q_start[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int first = p.q_start[lo], end = p.q_start[lo + 1];
  if (row < first || row >= end) return;
  const int n = end - first, i = static_cast<int>(row) - first;
  const int keys = min(p.kv_len[lo], p.bt_stride * p.page_size), past = p.kv_len[lo] - n, pos = past + i;
  const E* const q = static_cast<const E*>(p.q) + row * p.q_row + head * p.q_head;
  const int kvh = head / (p.hq / p.hkv);
  constexpr int N = D / 32;
  float qv[N], o[N], m = -INFINITY, l = 0.f;
  for (int d = 0; d < N; ++d) qv[d] = to_float(q[lane + 32 * d]) * p.scale, o[d] = 0.f;
  for (int key = 0; key < keys; ++key) {
    bool seen;
    if (p.tree) {
      const int j = key - past;
      seen = j < 0 || (j < 32 * p.words && j < n && (p.tree[row * p.words + j / 32] >> (j % 32) & 1));
    } else {
      seen = key <= pos && (key > pos - static_cast<long long>(p.window) || key < p.sinks);
    }
    if (!seen) continue;
    const long long at = ((static_cast<long long>(p.block_table[static_cast<long long>(lo) * p.bt_stride + key / p.page_size]) * p.page_size + key % p.page_size) * p.hkv + kvh) * D;
    const E *const k = static_cast<const E*>(p.k_cache) + at, *const v = static_cast<const E*>(p.v_cache) + at;
    float s = 0.f;
    for (int d = 0; d < N; ++d) s += qv[d] * to_float(k[lane + 32 * d]);
    for (int bit = 16; bit; bit >>= 1) s += __shfl_xor_sync(0xffffffffu, s, bit);
    const float top = fmaxf(m, s), keep = expf(m - top), w = expf(s - top);
    m = top;
    l = l * keep + w;
    for (int d = 0; d < N; ++d) o[d] = o[d] * keep + w * to_float(v[lane + 32 * d]);
  }
  E* const out = static_cast<E*>(p.out) + row * p.out_row + head * p.out_head;
  for (int d = 0; d < N; ++d) out[lane + 32 * d] = static_cast<E>(l > 0.f ? o[d] / l : 0.f);
}

// Where a call that names no status word leaves its bits.
__device__ int g_masked_attention_status;

}  // namespace

cudaError_t launch_masked_attention(const MaskedAttnParams& p, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    return launch_chained(kernel, dim3(static_cast<unsigned>((static_cast<long long>(p.tokens) * p.hq + 7) / 8)), dim3(256), 0, stream, p);
  };
  if (p.fp16) return p.head_dim == 64 ? go(masked_attention_kernel<__half, 64>) : go(masked_attention_kernel<__half, 128>);
  return p.head_dim == 64 ? go(masked_attention_kernel<__nv_bfloat16, 64>) : go(masked_attention_kernel<__nv_bfloat16, 128>);
}

}  // namespace mf

using namespace mf;

extern "C" size_t monofab_masked_attention_ws_bytes(int tokens, int hq, int hkv, int head_dim) {
  (void)tokens, (void)hq, (void)hkv, (void)head_dim;
  return 16;
}

extern "C" int monofab_masked_attention(const monofab_masked_attention_args* a, void* stream) {
  if (!a) return fail(MONOFAB_EINVAL, "masked_attention: NULL argument");
  if (a->tokens < 0 || a->requests < 0 || a->n_pages < 1 || a->bt_stride < 1)
    return fail(MONOFAB_EINVAL, "masked_attention: tokens=%d, requests=%d, n_pages=%d, bt_stride=%d", a->tokens, a->requests, a->n_pages, a->bt_stride);
  if (a->hkv < 1 || a->hq < a->hkv || a->hq % a->hkv) return fail(MONOFAB_EINVAL, "masked_attention: hq=%d must be a multiple of hkv=%d", a->hq, a->hkv);
  if (a->hq / a->hkv > 128) return fail(MONOFAB_EINVAL, "masked_attention: %d query heads for a KV head, at most 128", a->hq / a->hkv);
  if (a->head_dim != 64 && a->head_dim != 128) return fail(MONOFAB_EINVAL, "masked_attention: head_dim=%d must be 64 or 128", a->head_dim);
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
  if ((at16 & 15) || ((a->q_row | a->q_head | a->out_row | a->out_head) & 7) || a->q_row < 0 || a->q_head < 0)
    return fail(MONOFAB_EINVAL, "masked_attention: rows and heads of q and out, the caches and the workspace must start at multiples of 16 bytes");
  if (a->ws_bytes < static_cast<int64_t>(monofab_masked_attention_ws_bytes(a->tokens, a->hq, a->hkv, a->head_dim)))
    return fail(MONOFAB_EINVAL, "masked_attention: a workspace of %lld bytes is smaller than monofab_masked_attention_ws_bytes says", static_cast<long long>(a->ws_bytes));
  MF_CUDA(launch_masked_attention(*a, static_cast<cudaStream_t>(stream)));
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
