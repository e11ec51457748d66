"""Paged-KV GQA attention for mixed prefill / decode batches (head_dim 128).

Host mirror of the reference's attention stage (monoserve/runtime/lane.py:423-520
builds, per request, prefill tiles per (q head, 128-row block, KV chunk) and decode
tiles per (KV head, chunk); `req_info` rows are {first query row, position of that
row, query rows, keys visible}).  Here a work item is (request, KV head, block of
query tokens, key range); long items are split over key ranges for load balance and
merged by a second small kernel.
"""
import ctypes
import functools
import math
import struct

import torch

from monoserve_b200 import _C

SCALE_LOG2 = math.log2(math.e) / math.sqrt(128.0)   # monoserve/runtime/lane.py:238


SM_COUNT = 148          # CTAs that run at once: one work item per SM
MIN_PART_TILES = 4      # a part shorter than four 128-key tiles is not worth a merge


def plan_items(req_info, hq, hkv, sms=SM_COUNT, part_tiles=None):
    """The work list of one attention call, as the reference's lane builds prefill
    tiles per (block, KV chunk) and decode tiles per (KV head, chunk)
    (monoserve/runtime/lane.py:423-520), with the chunk length chosen for load balance.

    req_info: rows of (first query row, position of that row, query rows, keys visible),
    one per request (row index = block-table row).  Returns (items int32 [n, 12],
    merge int32 [m, 8], workspace rows).  Items are ordered longest first, so that the
    SMs that free up last take the shortest ones.
    """
    group = hq // hkv
    per_block = 128 // group
    blocks = []
    for req, (row0, pos0, rows, kv_len) in enumerate(req_info):
        for b in range(0, rows, per_block):
            n = min(per_block, rows - b)
            kv_end = min(kv_len, pos0 + b + n)
            blocks.append((req, row0 + b, n, pos0 + b, kv_len, -(-max(kv_end, 0) // 128)))
    total = sum(t for *_, t in blocks) * hkv
    if part_tiles is None:
        # aim at two rounds of equally long parts over the SMs
        part_tiles = max(MIN_PART_TILES, -(-total // (2 * sms)))
    items, merge, ws_rows = [], [], 0
    for req, row0, n, pos0, kv_len, tiles in blocks:
        parts = max(1, -(-tiles // part_tiles)) if tiles >= 2 * MIN_PART_TILES else 1
        per_part = -(-tiles // parts)
        parts = -(-tiles // per_part) if tiles else 1
        for h in range(hkv):
            if parts == 1:
                items.append((tiles, [req, h, row0, n, pos0, kv_len, 0, 0, -1, 0, 0, 0]))
                continue
            stride = n * group
            merge.append([row0, n, h, ws_rows, parts, stride, 0, 0])
            for part in range(parts):
                t0, t1 = part * per_part, min(tiles, (part + 1) * per_part)
                items.append((t1 - t0, [req, h, row0, n, pos0, kv_len, t0 * 128, t1 * 128, ws_rows, 0, 0, 0]))
                ws_rows += stride
    items.sort(key=lambda it: -it[0])
    return (torch.tensor([it for _, it in items], dtype=torch.int32).reshape(-1, 12),
            torch.tensor(merge, dtype=torch.int32).reshape(-1, 8), ws_rows)


def build_items(req_info, hq, hkv):
    """The unsplit work list: one item per (request, block of query tokens, KV head)."""
    return plan_items(req_info, hq, hkv, part_tiles=1 << 30)[0]


class AttentionPlan:
    """The work list of one batch shape, planned once and kept on the device with its
    split workspace; `run` only launches.  (The reference's lane rebuilds its attention
    tiles per step on the host too: monoserve/runtime/lane.py:423-520.)"""

    def __init__(self, req_info, hq, hkv, split=True, part_tiles=None, device="cuda"):
        self.hq, self.hkv = hq, hkv
        items, merge, self.ws_rows = plan_items(req_info, hq, hkv, part_tiles=part_tiles if split else 1 << 30)
        self.items, self.merge = items.to(device), merge.to(device)
        self.ws = torch.empty(self.ws_rows * 130, dtype=torch.float32, device=device) if self.ws_rows else None
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def run(self, q, k_cache, v_cache, block_table, out=None, stream=None, check=True):
        T, hq, D = q.shape
        n_pages, page_size, hkv, _ = k_cache.shape
        assert D == 128 and (hq, hkv) == (self.hq, self.hkv)
        assert q.dtype == torch.bfloat16 and q.is_cuda and q.is_contiguous()
        assert k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.shape == v_cache.shape
        assert block_table.dtype == torch.int32 and block_table.is_cuda and block_table.is_contiguous()
        if out is None:
            out = torch.empty_like(q)
        st = stream if stream is not None else torch.cuda.current_stream()
        _C.check(_C.lib.monofab_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                          block_table.data_ptr(), block_table.shape[1], self.items.data_ptr(),
                                          self.items.shape[0], T, hq, hkv, page_size, n_pages, SCALE_LOG2,
                                          self.ws.data_ptr() if self.ws is not None else None, self.ws_rows,
                                          self.merge.data_ptr() if self.merge.shape[0] else None, self.merge.shape[0],
                                          self.status.data_ptr(), ctypes.c_void_p(st.cuda_stream)))
        if check and int(self.status.item()):
            raise RuntimeError(f"monofab: attention kernel reported status {int(self.status.item())}")
        return out


def paged_attention(q, k_cache, v_cache, block_table, req_info, out=None, stream=None, split=True, part_tiles=None):
    """q bf16 [T, hq, 128]; k_cache / v_cache bf16 [pages, page_size, hkv, 128];
    block_table int32 [requests, stride]; req_info as in plan_items.  split=False keeps
    every (request, block, KV head) in one work item.  Returns bf16 [T, hq, 128]."""
    plan = AttentionPlan(req_info, q.shape[1], k_cache.shape[2], split=split, part_tiles=part_tiles)
    return plan.run(q, k_cache, v_cache, block_table, out=out, stream=stream)


K_ATTN_PREFILL, K_ATTN_DECODE, K_ATTN_MERGE = 33, 34, 35


def fabric_maps(fab, q, k_cache, v_cache):
    """Tensor maps of q and the paged caches in a fabric's table: (q_map, q_map_small or 0, k_map, v_map)."""
    T, hq, _ = q.shape
    n_pages, page, hkv, _ = k_cache.shape
    group = hq // hkv
    dims, strides = [128, hq, T], [256, hq * 256]
    q_map = fab.tensor_map(q.data_ptr(), dims, strides, [64, group, 128 // group])
    q_small = fab.tensor_map(q.data_ptr(), dims, strides, [64, group, 32 // group]) if 32 % group == 0 else 0
    # one box = one page's keys of one KV head, both halves of the head dimension, in groups of eight keys
    row = hkv * 256
    kd, ks, kb = [64, 8, 2 * hkv, page // 8, n_pages], [row, 128, 8 * row, page * row], [64, 8, 2, page // 8, 1]
    return q_map, q_small, fab.tensor_map(k_cache.data_ptr(), kd, ks, kb), fab.tensor_map(v_cache.data_ptr(), kd, ks, kb)


def fabric_tiles(items, merge, args_ptr, kind=K_ATTN_PREFILL):
    """The work list of plan_items as fabric tiles: (attention item tiles, merge tiles), each a
    uint64 [n, 8] array.  Tile fields: see make_attn_work / tile_attn_merge in csrc/fabric_seq_tiles.cuh."""
    import numpy as np
    from monoserve_b200.fabric import tile_array
    it = items.numpy().astype(np.int64).reshape(-1, 12)
    tiles = tile_array(kind, i0=it[:, 2], i1=it[:, 3] | (it[:, 1] << 16), i2=it[:, 6], i3=np.maximum(it[:, 7], 0),
                       a0=args_ptr, a1=it[:, 0] | ((it[:, 8] + 1) << 32), a2=it[:, 4] | (it[:, 5] << 32))
    mg = merge.numpy().astype(np.int64).reshape(-1, 8)
    merges = tile_array(K_ATTN_MERGE, i0=mg[:, 0], i1=mg[:, 1] | (mg[:, 2] << 16), i2=mg[:, 3],
                        i3=mg[:, 4] | (mg[:, 5] << 16), a0=args_ptr)
    return tiles, merges


# ------------------------------------------------------------------ windows and sinks, trees of drafted tokens

_HALVES = (torch.bfloat16, torch.float16)
_masked_args = struct.Struct("10Q5q12if4x")   # monofab_masked_attention_args of include/monofab.h


# The current stream's handle of a device, without the object that torch.cuda.current_stream makes of it (4 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _no(what):
    raise ValueError("monofab: " + what)


def _refuse(ok, what):
    ok or _no(what)


def _stream_of(index, stream):
    stream is None or stream.device.index == index or _no("the stream belongs to another device than the tensors")
    return stream


def _apart(row, rows, head, heads, D):
    """Whether `rows` by `heads` runs of D values, at these strides, have no value in common."""
    (near, n), (far, m) = sorted([(row, rows), (head, heads)])
    if near >= D and far >= (n - 1) * near + D:   # one inside the other, as nearly all are
        return True
    # else two runs lie a * near - b * far apart, a < n, b < m: the nearest a of each b, those of b = 0 one step
    return (n == 1 or near >= D) and all(abs(min(n - 1, max(0, a)) * near - b * far) >= D for b in range(1, m) for a in (b * far // near, b * far // near + 1))


@functools.lru_cache(maxsize=None)
def _masked_ws_bytes(device_index, head_dim):
    n = _C.lib.monofab_masked_attention_ws_bytes(head_dim)
    if n < 0:
        _C.check(n)
    return n


def _masked_attention(q, k_cache, v_cache, block_table, q_start, kv_len, window, sinks, tree, scale, out, stream, status):
    shape, cache = q.shape, k_cache.shape
    len(shape) == 3 and len(cache) == 4 and v_cache.shape == cache or \
        _no("q is [tokens, hq, head_dim], the caches are [pages, page_size, hkv, head_dim]")
    T, hq, D = shape
    n_pages, page, hkv, Dk = cache
    D == Dk and D in (64, 128) or _no(f"head_dim must be 64 or 128 in q and the caches, not {D} and {Dk}")
    dtype = q.dtype
    dtype in _HALVES and k_cache.dtype is dtype and v_cache.dtype is dtype or _no("q and the caches are bf16 or fp16, all the same")
    hkv >= 1 and hq >= 1 and hq % hkv == 0 and hq // hkv <= 128 or _no(f"hq={hq} must be a multiple of hkv={hkv}, at most 128 times")
    page in (8, 16, 32, 64, 128) or _no(f"page_size={page} must be 8, 16, 32, 64 or 128")
    k_cache.is_contiguous() and v_cache.is_contiguous() or _no("the caches must be contiguous")
    tables = block_table.shape
    len(tables) == 2 and q_start.dim() == 1 and kv_len.dim() == 1 or _no("block_table is [requests, pages], q_start and kv_len are vectors")
    R = kv_len.shape[0]
    tables[0] == R and q_start.shape[0] == R + 1 or _no(f"{R} requests: block_table needs as many rows, q_start one more entry")
    small = (block_table, q_start, kv_len) if tree is None else (block_table, q_start, kv_len, tree)
    index, here = q.get_device(), True
    for t in small:
        t.dtype is torch.int32 and t.is_contiguous() or _no("block_table, q_start, kv_len and tree are contiguous int32")
        here = here and t.get_device() == index
    if tree is None:
        1 <= window < 1 << 31 and 0 <= sinks < 1 << 31 or _no(f"window={window} must be positive, sinks={sinks} not negative")
        words = tree_at = 0
    else:
        window = sinks = 0
        tree.dim() == 2 and tree.shape[0] == T and (tree.shape[1] >= 1 or T == 0) or _no("tree is [tokens, words]")
        words, tree_at = tree.shape[1], tree.data_ptr()
    scale = D ** -0.5 if scale is None else float(scale)
    0.0 < scale < math.inf or _no("the scale must be positive and finite")
    out is None or (out.shape == shape and out.dtype == dtype) or _no("out has the shape and type of q")

    out_strides = hq * D, D
    for t in (q,) if out is None else (out, q):   # strides of rows and heads; that of a single one may be anything
        row, head, last = t.stride()
        if T <= 1 or hq == 1:
            row, head = row if T > 1 else hq * D, head if hq > 1 else D
        T == 0 or (last == 1 and (row | head) % 8 == 0 and row > 0 and head > 0 and t.data_ptr() % 16 == 0) or \
            _no("the heads of q and out must be contiguous and start at multiples of 16 bytes")
        if t is out:
            T == 0 or _apart(row, T, head, hq, D) or _no("rows and heads of out must not overlap")
            out_strides = row, head
    index >= 0 and here and k_cache.get_device() == index and v_cache.get_device() == index and \
        (out is None or out.get_device() == index) and (status is None or status.get_device() == index) or _no("all tensors must be on one CUDA device")
    status is None or (status.dtype == torch.int32 and status.numel() >= 1) or _no("status is int32")
    if stream is not None or torch.cuda.current_device() != index:
        with torch.cuda.device(index), torch.cuda.stream(_stream_of(index, stream)):   # what is allocated in the call belongs to its stream
            return _masked_attention(q, k_cache, v_cache, block_table, q_start, kv_len, window, sinks, tree, scale, out, None, status)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    if T == 0 or R == 0:
        return out
    ws_bytes = _masked_ws_bytes(index, D)
    ws = block_table.new_empty(ws_bytes >> 2)
    args = _masked_args.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), q_start.data_ptr(),
                             kv_len.data_ptr(), tree_at, ws.data_ptr(), 0 if status is None else status.data_ptr(), row, head, *out_strides, ws_bytes,
                             T, R, hq, hkv, D, page, n_pages, tables[1], words, window, sinks, dtype is torch.float16, scale)
    rc = _C.lib.monofab_masked_attention(args, _raw_stream(index))
    if rc:
        _C.check(rc)
    return out


def sliding_attention(q, k_cache, v_cache, block_table, q_start, kv_len, window, sinks=0, scale=None, out=None, stream=None, status=None):
    """Attention over a paged cache within a window, with the first `sinks` keys visible to all: a row at position p sees
    key j if j <= p and (j > p - window or j < sinks).  Prompts, portions of prompts and single tokens in one ragged batch.

    q [T, hq, D], D 64 or 128, bf16 or fp16, rows and heads at any stride of 16 bytes; k_cache / v_cache
    [pages, page_size, hkv, D]; block_table int32 [requests, stride]; q_start int32 [requests + 1]: request r's rows are
    q_start[r] .. q_start[r + 1] - 1; kv_len int32 [requests]: its keys, those of its rows the last of them.  The lengths are read
    on the device: a call captured in a CUDA graph can be replayed with others.  Returns [T, hq, D] (`out`, which may be q
    itself, or else shares no memory with it): rows that see no key are zeros, rows of no request keep what they hold (are undefined in a new tensor).
    A bounded wait that ran out is reported in `status` (int32 on the device), or to attention_status().  Values that some row
    of a request sees must be finite; what none sees may hold anything.  A score of plus infinity or no number makes the rows
    that see it NaN; minus infinity has weight zero, and rows whose scores are all that are zeros.  Scores, sums and outputs are in
    32 bits; a weight is rounded once, to the type of V, for its product.  Scores may be 1e7 in magnitude (bf16: 5e8).  At most 16384 requests."""
    return _masked_attention(q, k_cache, v_cache, block_table, q_start, kv_len, int(window), int(sinks), None, scale, out, stream, status)


def tree_attention(q, k_cache, v_cache, block_table, q_start, kv_len, tree, scale=None, out=None, stream=None, status=None):
    """Attention of drafted token trees over a paged cache: a request's rows are its drafted tokens, whose keys are the last
    ones of its kv_len.  A row sees all keys in front of them (the past), and of drafted token d the key if bit d % 32 of
    tree[row, d // 32] is set.  tree: int32 [T, words] (tree_bits makes it from parents); drafted tokens from 32 * words on
    are seen by none.  Everything else as in sliding_attention."""
    return _masked_attention(q, k_cache, v_cache, block_table, q_start, kv_len, 0, 0, tree, scale, out, stream, status)


def tree_bits(parents, words=None):
    """The words of one request's tree for tree_attention, int32 [drafts, words] on the host: parents[i] is the drafted token that
    token i follows, an earlier one, or -1 where it follows the past.  A token sees itself and what it follows."""
    seen = []
    for i, parent in enumerate(parents):
        _refuse(-1 <= parent < i, f"token {i} cannot follow token {parent}")
        seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
    need = max(1, -(-len(seen) // 32))
    words = need if words is None else words
    _refuse(words >= need, f"{len(seen)} drafted tokens need {need} words")
    signed = [[(b >> 32 * w & 0xffffffff) - (1 << 32 if b >> 32 * w + 31 & 1 else 0) for w in range(words)] for b in seen]
    return torch.tensor(signed, dtype=torch.int32).reshape(len(seen), words)


def attention_status(device=None):
    """The status bits (include/monofab.h) that sliding_attention and tree_attention calls without a status of their own have left
    on the device since the last time it was asked.  Waits for the device."""
    out = ctypes.c_int32()
    with torch.cuda.device(device):
        _C.check(_C.lib.monofab_masked_attention_status(ctypes.byref(out)))
    return out.value
