"""Operators on a paged KV cache as launches on a stream: the append of new rows with the norms and the rotation in the
same pass, pages shared by sequences that fork, pages copied and accepted drafts' rows moved in all layers at once.

The caches are those of the attention (monoserve_b200/attention.py): [pages, page_size, hkv, head_dim], K and V apart, a
tensor per layer; page 0 is the sink that unused block-table entries point at (monoserve_b200/engine.py:PagePool).  A
slot is page * page_size + row in the page.  Like every launch, these wait for a resident fabric to stop.
"""
import struct

import torch

from monoserve_b200 import _C
from monoserve_b200.attention import _HALVES, _no, _raw_stream, _refuse, _stream_of
from monoserve_b200.engine import PagePool


_rope_args = struct.Struct("9Q3q8if4x")   # monofab_qk_rope_args of include/monofab.h


def qk_rope(qkv, positions, slots, k_cache, v_cache, cos_sin, hq, q_norm=None, k_norm=None, eps=1e-6, interleaved=False, q_out=None, stream=None):
    """q and k heads of a projection normed and turned, k and v appended to the caches, q returned.

    qkv [T, (hq + 2 hkv) D], bf16 or fp16, rows at any stride of 8 bytes: hq q heads, then hkv k heads, then hkv v heads;
    k_cache / v_cache [pages, page_size, hkv, D], D 64, 128 or 256; positions, slots int32 [T]; cos_sin fp32
    [max_pos, rot / 2, 2] (lane_base.rope_table), rot a multiple of 8 up to D; q_norm / k_norm [D] in qkv's type, or None for no
    norm.  A head x becomes x * rsqrt(mean(x^2) + eps) * norm, and of its first rot dims the pairs (d, d + rot / 2), or
    (2 d, 2 d + 1) if `interleaved`, are turned by the row of the table of its position (outside the table: the nearest
    row).  32-bit arithmetic, one rounding.  Slots outside the cache store nothing: -1 for padding.  q_out [T, hq, D] may be the q
    heads of qkv themselves (qkv.view(T, -1, D)[:, :hq])."""
    cache, dtype, index = k_cache.shape, qkv.dtype, qkv.get_device()
    qkv.dim() == 2 and len(cache) == 4 and v_cache.shape == cache or _no("qkv is [T, heads * D], the caches are [pages, page_size, hkv, D]")
    T, columns = qkv.shape
    n_pages, page, hkv, D = cache
    D in (64, 128, 256) or _no(f"head_dim must be 64, 128 or 256, not {D}")
    hq >= 1 and columns == (hq + 2 * hkv) * D or _no(f"qkv has {columns} columns, not those of {hq} + 2 * {hkv} heads of {D}")
    dtype in _HALVES and k_cache.dtype is dtype and v_cache.dtype is dtype or _no("qkv and the caches are bf16 or fp16, all the same")
    k_cache.is_contiguous() and v_cache.is_contiguous() or _no("the caches must be contiguous")
    n_pages * page < 1 << 31 or _no("the caches have more slots than int32 can name")
    for t in (positions, slots):
        t.shape == (T,) and t.dtype == torch.int32 and t.is_contiguous() or _no("positions and slots are int32 [T]")
    table = cos_sin.shape
    len(table) == 3 and table[2] == 2 and cos_sin.dtype == torch.float32 and cos_sin.is_contiguous() or _no("cos_sin is fp32 [max_pos, rot / 2, 2]")
    rot = 2 * table[1]
    table[0] >= 1 and rot % 8 == 0 and rot <= D or _no(f"rot={rot} must be a multiple of 8 up to {D}")
    norms = [w for w in (q_norm, k_norm) if w is not None]
    for w in norms:
        w.shape == (D,) and w.dtype == dtype and w.is_contiguous() or _no("q_norm and k_norm are [D] in the type of qkv")
    eps >= 0 or _no("eps must not be negative")
    ld, step = qkv.stride()
    T == 0 or (step == 1 and ld % 4 == 0 and ld >= columns * (T > 1)) or _no("rows of qkv must be contiguous and start at multiples of 8 bytes")
    tensors = [k_cache, v_cache, positions, slots, cos_sin, *norms]
    if q_out is not None:
        row, head, last = q_out.stride()
        q_out.shape == (T, hq, D) and q_out.dtype == dtype and last == 1 and (hq == 1 or head == D) and row % 4 == 0 and \
            (T <= 1 or row >= hq * D) or _no("q_out is [T, hq, D] with contiguous rows that start at multiples of 8 bytes")
        tensors.append(q_out)
    for t in tensors:
        t.get_device() == index and index >= 0 or _no("all tensors must be on one CUDA device")
    if stream is not None or torch.cuda.current_device() != index:
        with torch.cuda.device(index), torch.cuda.stream(_stream_of(index, stream)):   # what is allocated in the call belongs to its stream
            return qk_rope(qkv, positions, slots, k_cache, v_cache, cos_sin, hq, q_norm, k_norm, eps, interleaved, q_out)
    if q_out is None:
        q_out = qkv.new_empty((T, hq, D))
        row = hq * D
    args = _rope_args.pack(qkv.data_ptr(), positions.data_ptr(), slots.data_ptr(), cos_sin.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(),
                           0 if k_norm is None else k_norm.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ld, row,
                           n_pages * page, T, hq, hkv, D, rot, table[0], bool(interleaved), dtype is torch.float16, eps)
    rc = _C.lib.monofab_qk_rope(args, _raw_stream(index))
    if rc:
        _C.check(rc)
    return q_out


class SharedPages(PagePool):
    """A page pool whose pages several sequences can hold: a page is free again when as many have given it as had it."""

    def __init__(self, n_pages):
        super().__init__(n_pages)
        self.n_pages = n_pages
        self.holders = [0] * n_pages

    def take(self, n):
        pages = super().take(n)
        for p in pages:
            self.holders[p] = 1
        return pages

    def share(self, pages):
        """Another sequence holds these pages, too."""
        pages = list(pages)
        self._held(pages)
        for p in pages:
            self.holders[p] += 1
        return pages

    def _held(self, pages):
        _refuse(all(0 < p < self.n_pages and self.holders[p] > 0 for p in pages), "only pages that a sequence holds can be shared")

    def give(self, pages):
        """A sequence lets go of these pages.  Nothing changes where one of them is not held."""
        pages = list(pages)   # gone through twice
        left = {}
        for p in pages:
            _refuse(0 < p < self.n_pages and left.setdefault(p, self.holders[p]) > 0, f"page {p} is held by no sequence")
            left[p] -= 1
        for p, n in left.items():
            self.holders[p] = n
        super().give([p for p in dict.fromkeys(pages) if left[p] == 0])

    def fork(self, pages, length, page_size):
        """The pages of a new sequence that starts as the first `length` tokens of one with these pages, and the copies
        [(from, to)] to make for it: it shares the full pages, and gets its own copy of the one that it will go on filling."""
        full, rest = divmod(length, page_size)
        _refuse(0 <= length <= len(pages) * page_size, f"{length} tokens in {len(pages)} pages of {page_size}")
        self._held(pages[:full + (rest > 0)])   # before a page is taken
        own = self.take(1) if rest else []
        return self.share(pages[:full]) + own, [(pages[full], p) for p in own]

    def compact(self, sequences):
        """Moves held pages to the lowest numbers.  sequences: lists of pages, all that are held; their entries are
        replaced.  Returns the copies [(from, to)] to make before anybody reads the new pages."""
        seen = [0] * self.n_pages
        sequences = list(sequences)   # gone through twice
        for pages in sequences:
            _refuse(hasattr(pages, "__setitem__"), "compact replaces the entries of the sequences' lists")
            for p in pages:
                _refuse(0 < p < self.n_pages, f"page {p} is no page of the pool")
                seen[p] += 1
        _refuse(seen == self.holders, "compact needs the pages of every sequence that holds some")
        held = [p for p in range(1, self.n_pages) if self.holders[p]]
        holes = [p for p in range(1, len(held) + 1) if not self.holders[p]]
        moves = dict(zip([p for p in held if p > len(held)], holes))
        for pages in sequences:
            pages[:] = [moves.get(p, p) for p in pages]
        for a, b in moves.items():
            self.holders[b], self.holders[a] = self.holders[a], 0
        self.free = list(range(self.n_pages - 1, len(held), -1))
        return list(moves.items())


class CachePages:
    """The cache tensors of all layers as one object whose pages and rows are moved together, one launch for all of them.

    pages = CachePages(kv.k + kv.v)      # [pages, page_size, hkv, D] each, kept alive and in place by the caller
    pages.copy(src, dst); pages.accept(block_table, base, path, count); pages.check()
    """

    def __init__(self, tensors):
        tensors = list(tensors)
        _refuse(tensors and all(t.dim() == 4 for t in tensors), "cache tensors are [pages, page_size, hkv, D]")
        t0 = tensors[0]
        _refuse(all(t.shape == t0.shape and t.dtype == t0.dtype and t.device == t0.device and t.is_contiguous() for t in tensors),
                "cache tensors must be contiguous and have one shape, type and device")
        self.n_pages, self.page_size = t0.shape[:2]
        self.row_bytes = t0.shape[2] * t0.shape[3] * t0.element_size()
        _refuse(self.n_pages >= 1 and self.page_size >= 1 and self.row_bytes >= 16 and self.row_bytes % 16 == 0 and all(t.data_ptr() % 16 == 0 for t in tensors),
                "rows of a cache tensor must be multiples of 16 bytes")
        at, size = sorted(t.data_ptr() for t in tensors), t0.numel() * t0.element_size()
        _refuse(len(tensors) <= 65535 and all(b - a >= size for a, b in zip(at, at[1:])), "at most 65535 cache tensors, each of them once and in memory of its own")
        _refuse(t0.is_cuda, "cache tensors must be on a CUDA device")
        self.tensors, self.device = tensors, t0.device
        self._table = torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64).to(self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._at, self._status_at = self._table.data_ptr(), self.status.data_ptr()
        torch.cuda.current_stream(self.device).synchronize()   # both are there for calls on any stream

    def _indexes(self, name, t, *shape):
        at = t.shape
        t.dtype == torch.int32 and t.is_contiguous() and t.device == self.device and len(at) == len(shape) or \
            _no(f"{name} is int32 on the device of the cache, of shape {list(shape)}")
        for s, n in zip(shape, at):
            s in (-1, n) or _no(f"{name} is int32 on the device of the cache, of shape {list(shape)}")
        return at

    def _elsewhere(self, stream):
        return stream is not None or torch.cuda.current_device() != self.device.index

    def copy(self, src, dst, stream=None):
        """Page dst[i] takes what page src[i] holds, in all tensors.  src, dst: int32 tensors on the device, or host lists.  One page
        may go to many, but a destination may be no other pair's source or destination: lists are refused, of tensors such
        pairs (and pages that do not exist) are left out, which check() tells.  A page and itself: nothing (padding)."""
        if self._elsewhere(stream):
            with torch.cuda.device(self.device), torch.cuda.stream(_stream_of(self.device.index, stream)):
                return self.copy(src, dst)
        if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            src, dst = list(src), list(dst)
            len(src) == len(dst) and all(0 <= p < self.n_pages for p in src + dst) or _no("src and dst are as many page numbers of the cache")
            pairs = [(s, d) for s, d in zip(src, dst) if s != d]
            src, dst = [s for s, _ in pairs], [d for _, d in pairs]
            len(set(dst)) == len(dst) and not set(dst) & set(src) or _no("a destination is another pair's source or destination")
            src, dst = torch.tensor([src, dst], dtype=torch.int32).to(self.device)
        isinstance(src, torch.Tensor) and isinstance(dst, torch.Tensor) or _no("src and dst are both tensors or both lists")
        n, = self._indexes("src", src, -1)
        self._indexes("dst", dst, n)
        n <= 65535 or _no("at most 65535 pages a call")
        rc = _C.lib.monofab_page_copy(self._at, len(self.tensors), src.data_ptr(), dst.data_ptr(), n, self.n_pages, self.page_size * self.row_bytes,
                                      self._status_at, _raw_stream(self.device.index))
        if rc:
            _C.check(rc)

    def accept(self, block_table, base, path, count, stream=None):
        """The rows of accepted drafts move to the places behind their sequence, in all tensors: of request r, row base[r] + path[r, i]
        to row base[r] + i for i < count[r], as they were before the call.  block_table int32 [requests, stride], base and
        count int32 [requests], path int32 [requests, most <= 2048], on the device.  Rows in places that do not exist stay,
        which check() tells.  Requests must not share the pages of these rows."""
        if self._elsewhere(stream):
            with torch.cuda.device(self.device), torch.cuda.stream(_stream_of(self.device.index, stream)):
                return self.accept(block_table, base, path, count)
        R, width = self._indexes("block_table", block_table, -1, -1)
        self._indexes("base", base, R)
        self._indexes("count", count, R)
        _, most = self._indexes("path", path, R, -1)
        most <= 2048 and R <= 65535 and width >= 1 or _no("at most 2048 rows of a path, 65535 requests")
        rc = _C.lib.monofab_accept_rows(self._at, len(self.tensors), block_table.data_ptr(), width, base.data_ptr(), path.data_ptr(), count.data_ptr(), R,
                                        most, self.page_size, self.n_pages, self.row_bytes, self._status_at, _raw_stream(self.device.index))
        if rc:
            _C.check(rc)

    def check(self):
        """Raises if a copy or an accept since the last check left something out, on whatever stream it was called or replayed.
        Waits for the device (and so for a resident fabric to stop)."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self.device)   # the bits of a call on another stream come behind this
            raise RuntimeError(f"monofab: pages or rows were left out, status {bits}")
