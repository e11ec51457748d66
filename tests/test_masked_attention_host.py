"""What sliding_attention, tree_attention, qk_rope and the cache's page operations refuse, before any launch, and the
host side of trees and shared pages."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def attention_args(T=4, hq=8, hkv=2, D=128, page=16, R=2, dtype=BF):
    return dict(q=torch.zeros(T, hq, D, dtype=dtype), k_cache=torch.zeros(3, page, hkv, D, dtype=dtype), v_cache=torch.zeros(3, page, hkv, D, dtype=dtype),
                block_table=torch.zeros(R, 2, dtype=torch.int32), q_start=torch.zeros(R + 1, dtype=torch.int32), kv_len=torch.zeros(R, dtype=torch.int32))


@pytest.mark.parametrize("change,what", [
    (dict(D=96), "head_dim"), (dict(D=256), "head_dim"), (dict(hq=9), "multiple of hkv"), (dict(hq=258, hkv=2), "at most 128 times"),
    (dict(page=24), "page_size"), (dict(page=256), "page_size"), (dict(dtype=torch.float32), "bf16 or fp16")])
def test_attention_refuses_shapes(change, what):
    from monoserve_b200.attention import sliding_attention, tree_attention
    a = attention_args(**change)
    with pytest.raises(ValueError, match=what):
        sliding_attention(**a, window=5)
    with pytest.raises(ValueError, match=what):
        tree_attention(**a, tree=torch.zeros(4, 1, dtype=torch.int32))


def test_attention_refuses_arguments():
    from monoserve_b200.attention import sliding_attention, tree_attention

    def refused(what, window=5, fn=sliding_attention, **kw):
        a = attention_args()
        a.update(kw)
        if fn is sliding_attention:
            a["window"] = window
        with pytest.raises(ValueError, match=what):
            fn(**a)

    refused("window", window=0)
    refused("sinks", sinks=-1)
    refused("scale", scale=0.0)
    refused("scale", scale=float("nan"))
    refused("scale", scale=-1.0)
    refused("2 requests", q_start=torch.zeros(2, dtype=torch.int32))
    refused("2 requests", block_table=torch.zeros(3, 2, dtype=torch.int32))
    refused("int32", kv_len=torch.zeros(2, dtype=torch.int64))
    refused("all the same", v_cache=torch.zeros(3, 16, 2, 128, dtype=torch.float16))
    refused("contiguous", k_cache=torch.zeros(3, 16, 2, 256, dtype=BF)[..., ::2])
    refused("caches are", k_cache=torch.zeros(4, 16, 2, 128, dtype=BF))
    refused("shape and type", out=torch.zeros(4, 8, 64, dtype=BF))
    refused("16 bytes", q=torch.zeros(4, 8, 129, dtype=BF)[..., :128])
    refused("16 bytes", q=torch.zeros(4 * 8 * 128 + 1, dtype=BF)[1:].view(4, 8, 128))
    refused("one CUDA device")
    refused("tree is", fn=tree_attention, tree=torch.zeros(3, 1, dtype=torch.int32))
    refused("tree is", fn=tree_attention, tree=torch.zeros(4, 0, dtype=torch.int32))
    refused("int32", fn=tree_attention, tree=torch.zeros(4, 1, dtype=torch.int64))


def test_attention_entry_point_refuses():
    from monoserve_b200 import _C
    z = (ctypes.c_uint8 * 64)()
    at = (ctypes.addressof(z) + 15) & ~15
    good = dict(q=at, k_cache=at, v_cache=at, out=at, block_table=at, q_start=at, kv_len=at, ws=at, q_row=1024, q_head=128, out_row=1024, out_head=128,
                ws_bytes=1 << 40, tokens=1, requests=1, hq=8, hkv=2, head_dim=128, page_size=16, n_pages=1, bt_stride=1, window=1, scale=1.0)

    def refused(what, **kw):
        a = _C.MaskedAttentionArgsC(**{**good, **kw})
        assert _C.lib.monofab_masked_attention(ctypes.byref(a), None) == -1
        assert what in _C.lib.monofab_last_error(), _C.lib.monofab_last_error()

    refused(b"head_dim", head_dim=96)
    refused(b"page_size", page_size=24)
    refused(b"multiple of hkv", hq=7)
    refused(b"at most 128", hq=258, hkv=2)
    refused(b"scale", scale=0.0)
    refused(b"window", window=0)
    refused(b"words", tree=at, words=0)
    refused(b"NULL", q=None)
    refused(b"NULL", ws=None)
    refused(b"16 bytes", q=at + 2)
    refused(b"16 bytes", out_row=1025)
    refused(b"2^30", bt_stride=1 << 28)
    refused(b"workspace", ws_bytes=0)
    refused(b"at most 16384", requests=16385)
    assert _C.lib.monofab_masked_attention(None, None) == -1
    a = _C.MaskedAttentionArgsC(**{**good, "tokens": 0})
    assert _C.lib.monofab_masked_attention(ctypes.byref(a), None) == 0   # nothing to do


def test_tree_bits():
    from monoserve_b200.attention import tree_bits
    assert tree_bits([-1, 0, 0, 2, -1]).tolist() == [[1], [3], [5], [13], [16]]
    long = tree_bits(range(-1, 63))
    assert long.shape == (64, 2) and long[63].tolist() == [-1, -1] and long[31].tolist() == [-1, 0] and long[32].tolist() == [-1, 1]
    assert tree_bits([-1], words=3).tolist() == [[1, 0, 0]] and tree_bits([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError):
            tree_bits(bad)
    with pytest.raises(ValueError):
        tree_bits([-1] * 33, words=1)


def rope_args(T=3, hq=4, hkv=2, D=128, dtype=BF, rot=None):
    return dict(qkv=torch.zeros(T, (hq + 2 * hkv) * D, dtype=dtype), positions=torch.zeros(T, dtype=torch.int32), slots=torch.zeros(T, dtype=torch.int32),
                k_cache=torch.zeros(2, 16, hkv, D, dtype=dtype), v_cache=torch.zeros(2, 16, hkv, D, dtype=dtype),
                cos_sin=torch.zeros(8, (rot or D) // 2, 2), hq=hq)


@pytest.mark.parametrize("change,what", [(dict(D=96), "head_dim"), (dict(dtype=torch.float32), "bf16 or fp16"), (dict(rot=20), "rot"), (dict(rot=136), "rot")])
def test_qk_rope_refuses_shapes(change, what):
    from monoserve_b200.cache import qk_rope
    with pytest.raises(ValueError, match=what):
        qk_rope(**rope_args(**change))


@pytest.mark.parametrize("change,what", [
    (dict(hq=5), "columns"), (dict(slots=torch.zeros(3, dtype=torch.int64)), "int32"), (dict(positions=torch.zeros(2, dtype=torch.int32)), "int32"),
    (dict(q_norm=torch.zeros(64, dtype=BF)), "q_norm"), (dict(k_norm=torch.zeros(128)), "q_norm"), (dict(eps=-1.0), "eps"),
    (dict(qkv=torch.zeros(3, 1026, dtype=BF)[:, 1:1025]), "8 bytes"), (dict(q_out=torch.zeros(3, 4, 256, dtype=BF)[..., ::2]), "q_out"), (dict(), "one CUDA device")])
def test_qk_rope_refuses_arguments(change, what):
    from monoserve_b200.cache import qk_rope
    with pytest.raises(ValueError, match=what):
        qk_rope(**{**rope_args(), **change})


def test_cache_entry_points_refuse():
    from monoserve_b200 import _C
    at = 1 << 20   # never read: the calls are refused first

    def refused(what, rc):
        assert rc == -1 and what in _C.lib.monofab_last_error(), (rc, _C.lib.monofab_last_error())

    lib = _C.lib
    good = dict(qkv=at, positions=at, slots=at, cos_sin=at, q_out=at, k_cache=at, v_cache=at, n_slots=1, T=1, hq=1, hkv=1, head_dim=128, rot=128,
                max_pos=1, eps=1e-6)

    def rope(**kw):
        return lib.monofab_qk_rope(ctypes.byref(_C.QkRopeArgsC(**{**good, **kw})), None)

    refused(b"head_dim", rope(head_dim=96))
    refused(b"rot", rope(rot=12))
    refused(b"rot", rope(rot=136))
    refused(b"NULL", rope(qkv=None))
    refused(b"NULL", rope(v_cache=None))
    refused(b"8 bytes", rope(qkv=at + 2))
    refused(b"8 bytes", rope(ld_out=130))
    refused(b"eps", rope(eps=float("nan")))
    refused(b"max_pos", rope(max_pos=0))
    refused(b"hq", rope(hq=1 << 17))
    refused(b"NULL", lib.monofab_qk_rope(None, None))
    assert rope(T=0) == 0
    refused(b"page_bytes", lib.monofab_page_copy(at, 1, at, at, 1, 1, 24, at, None))
    refused(b"65535", lib.monofab_page_copy(at, 1, at, at, 65536, 1, 32, at, None))
    refused(b"NULL", lib.monofab_page_copy(at, 1, at, None, 1, 1, 32, at, None))
    refused(b"row_bytes", lib.monofab_accept_rows(at, 1, at, 1, at, at, at, 1, 1, 16, 1, 8, at, None))
    refused(b"at most 2048", lib.monofab_accept_rows(at, 1, at, 1, at, at, at, 1, 2049, 16, 1, 16, at, None))
    refused(b"NULL", lib.monofab_accept_rows(at, 1, at, 1, at, at, at, 1, 1, 16, 1, 16, None, None))
    assert lib.monofab_page_copy(at, 1, at, at, 0, 1, 32, at, None) == 0
    assert lib.monofab_accept_rows(at, 1, at, 1, at, at, at, 0, 1, 16, 1, 16, at, None) == 0


def test_packed_arguments_are_the_structs():
    """What the wrappers pack is laid out as the structs of the header."""
    from monoserve_b200 import _C, attention, cache
    for packer, struct in ((attention._masked_args, _C.MaskedAttentionArgsC), (cache._rope_args, _C.QkRopeArgsC)):
        names = [n for n, _ in struct._fields_ if n != "reserved"]
        a = struct.from_buffer_copy(packer.pack(*range(1, len(names) + 1)))
        assert packer.size == ctypes.sizeof(struct)
        assert [getattr(a, n) for n in names] == list(range(1, len(names) + 1))


def test_cache_pages_refuse():
    from monoserve_b200.cache import CachePages
    t = torch.zeros(4, 16, 2, 64, dtype=BF)
    for tensors, what in (([], "are"), ([t, t[:3]], "one shape"), ([t, t.half()], "one shape"), ([t[..., ::2]], "one shape"),
                          ([torch.zeros(4, 16, 1, 4, dtype=BF)], "16 bytes"), ([t, t], "each of them once"), ([t], "CUDA device")):
        with pytest.raises(ValueError, match=what):
            CachePages(tensors)


def test_shared_pages_fork_and_give():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(10)
    a = pool.take(3)                               # 40 tokens in pages of 16
    b, copies = pool.fork(a, 40, 16)
    assert b[:2] == a[:2] and b[2] not in a and copies == [(a[2], b[2])]
    c, none = pool.fork(a, 32, 16)
    assert c == a[:2] and none == [] and pool.available() == 9 - 4
    pool.give(a)
    assert pool.available() == 9 - 3               # the first two are held by b and c
    pool.give(b)
    assert pool.available() == 9 - 2
    with pytest.raises(ValueError):
        pool.give([c[0], c[0]])                    # once too often: nothing changes
    pool.give(c)
    assert sorted(pool.free) == list(range(1, 10)) and not any(pool.holders)
    for bad in ([0], [1], [10], [-1]):
        with pytest.raises(ValueError):
            pool.give(bad)
        with pytest.raises(ValueError):
            pool.share(bad)
    with pytest.raises(MemoryError):
        pool.take(10)
    assert pool.available() == 9
    with pytest.raises(ValueError):
        pool.fork([1], 17, 16)


def test_a_fork_without_room_changes_nothing():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(3)
    a = pool.take(2)
    with pytest.raises(MemoryError):
        pool.fork(a, 20, 16)
    assert pool.holders == [0, 1, 1]


def test_shared_pages_compact():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(20)
    a, b, c = pool.take(4), pool.take(5), pool.take(3)
    d, _ = pool.fork(c, 32, 16)
    pool.give(a)
    b0, c0 = list(b), list(c)
    with pytest.raises(ValueError):
        pool.compact([b, c])                       # d holds pages, too
    moves = dict(pool.compact([b, c, d]))
    assert sorted(set(b + c + d)) == list(range(1, 9))
    assert b == [moves.get(p, p) for p in b0] and c == [moves.get(p, p) for p in c0] and d == c[:2]
    assert not set(moves) & set(moves.values()) and pool.available() == 11
    assert sorted(pool.free) == list(range(9, 20)) and pool.take(1) == [9]


def test_a_fork_of_pages_that_are_not_held_takes_none():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(6)
    a = pool.take(2)
    for pages in ([a[0], 5], [5, a[0]]):
        with pytest.raises(ValueError, match="holds"):
            pool.fork(pages, 20, 16)
    assert pool.available() == 3 and sum(pool.holders) == 2
    assert pool.fork([a[0], 5], 16, 16) == ([a[0]], [])   # the page behind the prefix does not matter


def test_a_stream_of_another_device_is_refused():
    from types import SimpleNamespace
    from monoserve_b200.attention import _stream_of
    stream = SimpleNamespace(device=torch.device("cuda", 1))
    assert _stream_of(1, stream) is stream and _stream_of(0, None) is None
    with pytest.raises(ValueError, match="another device"):
        _stream_of(0, stream)


def test_workspaces_are_for_the_head_dims_that_there_are():
    from monoserve_b200 import _C
    for dim in (-1, 0, 96, 256):
        assert _C.lib.monofab_masked_attention_ws_bytes(dim) == -1 and b"head_dim" in _C.lib.monofab_last_error()


def test_pages_given_by_an_iterator_are_free_again():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(6)
    a = pool.take(3)
    pool.give(p for p in a)
    assert sorted(pool.free) == [1, 2, 3, 4, 5] and not any(pool.holders)


def test_compact_takes_an_iterator_and_refuses_what_it_cannot_replace():
    from monoserve_b200.cache import SharedPages
    pool = SharedPages(9)
    a, b, c = pool.take(3), pool.take(2), pool.take(2)
    pool.give(a)
    with pytest.raises(ValueError, match="lists"):
        pool.compact([b, tuple(c)])
    assert b == [4, 5] and pool.holders == [0, 0, 0, 0, 1, 1, 1, 1, 0]   # nothing has changed
    assert pool.compact(s for s in [b, c]) == [(5, 1), (6, 2), (7, 3)]
    assert b == [4, 1] and c == [2, 3] and pool.holders == [0, 1, 1, 1, 1, 0, 0, 0, 0]


def test_an_out_whose_rows_overlap_is_refused():
    """Where several rows or heads share memory, which of their results stays would be left to chance."""
    from monoserve_b200.attention import _apart, sliding_attention

    def call(row, head, T=4, hq=8, buffer=torch.zeros(1 << 16, dtype=BF)):
        sliding_attention(**{**attention_args(T=T, hq=hq), "out": torch.as_strided(buffer, (T, hq, 128), (row, head, 1))}, window=5)

    for row, head in ((64, 4096), (1024, 64), (512, 128), (256, 512), (8, 8), (128, 128), (384, 256)):
        with pytest.raises(ValueError, match="must not overlap"):
            call(row, head)
    # apart: contiguous, wider, heads first, interleaved; single rows and heads at any stride
    for row, head in ((1024, 128), (2048, 136), (128, 512), (256, 1024), (1536, 128)):
        with pytest.raises(ValueError, match="one CUDA device"):
            call(row, head)
    with pytest.raises(ValueError, match="one CUDA device"):
        call(8, 128, T=1)
    for n, m, D in ((1, 1, 8), (1, 5, 8), (4, 3, 8), (5, 5, 16), (7, 2, 8)):   # against every pair of runs
        for row in range(8, 160, 8):
            for head in range(8, 160, 8):
                runs = sorted(i * row + j * head for i in range(n) for j in range(m))
                assert _apart(row, n, head, m, D) == all(y - x >= D for x, y in zip(runs, runs[1:])), (n, m, D, row, head)


def test_cache_tensors_that_share_pages_are_refused():
    from monoserve_b200.cache import CachePages
    t = torch.zeros(10, 16, 2, 64, dtype=BF)
    for tensors in ([t[:4], t[2:6]], [t[6:], t[:4], t[3:7]], [t[:4], t[:4]]):
        with pytest.raises(ValueError, match="each of them once"):
            CachePages(tensors)
    with pytest.raises(ValueError, match="CUDA device"):
        CachePages([t[6:], t[:4]])
