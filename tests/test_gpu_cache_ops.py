"""qk_rope against its formula in 64 bits, and the cache's page and row moves against the same moves on the host."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def rope_inputs(T, hq, hkv, D, rot, dtype, seed, page=16, norms=True, max_pos=5000):
    from monoserve_b200.lane_base import rope_table
    g = torch.Generator().manual_seed(seed)
    n_pages = -(-T // page) + 2
    return dict(qkv=torch.randn(T, (hq + 2 * hkv) * D, generator=g).to(dtype), positions=torch.randint(0, max_pos, (T,), generator=g, dtype=torch.int32),
                slots=(torch.randperm((n_pages - 1) * page, generator=g)[:T] + page).to(torch.int32),
                k_cache=torch.full((n_pages, page, hkv, D), 9.0).to(dtype), v_cache=torch.full((n_pages, page, hkv, D), 9.0).to(dtype),
                cos_sin=rope_table(1e6, rot, max_pos), hq=hq, q_norm=(torch.randn(D, generator=g) + 1).to(dtype) if norms else None,
                k_norm=(torch.randn(D, generator=g) + 1).to(dtype) if norms else None)


def rope_reference(qkv, positions, slots, k_cache, v_cache, cos_sin, hq, q_norm, k_norm, eps=1e-6, interleaved=False):
    """(q, k_cache, v_cache) in 64 bits, and for the heads how far each may be off apart from its rounding."""
    hkv, D = k_cache.shape[2:]
    x = qkv.double().view(len(qkv), hq + 2 * hkv, D)
    rot = 2 * cos_sin.shape[1]
    cs = cos_sin[positions.long().clamp(0, len(cos_sin) - 1)].double()[:, None]

    def head(h, w):
        y = h if w is None else h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
        out, size = y.clone(), y.abs()
        i = torch.arange(rot // 2)
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        a, b = y[..., first], y[..., second]
        out[..., first], out[..., second] = a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]
        size[..., first] = size[..., second] = a.abs() + b.abs()
        return out, size

    q, q_size = head(x[:, :hq], q_norm)
    k, k_size = head(x[:, hq:hq + hkv], k_norm)
    kc, vc, k_far = k_cache.double(), v_cache.double(), torch.zeros_like(k_cache, dtype=torch.float64)
    there = (slots >= 0) & (slots < kc.shape[0] * kc.shape[1])
    at = slots[there].long()
    kc.view(-1, hkv, D)[at], vc.view(-1, hkv, D)[at], k_far.view(-1, hkv, D)[at] = k[there], x[there, hq + hkv:], k_size[there]
    # 32-bit steps of half 2^-23 each: D for the sum of squares (half of it through the root), eight more for the root, the
    # products and the turn
    far = (D / 2 + 8) * 2.0 ** -24
    return q, kc, vc, far * q_size, far * k_far


def check_rope(a, got, interleaved=False):
    q, kc, vc, q_far, k_far = rope_reference(**a, interleaved=interleaved)
    half = torch.finfo(a["qkv"].dtype).eps / 2
    least = 2.0 ** -25 if a["qkv"].dtype == FP else 0.0   # half a step of fp16's smallest values
    for out, ref, far in ((got[0], q, q_far), (got[1], kc, k_far)):
        err = (out.double().cpu() - ref).abs()
        assert bool((err <= half * ref.abs() + (1 + half) * far + least).all()), float((err - half * ref.abs()).max())
    assert torch.equal(got[2].double().cpu(), vc)


def run_rope(a, **kw):
    from monoserve_b200.cache import qk_rope
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    d.update(kw)
    q = qk_rope(**d)
    return q, d["k_cache"], d["v_cache"]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (64, 8), (128, 128), (128, 64), (128, 24), (256, 256), (256, 64)])
def test_qk_rope(dtype, interleaved, D, rot):
    for T, hq, hkv, norms in ((1, 32, 4, True), (37, 12, 4, True), (300, 5, 5, True), (9, 8, 1, False)):
        a = rope_inputs(T, hq, hkv, D, rot, dtype, seed=T + D, norms=norms)
        check_rope(a, run_rope(a, interleaved=interleaved), interleaved)


def test_qk_rope_without_turning_one_norm_and_many_heads():
    a = rope_inputs(50, 96, 8, 128, 128, BF, seed=1)
    a["k_norm"] = None
    check_rope(a, run_rope(a))
    a = rope_inputs(50, 96, 8, 128, 128, BF, seed=2)
    a["cos_sin"] = torch.zeros(4, 0, 2)
    check_rope(a, run_rope(a))


def test_qk_rope_padding_far_positions_and_bad_slots():
    a = rope_inputs(40, 32, 4, 128, 128, BF, seed=3)
    a["slots"][::3] = -1
    a["slots"][1] = 1 << 30
    a["slots"][4] = a["k_cache"].shape[0] * 16   # one past the last
    a["positions"][2], a["positions"][5] = 4999, 1 << 30
    a["positions"][7] = -5
    check_rope(a, run_rope(a))


def test_qk_rope_in_place_and_strided():
    a = rope_inputs(65, 32, 4, 128, 128, BF, seed=4)
    want = run_rope(a)
    wide = torch.full((65, 41 * 128), 5.0, dtype=BF, device="cuda")
    wide[:, :40 * 128] = a["qkv"].cuda()
    got = run_rope(a, qkv=wide[:, :40 * 128])
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    q_view = wide.view(65, 41, 128)[:, :32]
    got = run_rope(a, qkv=wide[:, :40 * 128], q_out=q_view)
    assert torch.equal(q_view, want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert torch.equal(wide[:, 32 * 128:40 * 128].cpu(), a["qkv"][:, 32 * 128:]) and bool((wide[:, 40 * 128:] == 5).all())


def test_qk_rope_of_nothing_zeros_and_a_captured_call():
    from monoserve_b200.cache import qk_rope
    a = rope_inputs(8, 4, 2, 64, 64, FP, seed=5)
    none = {k: (v[:0] if k in ("qkv", "positions", "slots") else v) for k, v in a.items()}
    assert run_rope(none)[0].shape == (0, 4, 64)
    a["qkv"][0] = 0
    check_rope(a, run_rope(a))
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    qk_rope(**d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = qk_rope(**d)
    b = rope_inputs(8, 4, 2, 64, 64, FP, seed=6)
    for k in ("qkv", "positions", "slots"):
        d[k].copy_(b[k])
    d["k_cache"].fill_(9)
    d["v_cache"].fill_(9)
    graph.replay()
    torch.cuda.synchronize()
    check_rope({**a, **{k: b[k] for k in ("qkv", "positions", "slots")}}, (q, d["k_cache"], d["v_cache"]))


def test_qk_rope_cache_past_32_bits():
    a = rope_inputs(20, 4, 8, 128, 128, BF, seed=7, page=64)
    far = (1 << 31) // (64 * 8 * 128) + 5
    n = a["k_cache"].shape[0]
    big = [torch.empty(far + n, 64, 8, 128, dtype=BF, device="cuda") for _ in range(2)]
    for b in big:
        b[far:] = 9
    q, kc, vc = run_rope(a, k_cache=big[0], v_cache=big[1], slots=a["slots"].cuda() + far * 64)
    check_rope(a, (q, kc[far:], vc[far:]))


def test_qk_rope_many_rows():
    a = rope_inputs(5000, 32, 4, 128, 128, BF, seed=8)
    check_rope(a, run_rope(a))


# ---------------------------------------------------------------------------------------------------- pages and rows

def cache(layers, n_pages, page, hkv, D, seed, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n_pages, page, hkv, D, generator=g).to(dtype) for _ in range(2 * layers)]


@pytest.mark.parametrize("page,hkv,D", [(16, 4, 128), (64, 8, 128), (8, 1, 8), (32, 3, 24)])
@pytest.mark.parametrize("pairs", [1, 7, 100])
def test_copy_pages(page, hkv, D, pairs):
    from monoserve_b200.cache import CachePages
    host = cache(3, 2 * pairs + 3, page, hkv, D, seed=pairs + page)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    order = torch.randperm(2 * pairs + 3, generator=torch.Generator().manual_seed(pairs)).to(torch.int32)
    src, dst = order[:pairs].clone(), order[pairs:2 * pairs].clone()
    if pairs > 2:
        src[1] = src[0]           # one page to two places
        src[2] = dst[2]           # nothing to do
    pages.copy(src.cuda(), dst.cuda())
    pages.check()
    for t in host:
        t[dst.long()] = t[src.long()].clone()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))


def test_copy_pages_from_lists_and_of_nothing():
    from monoserve_b200.cache import CachePages
    host = cache(1, 9, 16, 2, 64, seed=3)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    pages.copy([1, 1, 4, 5], [2, 3, 4, 6])
    pages.copy([], [])
    pages.check()
    for t in host:
        t[2], t[3], t[6] = t[1], t[1], t[5]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))
    for src, dst in (([1, 2], [3, 3]), ([1, 2], [2, 4]), ([1], [9]), ([-1], [2]), ([1, 2], [3])):
        with pytest.raises(ValueError):
            pages.copy(src, dst)
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    for src, dst in ((i, i[:1]), (i.long(), i.long()), (i.cpu(), i), (i[:, None], i[:, None])):
        with pytest.raises(ValueError):
            pages.copy(src, dst)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))


def test_copies_that_depend_on_their_order_are_left_out():
    from monoserve_b200.cache import CachePages
    host = cache(2, 12, 16, 2, 64, seed=4)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    src = torch.tensor([1, 2, 4, 6, 8, 12, 3, -1], dtype=torch.int32)
    dst = torch.tensor([2, 3, 5, 7, 7, 9, 10, 11], dtype=torch.int32)
    pages.copy(src.cuda(), dst.cuda())
    with pytest.raises(RuntimeError, match="left out"):
        pages.check()
    pages.check()
    for t in host:   # 1 -> 2 -> 3 -> 10 is a chain, 7 is taken twice, 12 and -1 are no pages
        t[5] = t[4]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))


def accept_reference(host, bt, base, path, count, page):
    for t in host:
        old = t.clone()
        for r in range(len(base)):
            for i in range(min(int(count[r]), path.shape[1])):
                (a, x), (b, y) = (divmod(int(base[r]) + j, page) for j in (int(path[r, i]), i))
                t[bt[r, b], y] = old[bt[r, a], x]


@pytest.mark.parametrize("page,hkv,D,most", [(16, 4, 128, 9), (8, 1, 8, 30), (64, 8, 128, 100), (16, 3, 24, 1), (16, 2, 64, 700)])
def test_accept_rows(page, hkv, D, most):
    """Paths that run upwards, that run anywhere among the drafts and that name a draft twice, over the ends of pages."""
    from monoserve_b200.cache import CachePages
    g = torch.Generator().manual_seed(most)
    R, room = 5, 2 * most + 5
    base = torch.randint(0, 40, (R,), generator=g, dtype=torch.int32)
    need = -(-(40 + room) // page)
    host = cache(2, R * need + 1, page, hkv, D, seed=most)
    bt = (torch.randperm(R * need, generator=g) + 1).view(R, need).to(torch.int32)
    path = torch.stack([torch.randperm(room, generator=g)[:most] for _ in range(R)]).to(torch.int32)
    path[1] = path[1].sort().values
    path[2] = torch.randint(0, room, (most,), generator=g)
    path[3] = torch.arange(most)
    count = torch.tensor([most, most, most, most, 0], dtype=torch.int32)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    pages.accept(bt.cuda(), base.cuda(), path.cuda(), count.cuda())
    pages.check()
    accept_reference(host, bt, base, path, count, page)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))


def test_accept_rows_that_are_not_there_stay():
    from monoserve_b200.cache import CachePages
    host = cache(1, 6, 16, 2, 64, seed=6)
    bt = torch.tensor([[1, 2], [3, 9]], dtype=torch.int32)        # page 9 does not exist
    base = torch.tensor([10, 12], dtype=torch.int32)
    path = torch.tensor([[3, -1, 30, 5], [1, 6, 2, 3]], dtype=torch.int32)
    count = torch.tensor([9, 3], dtype=torch.int32)               # of four; a count past the path ends with it
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    pages.accept(bt.cuda(), base.cuda(), path.cuda(), count.cuda())
    with pytest.raises(RuntimeError, match="left out"):
        pages.check()
    for t in host:
        old = t.clone()
        t[1, 10], t[1, 13] = old[1, 13], old[1, 15]               # request 0: rows 0 and 3; -1 and 30 are left out
        t[3, 12], t[3, 14] = old[3, 13], old[3, 14]               # request 1: rows 0 and 2; row 1 comes from page 9
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))
    for bad in (dict(base=base[:1]), dict(path=path.long()), dict(count=count[None]), dict(block_table=bt[:, :0])):
        a = {k: v.cuda() for k, v in dict(dict(block_table=bt, base=base, path=path, count=count), **bad).items()}
        with pytest.raises(ValueError):
            pages.accept(**a)


def test_moves_in_a_graph_and_on_a_stream():
    from monoserve_b200.cache import CachePages
    host = cache(2, 9, 16, 2, 64, seed=8)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    src, dst = torch.tensor([1, 2], dtype=torch.int32).cuda(), torch.tensor([3, 4], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pages.copy([7], [8], stream=side)
    pages.copy(src, dst, stream=side)
    side.synchronize()
    for t in host:
        t[8], t[3], t[4] = t[7], t[1], t[2]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.copy(src, dst)
    src.copy_(torch.tensor([5, 6]))
    graph.replay()
    pages.check()
    for t in host:
        t[3], t[4] = t[5], t[6]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))


def test_a_step_of_speculative_decoding():
    """Append, tree attention, acceptance, a fork and the next token, as a server runs them: the next token's attention is that
    of a cache into which only the accepted tokens were ever written."""
    from monoserve_b200.attention import attention_status, sliding_attention, tree_attention, tree_bits
    from monoserve_b200.cache import CachePages, SharedPages, qk_rope
    from monoserve_b200.lane_base import rope_table
    hq, hkv, D, page, past = 8, 2, 128, 16, 37
    g = torch.Generator().manual_seed(9)
    table, pool = rope_table(1e6, D, 4096).cuda(), SharedPages(24)
    kc, vc, kc2, vc2 = (torch.zeros(24, page, hkv, D, dtype=BF, device="cuda") for _ in range(4))
    norm = torch.ones(D, dtype=BF, device="cuda")
    rows = lambda n: torch.randn(n, (hq + 2 * hkv) * D, generator=g).to(BF).cuda()   # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()                         # noqa: E731
    seq = pool.take(4)

    def append(qkv, positions, pages, caches, at=None):
        at = positions if at is None else at
        return qk_rope(qkv, i32(positions), i32([pages[p // page] * page + p % page for p in at]), *caches, table, hq, q_norm=norm, k_norm=norm)

    prompt, drafts, last = rows(past), rows(7), rows(1)
    parents = [-1, 0, 0, 1, 2, 2, 5]
    depth = [0, 1, 1, 2, 2, 2, 3]
    path = [0, 2, 5, 6]
    bt = torch.zeros(1, 6, dtype=torch.int32, device="cuda")
    bt[0, :4] = i32(seq)
    for caches in ((kc, vc), (kc2, vc2)):
        q = append(prompt, list(range(past)), seq, caches)
        sliding_attention(q, *caches, bt, i32([0, past]), i32([past]), 1 << 30)
    # drafts lie in the cache one behind the other, but stand at the positions of their depths
    q = append(drafts, [past + d for d in depth], seq, (kc, vc), at=[past + i for i in range(7)])
    tree = tree_attention(q, kc, vc, bt, i32([0, 7]), i32([past + 7]), tree_bits(parents).cuda())
    CachePages([kc, vc]).accept(bt, i32([past]), i32([path]), i32([4]))
    q2 = append(drafts[path], [past + d for d in range(4)], seq, (kc2, vc2))
    plain = sliding_attention(q2, kc2, vc2, bt, i32([0, 4]), i32([past + 4]), 1 << 30)
    n = past + 4
    for a, b in ((kc, kc2), (vc, vc2)):
        a, b = (t[seq].flatten(0, 1)[:n] for t in (a, b))
        assert torch.equal(a, b)
    # the same keys in another order: weights are rounded at other reference points, each result by half a step
    err = (tree[path].double() - plain.double()).abs()
    assert bool((err <= 2 * (2 * 2.0 ** -8 + 3e-4) * 6).all())
    fork, copies = pool.fork(seq, n, page)
    assert len(copies) == 1
    CachePages([kc, vc]).copy(*zip(*copies))
    bt2 = torch.zeros(2, 6, dtype=torch.int32, device="cuda")
    bt2[0, :4] = bt[0, :4]
    bt2[1, :len(fork)] = i32(fork)
    for pages in (seq, fork):
        q = append(last, [n], pages, (kc, vc))
    both = sliding_attention(q.expand(2, hq, D).contiguous(), kc, vc, bt2, i32([0, 1, 2]), i32([n + 1, n + 1]), 1 << 30)
    q = append(last, [n], seq, (kc2, vc2))
    want = sliding_attention(q, kc2, vc2, bt, i32([0, 1]), i32([n + 1]), 1 << 30)
    assert torch.equal(both[0], want[0]) and torch.equal(both[1], want[0])
    assert attention_status() == 0


def test_pages_copied_to_themselves_are_padding():
    """Of lists and of tensors alike: as often as one likes, and beside a copy to or from the same page."""
    from monoserve_b200.cache import CachePages
    host = cache(2, 9, 16, 2, 64, seed=44)
    dev = [t.cuda() for t in host]
    pages = CachePages(dev)
    src, dst = [0, 1, 0, 3, 5, 2, 0], [0, 2, 0, 3, 3, 2, 0]
    for a, b in ((src, dst), [torch.tensor(t, dtype=torch.int32).cuda() for t in (src, dst)]):
        pages.copy(a, b)
        pages.check()
        for t in host:
            t[2], t[3] = t[1], t[5]
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, host))
    out_of_range = torch.tensor([9, -1], dtype=torch.int32).cuda()
    pages.copy(out_of_range, out_of_range)
    with pytest.raises(RuntimeError, match="left out"):
        pages.check()
    for a, b in ((src, out_of_range), (out_of_range, dst)):
        with pytest.raises(ValueError, match="both"):
            pages.copy(a, b)


def test_a_check_waits_for_calls_on_other_streams():
    """The side stream is busy when its call is made, so that the call has not run when check() is asked."""
    from monoserve_b200.cache import CachePages
    pages = CachePages([t.cuda() for t in cache(1, 9, 16, 2, 64, seed=45)])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()   # noqa: E731
    missing, page, one, zero, table = i32([9]), i32([2]), i32([1]), i32([0]), i32([[1, 9]])
    far = i32([[20]])   # row 20 of the table's pages is in page 9
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.copy(missing, page)

    def replayed():
        with torch.cuda.stream(side):
            graph.replay()

    torch.cuda.synchronize()
    for call in (lambda: pages.copy(missing, page, stream=side), lambda: pages.accept(table, zero, far, one, stream=side), replayed):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)   # cycles: some 50 ms
        call()
        with pytest.raises(RuntimeError, match="left out"):
            pages.check()
        pages.check()
