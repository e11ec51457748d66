"""sliding_attention and tree_attention against the formula in 64 bits (tests/masked_attention_cases.py), at the lengths,
masks, strides and orders where they can go wrong."""
import pytest
import torch

from tests.masked_attention_cases import make, reference, sliding_mask, tolerance, tree_mask

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def on_gpu(*tensors):
    return [t.cuda() for t in tensors]


def run_sliding(batch, window, sinks, **kw):
    from monoserve_b200.attention import sliding_attention
    return sliding_attention(*on_gpu(*batch), window, sinks=sinks, **kw)


def check(out, batch, masks, scale=None):
    from monoserve_b200.attention import attention_status
    assert attention_status() == 0
    ref, weighted = reference(*batch, masks, scale=scale)
    tol = tolerance(ref, weighted, batch[0].dtype, int(batch[5].max()))
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def sliding_masks(batch, window, sinks):
    start, kv = batch[4].tolist(), batch[5].tolist()
    return [sliding_mask(b - a, L, window, sinks) for a, b, L in zip(start, start[1:], kv)]


HEADS = [(32, 4), (12, 4), (6, 6), (12, 1)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_sliding_ragged_batch(dtype, dim, hq, hkv):
    """Prompts, portions and single tokens together, windows and sinks inside, at and across the 128-key tiles."""
    batch = make([1, 5, 0, 33, 130, 1], [0, 700, 50, 3, 260, 2049], hq, hkv, dim, 16, dtype, seed=hq + dim)
    for window, sinks in ((1, 0), (7, 3), (128, 0), (129, 130), (500, 17), (1 << 31 - 1, 0)):
        check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128])
def test_sliding_single_tokens_of_all_lengths(page):
    past = [0, 1, 15, 126, 127, 128, 129, 255, 256, 1000, 4095, 9000]
    batch = make([1] * len(past), past, 32, 4, 128, page, BF, seed=page)
    for window, sinks in ((4096, 4), (1024, 0), (100000, 0), (200, 300)):
        check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


@pytest.mark.parametrize("window,sinks", [(1024, 4), (100000, 0), (130, 600)])
def test_sliding_long_prompts(window, sinks):
    batch = make([1500, 777], [0, 901], 32, 4, 128, 16, BF, seed=5)
    check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


def test_one_long_context():
    """A context long enough to be split over every SM."""
    batch = make([1], [100_000], 8, 1, 128, 64, BF, seed=6)
    for window, sinks in ((1 << 30, 0), (70_001, 129)):
        check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


@pytest.mark.parametrize("dim", [64, 128])
def test_what_no_row_sees_may_hold_anything(dim):
    """Keys between the sinks and the window, behind the last one and in other pages are NaN; so are pages nobody owns."""
    batch = make([1, 3, 40], [300, 900, 513], 32, 4, dim, 16, BF, seed=7, fill=float("nan"))
    q, kc, vc, bt, start, kv = batch
    window, sinks = 70, 5
    for r, (a, b, L) in enumerate(zip(start.tolist(), start.tolist()[1:], kv.tolist())):
        for j in range(sinks, L - (b - a) - window + 1):
            kc[bt[r, j // 16], j % 16] = float("nan")
            vc[bt[r, j // 16], j % 16] = float("inf")
    check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


def test_rows_that_see_nothing_and_rows_of_nobody():
    """More rows than keys: the rows in front of the first key are zeros; rows behind the last request are left alone, those
    of requests without keys are zeros."""
    from monoserve_b200.attention import sliding_attention
    q, kc, vc, bt, start, kv = make([6, 2, 4], [10, 0, 20], 32, 4, 128, 16, BF, seed=8)
    kv = torch.tensor([4, 0, 24], dtype=torch.int32)
    q = torch.cat([q, q[:3]])
    out = torch.full_like(q, 7.0).cuda()
    args = on_gpu(q, kc, vc, bt, start, kv)
    sliding_attention(*args, 100, out=out)
    masks = [sliding_mask(6, 4, 100, 0), torch.zeros(2, 0, dtype=torch.bool), sliding_mask(4, 24, 100, 0)]
    batch = (q[:12], kc, vc, bt, start, kv)
    check(out[:12], batch, masks)
    assert bool((out[:2] == 0).all()) and bool((out[6:8] == 0).all()) and bool((out[12:] == 7).all())


def test_keys_end_with_the_block_table():
    batch = make([2], [62], 4, 4, 64, 16, BF, seed=9)
    q, kc, vc, bt, start, kv = batch
    kv = kv + 30   # 94 keys said, 64 there: the rows are at positions 92 and 93
    batch = (q, kc, vc, bt, start, kv)
    check(run_sliding(batch, 40, 3), batch, sliding_masks(batch, 40, 3))
    check(run_sliding(batch, 20, 0), batch, sliding_masks(batch, 20, 0))


def random_trees(rows, seed, empty=False):
    g = torch.Generator().manual_seed(seed)
    words = max(1, -(-max(rows) // 32))
    t = torch.randint(-(1 << 31), 1 << 31, (sum(rows), words), generator=g).to(torch.int32)
    if empty:
        t[::2] = 0
    return t


def tree_masks(batch, tree):
    start, kv = batch[4].tolist(), batch[5].tolist()
    return [tree_mask(tree[a:b], b - a, L) for a, b, L in zip(start, start[1:], kv)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_tree_any_bits(dtype, dim, hq, hkv):
    """Any bits, also those of later tokens; drafted tokens that begin anywhere in a tile of keys; rows that see nothing."""
    from monoserve_b200.attention import tree_attention
    rows, past = [1, 8, 33, 64, 100, 7, 0], [0, 127, 250, 1000, 128, 0, 40]
    batch = make(rows, past, hq, hkv, dim, 16, dtype, seed=hq * dim)
    for empty in (False, True):
        tree = random_trees(rows, hq, empty)
        check(tree_attention(*on_gpu(*batch), tree.cuda()), batch, tree_masks(batch, tree))


def test_tree_of_parents_and_few_words():
    from monoserve_b200.attention import tree_attention, tree_bits
    parents = [-1, 0, 0, 1, 1, 2, -1, 6] + list(range(7, 39))
    bits = tree_bits(parents)
    assert bits.shape == (40, 2)
    batch = make([40], [333], 32, 4, 128, 16, BF, seed=11)
    check(tree_attention(*on_gpu(*batch), bits.cuda()), batch, tree_masks(batch, bits))
    short = bits[:, :1].contiguous()   # drafted tokens from 32 on are seen by none
    check(tree_attention(*on_gpu(*batch), short.cuda()), batch, tree_masks(batch, short))


def test_a_chain_is_causal_attention():
    from monoserve_b200.attention import sliding_attention, tree_attention, tree_bits
    batch = on_gpu(*make([16, 16], [500, 77], 32, 4, 128, 16, BF, seed=12))
    chain = torch.cat([tree_bits(range(-1, 15))] * 2).cuda()
    assert torch.equal(tree_attention(*batch, chain), sliding_attention(*batch, 1 << 30))


@pytest.mark.parametrize("rows", [[1] * 5, [40, 1, 300]])
def test_strides_of_q_and_out(rows):
    """q as a view of a projection's rows, out as a view of a wider buffer, and out in the place of q: the same bits."""
    from monoserve_b200.attention import sliding_attention
    past = [100 * (r + 1) for r in range(len(rows))]
    q, kc, vc, bt, start, kv = on_gpu(*make(rows, past, 32, 4, 128, 16, BF, seed=13))
    want = sliding_attention(q, kc, vc, bt, start, kv, 150, sinks=2)
    qkv = torch.zeros(len(q), 40, 128, dtype=BF, device="cuda")
    qkv[:, :32] = q
    wide = torch.full((len(q), 33, 160), 3.0, dtype=BF, device="cuda")
    sliding_attention(qkv[:, :32], kc, vc, bt, start, kv, 150, sinks=2, out=wide[:, :32, 8:136])
    assert torch.equal(wide[:, :32, 8:136], want)
    assert bool((wide[:, 32] == 3).all()) and bool((wide[:, :, :8] == 3).all()) and bool((wide[:, :, 136:] == 3).all())
    sliding_attention(qkv[:, :32], kc, vc, bt, start, kv, 150, sinks=2, out=qkv[:, :32])
    assert torch.equal(qkv[:, :32], want) and bool((qkv[:, 32:] == 0).all())
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(sliding_attention(heads_first, kc, vc, bt, start, kv, 150, sinks=2), want)


def test_the_same_bits_every_time():
    from monoserve_b200.attention import sliding_attention
    batch = on_gpu(*make([1, 1, 200, 1], [9000, 3000, 500, 20], 32, 4, 128, 16, BF, seed=14))
    want = sliding_attention(*batch, 1 << 30)
    assert all(torch.equal(sliding_attention(*batch, 1 << 30), want) for _ in range(20))


def test_a_captured_call_takes_the_lengths_of_its_replay():
    from monoserve_b200.attention import sliding_attention
    long = make([1, 1, 1], [700, 2000, 5000], 32, 4, 128, 16, BF, seed=15)
    q, kc, vc, bt, start, kv = on_gpu(*long)
    sliding_attention(q, kc, vc, bt, start, kv, 900, sinks=4)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = sliding_attention(q, kc, vc, bt, start, kv, 900, sinks=4)
    for lens in ([701, 2001, 5001], [3, 1500, 1], [701, 0, 4999]):
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        batch = (*long[:5], torch.tensor(lens, dtype=torch.int32))
        check(out, batch, [sliding_mask(1, L, 900, 4) if L else torch.zeros(1, 0, dtype=torch.bool) for L in lens])


def test_calls_on_two_streams_and_two_graphs_at_once():
    """Calls that overlap do not share a workspace."""
    from monoserve_b200.attention import sliding_attention
    batches = [on_gpu(*make([1, 1], [6000 + s, 3000], 32, 4, 128, 16, BF, seed=16 + s)) for s in range(2)]
    want = [sliding_attention(*b, 1 << 30) for b in batches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[sliding_attention(*b, 1 << 30, stream=st) for _ in range(8)] for b, st in zip(batches, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)
    graphs, outs = [], []
    for b in batches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sliding_attention(*b, 1 << 30))
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_a_cache_past_32_bits():
    """Pages whose first value lies past 2^31 values."""
    from monoserve_b200.attention import sliding_attention
    batch = make([1, 20], [200, 100], 8, 8, 128, 64, BF, seed=18, extra_pages=1)
    q, kc, vc, bt, start, kv = batch
    n = kc.shape[0]
    far = (1 << 31) // kc[0].numel() + 3
    big = [torch.empty(far + n, *kc.shape[1:], dtype=BF, device="cuda") for _ in range(2)]
    for b, c in zip(big, (kc, vc)):
        b[far:] = c.cuda()
    out = sliding_attention(q.cuda(), *big, (bt + far).cuda(), start.cuda(), kv.cuda(), 150)
    check(out, batch, sliding_masks(batch, 150, 0))


def test_many_requests_most_of_them_empty():
    rows = [1 if r % 37 == 0 else 0 for r in range(1500)]
    past = [r % 400 for r in range(1500)]
    batch = make(rows, past, 4, 2, 64, 16, FP, seed=19)
    check(run_sliding(batch, 100, 1), batch, sliding_masks(batch, 100, 1))


def test_scale_and_large_scores():
    """Weights that are all but zero and maxima that grow from tile to tile."""
    q, kc, vc, bt, start, kv = make([1, 70], [1000, 500], 8, 2, 128, 16, BF, seed=20)
    batch = (q, kc, vc, bt, start, kv)
    check(run_sliding(batch, 1 << 30, 0, scale=1e-4), batch, sliding_masks(batch, 1 << 30, 0), scale=1e-4)
    ramp = torch.arange(kc.shape[0] * 16).view(-1, 16, 1, 1) / 1024
    batch = (q.sign(), (kc.sign() * ramp).to(BF), vc, bt, start, kv)
    out = run_sliding(batch, 1 << 30, 0, scale=1.0)
    ref, weighted = reference(*batch, sliding_masks(batch, 1 << 30, 0), scale=1.0)
    # 128 exact products below 1.8: their 32-bit sum is off by less than 128 * 2^-24 * 128 * 1.8 = 1.8e-3
    tol = tolerance(ref, weighted, BF, 1100) + 1.8e-3 * weighted
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def test_as_many_requests_as_a_call_takes():
    R = 16384
    rows, past = [1] * R, [r % 3 for r in range(R)]
    batch = make(rows, past, 1, 1, 64, 8, BF, seed=21)
    check(run_sliding(batch, 2, 0), batch, sliding_masks(batch, 2, 0))


def test_a_status_word_of_ones_own():
    from monoserve_b200.attention import attention_status, sliding_attention
    batch = on_gpu(*make([3], [200], 8, 2, 64, 16, FP, seed=22))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = sliding_attention(*batch, 50)
    assert torch.equal(sliding_attention(*batch, 50, status=status), want)
    assert status.item() == 0 and attention_status() == 0
    q, *rest = batch
    assert sliding_attention(q[:0], *rest[:3], torch.zeros(2, dtype=torch.int32, device="cuda"), rest[4], 50).shape == (0, 8, 64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert sliding_attention(q[:0], *rest[:2], rest[2][:0], none.new_zeros(1), none, 50).shape == (0, 8, 64)


def test_groups_of_128_and_wide_kv_heads():
    for hq, hkv, rows in ((128, 1, [1, 3]), (256, 2, [2, 1]), (40, 40, [200, 1]), (24, 8, [90, 43])):
        batch = make(rows, [300, 129], hq, hkv, 64, 32, BF, seed=hq)
        check(run_sliding(batch, 200, 7), batch, sliding_masks(batch, 200, 7))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hkv", [(32, 4), (12, 4), (5, 5), (16, 1), (96, 8)])
def test_batches_of_few_rows(dtype, hq, hkv):
    """At most 16 rows of a KV head a request on the mean: those requests' rows are the columns of the products, others among
    them (of a pair, too) are not. Windows, sinks and trees; every kind of item behind every other."""
    from monoserve_b200.attention import tree_attention
    group = hq // hkv
    few = max(1, 16 // group)
    rows = [1, few, 0, 1, few, 0, 0, 1, 1, 0, 0, 0, 0, 1]
    past = [3000, 700, 10, 0, 129, 5, 7, 128, 2048, 0, 0, 1, 2, 60]
    big = 16 // group * len(rows) - sum(rows)   # as many more as the mean allows
    if big > 0:
        rows[9], past[9] = big, 333
    batch = make(rows, past, hq, hkv, 128, 16, dtype, seed=hq + 31)
    assert sum(rows) * group <= 16 * len(rows)
    for window, sinks in ((1 << 30, 0), (100, 3), (129, 140), (1, 0)):
        check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))
    for empty in (False, True):
        tree = random_trees(rows, hq, empty)
        check(tree_attention(*on_gpu(*batch), tree.cuda()), batch, tree_masks(batch, tree))


def test_few_rows_whose_maxima_grow_and_unseen_values():
    """Maxima that grow from tile to tile, so that sums are rescaled, and NaN in what nobody sees."""
    q, kc, vc, bt, start, kv = make([1, 1, 1], [3000, 1000, 1], 32, 4, 128, 16, BF, seed=33, fill=float("nan"))
    ramp = torch.zeros(kc.shape[0])
    for r, L in enumerate(kv.tolist()):
        for j in range(-(-L // 16)):
            ramp[bt[r, j]] = (j + 1) / 128
    batch = (q.sign(), (kc.sign() * ramp[:, None, None, None]).to(BF), vc, bt, start, kv)
    out = run_sliding(batch, 1 << 30, 0, scale=1.0)
    ref, weighted = reference(*batch, sliding_masks(batch, 1 << 30, 0), scale=1.0)
    # 128 exact products of at most 1.5: their 32-bit sum is off by less than 128 * 2^-24 * 128 * 1.5 = 1.5e-3
    tol = tolerance(ref, weighted, BF, 3100) + 1.5e-3 * weighted
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1, 3], [5, 40, 33], [70, 9, 150]])
def test_drafted_tokens_that_no_row_sees_may_hold_anything(dim, rows):
    """Padded drafts, whose rows of the cache nobody has written: every third token is seen by none, itself included."""
    from monoserve_b200.attention import tree_attention
    batch = make(rows, [300, 0, 120], 32, 4, dim, 16, BF, seed=dim + rows[0], fill=float("nan"))
    q, kc, vc, bt, start, kv = batch
    tree = random_trees(rows, 5)
    for r, (a, b, L) in enumerate(zip(start.tolist(), start.tolist()[1:], kv.tolist())):
        for d in range(1, b - a, 3):
            bit = 1 << d % 32
            tree[a:b, d // 32] &= ~bit if bit < 1 << 31 else (1 << 31) - 1
            tree[a + d] = 0
            j = L - (b - a) + d
            kc[bt[r, j // 16], j % 16] = float("nan")
            vc[bt[r, j // 16], j % 16] = float("inf" if d % 2 else "nan")
            q[a + d] = float("nan")
    out = tree_attention(*on_gpu(*batch), tree.cuda())
    padded = torch.cat([torch.arange(n) % 3 == 1 for n in rows])
    clean = q.clone()
    clean[padded] = 0
    got = out.cpu()
    past = torch.cat([torch.full((n,), int(L) > n) for n, L in zip(rows, kv)])
    assert bool(got[padded & past].isnan().all())         # a padded row's own queries are no numbers, and it sees the past
    assert bool((got[padded & ~past] == 0).all())         # or nothing
    masks = tree_masks(batch, tree)
    ref, weighted = reference(clean, kc, vc, bt, start, kv, masks)
    err = (got.double() - ref).abs()[~padded]
    assert bool((err <= tolerance(ref, weighted, BF, int(kv.max()))[~padded]).all())


@pytest.mark.parametrize("rows", [[1, 1], [20, 1], [200, 3]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_score_that_is_no_number_shows_in_the_rows_that_see_it(rows, bad):
    """One key at each column of a 16-column pattern, whichever way its weight is worked out; other rows are as ever."""
    q, kc, vc, bt, start, kv = make(rows, [260, 700], 8, 1, 128, 16, BF, seed=41)
    q = q.abs() + 0.125   # with a key of infinities: a score of infinity
    for column in range(16):
        key = 100 + column
        keys = kc.clone()
        keys[bt[0, key // 16], key % 16] = bad
        batch = (q, keys, vc, bt, start, kv)
        window = 260 + rows[0] // 2 - key   # seen by the first half of the request's rows; by a single one
        window += rows[0] == 1
        out = run_sliding(batch, window, 0).cpu()
        sees = sliding_mask(rows[0], 260 + rows[0], window, 0)[:, key]
        assert bool(sees.any())
        assert bool(out[:rows[0]][sees].isnan().all())
        good = torch.cat([~sees, torch.ones(rows[1], dtype=torch.bool)])
        ref, weighted = reference(q, kc, vc, bt, start, kv, sliding_masks(batch, window, 0))
        tol = tolerance(ref, weighted, BF, 800)
        assert bool(((out.double() - ref).abs() <= tol)[good].all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_len", [[4, 0, 24], [39, 1, 3], [300, 2, 4]])
def test_trees_with_fewer_keys_than_rows(dim, kv_len):
    """The first drafted tokens have no key: their bits say nothing, and rows that see none of the others are zeros."""
    from monoserve_b200.attention import tree_attention
    rows = [40, 2, 4]
    q, kc, vc, bt, start, _ = make(rows, [300, 0, 20], 32, 4, dim, 16, BF, seed=77)
    for empty in (False, True):
        tree = random_trees(rows, 78, empty)
        batch = (q, kc, vc, bt, start, torch.tensor(kv_len, dtype=torch.int32))
        check(tree_attention(*on_gpu(*batch), tree.cuda()), batch, tree_masks(batch, tree))


def far_below_the_reference(out, weighted, keys_per_one):
    """As tolerance() for fp16, whose weights have steps of 2^-31 of their reference at worst: half of that for each key, times
    keys_per_one, the keys times |v| for each whole unit of the sum of weights."""
    half = torch.finfo(FP).eps / 2
    return half * out.abs() + (half + 3e-4) * weighted + keys_per_one * 2.0 ** -32 + 2.0 ** -25


@pytest.mark.parametrize("dim,hq,rows", [(128, 8, [1]), (128, 8, [5]), (128, 8, [40]), (64, 8, [1]), (64, 2, [200])])
def test_fp16_weights_far_below_the_largest_count(dim, hq, rows):
    """One key of 64 has nearly all the weight and no value; 63 others have 2^-26 of it each and large values, which are the output.
    As columns and as rows of the products, of one stream's rows and of two."""
    q, kc, vc, bt, start, kv = make(rows, [640], hq, 1, dim, 16, FP, seed=51)
    q.zero_(), kc.zero_(), vc.fill_(1000.0)
    q[:, :, 0] = 1
    for j in range(0, int(kv[0]), 64):
        kc[bt[0, j // 16], j % 16, :, 0] = 18.0   # 18 log2(e) = 25.97
        vc[bt[0, j // 16], j % 16] = 0
    batch = (q, kc, vc, bt, start, kv)
    out = run_sliding(batch, 1 << 30, 0, scale=1.0).double().cpu()
    ref, weighted = reference(*batch, sliding_masks(batch, 1 << 30, 0), scale=1.0)
    assert float(ref.min()) > 8e-4
    err = (out - ref).abs()
    assert bool((err <= far_below_the_reference(ref, weighted, 64 * 1000)).all()), float((err / ref).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_fp16_weights_of_ragged_batches(dim, hq, hkv):
    """The sum of a row's weights is one at least in units of its largest, which is its reference or above it."""
    batch = make([1, 5, 0, 33, 130, 1], [0, 700, 50, 3, 260, 2049], hq, hkv, dim, 16, FP, seed=hq + dim + 52)
    for window, sinks in ((7, 3), (500, 17), (1 << 30, 0)):
        out = run_sliding(batch, window, sinks, scale=0.5).double().cpu()   # peaked: scores of several times the usual ones
        ref, weighted = reference(*batch, sliding_masks(batch, window, sinks), scale=0.5)
        # a weight's exponent is off by 128 * 2^-24 * 128 * 0.5 = 4.9e-4 at most and its power of two by 2^-13; so is the sum
        tol = far_below_the_reference(ref, weighted, int(batch[5].max()) * 6) + 2 * 6.2e-4 * weighted
        err = (out - ref).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[1], [10], [40]])
@pytest.mark.parametrize("window", [1, 20, 2000, (1 << 31) - 700, (1 << 31) - 1])
@pytest.mark.parametrize("sinks", [0, 5, 300])
def test_positions_up_to_the_largest(dim, rows, window, sinks):
    """As many keys as an int32 can say, of which the block table has the first 640: most windows lie behind all of them."""
    q, kc, vc, bt, start, _ = make(rows, [640 - rows[0]], 8, 1, dim, 16, BF, seed=54)
    L = (1 << 31) - 1
    p, j = torch.arange(L - rows[0], L)[:, None], torch.arange(640)[None]
    mask = (j > p - window) | (j < sinks)
    batch = (q, kc, vc, bt, start, torch.tensor([L], dtype=torch.int32))
    out = run_sliding(batch, window, sinks)
    ref, weighted = reference(*batch, [mask])
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tolerance(ref, weighted, BF, 640)).all()), float(err.max())


NO_WINDOW = (1 << 31) - 1   # the largest numbers that a call takes


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [1, 20, 0, 150]])
@pytest.mark.parametrize("window,sinks", [(NO_WINDOW, 0), (NO_WINDOW, NO_WINDOW), (1, NO_WINDOW), (100, NO_WINDOW), (130, 200)])
def test_the_largest_windows_and_sinks(dim, rows, window, sinks):
    """As columns (dim 128, single tokens) and as rows of the products."""
    batch = make(rows, [700, 129, 5, 0], 32, 4, dim, 16, BF, seed=53)
    check(run_sliding(batch, window, sinks), batch, sliding_masks(batch, window, sinks))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1], [9, 1], [20, 1], [200, 3]])
def test_a_score_of_minus_infinity_has_no_weight(dim, rows):
    """As the formula says: the power of minus infinity is zero. Rows whose scores are all that are zeros, as those that see no key."""
    n = rows[0]
    q, kc, vc, bt, start, kv = make(rows, [260, 700], 8, 1, dim, 16, BF, seed=55)
    q = q.abs() + 0.125
    for j in range(260 - 10, 260 + (n + 1) // 2):   # keys in front of the rows, and of the first half of them
        kc[bt[0, j // 16], j % 16] = -float("inf")
    batch = (q, kc, vc, bt, start, kv)
    for window, sinks in ((8, 0), (8, 3), (1 << 30, 0)):
        out = run_sliding(batch, window, sinks)
        check(out, batch, sliding_masks(batch, window, sinks))
        if (window, sinks) == (8, 0):
            assert bool((out[:(n + 1) // 2] == 0).all())


def test_every_ancestor_of_a_drafted_token_counts():
    """A tree behind a short past, within a bound for each element that no other tree's result would keep: any one bit of the
    oracle's masks turned over shows in its row."""
    from monoserve_b200.attention import attention_status, tree_attention, tree_bits
    batch = make([7], [37], 8, 2, 128, 16, BF, seed=56)
    tree = tree_bits([-1, 0, 0, 1, 2, 2, 5])
    out = tree_attention(*on_gpu(*batch), tree.cuda()).double().cpu()
    assert attention_status() == 0

    def off(words):
        ref, weighted = reference(*batch, tree_masks(batch, words))
        return ((out - ref).abs() / tolerance(ref, weighted, BF, 44)).amax((1, 2))

    assert bool((off(tree) <= 1).all())
    for row in range(7):
        for d in range(7):
            other = tree.clone()
            other[row, 0] ^= 1 << d
            assert float(off(other)[row]) > 1, (row, d)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1, 1], [9, 40, 1]])
def test_pages_that_do_not_exist_read_as_zeros(dim, rows):
    from monoserve_b200.attention import tree_attention
    q, kc, vc, bt, start, kv = make(rows, [300, 500, 90], 32, 4, dim, 16, BF, seed=57)
    n = kc.shape[0]
    bad = bt.clone()
    for r, column, page in ((0, 1, -1), (0, 12, n), (0, 18, n + 1000), (1, 0, -1000), (1, 20, n), (1, 31, -1), (2, 5, n)):
        bad[r, column] = page
    zeros = torch.where((bad < 0) | (bad >= n), n, bad)   # the oracle has a page of zeros for them
    kz, vz = (torch.cat([t, torch.zeros_like(t[:1])]) for t in (kc, vc))
    oracle = (q, kz, vz, zeros, start, kv)
    for window, sinks in ((1 << 30, 0), (150, 20)):
        check(run_sliding((q, kc, vc, bad, start, kv), window, sinks), oracle, sliding_masks(oracle, window, sinks))
    tree = random_trees(rows, 58)
    check(tree_attention(*on_gpu(q, kc, vc, bad, start, kv), tree.cuda()), oracle, tree_masks(oracle, tree))


@pytest.mark.parametrize("dim", [64, 128])
def test_row_starts_that_are_no_ascending_places(dim):
    """Taken within [0, tokens]; a request that ends in front of its begin has no rows, and rows of nobody stay."""
    from monoserve_b200.attention import sliding_attention
    q, kc, vc, bt, _, kv = make([3, 0, 7, 0, 4], [90, 200, 0, 30, 500], 32, 4, dim, 16, BF, seed=59)
    T = len(q)
    said = torch.tensor([-5, 3, 2, 10, 9, 1 << 30], dtype=torch.int32)
    taken = [(0, 3), (3, 3), (2, 10), (10, 10), (9, T)]
    out = torch.full_like(q, 5.0).cuda()
    # requests 0 and 2 say rows 2 both, 2 and 4 row 9: the test looks at the others
    sliding_attention(*on_gpu(q, kc, vc, bt, said, kv), 100, sinks=3, out=out)
    for r, (a, b) in enumerate(taken):
        if a == b:
            continue
        one = (q[a:b], kc, vc, bt[r:r + 1], torch.tensor([0, b - a], dtype=torch.int32), kv[r:r + 1])
        ref, weighted = reference(*one, sliding_masks(one, 100, 3))
        err = ((out[a:b].double().cpu() - ref).abs() <= tolerance(ref, weighted, BF, 600)).all(2).all(1)
        assert all(bool(err[i - a]) for i in range(a, b) if i not in (2, 9)), (r, err)
    said = torch.tensor([4, 7, 7, 7, 7, 9], dtype=torch.int32)   # rows 0 .. 3 and 9 .. are nobody's
    out.fill_(5.0)
    sliding_attention(*on_gpu(q, kc, vc, bt, said, kv), 100, sinks=3, out=out)
    assert bool((out[:4] == 5).all()) and bool((out[9:] == 5).all()) and not bool((out[4:9] == 5).any())


def test_calls_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor
    from monoserve_b200.attention import attention_status, sliding_attention
    batches = [on_gpu(*make([1, 1 + 20 * s], [3000 + s, 700], 32, 4, 64 * (1 + s % 2), 16, BF, seed=60 + s)) for s in range(4)]
    want = [sliding_attention(*b, 500, sinks=2) for b in batches]
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        outs = [sliding_attention(*batches[i], 500, sinks=2, stream=stream) for _ in range(20)]
        stream.synchronize()
        return all(torch.equal(o, want[i]) for o in outs)

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))
    assert attention_status() == 0


@pytest.mark.parametrize("dtype,size", [(FP, 1 << 23), (BF, 1 << 28)])
@pytest.mark.parametrize("dim,rows", [(64, [1, 30]), (128, [1, 1]), (128, [40, 3])])
def test_scores_as_large_as_may_be(dtype, size, dim, rows):
    """Scores of about `size`, exact, most of them a whole step below the largest ones: the output is the mean of those' values.
    They come in later tiles for some rows, so that references move."""
    q, kc, vc, bt, start, kv = make(rows, [700, 400], 8, 2, dim, 16, dtype, seed=61)
    q.zero_(), kc.zero_()
    q[:, :, 0] = 1 << 8
    g = torch.Generator().manual_seed(62)
    kc[..., 0] = torch.randint(-3, 1, kc.shape[:3], generator=g).to(dtype) * (size >> 15) + (size >> 8)   # steps of 2^-7 of `size`
    batch = (q, kc, vc, bt, start, kv)
    for window, sinks in ((1 << 30, 0), (200, 3)):
        check(run_sliding(batch, window, sinks, scale=1.0), batch, sliding_masks(batch, window, sinks), scale=1.0)
