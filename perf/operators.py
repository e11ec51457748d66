"""The operators of speculative and streaming decoding over a paged cache, in plain form and as calls of this library.

    rope      norms of queries and keys for each head, position rotation and append to the cache (monoserve_b200/cache.py)
    sliding   attention over a paged cache within a window, with a few first tokens that stay visible (monoserve_b200/attention.py)
    tree      attention of drafted token trees over a paged cache (monoserve_b200/attention.py)
    copy      pages of a cache copied in all layers: sequences forked (monoserve_b200/cache.py)
    accept    the accepted drafts' rows moved behind the sequence, in all layers (monoserve_b200/cache.py)

Sizes are those of the attention benchmark and tests (monoserve_b200/benchmarks/attention.py: contexts of 512 to 8192, prompts of
2048, pages of 16 and 64, heads 32 / 4, 96 / 8 and 12 / 4) and generic ones around them.
Lengths belong to a case (drawn from its "lens"); the seed of prepare() makes the contents.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = [(32, 4), (96, 8), (12, 4)]
EPS = 1e-6


def listed():
    return [
        # four sequences decode one token each: nothing but latency; 16-bit floats, small heads, neighbouring pairs turned
        dict(name="rope_step", kind="rope", tokens=4, hq=12, hkv=4, dim=64, rot=64, pairs="neighbours", page=64, past=4000, dtype="fp16", lens=1),
        # four ragged prompts of about 2048 tokens in one pass
        dict(name="rope_prompts", kind="rope", tokens=8191, hq=32, hkv=4, dim=128, rot=128, pairs="halves", page=16, past=0, dtype="bf16", lens=2),
        # two streams past their window, one token each: latency
        dict(name="sliding_step", kind="sliding", requests=2, rows=1, past_lo=1500, past_hi=5000, hq=12, hkv=4, dim=64, page=64, window=1000, sinks=5, dtype="fp16", lens=3),
        # a full decode batch of a server, most sequences longer than the window
        dict(name="sliding_decode", kind="sliding", requests=128, rows=1, past_lo=512, past_hi=8192, hq=32, hkv=4, dim=128, page=16, window=4096, sinks=4, dtype="bf16", lens=4),
        # four ragged prompts, portions of longer ones among them
        dict(name="sliding_prompts", kind="sliding", requests=4, rows=2048, past_lo=0, past_hi=2048, hq=32, hkv=4, dim=128, page=16, window=1024, sinks=4, dtype="bf16", lens=5),
        # one sequence verifies eight drafted tokens: latency
        dict(name="tree_step", kind="tree", requests=1, rows=8, past_lo=1900, past_hi=2100, hq=32, hkv=4, dim=128, page=16, dtype="bf16", lens=6),
        # a batch verifies up to 16 drafts each
        dict(name="tree_batch", kind="tree", requests=32, rows=16, past_lo=512, past_hi=8192, hq=32, hkv=4, dim=128, page=16, dtype="bf16", lens=7),
        # big trees over long contexts, many query heads
        dict(name="tree_long", kind="tree", requests=4, rows=64, past_lo=30000, past_hi=60000, hq=96, hkv=8, dim=128, page=64, dtype="bf16", lens=8),
        # one sequence is forked once: its last page in 48 layers
        dict(name="copy_fork", kind="copy", layers=48, pages=64, pairs=1, hkv=4, dim=128, page=16, dtype="bf16"),
        # a pool is compacted, or 32 sequences get pages of their own
        dict(name="copy_many", kind="copy", layers=48, pages=401, pairs=131, hkv=4, dim=128, page=16, dtype="bf16"),
        # one sequence takes over the drafts it accepted
        dict(name="accept_step", kind="accept", layers=48, requests=1, drafts=16, most=5, hkv=4, dim=128, page=16, dtype="bf16", lens=9),
        # a batch of trees, up to ten accepted each
        dict(name="accept_batch", kind="accept", layers=48, requests=64, drafts=31, most=10, hkv=4, dim=128, page=16, dtype="bf16", lens=10),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rope", "sliding", "sliding", "tree", "tree", "copy", "accept"])
    hq, hkv = rng.choice(HEADS)
    c = dict(kind=kind, hkv=hkv, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64]), dtype=rng.choice(["bf16", "fp16"]))
    if kind == "rope":
        c.update(tokens=_spread(rng, 1, 2800), hq=hq, rot=rng.choice([32, 64]), pairs=rng.choice(["halves", "neighbours"]),
                 past=rng.randrange(0, 5000), lens=rng.randrange(1 << 30))
    elif kind == "sliding":
        rows = rng.choice([1, 1, _spread(rng, 2, 600)])
        lo = _spread(rng, 1, 4000)
        c.update(requests=_spread(rng, 1, 100 if rows == 1 else 8), rows=rows, past_lo=lo, past_hi=lo + _spread(rng, 1, 4000), hq=hq,
                 window=_spread(rng, 1, 4096), sinks=rng.choice([0, 1, 4, rng.randrange(2, 300)]), lens=rng.randrange(1 << 30))
    elif kind == "tree":
        lo = _spread(rng, 1, 8000)
        c.update(requests=_spread(rng, 1, 24), rows=_spread(rng, 1, 64), past_lo=lo, past_hi=lo + _spread(rng, 1, 8000), hq=hq, lens=rng.randrange(1 << 30))
    elif kind == "copy":
        pairs = _spread(rng, 1, 100)
        c.update(layers=rng.randrange(2, 49), pages=2 * pairs + rng.randrange(1, 60), pairs=pairs)
    else:
        most = rng.randrange(1, 12)
        c.update(layers=rng.randrange(2, 49), requests=_spread(rng, 1, 64), drafts=2 * most + rng.randrange(0, 40), most=most, lens=rng.randrange(1 << 30))
    return c


# ------------------------------------------------------------------------------------------------ lengths and inputs

def _lengths(case):
    """(rows, keys) of each request: rows are ragged where there is more than one, keys are the past and the rows."""
    rng = random.Random(case["lens"])
    most = case["rows"]
    rows = [most if most == 1 else rng.randint(max(1, most // 2), most) for _ in range(case["requests"])]
    return rows, [rng.randint(case["past_lo"], case["past_hi"]) + n for n in rows]


def _counts(case):
    """How many drafts each request accepts."""
    return [1 + (7 * r) % case["most"] for r in range(case["requests"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) + 1)


def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _table(g, need):
    """A block table int32 [requests][most pages] of shuffled pages; page 0 is no sequence's. Also the number of pages."""
    n = sum(need) + 1
    order = torch.randperm(n - 1, generator=g, device="cuda").to(torch.int32) + 1
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = order[at:at + k]
        at += k
    return table, n


def _tree(rng, rows):
    """Which drafted tokens each drafted token sees, as int32 words of 32: itself and its ancestors in a random tree."""
    words = -(-max(rows) // 32)
    bits = []
    for n in rows:
        seen = []
        for i in range(n):
            parent = rng.randrange(max(0, i - 6), i) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        bits += seen
    word = [[(b >> 32 * w) & 0xffffffff for w in range(words)] for b in bits]
    return torch.tensor([[v - (1 << 32) if v >> 31 else v for v in row] for row in word], dtype=torch.int32)


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(int(seed))
    dtype, dim, page, hkv = DTYPES[case["dtype"]], case["dim"], case["page"], case["hkv"]
    s = dict(case=case)
    if case["kind"] == "rope":
        T, hq = case["tokens"], case["hq"]
        where = random.Random(case["lens"])
        n_pages = -(-T // page) + 3
        s["qkv"] = _normal(g, dtype, T, (hq + 2 * hkv) * dim)
        s["k_cache"], s["v_cache"] = (torch.zeros(n_pages, page, hkv, dim, dtype=dtype, device="cuda") for _ in range(2))
        s["slots"] = torch.randperm((n_pages - 1) * page, generator=g, device="cuda")[:T].to(torch.int32) + page
        most = case["past"] + T
        s["positions"] = torch.tensor([where.randrange(most) for _ in range(T)] if case["past"] else [i % 2048 for i in range(T)],
                                      dtype=torch.int32, device="cuda")
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-2 * torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) / case["rot"])
        s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        s["q_norm"], s["k_norm"] = (_normal(g, dtype, dim) * 0.1 + 1 for _ in range(2))
        return s
    if case["kind"] in ("sliding", "tree"):
        rows, keys = _lengths(case)
        s["block_table"], n_pages = _table(g, [-(-k // page) for k in keys])
        s["q"] = _normal(g, dtype, sum(rows), case["hq"], dim)
        s["k_cache"], s["v_cache"] = (_normal(g, dtype, n_pages, page, hkv, dim) for _ in range(2))
        s["q_start"] = torch.tensor([sum(rows[:r]) for r in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
        s["kv_len"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
        s["most_rows"], s["most_keys"] = max(rows), max(keys)
        if case["kind"] == "tree":
            s["tree"] = _tree(rng, rows).cuda()
        return s
    L = case["layers"]
    if case["kind"] == "copy":
        n_pages = case["pages"]
        order = torch.randperm(n_pages - 1, generator=g, device="cuda").to(torch.int32) + 1
        s["src"], s["dst"] = order[:case["pairs"]].contiguous(), order[case["pairs"]:2 * case["pairs"]].contiguous()
    else:
        R, n, counts = case["requests"], case["drafts"], _counts(case)
        where = random.Random(case["lens"])
        past = [where.randrange(1, 4 * page) for _ in range(R)]
        s["block_table"], n_pages = _table(g, [-(-(p + n) // page) for p in past])
        s["base"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        # the first draft is the root and stays; the others lie behind the places that are taken
        paths = [[0] + sorted(rng.sample(range(c, n), c - 1)) + [0] * (case["most"] - c) for c in counts]
        s["path"], s["count"] = torch.tensor(paths, dtype=torch.int32, device="cuda"), torch.tensor(counts, dtype=torch.int32, device="cuda")
    s["k"], s["v"] = (_normal(g, dtype, L, n_pages, page, hkv, dim) for _ in range(2))
    if own:   # what a program makes once for its cache
        from monoserve_b200.cache import CachePages
        s["pages"] = CachePages(list(s["k"]) + list(s["v"]))
    return s


# -------------------------------------------------------------------------------------------------------- plain form

def _rope_plain(s):
    c, qkv = s["case"], s["qkv"]
    hq, hkv, dim, rot = c["hq"], c["hkv"], c["dim"], c["rot"]
    x = qkv.float().view(-1, hq + 2 * hkv, dim)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    w = torch.cat([s["q_norm"].float().expand(hq, dim), s["k_norm"].float().expand(hkv, dim)])
    y = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    cs = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin, turned = cs[..., 0], cs[..., 1], y[..., :rot]
    if c["pairs"] == "halves":
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    y = torch.cat([turned, y[..., rot:]], -1).to(qkv.dtype)
    slots = s["slots"].long()
    s["k_cache"].view(-1, hkv, dim)[slots] = y[:, hq:]
    s["v_cache"].view(-1, hkv, dim)[slots] = v.to(qkv.dtype)
    return dict(q=y[:, :hq].contiguous(), k_cache=s["k_cache"], v_cache=s["v_cache"])


def _padded(s, most):
    """q in a batch [requests][most rows], which of its rows there are, and their positions."""
    start, keys = s["q_start"].long(), s["kv_len"].long()
    i = torch.arange(most, device="cuda")
    there = i < (start[1:] - start[:-1])[:, None]
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    return row, there, (keys - (start[1:] - start[:-1]))[:, None] + i


def _gather(s, at):
    """Rows [requests][n] of K and V, 32 bits, at positions `at` of each request."""
    page = s["case"]["page"]
    slot = s["block_table"].gather(1, at // page).long() * page + at % page
    return s["k_cache"].flatten(0, 1)[slot].float(), s["v_cache"].flatten(0, 1)[slot].float()


def _attend_plain(s, row, there, k, v, mask):
    """softmax of the masked scores times v, rows without a visible key zero. mask: [requests][rows][keys]."""
    c, q = s["case"], s["q"]
    R, m = row.shape
    hq, hkv, dim = c["hq"], c["hkv"], c["dim"]
    x = q[row].float().view(R, m, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(R, hkv, -1, dim)
    scores = (x @ k.permute(0, 2, 3, 1)) * dim ** -0.5
    scores = scores.view(R, hkv, hq // hkv, m, -1).masked_fill(~mask[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0, top)).exp()
    total = p.sum(-1, keepdim=True)
    o = p.flatten(2, 3) @ v.permute(0, 2, 1, 3)
    o = o.view(R, hkv, hq // hkv, m, dim) / torch.where(total == 0, 1, total)
    out = torch.empty_like(q)
    out[row[there]] = o.permute(0, 3, 1, 2, 4).reshape(R, m, hq, dim)[there].to(q.dtype)
    return out


def _sliding_plain(s):
    c = s["case"]
    row, there, pos = _padded(s, s["most_rows"])
    keys, window, sinks = s["kv_len"].long(), c["window"], c["sinks"]
    span = torch.arange(min(window - 1 + s["most_rows"], s["most_keys"]), device="cuda")
    first = (pos[:, :1] - window + 1).clamp(min=0)
    near, far = first + span, torch.arange(sinks, device="cuda").expand(len(keys), sinks)
    at = torch.cat([far, near], 1)
    seen = (at[:, None] <= pos[..., None]) & (at < keys[:, None])[:, None]
    inside = at[:, None] > pos[..., None] - window
    inside[..., :sinks] = ~inside[..., :sinks]   # a sink inside the window is counted there
    k, v = _gather(s, at.clamp(max=s["block_table"].shape[1] * c["page"] - 1))
    return _attend_plain(s, row, there, k, v, seen & inside)


def _tree_plain(s):
    row, there, pos = _padded(s, s["most_rows"])
    at = torch.arange(s["most_keys"], device="cuda").expand(len(pos), -1)
    draft = at - pos[:, :1]
    n = 32 * s["tree"].shape[1]
    word = s["tree"].long()[row].gather(2, (draft.clamp(0, n - 1) // 32)[:, None].expand(-1, row.shape[1], -1))
    bit = (word >> (draft.clamp(0, n - 1) % 32)[:, None]) & 1
    rows = s["kv_len"][:, None].long() - pos[:, :1]
    mask = (draft < 0)[:, None] | ((draft >= 0) & (draft < rows))[:, None] & (bit > 0)
    return _attend_plain(s, row, there, *_gather(s, at), mask)


def _accept_plain(s):
    page, most = s["case"]["page"], s["path"].shape[1]
    i = torch.arange(most, device="cuda")
    taken = i < s["count"][:, None]

    def slot(at):
        at = at.long()
        return torch.where(taken, s["block_table"].gather(1, at // page).long() * page + at % page, 0)

    src, dst = slot(s["base"][:, None] + s["path"]).flatten(), slot(torch.where(taken, s["base"][:, None] + i, 0)).flatten()
    k, v = s["k"].flatten(1, 2), s["v"].flatten(1, 2)
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return dict(k=s["k"], v=s["v"])


def _copy_plain(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    return dict(k=s["k"], v=s["v"])


# ------------------------------------------------------------------------------------------------------- both of them

def _run_own(s):
    c = s["case"]
    if c["kind"] == "rope":
        from monoserve_b200.cache import qk_rope
        q = qk_rope(s["qkv"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["cos_sin"], c["hq"], q_norm=s["q_norm"],
                    k_norm=s["k_norm"], eps=EPS, interleaved=c["pairs"] == "neighbours")
        return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    if c["kind"] == "sliding":
        from monoserve_b200.attention import sliding_attention
        return sliding_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["q_start"], s["kv_len"], c["window"], sinks=c["sinks"])
    if c["kind"] == "tree":
        from monoserve_b200.attention import tree_attention
        return tree_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["q_start"], s["kv_len"], s["tree"])
    if c["kind"] == "copy":
        s["pages"].copy(s["src"], s["dst"])
    else:
        s["pages"].accept(s["block_table"], s["base"], s["path"], s["count"])
    return dict(k=s["k"], v=s["v"])


def run(state):
    if own:
        return _run_own(state)
    plain = dict(rope=_rope_plain, sliding=_sliding_plain, tree=_tree_plain, copy=_copy_plain, accept=_accept_plain)
    return plain[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------- the floor

def _visible(case, n, L):
    """(keys that any row of a request sees, pairs of a row and a key it sees); of a tree, past and one chain of drafts as long as
    its rows' numbers at most."""
    if case["kind"] == "tree":
        return L, n * (L - n) + n * (n + 1) // 2
    w, z, p0 = case["window"], case["sinks"], L - n
    lo = max(0, p0 - w + 1)
    seen = L - lo + min(z, lo)
    # rows p0 .. L - 1: keys inside the window, and the sinks in front of it
    below = max(0, min(L, w) - p0)   # rows that see every key up to themselves
    a = sum_to(p0 + below) - sum_to(p0) + (n - below) * w
    front = sum(min(z, max(0, p - w + 1)) for p in range(p0, L))
    return seen, a + front


def sum_to(n):
    return n * (n + 1) // 2


def work(case):
    size = 2
    if case["kind"] == "rope":
        values = case["tokens"] * (case["hq"] + 2 * case["hkv"]) * case["dim"]
        distinct = min(case["tokens"], case["past"] + case["tokens"] if case["past"] else 2048)
        return dict(bytes=2 * size * values + distinct * case["rot"] * 4 + 8 * case["tokens"], flops=8 * values)
    if case["kind"] in ("sliding", "tree"):
        rows, keys = _lengths(case)
        per = [_visible(case, n, L) for n, L in zip(rows, keys)]
        io = 2 * sum(rows) * case["hq"] * case["dim"] * size
        return dict(bytes=io + 2 * sum(k for k, _ in per) * case["hkv"] * case["dim"] * size,
                    flops=4 * case["dim"] * case["hq"] * sum(p for _, p in per))
    row = case["hkv"] * case["dim"] * size
    if case["kind"] == "copy":
        return dict(bytes=2 * 2 * case["layers"] * case["pairs"] * case["page"] * row, flops=0)
    moved = sum(c - 1 for c in _counts(case))
    return dict(bytes=2 * 2 * case["layers"] * max(1, moved) * row, flops=0)


# ------------------------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("copy", "accept"):   # moved, not computed
        if case["kind"] == "copy":
            moves = list(zip(s["src"].tolist(), s["dst"].tolist()))
        else:
            page, table, moves = case["page"], s["block_table"].tolist(), []
            for r, (p, path, c) in enumerate(zip(s["base"].tolist(), s["path"].tolist(), s["count"].tolist())):
                for i in range(c):
                    moves.append(tuple((table[r][at // page], at % page) for at in (p + path[i], p + i)))
        old, new = (s["k"], s["v"]), (s["k"].double(), s["v"].double())
        for a, b in moves:
            for x, y in zip(old, new):
                y[(slice(None), *b) if isinstance(b, tuple) else (slice(None), b)] = x[(slice(None), *a) if isinstance(a, tuple) else (slice(None), a)].double()
        return dict(k=new[0], v=new[1])
    hq, hkv, dim, page = case.get("hq"), case["hkv"], case["dim"], case["page"]
    if case["kind"] == "rope":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, dim)
        rot, half = case["rot"], case["rot"] // 2
        first = torch.arange(half, device="cuda") if case["pairs"] == "halves" else 2 * torch.arange(half, device="cuda")
        second = first + (half if case["pairs"] == "halves" else 1)
        z = torch.complex(*s["cos_sin"][s["positions"].long()].double().unbind(-1))[:, None]

        def turn(h, w):
            h = h / (h.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            t = torch.complex(h[..., first], h[..., second]) * z
            h[..., first], h[..., second] = t.real, t.imag
            return h

        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        page_of, offset = s["slots"].long() // page, s["slots"].long() % page
        k_cache[page_of, offset] = turn(x[:, hq:hq + hkv], s["k_norm"])
        v_cache[page_of, offset] = x[:, hq + hkv:]
        return dict(q=turn(x[:, :hq], s["q_norm"]), k_cache=k_cache, v_cache=v_cache)
    rows, keys = _lengths(case)
    out = torch.zeros(sum(rows), hq, dim, dtype=torch.float64, device="cuda")
    at = 0
    for r, (n, L) in enumerate(zip(rows, keys)):
        pages = s["block_table"][r, :-(-L // page)].long()
        k, v = (t[pages].reshape(-1, hkv, dim)[:L].double() for t in (s["k_cache"], s["v_cache"]))
        key, p = torch.arange(L, device="cuda"), torch.arange(L - n, L, device="cuda")[:, None]
        if case["kind"] == "sliding":
            sees = (key <= p) & ((p - key < case["window"]) | (key < case["sinks"]))
        else:
            sees = torch.ones(n, L, dtype=torch.bool, device="cuda")
            j = torch.arange(n, device="cuda")
            sees[:, L - n:] = (s["tree"][at:at + n].long()[:, j // 32] >> (j % 32)) % 2 == 1
        for h in range(hq):
            e = torch.where(sees, s["q"][at:at + n, h].double() @ k[:, h * hkv // hq].T / math.sqrt(dim), -math.inf)
            e = torch.exp(e - e.max(-1, keepdim=True).values.clamp(min=-1e300))
            out[at:at + n, h] = e @ v[:, h * hkv // hq] / e.sum(-1, keepdim=True)
        at += n
    return out
