"""Performance cases of the KV-cache operators: attention of drafted trees, eviction by attention weight, attention over chosen blocks.

Kinds of cases:
  tree    attention of `rows` drafted tokens per sequence (a tree given as ancestor masks) over the cache; rows = 1 is plain decoding
  verify  a speculative step: rotation and append of the drafted tokens, their attention, the accepted path moved to its place
  weigh   the rows' attention weights added to the cache's book
  evict   caches pruned to `keep` entries each, into other caches
  step    decoding under a budget: append, attention, weights, and eviction in place back to `keep` entries
  blocks  block means brought up to date, then attention over the `nsel` blocks that each row scores highest
"""
import math
import random

import torch

own = False

ENGINE_CAP = 4096          # positions of one of the engines' caches
FIRST, RECENT = 4, 32      # entries that an eviction never takes: the first ones and the latest


def listed():
    oss, qwen = {"heads": 64, "kv": 8, "dim": 64}, {"heads": 32, "kv": 4, "dim": 128}
    return [
        # one token of one conversation, the engine's own shape: latency alone
        {"name": "tree 1x1 f32 73", "kind": "tree", "n": 1, "rows": 1, "ctx": 73, **oss, "bf16": False, "window": 0},
        # a short draft in a sliding-window layer
        {"name": "tree 1x8 f32 1900 window", "kind": "tree", "n": 1, "rows": 8, "ctx": 1900, **oss, "bf16": False, "window": 128},
        # a draft tree of the second engine late in a long conversation
        {"name": "tree 1x26 f32 3700", "kind": "tree", "n": 1, "rows": 26, "ctx": 3700, **qwen, "bf16": False, "window": 0},
        # a loaded server, every sequence with the widest tree; the half-size cache
        {"name": "tree 16x64 bf16 2000", "kind": "tree", "n": 16, "rows": 64, "ctx": 2000, **oss, "bf16": True, "window": 0},
        # a lightly loaded server's whole speculative step
        {"name": "verify 5x13 f32 1211", "kind": "verify", "n": 5, "rows": 13, "ctx": 1211, **oss, "bf16": False, "window": 0},
        # one new token of each of many sequences counted into the book
        {"name": "weigh 24x1 f32 3801", "kind": "weigh", "n": 24, "rows": 1, "ctx": 3801, **oss, "bf16": False, "window": 0},
        # accepted rows of wider drafts
        {"name": "weigh 7x37 bf16 2500", "kind": "weigh", "n": 7, "rows": 37, "ctx": 2500, **qwen, "bf16": True, "window": 0},
        # one full cache pruned to a quarter
        {"name": "evict 1 f32 4096 to 1024", "kind": "evict", "n": 1, "rows": 0, "ctx": 4096, "keep": 1024, **oss, "bf16": False},
        # a server's sweep over its sequences, ragged, some of them shorter than the budget
        {"name": "evict 32 bf16 3900 to 2001", "kind": "evict", "n": 32, "rows": 0, "ctx": 3900, "keep": 2001, **qwen, "bf16": True},
        # steady decoding of sequences that stand at their budget
        {"name": "step 12 f32 1023", "kind": "step", "n": 12, "rows": 1, "ctx": 1023, "keep": 1023, **oss, "bf16": False},
        # one token over a long document
        {"name": "blocks 1 bf16 61000", "kind": "blocks", "n": 1, "rows": 1, "ctx": 61000, "block": 64, "nsel": 32, **qwen, "bf16": True},
        # a piece of a prompt: every row chooses for itself
        {"name": "blocks 1x201 f32 9001", "kind": "blocks", "n": 1, "rows": 201, "ctx": 9001, "block": 32, "nsel": 24, **oss, "bf16": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "weigh", "evict", "step", "blocks", "blocks"])
    heads, kv, dim = rng.choice([(64, 8, 64), (32, 4, 128), (8, 2, 64), (20, 4, 128), (6, 6, 64), (32, 2, 128)])
    c = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "bf16": rng.random() < 0.5}
    if kind in ("tree", "verify", "weigh"):
        n, rows = _log(rng, 1, 16), _log(rng, 1, 64)
        most = min(4000, 16 * 64 * 2000 * 64 * 64 // (n * rows * heads * dim), 1100_000_000 // (n * kv * dim * 8))
        return {**c, "n": n, "rows": rows, "ctx": _log(rng, 1, max(2, most)), "window": rng.choice([0, 0, 128, 37]) if dim == 64 else 0}
    if kind == "evict":
        n, ctx = _log(rng, 1, 32), _log(rng, 100, 4000)
        return {**c, "n": n, "rows": 0, "ctx": ctx, "keep": rng.randint(FIRST + RECENT + 1, ctx)}
    if kind == "step":
        ctx = _log(rng, 64, 3000)
        return {**c, "n": _log(rng, 1, 24), "rows": 1, "ctx": ctx, "keep": ctx}
    block, nsel = rng.choice([16, 32, 64, 128]), rng.randint(3, 32)
    if rng.random() < 0.5:          # decoding: a row per sequence
        n = _log(rng, 1, 16)
        return {**c, "n": n, "rows": 1, "ctx": _log(rng, 1, min(60000, 800_000 // (n * kv) * 128 // dim)), "block": block, "nsel": nsel}
    rows = _log(rng, 2, 200)
    return {**c, "n": 1, "rows": rows, "ctx": rows + _log(rng, 1, 9000), "block": block, "nsel": min(nsel, 24 * 32 // block + 2)}


def _lens(case):
    """Cached entries of each sequence before the call: the first has `ctx`, the others half of it and more."""
    r = random.Random(case["ctx"] * 1000 + case["n"])
    if case["kind"] == "step":
        return [case["ctx"]] * case["n"]
    return [case["ctx"]] + [r.randint((case["ctx"] + 1) // 2, case["ctx"]) for _ in range(case["n"] - 1)]


def _trees(case):
    """Parents of each sequence's drafted tokens (-1: follows the cached ones) and how many it has; the first has them all."""
    r = random.Random(case["rows"] * 100 + case["n"])
    rows = case["rows"]
    counts = [rows] + [r.randint((rows + 1) // 2, rows) for _ in range(case["n"] - 1)]
    parents = [[-1 if i == 0 else max(-1, i - 1 - int(r.expovariate(0.7))) for i in range(rows)] for _ in counts]
    return parents, counts


def _masks(parents):
    out = []
    for p in parents:
        m = []
        for i, j in enumerate(p):
            m.append((1 << i) | (m[j] if j >= 0 else 0))
        out.append(m)
    return out


def _cap(case):
    need = case["ctx"] + case["rows"] + 1
    return ENGINE_CAP if need <= ENGINE_CAP else (need + 63) // 64 * 64


class _State:
    kv = dst = None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    s = _State()
    s.case, n, rows, kind = case, case["n"], case["rows"], case["kind"]
    H, kvh, hd, cap = case["heads"], case["kv"], case["dim"], _cap(case)
    kind_t = torch.bfloat16 if case["bf16"] else torch.float32

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def ints(v, t=torch.int32):
        return torch.tensor(v, dtype=t, device=dev)

    s.scale, s.cap = 1.0 / math.sqrt(hd), cap
    lens = _lens(case)
    s.len = ints(lens)
    s.k = torch.empty((n, kvh, cap, hd), dtype=kind_t, device=dev).normal_(generator=g)
    s.v = torch.empty((n, kvh, cap, hd), dtype=kind_t, device=dev).normal_(generator=g)
    s.k[..., ::8] *= 3          # a few strong dimensions, as keys have
    s.weight = randn(n, kvh, cap).mul_(1.5).exp_()
    s.pos = torch.arange(cap, device=dev, dtype=torch.int32).repeat(n, kvh, 1)
    s.sinks = randn(H) if hd == 64 else None
    if kind == "evict":
        # the positions that earlier evictions left, in no order
        s.pos = torch.argsort(torch.rand((n, kvh, cap), generator=g, device=dev), dim=-1).to(torch.int32)
        s.end, m = ints([cap] * n), min(case["keep"], cap)
        s.k2, s.v2 = torch.zeros((n, kvh, m, hd), dtype=kind_t, device=dev), torch.zeros((n, kvh, m, hd), dtype=kind_t, device=dev)
        s.weight2, s.pos2 = torch.zeros((n, kvh, m), device=dev), torch.zeros((n, kvh, m), dtype=torch.int32, device=dev)
        s.map, s.new_len = torch.zeros((n, kvh, m), dtype=torch.int32, device=dev), ints([0] * n)
        return s
    if kind == "blocks":
        # one row per sequence, or the last `rows` positions of one sequence
        R, nb = (n if rows == 1 else rows), cap // case["block"]
        s.seq = ints(list(range(n)) if rows == 1 else [0] * rows)
        s.lens = s.len.clone() if rows == 1 else ints([case["ctx"] - rows + i + 1 for i in range(rows)])
        s.since = s.len - rows
        blocks = s.k[:, :, : nb * case["block"]].reshape(n, kvh, nb, case["block"], hd)
        s.means = blocks.double().mean(3).float()
        s.q = randn(R, H * hd)
        s.sel = torch.zeros((R, kvh, case["nsel"]), dtype=torch.int32, device=dev)
        s.out, s.lse = torch.zeros((R, H * hd), device=dev), torch.zeros((R, H), device=dev)
        return s
    parents, counts = _trees(case)
    masks = _masks(parents)
    s.count = ints(counts) if n > 1 else None
    s.mask = ints([[m - (1 << 64) if m >> 63 else m for m in row] for row in masks], torch.int64) if rows > 1 else None
    s.rows = None
    s.q = randn(n, rows, H * hd)
    s.out, s.lse = torch.zeros((n, rows, H * hd), device=dev), torch.zeros((n, rows, H), device=dev)
    if kind in ("verify", "step"):
        s.qkv = randn(n, rows, (H + 2 * kvh) * hd)
        s.at = ints([[ln + bin(m).count("1") - 1 for m in row] for ln, row in zip(lens, masks)])
        angle = torch.arange(ENGINE_CAP, device=dev, dtype=torch.float64)[:, None] * 150000.0 ** (-torch.arange(hd // 2, device=dev, dtype=torch.float64) / (hd // 2))
        s.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    if kind == "verify":
        # the accepted path: from a node drawn at random back to its root
        picks = torch.rand(n, generator=g, device=dev).tolist()
        paths = []
        for p, c, u in zip(parents, counts, picks):
            i, path = int(u * c), []
            while i >= 0:
                path.append(i)
                i = p[i]
            paths.append(path[::-1])
        s.path, s.npath, s.new_len = ints([p + [-1] * (rows - len(p)) for p in paths]), ints([len(p) for p in paths]), ints([0] * n)
    if kind == "weigh":
        s.lse = _attend(s.q.view(n, rows, kvh, -1, hd), *_cached(s, cap), _visible(s, cap), s.scale, s.sinks)[1].reshape(n, rows, H)
        s.rows = torch.randint(1, 1 << 62, (n,), generator=g, device=dev) if rows > 1 else None     # the accepted rows
    if kind == "step":
        s.end = ints([ln + 1 for ln in lens])
        s.full = s.len + 1
        s.map, s.new_len = torch.zeros((n, kvh, case["keep"]), dtype=torch.int32, device=dev), ints([0] * n)
    return s


# ---------------------------------------------------------------- the operators in their plain form
def _cached(s, width):
    return s.k[:, :, :width].float(), s.v[:, :, :width].float()


def _count(s):
    return s.count if s.count is not None else torch.full_like(s.len, s.case["rows"])


def _bits(s):
    """[sequence][row][node]: whether the row sees the node."""
    rows = s.case["rows"]
    j = torch.arange(rows, device=s.len.device)
    bits = (j[None, :] <= j[:, None]).expand(len(s.len), rows, rows) if s.mask is None else ((s.mask[:, :, None] >> j) & 1).bool()
    return bits & (j < _count(s)[:, None])[:, None, :]


def _visible(s, width):
    """[sequence][row][slot]"""
    rows, window = s.case["rows"], s.case.get("window", 0)
    j, t = torch.arange(rows, device=s.len.device), torch.arange(width, device=s.len.device)
    bits, length = _bits(s), s.len[:, None, None].long()
    depth = (bits & (j[:, None] != j)).sum(-1)
    node = t - length                                            # [n][1][width]
    inside = (node >= 0) & (node < rows)
    drafted = torch.gather(bits, 2, node.clamp(0, rows - 1).expand(-1, rows, -1)) & inside
    seen = (node < 0) | drafted
    if window:
        of_node = torch.gather(depth, 1, node[:, 0].clamp(0, rows - 1))[:, None, :]
        seen &= torch.where(node < 0, depth[:, :, None] - node < window, depth[:, :, None] - of_node < window)
    return seen


def _scores(q, k, seen, scale):
    """[n][kv][rows][g][width], -inf where nothing is seen"""
    n, rows, kvh, per, hd = q.shape
    s = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(n, kvh, rows * per, hd), k.transpose(2, 3)).mul_(scale).view(n, kvh, rows, per, -1)
    return s.masked_fill_(~seen[:, None, :, None, :], -math.inf)


def _attend(q, k, v, seen, scale, sinks):
    """q [n][rows][kv][g][dim], k and v [n][kv][width][dim], seen [n][rows][width] -> out as q, lse [n][rows][kv][g]"""
    n, rows, kvh, per, hd = q.shape
    s = _scores(q, k, seen, scale)
    top = s.amax(-1)
    if sinks is not None:
        sink = sinks.view(kvh, 1, per)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top[..., None]).exp_()
    total = p.sum(-1)
    if sinks is not None:
        total = total + (sink - top).exp()
    out = torch.matmul(p.view(n, kvh, rows * per, -1), v).view(n, kvh, rows, per, hd)
    out = out / torch.where(total == 0, torch.ones_like(total), total)[..., None]
    return out.permute(0, 2, 1, 3, 4), (top + total.log()).permute(0, 2, 1, 3)


def _plain_append(s):
    case = s.case
    n, rows, H, kvh, hd = case["n"], case["rows"], case["heads"], case["kv"], case["dim"]
    x = s.qkv.view(n, rows, H + 2 * kvh, hd)
    cos, sin = s.rope[s.at.long()].unbind(-1)
    cos, sin, a, b = cos[:, :, None], sin[:, :, None], x[:, :, : H + kvh, : hd // 2], x[:, :, : H + kvh, hd // 2 :]
    turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    i = torch.arange(rows, device=x.device)
    live = i < _count(s)[:, None]
    at_seq, at_row = live.nonzero(as_tuple=True)
    slot = (s.len[:, None] + i)[live].long()
    s.q.view(n, rows, H, hd)[at_seq, at_row] = turned[at_seq, at_row, :H]
    s.k[at_seq, :, slot] = turned[at_seq, at_row, H:].to(s.k.dtype)
    s.v[at_seq, :, slot] = x[at_seq, at_row, H + kvh :].to(s.v.dtype)
    s.weight[at_seq, :, slot] = 0.0
    s.pos[at_seq, :, slot] = s.at[live][:, None].expand(-1, kvh)


def _plain_tree(s):
    case = s.case
    n, rows, kvh, hd = case["n"], case["rows"], case["kv"], case["dim"]
    width = min(s.cap, case["ctx"] + rows)
    out, lse = _attend(s.q.view(n, rows, kvh, -1, hd), *_cached(s, width), _visible(s, width), s.scale, s.sinks)
    live = (torch.arange(rows, device=out.device) < _count(s)[:, None])[:, :, None]
    s.out.copy_(torch.where(live, out.reshape(n, rows, -1), s.out))
    s.lse.copy_(torch.where(live, lse.reshape(n, rows, -1), s.lse))


def _plain_commit(s):
    rows = s.case["rows"]
    i = torch.arange(rows, device=s.len.device)
    live = i < s.npath[:, None]
    at_seq, _ = live.nonzero(as_tuple=True)
    src, dst = (s.len[:, None] + s.path)[live].long(), (s.len[:, None] + i)[live].long()
    for book in (s.k, s.v, s.weight, s.pos):
        book[at_seq, :, dst] = book[at_seq, :, src]
    s.new_len.copy_(s.len + s.npath)


def _plain_weigh(s):
    case = s.case
    n, rows, kvh, hd = case["n"], case["rows"], case["kv"], case["dim"]
    width = min(s.cap, case["ctx"] + rows)
    i = torch.arange(rows, device=s.len.device)
    live = i < _count(s)[:, None]
    if s.rows is not None:
        live = live & ((s.rows[:, None] >> i) & 1).bool()
    x = _scores(s.q.view(n, rows, kvh, -1, hd), s.k[:, :, :width].float(), _visible(s, width) & live[:, :, None], s.scale)
    x.sub_(torch.where(live[:, :, None], s.lse, torch.zeros_like(s.lse)).view(n, rows, kvh, -1).permute(0, 2, 1, 3)[..., None]).exp_()
    s.weight[:, :, :width] += x.sum((2, 3))


def _plain_evict(s, length, keep, k, v, weight, pos):
    """The caches k, v with their books become, or with others given are copied to, those of the kept entries."""
    n, kvh = s.weight.shape[:2]
    width = s.case["ctx"] + s.case["rows"]
    t = torch.arange(width, device=length.device)
    inside = (t < length[:, None])[:, None]
    at, w = s.pos[:, :, :width], s.weight[:, :, :width]
    safe = (at < FIRST) | (at >= (s.end - RECENT)[:, None, None])
    key = torch.where(inside, torch.where(safe, torch.full_like(w, math.inf), w), torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    m = torch.clamp(length, max=keep)[:, None, None]
    kept = torch.zeros((n, kvh, width), dtype=torch.bool, device=t.device).scatter_(2, order, (t < m).expand(n, kvh, -1))
    beyond = torch.where(kept & (t >= m), t, torch.full_like(t, width)).sort(-1).values
    hole = ~kept & (t < m)
    nth = (hole.cumsum(-1) - 1).clamp(min=0)
    source = torch.where(hole, torch.gather(beyond, 2, nth), t)[:, :, :keep]
    live = t[:keep] < m
    s.map.copy_(torch.where(live, source, torch.full_like(source, -1)))
    s.new_len.copy_(m[:, 0, 0])
    a, b, d = live.expand(n, kvh, -1).nonzero(as_tuple=True)
    src = source[a, b, d]
    k[a, b, d], v[a, b, d] = s.k[a, b, src], s.v[a, b, src]
    weight[a, b, d], pos[a, b, d] = s.weight[a, b, src], s.pos[a, b, src]


def _plain_means(s):
    case = s.case
    n, kvh, hd, block = case["n"], case["kv"], case["dim"], case["block"]
    lo = (case["ctx"] - case["rows"]) // block if n == 1 else 0
    hi = case["ctx"] // block
    if hi <= lo:
        return
    b = torch.arange(lo, hi, device=s.len.device)
    due = (b >= (s.since // block)[:, None]) & (b < (s.len // block)[:, None])
    if n == 1:
        s.means[:, :, lo:hi] = s.k[:, :, lo * block : hi * block].view(n, kvh, -1, block, hd).double().mean(3).float()
        return
    a, b = due.nonzero(as_tuple=True)
    b = b + lo
    t = b[:, None] * block + torch.arange(block, device=b.device)
    s.means[a, :, b] = s.k[a[:, None], :, t].double().mean(1).float()


def _plain_blocks(s):
    case = s.case
    kvh, hd, block, nsel = case["kv"], case["dim"], case["block"], case["nsel"]
    R, seq = len(s.seq), s.seq.long()
    nb = -(-case["ctx"] // block)
    q = s.q.view(R, kvh, -1, hd)
    full = min(nb, s.means.shape[2])
    score = torch.full((R, kvh, nb), -math.inf, device=q.device)
    if len(s.len) == 1:         # every row scores the same means
        x = torch.matmul(q.double().transpose(0, 1).reshape(1, kvh, -1, hd), s.means[:, :, :full].double().transpose(2, 3))
        score[:, :, :full] = x.view(kvh, R, -1, full).amax(2).transpose(0, 1).float()
    else:
        score[:, :, :full] = torch.matmul(q.double(), s.means[seq, :, :full].double().transpose(2, 3)).amax(2).float()
    j = torch.arange(nb, device=q.device)
    have = (-(-s.lens // block))[:, None, None]
    score = torch.where((j < 1) | (j >= have - 2), torch.full_like(score, math.inf), score)
    score = torch.where(j < have, score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :, :nsel]
    sel = torch.where(order < have, order, torch.full_like(order, nb)).sort(-1).values
    s.sel.fill_(-1)
    s.sel[:, :, : sel.shape[2]] = torch.where(sel < nb, sel, torch.full_like(sel, -1))
    t = (sel[..., None] * block + torch.arange(block, device=q.device)).view(R, kvh, -1)
    seen = t < s.lens[:, None, None]
    t = t.clamp(max=case["ctx"] - 1)
    head = torch.arange(kvh, device=q.device)[:, None]
    k, v = s.k[seq[:, None, None], head, t].float(), s.v[seq[:, None, None], head, t].float()
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s.scale).masked_fill_(~seen[:, :, None], -math.inf)
    top = x.amax(-1)
    if s.sinks is not None:
        top = torch.maximum(top, s.sinks.view(kvh, -1))
    p = x.sub_(top[..., None]).exp_()
    total = p.sum(-1)
    if s.sinks is not None:
        total = total + (s.sinks.view(kvh, -1) - top).exp()
    s.out.copy_((torch.matmul(p, v) / total[..., None]).view(R, -1))
    s.lse.copy_((top + total.log()).view(R, -1))


# ---------------------------------------------------------------- a pass
def run(s):
    case, kind = s.case, s.case["kind"]
    n, rows, H, keep = case["n"], case["rows"], case["heads"], case.get("keep")
    if own:
        import cpubrrr_b200 as B
        if s.kv is None:
            s.kv = B.KvCache(s.k, s.v, n, case["kv"], case["dim"], s.cap, bf16=case["bf16"], weight=s.weight, pos=s.pos)
            if kind == "evict":
                s.dst = B.KvCache(s.k2, s.v2, n, case["kv"], case["dim"], s.k2.shape[2], bf16=case["bf16"], weight=s.weight2, pos=s.pos2)
        kv, st = s.kv, torch.cuda.current_stream().cuda_stream
    if kind in ("verify", "step"):
        if own:
            kv.append(n, rows, s.len, s.qkv, n_head=H, q=s.q, at=s.at, rope=s.rope, n_rope=ENGINE_CAP, count=s.count, stream=st)
        else:
            _plain_append(s)
    if kind in ("tree", "verify", "step"):
        if own:
            kv.attn_tree(n, rows, s.len, s.q, H, s.out, s.scale, count=s.count, mask=s.mask, len_hint=case["ctx"], window=case.get("window", 0), sinks=s.sinks, lse=s.lse,
                         stream=st)
        else:
            _plain_tree(s)
    if kind == "tree":
        return {"out": s.out, "lse": s.lse}
    if kind == "verify":
        if own:
            kv.commit(n, rows, s.len, s.path, s.npath, new_len=s.new_len, stream=st)
        else:
            _plain_commit(s)
        return {"q": s.q, "out": s.out, "lse": s.lse, "k": s.k, "v": s.v, "weight": s.weight, "pos": s.pos, "len": s.new_len}
    if kind in ("weigh", "step"):
        if own:
            kv.weigh(n, rows, s.len, s.q, H, s.lse, s.scale, count=s.count, mask=s.mask, picked=s.rows, len_hint=case["ctx"], window=case.get("window", 0), stream=st)
        else:
            _plain_weigh(s)
    if kind == "weigh":
        return {"weight": s.weight}
    if kind == "evict":
        if own:
            kv.evict(n, s.len, keep, FIRST, RECENT, s.end, s.map, dst=s.dst, new_len=s.new_len, len_hint=case["ctx"], stream=st)
        else:
            _plain_evict(s, s.len, keep, s.k2, s.v2, s.weight2, s.pos2)
        return {"k": s.k2, "v": s.v2, "weight": s.weight2, "pos": s.pos2, "map": s.map, "len": s.new_len}
    if kind == "step":
        if own:
            kv.evict(n, s.full, keep, FIRST, RECENT, s.end, s.map, new_len=s.new_len, len_hint=case["ctx"] + 1, stream=st)
        else:
            _plain_evict(s, s.full, keep, s.k, s.v, s.weight, s.pos)
        slot = slice(0, keep)       # what lies behind the new length is nobody's
        return {"q": s.q, "out": s.out, "lse": s.lse, "k": s.k[:, :, slot], "v": s.v[:, :, slot], "weight": s.weight[:, :, slot], "pos": s.pos[:, :, slot], "map": s.map,
                "len": s.new_len}
    if own:
        kv.means(n, s.len, case["block"], s.means, since=s.since, len_hint=rows, stream=st)
        kv.attn_blocks(len(s.seq), s.seq, s.lens, case["block"], s.means, case["nsel"], 1, 2, s.q, H, s.out, s.scale, s.sel, len_hint=case["ctx"], sinks=s.sinks, lse=s.lse,
                       stream=st)
    else:
        _plain_means(s)
        _plain_blocks(s)
    return {"means": s.means, "sel": s.sel, "out": s.out, "lse": s.lse}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, rows, H, kvh, hd, kind = case["n"], case["rows"], case["heads"], case["kv"], case["dim"], case["kind"]
    size, lens = 2 if case["bf16"] else 4, _lens(case)
    entry = kvh * hd * size
    if kind == "evict":
        kept = [min(x, case["keep"]) for x in lens]
        return {"bytes": sum(x * kvh * 8 for x in lens) + sum(kept) * (4 * entry + kvh * 12), "flops": 0}
    if kind == "blocks":
        block, nsel = case["block"], case["nsel"]
        seen = lens if rows == 1 else [case["ctx"] - rows + i + 1 for i in range(rows)]
        taken = [min(x, nsel * block) for x in seen]
        scored = [x // block for x in seen]
        # a row's blocks are its own choice; what several rows of one sequence choose in common is read once
        read = sum(taken) if rows == 1 else min(case["ctx"], sum(taken))
        by = read * 2 * entry + (sum(scored) if rows == 1 else scored[-1]) * kvh * hd * 4 + len(seen) * (2 * H * hd + H + kvh * nsel) * 4
        return {"bytes": by, "flops": sum(4 * x * H * hd for x in taken) + sum(2 * x * H * hd for x in scored)}
    parents, counts = _trees(case)
    window, slots, pairs = case.get("window", 0), 0, 0
    for ln, c, masks in zip(lens, counts, _masks(parents)):
        depths = [bin(m).count("1") - 1 for m in masks[:c]]
        seen = [min(ln, max(0, window - d - 1)) if window else ln for d in depths]
        slots += max(seen) + c
        pairs += sum(x + d + 1 for x, d in zip(seen, depths))
    tokens = sum(counts)
    attend = {"bytes": slots * 2 * entry + tokens * (2 * H * hd + H) * 4, "flops": 4 * pairs * H * hd}
    if kind == "tree":
        return attend
    append = tokens * ((2 * H + 2 * kvh) * hd * 4 + 2 * entry)
    if kind == "verify":
        return {"bytes": append + attend["bytes"], "flops": attend["flops"]}
    weigh = {"bytes": slots * (entry + kvh * 8) + tokens * (H * hd + H) * 4, "flops": 2 * pairs * H * hd}
    if kind == "weigh":
        return weigh
    # the weights may be formed from scores that the attention has at hand: K is counted once
    return {"bytes": append + attend["bytes"] + slots * kvh * 16, "flops": attend["flops"]}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_row(q, k, v, seen, scale, sinks):
    """One row: q [kv][g][dim], k and v [kv][width][dim], seen [width] or [kv][width]."""
    x = torch.einsum("hgd,htd->hgt", q, k) * scale
    x = torch.where(seen if seen.dim() == 1 else seen[:, None], x, torch.tensor(-math.inf, dtype=x.dtype, device=x.device))
    if sinks is not None:
        x = torch.cat([x, sinks.view(x.shape[0], -1, 1)], -1)
    lse = torch.logsumexp(x, -1)
    p = (x - lse[..., None]).exp()
    p = torch.nan_to_num(p, nan=0.0)
    return torch.einsum("hgt,htd->hgd", p[..., : k.shape[1]], v), lse, p[..., : k.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    n, rows, H, kvh, hd, kind = case["n"], case["rows"], case["heads"], case["kv"], case["dim"], case["kind"]
    dev, lens = s.k.device, _lens(case)
    sinks = None if s.sinks is None else s.sinks.double()
    if kind == "evict":
        k, v, w, pos = (torch.zeros_like(x) for x in (s.k2, s.v2, s.weight2, s.pos2))
        _exact_evict(s, lens, case["keep"], k, v, w, pos)
        return {"k": k.double(), "v": v.double(), "weight": w.double(), "pos": None, "map": None, "len": None}
    if kind == "blocks":
        if len(s.seq) * case["nsel"] * case["block"] * kvh > 20_000_000:
            return None
        means, out, lse = s.means.double(), torch.zeros_like(s.out, dtype=torch.float64), torch.zeros_like(s.lse, dtype=torch.float64)
        for b, ln in enumerate(lens):
            for j in range(max(0, ln - rows) // case["block"], ln // case["block"]):
                means[b, :, j] = s.k[b, :, j * case["block"] : (j + 1) * case["block"]].double().mean(1)
        stored = means.float().double()
        for r in range(len(s.seq)):
            b, ln = int(s.seq[r]), int(s.lens[r])
            nb, block = -(-ln // case["block"]), case["block"]
            q = s.q[r].view(kvh, -1, hd).double()
            score = torch.einsum("hgd,hjd->hgj", q, stored[b, :, : ln // block]).amax(1).float().cpu().numpy()
            for h in range(kvh):
                must = sorted({j for j in range(nb) if j < 1 or j >= nb - 2})
                free = sorted((j for j in range(nb) if j not in must), key=lambda j: (-score[h, j], j))
                chosen = sorted(must + free[: max(0, case["nsel"] - len(must))])
                t = torch.cat([torch.arange(j * block, min(ln, (j + 1) * block), device=dev) for j in chosen])
                o, z, _ = _exact_row(q[h : h + 1], s.k[b, h : h + 1, t].double(), s.v[b, h : h + 1, t].double(), torch.ones(len(t), dtype=torch.bool, device=dev), s.scale,
                                     None if sinks is None else sinks.view(kvh, -1)[h])
                out[r].view(kvh, -1, hd)[h], lse[r].view(kvh, -1)[h] = o[0], z[0]
        return {"means": means, "sel": None, "out": out, "lse": lse}
    parents, counts = _trees(case)
    masks = _masks(parents)
    window = case.get("window", 0)
    out, lse = torch.zeros_like(s.out, dtype=torch.float64), torch.zeros_like(s.lse, dtype=torch.float64)
    weight, q_all, keys, values = s.weight.double(), s.q.double(), s.k, s.v
    if kind in ("verify", "step"):
        x = s.qkv.double().view(n, rows, -1, hd)
        q_all, kd, vd = q_all.clone(), s.k.double(), s.v.double()
        for b in range(n):
            for i in range(counts[b]):
                p = int(s.at[b, i])
                c, d = s.rope[p, :, 0].double(), s.rope[p, :, 1].double()
                lo, hi = x[b, i, : H + kvh, : hd // 2], x[b, i, : H + kvh, hd // 2 :]
                turned = torch.cat([lo * c - hi * d, hi * c + lo * d], -1)
                q_all[b, i] = turned[:H].reshape(-1)
                kd[b, :, lens[b] + i], vd[b, :, lens[b] + i] = turned[H:], x[b, i, H + kvh :]
                weight[b, :, lens[b] + i] = 0.0
                s.pos[b, :, lens[b] + i] = p
        keys, values = kd.to(s.k.dtype), vd.to(s.v.dtype)
    picked = s.rows.tolist() if kind == "weigh" and s.rows is not None else [-1] * n
    for b in range(n):
        width = lens[b] + rows
        t = torch.arange(width, device=dev)
        k, v = keys[b, :, :width].double(), values[b, :, :width].double()
        depth = [bin(m & ((1 << counts[b]) - 1)).count("1") - 1 for m in masks[b]]
        for i in range(counts[b]):
            seen = t < lens[b]
            if window:
                seen &= t > lens[b] + depth[i] - window
            for j in range(counts[b]):
                if masks[b][i] >> j & 1 and (not window or depth[i] - depth[j] < window):
                    seen[lens[b] + j] = True
            o, z, p = _exact_row(q_all[b, i].view(kvh, -1, hd), k, v, seen, s.scale, sinks)
            out[b, i], lse[b, i] = o.reshape(-1), z.reshape(-1)
            if kind == "weigh":         # the logarithms of the sums are given
                p = (torch.einsum("hgd,htd->hgt", q_all[b, i].view(kvh, -1, hd), k) * s.scale - s.lse[b, i].double().view(kvh, -1, 1)).exp() * seen
            if kind in ("weigh", "step") and picked[b] >> i & 1:
                weight[b, :, :width] += p.sum(1)
    if kind == "tree":
        return {"out": out, "lse": lse}
    if kind == "weigh":
        return {"weight": weight}
    if kind == "verify":
        k, v, w = kd, vd, weight
        for b in range(n):
            path = [lens[b] + x for x in s.path[b, : int(s.npath[b])].tolist()]
            to = slice(lens[b], lens[b] + len(path))
            k[b, :, to], v[b, :, to], w[b, :, to] = k[b, :, path].clone(), v[b, :, path].clone(), w[b, :, path].clone()
        return {"q": q_all, "out": out, "lse": lse, "k": k, "v": v, "weight": w, "pos": None, "len": None}
    s.k, s.v, s.weight = kd, vd, weight
    k, v, w, pos = kd.clone(), vd.clone(), weight.clone(), s.pos.clone()
    _exact_evict(s, [x + 1 for x in lens], case["keep"], k, v, w, pos)
    m = case["keep"]
    return {"q": q_all, "out": out, "lse": lse, "k": k[:, :, :m], "v": v[:, :, :m], "weight": w[:, :, :m], "pos": None, "map": None, "len": None}


def _exact_evict(s, lens, keep, k, v, weight, pos):
    end = s.end.tolist()
    for b, ln in enumerate(lens):
        m = min(ln, keep)
        for h in range(s.weight.shape[1]):
            w, at = s.weight[b, h, :ln].tolist(), s.pos[b, h, :ln].tolist()
            ranked = sorted(range(ln), key=lambda t: (not (at[t] < FIRST or at[t] >= end[b] - RECENT), -w[t], t))
            kept = sorted(ranked[:m])
            held, spare = set(kept), [t for t in kept if t >= m]
            source = [t if t in held else spare.pop(0) for t in range(m)]
            src = torch.tensor(source, device=s.k.device)
            k[b, h, :m], v[b, h, :m], weight[b, h, :m], pos[b, h, :m] = s.k[b, h, src], s.v[b, h, src], s.weight[b, h, src], s.pos[b, h, src]
