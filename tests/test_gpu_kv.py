"""KV-cache operators on the GPU against their 64-bit restatement (kv_ref.py).

Tolerances.  Scores are sums of head_dim products formed to about 22 bits and added in single precision, partly by truncating adders: with at most
head_dim / 8 = 16 dependent sums of 2^-24 each, |score| around 3 (the inputs here: unit normal, scale 1 / sqrt(dim)) and e^x turning an absolute error into
a relative one, a weight is off by at most 2 x 16 x 3 x 2^-24 = 6e-6 and an output, a mean of values under such weights, by the same in the 2-norm; sums of
partial results add less than 1e-6.  So: 1e-5 of the 2-norm, and 1e-5 absolute on lse (plus its own rounding, 2^-24 relative).  Dropping the low
part of any operand (11 bits left) would be off by 1e-4 and more.  bf16 caches hold the values the reference reads, so the same holds."""
import math

import numpy as np
import pytest

import kv_ref as R

pytestmark = pytest.mark.gpu

NORM, LSE = 1e-5, 1e-5


class Setup:
    """A cache with random values: torch tensors in device memory, and the values as 64-bit arrays.  Strides and layout as asked for; memory between heads is NaN."""

    def __init__(self, dev, seed, n_seq, nkv, hd, cap, bf16=False, pad=0, heads_outside=False):
        import torch
        self.torch, self.dev, self.rng = torch, dev, np.random.default_rng(seed)
        self.n_seq, self.nkv, self.hd, self.cap, self.bf16 = n_seq, nkv, hd, cap, bf16
        t = torch.bfloat16 if bf16 else torch.float32
        shape = (nkv, n_seq, cap * hd + pad) if heads_outside else (n_seq, nkv, cap * hd + pad)
        self.raw = [torch.full(shape, float("nan"), dtype=t, device=dev) for _ in range(2)]
        if heads_outside:
            self.hs, self.ss = n_seq * (cap * hd + pad), cap * hd + pad
        else:
            self.hs, self.ss = cap * hd + pad, nkv * (cap * hd + pad)
        self.heads_outside = heads_outside
        for x in self.raw:
            self.rows(x).copy_(torch.from_numpy(self.rng.standard_normal((n_seq, nkv, cap, hd)).astype(np.float32)))
        self.weight = torch.zeros((n_seq, nkv, cap), device=dev)
        self.pos = torch.zeros((n_seq, nkv, cap), dtype=torch.int32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)

    def rows(self, x):
        x = x[:, :, : self.cap * self.hd].unflatten(2, (self.cap, self.hd))
        return x.transpose(0, 1) if self.heads_outside else x

    @property
    def k(self):
        return self.rows(self.raw[0])

    @property
    def v(self):
        return self.rows(self.raw[1])

    def view(self, B):
        dense = self.hs == self.cap * self.hd and self.ss == self.nkv * self.hs
        return B.KvCache(self.raw[0], self.raw[1], self.n_seq, self.nkv, self.hd, self.cap, bf16=self.bf16, head_stride=0 if dense else self.hs, seq_stride=0 if dense else self.ss,
                         weight=self.weight, pos=self.pos, err=self.err)

    def values(self):
        return self.k.double().cpu().numpy(), self.v.double().cpu().numpy()

    def f32(self, *shape):
        return self.rng.standard_normal(shape).astype(np.float32)

    def up(self, a, dtype=None):
        a = np.ascontiguousarray(a, dtype=dtype)
        if a.dtype == np.uint64:
            a = a.view(np.int64)
        return self.torch.from_numpy(a).to(self.dev)

    def ok(self):
        return int(self.err.item()) == 0


def random_tree(rng, rows):
    masks = []
    for i in range(rows):
        j = int(rng.integers(-1, i)) if i else -1
        masks.append(1 << i | (masks[j] if j >= 0 else 0))
    return masks


def close(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= NORM * norm if norm else not got.any(), (np.linalg.norm(got - want), norm)


def close_lse(got, want):
    got = np.asarray(got, np.float64)
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin])
    off = np.abs(got[fin] - want[fin])
    assert (off <= LSE + np.abs(want[fin]) * 2.0**-24).all(), off.max()


TREES = [
    # n_seq, n, rows, lengths, heads, kv, dim, bf16, window, counts, masks, seq, sinks
    dict(n=1, rows=1, lens=[0], heads=8, kv=2, hd=64, masks="chain"),
    dict(n=1, rows=1, lens=[1], heads=2, kv=2, hd=128, masks="chain"),
    dict(n=1, rows=1, lens=[72], heads=64, kv=8, hd=64, masks="chain", sinks=True),
    dict(n=3, rows=2, lens=[0, 7, 8], heads=8, kv=1, hd=64, masks="tree", bf16=True),
    dict(n=2, rows=5, lens=[15, 200], heads=12, kv=4, hd=128, masks="tree"),
    dict(n=2, rows=7, lens=[300, 33], heads=20, kv=4, hd=64, masks="tree", counts=[7, 3], sinks=True, window=37),
    dict(n=1, rows=64, lens=[129], heads=8, kv=1, hd=64, masks="tree"),
    dict(n=2, rows=64, lens=[63, 511], heads=4, kv=2, hd=128, masks="tree", bf16=True, counts=[64, 49]),
    dict(n=1, rows=64, lens=[100], heads=2, kv=1, hd=64, masks="chain", window=5, sinks=True),
    dict(n=2, rows=33, lens=[1000, 1], heads=16, kv=1, hd=128, masks="any"),
    dict(n=3, rows=9, lens=[40, 41, 0], heads=6, kv=6, hd=64, masks="any", window=1, bf16=True),
    dict(n=2, rows=3, lens=[0, 0], heads=8, kv=4, hd=64, masks="none"),
    dict(n=2, rows=3, lens=[0, 0], heads=8, kv=4, hd=64, masks="none", sinks=True),
    dict(n=2, rows=3, lens=[5, 17], heads=8, kv=4, hd=64, masks="chain", counts=[0, 2]),
    dict(n=3, rows=4, lens=[250, 3, 77], heads=8, kv=4, hd=64, masks="tree", seq=[4, 0, 4], pad=8),
    dict(n=2, rows=13, lens=[777, 500], heads=14, kv=2, hd=128, masks="tree", seq=[1, 2], heads_outside=True, bf16=True),
    dict(n=1, rows=17, lens=[2113], heads=32, kv=4, hd=128, masks="tree"),
    dict(n=1, rows=40, lens=[1500], heads=15, kv=1, hd=64, masks="tree", window=128, sinks=True),
]


def prepared_tree(dev, c, seed=1):
    rng = np.random.default_rng(seed)
    n, rows = c["n"], c["rows"]
    seq = c.get("seq") or list(range(n))
    s = Setup(dev, seed, max(seq) + 1, c["kv"], c["hd"], max(c["lens"]) + rows + 3, c.get("bf16", False), c.get("pad", 0), c.get("heads_outside", False))
    s.rows_n, s.lens, s.seq = rows, c["lens"], seq
    s.counts = c.get("counts") or [rows] * n
    s.masks = {"chain": lambda: [R.chain(rows)] * n, "tree": lambda: [random_tree(rng, rows) for _ in range(n)],
               "any": lambda: [[int(x) for x in rng.integers(0, 1 << 63, rows)] for _ in range(n)], "none": lambda: [[0] * rows] * n}[c["masks"]]()
    s.q = s.f32(n, rows, c["heads"], c["hd"])
    s.sinks = s.f32(c["heads"]) if c.get("sinks") else None
    s.scale, s.window, s.heads = 1 / math.sqrt(c["hd"]), c.get("window", 0), c["heads"]
    # what no row of an entry sees holds NaN
    for q in set(seq):
        used = set()
        for b in range(n):
            if seq[b] == q:
                used |= {t for i in range(s.counts[b]) for t in range(s.lens[b] + s.counts[b]) if R.sees(s.masks[b], s.counts[b], s.lens[b], s.window, i, t)}
        idle = [t for t in range(s.cap) if t not in used]
        s.k[q, :, idle] = float("nan")
        s.v[q, :, idle] = float("inf")
    return s


def run_tree(B, s, c, lse=True, hint=0, stream=None, out=None):
    import torch
    n, rows = c["n"], c["rows"]
    out = torch.full((n, rows, c["heads"] * c["hd"]), 7.0, device=s.dev) if out is None else out
    z = torch.full((n, rows, c["heads"]), 7.0, device=s.dev) if lse else None
    s.view(B).attn_tree(n, rows, s.up(s.lens, np.int32), s.up(s.q), c["heads"], out, s.scale, seq=s.up(s.seq, np.int32) if "seq" in c else None,
                        count=s.up(s.counts, np.int32) if "counts" in c else None, mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)), len_hint=hint,
                        window=s.window, sinks=None if s.sinks is None else s.up(s.sinks), lse=z, stream=stream)
    torch.cuda.synchronize()
    return out, z


@pytest.mark.parametrize("c", TREES, ids=lambda c: "-".join(str(c[k]) for k in ("n", "rows", "lens", "heads", "kv", "hd", "masks")))
def test_tree(brrr, dev, c):
    s = prepared_tree(dev, c)
    out, lse = run_tree(brrr, s, c)
    assert s.ok()
    k, v = s.values()
    want, want_lse, _ = R.tree(s.q.astype(np.float64), k, v, s.seq, s.lens, s.counts, s.masks, s.scale, s.window, s.sinks)
    out, lse = out.cpu().numpy().reshape(want.shape), lse.cpu().numpy()
    for b in range(c["n"]):
        m = s.counts[b]
        if m:
            close(out[b, :m], want[b, :m])
            close_lse(lse[b, :m], want_lse[b, :m])
        assert (out[b, m:] == 7.0).all() and (lse[b, m:] == 7.0).all()      # rows behind the count
    again, _ = run_tree(brrr, s, c, lse=False, hint=0)
    assert np.array_equal(again.cpu().numpy().reshape(out.shape), out)
    inplace = s.up(s.q).view(c["n"], c["rows"], -1)
    args = dict(seq=s.up(s.seq, np.int32) if "seq" in c else None, count=s.up(s.counts, np.int32) if "counts" in c else None,
                mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)), window=s.window, sinks=None if s.sinks is None else s.up(s.sinks))
    s.view(brrr).attn_tree(c["n"], c["rows"], s.up(s.lens, np.int32), inplace, c["heads"], inplace, s.scale, **args)
    for b in range(c["n"]):
        assert np.array_equal(inplace.cpu().numpy().reshape(out.shape)[b, : s.counts[b]], out[b, : s.counts[b]])
    for hint in (1, s.cap, 1 << 20):                                          # a hint is no more than that
        other, _ = run_tree(brrr, s, c, lse=False, hint=hint)
        for b in range(c["n"]):
            if s.counts[b]:
                close(other.cpu().numpy().reshape(out.shape)[b, : s.counts[b]], want[b, : s.counts[b]])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_rows_do_not_touch_what_other_rows_see(brrr, dev, bf16, hd):
    """A drafted row whose key and value are no numbers, and cached slots that the window hides from the deeper rows alone: only rows that see them are concerned."""
    c = dict(n=1, rows=9, lens=[60], heads=8, kv=2, hd=hd, masks="tree", bf16=bf16)
    s = prepared_tree(dev, c)
    masks = [1, 3, 5, 9, 16 | 1, 32 | 2 | 1, 64, 128 | 64, 256]
    s.masks, s.window = [masks], 20
    k, v = s.values()
    bad_rows = {i for i in range(9) if masks[i] >> 2 & 1 or i in (6, 8)}
    s.v[0, :, 62] = float("inf"); s.k[0, :, 62] = float("nan")     # row 2
    s.v[0, :, 41] = float("nan"); s.k[0, :, 41] = float("-inf")    # seen by depth 0 alone: rows 0, 6 and 8
    bad_rows |= {0}
    k[0, :, [62, 41]] = 0; v[0, :, [62, 41]] = 0
    out, _ = run_tree(brrr, s, c)
    out = out.cpu().numpy().reshape(9, 8, hd)
    want = R.tree(s.q.astype(np.float64), k, v, [0], [60], [9], s.masks, s.scale, 20)[0][0]
    for i in set(range(9)) - bad_rows:
        close(out[i], want[i])


def test_tree_leaves_out_what_does_not_fit(brrr, dev):
    import torch
    c = dict(n=6, rows=4, lens=[10, -1, 30, 31, 10, 10], heads=4, kv=2, hd=64, masks="chain", seq=[0, 0, 0, 0, 3, -1])
    s = Setup(dev, 5, 2, 2, 64, 34)
    q = s.f32(6, 4, 4, 64)
    out = torch.full((6, 4, 256), 7.0, device=dev)
    s.view(brrr).attn_tree(6, 4, s.up(c["lens"], np.int32), s.up(q), 4, out, 0.125, seq=s.up(c["seq"], np.int32))
    torch.cuda.synchronize()
    assert not s.ok()
    k, v = s.values()
    for b in range(6):
        if b in (0, 2):
            close(out[b].cpu().numpy().reshape(4, 4, 64), R.tree(q[b:b + 1].astype(np.float64), k, v, [0], [c["lens"][b]], [4], [R.chain(4)], 0.125)[0][0])
        else:
            assert (out[b] == 7.0).all()
    s.err.zero_()
    out.fill_(7.0)
    s.view(brrr).attn_tree(2, 4, s.up([3, 3], np.int32), s.up(q), 4, out, 0.125, count=s.up([5, -1], np.int32))
    torch.cuda.synchronize()
    assert not s.ok() and (out == 7.0).all()


def test_tree_large_scores_and_sinks(brrr, dev):
    """Scores of hundreds, of either sign: the running maximum carries them; a sink far above takes all weight, one far below none."""
    c = dict(n=1, rows=3, lens=[400], heads=4, kv=1, hd=64, masks="tree")
    s = prepared_tree(dev, c)
    s.scale = 30.0
    s.sinks = np.float32([1e4, -1e4, 0.0, -np.inf])
    out, lse = run_tree(brrr, s, c)
    k, v = s.values()
    want, want_lse, _ = R.tree(s.q.astype(np.float64), k, v, [0], [400], [3], s.masks, 30.0, 0, s.sinks.astype(np.float64))
    # a score of 1000 carries 16 x 2^-24 x 1000 = 1e-3 of absolute error into the exponent
    assert np.abs(out.cpu().numpy().reshape(want.shape) - want).max() < 4e-3 and np.abs(lse.cpu().numpy() - want_lse).max() < 2e-3


def test_offsets_beyond_32_bits(brrr, dev):
    """The second sequence stands more than 2^32 values behind the first."""
    import torch
    stride, cap, hd, kv = (1 << 32) + 64, 130, 64, 2
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB of device memory")
    buf = [torch.empty(stride + kv * cap * hd, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    rng = np.random.default_rng(3)
    x = [torch.from_numpy(rng.standard_normal((kv, cap, hd)).astype(np.float32)).to(dev).bfloat16() for _ in range(2)]
    for b, y in zip(buf, x):
        b[stride:] = y.flatten()
    weight, pos, err = torch.zeros((2, kv, cap), device=dev), torch.arange(cap, dtype=torch.int32, device=dev).repeat(2, kv, 1), torch.zeros(1, dtype=torch.int32, device=dev)
    view = brrr.KvCache(buf[0], buf[1], 2, kv, hd, cap, bf16=True, seq_stride=stride, weight=weight, pos=pos, err=err)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.from_numpy(rng.standard_normal((1, 2, 4, hd)).astype(np.float32)).to(dev)
    out, lse = torch.zeros((1, 2, 4 * hd), device=dev), torch.zeros((1, 2, 4), device=dev)
    seq, ln = i32(1), i32(120)
    view.attn_tree(1, 2, ln, q, 4, out, 0.125, seq=seq, lse=lse)
    k, v = (y.double().cpu().numpy()[None] for y in x)
    want, _, weights = R.tree(q.double().cpu().numpy(), k, v, [0], [120], [2], [R.chain(2)], 0.125)
    close(out.cpu().numpy().reshape(want.shape), want)
    view.weigh(1, 2, ln, q, 4, lse, 0.125, seq=seq)
    book = np.zeros((kv, cap))
    for _, _, h, slots, w in weights:
        book[h // 2, slots] += w
    close(weight[1].cpu().numpy(), book)
    means, sel = torch.zeros((2, kv, cap // 16, hd), device=dev), torch.zeros((1, kv, 3), dtype=torch.int32, device=dev)
    view.means(1, ln, 16, means, seq=seq)
    want = k[0, :, :112].reshape(kv, 7, 16, hd).mean(2)
    assert np.array_equal(means[1, :, :7].cpu().numpy(), want.astype(np.float32)) and not means[0].any()
    view.attn_blocks(1, seq, ln, 16, means, 3, 1, 1, q[:, :1].contiguous(), 4, out[:, :1].contiguous(), 0.125, sel)
    for h in range(kv):
        assert sel[0, h].tolist() == R.choose(q[0, 0].cpu().numpy()[2 * h: 2 * h + 2], means[1, h].cpu().numpy(), 120, 16, 3, 1, 1)
    kept = torch.zeros((1, kv, 40), dtype=torch.int32, device=dev)
    view.evict(1, ln, 40, 2, 5, i32(120), kept, seq=seq)
    torch.cuda.synchronize()
    for h in range(kv):
        src = R.evict(book[h, :120].astype(np.float32), list(range(120)), 40, 2, 5, 120)
        assert torch.equal(buf[0][stride + h * cap * hd:][: 40 * hd].view(40, hd), x[0][h][torch.tensor(kept[0, h].tolist(), device=dev)])
        assert kept[0, h].tolist() == src
    assert int(err) == 0


# ---------------------------------------------------------------- many rows: the kernels of 128-row tiles
WIDE = [
    dict(n=1, rows=64, lens=[700], heads=64, kv=4, hd=64, masks="tree"),
    dict(n=3, rows=33, lens=[1301, 0, 640], heads=64, kv=4, hd=64, masks="any", counts=[33, 17, 33], sinks=True),
    dict(n=2, rows=64, lens=[1025, 1152], heads=32, kv=2, hd=64, masks="tree", window=200),
    dict(n=4, rows=64, lens=[130, 127, 129, 64], heads=48, kv=6, hd=64, masks="chain", seq=[4, 1, 0, 2], pad=16),
    dict(n=2, rows=40, lens=[900, 77], heads=48, kv=3, hd=128, masks="tree"),
    dict(n=2, rows=64, lens=[511, 1090], heads=32, kv=2, hd=128, masks="any", window=64, sinks=True),
    dict(n=3, rows=50, lens=[641, 640, 639], heads=48, kv=4, hd=128, masks="chain", counts=[50, 1, 49], heads_outside=True),
    dict(n=1, rows=61, lens=[1999], heads=32, kv=2, hd=64, masks="tree", bf16=True),
    dict(n=2, rows=64, lens=[500, 1301], heads=64, kv=4, hd=64, masks="any", bf16=True, counts=[0, 64], sinks=True, window=333),
    dict(n=24, rows=64, lens=[30 + 2 * i for i in range(24)], heads=16, kv=2, hd=64, masks="tree", bf16=True),
    dict(n=2, rows=47, lens=[1280, 831], heads=32, kv=2, hd=128, masks="tree", bf16=True, seq=[2, 2], pad=8),
    dict(n=1, rows=64, lens=[2500], heads=16, kv=1, hd=128, masks="chain", bf16=True, window=1000),
]


def reference(s, c, q, scale):
    """The definition in 64 bits on the GPU, entry by entry: out, lse, and the weights of every row [n][rows][heads][slots]."""
    import torch
    k, v = s.k.double().nan_to_num(0.0, 0.0, 0.0), s.v.double().nan_to_num(0.0, 0.0, 0.0)       # what is no number here nobody sees
    n, rows, heads, hd = q.shape
    out, lse, weights = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device), []
    for b in range(n):
        m, ln = s.counts[b], s.lens[b]
        if not m:
            weights.append(None)
            continue
        live = [x & ((1 << m) - 1) for x in s.masks[b][:m]]
        seen = torch.zeros((m, ln + m), dtype=torch.bool, device=q.device)
        for i in range(m):
            di = R.depth(live[i], i)
            seen[i, max(0, ln + di + 1 - s.window) if s.window else 0: ln] = True
            seen[i, ln:] = torch.tensor([bool(live[i] >> j & 1) and (not s.window or di - R.depth(live[j], j) < s.window) for j in range(m)], device=q.device)
        per = heads // c["kv"]
        x = torch.einsum("ihd,htd->iht", q[b, :m].double(), k[s.seq[b], :, : ln + m].repeat_interleave(per, 0)) * scale
        x = x.masked_fill(~seen[:, None], -math.inf)
        full = x if s.sinks is None else torch.cat([x, s.up(s.sinks).double().view(1, -1, 1).expand(m, -1, 1)], -1)
        lse[b, :m] = torch.logsumexp(full, -1)
        w = torch.exp(x - lse[b, :m, :, None]).nan_to_num(0.0)
        out[b, :m] = torch.einsum("iht,htd->ihd", w, v[s.seq[b], :, : ln + m].repeat_interleave(per, 0))
        weights.append(w)
    return out, lse, weights


@pytest.mark.parametrize("scale", [1.0, -1.3])
@pytest.mark.parametrize("c", WIDE, ids=lambda c: "-".join(str(c[k]) for k in ("n", "rows", "heads", "kv", "hd", "masks")) + ("-bf16" if c.get("bf16") else ""))
def test_wide_trees_and_their_weights(brrr, dev, c, scale):
    import torch
    s = prepared_tree(dev, c, seed=31)
    s.scale *= scale
    n, rows, per = c["n"], c["rows"], c["heads"] // c["kv"]
    want, want_lse, weights = reference(s, c, s.up(s.q), s.scale)
    for hint in (0, 1):              # a small hint sends the same call to the kernel of 16-row tiles
        out, lse = run_tree(brrr, s, c, hint=hint)
        assert s.ok()
        again, _ = run_tree(brrr, s, c, hint=hint)
        assert torch.equal(out, again)
        same = s.up(s.q).view(out.shape)
        s.view(brrr).attn_tree(n, rows, s.up(s.lens, np.int32), same, c["heads"], same, s.scale, seq=s.up(s.seq, np.int32) if "seq" in c else None,
                               count=s.up(s.counts, np.int32) if "counts" in c else None, mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)),
                               len_hint=hint, window=s.window, sinks=None if s.sinks is None else s.up(s.sinks))
        for b in range(n):
            assert torch.equal(same[b, : s.counts[b]], out[b, : s.counts[b]])
        for b in range(n):
            m = s.counts[b]
            if m:
                close(out[b, :m].cpu().numpy().reshape(m, c["heads"], c["hd"]), want[b, :m].cpu().numpy())
                close_lse(lse[b, :m].cpu().numpy(), want_lse[b, :m].cpu().numpy())
            assert (out[b, m:] == 7.0).all() and (lse[b, m:] == 7.0).all()
    if "seq" in c and len(set(s.seq)) < n:
        return                       # a sequence may be weighed once in a call
    picked = [int(x) for x in s.rng.integers(0, 1 << 63, n)]
    for pick in (None, picked):
        s.weight.fill_(1.0)
        s.view(brrr).weigh(n, rows, s.up(s.lens, np.int32), s.up(s.q), c["heads"], lse, s.scale, seq=s.up(s.seq, np.int32) if "seq" in c else None,
                           count=s.up(s.counts, np.int32) if "counts" in c else None, mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)),
                           picked=None if pick is None else s.up(np.array(pick, np.uint64)), window=s.window)
        torch.cuda.synchronize()
        assert s.ok()
        book = torch.ones(s.weight.shape, dtype=torch.float64, device=dev)
        for b in range(n):
            m = s.counts[b]
            if m:
                rows_in = torch.tensor([pick is None or bool(pick[b] >> i & 1) for i in range(m)], device=dev)
                book[s.seq[b], :, : s.lens[b] + m] += (weights[b] * rows_in[:, None, None]).sum(0).view(c["kv"], per, -1).sum(1)
        close(s.weight.cpu().numpy(), book.cpu().numpy())
        untouched = book == 1.0
        assert (s.weight[untouched] == 1.0).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_wide_rows_do_not_touch_what_other_rows_see(brrr, dev, bf16, hd):
    """As for few rows: drafted rows and cached slots that are no numbers concern the rows that see them, in outputs and in the book."""
    import torch
    c = dict(n=1, rows=64, lens=[900], heads=32, kv=2, hd=hd, masks="tree", bf16=bf16)
    s = prepared_tree(dev, c, seed=9)
    s.masks, s.window = [[1 << i | (s.masks[0][i] & 1) for i in range(64)]], 300       # rows see row 0 or nobody but themselves
    s.masks[0][0] = 1
    s.k.nan_to_num_(0.1), s.v.nan_to_num_(0.2, 0.3, 0.4)
    want, _, weights = reference(s, c, s.up(s.q), s.scale)
    s.v[0, :, 917] = float("inf"); s.k[0, :, 917] = float("nan")      # row 17
    s.v[0, 1, 930, 3] = float("nan")                                  # row 30, one dimension of one head
    shallow = [i for i in range(64) if R.depth(s.masks[0][i], i) == 0]
    s.v[0, :, 601] = float("nan"); s.k[0, :, 601] = float("inf")      # seen by depth 0 alone (601 = 900 + 0 + 1 - 300)
    out, lse = run_tree(brrr, s, c)
    out = out.cpu().numpy().reshape(64, 32, hd)
    fine = [i for i in range(64) if i not in shallow and i not in (17, 30)]
    close(out[fine], want[0, fine].cpu().numpy())
    close(out[30, :16], want[0, 30, :16].cpu().numpy()) if 30 not in shallow else None
    picked = sum(1 << i for i in fine)
    s.view(brrr).weigh(1, 64, s.up(s.lens, np.int32), s.up(s.q), 32, lse, s.scale, mask=s.up(np.array(s.masks, np.uint64)), picked=s.up(np.array([picked], np.uint64)), window=300)
    torch.cuda.synchronize()
    book = (weights[0][fine].sum(0)).view(2, 16, -1).sum(1)
    close(s.weight[0, :, :964].cpu().numpy(), book.cpu().numpy())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sinks", [False, True])
def test_wide_rows_that_see_nothing(brrr, dev, bf16, hd, sinks):
    """Rows without a slot stand between rows that have some: zeros, the sink or -infinity, and nothing in the book."""
    import torch
    c = dict(n=2, rows=64, lens=[0, 150], heads=32, kv=2, hd=hd, masks="tree", bf16=bf16, sinks=sinks)
    s = prepared_tree(dev, c, seed=12)
    s.k.nan_to_num_(0.1), s.v.nan_to_num_(0.2, 0.3, 0.4)
    s.masks = [[m if i % 3 else 0 for i, m in enumerate(masks)] for masks in s.masks]
    want, want_lse, weights = reference(s, c, s.up(s.q), s.scale)
    assert (want_lse[0, ::3] == -math.inf).all() != sinks
    for hint in (0, 1):
        out, lse = run_tree(brrr, s, c, hint=hint)
        close(out.cpu().numpy().reshape(want.shape), want.cpu().numpy())
        close_lse(lse.cpu().numpy(), want_lse.cpu().numpy())
        assert not out[0, ::3].any()
    s.weight.fill_(1.0)
    s.view(brrr).weigh(2, 64, s.up(s.lens, np.int32), s.up(s.q), 32, lse, s.scale, mask=s.up(np.array(s.masks, np.uint64)))
    torch.cuda.synchronize()
    book = torch.ones(s.weight.shape, dtype=torch.float64, device=dev)
    for b in range(2):
        book[b, :, : s.lens[b] + 64] += weights[b].sum(0).view(2, 16, -1).sum(1)
    assert s.ok()
    close(s.weight.cpu().numpy(), book.cpu().numpy())


def test_wide_rows_far_beyond_32_bits(brrr, dev):
    import torch
    stride, cap, hd, kv, rows, heads, ln = (1 << 32) + 64, 1000, 64, 2, 64, 32, 900
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB of device memory")
    buf = [torch.empty(stride + kv * cap * hd, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    rng = np.random.default_rng(5)
    x = [torch.from_numpy(rng.standard_normal((1, kv, cap, hd)).astype(np.float32)).to(dev).bfloat16() for _ in range(2)]
    for b, y in zip(buf, x):
        b[stride:] = y.flatten()
    weight, err = torch.zeros((2, kv, cap), device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    view = brrr.KvCache(buf[0], buf[1], 2, kv, hd, cap, bf16=True, seq_stride=stride, weight=weight, err=err)
    q = torch.from_numpy(rng.standard_normal((1, rows, heads, hd)).astype(np.float32)).to(dev)
    out, lse, seq, lens = torch.zeros((1, rows, heads * hd), device=dev), torch.zeros((1, rows, heads), device=dev), torch.ones(1, dtype=torch.int32, device=dev), \
        torch.full((1,), ln, dtype=torch.int32, device=dev)
    view.attn_tree(1, rows, lens, q, heads, out, 0.125, seq=seq, lse=lse)
    view.weigh(1, rows, lens, q, heads, lse, 0.125, seq=seq)
    torch.cuda.synchronize()

    class Near:
        k, v, counts, lens, masks, window, sinks, seq = x[0], x[1], [rows], [ln], [R.chain(rows)], 0, None, [0]
    want, want_lse, weights = reference(Near, dict(kv=kv), q, 0.125)
    close(out.cpu().numpy().reshape(want.shape), want.cpu().numpy())
    close_lse(lse.cpu().numpy(), want_lse.cpu().numpy())
    close(weight[1, :, : ln + rows].cpu().numpy(), weights[0].sum(0).view(kv, 16, -1).sum(1).cpu().numpy())
    assert int(err) == 0 and not weight[0].any()


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("hd,bf16,turn,nh,out_q", [(64, False, True, 9, True), (128, True, True, 6, True), (64, True, False, 0, False), (128, False, False, 3, True), (64, False, True, 6, False)])
def test_append(brrr, dev, hd, bf16, turn, nh, out_q):
    """Keys, values, rotated queries and books of ragged rows, bit for bit; nothing else changes."""
    import torch
    n, rows, kv = 3, 5, 3
    s = Setup(dev, 11, 4, kv, hd, 40, bf16, pad=16)
    seq, lens, counts = [3, 0, 2], [35, 0, 20], [5, 2, 0]
    ld = (nh + 2 * kv) * hd + 8
    x = s.f32(n, rows, ld)
    at = s.rng.integers(0, 50, (n, rows)).astype(np.int32)
    rope = s.f32(50, hd // 2, 2)
    s.weight += 3.0
    s.pos += 9
    before = [t.clone() for t in (*s.raw, s.weight, s.pos)]
    q = torch.full((n, rows, max(nh, 1), hd), 7.0, device=dev)
    s.view(brrr).append(n, rows, s.up(lens, np.int32), s.up(x), n_head=nh, q=q if out_q else None, at=s.up(at), rope=s.up(rope) if turn else None, n_rope=50 if turn else 0,
                        count=s.up(counts, np.int32), seq=s.up(seq, np.int32), ld=ld)
    torch.cuda.synchronize()
    assert s.ok()
    got = [s.k.float().cpu().numpy(), s.v.float().cpu().numpy(), s.weight.cpu().numpy(), s.pos.cpu().numpy()]
    after = [t.clone() for t in (*s.raw, s.weight, s.pos)]
    for t, old in zip((*s.raw, s.weight, s.pos), before):
        t.copy_(old)
    want = [s.k.float().cpu().numpy(), s.v.float().cpu().numpy(), s.weight.cpu().numpy(), s.pos.cpu().numpy()]
    want_q = np.full((n, rows, max(nh, 1), hd), 7.0, np.float32)
    for b in range(n):
        for i in range(counts[b]):
            r = x[b, i, : (nh + 2 * kv) * hd].reshape(-1, hd)
            y = R.rotate(r[: nh + kv], rope[at[b, i]]) if turn else r[: nh + kv]
            want_q[b, i, :nh] = y[:nh]
            k, v = torch.from_numpy(y[nh:].copy()), torch.from_numpy(r[nh + kv:].copy())
            want[0][seq[b], :, lens[b] + i] = (k.bfloat16() if bf16 else k).float().numpy()
            want[1][seq[b], :, lens[b] + i] = (v.bfloat16() if bf16 else v).float().numpy()
            want[2][seq[b], :, lens[b] + i] = 0
            want[3][seq[b], :, lens[b] + i] = at[b, i]
    for a, b in zip(got, want):
        assert np.array_equal(a, b, equal_nan=True)
    if out_q and nh:
        assert np.array_equal(q.cpu().numpy(), want_q)
    gap = [t[:, :, s.cap * hd:] for t in after[:2]]
    assert all(bool(g.isnan().all()) for g in gap)


def test_append_leaves_out(brrr, dev):
    """A second entry of one sequence, lengths and positions that do not fit, sequences that are none: nothing of them is written."""
    import torch
    s = Setup(dev, 2, 3, 2, 64, 16)
    before = s.k.clone()
    x = s.f32(6, 2, 4 * 64)
    rope = s.f32(8, 32, 2)
    at = np.zeros((6, 2), np.int32)
    at[0, 1] = 8
    at[3, 0] = -1
    s.view(brrr).append(6, 2, s.up([4, 15, 4, 5, 2, 1], np.int32), s.up(x), rope=s.up(rope), n_rope=8, at=s.up(at), seq=s.up([1, 0, 1, 2, 3, -7], np.int32))
    torch.cuda.synchronize()
    assert not s.ok()
    changed = (s.k != before).any(-1)
    assert changed.nonzero().tolist() == [[1, 0, 4], [1, 1, 4], [2, 0, 6], [2, 1, 6]]


# ---------------------------------------------------------------- commit
@pytest.mark.parametrize("hd,bf16", [(64, True), (128, False), (64, False), (128, True)])
def test_commit(brrr, dev, hd, bf16):
    import torch
    n, rows, kv = 5, 64, 2
    s = Setup(dev, 4, 6, kv, hd, 90, bf16, pad=8)
    s.weight.copy_(torch.from_numpy(s.f32(6, kv, 90)))
    s.pos.copy_(torch.arange(6 * kv * 90, dtype=torch.int32).view(6, kv, 90))
    seq, lens = [5, 0, 2, 3, 1], [26, 10, 0, 25, 88]
    paths = [[0, 1, 5, 63], [], list(range(64)), [63, 0, 0, 1], [1]]
    path = np.full((n, rows), -1, np.int32)
    for b, p in enumerate(paths):
        path[b, : len(p)] = p
    want = [t.clone() for t in (s.k, s.v, s.weight, s.pos)]
    for b, p in enumerate(paths):
        for t in want:
            t[seq[b], :, lens[b]: lens[b] + len(p)] = t[seq[b]][:, [lens[b] + x for x in p]].clone()
    new_len = torch.zeros(n, dtype=torch.int32, device=dev)
    s.view(brrr).commit(n, rows, s.up(lens, np.int32), s.up(path), s.up([len(p) for p in paths], np.int32), seq=s.up(seq, np.int32), new_len=new_len)
    torch.cuda.synchronize()
    assert s.ok() and new_len.tolist() == [a + len(p) for a, p in zip(lens, paths)]
    for a, b in zip((s.k, s.v, s.weight, s.pos), want):
        assert torch.equal(a, b)


def test_commit_leaves_out(brrr, dev):
    import torch
    s = Setup(dev, 4, 5, 2, 64, 20)
    before = [t.clone() for t in (s.k, s.v)]
    path = np.array([[1, 2], [2, 0], [1, 3], [-1, 0], [0, 1], [1, 1], [1, 0]], np.int32)
    new_len = torch.zeros(7, dtype=torch.int32, device=dev)
    lens = [4, 4, 4, 4, 4, 19, 4]
    s.view(brrr).commit(7, 3, s.up(lens, np.int32), s.up(np.pad(path, ((0, 0), (0, 1)))), s.up([2, 4, 2, 1, 2, 1, 1], np.int32), seq=s.up([0, 1, 2, 3, 0, 4, 5], np.int32), new_len=new_len)
    torch.cuda.synchronize()
    assert not s.ok() and new_len.tolist() == [6, 4, 4, 4, 4, 19, 4]
    assert torch.equal(s.k[1:], before[0][1:]) and torch.equal(s.v[1:], before[1][1:])
    assert torch.equal(s.k[0, :, 4:6], before[0][0, :, 5:7])


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("c", [c for c in TREES if "seq" not in c], ids=lambda c: "-".join(str(c[k]) for k in ("n", "rows", "lens", "heads", "kv", "hd", "masks")))
@pytest.mark.parametrize("pick", [False, True])
def test_weigh(brrr, dev, c, pick):
    import torch
    s = prepared_tree(dev, c, seed=2)
    _, lse = run_tree(brrr, s, c)
    k, v = s.values()
    n, rows, per = c["n"], c["rows"], c["heads"] // c["kv"]
    picked = [int(x) for x in s.rng.integers(0, 1 << 63, n)] if pick else [(1 << 64) - 1] * n
    book = np.abs(s.f32(s.n_seq, c["kv"], s.cap))
    s.weight.copy_(torch.from_numpy(book))
    want = book.astype(np.float64)
    seen = np.zeros(want.shape, bool)
    for b, i, h, slots, w in R.tree(s.q.astype(np.float64), k, v, s.seq, s.lens, s.counts, s.masks, s.scale, s.window, s.sinks)[2]:
        if picked[b] >> i & 1 and len(slots):
            want[s.seq[b], h // per, slots] += w
            seen[s.seq[b], h // per, slots] = True
    for hint in (0, 1):
        s.weight.copy_(torch.from_numpy(book))
        s.view(brrr).weigh(n, rows, s.up(s.lens, np.int32), s.up(s.q), c["heads"], lse, s.scale, count=s.up(s.counts, np.int32) if "counts" in c else None,
                           mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)), picked=s.up(np.array(picked, np.uint64)) if pick else None, len_hint=hint,
                           window=s.window)
        torch.cuda.synchronize()
        got = s.weight.cpu().numpy()
        assert s.ok() and np.array_equal(got[~seen], book[~seen])
        close(got[seen] - book[seen].astype(np.float64) + 1.0, want[seen] - book[seen] + 1.0) if seen.any() else None


def test_weigh_leaves_out(brrr, dev):
    import torch
    s = Setup(dev, 6, 3, 2, 64, 50)
    q, lse = s.up(s.f32(4, 2, 2, 64)), s.up(np.full((4, 2, 2), 5.0, np.float32))
    s.view(brrr).weigh(4, 2, s.up([10, 49, 10, 10], np.int32), q, 2, lse, 0.125, seq=s.up([1, 0, 1, 7], np.int32))
    torch.cuda.synchronize()
    assert not s.ok() and not s.weight[0].any() and not s.weight[2].any()
    once = s.weight.clone()
    s.err.zero_()
    s.weight.zero_()
    s.view(brrr).weigh(1, 2, s.up([10], np.int32), q, 2, lse, 0.125, seq=s.up([1], np.int32))
    torch.cuda.synchronize()
    assert s.ok() and torch.equal(s.weight, once) and bool((once[1, :, :12] > 0).all())


# ---------------------------------------------------------------- eviction
EVICT = [dict(n=1, lens=[1], keep=1, first=0, recent=0), dict(n=1, lens=[2], keep=1, first=0, recent=1), dict(n=3, lens=[0, 5, 33], keep=5, first=1, recent=2),
         dict(n=2, lens=[1025, 1024], keep=1024, first=4, recent=64, hd=128), dict(n=2, lens=[4000, 3999], keep=31, first=0, recent=31, bf16=True),
         dict(n=2, lens=[3000, 64], keep=64, first=64, recent=0, hd=128, bf16=True), dict(n=2, lens=[2500, 999], keep=1300, first=4, recent=100, seq=[2, 0]),
         dict(n=1, lens=[700], keep=350, first=0, recent=0, book="ties"), dict(n=1, lens=[700], keep=97, first=3, recent=9, book="odd"),
         dict(n=1, lens=[96], keep=64, first=0, recent=0, book="ties"), dict(n=1, lens=[33000], keep=20011, first=100, recent=1000, kv=1),
         dict(n=1, lens=[50001], keep=30011, first=7, recent=100, kv=1, book="ties"), dict(n=1, lens=[7001], keep=3500, first=0, recent=0, kv=2, book="odd")]


def evict_setup(dev, c, seed):
    import torch
    seq = c.get("seq") or list(range(c["n"]))
    s = Setup(dev, seed, max(seq) + 1, c.get("kv", 3), c.get("hd", 64), max(max(c["lens"]), c["keep"]) + 5, c.get("bf16", False), pad=8)
    w = np.exp(2 * s.f32(s.n_seq, s.nkv, s.cap))
    if c.get("book") == "ties":
        w = s.rng.integers(0, 3, w.shape).astype(np.float32)
    if c.get("book") == "odd":
        w = s.rng.choice(np.float32([0.0, -0.0, np.nan, -np.nan, np.inf, -np.inf, -1.0, 1e-42, 2.0]), w.shape)
    s.weight.copy_(torch.from_numpy(w.astype(np.float32)))
    s.pos.copy_(torch.from_numpy(np.stack([[s.rng.permutation(s.cap) for _ in range(s.nkv)] for _ in range(s.n_seq)]).astype(np.int32)))
    s.seq, s.end = seq, [s.cap] * c["n"]
    return s


def evict_want(s, c):
    w, p = s.weight.cpu().numpy(), s.pos.cpu().numpy()
    return [[R.evict(w[s.seq[b], h, : c["lens"][b]], p[s.seq[b], h, : c["lens"][b]], c["keep"], c["first"], c["recent"], s.end[b]) for h in range(s.nkv)] for b in range(c["n"])]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("c", EVICT, ids=lambda c: f"{c['lens']}-{c['keep']}-{c.get('book', '')}")
def test_evict(brrr, dev, c, inplace):
    import torch
    s = evict_setup(dev, c, 8)
    want = evict_want(s, c)
    old = [t.clone() for t in (s.k, s.v, s.weight, s.pos)]
    d = None if inplace else Setup(dev, 9, s.n_seq, s.nkv, s.hd, c["keep"] + 2, s.bf16, heads_outside=True)
    to = s if inplace else d
    untouched = [t.clone() for t in (to.k, to.v, to.weight, to.pos)]
    kept = torch.full((c["n"], s.nkv, c["keep"]), 5, dtype=torch.int32, device=dev)
    new_len = torch.zeros(c["n"], dtype=torch.int32, device=dev)
    s.view(brrr).evict(c["n"], s.up(c["lens"], np.int32), c["keep"], c["first"], c["recent"], s.up(s.end, np.int32), kept, seq=s.up(s.seq, np.int32) if "seq" in c else None,
                       dst=None if inplace else d.view(brrr), new_len=new_len)
    torch.cuda.synchronize()
    assert s.ok() and new_len.tolist() == [min(x, c["keep"]) for x in c["lens"]]
    for b in range(c["n"]):
        for h in range(s.nkv):
            src = want[b][h]
            assert kept[b, h].tolist() == src + [-1] * (c["keep"] - len(src))
            at = torch.tensor(src, dtype=torch.long, device=dev)
            for now, was, rest in zip((to.k, to.v, to.weight, to.pos), old, untouched):
                assert torch.equal(now[s.seq[b], h, : len(src)].nan_to_num(99.0), was[s.seq[b], h][at].nan_to_num(99.0))
                assert torch.equal(now[s.seq[b], h, len(src):].nan_to_num(99.0), rest[s.seq[b], h, len(src):].nan_to_num(99.0))
    idle = [q for q in range(s.n_seq) if q not in s.seq]
    for now, rest in zip((to.k, to.v, to.weight, to.pos), untouched):
        assert torch.equal(now[idle].nan_to_num(99.0), rest[idle].nan_to_num(99.0))


def test_evict_leaves_out(brrr, dev):
    import torch
    c = dict(n=5, lens=[30, 30, 36, -1, 30], keep=10, first=0, recent=0)
    s = evict_setup(dev, dict(c, lens=[30] * 5, seq=[1, 1, 0, 2, 0]), 3)
    old = [t.clone() for t in (s.k, s.weight)]
    kept, new_len = torch.zeros((5, 3, 10), dtype=torch.int32, device=dev), torch.zeros(5, dtype=torch.int32, device=dev)
    s.view(brrr).evict(5, s.up(c["lens"], np.int32), 10, 0, 0, None, kept, seq=s.up([1, 1, 0, 2, 9], np.int32), new_len=new_len)
    torch.cuda.synchronize()
    assert not s.ok() and bool((kept[1:] == -1).all()) and new_len.tolist() == [10, 30, 36, -1, 30]
    assert torch.equal(s.k[[0, 2]], old[0][[0, 2]])
    src = R.evict(old[1][1, 0, :30].cpu().numpy(), [0] * 30, 10, 0, 0, 0)
    assert kept[0, 0].tolist() == src


# ---------------------------------------------------------------- block means and chosen blocks
@pytest.mark.parametrize("block,bf16,hd", [(16, False, 64), (32, True, 128), (64, False, 128), (128, True, 64)])
def test_means(brrr, dev, block, bf16, hd):
    import torch
    s = Setup(dev, 3, 4, 2, hd, 5 * block + 7, bf16, pad=8)
    seq, since, lens = [3, 0, 1], [0, block + 1, 3 * block], [5 * block + 7, 3 * block - 1, 3 * block]
    for hint in (0, 1):
        means = torch.full((4, 2, 5, hd), 7.0, device=dev)
        s.view(brrr).means(3, s.up(lens, np.int32), block, means, seq=s.up(seq, np.int32), since=s.up(since, np.int32), len_hint=hint)
        torch.cuda.synchronize()
        want = np.full((4, 2, 5, hd), 7.0, np.float32)
        k = s.values()[0]
        for b in range(3):
            for j in range(since[b] // block, lens[b] // block):
                want[seq[b], :, j] = k[seq[b], :, j * block: (j + 1) * block].mean(1)
        assert s.ok() and np.array_equal(means.cpu().numpy(), want)      # both sums are good to 2^-50: the one rounding agrees
    means.fill_(7.0)
    s.view(brrr).means(3, s.up([-1, 5 * block + 8, block], np.int32), block, means, seq=s.up([0, 1, 4], np.int32))
    torch.cuda.synchronize()
    assert not s.ok() and (means == 7.0).all()


BLOCKS = [dict(lens=[1], block=16, nsel=1, first=0, local=1, heads=2, kv=2), dict(lens=[0, 16, 17], block=16, nsel=3, first=1, local=2, heads=8, kv=2),
          dict(lens=[500, 33, 499], block=16, nsel=5, first=1, local=1, heads=64, kv=8, sinks=True), dict(lens=[2000], block=32, nsel=20, first=0, local=3, heads=32, kv=4, hd=128),
          dict(lens=[640, 639], block=64, nsel=10, first=2, local=8, heads=12, kv=2, bf16=True), dict(lens=[3000], block=16, nsel=181, first=1, local=2, heads=5, kv=1, bf16=True, hd=128),
          dict(lens=[900 + i for i in range(70)], block=128, nsel=4, first=1, local=1, heads=16, kv=1, hd=128, prompt=True),
          dict(lens=[5000, 300], block=16, nsel=7, first=1, local=1, heads=6, kv=3, ties=True), dict(lens=[4100], block=16, nsel=200, first=0, local=1, heads=8, kv=1, ties=True)]


@pytest.mark.parametrize("c", BLOCKS, ids=lambda c: f"{c['lens'][:3]}-{c['block']}-{c['nsel']}-{c['heads']}-{c['kv']}")
def test_blocks(brrr, dev, c):
    import torch
    rows, hd, kv, block, nsel = len(c["lens"]), c.get("hd", 64), c["kv"], c["block"], c["nsel"]
    seq = [1] * rows if c.get("prompt") else list(range(rows))
    s = Setup(dev, 21, max(seq) + 1, kv, hd, max(c["lens"]) + 3, c.get("bf16", False), pad=8)
    q = s.f32(rows, c["heads"], hd)
    means = torch.full((s.n_seq, kv, s.cap // block, hd), float("nan"), device=dev)
    view = s.view(brrr)
    longest = {b: max(x for x, y in zip(c["lens"], seq) if y == b) for b in set(seq)}
    view.means(len(longest), s.up([longest[b] for b in longest], np.int32), block, means, seq=s.up(list(longest), np.int32))
    if c.get("ties"):       # few different means, some of them not numbers
        m = means.cpu().numpy()
        m[:] = s.f32(1, kv, 3, hd)[:, :, s.rng.integers(0, 3, m.shape[2])]
        m[0, 0, 5:9] = np.nan
        means.copy_(torch.from_numpy(m))
    for b in set(seq):
        s.k[b, :, longest[b]:] = float("nan"); s.v[b, :, longest[b]:] = float("inf")
    sinks = s.f32(c["heads"]) if c.get("sinks") else None
    out, lse = torch.full((rows, c["heads"] * hd), 7.0, device=dev), torch.full((rows, c["heads"]), 7.0, device=dev)
    sel = torch.full((rows, kv, nsel), 77, dtype=torch.int32, device=dev)
    scale = 1 / math.sqrt(hd)
    view.attn_blocks(rows, s.up(seq, np.int32) if c.get("prompt") else None, s.up(c["lens"], np.int32), block, means, nsel, c["first"], c["local"], s.up(q), c["heads"], out, scale, sel,
                     sinks=None if sinks is None else s.up(sinks), lse=lse)
    torch.cuda.synchronize()
    assert s.ok()
    k, v = s.values()
    m, got = means.cpu().numpy(), out.cpu().numpy().reshape(rows, c["heads"], hd)
    per = c["heads"] // kv
    want, want_lse = np.zeros(got.shape), np.zeros(got.shape[:2])
    for r in range(rows):
        for h in range(kv):
            chosen = R.choose(q[r, h * per: (h + 1) * per], m[seq[r], h], c["lens"][r], block, nsel, c["first"], c["local"])
            assert sel[r, h].tolist() == chosen + [-1] * (nsel - len(chosen))
            slots = [t for j in chosen for t in range(j * block, min((j + 1) * block, c["lens"][r]))]
            for g in range(h * per, (h + 1) * per):
                want[r, g], want_lse[r, g], _ = R.attend(q[r, g].astype(np.float64), k[seq[r], h], v[seq[r], h], slots, scale, None if sinks is None else float(sinks[g]))
    close(got, want)
    close_lse(lse.cpu().numpy(), want_lse)
    for hint in (1, 1 << 20):
        other = torch.zeros_like(out)
        view.attn_blocks(rows, s.up(seq, np.int32), s.up(c["lens"], np.int32), block, means, nsel, c["first"], c["local"], s.up(q), c["heads"], other, scale, sel, len_hint=hint,
                         sinks=None if sinks is None else s.up(sinks))
        torch.cuda.synchronize()
        close(other.cpu().numpy().reshape(want.shape), want)
    inplace = s.up(q).view(rows, -1)
    view.attn_blocks(rows, s.up(seq, np.int32), s.up(c["lens"], np.int32), block, means, nsel, c["first"], c["local"], inplace, c["heads"], inplace, scale, sel,
                     sinks=None if sinks is None else s.up(sinks))
    assert torch.equal(inplace, out)


def test_blocks_leave_out(brrr, dev):
    import torch
    s = Setup(dev, 6, 2, 2, 64, 50)
    means = torch.zeros((2, 2, 3, 64), device=dev)
    out, sel = torch.full((4, 4 * 64), 7.0, device=dev), torch.full((4, 2, 2), 77, dtype=torch.int32, device=dev)
    s.view(brrr).attn_blocks(4, s.up([0, 2, 1, -1], np.int32), s.up([20, 20, 51, 20], np.int32), 16, means, 2, 0, 1, s.up(s.f32(4, 4, 64)), 4, out, 0.125, sel)
    torch.cuda.synchronize()
    assert not s.ok() and (out[1:] == 7.0).all() and (sel[1:] == 77).all() and not (out[0] == 7.0).any()


# ---------------------------------------------------------------- together
def test_a_decoding_loop_with_drafts_and_a_budget(brrr, dev):
    """What a server does with the set: drafted rows appended, attended, the accepted path weighed and committed, caches pruned in place, block means renewed and
    one row attended over chosen blocks; each round against the restatement on the cache as it then stands."""
    import torch
    n, rows, heads, kv, hd, cap, keep = 3, 6, 8, 2, 64, 160, 96
    rng = np.random.default_rng(77)
    s = Setup(dev, 78, n, kv, hd, cap)
    rope = s.f32(4096, hd // 2, 2)
    rope /= np.linalg.norm(rope, axis=2, keepdims=True)
    view, i32 = s.view(brrr), lambda v: s.up(v, np.int32)
    lens, ends = [0, 40, 90], [0, 40, 90]
    for b in range(n):
        s.pos[b, :, : lens[b]] = torch.arange(lens[b], dtype=torch.int32)
    means = torch.zeros((n, kv, cap // 16, hd), device=dev)
    d_rope = s.up(rope)
    for turn in range(9):
        masks = [random_tree(rng, rows) for _ in range(n)]
        counts = [int(rng.integers(1, rows + 1)) for _ in range(n)]
        at = np.array([[ends[b] + R.depth(masks[b][i], i) for i in range(rows)] for b in range(n)], np.int32)
        x = s.f32(n, rows, (heads + 2 * kv) * hd)
        q, out, lse = torch.zeros((n, rows, heads * hd), device=dev), torch.zeros((n, rows, heads * hd), device=dev), torch.zeros((n, rows, heads), device=dev)
        dl, dc, dm = i32(lens), i32(counts), s.up(np.array(masks, np.uint64))
        view.append(n, rows, dl, s.up(x), n_head=heads, q=q, at=i32(at), rope=d_rope, n_rope=4096, count=dc)
        view.attn_tree(n, rows, dl, q, heads, out, 0.125, count=dc, mask=dm, lse=lse)
        k, v = s.values()
        want, _, weights = R.tree(q.double().cpu().numpy().reshape(n, rows, heads, hd), k, v, range(n), lens, counts, masks, 0.125)
        for b in range(n):
            close(out[b, : counts[b]].cpu().numpy().reshape(-1, heads, hd), want[b, : counts[b]])
        tips = [int(rng.integers(0, c)) for c in counts]
        paths = [[i for i in range(rows) if masks[b][tips[b]] >> i & 1] for b in range(n)]
        picked = [sum(1 << i for i in p) for p in paths]
        book = s.weight.double().cpu().numpy()
        for b, i, h, slots, w in weights:
            if picked[b] >> i & 1:
                book[b, h // 4, slots] += w
        view.weigh(n, rows, dl, q, heads, lse, 0.125, count=dc, mask=dm, picked=s.up(np.array(picked, np.uint64)))
        close(s.weight.cpu().numpy(), book)
        new_len = torch.zeros(n, dtype=torch.int32, device=dev)
        view.commit(n, rows, dl, i32([p + [-1] * (rows - len(p)) for p in paths]), i32([len(p) for p in paths]), new_len=new_len)
        lens = [a + len(p) for a, p in zip(lens, paths)]
        ends = [a + len(p) for a, p in zip(ends, paths)]
        assert new_len.tolist() == lens
        w, p = s.weight.cpu().numpy(), s.pos.cpu().numpy()
        src = [[R.evict(w[b, h, : lens[b]], p[b, h, : lens[b]], keep, 4, 16, ends[b]) for h in range(kv)] for b in range(n)]
        k, v = s.values()
        kept, pruned = torch.zeros((n, kv, keep), dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
        view.evict(n, new_len, keep, 4, 16, i32(ends), kept, new_len=pruned)
        lens = [min(a, keep) for a in lens]
        assert pruned.tolist() == lens
        for b in range(n):
            for h in range(kv):
                assert np.array_equal(s.k[b, h, : lens[b]].double().cpu().numpy(), k[b, h, src[b][h]])
                assert np.array_equal(s.pos[b, h, : lens[b]].cpu().numpy(), p[b, h, src[b][h]])
        view.means(n, pruned, 16, means)
        sel, o = torch.zeros((n, kv, 4), dtype=torch.int32, device=dev), torch.zeros((n, heads * hd), device=dev)
        q1 = q[:, 0].contiguous()
        view.attn_blocks(n, None, pruned, 16, means, 4, 1, 1, q1, heads, o, 0.125, sel)
        torch.cuda.synchronize()
        k, v = s.values()
        qn, mn = q1.cpu().numpy().reshape(n, heads, hd), means.cpu().numpy()
        for b in range(n):
            for h in range(heads):
                chosen = R.choose(qn[b, h // 4 * 4: h // 4 * 4 + 4], mn[b, h // 4], lens[b], 16, 4, 1, 1)
                assert [x for x in sel[b, h // 4].tolist() if x >= 0] == chosen
                slots = [t for j in chosen for t in range(16 * j, min(16 * j + 16, lens[b]))]
                close(o[b].cpu().numpy().reshape(heads, hd)[h], R.attend(qn[b, h].astype(np.float64), k[b, h // 4], v[b, h // 4], slots, 0.125)[0])
        assert s.ok()


def test_graphs_and_streams(brrr, dev):
    """The set captured into two graphs that are replayed on two streams at once over one cache (reading calls share nothing), and the writing calls in a graph of their own:
    the same bits as the eager calls; lengths are read when the graph runs."""
    import torch
    c = dict(n=2, rows=11, lens=[600, 410], heads=16, kv=2, hd=64, masks="tree")
    s = prepared_tree(dev, c)
    wide = prepared_tree(dev, dict(n=1, rows=64, lens=[700], heads=64, kv=4, hd=64, masks="tree", bf16=True))
    wq, wmask, wlen, wview = wide.up(wide.q), wide.up(np.array(wide.masks, np.uint64)), wide.up([700], np.int32), wide.view(brrr)
    view = s.view(brrr)
    s.k.nan_to_num_(0.0), s.v.nan_to_num_(0.0, 0.0, 0.0)
    n, rows = 2, 11
    q, mask, lens = s.up(s.q), s.up(np.array(s.masks, np.uint64)), s.up(s.lens, np.int32)
    means = torch.zeros((2, 2, s.cap // 16, 64), device=dev)
    view.means(2, lens, 16, means)
    q1 = q[:, 0].contiguous()

    def bufs():
        return (torch.zeros((n, rows, 16 * 64), device=dev), torch.zeros((n, rows, 16), device=dev), torch.zeros((2, 2, 5), dtype=torch.int32, device=dev), torch.zeros((2, 16 * 64), device=dev),
                torch.zeros((1, 64, 64 * 64), device=dev))

    def read(o, st):
        view.attn_tree(n, rows, lens, q, 16, o[0], 0.125, mask=mask, lse=o[1], stream=st)
        view.attn_blocks(2, None, lens, 16, means, 5, 1, 1, q1, 16, o[3], 0.125, o[2], stream=st)
        wview.attn_tree(1, 64, wlen, wq, 64, o[4], 0.125, mask=wmask, stream=st)
    eager = bufs()
    read(eager, None)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        o, g = bufs(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            read(o, torch.cuda.current_stream().cuda_stream)
        graphs.append(g), outs.append(o)
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, eager))
    lens.copy_(s.up([101, 3], np.int32))
    read(eager, None)
    for g in graphs:
        g.replay()
        torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, eager))
    # writing calls: append, weigh, commit, evict
    keep = 40
    x, at = s.up(s.f32(n, rows, 4 * 64)), s.up(np.arange(n * rows).reshape(n, rows), np.int32)
    path, npath, end = s.up(np.tile(np.arange(rows), (n, 1)), np.int32), s.up([3, 11], np.int32), s.up([120, 20], np.int32)
    kept, l1, l2 = torch.zeros((n, 2, keep), dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)

    def write(st):
        view.append(n, rows, lens, x, at=at, stream=st)
        view.weigh(n, rows, lens, q, 16, eager[1], 0.125, mask=mask, stream=st)
        view.commit(n, rows, lens, path, npath, new_len=l1, stream=st)
        view.evict(n, l1, keep, 2, 4, end, kept, new_len=l2, stream=st)
    start = [t.clone() for t in (*s.raw, s.weight, s.pos)]
    write(None)
    torch.cuda.synchronize()
    want = [t.clone() for t in (*s.raw, s.weight, s.pos, kept, l1, l2)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        write(torch.cuda.current_stream().cuda_stream)
    for t, a in zip((*s.raw, s.weight, s.pos), start):
        t.copy_(a)
    kept.zero_(), l1.zero_(), l2.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert l2.tolist() == [40, 14] and s.ok()
    for a, b in zip((*s.raw, s.weight, s.pos, kept, l1, l2), want):
        assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))


def test_memory_that_is_not_this_devices(brrr, dev):
    import torch
    host = torch.zeros((1, 1, 16, 64)).pin_memory()
    x = torch.zeros(64 * 3, device=dev)
    with pytest.raises(brrr.BrrrError):
        brrr.KvCache(host, host, 1, 1, 64, 16).attn_tree(1, 1, torch.zeros(1, dtype=torch.int32, device=dev), x, 1, x, 1.0)
