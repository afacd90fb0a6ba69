"""KV-cache operators at the limits of what their header allows, on the GPU: the largest finite numbers, more protected entries than are kept, the widest window,
destinations between the source's heads, long lists of blocks, every piece of an operand.  The restatement, the set-up and, where none is derived here, the tolerances
are those of test_gpu_kv.py."""
import math

import numpy as np
import pytest

import kv_ref as R
from test_gpu_kv import Setup, close, close_lse, prepared_tree, reference, run_tree

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the largest finite numbers
def fill_idle(s, bf16):
    """What no row sees holds the type's largest and lowest value in turn."""
    import torch
    big = torch.finfo(torch.bfloat16 if bf16 else torch.float32).max
    sign = torch.where(torch.arange(s.hd, device=s.dev) % 2 == 0, 1.0, -1.0).to(s.k.dtype)
    for x in (s.k, s.v):
        idle = ~torch.isfinite(x[..., 0])
        x[idle] = sign * big
    return big, sign


LARGEST = [dict(n=2, rows=1, lens=[72, 9], heads=16, kv=2, masks="chain", sinks=True), dict(n=2, rows=7, lens=[301, 33], heads=8, kv=4, masks="tree", counts=[7, 3], window=37),
           dict(n=1, rows=64, lens=[700], heads=32, kv=2, masks="tree"), dict(n=2, rows=64, lens=[511, 1090], heads=32, kv=2, masks="any", window=64, sinks=True)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("c", LARGEST, ids=lambda c: "-".join(str(c[k]) for k in ("n", "rows", "lens", "heads", "kv", "masks")))
def test_tree_largest_numbers_in_slots_that_nobody_sees(brrr, dev, c, hd, bf16):
    import torch
    c = dict(c, hd=hd, bf16=bf16)
    s = prepared_tree(dev, c)
    fill_idle(s, bf16)
    want, want_lse, weights = reference(s, c, s.up(s.q), s.scale)
    for hint in (0, 1):              # a small hint: the kernel of 16-row tiles
        out, lse = run_tree(brrr, s, c, hint=hint)
        assert s.ok()
        for b in range(c["n"]):
            m = s.counts[b]
            close(out[b, :m].cpu().numpy().reshape(m, c["heads"], hd), want[b, :m].cpu().numpy())
            close_lse(lse[b, :m].cpu().numpy(), want_lse[b, :m].cpu().numpy())
    s.view(brrr).weigh(c["n"], c["rows"], s.up(s.lens, np.int32), s.up(s.q), c["heads"], lse, s.scale, count=s.up(s.counts, np.int32),
                       mask=None if c["masks"] == "chain" else s.up(np.array(s.masks, np.uint64)), window=s.window)
    torch.cuda.synchronize()
    book = torch.zeros(s.weight.shape, dtype=torch.float64, device=dev)
    for b in range(c["n"]):
        book[b, :, : s.lens[b] + s.counts[b]] += weights[b].sum(0).view(c["kv"], c["heads"] // c["kv"], -1).sum(1)
    close(s.weight.cpu().numpy(), book.cpu().numpy())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("at", [7, 41, 62])
def test_tree_rows_that_see_the_largest_value(brrr, dev, at, hd, bf16):
    """One slot's value is the largest finite one - seen by all rows (7, in a step that everybody sees whole), by the shallow ones (41), by one drafted row and those
    behind it (62): weighted it stays in single precision, and the others do not notice it."""
    import torch
    c = dict(n=1, rows=9, lens=[60], heads=8, kv=2, hd=hd, masks="tree", bf16=bf16)
    s = prepared_tree(dev, c)
    s.masks, s.window = [[1, 3, 5, 9, 16 | 1, 32 | 2 | 1, 64, 128 | 64, 256]], 20 if at == 41 else 0
    s.k.nan_to_num_(0.1), s.v.nan_to_num_(0.2, 0.3, 0.4)
    big = torch.finfo(s.v.dtype).max
    s.v[0, :, at, ::2], s.v[0, :, at, 1::2] = big, -big
    k, v = s.values()
    want, want_lse, _ = R.tree(s.q.astype(np.float64), k, v, [0], [60], [9], s.masks, s.scale, s.window)
    out, lse = run_tree(brrr, s, c)
    for i in range(9):
        close(out[0, i].cpu().numpy().reshape(8, hd), want[0, i])
    close_lse(lse.cpu().numpy(), want_lse)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads", [8, 32])
def test_blocks_largest_numbers_behind_the_end(brrr, dev, heads, hd, bf16):
    import torch
    kv, lens, block, nsel = 2, [500, 33, 5], 32, 4
    s = Setup(dev, 13, 3, kv, hd, 520, bf16)
    means, view = torch.zeros((3, kv, 520 // block, hd), device=dev), s.view(brrr)
    view.means(3, s.up(lens, np.int32), block, means)
    for b in range(3):
        s.k[b, :, lens[b]:] = float("nan"); s.v[b, :, lens[b]:] = float("nan")
    fill_idle(s, bf16)
    q = s.f32(3, heads, hd)
    out, lse, sel = torch.zeros((3, heads * hd), device=dev), torch.zeros((3, heads), device=dev), torch.zeros((3, kv, nsel), dtype=torch.int32, device=dev)
    view.attn_blocks(3, None, s.up(lens, np.int32), block, means, nsel, 1, 1, s.up(q), heads, out, 0.125, sel, lse=lse)
    torch.cuda.synchronize()
    assert s.ok()
    k, v = s.values()
    per, m = heads // kv, means.cpu().numpy()
    for r in range(3):
        for h in range(heads):
            chosen = R.choose(q[r, h // per * per: (h // per + 1) * per], m[r, h // per], lens[r], block, nsel, 1, 1)
            slots = [t for j in chosen for t in range(j * block, min((j + 1) * block, lens[r]))]
            want, z, _ = R.attend(q[r, h].astype(np.float64), k[r, h // per], v[r, h // per], slots, 0.125)
            close(out[r].cpu().numpy().reshape(heads, hd)[h], want)
            close_lse(lse[r, h].cpu().numpy()[None], np.array([z]))


# ---------------------------------------------------------------- more protected entries than are kept
CROWDED = [dict(lens=[5], keep=3, first=0, recent=1, spread=1, cap=8, kv=1), dict(lens=[700, 31], keep=50, first=20, recent=30, spread=40, cap=705),
           dict(lens=[700, 333], keep=50, first=50, recent=0, spread=60, cap=705, book="odd"), dict(lens=[3000, 64], keep=64, first=0, recent=64, spread=3000, cap=3001, book="ties"),
           dict(lens=[4096], keep=1000, first=500, recent=0, spread=2048, cap=4096), dict(lens=[4096], keep=1025, first=1025, recent=0, spread=1, cap=4096, book="odd"),
           dict(lens=[50001], keep=1000, first=700, recent=300, spread=2000, cap=50010, kv=1, book="odd"), dict(lens=[47000], keep=8001, first=1, recent=0, spread=3, cap=47001, kv=1)]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("c", CROWDED, ids=lambda c: f"{c['lens']}-{c['keep']}-{c['spread']}-{c.get('book', '')}")
def test_evict_with_more_protected_entries_than_are_kept(brrr, dev, c, inplace):
    """Positions that many entries share: among the protected ones the larger weight comes first, NaN last of them and still before every other entry."""
    import torch
    n, nkv, keep, first, recent = len(c["lens"]), c.get("kv", 2), c["keep"], c["first"], c["recent"]
    s = Setup(dev, 17, n, nkv, 64, c["cap"])
    w = np.exp(2 * s.f32(n, nkv, s.cap))
    if c.get("book") == "ties":
        w = s.rng.integers(0, 3, w.shape)
    if c.get("book") == "odd":
        w = s.rng.choice(np.float32([0.0, -0.0, np.nan, -np.nan, np.inf, -np.inf, -1.0, 1e-42, 2.0, 3.0e38]), w.shape)
    if c["lens"] == [5]:
        w[0, 0, :5] = [1, 2, 3, 4, 5]
    s.weight.copy_(torch.from_numpy(w.astype(np.float32)))
    s.pos.copy_(torch.from_numpy(s.rng.integers(0, c["spread"], w.shape).astype(np.int32)))
    end = c["spread"]
    weight, pos = s.weight.cpu().numpy(), s.pos.cpu().numpy()
    old = [t.clone() for t in (s.k, s.v, s.weight, s.pos)]
    d = s if inplace else Setup(dev, 18, n, nkv, 64, keep)
    kept, new_len = torch.zeros((n, nkv, keep), dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    s.view(brrr).evict(n, s.up(c["lens"], np.int32), keep, first, recent, s.up([end] * n, np.int32), kept, dst=None if inplace else d.view(brrr), new_len=new_len)
    torch.cuda.synchronize()
    assert s.ok() and new_len.tolist() == [min(x, keep) for x in c["lens"]]
    for b in range(n):
        for h in range(nkv):
            src = R.evict(weight[b, h, : c["lens"][b]], pos[b, h, : c["lens"][b]], keep, first, recent, end)
            assert kept[b, h].tolist() == src + [-1] * (keep - len(src))
            if c["lens"] == [5]:
                assert sorted(src) == [2, 3, 4]
            at = torch.tensor(src, dtype=torch.long, device=dev)
            for now, was in zip((d.k, d.v, d.weight, d.pos), old):
                assert torch.equal(now[b, h, : len(src)].nan_to_num(99.0), was[b, h][at].nan_to_num(99.0))


# ---------------------------------------------------------------- the widest window
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,heads,kv,hd", [(1, 8, 8, 64), (5, 16, 4, 128), (64, 32, 2, 64), (64, 32, 2, 128)])
def test_a_window_that_hides_nothing_changes_no_bit(brrr, dev, rows, heads, kv, hd, bf16):
    """A window is a limit on what is seen and on the work, never more work than without one: one that hides nothing splits the slots as none does, up to the largest."""
    import torch
    c = dict(n=1, rows=rows, lens=[2000], heads=heads, kv=kv, hd=hd, masks="tree", bf16=bf16)
    s = prepared_tree(dev, c)
    want, want_lse = run_tree(brrr, s, c)
    for window in (1 << 20, (1 << 31) - 64, (1 << 31) - 1):
        s.window = window
        out, lse = run_tree(brrr, s, c)
        assert s.ok() and torch.equal(out, want) and torch.equal(lse, want_lse)
        books = []
        for x in (0, window):
            s.weight.zero_()
            s.view(brrr).weigh(1, rows, s.up(s.lens, np.int32), s.up(s.q), heads, lse, s.scale, mask=s.up(np.array(s.masks, np.uint64)), window=x)
            books.append(s.weight.clone())
        assert torch.equal(*books) and bool(books[0].any())


# ---------------------------------------------------------------- destinations between the source's heads
@pytest.mark.parametrize("layout", ["sequences", "heads", "halves"])
def test_evict_into_rows_between_the_sources(brrr, dev, layout):
    """One allocation holds both caches, whose heads alternate: sequences inside a head, heads of a sequence one by one, a source in the first half of every row."""
    import torch
    n, nkv, hd, cap, keep = 2, 3, 64, 40, 16
    rng = np.random.default_rng(4)
    shape = {"sequences": (nkv, 2 * n, cap * hd), "heads": (n, nkv, 2, cap * hd), "halves": (n, 2 * nkv, cap * hd)}[layout]
    raw = [torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dev) for _ in range(2)]
    if layout == "sequences":
        at, strides = [(0, 0), (0, n)], dict(head_stride=2 * n * cap * hd, seq_stride=cap * hd)
        rows = lambda x, i: x[:, i * n: (i + 1) * n].transpose(0, 1)  # noqa: E731
    elif layout == "heads":
        at, strides = [(0, 0, 0), (0, 0, 1)], dict(head_stride=2 * cap * hd, seq_stride=2 * nkv * cap * hd)
        rows = lambda x, i: x[:, :, i]  # noqa: E731
    else:
        at, strides = [(0, 0), (0, nkv)], dict(head_stride=cap * hd, seq_stride=2 * nkv * cap * hd)
        rows = lambda x, i: x[:, i * nkv: (i + 1) * nkv]  # noqa: E731
    weight, pos = torch.rand((2, n, nkv, cap), device=dev), torch.arange(cap, dtype=torch.int32, device=dev).repeat(2, n, nkv, 1)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    src, dst = (brrr.KvCache(raw[0][i], raw[1][i], n, nkv, hd, cap, weight=weight[j], pos=pos[j], err=err, **strides) for j, i in enumerate(at))
    old, books = [x.clone() for x in raw], weight.clone()
    lens, kept = [33, 40], torch.zeros((n, nkv, keep), dtype=torch.int32, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    src.evict(n, i32(lens), keep, 2, 3, i32(lens), kept, dst=dst)
    torch.cuda.synchronize()
    assert int(err) == 0
    for x, was in zip(raw, old):
        assert torch.equal(rows(x, 0), rows(was, 0)) and torch.equal(rows(x, 1).unflatten(-1, (cap, hd))[:, :, keep:], rows(was, 1).unflatten(-1, (cap, hd))[:, :, keep:])
    for b in range(n):
        for h in range(nkv):
            want = R.evict(books[0, b, h, : lens[b]].cpu().numpy(), list(range(lens[b])), keep, 2, 3, lens[b])
            assert kept[b, h].tolist() == want
            for x, was in zip(raw, old):
                assert torch.equal(rows(x, 1)[b, h].view(cap, hd)[:keep], rows(was, 0)[b, h].view(cap, hd)[torch.tensor(want, device=dev)])
            assert torch.equal(weight[1, b, h, :keep], books[0, b, h][torch.tensor(want, device=dev)])


# ---------------------------------------------------------------- long lists of blocks
@pytest.mark.parametrize("hd,bf16,heads", [(64, True, 4), (128, False, 16), (128, True, 9)])
@pytest.mark.parametrize("blocks,nsel,ties", [(1023, 5, False), (1025, 40, True), (5000, 256, False), (5001, 17, True), (16384, 33, True), (16384, 256, False)])
def test_blocks_of_long_caches(brrr, dev, blocks, nsel, ties, hd, bf16, heads):
    """Up to the largest number of blocks, full and short sequences in one call: the choice is the restatement's, block by block."""
    import torch
    block, rows, kv = 16, 3, 1
    s = Setup(dev, 29, 1, kv, hd, blocks * block + 3, bf16)
    lens = [s.cap, blocks * block // 3 + 5, block]
    means = torch.full((1, kv, blocks, hd), float("nan"), device=dev)
    view = s.view(brrr)
    view.means(1, s.up([s.cap], np.int32), block, means)
    if ties:
        few = s.up(s.f32(40, hd) / 4)
        means[0, 0] = few[torch.from_numpy(s.rng.integers(0, 40, blocks)).to(dev)]
        means[0, 0, 7: blocks: 100] = float("nan")
    q = s.f32(rows, heads, hd)
    m = means[0, 0].cpu().numpy()
    k, v = s.values()
    chosen = [R.choose(q[r], m, lens[r], block, nsel, 1, 2) for r in range(rows)]
    for hint in (0, 100):
        out, lse = torch.zeros((rows, heads * hd), device=dev), torch.zeros((rows, heads), device=dev)
        sel = torch.full((rows, kv, nsel), 77, dtype=torch.int32, device=dev)
        view.attn_blocks(rows, s.up([0] * rows, np.int32), s.up(lens, np.int32), block, means, nsel, 1, 2, s.up(q), heads, out, 1 / math.sqrt(hd), sel, len_hint=hint, lse=lse)
        torch.cuda.synchronize()
        assert s.ok()
        for r in range(rows):
            assert sel[r, 0].tolist() == chosen[r] + [-1] * (nsel - len(chosen[r]))
            slots = [t for j in chosen[r] for t in range(j * block, min((j + 1) * block, lens[r]))]
            for h in range(heads):
                want, z, _ = R.attend(q[r, h].astype(np.float64), k[0, 0], v[0, 0], slots, 1 / math.sqrt(hd))
                close(out[r].cpu().numpy().reshape(heads, hd)[h], want)
                close_lse(lse[r, h].cpu().numpy()[None], np.array([z]))


# ---------------------------------------------------------------- every piece of an operand
def cut16(x):
    """x without what a third piece of eight bits would hold."""
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32).astype(np.float64) + \
        (np.ascontiguousarray(x - (x.view(np.uint32) & 0xFFFF0000).view(np.float32)).view(np.uint32) & 0xFFFF0000).view(np.float32)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("hint", [0, 1])
def test_no_piece_of_an_operand_is_lost(brrr, dev, hint, hd, bf16):
    """Rows of one or two slots, where sums hide nothing: hint 0 goes to the kernels of 128-row tiles (three pieces of eight bits), 1 to those of 16 rows (tf32 twice).

    Relative bounds, each from its roundings.  VALUE, a row that sees one slot returns its value: 24 bits in three pieces are exact, two tf32 parts leave out 2^-22 at
    most, the division and the product 2^-22 + 2^-24: 2^-20.  SCORE, the log-sum of such a row whose query has one dimension is one product: what is left out of a
    product 2^-21 (mid x lo twice; tf32: 2^-21 as well), three additions that matter, truncated, 3 x 2^-23, five roundings of the scale and the logarithms'
    factors 5 x 2^-24: 1.2e-6 < 2^-19.  WEIGHT, values 1 and 0 under scores 0 and s with |s| < 3: an exponent of 4.4 off by 3 x 2^-24 of it changes a weight by
    5.5e-7, the power, the pieces and the division by 2^-22 each: 1.3e-6 < 2^-19.  BOOK, e^s with s < 8: 8 times the bound of a score, 9.6e-6, and the power's 2^-22: 1.2e-5.
    16 bits of one operand are off by up to 2^-15: each bound is checked to see that."""
    import torch
    value, score, weight, book = 2.0**-20, 2.0**-19, 2.0**-19, 1.2e-5
    rows, heads, kv, cap = 64, 32, 2, 4000
    per, half = heads // kv, rows // 2
    s = Setup(dev, 41, 1, kv, hd, cap, bf16)
    view, out, lse = s.view(brrr), torch.zeros((1, rows, heads * hd), device=dev), torch.zeros((1, rows, heads), device=dev)

    def run(masks, q):
        view.attn_tree(1, rows, s.up([0], np.int32), s.up(q), heads, out, 0.125, mask=s.up(np.array([masks], np.uint64)), len_hint=hint, lse=lse)
        torch.cuda.synchronize()
        assert s.ok()
        return out.double().cpu().numpy().reshape(rows, heads, hd), lse.double().cpu().numpy()[0]

    def off(got, want):
        return (np.abs(got - want) / np.abs(want)).max()

    # one slot each: its value, its score
    k, v = s.values()
    q = np.zeros((rows, heads, hd), np.float32)
    i, h = np.meshgrid(np.arange(rows), np.arange(heads), indexing="ij")
    d = (5 * i + h) % hd
    key = k[0, h // per, i, d]
    q[i, h, d] = (s.rng.uniform(32, 64, (rows, heads)) / key).astype(np.float32)          # scaled scores of 4 to 8
    one = q[i, h, d]
    o, z = run([1 << i for i in range(rows)], q)
    assert off(o, v[0, h // per, i]) < value
    assert off(z, 0.125 * one.astype(np.float64) * key) < score < off(0.125 * cut16(one) * key, 0.125 * one.astype(np.float64) * key)
    s.weight.zero_()
    view.weigh(1, rows, s.up([0], np.int32), s.up(q), heads, torch.zeros_like(lse), 0.125, mask=s.up(np.array([[1 << i for i in range(rows)]], np.uint64)))
    want, less = (np.exp(0.125 * x * key).reshape(rows, kv, per).sum(2).T for x in (one.astype(np.float64), cut16(one)))
    got = s.weight[0, :, :rows].double().cpu().numpy()
    assert off(got, want) < book < off(less, want)
    if not bf16:
        k32, v32 = key.astype(np.float32), v[0].astype(np.float32)
        assert score < off(one * cut16(k32), one * key) and value < off(cut16(v32), v[0]) and book < off(np.exp(0.125 * one * cut16(k32)), np.exp(0.125 * one * key))
    # two slots: row i < 32 sees itself, of key 0 and value 1, and slot 32 + i, whose value is 0
    s.k[:, :, :half], s.v[:, :, :half], s.v[:, :, half: rows] = 0.0, 1.0, 0.0
    s.k[:, :, half: rows] = 1.0
    x = s.rng.uniform(0.5, 3, (rows, heads)).astype(np.float32)
    q[:] = 0.0
    q[:, :, 3] = 8 * x
    o, _ = run([1 << i | 1 << (half + i % half) for i in range(rows)], q)
    want = 1 / (1 + np.exp(x[:half].astype(np.float64)))
    p = np.exp(-x[:half].astype(np.float64))
    assert off(o[:half], want[:, :, None]) < weight < off(cut16(p.astype(np.float32)) / (1 + p), want)
