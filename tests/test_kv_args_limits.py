"""Refusals of the KV-cache operators at the limits of their arguments; nothing here touches a device."""
import ctypes as C

import pytest

from test_kv_args import ARG, P, view

CUDA = 3            # what an accepted call returns where there is no device, or where its memory is nobody's


@pytest.mark.parametrize("scale,want", [(1.5e38, True), (-3.4e38, True), (1.0001e38, True), (1e38, False), (-1e38, False), (0.0, False)])
def test_scales_whose_powers_of_two_leave_single_precision(brrr, scale, want):
    """log2(e) x 3e38 is infinite, and a score of zero times that no number."""
    L, v = brrr.lib(), view(brrr)
    r = C.byref(v)
    calls = [L.brrr_attn_tree(r, 1, 1, None, P, None, None, 0, P, 4, scale, 0, None, P, None, None), L.brrr_kv_weigh(r, 1, 1, None, P, None, None, None, 0, P, 4, scale, 0, P, None),
             L.brrr_attn_blocks(r, 1, None, P, 16, P, 4, 1, 1, 0, P, 4, scale, None, P, P, None, None)]
    if want:
        assert calls == [ARG] * 3
    elif not __import__("torch").cuda.is_available():
        assert calls == [CUDA] * 3


class OnDevice:
    """A tensor as one of device 0 would look to the class."""

    def __init__(self, x):
        self.x, self.dtype, self.shape, self.device = x, x.dtype, x.shape, "cuda:0"

    def __getattr__(self, name):
        return getattr(self.x, name)

    def get_device(self):
        return 0

    def data_ptr(self):
        return P


def test_the_class_reads_no_array_as_another_type(brrr):
    """Lengths that are floats, or queries that are integers, have the right size and would be read as what they are not."""
    import torch

    def a(dtype, n=64 * 12 * 3):
        return OnDevice(torch.zeros(n, dtype=dtype))
    f, i, w, h = a(torch.float32), a(torch.int32), a(torch.int64), a(torch.float16)
    kv = brrr.KvCache(P, 2 * P, 3, 4, 64, 16, weight=f, pos=i, err=i)
    for bad in (dict(weight=i), dict(pos=f), dict(err=f), dict(pos=w), dict(weight=a(torch.float64))):
        with pytest.raises(brrr.BrrrError, match="is wanted"):
            brrr.KvCache(P, 2 * P, 3, 4, 64, 16, **{**dict(weight=f, pos=i, err=i), **bad})
    i = a(torch.int32)
    calls = {
        "append": (lambda **k: kv.append(1, 1, k.pop("length"), k.pop("qkv"), n_head=4, n_rope=1, **k), dict(length=i, qkv=f, seq=i, count=i, at=i, rope=f, q=f)),
        "attn_tree": (lambda **k: kv.attn_tree(1, 1, k.pop("length"), k.pop("q"), 4, k.pop("out"), 1.0, **k), dict(length=i, q=f, out=f, seq=i, count=i, mask=w, sinks=f, lse=f)),
        "commit": (lambda **k: kv.commit(1, 1, k.pop("length"), k.pop("path"), k.pop("npath"), **k), dict(length=i, path=i, npath=i, seq=i, new_len=i)),
        "weigh": (lambda **k: kv.weigh(1, 1, k.pop("length"), k.pop("q"), 4, k.pop("lse"), 1.0, **k), dict(length=i, q=f, lse=f, seq=i, count=i, mask=w, picked=w)),
        "evict": (lambda **k: kv.evict(1, k.pop("length"), 4, 1, 1, k.pop("end"), k.pop("map"), **k), dict(length=i, end=i, map=i, seq=i, new_len=i)),
        "means": (lambda **k: kv.means(1, k.pop("length"), 16, k.pop("means"), **k), dict(length=i, means=f, seq=i, since=i)),
        "attn_blocks": (lambda **k: kv.attn_blocks(1, k.pop("seq"), k.pop("length"), 16, k.pop("means"), 4, 1, 1, k.pop("q"), 4, k.pop("out"), 1.0, k.pop("sel"), **k),
                        dict(seq=i, length=i, means=f, q=f, out=f, sel=i, sinks=f, lse=f)),
    }
    for name, (call, good) in calls.items():
        with pytest.raises(brrr.BrrrError, match=f"brrr_(kv|attn)_{name.split('_')[-1]}"):          # the arrays are taken; the memory is nobody's
            call(**good)
        for arg, x in good.items():
            for bad in (f, i, w, h):
                if bad.dtype != x.dtype:
                    with pytest.raises(brrr.BrrrError, match="is wanted"):
                        call(**{**good, arg: bad})
    unsigned = dict(length=a(torch.uint32), q=f, out=f, mask=a(torch.uint64))
    with pytest.raises(brrr.BrrrError, match="brrr_attn_tree"):
        calls["attn_tree"][0](**unsigned)


def test_a_destination_may_stand_between_the_sources_heads(brrr):
    """Random layouts of two views over one stretch of memory: refused exactly where two rows share a byte."""
    import random

    import torch
    L, rng, seen = brrr.lib(), random.Random(5), {True: 0, False: 0}

    def layout():
        n_seq, nkv, cap = rng.randint(1, 3), 2, rng.randint(1, 3)
        head = cap * 64
        inner = head + rng.choice([0, 0, 64, 200])
        if rng.random() < 0.5:
            hs, ss = inner, inner * (nkv - 1) + head + rng.choice([0, 8, 400, 1000])
        else:
            hs, ss = inner * (n_seq - 1) + head + rng.choice([0, 8, 400, 1000]), inner
        if rng.random() < 0.2:
            hs = ss = 0
        return dict(n_seq=n_seq, n_head_kv=nkv, cap=cap, head_stride=hs, seq_stride=ss)

    def bytes_of(at, c):
        head = c["cap"] * 64
        hs = c["head_stride"] or head
        ss = c["seq_stride"] or hs * c["n_head_kv"]
        return {at + 4 * (s * ss + h * hs) + i for s in range(c["n_seq"]) for h in range(c["n_head_kv"]) for i in range(0, 4 * head, 16)}
    for _ in range(600):
        a, b = layout(), layout()
        at, to = P, P + 16 * rng.randint(0, 700)
        src, dst = view(brrr, **a, k=at, v=2 * P), view(brrr, **b, k=to, v=6 * P, weight=7 * P, pos=8 * P)
        overlap = bool(bytes_of(at, a) & bytes_of(to, b))
        got = L.brrr_kv_evict(C.byref(src), C.byref(dst), 1, None, P, 1, 0, 0, None, P, None, 0, None)
        seen[overlap] += 1
        assert (got == ARG) == overlap or (not overlap and torch.cuda.is_available()), (a, b, to - at)
        assert got in (ARG, CUDA)
    assert min(seen.values()) > 50, seen
