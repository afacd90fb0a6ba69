"""Refusals of the KV-cache operators: everything the host can see is checked before anything touches a device."""
import ctypes as C

import pytest

ARG, RANGE = 1, 5
P = 1 << 20          # an aligned address nobody reads


def view(B, **kw):
    d = dict(k=P, v=2 * P, type=0, n_seq=3, n_head_kv=4, head_dim=64, cap=100, head_stride=0, seq_stride=0, weight=3 * P, pos=4 * P, err=5 * P)
    d.update(kw)
    return B._lib.Kv(*[d[n] for n, _ in B._lib.Kv._fields_])


BAD_VIEWS = [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=2 * P + 4), dict(type=2), dict(type=-1), dict(n_seq=0), dict(n_head_kv=0), dict(n_head_kv=513),
             dict(head_dim=96), dict(head_dim=0), dict(cap=0), dict(cap=(1 << 19) + 1), dict(head_stride=-64), dict(head_stride=6404), dict(head_stride=6392),
             dict(seq_stride=6400 * 4 - 8), dict(seq_stride=6408), dict(n_head_kv=1, head_stride=8, seq_stride=6392), dict(head_stride=6400, seq_stride=1 << 51),
             dict(weight=3 * P + 2), dict(pos=4 * P + 1), dict(err=5 * P + 3)]


@pytest.mark.parametrize("bad", BAD_VIEWS, ids=str)
def test_views_that_describe_no_cache(brrr, bad):
    L, v = brrr.lib(), view(brrr, **bad)
    r = C.byref(v)
    assert L.brrr_kv_append(r, 1, 1, None, P, None, None, P, 0, 4, None, 0, None, None) == ARG
    assert L.brrr_attn_tree(r, 1, 1, None, P, None, None, 0, P, 4, 1.0, 0, None, P, None, None) == ARG
    assert L.brrr_kv_commit(r, 1, 1, None, P, P, P, None, None) == ARG
    assert L.brrr_kv_weigh(r, 1, 1, None, P, None, None, None, 0, P, 4, 1.0, 0, P, None) == ARG
    assert L.brrr_kv_evict(r, None, 1, None, P, 10, 0, 0, None, P, None, 0, None) == ARG
    assert L.brrr_kv_means(r, 1, None, None, P, 16, 0, P, None) == ARG
    assert L.brrr_attn_blocks(r, 1, None, P, 16, P, 4, 1, 1, 0, P, 4, 1.0, None, P, P, None, None) == ARG


def test_no_view(brrr):
    L = brrr.lib()
    assert L.brrr_attn_tree(None, 1, 1, None, P, None, None, 0, P, 4, 1.0, 0, None, P, None, None) == ARG
    assert L.brrr_kv_commit(None, 1, 1, None, P, P, P, None, None) == ARG


def refuse(fn, good, cases, want=ARG):
    """fn(**arguments) with one argument at a time replaced."""
    for name, values in cases.items():
        for x in values:
            assert fn(**{**good, name: x}) == want, (name, x)


def test_append(brrr):
    L, v = brrr.lib(), view(brrr)

    def call(n=1, rows=1, seq=None, len=P, count=None, at=None, qkv=P, ld=0, nh=8, rope=None, n_rope=0, q=None):
        return L.brrr_kv_append(C.byref(v), n, rows, seq, len, count, at, qkv, ld, nh, rope, n_rope, q, None)
    refuse(call, {}, dict(n=[0, -1, 4, 65536], rows=[0, -1, 101], len=[None], qkv=[None, P + 4], ld=[8, 1020, 1026], nh=[-1, 3, 68], q=[P + 8], rope=[P]))
    refuse(call, dict(nh=0), dict(q=[P]))
    refuse(call, dict(rope=P), dict(n_rope=[0, -5]))


def test_tree_and_weigh(brrr):
    L, v, bare = brrr.lib(), view(brrr), view(brrr, weight=None)

    def tree(n=1, rows=1, seq=None, len=P, count=None, mask=None, q=P, nh=8, scale=1.0, window=0, sinks=None, out=P, lse=None):
        return L.brrr_attn_tree(C.byref(v), n, rows, seq, len, count, mask, 0, q, nh, scale, window, sinks, out, lse, None)

    def weigh(n=1, rows=1, seq=None, len=P, count=None, mask=None, picked=None, q=P, nh=8, scale=1.0, window=0, lse=P, v=v):
        return L.brrr_kv_weigh(C.byref(v), n, rows, seq, len, count, mask, picked, 0, q, nh, scale, window, lse, None)
    both = dict(n=[0, -1, 4, 65536], rows=[0, 65, -2], seq=[P + 2], len=[None, P + 1], count=[P + 2], mask=[P + 4], q=[None, P + 4], nh=[0, -4, 6, 68], window=[-1],
                scale=[float("nan"), float("inf"), -float("inf")])
    refuse(tree, {}, {**both, "out": [None, P + 8], "sinks": [P + 1], "lse": [P + 2]})
    refuse(weigh, {}, {**both, "picked": [P + 4], "lse": [None, P + 2], "v": [bare]})


def test_commit(brrr):
    L, v = brrr.lib(), view(brrr)

    def call(n=1, rows=1, len=P, path=P, npath=P, new_len=None):
        return L.brrr_kv_commit(C.byref(v), n, rows, None, len, path, npath, new_len, None)
    refuse(call, {}, dict(n=[0, 4], rows=[0, 65], len=[None], path=[None], npath=[None], new_len=[P]))


def test_evict(brrr):
    L, v = brrr.lib(), view(brrr)

    def call(v=v, dst=None, n=1, len=P, keep=50, first=4, recent=8, end=P, map=P, new_len=None):
        return L.brrr_kv_evict(C.byref(v), None if dst is None else C.byref(dst), n, None, len, keep, first, recent, end, map, new_len, 0, None)
    far = dict(k=16 * P, v=17 * P, weight=18 * P, pos=19 * P)
    size = 3 * 4 * 100 * 64 * 4
    refuse(call, {}, dict(v=[view(brrr, weight=None), view(brrr, pos=None)], n=[0, 4, 65536], len=[None], keep=[0, -1, 101, 11], first=[-1, 51, 43], recent=[-1, 47], end=[None],
                          map=[None], new_len=[P]))
    refuse(call, {}, dict(dst=[view(brrr), view(brrr, **{**far, "type": 1}), view(brrr, **{**far, "n_head_kv": 2}), view(brrr, **{**far, "head_dim": 128}),
                               view(brrr, **{**far, "cap": 49}), view(brrr, **{**far, "weight": None}), view(brrr, **{**far, "pos": None}),
                               view(brrr, **{**far, "k": P + size - 16}), view(brrr, **{**far, "v": P}), view(brrr, **{**far, "pos": 3 * P})]))
    refuse(call, dict(n=3), dict(dst=[view(brrr, **{**far, "n_seq": 2})]))


def test_means_and_blocks(brrr):
    L, v = brrr.lib(), view(brrr)

    def means(n=1, len=P, block=16, means=P):
        return L.brrr_kv_means(C.byref(v), n, None, None, len, block, 0, means, None)

    def blocks(v=v, rows=1, len=P, block=16, means=P, nsel=4, first=1, local=1, q=P, nh=8, sel=P, out=P):
        return L.brrr_attn_blocks(C.byref(v), rows, None, len, block, means, nsel, first, local, 0, q, nh, 1.0, None, sel, out, None, None)
    refuse(means, {}, dict(n=[0, 4], len=[None], block=[0, 8, 48, 256], means=[None, P + 8]))
    refuse(blocks, {}, dict(rows=[0, 4, 65536], len=[None], block=[0, 24], means=[None, P + 4], nsel=[0, 257, 1], first=[-1, 4], local=[0, 4], q=[None, P + 4], nh=[0, 5, 68], sel=[None],
                            out=[None, P + 4]))
    refuse(blocks, {}, dict(v=[view(brrr, cap=1 << 19)]), RANGE)


def test_the_binding_passes_what_the_header_says(brrr):
    """The structure has the header's fields in its order, and the class refuses through the same checks."""
    import os
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "brrr.h")).read()
    body = re.search(r"typedef struct brrr_kv \{(.*?)\} brrr_kv;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for line in body.split(";") for n in re.findall(r"\**(\w+)\s*(?:,|$)", line.strip())]
    assert names == [n for n, _ in brrr._lib.Kv._fields_]
    kv = brrr.KvCache(P, 2 * P, 3, 4, 64, 100)
    with pytest.raises(brrr.BrrrError, match="brrr_kv_weigh.*argument"):
        kv.weigh(1, 1, P, P, 8, P, 1.0)
    assert kv.TREE_MAX == int(re.search(r"#define BRRR_TREE_MAX (\d+)", src).group(1))


def test_the_class_takes_tensors_of_the_right_kind_only(brrr):
    """Arrays of another value size, with strides, or in host memory beside a device cache never become addresses."""
    import torch
    kv = brrr.KvCache(P, 2 * P, 3, 4, 64, 100, weight=3 * P, pos=4 * P)
    i32, i64 = torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    k = torch.zeros((1, 2, 16, 64))
    for bad in (k.half(), k.bfloat16(), k.int(), k[:, :1], k.view(-1)[1:]):          # another type, memory that ends early
        with pytest.raises(brrr.BrrrError, match="values of torch.float32"):
            brrr.KvCache(k, bad if bad.dtype != k.dtype else bad.clone(), 1, 2, 64, 16)
    with pytest.raises(brrr.BrrrError, match="values of torch.bfloat16"):
        brrr.KvCache(k.half(), k.half(), 1, 2, 64, 16, bf16=True)
    with pytest.raises(brrr.BrrrError, match="values of torch.float32"):
        brrr.KvCache(k, k, 1, 2, 64, 16, head_stride=16 * 64 + 8)
    assert brrr.KvCache(k[:, 1:], k[:, 1:], 1, 1, 64, 16, head_stride=8).view.cap == 16          # one head: its stride says nothing
    here, there = brrr.KvCache(k, k, 1, 2, 64, 16), brrr.KvCache(k, k, 1, 2, 64, 16)
    there._dev = 1
    with pytest.raises(brrr.BrrrError, match="another device"):
        here.evict(1, P, 5, 0, 0, None, P, dst=there)
    for call in (lambda: kv.attn_tree(1, 1, i32, P, 8, P, 1.0), lambda: kv.commit(1, 1, P, i64, P), lambda: kv.evict(1, i64, 5, 0, 0, None, P),
                 lambda: kv.weigh(1, 1, P, P, 8, P, 1.0, picked=i32)):
        with pytest.raises(brrr.BrrrError, match="cache's device"):
            call()
