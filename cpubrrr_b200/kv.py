"""KV caches outside an engine: draft trees, eviction by attention weight, attention over chosen blocks.

`KvCache` is a view of device memory that the caller owns (brrr_kv of include/brrr.h, where every call is described); its
methods are the C entry points with the optional arguments by name.  Device arrays are given as addresses or as anything
with data_ptr() (a contiguous torch tensor); `stream` is a cudaStream_t as an integer (None: the default stream).
"""
import ctypes as C

from ._lib import Kv, check, lib


def _p(x):
    return x if x is None or isinstance(x, int) else x.data_ptr()


class KvCache:
    F32, BF16 = 0, 1
    TREE_MAX = 64

    def __init__(self, k, v, n_seq, n_head_kv, head_dim, cap, bf16=False, head_stride=0, seq_stride=0, weight=None, pos=None, err=None):
        self._held = (k, v, weight, pos, err)      # the memory stays as long as the view
        self.view = Kv(_p(k), _p(v), int(bool(bf16)), n_seq, n_head_kv, head_dim, cap, head_stride, seq_stride, _p(weight), _p(pos), _p(err))
        self._ref = C.byref(self.view)

    def append(self, n, rows, length, qkv, n_head=0, q=None, at=None, rope=None, n_rope=0, count=None, seq=None, ld=0, stream=None):
        """Rows of q | k | v into the cache at slots length[b] + i, rotated by their positions; rotated q to `q`."""
        check(lib().brrr_kv_append(self._ref, n, rows, _p(seq), _p(length), _p(count), _p(at), _p(qkv), ld, n_head, _p(rope), n_rope, _p(q), stream), "brrr_kv_append")

    def attn_tree(self, n, rows, length, q, n_head, out, scale, seq=None, count=None, mask=None, len_hint=0, window=0, sinks=None, lse=None, stream=None):
        """Attention of drafted tokens (ancestor masks; None: a chain) over the cache and their own entries."""
        check(lib().brrr_attn_tree(self._ref, n, rows, _p(seq), _p(length), _p(count), _p(mask), len_hint, _p(q), n_head, scale, window, _p(sinks), _p(out), _p(lse),
                                   stream), "brrr_attn_tree")

    def commit(self, n, rows, length, path, npath, seq=None, new_len=None, stream=None):
        """The accepted rows of each tree to the slots behind the cached entries."""
        check(lib().brrr_kv_commit(self._ref, n, rows, _p(seq), _p(length), _p(path), _p(npath), _p(new_len), stream), "brrr_kv_commit")

    def weigh(self, n, rows, length, q, n_head, lse, scale, seq=None, count=None, mask=None, picked=None, len_hint=0, window=0, stream=None):
        """The attention weights of the rows (of those whose bit in `picked` is set) added to the cache's book."""
        check(lib().brrr_kv_weigh(self._ref, n, rows, _p(seq), _p(length), _p(count), _p(mask), _p(picked), len_hint, _p(q), n_head, scale, window, _p(lse), stream),
              "brrr_kv_weigh")

    def evict(self, n, length, keep, first, recent, end, map, seq=None, dst=None, new_len=None, len_hint=0, stream=None):
        """The `keep` entries of each head with the largest weights (and the first and latest ones) in place, or into another KvCache."""
        check(lib().brrr_kv_evict(self._ref, None if dst is None else dst._ref, n, _p(seq), _p(length), keep, first, recent, _p(end), _p(map), _p(new_len), len_hint,
                                  stream), "brrr_kv_evict")

    def means(self, n, length, block, means, seq=None, since=None, len_hint=0, stream=None):
        """Means of the keys of the whole blocks between since[b] and length[b]."""
        check(lib().brrr_kv_means(self._ref, n, _p(seq), _p(since), _p(length), block, len_hint, _p(means), stream), "brrr_kv_means")

    def attn_blocks(self, rows, seq, length, block, means, nsel, first, local, q, n_head, out, scale, sel, len_hint=0, sinks=None, lse=None, stream=None):
        """Attention of each row over the nsel blocks of its sequence that it scores highest; the choice goes to `sel`."""
        check(lib().brrr_attn_blocks(self._ref, rows, _p(seq), _p(length), block, _p(means), nsel, first, local, len_hint, _p(q), n_head, scale, _p(sinks), _p(sel),
                                     _p(out), _p(lse), stream), "brrr_attn_blocks")
