"""KV caches outside an engine: draft trees, eviction by attention weight, attention over chosen blocks.

`KvCache` is a view of device memory that the caller owns (brrr_kv of include/brrr.h, where every call is described); its
methods are the C entry points with the optional arguments by name.  Device arrays are given as addresses or as anything
with data_ptr() (a contiguous torch tensor); `stream` is a cudaStream_t as an integer (None: the default stream).
What only the device can see - an entry that does not fit - sets the word `err`; without one it is left out silently.
"""
import ctypes as C

from ._lib import BrrrError, Kv, check, lib


class _Kind(set):
    """What an array may hold: the tensor types of these names, each entered when it is first met."""

    def __init__(self, *names):
        super().__init__()
        self.names = names

    def meets(self, dtype):
        if str(dtype) in self.names:
            self.add(dtype)
        return dtype in self


REAL, INT, WORD = _Kind("torch.float32"), _Kind("torch.int32", "torch.uint32"), _Kind("torch.int64", "torch.uint64")


class KvCache:
    F32, BF16 = 0, 1
    TREE_MAX = 64

    def __init__(self, k, v, n_seq, n_head_kv, head_dim, cap, bf16=False, head_stride=0, seq_stride=0, weight=None, pos=None, err=None):
        self._held = (k, v, weight, pos, err)      # the memory stays as long as the view
        self._dev = None if isinstance(k, int) or k is None else k.get_device()
        # k and v may have any strides: head_stride and seq_stride describe them
        book, head = n_seq * n_head_kv * cap, cap * head_dim
        hs = head_stride if head_stride and n_head_kv > 1 else head
        values = (n_seq - 1) * (seq_stride if seq_stride and n_seq > 1 else hs * n_head_kv) + (n_head_kv - 1) * hs + head
        self.view = Kv(self._rows(k, values, bf16), self._rows(v, values, bf16), int(bool(bf16)), n_seq, n_head_kv, head_dim, cap, head_stride, seq_stride,
                       self._at(weight, book), self._at(pos, book, INT), self._at(err, 1, INT))
        self._ref = C.byref(self.view)
        self._lib = lib()

    def _rows(self, x, need, bf16):
        """The address of keys or values; behind a tensor's first value its memory has to hold all of them."""
        if x is None or isinstance(x, int):
            return x
        dtype, left = "torch.bfloat16" if bf16 else "torch.float32", x.untyped_storage().nbytes() // x.element_size() - x.storage_offset()
        if str(x.dtype) != dtype or left < need or x.get_device() != self._dev:
            raise BrrrError(f"KvCache: {need} values of {dtype} on one device are wanted, not {left} of {x.dtype} on {x.device}")
        return x.data_ptr()

    def _at(self, x, need, kind=REAL):
        """The address of a device array; a tensor has to be dense, of values of that kind, of `need` of them at least and on the cache's device."""
        if x is None:
            return None
        try:
            here = x.get_device()
        except AttributeError:
            return x                               # an address
        if (x.dtype not in kind and not kind.meets(x.dtype)) or x.numel() < need or not x.is_contiguous() or (here != self._dev and (here < 0 or self._dev is not None)):
            raise BrrrError(f"KvCache: a contiguous array of {need} or more values of {kind.names[0]} on the cache's device is wanted, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return x.data_ptr()

    def append(self, n, rows, length, qkv, n_head=0, q=None, at=None, rope=None, n_rope=0, count=None, seq=None, ld=0, stream=None):
        """Rows of q | k | v into the cache at slots length[b] + i, rotated by their positions `at` (None: the slots' numbers, wrong in a tree and after an
        eviction in place); rotated q to `q`."""
        p, v = self._at, self.view
        width = (n_head + 2 * v.n_head_kv) * v.head_dim
        check(self._lib.brrr_kv_append(self._ref, n, rows, p(seq, n, INT), p(length, n, INT), p(count, n, INT), p(at, n * rows, INT), p(qkv, (n * rows - 1) * (ld or width) + width), ld, n_head,
                                       p(rope, n_rope * v.head_dim), n_rope, p(q, n * rows * n_head * v.head_dim), stream), "brrr_kv_append")

    def attn_tree(self, n, rows, length, q, n_head, out, scale, seq=None, count=None, mask=None, len_hint=0, window=0, sinks=None, lse=None, stream=None):
        """Attention of drafted tokens (ancestor masks; None: a chain) over the cache and their own entries."""
        p, heads = self._at, n * rows * n_head
        values = heads * self.view.head_dim
        check(self._lib.brrr_attn_tree(self._ref, n, rows, p(seq, n, INT), p(length, n, INT), p(count, n, INT), p(mask, n * rows, WORD), len_hint, p(q, values), n_head, scale, window,
                                       p(sinks, n_head), p(out, values), p(lse, heads), stream), "brrr_attn_tree")

    def commit(self, n, rows, length, path, npath, seq=None, new_len=None, stream=None):
        """The accepted rows of each tree to the slots behind the cached entries."""
        p = self._at
        check(self._lib.brrr_kv_commit(self._ref, n, rows, p(seq, n, INT), p(length, n, INT), p(path, n * rows, INT), p(npath, n, INT), p(new_len, n, INT), stream), "brrr_kv_commit")

    def weigh(self, n, rows, length, q, n_head, lse, scale, seq=None, count=None, mask=None, picked=None, len_hint=0, window=0, stream=None):
        """The attention weights of the rows (of those whose bit in `picked` is set) added to the cache's book."""
        p, heads = self._at, n * rows * n_head
        check(self._lib.brrr_kv_weigh(self._ref, n, rows, p(seq, n, INT), p(length, n, INT), p(count, n, INT), p(mask, n * rows, WORD), p(picked, n, WORD), len_hint,
                                      p(q, heads * self.view.head_dim), n_head, scale, window, p(lse, heads), stream), "brrr_kv_weigh")

    def evict(self, n, length, keep, first, recent, end, map, seq=None, dst=None, new_len=None, len_hint=0, stream=None):
        """The `keep` entries of each head with the largest weights (and the first and latest ones) in place, or into another KvCache."""
        p = self._at
        if dst is not None and None not in (dst._dev, self._dev) and dst._dev != self._dev:
            raise BrrrError("KvCache: dst is on another device")
        check(self._lib.brrr_kv_evict(self._ref, None if dst is None else dst._ref, n, p(seq, n, INT), p(length, n, INT), keep, first, recent, p(end, n, INT),
                                      p(map, n * self.view.n_head_kv * keep, INT), p(new_len, n, INT), len_hint, stream), "brrr_kv_evict")

    def means(self, n, length, block, means, seq=None, since=None, len_hint=0, stream=None):
        """Means of the keys of the whole blocks between since[b] and length[b]."""
        p = self._at
        check(self._lib.brrr_kv_means(self._ref, n, p(seq, n, INT), p(since, n, INT), p(length, n, INT), block, len_hint, p(means, self._means(block)), stream), "brrr_kv_means")

    def attn_blocks(self, rows, seq, length, block, means, nsel, first, local, q, n_head, out, scale, sel, len_hint=0, sinks=None, lse=None, stream=None):
        """Attention of each row over the nsel blocks of its sequence that it scores highest; the choice goes to `sel`."""
        p, values = self._at, rows * n_head * self.view.head_dim
        check(self._lib.brrr_attn_blocks(self._ref, rows, p(seq, rows, INT), p(length, rows, INT), block, p(means, self._means(block)), nsel, first, local, len_hint, p(q, values), n_head,
                                         scale, p(sinks, n_head), p(sel, rows * self.view.n_head_kv * nsel, INT), p(out, values), p(lse, rows * n_head), stream), "brrr_attn_blocks")

    def _means(self, block):
        v = self.view
        return v.n_seq * v.n_head_kv * (v.cap // block) * v.head_dim if block > 0 else 0
