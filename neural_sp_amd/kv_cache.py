"""Paged key / value cache of a decoder's self-attention: fixed-size pages of every layer in one allocation, handed out to
the rows of a batch as they grow (ops.paged_attention reads and extends it, ops.paged_append fills in a prompt).

The page numbers live twice: in a host list per row, where pages are taken and returned, and in the int32 device table the
kernels read.  A row's pages are its own from `reserve` until `release`; nothing here waits for the device."""
import numpy as np
import torch

from neural_sp_amd import ops


class PagedKVCache(object):
    """n_layers x n_pages pages of `page_size` tokens x n_heads x head size, fp32 or bf16.

    k(l) / v(l): layer l's pages `[n_pages, n_heads, page_size, d]`; block_table `[n_rows, max_pages]` int32 on the device
    (-1: no page); lens `[n_rows]` int32 on the device (tokens stored; -1: the row is not in use)."""

    def __init__(self, n_layers, n_rows, max_len, n_heads, head_size, dtype, device, page_size=16, n_pages=None):
        if min(n_layers, n_rows, max_len, n_heads, head_size, page_size) < 1:
            raise ValueError('PagedKVCache: sizes are positive numbers')
        self.page_size = page_size
        self.max_pages = (max_len + page_size - 1) // page_size
        self.n_pages = n_rows * self.max_pages if n_pages is None else int(n_pages)
        self.device = torch.device(device)
        self._kv = torch.empty((n_layers, 2, self.n_pages, n_heads, page_size, head_size), device=self.device, dtype=dtype)
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._rows = [[] for _ in range(n_rows)]
        self._table = np.full((n_rows, self.max_pages), -1, dtype=np.int32)
        self.block_table = ops.h2d(self._table.copy(), self.device)
        self.lens = torch.full((n_rows,), -1, dtype=torch.int32, device=self.device)

    def k(self, layer):
        return self._kv[layer, 0]

    def v(self, layer):
        return self._kv[layer, 1]

    @property
    def free_pages(self):
        return len(self._free)

    def _numbers(self, rows):
        """each row once, as a number of 0 .. n_rows - 1 (negative ones count from the end); nothing is changed for a wrong one"""
        n = len(self._rows)
        rows = [int(r) for r in rows]
        for r in rows:
            if not -n <= r < n:
                raise IndexError('row %d of a cache of %d rows' % (r, n))
        return list(dict.fromkeys(r % n for r in rows))

    def reserve(self, rows, n_tokens):
        """pages for n_tokens tokens (in all, not in addition) of each of `rows`; all or none.  The caller's `lens` says how many
        of them are stored."""
        want = (int(n_tokens) + self.page_size - 1) // self.page_size
        if want > self.max_pages:
            raise ValueError('%d tokens: a row holds %d' % (n_tokens, self.max_pages * self.page_size))
        rows = self._numbers(rows)
        need = sum(max(0, want - len(self._rows[r])) for r in rows)
        if need > len(self._free):
            raise RuntimeError('PagedKVCache: %d pages wanted, %d free' % (need, len(self._free)))
        if need == 0:
            return
        for r in rows:
            while len(self._rows[r]) < want:
                self._table[r, len(self._rows[r])] = self._free[-1]
                self._rows[r].append(self._free.pop())
        self.block_table = ops.h2d(self._table.copy(), self.device)      # (a new tensor: launches under way keep theirs)

    def release(self, rows):
        """give the pages of `rows` back (the caller sets their `lens` to -1); launches in the stream so far still read them
        undisturbed, later ones of the same stream may write them for other rows"""
        for r in self._numbers(rows):
            self._free.extend(reversed(self._rows[r]))
            self._rows[r] = []
            self._table[r] = -1
        self.block_table = ops.h2d(self._table.copy(), self.device)
