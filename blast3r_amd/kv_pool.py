"""The pages of an 8-bit key/value cache on the device (``ba_kv_pool_*``, libba_hip.so).

A cache (``kv_cache.KVCache``) is written and read through lists of its blocks.  ``BlockPool`` keeps such lists: it knows of
each block how many lists hold it, gives blocks to sequences that grow, lets sequences share the blocks that they begin with,
and takes back what is no longer held.  Lists are about block numbers, so the caches of all layers of a network go by one
pool::

    pool = BlockPool(n_blocks)
    pages = torch.full((n_seqs, width), -1, dtype=torch.int32, device='cuda')
    moves = pool.grow(pages, lengths, n)                  # blocks for n more tokens of each sequence
    for cache in caches:
        cache.copy(*moves)                                # open blocks that others hold too, for their new owners
        cache.append(k, v, pages, lengths)
    pool.fork(pages, lengths, parents, children)          # children begin with their parents' blocks
    pool.free(pages, lengths, rows)                       # sequences that have ended

Nothing here synchronises and every call can be captured in a graph; results do not depend on the order in which threads run:
the lowest free block is taken first, and sequences are served in their order.  What a call cannot do for want of blocks it
counts in ``missing``.  The calls of one pool go one after the other (on one stream, or on streams that wait for each other).

A table is (n_seqs, blocks) int32, -1 where a list has no block (and 2^30 more than its number where one may not be written
to, see ``grow``).  A block must not be written to by two lists: after a fork
the open last block is shared, and ``grow`` is what gives each its own before new tokens are appended.
"""
import torch

from ._lib import (BaKvCompactArgs, BaKvCountArgs, BaKvForkArgs, BaKvFreeArgs, BaKvGrowArgs, BaKvPool, BaKvTable, BaKvTrimArgs,
                   launch, lib, written)

__all__ = ['BlockPool']

BLOCK = 64


def _fixed(name):
    return property(lambda self: getattr(self, name))


def _overlap(x, y):
    """Whether two tables have an entry in common."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    if y.data_ptr() < x.data_ptr():
        x, y = y, x
    (rows, width), stride = x.shape, x.stride(0) if x.shape[0] > 1 else x.shape[1]
    off = (y.data_ptr() - x.data_ptr()) // 4
    if off >= (rows - 1) * stride + width:
        return False
    if y.shape[0] > 1 and rows > 1 and y.stride(0) != stride:
        return True                                          # rows of other lengths: not looked at more closely
    return off % stride < width or off % stride + y.shape[1] > stride and off // stride + 1 < rows


class BlockPool:
    """Who holds the ``n_blocks`` blocks of a cache.

    counts   (n_blocks,) int32: the lists that hold each block (to be read; ``count`` sets it from lists)
    missing  (1,) int32: how many blocks the last ``grow`` wanted beyond those that were free
    """

    n_blocks, device, counts, missing = _fixed('_n_blocks'), _fixed('_device'), _fixed('_counts'), _fixed('_missing')

    def __init__(self, n_blocks, device='cuda'):
        if not 0 <= n_blocks < 1 << 30:
            raise ValueError(f'pool: bad sizes ({n_blocks} blocks)')
        self._counts = torch.zeros(n_blocks, dtype=torch.int32, device=device)
        if not self._counts.is_cuda:
            raise RuntimeError('pool: needs a GPU (it runs in libba_hip.so)')
        self._n_blocks, self._device = n_blocks, self._counts.device
        self._used = torch.zeros((n_blocks + 31) // 32, dtype=torch.int32, device=self._device)
        self._marks = torch.full((2 * n_blocks,), -1, dtype=torch.int32, device=self._device)
        self._missing = torch.zeros(1, dtype=torch.int32, device=self._device)
        self._lib, self._at = lib(), None
        if n_blocks % 32:                                   # bits past the last block are set
            self._used[-1] = -1 << n_blocks % 32

    def available(self):
        """(1,) int64 on the device: the free blocks."""
        free = torch.empty(1, dtype=torch.int64, device=self._device)
        a = self._args(BaKvFreeArgs)
        a.free = free.data_ptr()
        launch(self._lib.ba_kv_pool_free, a, self._device)
        return free

    def _args(self, kind):
        """The arguments of a call, with the pool's own."""
        at = self._counts.data_ptr()
        if at != self._at:
            self._at = at
            pool = BaKvPool(at, self._used.data_ptr(), self._marks.data_ptr(), self._n_blocks)
            self._kinds = {k: k(pool=pool) for k in (BaKvCountArgs, BaKvFreeArgs, BaKvForkArgs, BaKvTrimArgs, BaKvGrowArgs,
                                                     BaKvCompactArgs)}
        return kind.from_buffer_copy(self._kinds[kind])

    def _table(self, a, pages, name='pages'):
        shape, stride = pages.shape, pages.stride()
        if (len(shape) != 2 or pages.dtype is not torch.int32 or pages.device != self._device or
                stride[1] != 1 and shape[1] > 1 or stride[0] < shape[1] and shape[0] > 1):
            raise ValueError(f'pool: {name} must be (n_seqs, blocks) int32 on {self._device} with contiguous rows that do not '
                             'overlap')
        a.pages, a.stride, a.n_seqs, a.n_pages = pages.data_ptr(), stride[0], shape[0], shape[1]
        return shape

    def _ints(self, t, name, n=None):
        shape = t.shape
        if (t.dtype is not torch.int32 or t.device != self._device or len(shape) != 1 or n is not None and shape[0] != n or
                not t.is_contiguous()):
            raise ValueError(f'pool: {name} must be a contiguous int32 tensor of shape ({"n" if n is None else n},) on {self._device}')
        return t.data_ptr()

    def _launch(self, call, a, *changed):
        launch(call, a, self._device)
        written((self._counts, *changed))

    def _tables(self, a, tables):
        a.tables, a.n_tables = (BaKvTable * len(tables))(), len(tables)
        for i, t in enumerate(tables):
            self._table(a.tables[i], t)
        if any(_overlap(x, y) for i, x in enumerate(tables) for y in tables[:i]):
            raise ValueError('pool: tables overlap')

    def count(self, *tables):
        """Set the counts from tables: those of all lists that are in use.  For lists that were made or changed by hand, or
        read from a file."""
        a = self._args(BaKvCountArgs)
        self._tables(a, tables)
        self._launch(self._lib.ba_kv_pool_count, a)

    def grow(self, pages, lengths, new, max_new=None):
        """Blocks for ``new`` more tokens (a number, or (n_seqs,) int32) after the first ``lengths`` of each list, written into
        ``pages``; blocks that are there already stay, unless other lists hold them too.  max_new (default: what lists can
        hold) bounds ``new``, and a close bound saves time.  ``lengths`` stays as it is.

        Returns (src, dst, n) for ``KVCache.copy``: where new tokens would go to a block that has tokens and that other lists
        hold too, it is exchanged for another one in this list, and src has to be copied to dst before anything is appended
        (and before the next call on this pool).  One list after the other, so the last holder of a block keeps it.

        ``missing`` says how many blocks there were not.  Lists that there were none left for have -1 at the places of their
        new tokens.  A shared block that there was no other for stays in all lists that were to write there and hold it still,
        with 2^30 added to its number: its tokens are seen and read as ever.  Rows appended to either are left out, and
        ``lengths`` must not count them.  When blocks have been given back, the same call again gives such lists what they
        lacked."""
        a = self._args(BaKvGrowArgs)
        self._table(a.table, pages)
        S, width = a.table.n_seqs, a.table.n_pages
        a.lengths = self._ints(lengths, 'lengths', S)
        if isinstance(new, torch.Tensor):
            a.more = self._ints(new, 'new', S)
            most = width * BLOCK if max_new is None else max_new
        else:
            if new < 0:
                raise ValueError(f'pool: {new} new tokens')
            a.each = most = min(int(new), (1 << 31) - 1)
            if max_new is not None:
                most = max_new
        if most < 0:
            raise ValueError('pool: a negative bound on tokens')
        a.max_new = min(int(most), (1 << 31) - 1)
        moves = torch.empty(2 * S + 1, dtype=torch.int32, device=self._device).split_with_sizes((S, S, 1))
        at, missing = moves[2].data_ptr() - 8 * S, self._missing
        a.src, a.dst, a.n, a.missing = at, at + 4 * S, at + 8 * S, missing.data_ptr()
        self._launch(self._lib.ba_kv_pool_grow, a, pages, missing)
        return moves

    def fork(self, pages, lengths, parents, children, into=None):
        """Row children[i] becomes the list of row parents[i] ((n,) int32 each): it gives back the blocks that it held, holds
        its parent's blocks with tokens as well, and gets its length.  into: (pages, lengths) of the children, where they are in
        another table (which a reordering of all sequences needs), with lengths of its own.  Pairs that name a row that is not there, whose child a
        later pair has too, or whose child is a parent in the same table, change nothing."""
        to, to_lengths = (pages, lengths) if into is None else into
        a = self._args(BaKvForkArgs)
        S, width = self._table(a.from_, pages)
        T, wide = self._table(a.to, to)
        a.from_lengths, a.to_lengths = self._ints(lengths, 'lengths', S), self._ints(to_lengths, "the children's lengths", T)
        a.parents, a.children, a.n = self._ints(parents, 'parents'), self._ints(children, 'children', parents.shape[0]), parents.shape[0]
        if wide < width:
            raise ValueError("pool: children's lists must be as wide as their parents'")
        if to is not pages and (to.data_ptr() != pages.data_ptr() or to.stride() != pages.stride()) and _overlap(to, pages):
            raise ValueError('pool: the tables overlap')
        # (lengths of parents in another table are read while children's are written)
        same = to.data_ptr() == pages.data_ptr() and a.from_lengths == a.to_lengths
        if S and T and not same and a.from_lengths < a.to_lengths + 4 * T and a.to_lengths < a.from_lengths + 4 * S:
            raise ValueError("pool: the children's lengths overlap the parents'")
        if a.n:
            self._launch(self._lib.ba_kv_pool_fork, a, to, to_lengths)

    def free(self, pages, lengths, rows=None):
        """Give back the lists ``rows`` ((n,) int32; default: all): entries become -1, lengths 0."""
        a = self._args(BaKvTrimArgs)
        S, _ = self._table(a.table, pages)
        a.lengths, a.all = self._ints(lengths, 'lengths', S), 1
        if rows is not None:
            a.rows, a.n_rows = self._ints(rows, 'rows'), rows.shape[0]
            if not a.n_rows:
                return
        self._launch(self._lib.ba_kv_pool_trim, a, pages, lengths)

    def trim(self, pages, first=None, last=None):
        """Give back the blocks whose tokens all lie before ``first`` (a window that has moved on) or from ``last`` on (tokens
        that were drafted and refused); (n_seqs,) int32 each."""
        if first is None and last is None:
            raise ValueError('pool: trim by first, by last or by both')
        a = self._args(BaKvTrimArgs)
        S, _ = self._table(a.table, pages)
        if first is not None:
            a.first = self._ints(first, 'first', S)
        if last is not None:
            a.last = self._ints(last, 'last', S)
        self._launch(self._lib.ba_kv_pool_trim, a, pages)

    def compact(self, *tables, most=None):
        """Move the highest used blocks to the lowest free ones, ``most`` at a time at most (default: all), so that the used
        blocks come to be the first: ``tables`` (all that hold blocks of the pool) are changed, and (src, dst, n) is for
        ``KVCache.copy``, before the next call on this pool."""
        a = self._args(BaKvCompactArgs)
        self._tables(a, tables)
        most = self._n_blocks // 2 if most is None else min(int(most), self._n_blocks // 2)
        if most < 0:
            raise ValueError(f'pool: {most} moves')
        moves = torch.empty(2 * most + 1, dtype=torch.int32, device=self._device).split_with_sizes((most, most, 1))
        at = moves[2].data_ptr() - 8 * most
        a.most, a.src, a.dst, a.n = most, at, at + 4 * most, at + 8 * most
        self._launch(self._lib.ba_kv_pool_compact, a, *tables)
        return moves
