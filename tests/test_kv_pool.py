"""Pages of the 8-bit cache (BlockPool, KVCache.copy): refusals and what calls owe to torch (CPU); lists, counts and moves equal
to the oracle's, block copies, and a run of all of them with the cache's other calls (GPU).  All results are whole numbers or
copies: they are equal or wrong."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import tokens as otok
from test_tokens import _cache, _i32, _np

DEV = 'cuda:0'


# ---------------------------------------------------------------------------------- oracle pins (CPU)

def test_oracle_pool_known_answers():
    p = otok.Pool(6)
    rows, lens = np.full((3, 4), -1), [0, 0, 0]
    assert p.grow(rows, lens, [65, 1, 0]) == [] and rows.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4]
    lens = [65, 1, 0]
    table = rows.tolist()
    p.fork(table, lens, [0, 0], [2, 1], table, lens)        # the second child gives its block back
    assert table == [[0, 1, -1, -1]] * 3 and lens == [65, 65, 65] and p.counts == [3, 3, 0, 0, 0, 0]
    rows = np.array(table)
    assert p.grow(rows, lens, [1, 1, 64]) == [(1, 2), (1, 3)]              # the last holder keeps block 1
    assert rows.tolist() == [[0, 2, -1, -1], [0, 3, -1, -1], [0, 1, 4, -1]] and p.counts == [3, 1, 1, 1, 1, 0]
    assert p.grow(rows, [66, 66, 129], [128, 0, 64]) == [] and p.missing == 2 and rows.tolist()[0] == [0, 2, 5, -1]
    p.drop(rows[0])
    p.drop(rows[1])
    assert p.counts == [1, 1, 0, 0, 1, 0]
    assert p.compact([rows], 3) == [(4, 2)] and rows[2].tolist() == [0, 1, 2, -1] and p.counts == [1, 1, 1, 0, 0, 0]


# ---------------------------------------------------------------------------------- refusals (CPU)

def test_pool_entry_points_refuse_bad_arguments_without_a_gpu():
    from blast3r_amd import _lib
    L, p = _lib.lib(), 4096
    pool = _lib.BaKvPool(p, p, p, 40)
    table = lambda **kw: _lib.BaKvTable(**{**dict(pages=p, stride=4, n_seqs=2, n_pages=4), **kw})  # noqa: E731
    calls = {
        'count': (_lib.BaKvCountArgs, lambda t: dict(tables=ctypes.pointer(t), n_tables=1)),
        'grow': (_lib.BaKvGrowArgs, lambda t: dict(table=t, lengths=p, src=p, dst=p, n=p, missing=p)),
        'trim': (_lib.BaKvTrimArgs, lambda t: dict(table=t)),
        'fork': (_lib.BaKvForkArgs, lambda t: dict(from_=table(), to=t, from_lengths=p, to_lengths=p, parents=p, children=p, n=2)),
        'compact': (_lib.BaKvCompactArgs, lambda t: dict(tables=ctypes.pointer(t), n_tables=1, src=p, dst=p, n=p, most=3))}

    def refused(name, word, pool=pool, t=None, **kw):
        kind, fields = calls[name]
        call = getattr(L, 'ba_kv_pool_' + name)
        assert call(kind(pool=pool, **{**fields(t if t is not None else table()), **kw}), None) != 0 and word in L.ba_last_error().decode(), (name, word, L.ba_last_error())

    for name in calls:
        assert getattr(L, 'ba_kv_pool_' + name)(None, None) != 0
        for bad, word in ((_lib.BaKvPool(None, p, p, 40), 'null'), (_lib.BaKvPool(p, p, p, -1), 'bad sizes'), (_lib.BaKvPool(p, p, p, 1 << 30), 'bad sizes')):
            refused(name, word, pool=bad)
        for t, word in ((table(n_seqs=-1), 'bad sizes'), (table(n_pages=1 << 24), 'bad sizes'), (table(n_seqs=1 << 23), 'too many'), (table(pages=None), 'null')):
            refused(name, word, t=t)
    for bad, at, word in ((_lib.BaKvPool(None, p, p, 40), p, 'null'), (pool, None, 'null'), (_lib.BaKvPool(p, p, p, -1), p, 'bad sizes')):
        assert L.ba_kv_pool_free(_lib.BaKvFreeArgs(bad, at), None) != 0 and word in L.ba_last_error().decode()
    assert L.ba_kv_pool_free(None, None) != 0
    refused('count', 'bad tables', tables=None)
    refused('compact', 'bad tables', n_tables=-1)
    refused('grow', 'bad sizes', max_new=-1)
    refused('grow', 'too many blocks', t=table(n_seqs=1 << 20, n_pages=2047, stride=2047), max_new=1 << 30)
    for name in ('lengths', 'src', 'dst', 'n', 'missing'):
        refused('grow', 'null', **{name: None})
    for name in ('from_lengths', 'to_lengths', 'parents', 'children'):
        refused('fork', 'null', **{name: None})
    refused('fork', 'narrower', t=table(n_pages=3))
    refused('fork', 'bad sizes', n=-1)
    refused('fork', 'too many', n=65537)
    for at in (p, p + 4, p - 4):                             # lengths that are read and written, of tables of their own
        refused('fork', 'overlap', t=table(pages=1 << 20), to_lengths=at)
    refused('fork', 'overlap', to_lengths=p + 4)
    assert L.ba_kv_pool_fork(_lib.BaKvForkArgs(pool=pool, from_=table(), to=table()), None) == 0
    refused('compact', 'bad sizes', most=41)
    refused('compact', 'null', n=None)
    refused('trim', 'bad sizes', n_rows=-1)
    copy = dict(k=p, v=p, scales=p, n_blocks=3, heads=2, dim=64, src=p, dst=p, n=2)
    for kw, word in ((dict(dim=48), 'head size'), (dict(heads=0), 'bad sizes'), (dict(n=-1), 'bad sizes'), (dict(k=p + 8), 'aligned'), (dict(dst=None), 'null')):
        assert L.ba_kv_copy(_lib.BaKvCopyArgs(**{**copy, **kw}), None) != 0 and word in L.ba_last_error().decode(), (kw, L.ba_last_error())
    assert L.ba_kv_copy(_lib.BaKvCopyArgs(**{**copy, 'n': 0}), None) == 0


@pytest.fixture
def host(monkeypatch):
    from blast3r_amd import kv_cache, kv_pool
    calls = []
    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    for m in (kv_cache, kv_pool):
        monkeypatch.setattr(m, 'launch', lambda call, args, device: calls.append(args))
    return calls


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32)


def test_pool_refuses_host_tensors_and_bad_sizes():
    from blast3r_amd.kv_pool import BlockPool
    with pytest.raises(RuntimeError):
        BlockPool(4, device='cpu')
    for n in (-1, 1 << 30):
        with pytest.raises(ValueError):
            BlockPool(n, device='cpu')


def test_pool_refuses_bad_arguments(host):
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    pool = BlockPool(40, device='cpu')
    pages, lens = torch.full((2, 6), -1, dtype=torch.int32), _ints([0, 0])
    wide = torch.full((2, 12), -1, dtype=torch.int32)
    for bad in (pages.long(), pages[0], pages.t(), wide[:, ::2], pages[:1].expand(2, 6)):
        for call in (lambda: pool.count(bad), lambda: pool.grow(bad, lens, 1), lambda: pool.free(bad, lens), lambda: pool.trim(bad, first=lens),
                     lambda: pool.compact(bad), lambda: pool.fork(bad, lens, lens, lens), lambda: pool.fork(pages, lens, lens, lens, into=(bad, lens))):
            with pytest.raises(ValueError):
                call()
    for bad in (lens.long(), lens[:1], _ints([[0, 0]]), _ints([0, 0, 0, 0])[::2]):
        for call in (lambda: pool.grow(pages, bad, 1), lambda: pool.grow(pages, lens, bad), lambda: pool.free(pages, bad), lambda: pool.trim(pages, last=bad),
                     lambda: pool.fork(pages, bad, lens, lens), lambda: pool.fork(pages, lens, lens, bad)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: pool.grow(pages, lens, -1), lambda: pool.grow(pages, lens, 1, max_new=-1), lambda: pool.trim(pages), lambda: pool.compact(pages, pages),
                 lambda: pool.compact(pages, most=-1), lambda: pool.fork(pages, lens, lens, lens, into=(pages[:, :5], lens)),
                 lambda: pool.fork(wide, lens, lens, lens, into=(pages, lens)), lambda: pool.fork(pages, lens, lens, lens, into=(wide[:, :6].as_strided((2, 6), (6, 1)), _ints([0])))):
        with pytest.raises(ValueError):
            call()
    both = torch.full((6, 12), -1, dtype=torch.int32)         # tables in one buffer
    four = _ints([0] * 4)
    for x, y in ((both[:4], both[2:]), (both[:4], both[3:5]), (both[:, :7], both[:, 6:]), (both[:4, 3:], both[1:3, :4]), (both, both[2:3, 5:6]),
                 (both[2:3, 5:6], both), (both.view(12, 6), both[3:]), (both[:, 4:], both.view(-1)[8:68].view(5, 12)[:, 2:])):
        with pytest.raises(ValueError, match='overlap'):
            pool.compact(x, y)
        if y.shape[1] >= x.shape[1]:
            with pytest.raises(ValueError, match='overlap'):
                pool.fork(x, _ints([0] * len(x)), four, four, into=(y, _ints([0] * len(y))))
    other = torch.full((2, 6), -1, dtype=torch.int32)         # lengths in one buffer
    for to, x, y in ((other, lens, lens), (other, four[:2], four[1:3]), (pages, four[1:3], four[:2])):
        with pytest.raises(ValueError, match='lengths overlap'):
            pool.fork(pages, x, lens, lens, into=(to, y))
    with pytest.raises(AttributeError):
        pool.counts = pages
    c = KVCache(4, 1, 64, device='cpu')
    for args in ((lens.long(), lens), (lens, lens[:1]), (lens, _ints([0, 0, 0])), (lens, lens, lens), (_ints([[0]]), lens), (_ints([0, 0, 0, 0])[::2], lens)):
        with pytest.raises(ValueError):
            c.copy(*args)
    assert not host


def test_tensors_that_pool_calls_write_to_count_as_changed(host):
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    pool = BlockPool(40, device='cpu')
    pages, other, lens, ends = torch.full((2, 6), -1, dtype=torch.int32), torch.full((3, 6), -1, dtype=torch.int32), _ints([0, 0]), _ints([0, 0, 0])
    c = KVCache(40, 1, 64, device='cpu')
    calls = (
        (lambda: pool.count(pages), (pool.counts,)), (lambda: pool.grow(pages, lens, 1), (pool.counts, pages, pool.missing)),
        (lambda: pool.fork(pages, lens, lens, lens), (pool.counts, pages, lens)),
        (lambda: pool.fork(pages, lens, lens, lens, into=(other, ends)), (pool.counts, other, ends)),
        (lambda: pool.free(pages, lens), (pool.counts, pages, lens)), (lambda: pool.trim(other, first=ends), (pool.counts, other)),
        (lambda: pool.compact(pages, other), (pool.counts, pages, other)), (lambda: c.copy(lens, lens), (c.k, c.v, c.scales)))
    both = torch.full((6, 12), -1, dtype=torch.int32)
    everything = (pool.counts, pool.missing, pages, other, lens, ends, c.k, c.v, c.scales)
    for call, changed in calls:
        before = [t._version for t in everything]
        call()
        for t, v in zip(everything, before):
            assert t._version == v + (1 if any(t is u for u in changed) else 0)
    for x, y in ((both[:3], both[3:]), (both[:, :6], both[:, 6:]), (both[:, 3:8], both[:5, 8:]), (both[:0], both), (both[2:3], both[3:4])):
        pool.compact(x, y)
        if y.shape[1] >= x.shape[1]:
            pool.fork(x, _ints([0] * len(x)), lens, lens, into=(y, _ints([0] * len(y))))
    n = len(host)
    for call in (lambda: pool.free(pages, lens, rows=lens[:0]), lambda: pool.fork(pages, lens, lens[:0], lens[:0]), lambda: c.copy(lens[:0], lens[:0])):
        call()
    assert len(host) == n


def test_copies_of_factors_with_gradients_are_refused(host):
    from blast3r_amd.kv_cache import KVCache
    c = KVCache(2, 1, 64, device='cpu')
    w = KVCache.wrap(c.k, c.v, torch.ones(2, 1, 2, requires_grad=True))
    with pytest.raises(RuntimeError, match='gradient'):
        w.copy(_ints([0]), _ints([1]))
    assert not host


# ---------------------------------------------------------------------------------- parity (GPU)

class Both:
    """A pool and its oracle, and a table with its lengths."""

    def __init__(self, n_blocks, n_seqs, width):
        from blast3r_amd.kv_pool import BlockPool
        self.pool, self.o = BlockPool(n_blocks, device=DEV), otok.Pool(n_blocks)
        self.pages, self.lens = np.full((n_seqs, width), -1), [0] * n_seqs
        self.t = torch.full((n_seqs, width + 3), -7, dtype=torch.int32, device=DEV)[:, :width]       # rows that are not one after the other
        self.t.fill_(-1)
        self.tl = torch.zeros(n_seqs, dtype=torch.int32, device=DEV)

    def same(self):
        assert self.t.tolist() == self.pages.tolist() and self.tl.tolist() == [int(x) for x in self.lens]
        assert self.pool.counts.tolist() == self.o.counts and int(self.pool.available()) == self.o.counts.count(0)
        used = self.pool._used.cpu().numpy().view(np.uint32)
        bits = (used[:, None] >> np.arange(32, dtype=np.uint32) & 1).flatten()
        assert bits[:len(self.o.counts)].tolist() == [int(c > 0) for c in self.o.counts] and bits[len(self.o.counts):].all()
        assert bool(((self.pool._marks[:len(self.o.counts)] == -1) | (self.pool.counts == 0)).all())

    def moved(self, moves, got, size):
        src, dst, n = got
        assert int(n) == len(moves)
        assert src.tolist() == [m[0] for m in moves] + [-1] * (size - len(moves)) and dst.tolist() == [m[1] for m in moves] + [-1] * (size - len(moves))

    def grow(self, new, max_new=None):
        each = isinstance(new, int)
        got = self.pool.grow(self.t, self.tl, new if each else _i32(new), max_new=max_new)
        counts = [new] * len(self.lens) if each else [min(x, max_new) if max_new is not None else x for x in new]
        moves = self.o.grow(self.pages, self.lens, counts)
        self.moved(moves, got, len(self.lens))
        assert int(self.pool.missing) == self.o.missing
        return counts

    def advance(self, counts):
        self.lens = [x + max(0, n) for x, n in zip(self.lens, counts)]
        self.tl.copy_(_i32(self.lens))


@pytest.mark.gpu
@pytest.mark.parametrize('n_blocks,n_seqs,width,most,seed', [
    (1, 1, 1, 64, 0), (31, 3, 5, 70, 1), (32, 4, 8, 130, 2), (33, 40, 6, 1, 3), (200, 17, 30, 200, 4), (5000, 64, 120, 1, 5), (5000, 64, 120, 900, 6),
    (40000, 1500, 9, 100, 7), (70001, 20, 300, 5000, 8)])
def test_pool_against_oracle(n_blocks, n_seqs, width, most, seed):
    """Sequences that grow, fork, give back from either end, end and are moved together, in no order, also where blocks run
    out."""
    rng = np.random.default_rng(seed)
    b = Both(n_blocks, n_seqs, width)
    print(f'pool {n_blocks} {n_seqs} {width} {most}', flush=True)
    b.same()
    for step in range(12 if n_seqs < 1000 else 5):
        what = int(rng.integers(0, 6)) if step > 1 else 0
        print(f'  step {step}: {what}', flush=True)
        if what <= 1:
            new = rng.integers(0, most + 1, n_seqs).tolist() if rng.random() < 0.7 else most
            if not isinstance(new, int) and rng.random() < 0.3:
                new[int(rng.integers(0, n_seqs))] = -3
            counts = b.grow(new, max_new=None if isinstance(new, int) else most - int(rng.integers(0, 2)))
            b.advance(counts)
        elif what == 2:
            order = rng.permutation(n_seqs)
            k = max(1, n_seqs // 3)
            parents, children = rng.choice(order[:k], k).tolist(), order[k:2 * k].tolist()
            children = (children + [n_seqs, -1] * k)[:k]
            if k > 2:
                children[-1] = children[0]                  # the first of the two is left out
            b.pool.fork(b.t, b.tl, _i32(parents), _i32(children))
            rows = b.pages.tolist()
            b.o.fork(rows, b.lens, parents, children, rows, b.lens)
            b.pages = np.array(rows)
        elif what == 3:
            rows = rng.integers(-1, n_seqs + 1, max(1, n_seqs // 4)).tolist()       # some twice, some that are not there
            b.pool.free(b.t, b.tl, _i32(rows))
            for r in rows:
                if 0 <= r < n_seqs:
                    b.o.drop(b.pages[r])
                    b.lens[r] = 0
        elif what == 4:
            first, last = rng.integers(-70, 200, n_seqs), np.array(b.lens) + rng.integers(-100, 100, n_seqs)
            use = int(rng.integers(0, 3))
            b.pool.trim(b.t, first=_i32(first) if use != 1 else None, last=_i32(last) if use != 0 else None)
            for s in range(n_seqs):
                lo = max(0, int(first[s])) // 64 if use != 1 else 0
                hi = (max(0, int(last[s])) + 63) // 64 if use != 0 else 1 << 30
                b.o.drop(b.pages[s], keep=lambda x, lo=lo, hi=hi: lo <= x < hi)
            if use != 0:
                b.lens = [max(0, min(x, int(y))) for x, y in zip(b.lens, last)]
                b.tl.copy_(_i32(b.lens))
        else:
            some = None if rng.random() < 0.5 else int(rng.integers(0, n_blocks + 1))
            size = n_blocks // 2 if some is None else min(some, n_blocks // 2)
            got = b.pool.compact(b.t, most=some)
            b.moved(b.o.compact([b.pages], size), got, size)
        b.same()
    b.pool.count(b.t)
    b.o.count(b.pages)
    b.same()
    b.pool.free(b.t, b.tl)
    for row in b.pages:
        b.o.drop(row)
    b.lens = [0] * n_seqs
    b.same()
    assert not any(b.o.counts)


@pytest.mark.gpu
def test_all_sequences_reordered_into_another_table():
    """A step of a beam search: every row of the second table is a row of the first, whose lists then end.  Blocks that were
    shared by rows that all write get one copy less than they have holders."""
    b = Both(300, 8, 10)
    print('beam', flush=True)
    b.advance(b.grow([100, 5, 64, 0, 300, 129, 1, 63]))
    other, ends = torch.full((9, 12), -1, dtype=torch.int32, device=DEV), torch.zeros(9, dtype=torch.int32, device=DEV)
    rows, lens = np.full((9, 12), -1).tolist(), [0] * 9
    for parents in ([0, 0, 0, 4, 4, 1, 2, 3], [7, 7, 7, 7, 7, 7, 7, 7], [5, 4, 3, 2, 1, 0, 0, 0]):
        children = [8, 1, 2, 3, 4, 5, 6, 7]
        b.pool.fork(b.t, b.tl, _i32(parents), _i32(children), into=(other, ends))
        b.o.fork(b.pages.tolist(), b.lens, parents, children, rows, lens)
        b.pool.free(b.t, b.tl)
        for row in b.pages:
            b.o.drop(row)
        b.lens = [0] * 8
        b.same()
        table = np.array(rows)
        moves = b.o.grow(table, lens, [1] * 9)
        b.moved(moves, b.pool.grow(other, ends, 1), 9)
        rows, lens = table.tolist(), [x + 1 for x in lens]
        ends += 1
        assert other.tolist() == rows
        back = [8, 7, 6, 5, 4, 3, 2, 1]                      # and back
        wide = torch.full((8, 12), -1, dtype=torch.int32, device=DEV)
        b.pool.fork(other, ends, _i32(back), _i32(list(range(8))), into=(wide, b.tl))
        mine = np.full((8, 12), -1).tolist()
        b.o.fork(rows, lens, back, list(range(8)), mine, b.lens)
        b.pool.free(other, ends)
        for row in rows:
            b.o.drop(row)
        lens = [0] * 9
        b.t, b.pages = wide, np.array(mine)
        b.same()


@pytest.mark.gpu
@pytest.mark.parametrize('n_blocks', [100, 16384, 16385, 50000])
def test_lists_of_several_tables_counted_and_moved(n_blocks):
    """Two tables, one of them a part of a wider one, of more and fewer blocks than one workgroup counts; entries that are no
    block's; on another stream than the tensors were made on, and under inference mode."""
    from blast3r_amd.kv_pool import BlockPool
    rng = np.random.default_rng(n_blocks)
    pool, o = BlockPool(n_blocks, device=DEV), otok.Pool(n_blocks)
    one, two = rng.integers(-3, n_blocks + 3, (7, 9)), rng.integers(n_blocks // 2, n_blocks, (40, 33))
    one[0, 0], one[1, 1] = (1 << 31) - 1, -(1 << 31)
    a, wide = _i32(one), torch.full((40, 70), 7, dtype=torch.int32, device=DEV)
    b = wide[:, 30:63]
    b.copy_(_i32(two))
    print(f'tables {n_blocks}', flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        pool.count(a)
    torch.cuda.synchronize()
    o.count(one)
    assert pool.counts.tolist() == o.counts
    pool.count(a, b)
    o.count(one, two)
    assert pool.counts.tolist() == o.counts
    for most in (5, None):
        moves = o.compact([one, two], n_blocks // 2 if most is None else most)
        src, dst, n = pool.compact(a, b, most=most)
        assert int(n) == len(moves) and list(zip(src[:len(moves)].tolist(), dst[:len(moves)].tolist())) == moves
        assert bool((src[len(moves):] == -1).all()) and bool((dst[len(moves):] == -1).all())
        assert pool.counts.tolist() == o.counts and a.tolist() == one.tolist() and b.tolist() == two.tolist()
    assert bool((wide[:, :30] == 7).all()) and bool((wide[:, 63:] == 7).all())
    src, dst, n = pool.compact(a, b)
    assert int(n) == 0
    used = sum(x > 0 for x in o.counts)
    pages, lens = torch.full((3, 4), -1, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    pool.grow(pages, lens, 65)                               # what was free is at the end now
    free = n_blocks - used
    assert pages.flatten().tolist() == [used + 2 * (i // 4) + i % 4 if i % 4 < 2 and 2 * (i // 4) + i % 4 < free else -1 for i in range(12)]


@pytest.mark.gpu
@pytest.mark.parametrize('heads,dim,bits', [(1, 32, 'int8'), (5, 96, 'fp8'), (16, 64, 'int8'), (3, 256, 'fp8'), (8, 128, 'int8')])
def test_copy(heads, dim, bits):
    c, _ = _cache(20, heads, dim, bits)
    k, v, f = c.k.view(torch.uint8).clone(), c.v.view(torch.uint8).clone(), c.scales.clone()
    src, dst = [3, 19, -1, 7, 7, 20, 2, 4, 6], [0, 1, 5, 8, 9, 10, 2, -1, 11]
    print(f'copy {heads} {dim} {bits}', flush=True)

    def want(n):
        for a, b in list(zip(src, dst))[:n]:
            if 0 <= a < 20 and 0 <= b < 20:
                k[b], v[b], f[b] = k[a], v[a], f[a]
        assert torch.equal(c.k.view(torch.uint8), k) and torch.equal(c.v.view(torch.uint8), v) and torch.equal(c.scales, f)

    c.copy(_i32(src), _i32(dst), _i32([0]))
    want(0)
    c.copy(_i32(src), _i32(dst), _i32([4]))
    want(4)
    c.copy(_i32(src), _i32(dst), _i32([-3]))
    c.copy(_i32(src), _i32(dst), _i32([100]))
    want(9)
    c.k.view(torch.uint8)[3] = 1
    k[3] = 1
    c.copy(_i32(src), _i32(dst))
    want(9)
    from blast3r_amd.kv_cache import KVCache
    KVCache(0, heads, dim, device=DEV).copy(_i32(src), _i32(dst))


@pytest.mark.gpu
def test_copy_past_32_bit_offsets():
    from blast3r_amd.kv_cache import KVCache
    n = 70_000
    c = KVCache(n, 8, 128, torch.int8, device=DEV)
    print('copy past 4 GB', flush=True)
    c.k[n - 1], c.v[n - 2], c.scales[n - 1] = 5, 7, 3.0
    c.copy(_i32([n - 1, n - 2, n - 2]), _i32([1, 2, n - 3]))
    assert bool((c.k[1] == 5).all()) and bool((c.v[2] == 7).all()) and bool((c.v[n - 3] == 7).all()) and bool((c.scales[1] == 3.0).all())
    assert not c.k[2].any() and not c.v[1].any() and not c.k[0].any()


@pytest.mark.gpu
def test_samples_of_prompts_through_the_cache():
    """Prompts, samples forked from them, drafted tokens given back, a sequence that ends, blocks moved together: every
    sequence attends to the tokens that it was given, with its shared blocks read once as with every list by itself; the same
    through a captured graph."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    H, G, D, S = 2, 2, 64, 6
    rng = np.random.default_rng(0)
    cache, pool = KVCache(90, H, D, torch.int8, device=DEV), BlockPool(90, device=DEV)
    pages, lens = torch.full((S, 10), -1, dtype=torch.int32, device=DEV), torch.zeros(S, dtype=torch.int32, device=DEV)
    mirror = [([], []) for _ in range(S)]                   # keys and values of each sequence
    put = lambda x: torch.tensor(x, dtype=torch.float32, device=DEV).bfloat16()  # noqa: E731
    print('samples', flush=True)

    def append(counts):
        k, v = (np.float64(_np(put(rng.normal(size=(sum(counts), H, D))))) for _ in range(2))
        moves = pool.grow(pages, lens, _i32(counts), max_new=max(counts))
        assert int(pool.missing) == 0
        cache.copy(*moves)
        off = _i32(np.concatenate(([0], np.cumsum(counts))))
        cache.append(put(k), put(v), pages, lens, offsets=off, max_new=max(counts))
        lens.add_(_i32(counts))
        at = 0
        for s, n in enumerate(counts):
            mirror[s] = ([*mirror[s][0], *k[at:at + n]], [*mirror[s][1], *v[at:at + n]])
            at += n

    def check(shared=0, **kw):
        """Rows over codes against attention over the values that were appended.  int8 keeps a normal number to half of 1/127
        of its block's largest, 0.015 (0.0084 in the mean square); a block that grows token by token is recoded a few times:
        0.08 at most, 0.025.  Queries have length 1, so scores move by 0.025, 0.1 at most, and results by that times a value's
        distance from their mean, 0.8 on the average: 0.16 in all."""
        q = torch.nn.functional.normalize(put(rng.normal(size=(S, H * G, D))).float(), dim=-1).bfloat16()
        got = cache.attend(q, pages, lens, shared=shared, scale=1.0, **kw)
        for s in range(S):
            k, v = (np.array(x) for x in mirror[s])
            for h in range(H * G):
                if not len(k):
                    assert not got[s, h].any()
                    continue
                z = k[:, h // G] @ _np(q)[s, h]
                p = np.exp(z - z.max())
                assert np.abs(_np(got)[s, h] - p @ v[:, h // G] / p.sum()).max() < 0.2, (s, h)
        return q, got

    append([200, 0, 0, 70, 0, 0])
    check()
    pool.fork(pages, lens, _i32([0, 0, 3, 0]), _i32([1, 2, 4, 5]))
    for a, b in ((0, 1), (0, 2), (3, 4), (0, 5)):
        mirror[b] = (list(mirror[a][0]), list(mirror[a][1]))
    check()
    append([1, 1, 1, 1, 0, 1])                               # four samples of the first prompt: three copies
    assert int((pool.counts > 0).sum()) == 4 + 3 + 2 + 1 and pages[4, 1] != pages[3, 1]
    q, got = check()
    # rows of the first prompt alone: they share three blocks
    rows = torch.tensor([0, 1, 2, 5], device=DEV)
    alone = cache.attend(q[rows], pages[rows], lens[rows], scale=1.0)
    joint = cache.attend(q[rows], pages[rows], lens[rows], scale=1.0, shared=3)
    assert torch.equal(alone, got[rows]) and float((alone - joint).float().abs().max()) < 0.02
    pool.grow(pages, lens, 130)                              # drafted and refused
    pool.trim(pages, last=lens)
    check()
    append([64, 3, 1, 1, 5, 200])
    check()
    pool.free(pages, lens, _i32([0, 3]))
    mirror[0] = mirror[3] = ([], [])
    q, got = check()
    moves = pool.compact(pages)
    cache.copy(*moves)
    used = int((pool.counts > 0).sum())
    assert int(moves[2]) > 0 and int(pages.max()) == used - 1
    assert torch.equal(cache.attend(q, pages, lens, scale=1.0), got)
    append([30, 1, 1, 64, 1, 1])
    check()
    # a step captured: the blocks that it takes depend on what the pool holds at each replay
    new = torch.zeros((S, H, D), dtype=torch.bfloat16, device=DEV)

    def step():
        cache.copy(*pool.grow(pages, lens, 1))
        cache.append(new, new, pages, lens)
        lens.add_(1)
        return cache.attend(q, pages, lens, scale=1.0, cap=40.0)

    state = [t.clone() for t in (pages, lens, pool.counts, pool._used, pool._marks, cache.k, cache.v, cache.scales)]

    def reset():
        for t, x in zip((pages, lens, pool._counts, pool._used, pool._marks, cache.k, cache.v, cache.scales), state):
            t.copy_(x)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    outs = []
    for t in range(70):
        new.copy_(put(rng.normal(size=(S, H, D))))
        if t == 20:
            pool.free(pages, lens, _i32([1]))               # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        outs.append((y.clone(), new.clone()))
    end = pages.tolist(), lens.tolist(), pool.counts.tolist()
    reset()
    for t, (y, n) in enumerate(outs):
        new.copy_(n)
        if t == 20:
            pool.free(pages, lens, _i32([1]))
        assert torch.equal(step(), y), t
    assert end == (pages.tolist(), lens.tolist(), pool.counts.tolist())


@pytest.mark.gpu
def test_pool_calls_of_nothing():
    """No blocks, no lists, lists without places."""
    from blast3r_amd.kv_pool import BlockPool
    none = torch.full((0, 4), -1, dtype=torch.int32, device=DEV)
    thin = torch.full((3, 0), -1, dtype=torch.int32, device=DEV)
    some = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    print('pool of nothing', flush=True)
    for n in (0, 5):
        pool = BlockPool(n, device=DEV)
        for pages in (none, thin, some.clone()):
            lens = torch.zeros(pages.shape[0], dtype=torch.int32, device=DEV)
            pool.count(pages)
            src, dst, m = pool.grow(pages, lens, 100)
            assert src.tolist() == dst.tolist() == [-1] * len(lens) and int(m) == 0
            assert int(pool.missing) == (max(0, 6 - n) if pages.numel() else 0)
            pool.fork(pages, lens, _i32([0, 1]), _i32([1, 2]))
            pool.trim(pages, first=lens, last=lens)
            assert not pool.counts.any()
            src, dst, m = pool.compact(pages)
            assert int(m) == 0 and src.tolist() == [-1] * (n // 2)
            pool.free(pages, lens)
            pool.free(pages, lens, _i32([0, 7, -1, 0]))
            assert not pool.counts.any() and int(pool.available()) == n


@pytest.mark.gpu
@pytest.mark.parametrize('n_blocks', [1, 31, 32, 33, 5000, 100_000])
def test_free_blocks_counted_in_a_graph(n_blocks):
    """What ``available`` says is that of the present counts, at each replay."""
    from blast3r_amd.kv_pool import BlockPool
    print(f'free blocks of {n_blocks}', flush=True)
    pool = BlockPool(n_blocks, device=DEV)
    assert pool.available().tolist() == [n_blocks]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        free = pool.available()
    pages = torch.full((2, n_blocks // 2 + 1), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    left = n_blocks
    for n in (64, 0, 640, 64 * (n_blocks // 2)):
        pool.grow(pages, lens, n)
        lens += n
        left = n_blocks - int((pages >= 0).sum())
        g.replay()
        assert free.tolist() == pool.available().tolist() == [left] == [int((pool.counts == 0).sum())]
    pool.free(pages, lens)
    g.replay()
    assert free.tolist() == [n_blocks]


# ---------------------------------------------------------------------------------- blocks that run out

KEPT = 1 << 30


def test_oracle_keeps_shared_blocks_that_there_is_no_other_for():
    p = otok.Pool(4)
    p.counts = [1, 3, 1, 0]
    rows = np.array([[1, -1], [1, -1], [1, -1]])
    assert p.grow(rows, [5, 5, 5], [1, 1, 1]) == [(1, 3)] and p.missing == 1       # the third cannot have it alone
    assert rows[:, 0].tolist() == [3, 1 + KEPT, 1 + KEPT] and p.counts == [1, 2, 1, 1]
    assert p.grow(rows, [6, 5, 5], [1, 1, 0]) == [] and p.missing == 1 and rows[:, 0].tolist() == [3, 1 + KEPT, 1 + KEPT]
    p.drop(rows[0])
    assert p.counts == [1, 2, 1, 0] and p.grow(rows, [0, 5, 5], [0, 1, 1]) == [(1, 3)] and p.missing == 0
    assert rows[:, 0].tolist() == [-1, 3, 1] and p.counts == [1, 1, 1, 1]
    rows[1, 0], p.counts[3] = 2 + KEPT, 0
    assert p.grow(rows, [0, 5, 5], [0, 1, 1]) == [] and rows[1, 0] == 2            # no list beside it any more
    rows[1, 0] = 2 + KEPT
    table, lens = rows.tolist(), [0, 5, 5]
    p.fork(table, lens, [1], [0], table, lens)
    assert table[0][0] == 2 + KEPT and p.counts == [1, 1, 2, 0]
    rows = np.array(table)
    p.count(rows)
    assert p.counts == [0, 1, 2, 0] and p.compact([rows], 4) == [(2, 0)] and rows[:, 0].tolist() == [KEPT, KEPT, 1]
    p.drop(rows[0])
    assert p.counts == [1, 1, 0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize('n_seqs', [1, 2, 5, 64, 1500])
@pytest.mark.parametrize('spare', [0, 1, 3, 700])
@pytest.mark.parametrize('new', [1, 70, 200])
def test_shared_blocks_stay_where_there_is_no_other(n_seqs, spare, new):
    """Forks of a few sequences that all grow, with fewer free blocks than that takes, others than those that grow among the
    holders: lists, counts and moves as the oracle's; again after some have ended; lists counted, forked and moved with marks."""
    rng = np.random.default_rng(n_seqs * 7 + spare)
    print(f'out of blocks {n_seqs} {spare} {new}', flush=True)
    most = -(-n_seqs // 5)
    b = Both(most * 3 + spare, n_seqs, 6)
    b.advance(b.grow([int(rng.integers(64, 190)) if s < most else 0 for s in range(n_seqs)]))
    b.same()

    def fork(parents, children):
        b.pool.fork(b.t, b.tl, _i32(parents), _i32(children))
        rows = b.pages.tolist()
        b.o.fork(rows, b.lens, parents, children, rows, b.lens)
        b.pages = np.array(rows)

    if n_seqs > most:
        fork(rng.integers(0, most, n_seqs - most).tolist(), list(range(most, n_seqs)))
    b.same()
    seen = False
    for step in range(6):
        counts = [0 if rng.random() < 0.2 else int(rng.integers(1, new + 1)) for _ in range(n_seqs)]
        b.grow(counts, max_new=new)
        b.same()
        seen = seen or bool((b.pages >= KEPT).any())
        # lists that got all that they asked for have the tokens
        fine = [all(0 <= x < KEPT for x in row[length // 64:-(-(length + n) // 64)]) and length + n <= 6 * 64 for row, length, n in zip(b.pages, b.lens, counts)]
        b.advance([n if f else 0 for n, f in zip(counts, fine)])
        if step == 1 and n_seqs > 4:                        # a child of a marked list, in the place of another
            marked = np.flatnonzero((b.pages >= KEPT).any(1))
            if len(marked) > 1:
                fork([int(marked[0])], [int(marked[-1])])
                b.same()
        if step == 2:
            b.pool.count(b.t)
            b.o.count(b.pages)
            b.same()
        if step == 3:
            size = len(b.o.counts) // 2
            b.moved(b.o.compact([b.pages], size), b.pool.compact(b.t), size)
            b.same()
        rows = rng.permutation(n_seqs)[:max(1, n_seqs // 4)].tolist()
        b.pool.free(b.t, b.tl, _i32(rows))
        for r in rows:
            b.o.drop(b.pages[r])
            b.lens[r] = 0
        b.same()
    assert seen or n_seqs < 64 or spare > 3
    for s in range(n_seqs):                                 # the last one has its blocks for itself
        if s != n_seqs - 1:
            b.o.drop(b.pages[s])
    b.pool.trim(b.t, last=_i32([0] * (n_seqs - 1) + [6 * 64]))
    b.lens = [0] * (n_seqs - 1) + b.lens[-1:]
    b.tl.copy_(_i32(b.lens))
    b.grow([0] * (n_seqs - 1) + [1])
    b.same()
    assert not (b.pages >= KEPT).any()


@pytest.mark.gpu
@pytest.mark.parametrize('seed', range(4))
def test_tokens_of_every_list_through_a_cache_that_runs_full(seed):
    """Every sequence reads back, token by token, what it was given, while lists are forked, cut, ended and moved in a pool that
    is often too small: a step that had no blocks is not counted, is appended all the same, and is done again later.  Rows hold
    127, which makes the factor 1, so that whole numbers are kept exactly.  Attention sees the tokens of marked blocks: a query
    along one token's key gives its value."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    rng = np.random.default_rng(seed)
    S, D, n_blocks = 7, 32, 16
    cache, pool = KVCache(n_blocks, 1, D, torch.int8, device=DEV), BlockPool(n_blocks, device=DEV)
    pages, lens = torch.full((S, 6), -1, dtype=torch.int32, device=DEV), torch.zeros(S, dtype=torch.int32, device=DEV)
    tokens = [[] for _ in range(S)]                          # their numbers
    last, short, marked = 0, 0, 0

    def rows(ids):
        x = np.zeros((len(ids), 1, D))
        x[:, 0, 0] = 127
        for d in range(12):                                  # the number's bits, as +-100: keys point different ways
            x[:, 0, 1 + d] = np.where(np.asarray(ids, int) >> d & 1, 100, -100)
        return x

    def check():
        counts = [len(t) for t in tokens]
        off = _i32(np.concatenate(([0], np.cumsum(counts))))
        assert lens.tolist() == counts
        if not sum(counts):
            return
        got = cache.read(pages, torch.zeros_like(lens), off, sum(counts), max_count=max(counts), dtype=torch.float32)
        want = rows(sum(tokens, []))
        for x in got:
            assert np.array_equal(_np(x), want)
        # one token of each, its 12 bits against others': a score of 12e4 of 0.01 against 10e4 at most
        pick = [t[int(rng.integers(0, len(t)))] if t else 0 for t in tokens]
        q = rows(pick)
        q[:, 0, 0] = 0
        for kw in (dict(), dict(cap=900.0)):
            o = _np(cache.attend(torch.tensor(q, device=DEV).half(), pages, lens, causal=False, scale=0.005, **kw))
            for s in range(S):
                assert np.array_equal(o[s], rows([pick[s]])[0] if tokens[s] else np.zeros((1, D))), s

    print(f'full cache {seed}', flush=True)
    # at first four lists share an open block, and a fifth one takes all but one of the others
    first = {0: [100, 0, 0, 0, 0, 0, 0], 2: [0] * 4 + [384, 384, 64], 3: [1] * 7, 4: [1] * 7, 6: [1] * 7}
    for step in range(40):
        what = int(rng.integers(0, 8)) if step > 6 else {1: 5, 5: 6}.get(step, 0)
        if what < 5:
            counts = first[step] if step in first else [int(rng.integers(0, 3)) if rng.random() < 0.6 else int(rng.integers(0, 80)) for _ in range(S)]
            counts = [min(n, 6 * 64 - len(t)) for n, t in zip(counts, tokens)]
            if sum(counts):
                cache.copy(*pool.grow(pages, lens, _i32(counts), max_new=max(counts)))
                ids = [[last + sum(counts[:s]) + i for i in range(n)] for s, n in enumerate(counts)]
                last = (last + sum(counts)) % 3000
                x = torch.tensor(rows(sum(ids, [])), dtype=torch.float32, device=DEV)
                cache.append(x, x, pages, lens, offsets=_i32(np.concatenate(([0], np.cumsum(counts)))), max_new=max(counts))
                table = pages.tolist()
                for s, n in enumerate(counts):
                    if all(0 <= b < KEPT for b in table[s][len(tokens[s]) // 64:-(-(len(tokens[s]) + n) // 64)]):
                        tokens[s] = tokens[s] + ids[s]
                    else:
                        short += 1
                marked += sum(b >= KEPT for row in table for b in row)
                lens.copy_(_i32([len(t) for t in tokens]))
        elif what == 5:
            order = rng.permutation(S).tolist() if step > 6 else list(range(S))
            pool.fork(pages, lens, _i32([order[0]] * 3), _i32(order[1:4]))
            for c in order[1:4]:
                tokens[c] = list(tokens[order[0]])
        elif what == 6:
            gone = [int(rng.integers(0, S))] if step > 6 else [6]
            pool.free(pages, lens, _i32(gone))
            tokens[gone[0]] = []
        else:
            tokens = [t[:max(0, len(t) - int(rng.integers(0, 70)))] if rng.random() < 0.5 else t for t in tokens]
            lens.copy_(_i32([len(t) for t in tokens]))
            pool.trim(pages, last=lens)
            cache.copy(*pool.compact(pages))
        check()
    assert short > 3 and marked > 0, (short, marked)


def test_oracle_gives_back_shared_blocks_past_the_tokens():
    p = otok.Pool(6)
    p.counts = [1, 2, 2, 1, 0, 0]
    rows = np.array([[0, 1, 2], [3, 1, 2]])
    assert p.grow(rows, [64, 192], [64, 0]) == [] and rows.tolist() == [[0, 4, 2], [3, 1, 2]] and p.counts == [1, 1, 2, 1, 1, 0]
    assert p.grow(rows, [64, 64], [128, 128]) == [] and p.missing == 0     # nobody has tokens in block 2
    assert rows.tolist() == [[0, 4, 2], [3, 1, 5]] and p.counts == [1, 1, 1, 1, 1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize('n_blocks,n_seqs,width,new', [(40, 3, 6, 64), (300, 9, 20, 200), (300, 9, 20, 1300), (4000, 700, 6, 130), (6000, 1500, 5, 300)])
def test_lists_cut_short_give_up_what_others_hold(n_blocks, n_seqs, width, new):
    """Forks whose lengths are set back without a trim, and that grow again: blocks that the others still hold are exchanged
    without a copy, those of one's own stay."""
    rng = np.random.default_rng(new)
    print(f'cut short {n_blocks} {n_seqs} {new}', flush=True)
    b = Both(n_blocks, n_seqs, width)
    b.advance(b.grow([int(rng.integers(64, 64 * width)) if s < max(1, n_seqs // 4) else 0 for s in range(n_seqs)]))
    for step in range(5):
        parents = rng.integers(0, max(1, n_seqs // 4), n_seqs - max(1, n_seqs // 4)).tolist()
        children = list(range(max(1, n_seqs // 4), n_seqs))
        b.pool.fork(b.t, b.tl, _i32(parents), _i32(children))
        rows = b.pages.tolist()
        b.o.fork(rows, b.lens, parents, children, rows, b.lens)
        b.pages = np.array(rows)
        for k in range(2):
            b.lens = [int(rng.integers(0, x + 1)) if rng.random() < 0.7 else x for x in b.lens]
            b.tl.copy_(_i32(b.lens))
            b.grow([0 if rng.random() < 0.2 else int(rng.integers(1, new + 1)) for _ in range(n_seqs)], max_new=new)
            b.same()
    b.pool.trim(b.t, last=b.tl)
    for s in range(n_seqs):
        b.o.drop(b.pages[s], keep=lambda x, s=s: 64 * x < b.lens[s])
    b.same()


@pytest.mark.gpu
def test_tokens_of_others_stay_when_a_list_is_cut_short():
    """A child that takes back tokens down to the middle of what it shares, and appends others."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    cache, pool = KVCache(12, 1, 32, torch.int8, device=DEV), BlockPool(12, device=DEV)
    pages, lens = torch.full((2, 6), -1, dtype=torch.int32, device=DEV), _i32([0, 0])
    rng = np.random.default_rng(0)
    x, y = (torch.tensor(rng.integers(-126, 127, (n, 1, 32)), dtype=torch.float32, device=DEV) for n in (300, 200))
    x[:, :, 0], y[:, :, 0] = 127, 127                        # the factor is 1, and whole numbers are kept
    print('cut short, through the cache', flush=True)
    pool.grow(pages, lens, _i32([300, 0]))
    cache.append(x, x, pages, lens, offsets=_i32([0, 300, 300]))
    lens[0] = 300
    pool.fork(pages, lens, _i32([0]), _i32([1]))
    for cut in (128, 70, 0):
        lens[1] = cut
        cache.copy(*pool.grow(pages, lens, _i32([0, 200])))
        cache.append(y, y, pages, lens, offsets=_i32([0, 0, 200]))
        lens[1] += 200
        k, v = cache.read(pages, _i32([0, 0]), _i32([0, 300, 500 + cut]), 500 + cut, dtype=torch.float32)
        for got in (k, v):
            assert torch.equal(got[:300], x) and torch.equal(got[300:300 + cut], x[:cut]) and torch.equal(got[300 + cut:], y)


def test_caches_have_fewer_blocks_than_marks_leave_numbers_for():
    from blast3r_amd import _lib
    L, p = _lib.lib(), 4096
    same = dict(k=p, v=p, scales=p, heads=1, dim=64, bits=1, n_seqs=1, pages=p, n_pages=1, dtype=2, n_rows=1, rows_per_seq=1, max_rows=1, n_blocks=(1 << 30) + 1)
    at = dict(lengths=p, q=p, o=p, q_heads=1, scale=1.0, n_splits=1)
    for call, a in ((L.ba_kv_write, _lib.BaKvArgs(**same, starts=p, rk=p, rv=p)), (L.ba_kv_read, _lib.BaKvArgs(**same, starts=p, rk=p, rv=p)),
                    (L.ba_kv_attend, _lib.BaKvAttendArgs(**same, **at)), (L.ba_kv_attend_scored, _lib.BaKvScoredArgs(**same, **at))):
        assert call(ctypes.byref(a), None) != 0 and b'bad sizes' in L.ba_last_error()


@pytest.mark.gpu
def test_steps_that_run_out_of_blocks_in_a_graph():
    """A captured step of samples whose pool runs full, with sequences ended between the replays, as the same step run eagerly:
    lists, lengths, counts and codes are equal after each."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.kv_pool import BlockPool
    S = 6
    print('full pool in a graph', flush=True)

    def start():
        cache, pool = KVCache(9, 2, 32, torch.int8, device=DEV), BlockPool(9, device=DEV)
        pages, lens = torch.full((S, 4), -1, dtype=torch.int32, device=DEV), _i32([0] * S)
        x = torch.randn((90, 2, 32), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
        pool.grow(pages, lens, _i32([90, 0, 0, 0, 0, 0]))
        cache.append(x, x, pages, lens, offsets=_i32([0] + [90] * S))
        lens[0] = 90
        pool.fork(pages, lens, _i32([0] * 5), _i32([1, 2, 3, 4, 5]))
        new = torch.zeros((S, 2, 32), device=DEV)

        def step():
            cache.copy(*pool.grow(pages, lens, 1))
            cache.append(new, new, pages, lens)
            at = pages.gather(1, (lens // 64).long()[:, None])[:, 0]
            lens.add_(((at >= 0) & (at < KEPT)).int())       # of the lists that had room
            return cache.attend(new.bfloat16(), pages, lens)

        return cache, pool, pages, lens, new, step

    one, two = start(), start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        start()[-1]()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = one[-1]()
    seen = 0
    for t in range(60):
        x = torch.randn((S, 2, 32), device=DEV, generator=torch.Generator(device=DEV).manual_seed(t))
        for state in (one, two):
            state[4].copy_(x)
            if t in (10, 45):
                state[1].free(state[2], state[3], _i32([t // 10]))
        graph.replay()
        torch.cuda.synchronize()
        want = two[-1]()
        assert torch.equal(y, want), t
        seen += int((two[2] >= KEPT).any()) + int(two[1].missing > 0)
        for a, b in ((one[2], two[2]), (one[3], two[3]), (one[1].counts, two[1].counts), (one[1].missing, two[1].missing), (one[0].k, two[0].k), (one[0].v, two[0].v)):
            assert torch.equal(a, b), t
    assert seen > 10
