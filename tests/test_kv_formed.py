"""Attention over the 8-bit cache with capped scores, biases by distance, masks by row and lists that begin alike: oracle pins
and refusals (CPU), parity with the oracle (GPU).

Bars: those of tests/test_tokens.py's attention (weights in fp16, scores in fp32: 1.2e-3 sum p |v| and half a step of the output;
6e-4 for lse), in which what is new has room: a capped score is off by 4e-7 cap at most, 2e-5 of a weight for the caps here; a
bias that matters is below 2^6 in the exponents of 2, with three roundings of fp32, 1e-5.  Where distances are measured from
far tokens, lse adds slope times distance once: 2^-23 of it."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import tokens as otok
from test_tokens import HALF_STEP, _cache, _i32, _mirror, _np, _pages

DEV = 'cuda:0'


# ---------------------------------------------------------------------------------- oracle pins (CPU)

def test_oracle_with_nothing_formed_is_plain_attention():
    rng = np.random.default_rng(0)
    c = otok.Cache(rng.normal(size=(5, 2, 64, 32)), rng.normal(size=(5, 2, 64, 32)), np.ones((5, 2, 2)), 'int8')
    q = rng.normal(size=(9, 4, 32))
    for kw in (dict(), dict(causal=False), dict(window=20)):
        for x, y in zip(otok.attend(c, q, [[0, 2], [3, -1]], [100, 70], [3, 6], 0.2, **kw),
                        otok.attend_formed(c, q, [[0, 2], [3, -1]], [100, 70], [3, 6], 0.2, cap=1e9, slopes=[0.0] * 4,
                                           prefix=[0, -1], since=[0] * 9, until=[200] * 9, **kw)):
            assert np.allclose(x, y, rtol=1e-9, atol=1e-12)


def test_oracle_known_answers():
    """Two keys of scores 3 and 1 with values 1 and 0: the weights are known."""
    k, v = np.zeros((1, 1, 64, 32)), np.zeros((1, 1, 64, 32))
    k[0, 0, 0, 0], k[0, 0, 1, 0], v[0, 0, 0] = 3.0, 1.0, 1.0
    c = otok.Cache(k, v, np.ones((1, 1, 2)), 'int8')
    q = np.zeros((1, 1, 32))
    q[0, 0, 0] = 1.0
    run = lambda **kw: otok.attend_formed(c, q, [[0]], [2], [1], 1.0, **kw)[0][0, 0, 0]  # noqa: E731
    sig = lambda x: 1 / (1 + math.exp(-x))  # noqa: E731
    assert abs(run() - sig(2.0)) < 1e-12
    assert abs(run(cap=2.0) - sig(2 * math.tanh(1.5) - 2 * math.tanh(0.5))) < 1e-12
    assert abs(run(slopes=[0.5]) - sig(2.0 - 0.5)) < 1e-12                 # the first key is one token away
    assert run(since=[1]) == 0.0 and run(until=[1]) == 1.0 and run(since=[2]) == 0.0 and run(since=[1], prefix=[1]) == run()
    assert run(window=1) == 0.0 and abs(run(window=1, prefix=[1]) - sig(2.0)) < 1e-12


# ---------------------------------------------------------------------------------- refusals (CPU)

def test_formed_entry_point_refuses_bad_arguments_without_a_gpu():
    from blast3r_amd import _lib
    L = _lib.lib()
    p = 4096                                                # addresses that are only compared with each other
    good = dict(n_blocks=2, heads=2, dim=64, bits=0, n_seqs=1, n_pages=2, pages_stride=2, dtype=2, n_rows=3, rows_per_seq=3, max_rows=3,
                q_heads=4, scale=1.0, n_splits=1, k=p, v=p, scales=p, pages=p, lengths=p, q=p, o=p)
    assert L.ba_kv_attend_scored(None, None) != 0
    for word, kw in (('cap', dict(cap=-1.0)), ('cap', dict(cap=math.nan)), ('cap', dict(cap=1e4)), ('cap', dict(cap=math.inf)),
                     ('cap', dict(cap=1e-4)), ('shared', dict(shared=3, shared_parts=1)), ('shared', dict(shared=-1)),
                     ('shared_parts', dict(shared=1)), ('shared_parts', dict(shared_parts=1)), ('parts', dict(n_splits=65536, shared=1, shared_parts=1)),
                     ('null pointer', dict(shared=1, shared_parts=1)), ('too small', dict(shared=1, shared_parts=1, workspace=p, workspace_bytes=64)),
                     ('head size', dict(dim=48)), ('aligned', dict(k=p + 8)), ('null pointer', dict(q=None)), ('scale', dict(scale=0.0)),
                     ('too many', dict(n_seqs=1 << 23)), ('too many', dict(n_rows=(1 << 31) - 1, shared=1, shared_parts=1, offsets=p)),
                     ('fp16 or bf16', dict(dtype=0)), ('bad sizes', dict(window=-1))):
        a = _lib.BaKvScoredArgs(**{**good, **kw})
        assert L.ba_kv_attend_scored(ctypes.byref(a), None) != 0 and word in L.ba_last_error().decode(), (kw, L.ba_last_error())
    assert L.ba_kv_attend_scored(ctypes.byref(_lib.BaKvScoredArgs(**{**good, 'n_rows': 0})), None) == 0
    for kw in (dict(), dict(shared=2), dict(shared=1, window=5), dict(n_rows=0), dict(n_seqs=0, shared=1), dict(max_rows=0), dict(n_pages=0),
               dict(n_seqs=64, n_rows=64, rows_per_seq=1, max_rows=1, n_pages=300, shared=256), dict(n_rows=9000, max_rows=9000, n_pages=900, dim=256),
               dict(n_rows=9000, max_rows=9000, n_pages=900, since=p), dict(n_seqs=(1 << 31) - 1, heads=65536, q_heads=65536, n_rows=(1 << 31) - 1, max_rows=(1 << 31) - 1),
               dict(n_rows=(1 << 31) - 1, max_rows=(1 << 31) - 1, n_pages=(1 << 24) - 1)):
        a = _lib.BaKvScoredArgs(**{**good, **kw})
        L.ba_kv_scored_plan(a)
        assert 1 <= a.n_splits <= 64 or a.max_rows == 1 and a.n_splits <= 384
        assert a.shared_parts >= 1 if a.shared else a.shared_parts == 0
        assert a.tile in (0, 16, 32, 128, 256) and a.shared_tile in (0, 16, 32, 128, 256) and not (a.dim == 256 and a.tile == 256)
    plans = []                                               # a window wider than any list is none
    for window in (0, 1 << 35, (1 << 63) - 1):
        plans.append(_lib.BaKvScoredArgs(**{**good, 'window': window, 'n_pages': 300, 'max_rows': 1, 'rows_per_seq': 1, 'n_rows': 1}))
        L.ba_kv_scored_plan(plans[-1])
    assert plans[0].n_splits > 1 and len({(a.n_splits, a.tile) for a in plans}) == 1
    assert L.ba_kv_attend_scored(ctypes.byref(_lib.BaKvScoredArgs(**{**good, 'tile': 64})), None) != 0 and 'tiles' in L.ba_last_error().decode()
    assert L.ba_kv_attend_scored(ctypes.byref(_lib.BaKvScoredArgs(**{**good, 'shared_tile': 256, 'dim': 256})), None) != 0


@pytest.fixture
def host(monkeypatch):
    """KVCache over host tensors; the arguments of each launch are kept."""
    from blast3r_amd import kv_cache
    calls = []
    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    monkeypatch.setattr(kv_cache, 'launch', lambda call, args, device: calls.append(type(args).from_buffer_copy(args)))
    return calls


def test_python_refuses_bad_masks_and_scores(host):
    from torch.autograd import forward_ad

    from blast3r_amd.kv_cache import KVCache
    c = KVCache(4, 2, 64, device='cpu')
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q, pages, lens = torch.zeros(4, 4, 64, dtype=torch.bfloat16), i32([[0, 1], [2, 3]]), i32([5, 6])
    for kw in (dict(cap=0.0), dict(cap=-1.0), dict(cap=math.nan), dict(cap=1e9), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(4).double()),
               dict(slopes=torch.zeros(8)[::2]), dict(prefix=i32([1])), dict(prefix=lens.long()), dict(since=i32([1, 2])), dict(until=i32([0] * 5)),
               dict(until=i32([[0] * 4])), dict(shared=3), dict(shared=-1)):
        with pytest.raises(ValueError):
            c.attend(q, pages, lens, **kw)
    with pytest.raises(RuntimeError, match='gradient'):
        c.attend(q, pages, lens, slopes=torch.zeros(4, requires_grad=True))
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match='gradient'):
        c.attend(q, pages, lens, slopes=forward_ad.make_dual(torch.zeros(4), torch.zeros(4)))
    assert not host
    with torch.no_grad():
        c.attend(q, pages, lens, slopes=torch.zeros(4, requires_grad=True))
    c.attend(q, pages, lens, cap=50.0, prefix=i32([1, 2]), since=i32([0] * 4), until=i32([9] * 4), shared=1)
    a = host[-1]
    assert a.cap == 50.0 and a.n_splits >= 1 and a.prefix and a.since and a.until and not a.slopes
    assert a.shared == a.shared_parts == 0                  # two blocks are not worth another launch
    many, long = torch.zeros(64, 4, 64, dtype=torch.bfloat16), torch.zeros(64, 300, dtype=torch.int32)
    c.attend(many, long, torch.zeros(64, dtype=torch.int32), shared=256)
    assert host[-1].shared == 256 and host[-1].shared_parts >= 1
    c.attend(q, pages, lens)                                # what was there goes the way it went
    assert type(host[-1]).__name__ == 'BaKvAttendArgs' and type(a).__name__ == 'BaKvScoredArgs'
    for kw in (dict(cap=1.0), dict(shared=1)):
        c.attend(q[:0], i32(np.zeros((0, 2))), i32([]), **kw)


# ---------------------------------------------------------------------------------- parity (GPU)

class Planned:
    """The library with a plan of the test's choosing: parts and tiles of the sequences' own blocks and of the shared ones."""

    def __init__(self, shared, own=1, common=1, tile=0, shared_tile=0):
        from blast3r_amd import _lib
        self.lib, self.plan = _lib.lib(), (shared, own, common, tile, shared_tile)

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def ba_kv_scored_plan(self, a):
        a.shared, a.n_splits, a.shared_parts, a.tile, a.shared_tile = self.plan
        if not a.shared:
            a.shared_parts = 0


def _run(c, o, q, pages, lens, counts, scale=None, shared=0, uniform=False, max_new=None, out=None, **kw):
    """attend() and what the oracle says; rows within max_new are compared."""
    off = None if uniform else _i32(np.concatenate(([0], np.cumsum(counts))))
    dev = {n: (torch.tensor(np.asarray(x), dtype=torch.float32 if n == 'slopes' else torch.int32, device=DEV) if n in ('slopes', 'prefix', 'since', 'until') and x is not None else x)
           for n, x in kw.items()}
    got, lse = c.attend(q, _i32(pages), _i32(lens), offsets=off, max_new=max_new or max(max(counts), 1), scale=scale, return_lse=True, shared=shared,
                        out=out, **dev)
    want, want_lse, size = otok.attend_formed(o, _np(q), pages, lens, counts, scale or 1.0 / math.sqrt(q.shape[2]), **kw)
    assert np.array_equal(np.isnan(_np(got)), np.isnan(want))
    ok = ~np.isnan(want)
    step = HALF_STEP[q.dtype] * np.abs(want) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    err = np.abs(_np(got) - want)[ok]
    cap = 4e-7 * (kw.get('cap') or 0.0)                     # weights move by the errors of two capped scores at most
    bar = ((1.2e-3 + 2 * cap) * size + step)[ok]
    assert np.all(err <= bar), float(np.max(err / np.maximum(bar, 1e-300)))
    assert np.array_equal(_np(lse) == -math.inf, want_lse == -math.inf)
    fine = np.isfinite(want_lse)
    assert np.all(np.abs(_np(lse)[fine] - want_lse[fine]) <= 6e-4 + cap + 2.0 ** -22 * np.abs(want_lse[fine]))
    return got


def _masks(rng, lens, counts, kind):
    """since, until of the rows: documents in a row, frames, or anything, rows that see nothing among them."""
    since, until = [], []
    for length, n in zip(lens, counts):
        length = max(length, 1)
        edges = np.unique(np.concatenate(([0], rng.integers(0, length + 1, 1 + length // 60), [length])))
        for i in range(n):
            at = max(0, length - n + i)
            e = int(np.searchsorted(edges, at, side='right'))
            lo, hi = int(edges[e - 1]), int(edges[min(e, len(edges) - 1)])
            if kind == 'any':
                lo, hi = (int(x) for x in rng.integers(-5, length + 9, 2))
            since.append(lo)
            until.append(hi)
    return since, until


FORMED = [
    # dim, heads, group, lengths, counts, options
    (64, 2, 1, [1, 64, 65, 200], [1, 1, 1, 1], dict(cap=5.0)),
    (64, 1, 4, [700, 3, 0, 129], [1, 2, 1, 4], dict(slopes=True, prefix=[5, 1, 3, 70])),
    (128, 2, 8, [300, 900], [1, 1], dict(window=100, prefix=[64, 3])),
    (128, 1, 5, [333], [6], dict(mask='documents', cap=20.0)),
    (96, 2, 3, [100, 257], [10, 40], dict(window=37, prefix=[0, -4], slopes=True)),
    (64, 1, 1, [5, 90], [9, 33], dict(cap=1.0, prefix=[100, 80])),         # more rows than tokens; prefix past the length
    (32, 2, 2, [500], [70], dict(causal=False, mask='frames')),
    (64, 1, 2, [400, 191], [150, 63], dict(mask='documents', slopes=True)),
    (128, 1, 1, [330], [300], dict(causal=False, slopes=True)),            # tokens on both sides of a row
    (128, 2, 2, [600, 1], [250, 1], dict(mask='any', cap=50.0)),
    (256, 1, 2, [300], [80], dict(mask='any', causal=False, slopes=True, cap=7.0)),
    (256, 2, 1, [650], [1], dict(slopes=True, window=200, prefix=[10])),
    (32, 1, 16, [4000], [1], dict(window=64, prefix=[1], cap=30.0)),
    (64, 1, 1, [3000], [3], dict(mask='any', causal=False, prefix=[130])),
    (96, 2, 3, [190, 2500], [70, 1], dict(mask='frames', causal=False, prefix=[7, 1000])),
    (64, 2, 1, [70, 0, 1, 2100], [70, 0, 1, 300], dict(window=200, prefix=[64, 1, 1, 65], slopes=True)),
    (96, 1, 2, [1300], [200], dict(mask='documents', window=50)),
    (256, 1, 4, [700], [6], dict(mask='documents', causal=False, cap=12.0)),
    (32, 1, 2, [900], [300], dict(cap=3.0, slopes=True, causal=False, prefix=[500])),
]


def _case(rng, dim, heads, group, lens, counts, bits, opts, dtype, more=1):
    blocks = [max(1, (n + 63) // 64) for n in lens]
    c, o = _cache(sum(blocks) + 1, heads, dim, bits, seed=dim)
    pages = _pages(rng, blocks, sum(blocks) + 1, max(blocks) + 2)
    for s, n in enumerate(lens):                            # codes of places that hold no token yet may be anything
        if n % 64:
            p = int(pages[s, n // 64])
            c.k.view(torch.uint8)[p, :, n % 64:] = 0x7f
            c.v.view(torch.uint8)[p, :, :, n % 64:] = 0x7f
    opts = dict(opts)
    kind = opts.pop('mask', None)
    if kind:
        since, until = _masks(rng, lens, counts, kind)
        opts.update({'documents': dict(since=since), 'frames': dict(until=until), 'any': dict(since=since, until=until)}[kind])
    if opts.get('slopes'):
        opts['slopes'] = [float(np.float32(2.0 ** (-8.0 * (h + 1) / (heads * group)))) for h in range(heads * group)]
    x = torch.tensor(rng.normal(size=(sum(counts), heads * group + 1, dim)) * 2.0, dtype=torch.float32).to(dtype).to(DEV)
    return c, o, x[:, 1:], pages, opts


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dim,heads,group,lens,counts,opts', FORMED)
def test_formed_attention_against_oracle(bits, dim, heads, group, lens, counts, opts):
    rng = np.random.default_rng(sum(lens))
    for dtype in (torch.bfloat16, torch.float16):
        c, o, q, pages, kw = _case(rng, dim, heads, group, lens, counts, bits, opts, dtype)
        print(f'formed {bits} {dtype} {dim} {heads} {group} {lens} {counts} {opts}', flush=True)
        _run(c, o, q, pages, lens, counts, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize('counts', [[1], [3], [12], [40], [150], [300]])
def test_formed_attention_ranges(counts):
    """Factors far apart in neighbouring blocks, missing blocks, a NaN block that only some rows see, slopes from 2^-12 to 4 of
    either sign, caps from 1e-3 up, scores far past the cap."""
    rng = np.random.default_rng(counts[0])
    n = 64 * 20 - 11
    c, o = _cache(22, 1, 64, 'int8')
    pages = _pages(rng, [20], 22, 20)
    for b in range(20):
        e = int(rng.integers(-20, 20))
        c.scales[int(pages[0, b]), 0] = torch.tensor([2.0 ** (-7 - abs(e) / 4), 2.0 ** (2 * e)], device=DEV)
    pages[0, 3] = -1
    pages[0, 7] = 22
    o = _mirror(c, 'int8')
    x = rng.normal(size=(counts[0], 2, 64)) * np.exp(rng.normal(size=(counts[0], 2, 1)) * 2)
    x[0, 0] = 0.0
    q = torch.tensor(x, dtype=torch.float32).clamp(-8, 8).bfloat16().to(DEV)
    print(f'formed ranges {counts}', flush=True)
    for cap in (1e-3, 0.7, 40.0, 1e3):
        _run(c, o, q, pages, [n], counts, cap=cap)
    for slopes in ([2.0 ** -12, 4.0], [-0.01, 0.25], [0.0, 1.0]):
        _run(c, o, q, pages, [n], counts, slopes=slopes)
        _run(c, o, q, pages, [n], counts, slopes=slopes, causal=False, cap=30.0)
    c.scales[int(pages[0, 19]), 0, 0] = math.nan
    c.scales[int(pages[0, 2]), 0, 1] = math.nan
    o = _mirror(c, 'int8')
    _run(c, o, q, pages, [n], counts, window=64 * 10, cap=9.0)
    _run(c, o, q, pages, [n], counts, since=[64 * 3 + i % 200 for i in range(counts[0])], until=[64 * 19 + (i % 3 - 1) for i in range(counts[0])],
         slopes=[0.1, 0.02])
    _run(c, o, q, pages, [n], counts, since=[64 * 4] * counts[0], prefix=[64 * 2 + 1])
    q = q.clone()
    q[0, 1, 5] = math.nan                                   # a row of NaN scores, its neighbours as they were
    for kw in (dict(cap=20.0), dict(slopes=[0.01, 0.5]), dict(prefix=[64]), dict(cap=3.0, slopes=[0.01, 0.5])):
        _run(c, o, q, pages, [64 * 19], counts, window=64 * 12, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 20, 100])
def test_slopes_over_far_tokens_only(n):
    """Rows that see nothing but tokens far away: their biases differ by little beside their size.  Distances are measured from
    the nearest of them (with negative slopes: the farthest), so nothing is lost."""
    rng = np.random.default_rng(n)
    length = 64 * 400
    c, o = _cache(40, 1, 64, 'fp8')
    pages = np.full((1, 400), -1)
    pages[0, :20] = np.arange(20)                           # the blocks after the first 20 are not there
    pages[0, 380:] = 20 + np.arange(20)
    q = torch.tensor(rng.normal(size=(n, 2, 64)), dtype=torch.float32, device=DEV).bfloat16()
    print(f'far tokens {n}', flush=True)
    for slopes in ([0.5, 0.01], [-0.5, -0.003]):
        _run(c, o, q, pages, [length], [n], slopes=slopes, until=[1000 + i for i in range(n)])
        _run(c, o, q, pages, [length], [n], slopes=slopes, since=[length] * n, prefix=[700])


# ---------------------------------------------------------------------------------- lists that begin alike (GPU)

SHARED = [
    # dim, heads, group, shared blocks, lengths, counts, options
    (64, 2, 1, 1, [65, 64, 200, 70], [1, 1, 1, 1], {}),
    (128, 1, 4, 5, [700, 330, 320, 323], [1, 2, 0, 4], {}),
    (128, 2, 2, 20, [1281 + 7 * i for i in range(40)], [1] * 40, dict(cap=20.0)),
    (96, 2, 3, 3, [300, 457], [10, 40], dict(window=137)),
    (64, 1, 1, 4, [100, 290, 3], [9, 33, 3], {}),                          # sequences that end within the shared blocks
    (64, 1, 2, 10, [840, 660, 640], [150, 20, 0], dict(slopes=True)),
    (64, 4, 1, 12, [768 + 100] * 5, [100] * 5, dict(causal=False)),
    (256, 1, 2, 6, [500, 390], [80, 3], dict(prefix=[70, 1], window=60)),
    (32, 1, 8, 30, [2000, 1921], [5, 1], dict(cap=10.0, slopes=True)),
    (128, 1, 1, 9, [900, 700], [300, 90], dict(mask='any', causal=False)),
    (64, 2, 2, 7, [448, 448], [1, 1], {}),                                 # nothing of their own
    (128, 2, 4, 40, [2700], [1], {}),                                      # one sequence
]


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dim,heads,group,shared,lens,counts,opts', SHARED)
def test_shared_blocks_against_oracle(bits, dim, heads, group, shared, lens, counts, opts):
    rng = np.random.default_rng(sum(lens))
    c, o, q, pages, kw = _case(rng, dim, heads, group, lens, counts, bits, opts, torch.bfloat16)
    longest = int(np.argmax(lens))
    pages[:, :shared] = pages[longest, :shared]
    o = _mirror(c, bits)
    print(f'shared {bits} {dim} {heads} {group} {shared} {lens} {counts} {opts}', flush=True)
    uniform = len(set(counts)) == 1
    _run(c, o, q, pages, lens, counts, shared=shared, uniform=uniform, **kw)             # as it is planned
    real = c._lib
    for plan in ((), (1, 1, 16, 128), (2, 3, 32, 32), (2, 3, 16, 32), (3, 1, 32, 16), (3, 2, 128, 16), (1, 7, 0, 256 if dim < 256 else 128)):
        print(f'  plan {plan}', flush=True)
        c._lib = Planned(shared, *plan)
        a = _run(c, o, q, pages, lens, counts, shared=shared, uniform=uniform, **kw)
        assert torch.equal(a, _run(c, o, q, pages, lens, counts, shared=shared, uniform=uniform, **kw))
    c._lib = real


@pytest.mark.gpu
@pytest.mark.parametrize('counts', [[1] * 5, [40] * 5, [0, 3, 0, 90, 1]])
def test_shared_blocks_of_a_batch_with_empty_places(counts):
    """Places of the batch without a sequence (no tokens, no blocks) among others, the first one too."""
    rng = np.random.default_rng(sum(counts))
    lens = [0, 700, 0, 650, 500]
    c, o, q, pages, _ = _case(rng, 64, 2, 2, lens, counts, 'int8', {}, torch.bfloat16)
    pages[:, :7] = pages[1, :7]
    pages[0], pages[2] = -1, -1
    for plan in ((2, 2, 0, 0), (1, 1, 32, 128)):
        print(f'empty places {counts} {plan}', flush=True)
        c._lib = Planned(7, *plan)
        _run(c, o, q, pages, lens, counts, shared=7, uniform=len(set(counts)) == 1, max_new=max(counts))
        _run(c, o, q, pages, lens, counts, shared=7, uniform=len(set(counts)) == 1, cap=20.0, slopes=[0.1, 0.01, 0.2, 0.0])


@pytest.mark.gpu
@pytest.mark.parametrize('dim,heads,group,lens,counts,opts', [
    (64, 1, 2, [900, 191], [200, 63], dict(slopes=True)), (128, 2, 1, [1500], [300], dict(cap=9.0)), (256, 1, 1, [800], [150], dict(mask='any')),
    (96, 1, 3, [1200], [5], dict(prefix=[200], window=300)), (32, 1, 1, [700, 650], [300, 1], dict(mask='frames', causal=False))])
def test_every_plan_gives_the_result(dim, heads, group, lens, counts, opts):
    """Tiles of every size, and parts without blocks among them."""
    rng = np.random.default_rng(sum(lens))
    c, o, q, pages, kw = _case(rng, dim, heads, group, lens, counts, 'fp8', opts, torch.float16)
    for tile in (16, 32, 128, 256):
        for parts in (1, 2, 5, 40):
            print(f'plan {dim} {tile} {parts}', flush=True)
            c._lib = Planned(0, parts, 0, tile if dim < 256 else min(tile, 128))
            _run(c, o, q, pages, lens, counts, **kw)


@pytest.mark.gpu
def test_shared_rows_that_no_sequence_has_are_left_alone():
    """Rows past max_new, past the last sequence or before the first are not written, nor is their lse."""
    rng = np.random.default_rng(5)
    c, o = _cache(8, 2, 64, 'fp8')
    pages = np.array([[0, 1, 2, 3], [0, 1, 4, 5]])
    for n, most in ((3, 2), (40, 30), (200, 100)):
        lens, total = [200, 256], n + 5 + 4
        q = torch.tensor(rng.normal(size=(total, 4, 64)), dtype=torch.float32, device=DEV).bfloat16()
        y = torch.full_like(q, 7.0)
        print(f'shared bounds {n}', flush=True)
        off = _i32([2, 2 + n, 2 + n + 5])
        c._lib = Planned(2, 2, 2)
        _, lse = c.attend(q, _i32(pages), _i32(lens), offsets=off, max_new=most, out=y, shared=2, return_lse=True, cap=9.0)
        rows = _np(q)[2:2 + n + 5]
        want, _, size = otok.attend_formed(o, rows, pages, lens, [n, 5], 0.125, cap=9.0)
        done = np.r_[0:min(n, most), n:n + min(5, most)]
        assert np.all(np.abs(_np(y)[2:2 + n + 5] - want)[done] <= 1.2e-3 * size[done] + 2.0 ** -8 * np.abs(want[done]))
        rest = np.setdiff1d(np.arange(total), 2 + done)
        assert bool((y[torch.tensor(rest, device=DEV)] == 7.0).all())


@pytest.mark.gpu
def test_formed_calls_of_bad_lists_stay_inside():
    """Lengths past the lists, negative ones, offsets out of order, a cache without blocks: zeros or untouched rows."""
    from blast3r_amd.kv_cache import KVCache
    c, o = _cache(8, 2, 64, 'int8')
    none = KVCache(0, 2, 64, device=DEV)
    print('formed bad lists', flush=True)
    slopes = torch.tensor([0.1, 0.2], device=DEV)
    for n in (2, 40, 400):
        q = torch.randn((n, 2, 64), device=DEV).bfloat16()
        for kw in (dict(cap=5.0), dict(slopes=slopes), dict(prefix=_i32([9, 100000])), dict(shared=2), dict(shared=3, cap=4.0)):
            none._lib = c._lib = Planned(kw.get('shared', 0), 1, 2)
            got, lse = none.attend(q, _i32(np.zeros((2, 3))), _i32([150, 20]), return_lse=True, **kw)
            assert not got.any() and bool((lse == -math.inf).all())
            got = c.attend(q, _i32([[0, 1, -1], [9, 99, 1 << 30]]), _i32([100000, -5]), **kw)
            assert bool(torch.isfinite(got).all()) and not got[n // 2:].any()
            y = torch.full_like(q, 7.0)
            c.attend(q, _i32([[0, 1, 2]] * 2), _i32([50, 60]), offsets=_i32([n + 9, -2, n + 4]), out=y, **kw)
            assert bool((y == 7.0).all())
    c._lib = c._lib.lib
    assert not c.attend(q[:2], _i32(np.zeros((2, 0))), _i32([5, 6]), prefix=_i32([3, 4])).any()


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 5, 20, 100, 300])
def test_formed_queries_and_outputs_at_odd_places(n):
    """Queries and outputs that are not aligned for wide loads and stores, with heads and rows apart by odd numbers, in place
    too: as with aligned ones."""
    rng = np.random.default_rng(n)
    c, o = _cache(12, 2, 64, 'int8')
    pages, lens, counts = _pages(rng, [12], 12, 12), [700], [n]
    pages[:, 11] = -1
    real = c._lib
    base = torch.tensor(rng.normal(size=(2, n * 331 + 5)) * 2, dtype=torch.float32).bfloat16().to(DEV)
    q, y = (b[1:1 + n * 331].view(n, 331)[:, :4 * 67].unflatten(1, (4, 67))[..., 1:65] for b in base)
    print(f'odd places {n}', flush=True)
    for kw in (dict(cap=8.0), dict(slopes=[0.1, 0.0, 0.01, 0.3]), dict(prefix=[70], window=90), dict(cap=8.0, slopes=[0.1, 0.0, 0.01, 0.3], shared=3)):
        for plan in (None, (1, 0), (3, 2)):
            shared = kw.get('shared', 0)
            c._lib = real if plan is None else Planned(shared, plan[0], max(1, plan[1]))
            rest = base.clone()
            want = _run(c, o, q.contiguous(), pages, lens, counts, **kw)
            assert torch.equal(_run(c, o, q, pages, lens, counts, out=y, **kw), want)
            mine = torch.zeros_like(base[1], dtype=torch.bool)
            mine[1:1 + n * 331].view(n, 331)[:, :4 * 67].unflatten(1, (4, 67))[..., 1:65] = True
            assert torch.equal(base[1][~mine], rest[1][~mine]) and torch.equal(base[0], rest[0])
            z = q.clone()
            assert torch.equal(c.attend(z, _i32(pages), _i32(lens), out=z, shared=shared, **{
                k: (torch.tensor(v, device=DEV, dtype=torch.float32 if k == 'slopes' else torch.int32) if isinstance(v, list) else v)
                for k, v in kw.items() if k != 'shared'}), want)


@pytest.mark.gpu
def test_formed_attention_over_a_long_list_with_blocks_past_4_gigabytes():
    """400000 positions, of which a window, a prefix and single documents are there, in a cache of 9 GB."""
    from blast3r_amd.kv_cache import KVCache
    n, H, D, length = 70_000, 8, 128, 400_000
    c = KVCache(n, H, D, torch.int8, device=DEV)
    small, _ = _cache(8, H, D, 'int8')
    where = [0, 3, n - 1, n - 2, n - 5, 35_000, 5, n - 9]
    c.k[where], c.v[where], c.scales[where] = small.k, small.v, small.scales
    last = length // 64
    at = [0, 1, 3000, 3001, last - 2, last - 1, last, 4000]
    pages, short = np.full((1, last + 1), -1), np.full((1, last + 1), -1)
    pages[0, at], short[0, at] = where, np.arange(8)
    o = _mirror(small, 'int8')
    rng = np.random.default_rng(0)
    for m in (1, 30, 100):
        q = torch.tensor(rng.normal(size=(m, H, D)), dtype=torch.float32, device=DEV).bfloat16()
        slopes = [2.0 ** -(i + 6) for i in range(H)]
        print(f'long list {m}', flush=True)
        for kw in (dict(window=150, prefix=[100]), dict(slopes=slopes), dict(since=[3000 * 64 + 5] * m, until=[4001 * 64] * m, cap=20.0)):
            dev = {k: (torch.tensor(v, device=DEV, dtype=torch.float32 if k == 'slopes' else torch.int32) if isinstance(v, list) else v) for k, v in kw.items()}
            got = _np(c.attend(q, _i32(pages), _i32([length]), **dev))
            near = small.attend(q, _i32(short), _i32([length]), **dev)
            assert np.array_equal(got, _np(near))
            if m == 1:                                      # (the oracle goes through the whole list)
                want, _, size = otok.attend_formed(o, _np(q), short, [length], [m], 1 / math.sqrt(D), **kw)
                assert np.all(np.abs(got - want) <= 1.3e-3 * size + 2.0 ** -8 * np.abs(want))


def test_traces_of_formed_calls_are_refused(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    from blast3r_amd import kv_cache, kv_pool
    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32)  # noqa: E731
    c, pool = kv_cache.KVCache(2, 1, 64, device='cpu'), kv_pool.BlockPool(2, device='cpu')
    q, pages, lens = torch.zeros(1, 1, 64, dtype=torch.bfloat16), i32([[0, 1]]), i32([5])
    for f, args in ((lambda t: c.attend(t, pages, lens, cap=5.0), q), (lambda t: c.copy(t, lens), lens), (lambda t: pool.grow(pages, t, 1)[0], lens),
                    (lambda t: pool.trim(pages, first=t), lens), (lambda t: pool.fork(pages, lens, t, t), lens), (lambda t: pool.count(t), pages),
                    (lambda t: pool.compact(t)[0], pages)):
        with pytest.raises(RuntimeError, match='trace'):
            torch.jit.trace(f, (args,), check_trace=False)
        with pytest.raises(RuntimeError, match='trace'):
            make_fx(f)(args)


@pytest.mark.gpu
def test_formed_steps_in_a_graph_and_on_a_side_stream():
    """A step of samples that share a prompt, captured once and replayed with other inputs, lengths, masks and slopes, with
    eager work between the replays; the same on another stream."""
    c, _ = _cache(60, 2, 64, 'fp8')
    S = 6
    c._lib = Planned(20, 2, 2)
    pages = torch.cat((_i32([list(range(20))] * S), _i32(20 + np.arange(36).reshape(6, 6))), 1)
    q = torch.zeros((S, 8, 64), dtype=torch.bfloat16, device=DEV)
    lens, prefix, since = _i32([1280] * S), _i32([0] * S), _i32([0] * S)
    slopes = torch.zeros(8, device=DEV)

    def step():
        return c.attend(q, pages, lens, shared=20, cap=30.0, slopes=slopes, prefix=prefix, since=since)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    gen = torch.Generator(device=DEV).manual_seed(1)
    print('formed graph', flush=True)
    for t in range(12):
        q.copy_(torch.randn(q.shape, device=DEV, generator=gen) * 3)
        lens.copy_(torch.randint(1, 1280 + 384, (S,), device=DEV, generator=gen))
        prefix.copy_(torch.randint(0, 200, (S,), device=DEV, generator=gen))
        since.copy_(torch.randint(0, 1500, (S,), device=DEV, generator=gen))
        slopes.copy_(torch.rand(8, device=DEV, generator=gen) * 0.1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and torch.equal(y, other), t


@pytest.mark.gpu
@pytest.mark.parametrize('n', [1, 200])
def test_windows_wider_than_64_bits_hold(n):
    """The widest window there is, with rows whose positions are negative among others: as without one."""
    c, _ = _cache(12, 2, 64, 'int8')
    q = torch.randn((2 * n, 4, 64), device=DEV).bfloat16()
    pages, lens = _i32(np.arange(12).reshape(2, 6)), _i32([380, n // 2])
    print(f'widest window {n}', flush=True)
    for causal in (True, False):
        for kw in (dict(cap=9.0), dict(slopes=torch.rand(4, device=DEV)), dict(prefix=_i32([70, 5]))):
            want = c.attend(q, pages, lens, causal=causal, **kw)
            assert torch.equal(c.attend(q, pages, lens, causal=causal, window=(1 << 63) - 1, **kw), want)


# ---------------------------------------------------------------------------------- plans of large calls (CPU)

def test_plans_are_not_refused_where_one_part_is_not():
    """Whatever is planned for a call can be launched if the call can be without a plan; and its sums have room."""
    if torch.cuda.is_available():
        pytest.skip('would launch on addresses that are none')
    from blast3r_amd import _lib
    L, p = _lib.lib(), 4096
    rng = np.random.default_rng(0)
    base = dict(n_blocks=2, bits=0, dtype=2, scale=1.0, n_splits=1, k=p, v=p, scales=p, pages=p, lengths=p, q=p, o=p, workspace=p,
                workspace_bytes=(1 << 63) - 1)
    some = [dict(n_seqs=180, n_rows=3378240, max_rows=18768, heads=8, q_heads=64, dim=128, n_pages=20, shared=14, since=p),
            dict(n_seqs=65536, n_rows=65536, max_rows=1, heads=64, q_heads=64, dim=64, n_pages=64),
            dict(n_seqs=40000, n_rows=40000 * 32, max_rows=32, heads=64, q_heads=64, dim=256, n_pages=64),
            dict(n_seqs=1 << 22, n_rows=1 << 22, max_rows=1, heads=1, q_heads=1, dim=64, n_pages=64, shared=40),
            dict(n_seqs=1000, n_rows=4000000, max_rows=4000, heads=4, q_heads=32, dim=128, n_pages=300, shared=250)]
    log = lambda lo, hi: int(2.0 ** rng.uniform(lo, hi))  # noqa: E731
    while len(some) < 4000:
        heads, rows, seqs = log(0, 7), log(0, 15), log(0, 22)
        c = dict(n_seqs=seqs, n_rows=seqs * rows, max_rows=rows, heads=heads, q_heads=heads * log(0, 4), dim=int(rng.choice([32, 64, 96, 128, 256])), n_pages=log(0, 14))
        if c['n_rows'] >= 1 << 31:
            continue
        c['shared'] = int(rng.integers(0, c['n_pages'] + 1)) if rng.random() < 0.5 else 0
        c.update(since=p if rng.random() < 0.3 else None, prefix=p if rng.random() < 0.3 else None, window=log(0, 20) if rng.random() < 0.3 else 0,
                 causal=int(rng.integers(0, 2)), offsets=p if rng.random() < 0.5 else None)
        some.append(c)
    planned = 0
    for c in some:
        c = {**base, **c, 'rows_per_seq': 0 if c.get('offsets') else c['max_rows']}
        plain = _lib.BaKvScoredArgs(**{**c, 'shared': 0})
        assert L.ba_kv_attend_scored(ctypes.byref(plain), None) != 0
        if b'too many' in L.ba_last_error():
            continue
        a = _lib.BaKvScoredArgs(**c)
        L.ba_kv_scored_plan(a)
        n = a.n_splits + a.shared_parts
        planned += n > 1
        assert L.ba_kv_attend_scored(ctypes.byref(a), None) != 0 and b'too many' not in L.ba_last_error(), (c, L.ba_last_error())
        assert L.ba_kv_attend_workspace_bytes(a.n_rows, a.q_heads, a.dim, n) <= 8 << 30, c
    assert planned > 300


def test_parts_of_plain_calls_are_not_refused_where_one_is_not():
    """The same of plain attention: two parts of few rows were one workgroup, or as many rows to be joined, too many."""
    if torch.cuda.is_available():
        pytest.skip('would launch on addresses that are none')
    from blast3r_amd import _lib
    L, p = _lib.lib(), 4096
    rng = np.random.default_rng(1)
    log = lambda lo, hi: int(2.0 ** rng.uniform(lo, hi))  # noqa: E731
    some = [(65536, 64, 64, 64, 1, 64), (40000, 64, 64, 256, 32, 64), (1 << 22, 1, 1, 64, 1, 64), ((1 << 22) - 1, 1, 1, 64, 1, 64), (1 << 20, 1, 16, 32, 2, 9000)]
    some += [(log(8, 22), h, h * log(0, 4), int(rng.choice([32, 64, 96, 128, 256])), log(0, 10), log(0, 14)) for h in (log(0, 7) for _ in range(3000))]
    two = 0
    for seqs, heads, q_heads, dim, rows, pages in some:
        if seqs * rows >= 1 << 31:
            continue
        a = _lib.BaKvAttendArgs(n_blocks=2, bits=0, dtype=2, scale=1.0, n_splits=1, k=p, v=p, scales=p, pages=p, lengths=p, q=p, o=p, n_seqs=seqs, heads=heads,
                                q_heads=q_heads, dim=dim, n_rows=seqs * rows, rows_per_seq=rows, max_rows=rows, n_pages=pages, workspace=p, workspace_bytes=(1 << 63) - 1)
        assert L.ba_kv_attend(ctypes.byref(a), None) != 0
        if b'too many' in L.ba_last_error():
            continue
        a.n_splits = L.ba_kv_attend_splits(seqs, heads, q_heads, dim, rows, pages)
        two += a.n_splits > 1
        assert L.ba_kv_attend(ctypes.byref(a), None) != 0 and b'too many' not in L.ba_last_error(), (seqs, heads, q_heads, dim, rows, pages, L.ba_last_error())
    assert two > 300
    for bad in (((1 << 31) - 1, 65536, 65536, 256, (1 << 31) - 1, 1 << 24), (1 << 25, 65536, 65536, 64, (1 << 31) - 1, 9), (4, 4, 4, 0, 1, 9)):
        assert L.ba_kv_attend_splits(*bad) == 1


# ---------------------------------------------------------------------------------- windows wider than any list

WIDE = (1 << 40, (1 << 62) + 1, (1 << 63) - 1, 1 << 63, (1 << 64) + 3, 10 ** 30)


def test_wide_windows_are_not_cut_to_their_low_bits(host):
    from blast3r_amd.kv_cache import KVCache
    c = KVCache(4, 2, 64, device='cpu')
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q, pages, lens = torch.zeros(4, 4, 64, dtype=torch.bfloat16), i32([[0, 1], [2, 3]]), i32([5, 6])
    for window in WIDE:
        for kw in (dict(), dict(cap=5.0)):
            c.attend(q, pages, lens, window=window, **kw)
            assert host[-1].window >= 1 << 40


@pytest.mark.gpu
@pytest.mark.parametrize('n', [3, 20, 90, 300])
def test_windows_wider_than_any_list_are_none(n):
    """Of rows before the first token too, whose positions are below 0; through the C entry point as well."""
    from blast3r_amd import _lib
    c, o = _cache(12, 2, 64, 'int8')
    q = torch.randn((2 * n, 4, 64), device=DEV).bfloat16()
    pages, lens = _i32(np.arange(12).reshape(2, 6)), _i32([300, n - 2])
    print(f'wide windows {n}', flush=True)
    real = _lib.launch
    for kw in (dict(), dict(causal=False), dict(cap=9.0)):
        want = c.attend(q, pages, lens, return_lse=True, **kw)
        assert not want[0][n:n + 2].any() or kw.get('causal') is False
        for window in WIDE:
            for x, y in zip(c.attend(q, pages, lens, window=window, return_lse=True, **kw), want):
                assert torch.equal(x, y), (kw, window)
        from blast3r_amd import kv_cache
        for window in ((1 << 63) - 1, (1 << 63) - n):
            def put(call, args, device):
                args.window = window
                real(call, args, device)
            kv_cache.launch = put
            try:
                got = c.attend(q, pages, lens, window=1 << 40, return_lse=True, **kw)
            finally:
                kv_cache.launch = real
            for x, y in zip(got, want):
                assert torch.equal(x, y), (kw, window)


def test_plans_of_rows_with_a_first_token_of_their_own():
    """What a row's first token is, the host does not know: a few rows over a long list are planned as without, shared blocks
    are weighed alike, and a prompt packed with documents is taken whole, also in a table that is wider."""
    from blast3r_amd import _lib
    L, p = _lib.lib(), 4096

    def plan(**kw):
        a = _lib.BaKvScoredArgs(**{**dict(n_blocks=2, bits=1, dtype=2, scale=1.0, n_splits=1, heads=8, q_heads=32, dim=128, causal=1), **kw})
        L.ba_kv_scored_plan(a)
        return a.n_splits, a.tile, a.shared, a.shared_parts, a.shared_tile

    for seqs, rows, pages in ((1, 1, 1024), (1, 16, 1024), (1, 64, 1024), (1, 512, 1024), (4, 100, 300), (1, 1024, 256), (32, 16, 64)):
        kw = dict(n_seqs=seqs, n_rows=seqs * rows, max_rows=rows, rows_per_seq=rows, n_pages=pages)
        for shared in (0, pages // 4, pages - 3):
            assert plan(since=p, shared=shared, **kw) == plan(shared=shared, **kw)
    for seqs, rows, pages, shared in ((16, 768, 252, 240), (64, 768, 252, 240), (64, 2048, 288, 256)):
        kw = dict(n_seqs=seqs, n_rows=seqs * rows, max_rows=rows, rows_per_seq=rows, n_pages=pages, shared=shared)
        assert plan(since=p, **kw)[2:] == plan(**kw)[2:]
    for pages in (128, 2048):
        assert plan(since=p, n_seqs=1, n_rows=8192, max_rows=8192, rows_per_seq=8192, n_pages=pages) == (1, 128, 0, 0, 0)
