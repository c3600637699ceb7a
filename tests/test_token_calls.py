"""What the token operators' Python side owes to autograd, to tracing and to tensors that change hands (CPU: launches are
recorded instead of made), and calls of tests/test_tokens.py's operators that it leaves out (GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import tokens as otok
from test_tokens import HALF_STEP, _cache, _check, _np, _pages

DEV = 'cuda:0'


@pytest.fixture
def host(monkeypatch):
    """Rotary and KVCache over host tensors; the arguments of each launch are kept in the order of the calls."""
    from blast3r_amd import kv_cache, rotary
    calls = []

    def record(call, args, device):
        calls.append(type(args).from_buffer_copy(args))

    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    for m in (kv_cache, rotary):
        monkeypatch.setattr(m, 'launch', record)
    return calls


def _i32(x, device='cpu'):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


# ---------------------------------------------------------------------------------- tensors written to

def test_tensors_written_to_count_as_changed(host):
    """Each tensor that a call writes to gets a new version, so that a backward that saved it raises."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    rot, pos = Rotary(64, device='cpu'), _i32([0, 1, 2])
    w = torch.ones(3, 2, 64, requires_grad=True)
    x, k = torch.randn(3, 2, 64), torch.randn(3, 1, 64)
    y = (w * x).sum()                                       # saves x
    with torch.no_grad():
        assert rot(pos, x, out=x) is x
    assert x._version == 1
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    rot(pos, x, k, out=(x, k))
    assert x._version == 2 and k._version == 1
    rot(pos, x, k)
    assert x._version == 2 and k._version == 1              # only read
    c = KVCache(2, 1, 64, device='cpu')
    q, pages, lens = torch.zeros(1, 2, 64, dtype=torch.bfloat16), _i32([[0, 1]]), _i32([5])
    held = (c.k, c.v, c.scales)
    before = [t._version for t in held]
    rows = torch.zeros(1, 1, 64)
    c.append(rows, rows, pages, lens)
    assert [t._version for t in held] == [v + 1 for v in before] and rows._version == 0
    out = torch.zeros_like(q)
    c.attend(q, pages, lens, out=out)
    c.read(pages, lens, None, 1)
    assert out._version == 1 and q._version == 0 and [t._version for t in held] == [v + 1 for v in before]
    with torch.inference_mode():                            # no versions there
        z = torch.zeros(3, 2, 64)
        rot(pos, z, out=z)
    with torch.no_grad():
        rot(pos, z, out=z)


def test_outputs_that_require_a_gradient_are_refused(host):
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    rot, pos, x = Rotary(64, device='cpu'), _i32([0, 1, 2]), torch.randn(3, 2, 64)
    leaf = torch.zeros(3, 2, 64, requires_grad=True)
    with pytest.raises(ValueError, match='gradient'):
        rot(pos, x, out=leaf)
    with pytest.raises(ValueError, match='gradient'):
        rot(pos, x, x, out=(torch.zeros_like(x), leaf))
    c = KVCache(2, 1, 64, device='cpu')
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    out = torch.zeros_like(q).requires_grad_()
    with pytest.raises(RuntimeError, match='gradient'):
        c.attend(q, _i32([[0, 1]]), _i32([5]), out=out)
    assert not host
    with torch.no_grad():                                   # as torch's own operators take them
        rot(pos, x, out=leaf)
        c.attend(q, _i32([[0, 1]]), _i32([5]), out=out)
    assert len(host) == 2 and leaf._version == 1 and out._version == 1


def test_outputs_that_overlap_are_refused(host):
    """Rows are read and written in no order, so an output may be its own tensor as it stands, and otherwise neither another
    call's operand at another place nor one place under several rows."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    rot, pos = Rotary(64, device='cpu'), _i32([0, 1, 2])
    qkv = torch.zeros(3, 6, 64)
    q, k = qkv[:, :2], qkv[:, 2:4]
    other = torch.zeros(3, 2, 64).transpose(0, 1).reshape(-1).as_strided((3, 2, 64), (64, 192, 1))
    square = torch.zeros(3, 3, 64)
    for xs, out in (((q, k), (k, q)), ((q, q), (q, q)), ((q, k), (other, other)), ((q,), (q[:1].expand(3, 2, 64),)),
                    ((q,), (other[:, :1].expand(3, 2, 64),)), ((square,), (square.transpose(0, 1),)), ((q, k), (k, torch.zeros_like(k)))):
        with pytest.raises(ValueError, match='out'):
            rot(pos, *xs, out=out)
    c = KVCache(2, 1, 64, device='cpu')
    x = torch.zeros(3, 3, 64, dtype=torch.bfloat16)
    for out in (x.transpose(0, 1), x[:1].expand(3, 3, 64), x[:, :1].expand(3, 3, 64)):
        with pytest.raises(ValueError, match='out'):
            c.attend(x, _i32([[0, 1]]), _i32([5]), out=out)
    assert not host
    rot(pos, q, k, out=(q, k))                              # in place, in one buffer
    rot(pos, q, k, out=(other, qkv[:, 4:]))
    rot(pos[:1], q[:1], out=q[:1].as_strided((1, 2, 64), (7, 64, 1)))       # a stride that nothing uses
    c.attend(x, _i32([[0, 1]]), _i32([5]), out=x)
    c.attend(x, _i32([[0, 1]]), _i32([5]), out=torch.empty_like(x).transpose(0, 1))
    assert len(host) == 5


# ---------------------------------------------------------------------------------- forward mode

def test_forward_mode_tangents_go_through_rotary(host, monkeypatch):
    """The map is linear: a tangent is rotated as its tensor is, and one that is not there counts as zero."""
    from torch.autograd import forward_ad

    from blast3r_amd import rotary
    from blast3r_amd.rotary import Rotary

    def doubles(call, args, device):                        # stands for the rotation: y = 2 x, or x / 2 for the inverse
        for x, y, heads in ((args.x0, args.y0, args.heads0), (args.x1, args.y1, args.heads1))[:args.n_x]:
            src, dst = ((ctypes.c_float * (args.T * heads * args.dim)).from_address(p) for p in (x, y))
            dst[:] = [v * (0.5 if args.inverse else 2.0) for v in src]

    monkeypatch.setattr(rotary, 'launch', doubles)
    rot, pos = Rotary(64, device='cpu'), _i32([0, 1, 2])
    x, t, k = torch.randn(3, 2, 64), torch.randn(3, 2, 64), torch.randn(3, 1, 64)
    for inverse in (False, True):
        f = 0.5 if inverse else 2.0
        for mode in (torch.no_grad, torch.enable_grad):
            with forward_ad.dual_level(), mode():
                dual = forward_ad.make_dual(x, t)
                y = forward_ad.unpack_dual(rot(pos, dual, inverse=inverse))
                assert torch.equal(y.primal, f * x) and torch.equal(y.tangent, f * t)
                for a, b, ta, tb in ((dual, k, f * t, 0 * k), (k, dual, 0 * k, f * t)):
                    a, b = (forward_ad.unpack_dual(r).tangent for r in rot(pos, a, b, inverse=inverse))
                    assert torch.equal(a, ta) and torch.equal(b, tb)
                with pytest.raises(ValueError, match='out'):
                    rot(pos, dual, out=torch.zeros_like(x))
                with pytest.raises(ValueError, match='out'):
                    rot(pos, x, out=dual)
                assert forward_ad.unpack_dual(rot(pos, x)).tangent is None
    with forward_ad.dual_level():                           # reverse over forward
        w = k.clone().requires_grad_()
        y = forward_ad.unpack_dual(rot(pos, forward_ad.make_dual(w, w * 3))).tangent
        assert torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.full_like(w, 3.0 * 0.5))    # twice there, half of it back


def test_cache_refuses_forward_mode_tangents(host):
    from torch.autograd import forward_ad

    from blast3r_amd.kv_cache import KVCache
    c = KVCache(2, 1, 64, device='cpu')
    q, pages, lens = torch.zeros(1, 1, 64, dtype=torch.bfloat16), _i32([[0, 1]]), _i32([5])
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: c.attend(dual, pages, lens), lambda: c.attend(q, pages, lens, out=dual),
                     lambda: c.append(dual, q, pages, lens), lambda: c.append(q, dual, pages, lens)):
            with pytest.raises(RuntimeError, match='tangent'):
                call()
        assert not host
        c.append(q, q, pages, lens)
        c.attend(q, pages, lens)
        assert len(host) == 2


def test_factors_that_require_a_gradient_are_refused(host):
    """A wrapped cache's factors are fp32 tensors of the caller's: a gradient or tangent of them would be lost."""
    from torch.autograd import forward_ad

    from blast3r_amd.kv_cache import KVCache
    c = KVCache(2, 1, 64, device='cpu')
    w = KVCache.wrap(c.k, c.v, torch.ones(2, 1, 2, requires_grad=True))
    q, pages, lens = torch.zeros(1, 1, 64, dtype=torch.bfloat16), _i32([[0, 1]]), _i32([5])
    calls = [lambda w: w.attend(q, pages, lens), lambda w: w.read(pages, lens, None, 1), lambda w: w.append(q, q, pages, lens)]
    for call in calls:
        with pytest.raises(RuntimeError, match='gradient'):
            call(w)
    assert not host
    with torch.no_grad():
        for call in calls:
            call(w)
        assert len(host) == 3
        with forward_ad.dual_level():
            d = KVCache.wrap(c.k, c.v, forward_ad.make_dual(c.scales, torch.ones_like(c.scales)))
            for call in calls:
                with pytest.raises(RuntimeError, match='tangent'):
                    call(d)
    assert len(host) == 3


# ---------------------------------------------------------------------------------- tensors that change hands

def _calls(c, launched, blocks, heads, dim):
    """One call of each kind, all of which have to get the cache's present tensors."""
    q, rows = torch.zeros(1, heads, dim, dtype=torch.bfloat16), torch.zeros(1, heads, dim)
    pages, lens = _i32([[0]]), _i32([5])
    c.append(rows, rows, pages, lens)
    c.read(pages, lens, None, 1)
    c.attend(q, pages, lens)
    for a in launched[-3:]:
        assert (a.k, a.v, a.scales) == (c.k.data_ptr(), c.v.data_ptr(), c.scales.data_ptr())
        assert (a.n_blocks, a.heads, a.dim) == (blocks, heads, dim) == (c.n_blocks, c.heads, c.head_dim)


def test_cache_follows_tensors_put_in_place_of_its_own(host):
    from blast3r_amd.kv_cache import KVCache
    c = KVCache(2, 1, 64, device='cpu')
    _calls(c, host, 2, 1, 64)
    fp8 = torch.float8_e4m3fn
    more = torch.zeros(3, 1, 64, 64, dtype=torch.uint8)
    n = len(host)
    c.k = torch.cat((c.k.view(torch.uint8), more)).view(fp8)               # a cache that grows
    with pytest.raises(ValueError, match='v must be'):                      # and is not whole yet
        c.attend(torch.zeros(1, 1, 64, dtype=torch.bfloat16), _i32([[0]]), _i32([5]))
    c.v = torch.cat((c.v.view(torch.uint8), more)).view(fp8)
    with pytest.raises(ValueError, match='scales must be'):
        c.read(_i32([[0]]), _i32([5]), None, 1)
    assert len(host) == n
    c.scales = torch.cat((c.scales, torch.ones(3, 1, 2)))
    _calls(c, host, 5, 1, 64)
    for name in ('k', 'v', 'scales'):                                       # other memory behind the same tensors
        t = getattr(c, name)
        t.data = t.data.clone()
    _calls(c, host, 5, 1, 64)
    c.k, c.v, c.scales = torch.zeros(1, 2, 64, 32).char(), torch.zeros(1, 2, 32, 64).char(), torch.ones(1, 2, 2)
    _calls(c, host, 1, 2, 32)
    assert host[-1].bits == 1 and host[-1].scale == pytest.approx(32 ** -0.5) and c.dtype is torch.int8
    for name in ('n_blocks', 'heads', 'head_dim', 'device', 'dtype'):       # what the tensors say
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))


def test_rotary_says_what_it_was_made_with(host):
    """The kernels get what the constructor laid out: assignments that they would not see are refused."""
    from blast3r_amd.rotary import Rotary
    rot, pos, x = Rotary(64, axes=2, device='cpu'), torch.zeros(3, 2, dtype=torch.int32), torch.randn(3, 2, 64)
    for name in ('turns', 'frequencies', 'factor', 'head_dim', 'rotary_dim', 'layout', 'axes', 'device'):
        with pytest.raises(AttributeError):
            setattr(rot, name, getattr(rot, name))
    assert (rot.head_dim, rot.rotary_dim, rot.layout, rot.axes, rot.factor) == (64, 64, 'half', 2, 1.0)
    assert len(rot.frequencies) == 16 and rot.device == rot.turns.device
    rot(pos, x)
    assert host[-1].turns == rot.turns.data_ptr()
    rot.turns.data = rot.turns.data.clone()                 # other memory behind the same tensor
    rot(pos, x)
    assert host[-1].turns == rot.turns.data_ptr()


# ---------------------------------------------------------------------------------- tracing

def test_traces_are_refused(host, monkeypatch):
    """A launch is no operation of torch's: a trace would keep the allocation of its result and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from blast3r_amd import _lib, kv_cache, rotary
    rot, pos, x = rotary.Rotary(64, device='cpu'), _i32([0, 1, 2]), torch.randn(3, 2, 64)
    c = kv_cache.KVCache(2, 1, 64, device='cpu')
    q, pages, lens = torch.zeros(1, 1, 64, dtype=torch.bfloat16), _i32([[0, 1]]), _i32([5])
    for m in (kv_cache, rotary):
        monkeypatch.setattr(m, 'launch', _lib.launch)       # which ends before anything of the GPU's
    for f, args in ((lambda t: rot(pos, t), x), (lambda t: c.attend(t, pages, lens), q), (lambda t: c.append(t, t, pages, lens), q),
                    (lambda t: c.read(pages, t, None, 1), lens)):
        with pytest.raises(RuntimeError, match='trace'):
            torch.jit.trace(f, (args,), check_trace=False)
        with pytest.raises(RuntimeError, match='trace'):
            make_fx(f)(args)


# ---------------------------------------------------------------------------------- addresses and strides (GPU)

@pytest.mark.gpu
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
def test_append_of_fp32_rows_aligned_to_16_bytes_only(dim):
    """Rows whose addresses are 16 bytes past a multiple of 32 are written as aligned ones are."""
    from blast3r_amd.kv_cache import KVCache
    gen = torch.Generator(device=DEV).manual_seed(dim)
    base = torch.randn((2, 150 * 3 * dim + 8), device=DEV, generator=gen)
    k, v = (b[4:-4].view(150, 3, dim)[:, 1:] for b in base)
    assert k.data_ptr() % 32 == v.data_ptr() % 32 == 16
    print(f'append {dim}', flush=True)
    caches = [KVCache(4, 2, dim, torch.int8, device=DEV) for _ in range(2)]
    pages = _i32([[2, 0, 3, 1]], DEV)
    caches[0].append(k, v, pages, _i32([5], DEV))
    caches[1].append(k.contiguous(), v.contiguous(), pages, _i32([5], DEV))
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    assert torch.equal(caches[0].scales, caches[1].scales) and bool(caches[0].k.any()) and bool(caches[0].v.any())


# ---------------------------------------------------------------------------------- limits of the C entry points (CPU)

def _full(cls, **kw):
    """Arguments that pass every check, with addresses that are only compared with each other."""
    p = 4096
    names = {n for n, _ in cls._fields_}
    a = dict(k=p, v=p, scales=p, n_blocks=2, heads=2, dim=64, bits=0, n_seqs=1, pages=p, pages_stride=2, n_pages=2, dtype=2,
             starts=p, lengths=p, offsets=p, n_rows=3, max_rows=3, rk=p, rv=p, q=p, o=p, q_heads=4, scale=1.0, n_splits=1)
    return cls(**{**{n: x for n, x in a.items() if n in names}, **kw})


def _refused(call, args, word):
    from blast3r_amd import _lib
    assert call(ctypes.byref(args), None) != 0 and word in _lib.lib().ba_last_error().decode(), _lib.lib().ba_last_error()


@pytest.mark.parametrize('rows', [1 << 31, (1 << 63) - 62, (1 << 63) - 1])
def test_cache_calls_refuse_bounds_on_rows_past_32_bits(rows):
    """The number of blocks that a sequence may touch is rounded up from max_rows, which must not wrap."""
    from blast3r_amd import _lib
    L = _lib.lib()
    for call in (L.ba_kv_write, L.ba_kv_read):
        _refused(call, _full(_lib.BaKvArgs, max_rows=rows), 'bad sizes')
        _refused(call, _full(_lib.BaKvArgs, max_rows=3, rows_per_seq=rows, offsets=None), 'bad sizes')


def test_attention_checks_its_parts_before_it_launches():
    """Sizes that the join of the parts cannot take are refused before the parts are made, and the room that their sums
    need is not a number that wraps."""
    from blast3r_amd import _lib
    L = _lib.lib()
    most = (1 << 63) - 1
    for kw in (dict(n_rows=1 << 30, q_heads=2), dict(n_rows=(1 << 31) - 1, q_heads=65536, n_splits=65536)):
        _refused(L.ba_kv_attend, _full(_lib.BaKvAttendArgs, **{**dict(n_splits=2, workspace=4096, workspace_bytes=most), **kw}), 'too many')
        _refused(L.ba_kv_attend, _full(_lib.BaKvAttendArgs, **{**dict(n_splits=2, workspace=4096, workspace_bytes=64), **kw}), 'too many')


def test_attention_launches_have_less_than_2_32_threads():
    """2^23 workgroups of 512 threads are one too many."""
    from blast3r_amd import _lib
    a = _full(_lib.BaKvAttendArgs, dim=128, n_seqs=1 << 13, offsets=None, n_rows=1 << 18, rows_per_seq=256, max_rows=256,
              heads=1024, q_heads=1024)
    _refused(_lib.lib().ba_kv_attend, a, 'too many')


# ---------------------------------------------------------------------------------- many sequences without a bound on their rows

def test_ragged_calls_of_many_sequences_are_not_too_large(monkeypatch):
    """A call whose rows fit the chip many times over is no longer refused for the rows that each sequence might have:
    what comes after the checks of its size is the launch, which fails here for want of a GPU."""
    if torch.cuda.is_available():
        pytest.skip('would launch on addresses that are none')
    from blast3r_amd import _lib
    L = _lib.lib()
    for S in (4096, 70000):
        n = 200 * S
        for call, a in ((L.ba_kv_write, _full(_lib.BaKvArgs, n_seqs=S, n_rows=n, max_rows=n, heads=8)),
                        (L.ba_kv_read, _full(_lib.BaKvArgs, n_seqs=S, n_rows=n, max_rows=n, heads=8)),
                        (L.ba_kv_attend, _full(_lib.BaKvAttendArgs, n_seqs=S, n_rows=n, max_rows=n, heads=8, q_heads=32))):
            assert call(ctypes.byref(a), None) != 0
            assert b'too many' not in L.ba_last_error(), (S, L.ba_last_error())
    # what no launch can take, in rows or in sequences
    big = (1 << 31) - 1
    for kw in (dict(n_rows=big, max_rows=big, heads=4096, q_heads=4096), dict(n_seqs=1 << 22, heads=8, q_heads=8)):
        _refused(L.ba_kv_attend, _full(_lib.BaKvAttendArgs, **kw), 'too many')
        kw.pop('q_heads')
        _refused(L.ba_kv_write, _full(_lib.BaKvArgs, **kw), 'too many')


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [torch.float8_e4m3fn, torch.int8])
def test_ragged_calls_of_many_sequences_without_a_bound(bits):
    """3000 sequences: with max_new left out their rows are found by the offsets, and everything is as with a close bound."""
    from blast3r_amd.kv_cache import KVCache
    rng = np.random.default_rng(3)
    S, H, G, D = 3000, 8, 2, 32
    new = rng.integers(0, 41, S)
    new[[0, 1, 700, S - 2]] = 0
    new[[5, S - 1]] = 200
    held = rng.integers(0, 200, S)
    blocks = (held + new + 63) // 64
    pages = np.full((S, int(blocks.max())), -1)
    order, at = rng.permutation(int(blocks.sum())), 0
    for s, b in enumerate(blocks):
        pages[s, :b] = order[at:at + b]
        at += b
    n = int(new.sum())
    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((n, H, D), device=DEV, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn((n, H * G, D), device=DEV, generator=gen).bfloat16()
    pages, held_t, lens, off = _i32(pages, DEV), _i32(held, DEV), _i32(held + new, DEV), _i32(np.concatenate(([0], np.cumsum(new))), DEV)
    caches = [KVCache(int(blocks.sum()), H, D, bits, device=DEV) for _ in range(2)]
    out = []
    for c, most in zip(caches, (200, None)):
        print(f'many sequences {bits} {most}', flush=True)
        c.append(k, v, pages, held_t, offsets=off, max_new=most)
        o, lse = c.attend(q, pages, lens, offsets=off, max_new=most, return_lse=True)
        out.append((c.k.view(torch.uint8), c.v.view(torch.uint8), c.scales, o, lse, *c.read(pages, held_t, off, n, max_count=most)))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(b.any())


# ---------------------------------------------------------------------------------- attention: what test_tokens.py leaves out (GPU)

def _parts(S, heads, q_heads, dim, rows, n_pages):
    from blast3r_amd import _lib
    return _lib.lib().ba_kv_attend_splits(S, heads, q_heads, dim, rows, n_pages)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('tokens', [500, 3000])             # in one part, and in several
@pytest.mark.parametrize('dim,group,n', [(64, 2, 3), (128, 1, 1), (96, 3, 9), (64, 2, 50), (64, 1, 300), (128, 2, 130), (256, 1, 40)])
def test_attend_of_unaligned_queries_and_outputs(dim, group, n, tokens, dtype):
    """Queries and outputs at odd addresses with odd strides, the outputs' heads first: the same numbers as aligned ones, and
    nothing else of the outputs' memory is written."""
    heads, Hq = 2, 2 * group
    c, _ = _cache(60, heads, dim, 'int8', seed=dim)
    pages = _i32(_pages(np.random.default_rng(n), [(tokens + 63) // 64], 60, (tokens + 63) // 64), DEV)
    assert (_parts(1, heads, Hq, dim, n, pages.shape[1]) > 1) == (tokens == 3000)
    lens = _i32([tokens], DEV)
    x = (2 * torch.randn((n, Hq, dim), generator=torch.Generator().manual_seed(n))).to(dtype).to(DEV)
    print(f'attend unaligned {dim} {group} {n} {tokens} {dtype}', flush=True)
    want, want_lse = c.attend(x, pages, lens, return_lse=True)
    row = Hq * (dim + 3) + 4
    q = torch.zeros(n * row + 1, dtype=dtype, device=DEV)[1:].as_strided((n, Hq, dim), (row, dim + 3, 1), 1)
    q.copy_(x)
    head = n * (dim + 1) + 2
    base = torch.full((Hq * head + 1,), 7.0, dtype=dtype, device=DEV)
    out = base.as_strided((n, Hq, dim), (dim + 1, head, 1), 1)
    expect = base.clone()
    expect.as_strided(out.shape, out.stride(), 1).copy_(want)
    got, lse = c.attend(q, pages, lens, out=out, return_lse=True)
    assert got is out and torch.equal(base, expect) and torch.equal(lse, want_lse)
    base.fill_(7.0)
    c.attend(x, pages, lens, out=out)                       # one side at a time
    assert torch.equal(base, expect)
    assert torch.equal(c.attend(q, pages, lens), want)


@pytest.mark.gpu
@pytest.mark.parametrize('n,most', [(10, 7), (40, 20), (150, 40), (150, 130), (600, 300)])
@pytest.mark.parametrize('splits', [1, 2])
def test_attend_leaves_rows_past_the_bound_alone(n, most, splits):
    """Rows past max_rows of their sequence keep their outputs and their lse; the others are as in a call without them."""
    from blast3r_amd import _lib
    L = _lib.lib()
    heads, D, counts, lens = 2, 64, [n, 3], [3000, 1200]
    c, o = _cache(70, heads, D, 'fp8')
    pages = _pages(np.random.default_rng(n), [47, 19], 70, 47)
    q = torch.randn((n + 3, heads, D), generator=torch.Generator().manual_seed(n)).bfloat16().to(DEV)
    y, lse = torch.full_like(q, 7.0), torch.full((n + 3, heads), 5.0, device=DEV)
    p, off, ln = _i32(pages, DEV), _i32([0, n, n + 3], DEV), _i32(lens, DEV)
    size = L.ba_kv_attend_workspace_bytes(n + 3, heads, D, splits)
    work = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=DEV)
    a = _lib.BaKvAttendArgs(k=c.k.data_ptr(), v=c.v.data_ptr(), scales=c.scales.data_ptr(), n_blocks=70, heads=heads, dim=D, bits=0,
                            n_seqs=2, pages=p.data_ptr(), pages_stride=47, n_pages=47, dtype=2, lengths=ln.data_ptr(),
                            offsets=off.data_ptr(), n_rows=n + 3, max_rows=most, q=q.data_ptr(), o=y.data_ptr(), lse=lse.data_ptr(),
                            q_st=heads * D, q_sh=D, o_st=heads * D, o_sh=D, q_heads=heads, causal=1, scale=0.125, n_splits=splits,
                            workspace=work.data_ptr(), workspace_bytes=size)
    print(f'attend bound {n} {most} {splits}', flush=True)
    _lib.check(L.ba_kv_attend(ctypes.byref(a), _lib.stream_ptr(DEV)))
    assert bool((y[most:n] == 7.0).all()) and bool((lse[most:n] == 5.0).all())
    want, want_lse, size = otok.attend(o, _np(q), pages, lens, counts, 0.125)
    done = np.r_[0:most, n:n + 3]
    assert np.all(np.abs(_np(y) - want)[done] <= 1.2e-3 * size[done] + HALF_STEP[q.dtype] * np.abs(want[done]))
    assert np.all(np.abs(_np(lse) - want_lse)[done] <= 6e-4)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('dim,group,n,window', [(32, 1, 70, None), (32, 2, 150, None), (32, 2, 150, 1500), (256, 1, 70, None),
                                                (256, 2, 100, None), (256, 2, 100, 1300), (96, 1, 140, None)])
def test_attend_of_many_rows_in_several_parts(dim, group, n, window, dtype, bits):
    """Shared blocks (more than 32 rows) for the smallest and the largest heads, with the keys cut into parts."""
    tokens = 2300
    assert _parts(1, 1, group, dim, n, 36) > 1
    c, o = _cache(37, 1, dim, bits, seed=n)
    rng = np.random.default_rng(n)
    pages = _pages(rng, [36], 37, 36)
    q = torch.tensor(rng.normal(size=(n, group, dim)) * 2.0, dtype=torch.float32).to(dtype).to(DEV)
    print(f'attend parts {bits} {dtype} {dim} {group} {n} {window}', flush=True)
    _check(c, o, q, pages, [tokens], [n], True, window)
    _check(c, o, q, pages, [tokens], [n], False, window)


# ---------------------------------------------------------------------------------- derivatives, and a cache that grows (GPU)

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_rotary_in_forward_mode(dtype):
    """The tangent is the rotation of the tangent, also of one without contiguous heads, and of the gradient's."""
    from torch.autograd import forward_ad

    from blast3r_amd.rotary import Rotary
    rot = Rotary(64, axes=2, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda *s: torch.randn(s, device=DEV, generator=gen).to(dtype)  # noqa: E731
    pos = torch.randint(0, 99, (5, 2), device=DEV, generator=gen, dtype=torch.int32)
    q, k, t = mk(5, 4, 64), mk(5, 2, 64), mk(5, 64, 4).transpose(1, 2)
    y, z, dy, dt = rot(pos, q), rot(pos, k), rot(pos, t.contiguous()), rot(pos, t.contiguous(), inverse=True)
    for mode in (torch.no_grad, torch.enable_grad):
        with forward_ad.dual_level(), mode():
            a, b = rot(pos, forward_ad.make_dual(q, t), k)
            a, b = forward_ad.unpack_dual(a), forward_ad.unpack_dual(b)
            assert torch.equal(a.primal, y) and torch.equal(b.primal, z) and torch.equal(a.tangent, dy)
            assert b.tangent is None or not b.tangent.any()
    with forward_ad.dual_level():                           # forward over reverse
        w = q.clone().requires_grad_()
        (g,) = torch.autograd.grad(rot(pos, w), w, forward_ad.make_dual(q, t))
        assert torch.equal(forward_ad.unpack_dual(g).tangent, dt)


@pytest.mark.gpu
def test_growing_a_cache_by_assignment():
    from blast3r_amd.kv_cache import KVCache
    heads, D = 2, 64
    gen = torch.Generator(device=DEV).manual_seed(0)
    k, v, q = (torch.randn((200, heads, D), device=DEV, generator=gen).bfloat16() for _ in range(3))
    lens = _i32([200], DEV)
    big = KVCache(8, heads, D, torch.int8, device=DEV)
    big.append(k, v, _i32([[1, 0, 6, 7]], DEV), lens - 200)
    c = KVCache(2, heads, D, torch.int8, device=DEV)
    c.append(k[:100], v[:100], _i32([[1, 0]], DEV), lens - 200)
    for name, fresh in (('k', torch.zeros), ('v', torch.zeros), ('scales', torch.ones)):
        t = getattr(c, name)
        setattr(c, name, torch.cat((t, fresh((6, *t.shape[1:]), dtype=t.dtype, device=DEV))))
    c.append(k[100:], v[100:], _i32([[1, 0, 6, 7]], DEV), lens - 100)
    one, two = (x.read(_i32([[1, 0, 6, 7]], DEV), lens - 200, None, 200, dtype=torch.float32) for x in (c, big))
    # the second block was filled in two calls, and its codes may have been made anew: one step of its factor apart at most
    for a, b, f in zip(one, two, c.scales.unbind(-1)):
        assert torch.equal(a[:64], b[:64]) and torch.equal(a[128:], b[128:])
        assert bool(((a[64:128] - b[64:128]).abs() <= 1.01 * f[0][:, None]).all())
    assert c.n_blocks == 8 and c.attend(q, _i32([[1, 0, 6, 7]], DEV), lens).isfinite().all()


# ---------------------------------------------------------------------------------- factors that grow

def _growing(g, n=64, heads=1, dim=32):
    """n tokens whose largest value is g times that of the one before."""
    x = np.random.default_rng(0).uniform(-1, 1, (n, heads, dim))
    x[:, :, 0] = 1.0
    return np.float32(x * (g ** np.arange(n))[:, None, None])


@pytest.mark.parametrize('g', [1.0, 1.001, 1.0039, 1.01, 1.3, 2.5])
def test_int8_codes_lose_half_a_step_whenever_their_factor_grows(g):
    """The bound that the documents give: after n growths a value is within (n + 1) / 2 steps of the block's factor, and
    slow growth comes near it; e4m3 codes of normal size, whose factors at least double, stay within their 2^-4."""
    x = _growing(g)
    for bits in ('int8', 'fp8'):
        c = otok.Cache(np.zeros((1, 1, 64, 32)), np.zeros((1, 1, 64, 32)), np.ones((1, 1, 2)), bits)
        grown, f, n = np.zeros(64), 0.0, 0
        while n < 64:
            c.append(x[n:n + 1], x[n:n + 1], [[0]], [n], [1])
            before, f = f, c.scales[0, 0, 0]
            if not f <= 2.0 ** 60:                          # past the range of factors: NaN from here on
                assert x[n].max() > (127 if bits == 'int8' else 448) * 2.0 ** 60
                f = before
                break
            grown[:n] += f > before
            n += 1
            k, _, _ = c.sequence([0], n)
        grown, y = grown[:n], np.float64(x[:n])
        err = np.abs(k - y).max((1, 2))
        if bits == 'int8':
            assert np.all(err <= (grown + 1) / 2 * f * (1 + 1e-5))
            if g == 1.0039:
                assert grown[0] == 63 and err[0] > 25 * f
        else:
            normal = np.abs(y) >= 2.0 ** -6 * f
            assert np.all((np.abs(k - y) <= 2.0 ** -4 * np.abs(y))[normal])


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['int8', 'fp8'])
def test_append_of_single_tokens_that_grow(bits):
    """A factor that grows with each of 64 tokens: codes and factors as the oracle's throughout."""
    from blast3r_amd.kv_cache import KVCache
    from test_tokens import BITS, _mirror, _same
    x = _growing(1.0039, heads=2, dim=64)
    c = KVCache(1, 2, 64, BITS[bits], device=DEV)
    o = _mirror(c, bits)
    print(f'growing {bits}', flush=True)
    for t in range(64):
        r = torch.tensor(x[t:t + 1], device=DEV)
        c.append(r, r, _i32([[0]], DEV), _i32([t], DEV))
        o.append(x[t:t + 1], x[t:t + 1], [[0]], [t], [1])
    _same(c, o)
