"""Rotary positions, the 8-bit key/value cache and attention over it: oracle pins and refusals (CPU), parity with the
oracle (GPU).

Bars, derived from the arithmetic:
  * rotary: an angle is right to 2^-24 of a quarter turn and its sine and cosine to a few fp32 roundings, 4e-7 in all;
    the two products and their sum add 2^-23 of their size: |dy| <= 6e-7 (|a| + |b|) factor, and half a step of the
    output's type;
  * cache: codes and factors are equal to the oracle's, which rounds where the definition does;
    read values are the oracle's product rounded once;
  * attention: weights carry an fp16 rounding each in the numerator and in the denominator (2^-11 of p |v| each at most),
    scores an error of D roundings of fp32 of their terms (taken as 2^-24 * 8 sqrt(D) of the largest score, which is
    below 60 in the tests: 6e-5 for D = 256 in the exponent), and the output half a step of its type:
    |do| <= 1.2e-3 sum p |v| + half a step.  lse: its weights' roundings are 2^-12 of l on the average, 2^-11 at most,
    with the error of the scores: 6e-4.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import tokens as otok

DEV = 'cuda:0'
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BITS = {'fp8': torch.float8_e4m3fn, 'int8': torch.int8}


def _np(t):
    return t.detach().to('cpu', torch.float64).numpy()


# ---------------------------------------------------------------------------------- oracle pins (CPU)

def test_oracle_codes_equal_torchs_e4m3():
    x = torch.cat((torch.randn(20000, generator=torch.Generator().manual_seed(0)) * 60, torch.linspace(-0.04, 0.04, 4001)))
    x = x.clamp(-448, 448)
    assert np.array_equal(otok.nearest_code(_np(x), 'fp8'), _np(x.to(torch.float8_e4m3fn).float()))
    every = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[every.isfinite()]
    assert np.array_equal(otok.nearest_code(_np(every), 'fp8'), _np(every))


@pytest.mark.parametrize('amax,f', [(448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (0.0, 2.0 ** -60), (1e-30, 2.0 ** -60),
                                    (448.0 * 2.0 ** 60, 2.0 ** 60)])
def test_oracle_fit_e4m3(amax, f):
    assert otok.fit(amax, 'fp8') == f
    assert math.isnan(otok.fit(math.inf, 'fp8')) and math.isnan(otok.fit(1e30, 'fp8'))
    assert otok.fit(127.0, 'int8') == 1.0 and math.isnan(otok.fit(math.nan, 'int8'))


def test_oracle_attention_known_answers():
    """One key: its value; two equal keys: their mean; a key that no row sees, a row without keys."""
    k, v = np.zeros((1, 1, 64, 32)), np.zeros((1, 1, 64, 32))
    v[0, 0, 0], v[0, 0, 1], v[0, 0, 2] = 2.0, 4.0, np.nan
    c = otok.Cache(k, v, np.ones((1, 1, 2)), 'int8')
    q = np.ones((3, 1, 32))
    o, lse, _ = otok.attend(c, q[:2], [[0]], [2], [2], 0.3)
    assert np.all(o[0] == 2.0) and np.all(o[1] == 3.0) and np.allclose(lse[:, 0], [0.0, math.log(2.0)])
    o, lse, _ = otok.attend(c, q, [[0]], [2], [3], 0.3)                    # three rows, two tokens
    assert np.all(o[0] == 0.0) and lse[0, 0] == -math.inf and np.all(o[2] == 3.0)
    o, _, _ = otok.attend(c, q[:1], [[0]], [2], [1], 0.3, window=1)
    assert np.all(o == 4.0)


def test_frequencies():
    from blast3r_amd.rotary import rotary_frequencies
    f, m = rotary_frequencies(8)
    assert m == 1.0 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14)
    assert np.allclose(rotary_frequencies(8, scaling=dict(kind='linear', factor=4))[0], np.array(f) / 4, rtol=1e-14)
    b, _ = rotary_frequencies(8, scaling=dict(kind='base', factor=4))
    assert b[0] == 1.0 and abs(b[3] * 4 / f[3] - 1) < 1e-12               # the slowest pair 4 times slower
    r, m = rotary_frequencies(64, scaling=dict(kind='ramp', factor=8, length=4096, fast=32, slow=1))
    g, _ = rotary_frequencies(64)
    turns = 4096 * np.array(g) / (2 * math.pi)
    ratio = np.array(r) / np.array(g)
    assert np.all(ratio[turns >= 32] == 1.0) and np.allclose(ratio[turns <= 1], 1 / 8) and abs(m - (0.1 * math.log(8) + 1)) < 1e-15
    for bad in (dict(kind='cubic', factor=2), dict(kind='linear', factor=0.5), dict(kind='ramp', factor=2, length=9, fast=1, slow=1)):
        with pytest.raises(ValueError):
            rotary_frequencies(8, scaling=bad)
    for n in (0, 3):
        with pytest.raises(ValueError):
            rotary_frequencies(n)


# ---------------------------------------------------------------------------------- refusals (CPU)

def test_entry_points_refuse_bad_arguments_without_a_gpu():
    """Every check of the C entry points comes before any device call."""
    from blast3r_amd import _lib
    L = _lib.lib()

    def refused(call, a, word, **fields):
        keep = {n: getattr(a, n) for n in fields}
        for n, x in fields.items():
            setattr(a, n, x)
        assert call(ctypes.byref(a), None) != 0, (fields, word)
        assert word in L.ba_last_error().decode(), (L.ba_last_error(), word)
        for n, x in keep.items():
            setattr(a, n, x)

    r = _lib.BaRotaryArgs(n_x=1, dtype=2, B=1, T=4, dim=64, part=64, axes=2)
    r.heads0 = 2
    assert L.ba_rotary(None, None) != 0
    refused(L.ba_rotary, r, 'null pointer')
    refused(L.ba_rotary, r, 'one or two', n_x=3)
    refused(L.ba_rotary, r, 'whole pairs', part=66)
    refused(L.ba_rotary, r, 'whole pairs', part=62)
    refused(L.ba_rotary, r, 'head size', dim=1)
    refused(L.ba_rotary, r, 'interleaved', dim=65, interleaved=1)
    refused(L.ba_rotary, r, 'dtype', dtype=3)
    refused(L.ba_rotary, r, 'bad sizes', T=-1)
    refused(L.ba_rotary, r, 'bad sizes', T=1 << 41)
    assert L.ba_rotary(ctypes.byref(_lib.BaRotaryArgs(n_x=1, B=1, T=0, dim=64, part=64, axes=2, heads0=1)), None) == 0

    kv = dict(n_blocks=2, heads=2, dim=64, bits=0, n_seqs=1, n_pages=2, pages_stride=2, dtype=2, n_rows=3, rows_per_seq=3, max_rows=3)
    for call, a in ((L.ba_kv_write, _lib.BaKvArgs(**kv)), (L.ba_kv_read, _lib.BaKvArgs(**kv)),
                    (L.ba_kv_attend, _lib.BaKvAttendArgs(q_heads=4, scale=1.0, n_splits=1, **kv))):
        assert call(None, None) != 0
        refused(call, a, 'null pointer')
        for d in (0, 48, 160, 512):
            refused(call, a, 'head size', dim=d)
        refused(call, a, 'bits', bits=2)
        refused(call, a, 'bad sizes', n_seqs=-1)
        refused(call, a, 'bad sizes', n_rows=-1)
        refused(call, a, 'bad sizes', n_rows=1 << 31)
        refused(call, a, 'fp16 or bf16', dtype=3)
    a = _lib.BaKvAttendArgs(q_heads=4, scale=1.0, n_splits=1, **kv)
    refused(L.ba_kv_attend, a, 'multiple', q_heads=3)
    refused(L.ba_kv_attend, a, 'fp16 or bf16', dtype=0)
    refused(L.ba_kv_attend, a, 'scale', scale=0.0)
    refused(L.ba_kv_attend, a, 'scale', scale=math.nan)
    refused(L.ba_kv_attend, a, 'n_splits', n_splits=0)
    refused(L.ba_kv_attend, a, 'bad sizes', window=-1)
    refused(L.ba_kv_attend, a, 'without sequences', rows_per_seq=0)
    p = 4096                                                # addresses that are only compared with each other
    full = dict(k=p, v=p, scales=p, pages=p, lengths=p, q=p, o=p)
    refused(L.ba_kv_attend, a, 'aligned', **dict(full, k=p + 8))
    refused(L.ba_kv_attend, a, 'null pointer', **dict(full, n_splits=2))
    refused(L.ba_kv_attend, a, 'too small', **dict(full, n_splits=2, workspace=p, workspace_bytes=64))
    refused(L.ba_kv_attend, a, 'too many', **dict(full, n_seqs=1 << 23))
    assert L.ba_kv_attend_workspace_bytes(3, 4, 64, 2) == 3 * 4 * 2 * 66 * 4 and L.ba_kv_attend_workspace_bytes(3, 4, 64, 1) == 0


def test_python_refuses_host_tensors():
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    with pytest.raises(RuntimeError):
        KVCache(2, 1, 64, device='cpu')
    with pytest.raises(RuntimeError):
        Rotary(64, device='cpu')
    for kw in (dict(dtype=torch.float16), dict(head_dim=48), dict(heads=0)):
        with pytest.raises(ValueError):
            KVCache(**{**dict(n_blocks=1, heads=1, head_dim=64, device='cpu'), **kw})
    for kw in (dict(rotary_dim=66), dict(rotary_dim=30, axes=4), dict(axes=3), dict(layout='thirds'), dict(axes=0)):
        with pytest.raises(ValueError):
            Rotary(64, device='cpu', **kw)


@pytest.mark.gpu
def test_python_refuses_bad_arguments():
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    c = KVCache(4, 2, 64, device=DEV)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device=DEV)  # noqa: E731
    pages, lens = z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32)
    for args, kw in (((z(4, 2, 32), z(4, 2, 32), pages, lens), {}), ((z(4, 2, 64), z(4, 2, 64).half(), pages, lens), {}),
                     ((z(3, 2, 64), z(3, 2, 64), pages, lens), {}), ((z(4, 2, 64), z(4, 2, 64), pages.long(), lens), {}),
                     ((z(4, 2, 64), z(4, 2, 64), pages, lens[:1]), {}), ((z(4, 2, 64), z(4, 2, 64), pages, lens.cpu()), {}),
                     ((z(4, 2, 64), z(4, 2, 64), pages, lens), dict(offsets=lens)),
                     ((z(4, 2, 128)[..., ::2], z(4, 2, 64), pages, lens), {})):
        with pytest.raises(ValueError):
            c.append(*args, **kw)
    for q, kw in ((z(2, 3, 64), {}), (z(2, 2, 64).float(), {}), (z(2, 2, 64), dict(window=0)), (z(2, 2, 64), dict(scale=-1.0)),
                  (z(2, 2, 64), dict(out=z(2, 2, 64).half())), (z(3, 2, 64), {}), (z(2, 2, 32), {})):
        with pytest.raises(ValueError):
            c.attend(q, pages, lens, **kw)
    with pytest.raises(ValueError):
        c.read(pages, lens, None, 3)
    with pytest.raises(ValueError):
        KVCache.wrap(c.k, c.v.transpose(2, 3), c.scales)
    rot = Rotary(64, axes=2, device=DEV)
    pos = z(4, 2, dtype=torch.int32)
    for p, xs, kw in ((pos, (z(4, 2, 32),), {}), (pos[:, :1], (z(4, 2, 64),), {}), (pos[:3], (z(4, 2, 64),), {}),
                      (pos.float(), (z(4, 2, 64),), {}), (pos, (z(4, 2, 64), z(4, 2, 64).half()), {}),
                      (pos, (z(4, 2, 64),) * 3, {}), (pos, (z(4, 64, 2).transpose(1, 2),), {}),
                      (pos, (z(4, 2, 64),), dict(out=z(4, 1, 64))), (pos, (z(4, 2, 64).requires_grad_(),), dict(out=z(4, 2, 64)))):
        with pytest.raises(ValueError):
            rot(p, *xs, **kw)


# ---------------------------------------------------------------------------------- rotary (GPU)

def _rotary_bar(x, y, part, layout, axes, factor, dtype):
    """|a| + |b| of each element's pair, and half a step of the result."""
    n = part // axes
    size = np.abs(x).copy()
    for ax in range(axes):
        s = size[..., ax * n:(ax + 1) * n]
        a = np.abs(x[..., ax * n:(ax + 1) * n])
        if layout == 'half':
            both = a[..., :n // 2] + a[..., n // 2:]
            s[...] = np.concatenate((both, both), -1)
        else:
            both = a[..., 0::2] + a[..., 1::2]
            s[...] = np.repeat(both, 2, -1)
    return 6e-7 * factor * size + HALF_STEP[dtype] * np.abs(y) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


ROTARY = [
    # tokens, heads, dim, part, layout, axes, dtype
    (1, (4, 1), 128, 128, 'half', 1, torch.bfloat16),
    (37, (16, 16), 64, 64, 'half', 2, torch.bfloat16),
    (300, (5, 2), 96, 48, 'interleaved', 1, torch.float16),
    (129, (3, 3), 96, 96, 'half', 3, torch.float32),
    (65, (2, 1), 80, 20, 'half', 1, torch.bfloat16),               # sections that are no whole vectors
    (50, (2, 1), 82, 42, 'interleaved', 3, torch.float16),
    (33, (1, 1), 7, 6, 'half', 1, torch.float32),
    (2000, (24, 8), 256, 128, 'interleaved', 2, torch.bfloat16),   # several heads to a thread
]


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,heads,dim,part,layout,axes,dtype', ROTARY)
def test_rotary_against_oracle(tokens, heads, dim, part, layout, axes, dtype):
    from blast3r_amd.rotary import Rotary
    rng = np.random.default_rng(tokens)
    scaling = dict(kind='ramp', factor=8, length=8192) if part >= 48 else None
    rot = Rotary(dim, rotary_dim=part, layout=layout, axes=axes, scaling=scaling, device=DEV)
    pos = rng.integers(-1000, 1 << 21, (tokens, axes))
    pos[0] = 0
    pos[-1] = 2 ** 31 - 1
    p = torch.tensor(pos if axes > 1 else pos[:, 0], dtype=torch.int32, device=DEV)
    fused = torch.randn((tokens, sum(heads) + 1, dim), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    q, k = fused[:, :heads[0]], fused[:, heads[0]:heads[0] + heads[1]]
    print(f'rotary {tokens} {heads} {dim} {part} {layout} {axes} {dtype}', flush=True)
    for inverse in (False, True):
        got = rot(p, q, k, inverse=inverse)
        one = rot(p.long(), q, inverse=inverse)
        assert torch.equal(one, got[0])
        for x, y in zip((q, k), got):
            want = otok.rotary(_np(x), pos, rot.frequencies, part, layout, axes, rot.factor, inverse)
            assert np.all(np.abs(_np(y) - want) <= _rotary_bar(_np(x), want, part, layout, axes, rot.factor, dtype))
    # in place, over views of an unaligned buffer, and with a batch that shares its positions
    base = torch.empty(fused.numel() + 1, dtype=dtype, device=DEV)[1:].view(fused.shape)
    base.copy_(fused)
    y = base[:, :heads[0]]
    assert rot(p, y, out=y) is y and torch.equal(y, rot(p, q)) and torch.equal(base[:, heads[0]:], fused[:, heads[0]:])
    two = rot(p, torch.stack((q, 2 * q)))
    assert torch.equal(two[0], rot(p, q)) and torch.equal(two[1], rot(p, 2 * q))
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)                       # heads first
    assert torch.equal(rot(p, swapped), rot(p, q))


@pytest.mark.gpu
def test_rotary_gradient():
    """The gradient against the formula's (the opposite rotation) and against differences: the map is linear, so a
    difference quotient is the map itself up to the roundings of its terms."""
    from blast3r_amd.rotary import Rotary
    rot = Rotary(64, rotary_dim=48, axes=2, layout='interleaved', scaling=dict(kind='ramp', factor=4, length=512), device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    mk = lambda *s: torch.randn(s, device=DEV, generator=g)  # noqa: E731
    pos = torch.randint(-50, 5000, (9, 2), device=DEV, generator=g, dtype=torch.int32)
    x, k = mk(2, 9, 1, 64).requires_grad_(), mk(2, 9, 3, 64).requires_grad_()
    wide = x.expand(2, 9, 5, 64)                                                   # a head that five share
    y, z = rot(pos, wide, k)
    gy, gz = mk(2, 9, 5, 64), mk(2, 9, 3, 64)
    dx, dk = torch.autograd.grad((y, z), (x, k), (gy, gz))
    for got, grad, src in ((dx, gy, wide), (dk, gz, k)):
        want = np.stack([otok.rotary(_np(grad[b]), pos.cpu().numpy(), rot.frequencies, 48, 'interleaved', 2, rot.factor, True)
                         for b in range(2)])
        bar = np.stack([_rotary_bar(_np(grad[b]), want[b], 48, 'interleaved', 2, rot.factor, torch.float32) for b in range(2)])
        if got.shape[2] == 1:
            # the sum over the heads adds four roundings
            want, bar = want.sum(2, keepdims=True), bar.sum(2, keepdims=True) + 4 * 2.0 ** -24 * np.abs(want).sum(2, keepdims=True)
        assert np.all(np.abs(_np(got) - want) <= bar)
    u = mk(2, 9, 3, 64)
    with torch.no_grad():
        diff = (rot(pos, k + 0.5 * u).double() - rot(pos, k - 0.5 * u).double())
    a, b = float((diff * gz.double()).sum()), float((dk.double() * u.double()).sum())
    size = float((gz.abs().double() * (k.detach().abs() + u.abs()).double()).sum())
    assert abs(a - b) <= 4e-6 * size
    # the gradient's gradient: the map itself
    g1 = gz.clone().requires_grad_()
    (d1,) = torch.autograd.grad(rot(pos, x.detach().expand(2, 9, 5, 64), k)[1], (k,), (g1,), create_graph=True)
    (d2,) = torch.autograd.grad(d1, (g1,), (u,))
    with torch.no_grad():
        assert torch.equal(d1, dk) and torch.equal(d2, rot(pos, u))
    # a tensor that needs no gradient beside one that does; a broadcast gradient
    q2 = mk(2, 9, 3, 64)
    y, z = rot(pos, q2, k)
    (dk2,) = torch.autograd.grad(z.sum(), (k,))
    ones = otok.rotary(np.ones((9, 3, 64)), pos.cpu().numpy(), rot.frequencies, 48, 'interleaved', 2, rot.factor, True)
    assert np.all(np.abs(_np(dk2[0]) - ones) <= 3e-6)


# ---------------------------------------------------------------------------------- cache (GPU)

def _cache(n_blocks, heads, dim, bits, seed=0, spread=2):
    """A device cache with random codes and factors, and the oracle's copy."""
    from blast3r_amd.kv_cache import KVCache
    rng = np.random.default_rng(seed)
    c = KVCache(n_blocks, heads, dim, BITS[bits], device=DEV)
    for t in (c.k, c.v):
        x = torch.tensor(rng.normal(size=tuple(t.shape)) * 60, dtype=torch.float32)
        t.copy_((x.clamp(-448, 448) if bits == 'fp8' else x.round().clamp(-127, 127)).to(t.dtype))
    e = rng.integers(-7 - spread, -6 + spread, tuple(c.scales.shape))
    c.scales.copy_(torch.tensor(2.0 ** e * (1.0 if bits == 'fp8' else rng.uniform(0.6, 1.0, e.shape)), dtype=torch.float32))
    return c, _mirror(c, bits)


def _mirror(c, bits):
    return otok.Cache(_np(c.k.float()), _np(c.v.float()).transpose(0, 1, 3, 2), _np(c.scales), bits)


def _same(c, o):
    assert np.array_equal(_np(c.scales), o.scales, equal_nan=True)
    ok = ~np.isnan(o.scales)
    k, v = _np(c.k.float()), _np(c.v.float()).transpose(0, 1, 3, 2)
    assert np.array_equal(k[ok[..., 0]], o.k[ok[..., 0]]) and np.array_equal(v[ok[..., 1]], o.v[ok[..., 1]])
    assert np.isfinite(k).all() and np.isfinite(v).all()


def _pages(rng, blocks, n_blocks, width):
    order = rng.permutation(n_blocks)
    pages, at = np.full((len(blocks), width), -1), 0
    for s, n in enumerate(blocks):
        pages[s, :n] = order[at:at + n]
        at += n
    return pages


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dim,heads,dtype', [(64, 3, torch.bfloat16), (128, 2, torch.float16), (32, 1, torch.float32),
                                             (96, 5, torch.bfloat16), (256, 2, torch.float32)])
def test_append_and_read_against_oracle(bits, dim, heads, dtype):
    """Ragged appends within, across and at the ends of blocks; then single tokens, some of which outgrow their block."""
    rng = np.random.default_rng(dim)
    starts, counts = [0, 63, 64, 1, 100, 5, 60, 0, 17], [1, 1, 64, 62, 130, 0, 8, 200, 7]
    blocks = [(a + b + 70) // 64 + 1 for a, b in zip(starts, counts)]
    c, o = _cache(sum(blocks), heads, dim, bits, seed=dim)
    pages = _pages(rng, blocks, sum(blocks), max(blocks))
    n = sum(counts)
    fused = torch.tensor(rng.normal(size=(n, 2 * heads + 1, dim)) * rng.choice([0.1, 1.0, 5.0], (n, 1, 1)),
                         dtype=torch.float32).to(dtype).to(DEV)
    k, v = fused[:, :heads], fused[:, heads:2 * heads]
    off = np.concatenate(([0], np.cumsum(counts)))
    print(f'append {bits} {dim} {heads} {dtype}', flush=True)
    c.append(k, v, _i32(pages), _i32(starts), offsets=_i32(off), max_new=max(counts))
    o.append(_np(k), _np(v), pages, starts, counts)
    _same(c, o)
    lens = [a + b for a, b in zip(starts, counts)]
    for step, size in enumerate((0.01, 30.0, 1.0)):
        x = torch.tensor(rng.normal(size=(2, len(lens), heads, dim)) * size, dtype=torch.float32).to(dtype).to(DEV)
        if step == 1:                                       # an unaligned view, another order of heads
            buf = torch.empty(x.numel() + 3, dtype=dtype, device=DEV)[3:].view(2, heads, len(lens), dim).transpose(1, 2)
            buf.copy_(x)
            x = buf
        c.append(x[0], x[1], _i32(pages), _i32(lens))
        o.append(_np(x[0]), _np(x[1]), pages, lens, [1] * len(lens))
        _same(c, o)
        lens = [a + 1 for a in lens]
    first = [0, 63, 10, 0, 70, 0, 0, 1, 3]
    count = [a - b for a, b in zip(lens, first)]
    for out_type in (dtype, torch.float32):
        rk, rv = c.read(_i32(pages), _i32(first), _i32(np.concatenate(([0], np.cumsum(count)))), sum(count),
                        max_count=max(count), dtype=out_type)
        row = 0
        for s, (a, m) in enumerate(zip(first, count)):
            wk, wv, _ = o.sequence(pages[s], a + m)
            for got, want in ((rk, wk), (rv, wv)):
                want = torch.tensor(want[a:]).float().to(out_type)
                assert torch.equal(got[row:row + m].cpu(), want)
            row += m


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
def test_cache_edges(bits):
    """Zeros, the largest and the smallest factors, NaN and infinities, blocks that are not there, empty calls."""
    rng = np.random.default_rng(5)
    c, o = _cache(6, 2, 64, bits)
    pages = np.array([[0, 1], [2, -1], [7, 3], [4, 5]])
    x = np.float32(rng.normal(size=(4 * 100, 2, 64)))
    x[5] = 0.0
    x[0:100, 1] = 0.0                                       # a head of zeros
    x[300:330, 0] *= np.float32(2.0 ** -80)                 # below the least factor's step, beside larger ones
    x[364:400, 0] = np.float32(1e18)                        # near the largest factor
    k, v = x.copy(), x[::-1].copy()
    k[310, 1, 7], v[320, 0, 3], k[390, 1, 0] = np.nan, np.inf, 1e25
    put = lambda a: torch.tensor(a, device=DEV)  # noqa: E731
    print(f'cache edges {bits}', flush=True)
    c.append(put(k), put(v), _i32(pages), _i32([0, 0, 0, 0]))
    o.append(k, v, pages, [0, 0, 0, 0], [100] * 4)
    _same(c, o)
    assert np.isnan(o.scales).sum() == 3
    # a poisoned block stays so until its first place is written again
    t = np.float32(rng.normal(size=(4, 2, 64)))
    c.append(put(t), put(t), _i32(pages), _i32([100] * 4))
    o.append(t, t, pages, [100] * 4, [1] * 4)
    _same(c, o)
    c.append(put(t), put(t), _i32(pages), _i32([0, 64, 0, 64]))
    o.append(t, t, pages, [0, 64, 0, 64], [1] * 4)
    _same(c, o)
    rk, rv = c.read(_i32(pages), _i32([0, 32, 0, 63]), None, 4 * 90, dtype=torch.float32)
    for s, a in enumerate((0, 32, 0, 63)):
        wk, wv, _ = o.sequence(pages[s], a + 90)            # places past a block list or in no block read as zeros
        for got, want in ((rk, wk), (rv, wv)):              # the product, rounded to fp32
            assert np.array_equal(_np(got[90 * s:90 * s + 90]), np.float64(np.float32(want[a:])), equal_nan=True)
    before = c.k.view(torch.uint8).clone()
    e = torch.zeros((0, 2, 64), device=DEV)
    c.append(e, e, _i32(pages), _i32([0] * 4))
    c.append(put(x[:4]), put(x[:4]), _i32(pages), _i32([-1, 128, 1 << 30, 500]))      # starts out of range
    c.append(put(x[:4]), put(x[:4]), _i32(pages), _i32([0] * 4), offsets=_i32([4, 9, -3, 4, 4]))
    assert torch.equal(before, c.k.view(torch.uint8))
    assert c.read(_i32(pages), _i32([0] * 4), None, 0)[0].shape == (0, 2, 64)


# ---------------------------------------------------------------------------------- attention (GPU)

def _check(c, o, q, pages, lens, counts, causal=True, window=None, scale=None, uniform=False, max_new=None):
    off = None if uniform else _i32(np.concatenate(([0], np.cumsum(counts))))
    got, lse = c.attend(q, _i32(pages), _i32(lens), offsets=off, max_new=max_new or max(counts), causal=causal, window=window,
                        scale=scale, return_lse=True)
    want, want_lse, size = otok.attend(o, _np(q), pages, lens, counts, scale or 1.0 / math.sqrt(q.shape[2]), causal, window)
    assert np.array_equal(np.isnan(_np(got)), np.isnan(want))
    ok = ~np.isnan(want)
    step = HALF_STEP[q.dtype] * np.abs(want) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    err = np.abs(_np(got) - want)[ok]
    assert np.all(err <= (1.2e-3 * size + step)[ok]), float(np.max(err / np.maximum((1.2e-3 * size + step)[ok], 1e-300)))
    empty = want_lse == -math.inf
    assert np.array_equal(_np(lse) == -math.inf, empty)
    fine = np.isfinite(want_lse)
    assert np.all(np.abs(_np(lse)[fine] - want_lse[fine]) <= 6e-4)
    return got


ATTEND = [
    # dim, heads, group, lengths, counts, causal, window
    (64, 2, 1, [1, 64, 65, 200], [1, 1, 1, 1], True, None),
    (64, 1, 4, [700, 3, 0, 129], [1, 2, 1, 4], True, None),        # 16 rows, an empty sequence
    (128, 2, 8, [300, 900], [1, 1], True, 100),
    (128, 1, 5, [333], [6], True, None),                           # 30 rows
    (96, 2, 3, [100, 257], [10, 40], True, 37),                    # 120 rows; some before the window's tokens
    (64, 1, 1, [5, 90], [9, 33], True, None),                      # more rows than tokens: the first see none
    (32, 2, 2, [500], [70], False, None),
    (64, 1, 2, [400, 191], [150, 63], True, None),                 # two tiles of 32 to a wave
    (128, 1, 1, [330], [300], False, 90),
    (256, 1, 2, [300], [80], True, None),
    (256, 2, 1, [650], [1], True, None),
    (32, 1, 16, [4000], [1], True, None),
    (64, 1, 1, [3000], [1], True, 700),
    (256, 1, 4, [300], [6], True, None),                           # 24 rows of the largest head
    (32, 1, 5, [1500], [6], False, None),
    (96, 2, 3, [190, 2500], [70, 1], True, None),                  # 210 rows, and one token that shares their call
    (64, 2, 1, [70, 0, 1, 2100], [70, 0, 1, 300], True, 200),      # sequences without rows or tokens among others
    (128, 1, 2, [1300], [200], True, 500),
]


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dim,heads,group,lens,counts,causal,window', ATTEND)
def test_attend_against_oracle(bits, dim, heads, group, lens, counts, causal, window):
    rng = np.random.default_rng(sum(lens))
    blocks = [max(1, (n + 63) // 64) for n in lens]
    c, o = _cache(sum(blocks) + 1, heads, dim, bits, seed=dim)
    pages = _pages(rng, blocks, sum(blocks) + 1, max(blocks) + 2)
    for s, n in enumerate(lens):                            # codes of places that hold no token yet may be anything
        if n % 64:
            p = int(pages[s, n // 64])
            c.k.view(torch.uint8)[p, :, n % 64:] = 0x7f
            c.v.view(torch.uint8)[p, :, :, n % 64:] = 0x7f
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.tensor(rng.normal(size=(sum(counts), heads * group + 1, dim)) * 2.0, dtype=torch.float32).to(dtype).to(DEV)
        print(f'attend {bits} {dtype} {dim} {heads} {group} {lens} {counts}', flush=True)
        _check(c, o, x[:, 1:], pages, lens, counts, causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('counts', [[1], [3], [12], [40], [90]])
def test_attend_ranges(bits, counts, dtype):
    """Factors from 2^-40 to 2^40 (to 1 where outputs are fp16) in neighbouring blocks, queries of very different sizes, peaked rows, a NaN block that
    only some rows see, NaN queries, missing blocks."""
    rng = np.random.default_rng(counts[0])
    n = 64 * 20 - 11
    c, o = _cache(22, 1, 64, bits)
    pages = _pages(rng, [20], 22, 20)
    for b in range(20):                                     # values large where keys are small and the other way round
        e = int(rng.integers(-20, 20 if dtype == torch.bfloat16 else 1))
        c.scales[int(pages[0, b]), 0] = torch.tensor([2.0 ** (-7 - abs(e) / 4), 2.0 ** (2 * e)], device=DEV)
    pages[0, 3] = -1
    pages[0, 7] = 22
    o = _mirror(c, bits)
    x = rng.normal(size=(counts[0], 2, 64)) * np.exp(rng.normal(size=(counts[0], 2, 1)) * 2)
    x[0, 0] = 0.0
    x[-1, 1] *= 1e-20
    q = torch.tensor(x, dtype=torch.float32).clamp(-8, 8).to(dtype).to(DEV)
    print(f'attend ranges {bits} {counts} {dtype}', flush=True)
    _check(c, o, q, pages, [n], counts)
    _check(c, o, q, pages, [n], counts, scale=0.5)
    c.scales[int(pages[0, 19]), 0, 0] = math.nan            # the newest block: rows before it do not see it
    c.scales[int(pages[0, 2]), 0, 1] = math.nan
    o = _mirror(c, bits)
    _check(c, o, q, pages, [n], counts, window=64 * 10)
    _check(c, o, q, pages, [n], counts)
    c.scales[int(pages[0, 19]), 0] = torch.tensor([1.0, math.nan], device=DEV)      # its values: rows that see it in part or not
    o = _mirror(c, bits)
    _check(c, o, q, pages, [n], counts, window=64 * 10)
    q = q.clone()
    q[0, 1, 5] = math.nan
    o2 = _mirror(c, bits)
    _check(c, o2, q, pages, [64 * 19], counts, window=64 * 12)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', ['fp8', 'int8'])
def test_attend_one_key(bits):
    """A row that sees one token has its value: fp16 weights are the same in numerator and denominator, so all that is left
    are fp32 roundings (the weight's products, a reciprocal and a factor's: 2^-21 together) and half a step."""
    c, o = _cache(3, 2, 64, bits, seed=9)
    lens = [1, 50, 58]                                      # with 69 rows before it each stays within two blocks
    for n in (1, 20, 70):
        q = torch.randn((3 * n, 4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)).half() * 3
        got = _np(c.attend(q, _i32([[0, 1], [0, 1], [2, 1]]), _i32([n - 1 + x for x in lens]), window=1, max_new=n)).reshape(3, n, 4, 64)
        for s, pages in enumerate(([0, 1], [0, 1], [2, 1])):
            _, v, _ = o.sequence(pages, n - 1 + lens[s])
            for i in range(n):
                want = np.repeat(v[lens[s] - 1 + i], 2, 0)
                assert np.all(np.abs(got[s, i] - want) <= (2.0 ** -21 + 2.0 ** -11) * np.abs(want) + 2.0 ** -25), (n, s, i)


@pytest.mark.gpu
def test_attend_bounds():
    """max_new below a sequence's rows leaves the others as they are; lengths past the block list and below zero, offsets
    out of order and a cache without blocks stay inside the buffers."""
    from blast3r_amd.kv_cache import KVCache
    rng = np.random.default_rng(4)
    c, o = _cache(8, 2, 64, 'fp8')
    pages = _pages(rng, [4, 4], 8, 4)
    x = torch.tensor(rng.normal(size=(300, 2, 64)), dtype=torch.float32, device=DEV).bfloat16()
    print('attend bounds', flush=True)
    for n, most in ((10, 7), (150, 40)):
        off, lens = _i32([0, n, n + 3]), [200, 100]
        y = torch.full_like(x[:n + 3], 7.0)
        c.attend(x[:n + 3], _i32(pages), _i32(lens), offsets=off, max_new=most, out=y)
        want, _, size = otok.attend(o, _np(x[:n + 3]), pages, lens, [n, 3], 0.125)
        done = np.r_[0:most, n:n + 3]
        assert np.all(np.abs(_np(y) - want)[done] <= 1.2e-3 * size[done] + 2.0 ** -8 * np.abs(want[done]))
        rest = _np(y)[most:n]                               # up to a tile of them may be done all the same
        assert np.all((rest == 7.0) | (np.abs(rest - want[most:n]) <= 1.2e-3 * size[most:n] + 2.0 ** -8 * np.abs(want[most:n])))
    # 256 tokens is all that four blocks hold
    got = c.attend(x[:2], _i32(pages), _i32([100000, -5]))
    want, _, size = otok.attend(o, _np(x[:2]), pages, [256, 0], [1, 1], 0.125)
    assert np.all(np.abs(_np(got) - want) <= 1.2e-3 * size + 2.0 ** -8 * np.abs(want)) and not got[1].any()
    y = torch.full_like(x[:6], 7.0)
    c.attend(x[:6], _i32(pages), _i32([50, 60]), offsets=_i32([9, -2, 4]), out=y)
    assert bool((y == 7.0).all())
    none = KVCache(0, 2, 64, device=DEV)
    for n in (2, 40, 400):
        q = x[:1].expand(n, 2, 64)
        got, lse = none.attend(q, _i32(np.zeros((2, 3))), _i32([150, 20]), return_lse=True)
        assert not got.any() and bool((lse == -math.inf).all())
        assert not none.attend(q, _i32(np.zeros((2, 0))), _i32([150, 20])).any()
    none.append(x[:2], x[:2], _i32(np.zeros((2, 3))), _i32([0, 64]))
    assert not none.read(_i32(np.zeros((2, 3))), _i32([0, 64]), None, 4)[0].any()
    assert c.attend(x[:0], _i32(np.zeros((0, 3))), _i32([])).shape == (0, 2, 64)
    with pytest.raises(RuntimeError):
        c.attend(x[:2].requires_grad_(), _i32(pages), _i32([5, 6]))
    with pytest.raises(RuntimeError):
        c.append(x[:2].clone().requires_grad_(), x[:2], _i32(pages), _i32([5, 6]))


@pytest.mark.gpu
@pytest.mark.parametrize('causal,window', [(True, None), (True, 60), (False, 150)])
@pytest.mark.parametrize('n', [1, 20, 100, 300])
def test_attend_positions_past_the_block_list(n, causal, window):
    """Rows stand at the last positions of their sequence's length and row count, also where its tokens are more than its
    block list is wide (those past it are hidden) or its rows more than the tensor has."""
    rng = np.random.default_rng(n)
    c, o = _cache(8, 2, 64, 'int8')
    pages = _pages(rng, [2, 1], 8, 2)
    lens, counts = [128 + n // 2 + 5, 60], [n, 1]
    x = torch.tensor(rng.normal(size=(n + 1, 4, 64)), dtype=torch.float32, device=DEV).bfloat16()
    print(f'attend past the block list {n} {causal} {window}', flush=True)
    _check(c, o, x, pages, lens, counts, causal, window)
    more = np.concatenate((_np(x[:n]), np.zeros((7, 4, 64))))
    want, _, size = otok.attend(o, more, pages[:1], lens[:1], [n + 7], 0.125, causal, window)
    got = _np(c.attend(x[:n], _i32(pages[:1]), _i32(lens[:1]), offsets=_i32([0, n + 7]), causal=causal, window=window))
    assert np.all(np.abs(got - want[:n]) <= 1.2e-3 * size[:n] + 2.0 ** -8 * np.abs(want[:n]))


@pytest.mark.gpu
def test_attend_splits_join_to_one_pass():
    """Every number of parts gives the sums of one pass, to the roundings of fp32 and of the output."""
    from blast3r_amd._lib import BaKvAttendArgs, check, lib, stream_ptr
    L = lib()
    rng = np.random.default_rng(2)
    lens = [64 * 37 + 5, 64 * 3, 1, 0]
    for dim, q_heads, counts in ((64, 2, [1, 1, 1, 1]), (96, 6, [20, 20, 20, 20]), (128, 2, [100, 100, 100, 100])):
        c, o = _cache(64, 2, dim, 'int8')
        pages = _i32(_pages(rng, [38, 3, 1, 0], 64, 40))
        n = sum(counts)
        q = torch.randn((n, q_heads, dim), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half() * 2
        out = {}
        for splits in (1, 2, 3, 9, 64):
            print(f'attend splits {dim} {splits}', flush=True)
            y = torch.full_like(q, math.nan)
            work = torch.full((max(16, L.ba_kv_attend_workspace_bytes(n, q_heads, dim, splits)),), 255, dtype=torch.uint8, device=DEV)
            lengths = _i32(lens)
            a = BaKvAttendArgs(k=c.k.data_ptr(), v=c.v.data_ptr(), scales=c.scales.data_ptr(), n_blocks=64, heads=2, dim=dim, bits=1,
                               n_seqs=4, pages=pages.data_ptr(), pages_stride=40, n_pages=40, dtype=1, lengths=lengths.data_ptr(),
                               n_rows=n, rows_per_seq=counts[0], max_rows=counts[0], q=q.data_ptr(), o=y.data_ptr(),
                               q_st=q.stride(0), q_sh=q.stride(1), o_st=y.stride(0), o_sh=y.stride(1), q_heads=q_heads, causal=1,
                               scale=0.1, n_splits=splits, workspace=work.data_ptr(), workspace_bytes=work.numel())
            check(L.ba_kv_attend(ctypes.byref(a), stream_ptr(DEV)))
            out[splits] = y.float()
        for s in out:
            # weights are rounded relative to another reference: 2^-11 of sum p |v| apart at most
            assert torch.isfinite(out[s]).all() and float((out[s] - out[1]).abs().max()) <= 2e-3 * float(out[1].abs().max())
            assert float(out[s][-counts[3]:].abs().max()) == 0.0


@pytest.mark.gpu
def test_cache_past_32_bit_offsets():
    """A cache of 4.6 GB for the keys: blocks at its end are written, read and attended to."""
    from blast3r_amd.kv_cache import KVCache
    n, H, D = 70_000, 8, 128
    c = KVCache(n, H, D, torch.int8, device=DEV)
    pages = np.array([[n - 1, 3, n - 2]])
    rng = np.random.default_rng(1)
    k, v = (torch.tensor(rng.normal(size=(150, H, D)), dtype=torch.float32, device=DEV).bfloat16() for _ in range(2))
    print('cache of 9 GB', flush=True)
    c.append(k, v, _i32(pages), _i32([0]))
    small = otok.Cache(np.zeros((3, H, 64, D)), np.zeros((3, H, 64, D)), np.ones((3, H, 2)), 'int8')
    small.append(_np(k), _np(v), [[0, 1, 2]], [0], [150])
    rk, rv = c.read(_i32(pages), _i32([0]), None, 150, dtype=torch.float32)
    wk, wv, _ = small.sequence([0, 1, 2], 150)
    assert np.array_equal(_np(rk), np.float64(np.float32(wk))) and np.array_equal(_np(rv), np.float64(np.float32(wv)))
    q = torch.tensor(rng.normal(size=(1, H, D)), dtype=torch.float32, device=DEV).bfloat16()
    want, _, size = otok.attend(small, _np(q), [[0, 1, 2]], [150], [1], 1 / math.sqrt(D))
    got = _np(c.attend(q, _i32(pages), _i32([150])))
    assert np.all(np.abs(got - want) <= 1.2e-3 * size + 2.0 ** -8 * np.abs(want))


@pytest.mark.gpu
def test_tokens_in_a_graph_and_on_a_side_stream():
    """A step (rotate, append, attend) captured once and replayed with other inputs, lengths and blocks, with eager work
    between the replays; the same step on another stream than the tensors were made on."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    H, G, D, S = 2, 4, 64, 3
    rot = Rotary(D, device=DEV)
    caches = [KVCache(60, H, D, device=DEV) for _ in range(3)]
    pages = _i32(np.arange(60).reshape(3, 20))
    qkv = torch.zeros((S, H * (G + 2), D), dtype=torch.bfloat16, device=DEV)
    lens = torch.zeros(S, dtype=torch.int32, device=DEV)

    def step(c):
        q, k = rot(lens, qkv[:, :H * G], qkv[:, H * G:H * G + H])
        c.append(k, qkv[:, H * G + H:], pages, lens)
        return c.attend(q, pages, lens + 1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(KVCache(60, H, D, device=DEV))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(caches[0])
    gen = torch.Generator(device=DEV).manual_seed(1)
    for t in range(70):
        qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=gen))
        if t == 40:
            lens.copy_(_i32([700, 64, 5]))
        graph.replay()
        eager = step(caches[1])
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(caches[2])
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and torch.equal(y, other), t
        lens += 1
    for c in caches[1:]:
        assert torch.equal(c.k.view(torch.uint8), caches[0].k.view(torch.uint8)) and torch.equal(c.scales, caches[0].scales)


@pytest.mark.gpu
@pytest.mark.parametrize('bits,bar', [('fp8', 0.13), ('int8', 0.04)])
def test_example_of_online_frames(bits, bar):
    """examples/online_frames.py: rotary, append, attend over chosen frames and depth sampling together.  Attention over
    codes against attention over the unrounded keys and values: e4m3 is off by at most 2^-4 of a value (twice: keys through
    the weights, values), int8 by half of 1/127 of a block's largest value, about 2% of a value of ordinary size."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples', 'online_frames.py')
    spec = importlib.util.spec_from_file_location('online_frames', path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    error, depths, net = ex.run(frames=4, layers=2, width=512, heads=8, like=2, bits=BITS[bits], device=DEV)
    assert 0.0 < error < bar
    assert depths.shape == (1000, 6) and bool(torch.isfinite(depths).all())
