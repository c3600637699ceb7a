"""The timed cases of the token operators: rotary positions, the 8-bit key/value cache and attention over it.

They are what the depth and matching networks whose answers a bundle adjustment is fitted to do with each new frame:
the frame's tokens get their positions (``Rotary``), their keys and values are kept in 8 bits (``KVCache.append``, read
back with ``KVCache.read``), and queries attend to the kept tokens (``KVCache.attend``).  A frame of 512 x 384 pixels in
patches of 16 x 16 is 768 tokens.  With ``own`` false every operator is computed in its plain form (torch, 32 bits).

Cache layout: blocks of 64 tokens; ``k`` is (n_blocks, heads, 64, dim), ``v`` is (n_blocks, heads, dim, 64), one byte
each, ``scales`` (n_blocks, heads, 2) in fp32 holds the factors of a block's keys and values; ``pages`` (n_seqs, most
blocks) lists the blocks of each sequence.
"""
import math
import random

import torch

own = False

BLOCK = 64
DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BITS = {'fp8': torch.float8_e4m3fn, 'int8': torch.int8}
ROWS, COLS = 24, 32                  # the patches of a frame
SCALING = {'none': None, 'linear': dict(kind='linear', factor=4.0), 'base': dict(kind='base', factor=4.0),
           'ramp': dict(kind='ramp', factor=8.0, length=16384, fast=32.0, slow=1.0)}


# ------------------------------------------------------------------------------------------------ cases

def _rotary(name, tokens, q_heads, k_heads, dim, part, layout='half', axes=1, context=8192, scaled='none', dtype='bf16',
            grad=False):
    c = dict(op='rotary', tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim, part=part, layout=layout, axes=axes,
             context=context, scaled=scaled, dtype=dtype, grad=grad)
    return dict(c, name=name) if name else c


def _write(name, seqs, held, new, heads, dim, bits, dtype='bf16', salt=1):
    """held, new: (least, most) tokens of a sequence before the call and in it."""
    c = dict(op='write', seqs=seqs, held_lo=held[0], held_hi=held[1], new_lo=new[0], new_hi=new[1], heads=heads, dim=dim,
             bits=bits, dtype=dtype, salt=salt)
    return dict(c, name=name) if name else c


def _read(name, seqs, held, heads, dim, bits, dtype='bf16', salt=1):
    c = dict(op='read', seqs=seqs, held_lo=held[0], held_hi=held[1], heads=heads, dim=dim, bits=bits, dtype=dtype,
             salt=salt)
    return dict(c, name=name) if name else c


def _attend(name, seqs, new, held, q_heads, k_heads, dim, bits, dtype='bf16', causal=True, window=0, salt=1):
    """new: (least, most) queries of a sequence; held: its keys before them.  window 0: none."""
    c = dict(op='attend', seqs=seqs, new_lo=new[0], new_hi=new[1], held_lo=held[0], held_hi=held[1], q_heads=q_heads,
             k_heads=k_heads, dim=dim, bits=bits, dtype=dtype, causal=causal, window=window, salt=salt)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one sequence while it is generated: a launch
        _rotary('rotary token', 1, 32, 8, 128, 128),
        # queries and keys of 8 frames' patches, placed by row and column
        _rotary('rotary frames', 8 * ROWS * COLS, 16, 16, 64, 64, axes=2),
        # a training step on a long sequence: half of the head, interleaved, by-parts scaling, with its gradient
        _rotary('rotary long train', 32768, 32, 8, 128, 64, layout='interleaved', context=131072, scaled='ramp', grad=True),
        # one token for each of 64 sequences: most go to blocks that are open, whose codes may have to be made anew
        _write('write token', 64, (1, 8192), (1, 1), 8, 128, 'int8'),
        # the keys and values of 16 frames after 20 that are kept
        _write('write frames', 1, (20 * 768, 20 * 768), (16 * 768, 16 * 768), 16, 64, 'fp8'),
        # prompts of many lengths that continue sequences within a block
        _write('write ragged', 24, (0, 1000), (1, 1500), 5, 96, 'int8', dtype='fp16'),
        # a long sequence handed on in 16 bits
        _read('read long', 1, (131072, 131072), 8, 128, 'fp8'),
        # a query over the first frame
        _attend('attend token short', 1, (1, 1), (776, 776), 16, 16, 64, 'fp8'),
        # a step of 48 sequences of many lengths, four query heads to a key head
        _attend('attend tokens ragged', 48, (1, 1), (0, 8191), 32, 8, 128, 'int8'),
        # a query over 250 kept frames
        _attend('attend token long', 1, (1, 1), (250 * 768 - 1, 250 * 768 - 1), 16, 16, 64, 'fp8'),
        # a frame's tokens over its own and those of 32 kept frames
        _attend('attend frame', 1, (768, 768), (32 * 768, 32 * 768), 16, 16, 64, 'fp8', causal=False),
        # a chunk of a long prompt for two sequences
        _attend('attend chunk', 2, (2048, 2048), (14336, 14336), 32, 8, 128, 'int8'),
    ]


def _log(rng, lo, hi):
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    return n + (n == 3072)


def draw(rng):
    op = rng.choice(['rotary', 'write', 'read', 'attend', 'attend'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16'])
    bits = rng.choice(['fp8', 'int8'])
    salt = rng.randrange(1 << 20)
    if op == 'rotary':
        axes = rng.choice([1, 1, 2])
        dim = rng.choice([32, 64, 96, 128, 256])
        part = dim if rng.random() < 0.5 else dim // 2
        heads = rng.choice([(32, 8), (16, 16), (5, 1), (12, 3)])
        most = min(32768, 32768 * 40 * 128 // (sum(heads) * dim))
        return _rotary(None, _log(rng, 1, most), heads[0], heads[1], dim, part, rng.choice(['half', 'interleaved']), axes,
                       _log(rng, 40000, 1 << 20), rng.choice(list(SCALING)), rng.choice(['bf16', 'fp16', 'fp32']),
                       rng.random() < 0.3)
    dim = rng.choice([32, 64, 64, 96, 128, 128, 256])
    heads = rng.choice([1, 2, 5, 8, 16])
    if op == 'write':
        dtype = rng.choice(['bf16', 'fp16', 'fp32'])
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8_000_000 // (seqs * heads * dim)))
        return _write(None, seqs, (0, _log(rng, 1, 4096)), (rng.choice([0, 1, new]), new), heads, dim, bits, dtype, salt)
    if op == 'read':
        seqs = _log(rng, 1, 64)
        return _read(None, seqs, (0, _log(rng, 1, 64_000_000 // (seqs * heads * dim))), heads, dim, bits, dtype, salt)
    group = rng.choice([1, 2, 4, 8])
    heads = rng.choice([2, 5, 8])
    seqs = _log(rng, 1, 32)
    if rng.random() < 0.5:           # single tokens, or a few drafted ones
        new = rng.choice([1, 1, 2, 5])
        held = _log(rng, 1, min(160_000, 150_000_000 // (seqs * heads * dim)))
        low = rng.choice([0, held])
    else:                            # frames and chunks
        new = _log(rng, 6, 2048)
        held = _log(rng, 1, 16384)
        most = 250_000_000_000 // (4 * dim)
        while seqs > 1 and seqs * heads * group * new * (held + new) > most:
            seqs //= 2
        while held > 1 and seqs * heads * group * new * (held + new) > most:
            held //= 2
        while new > 6 and seqs * heads * group * new * (held + new) > most:
            new //= 2
        low = rng.choice([0, held])
    return _attend(None, seqs, (rng.choice([1, new]), new), (low, held), heads * group, heads, dim, bits, dtype,
                   rng.random() < 0.7, rng.choice([0, 0, 0, 100, 1000]), salt)


def _lengths(n, lo, hi, salt):
    """n lengths from lo to hi, the longest among them."""
    r = random.Random(salt)
    got = [r.randint(lo, hi) for _ in range(n)]
    got[r.randrange(n)] = hi
    return got


def _sizes(c):
    """(tokens held before the call, new tokens) of each sequence."""
    held = _lengths(c['seqs'], c['held_lo'], c['held_hi'], c['salt'])
    new = _lengths(c['seqs'], c['new_lo'], c['new_hi'], c['salt'] + 1) if 'new_lo' in c else [0] * c['seqs']
    return held, new


def work(c):
    es = 4 if c['dtype'] == 'fp32' else 2
    if c['op'] == 'rotary':
        n = c['tokens'] * (c['q_heads'] + c['k_heads'])
        ways = 2 if c['grad'] else 1
        return dict(bytes=ways * 2 * n * c['dim'] * es + 4 * c['tokens'] * c['axes'], flops=ways * 3 * n * c['part'])
    held, new = _sizes(c)
    if c['op'] == 'write':           # the call and the blocks it touched read back
        row = 2 * c['heads'] * c['dim'] * (es + 1)
        return dict(bytes=row * sum(new) + row * sum(h % BLOCK + n for h, n in zip(held, new) if n), flops=0)
    if c['op'] == 'read':
        return dict(bytes=2 * sum(held) * c['heads'] * c['dim'] * (1 + es), flops=0)
    keys = pairs = 0
    for h, n in zip(held, new):
        total, least = h + n, h + n
        for i in range(n):
            hi = h + i + 1 if c['causal'] else total
            lo = max(0, h + i + 1 - c['window']) if c['window'] else 0
            pairs += max(0, hi - lo)
            least = min(least, lo)
        keys += total - least
    return dict(bytes=2 * keys * c['k_heads'] * c['dim'] + 2 * sum(new) * c['q_heads'] * c['dim'] * es,
                flops=4 * c['dim'] * c['q_heads'] * pairs)


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(c):
    """Angle per position of each pair, and the factor of the result (64 bits)."""
    n = c['part'] // c['axes']
    base, scaling = 10000.0, SCALING[c['scaled']]
    if scaling and scaling['kind'] == 'base':
        base *= scaling['factor'] ** (n / max(n - 2, 1))
    f = [base ** (-2.0 * p / n) for p in range(n // 2)]
    m = 1.0
    if scaling and scaling['kind'] == 'linear':
        f = [x / scaling['factor'] for x in f]
    if scaling and scaling['kind'] == 'ramp':
        s = scaling['factor']
        keep = [min(1.0, max(0.0, (scaling['length'] * x / (2 * math.pi) - scaling['slow']) /
                             (scaling['fast'] - scaling['slow']))) for x in f]
        f = [g * x + (1 - g) * x / s for g, x in zip(keep, f)]
        m = 0.1 * math.log(s) + 1.0
    return f, m


def _codes(gen, shape, bits):
    x = torch.randn(shape, device=DEV, generator=gen) * (100.0 if bits == 'fp8' else 40.0)
    return x.clamp_(-448, 448).to(BITS['fp8']) if bits == 'fp8' else x.round_().clamp_(-127, 127).to(torch.int8)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(counts):
    return _int([0] + torch.tensor(counts).cumsum(0).tolist())


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c['dtype']]
    s = dict(case=c, dtype=dt)
    if c['op'] == 'rotary':
        T, Hq, Hk, D = c['tokens'], c['q_heads'], c['k_heads'], c['dim']
        qkv = torch.randn((T, Hq + 2 * Hk, D), device=DEV, generator=g).to(dt)       # as a projection leaves it
        s.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hk])
        if c['grad']:
            s['dq'] = torch.randn((T, Hq, D), device=DEV, generator=g).to(dt)
            s['dk'] = torch.randn((T, Hk, D), device=DEV, generator=g).to(dt)
            s['q'].requires_grad_(), s['k'].requires_grad_()
        at = torch.arange(T, device=DEV)
        if c['axes'] == 2:
            s['positions'] = torch.stack((at // COLS % ROWS, at % COLS), -1).int()
        else:
            s['positions'] = (at + torch.randint(0, c['context'] - T, (), device=DEV, generator=g)).int()
        f, m = _frequencies(c)
        # turns per position in units of 2^-40, which make the products with positions exact
        s['turns'] = torch.tensor([round(x / (2 * math.pi) * (1 << 40)) for x in f], dtype=torch.int64, device=DEV)
        s['factor'] = m
        if own:
            from blast3r_amd.rotary import Rotary
            s['rotary'] = Rotary(D, rotary_dim=c['part'], layout=c['layout'], axes=c['axes'],
                                 scaling=SCALING[c['scaled']], device=DEV)
        return s
    held, new = _sizes(c)
    H, D = c.get('heads') or c['k_heads'], c['dim']
    blocks = [max(1, -(-(h + n) // BLOCK)) for h, n in zip(held, new)]
    most, n_blocks = max(blocks), sum(blocks)
    order = torch.randperm(n_blocks, device=DEV, generator=g).int()                  # blocks lie in no order
    first = torch.tensor([0] + blocks, device=DEV).cumsum(0)[:-1]
    slot = torch.arange(most, device=DEV)
    s['pages'] = torch.where(slot < torch.tensor(blocks, device=DEV)[:, None],
                             order[(first[:, None] + slot).clamp_(max=n_blocks - 1)], 0).int()
    s['k'], s['v'] = _codes(g, (n_blocks, H, BLOCK, D), c['bits']), _codes(g, (n_blocks, H, D, BLOCK), c['bits'])
    u = torch.rand((n_blocks, H, 2), device=DEV, generator=g)
    s['scales'] = torch.exp2(torch.floor(u * 3) - 8) if c['bits'] == 'fp8' else 0.015 + 0.015 * u
    s['held'] = _int(held)
    s['lengths'] = _int([h + n for h, n in zip(held, new)])
    if c['op'] == 'write':
        s['new_k'] = torch.randn((sum(new), H, D), device=DEV, generator=g).to(dt)
        s['new_v'] = torch.randn((sum(new), H, D), device=DEV, generator=g).to(dt)
        s['offsets'], s['most_new'] = _offsets(new), max(new)
        back = [h % BLOCK + n if n else 0 for h, n in zip(held, new)]
        s['back_from'] = _int([h - h % BLOCK for h in held])
    else:
        back = held
        s['back_from'] = torch.zeros_like(s['held'])
    if c['op'] != 'attend':
        s['back'], s['n_back'], s['most_back'] = _offsets(back), sum(back), max(back)
    else:
        s['q'] = (2.0 * torch.randn((sum(new), c['q_heads'], D), device=DEV, generator=g)).to(dt)   # scores of a few units
        s['offsets'] = None if c['new_lo'] == c['new_hi'] else _offsets(new)
        s['counts'], s['rows'] = _int(new), _offsets(new)
        s['most_new'] = max(new)
    if own:
        from blast3r_amd.kv_cache import KVCache
        s['cache'] = KVCache.wrap(s['k'], s['v'], s['scales'])
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _pairs(x, c):
    """The two members of each pair, in 32 bits: (..., axes, pairs)."""
    r = x[..., :c['part']].float().unflatten(-1, (c['axes'], c['part'] // c['axes']))
    return r.chunk(2, -1) if c['layout'] == 'half' else (r[..., 0::2], r[..., 1::2])


def _rotate(x, cos, sin, c):
    a, b = _pairs(x, c)
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.cat(y, -1) if c['layout'] == 'half' else torch.stack(y, -1).flatten(-2)
    return torch.cat((y.flatten(-2), x[..., c['part']:].float()), -1).to(x.dtype)


def _plain_rotary(s):
    c = s['case']
    at = s['positions'].long().view(c['tokens'], 1, c['axes'], 1)
    turns = ((at * s['turns']) & ((1 << 40) - 1)).float() * 2.0 ** -40
    angle = (turns - (turns > 0.5).float()) * (2 * math.pi)
    cos, sin = angle.cos() * s['factor'], angle.sin() * s['factor']
    with torch.no_grad():
        out = dict(q=_rotate(s['q'], cos, sin, c), k=_rotate(s['k'], cos, sin, c))
        if c['grad']:
            out.update(dq=_rotate(s['dq'], cos, -sin, c), dk=_rotate(s['dk'], cos, -sin, c))
    return out


def _fit(amax, bits):
    """The factor of a block: the least power of two that brings fp8 codes to 448, amax / 127 for int8."""
    if bits == 'int8':
        return (amax / torch.full_like(amax, 127.0)).clamp(min=2.0 ** -60)     # a true division: torch takes 1 / 127 of a number
    m, e = torch.frexp(amax)                                     # amax = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e - 9 + (m > 0.875).int(), -60).clamp(min=-60))


def _encode(x, bits):
    return x.to(BITS['fp8']) if bits == 'fp8' else x.round().clamp(-127, 127).to(torch.int8)


def _plain_append(s):
    c = s['case']
    bits, S = c['bits'], c['seqs']
    touched = (BLOCK - 1 + s['most_new'] + BLOCK - 1) // BLOCK             # blocks that a sequence may touch
    held, offsets = s['held'].long(), s['offsets'].long()
    count = offsets[1:] - offsets[:-1]
    slot = (held // BLOCK)[:, None] + torch.arange(touched, device=DEV)
    at = slot[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)         # (S, touched, 64) token of each place
    fresh = (at >= held[:, None, None]) & (at < (held + count)[:, None, None])
    old = at < held[:, None, None]
    row = (offsets[:-1, None, None] + at - held[:, None, None]).clamp(0, max(0, s['new_k'].shape[0] - 1))
    # places without a new token go to an extra block that is thrown away
    spare = s['k'].shape[0]
    page = torch.where(fresh.any(-1), s['pages'].long().gather(1, slot.clamp(max=s['pages'].shape[1] - 1)), spare)
    for which, name, new in ((0, 'k', s['new_k']), (1, 'v', s['new_v'])):
        codes, scales = s[name], s['scales']
        x = new[row].float().masked_fill_(~fresh[..., None, None], 0.0)    # (S, touched, 64, H, D)
        scale = _fit(x.abs().amax((2, 4)), bits)                           # (S, touched, H)
        safe = page.clamp(max=spare - 1)
        before = scales[safe][..., which]
        scale = torch.where(old.any(-1)[..., None], torch.maximum(before, scale), scale)
        kept = codes.view(torch.uint8)[safe].view(codes.dtype).float()     # (S, touched, H, 64, D) or (.., D, 64)
        kept = kept.transpose(2, 3) if name == 'k' else kept.permute(0, 1, 4, 2, 3)
        ratio = torch.where(scale > before, before / scale, 1.0)
        again = _encode(kept * torch.where(old[..., None], ratio[:, :, None], 1.0)[..., None], bits)
        made = _encode(x * (1.0 / scale)[:, :, None, :, None], bits)
        both = torch.where(fresh[..., None, None], made.view(torch.uint8), again.view(torch.uint8))
        both = both.transpose(2, 3) if name == 'k' else both.permute(0, 1, 3, 4, 2)
        wide = torch.cat((codes.view(torch.uint8), torch.zeros_like(codes[:1]).view(torch.uint8)))
        wide[page] = both
        codes.view(torch.uint8).copy_(wide[:spare])
        tall = torch.cat((scales[..., which], torch.zeros_like(scales[:1, :, which])))
        tall[page] = scale
        scales[..., which] = tall[:spare]


def _plain_read(s):
    rows = torch.arange(s['n_back'], device=DEV)
    seq = torch.searchsorted(s['back'][1:].long(), rows, right=True)
    at = s['back_from'].long()[seq] + rows - s['back'].long()[seq]
    page, place = s['pages'].long()[seq, at // BLOCK], at % BLOCK
    kind, scale = s['k'].dtype, s['scales'][page]
    k = s['k'].view(torch.uint8)[page, :, place].view(kind).float() * scale[..., 0, None]
    v = s['v'].view(torch.uint8)[page, :, :, place].view(kind).float() * scale[..., 1, None]
    return k.to(s['dtype']), v.to(s['dtype'])


def _plain_attend(s):
    c = s['case']
    S, H, D, nq = c['seqs'], c['k_heads'], c['dim'], s['most_new']
    G = c['q_heads'] // H
    pages, kind, L = s['pages'].long(), s['k'].dtype, s['pages'].shape[1] * BLOCK
    scale = s['scales'][pages]                                             # (S, P, H, 2)
    k = s['k'].view(torch.uint8)[pages].view(kind).float().mul_(scale[..., 0, None, None])
    v = s['v'].view(torch.uint8)[pages].view(kind).float().mul_(scale[..., 1, None, None])
    k = k.permute(0, 2, 1, 3, 4).reshape(S, H, L, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(S, H, L, D)
    rows = s['rows'].long()
    i = torch.arange(nq, device=DEV)
    q = s['q'][(rows[:-1, None] + i).clamp(max=s['q'].shape[0] - 1)].float()           # (S, nq, Hq, D)
    q = q.view(S, nq, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * nq, D)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(S, H, G, nq, L)
    at = (s['lengths'] - s['counts']).long()[:, None, None] + i[:, None]               # (S, nq, 1)
    j = torch.arange(L, device=DEV)
    seen = (j < s['lengths'].long()[:, None, None]).expand(S, nq, L)
    if c['causal']:
        seen = seen & (j <= at)
    if c['window']:
        seen = seen & (j > at - c['window'])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, H, G * nq, L), v).view(S, H, G, nq, D)
    o = torch.where(total > 0, o / total, 0.0).to(s['dtype']).permute(0, 3, 1, 2, 4).reshape(S, nq, H * G, D)
    t = torch.arange(s['q'].shape[0], device=DEV)
    seq = torch.searchsorted(rows[1:], t, right=True)
    return o[seq, t - rows[seq]]


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    c = s['case']
    if c['op'] == 'rotary':
        if not own:
            return _plain_rotary(s)
        q, k = s['rotary'](s['positions'], s['q'], s['k'])
        if not c['grad']:
            return dict(q=q, k=k)
        dq, dk = torch.autograd.grad((q, k), (s['q'], s['k']), (s['dq'], s['dk']))
        return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)
    if c['op'] == 'attend':
        if not own:
            return dict(o=_plain_attend(s))
        return dict(o=s['cache'].attend(s['q'], s['pages'], s['lengths'], offsets=s['offsets'], max_new=s['most_new'],
                                        causal=c['causal'], window=c['window'] or None))
    out = {}
    if c['op'] == 'write':
        if own:
            s['cache'].append(s['new_k'], s['new_v'], s['pages'], s['held'], offsets=s['offsets'], max_new=s['most_new'])
        else:
            _plain_append(s)
        out['scales'] = s['scales']
    if own:
        out['k'], out['v'] = s['cache'].read(s['pages'], s['back_from'], s['back'], s['n_back'], max_count=s['most_back'],
                                             dtype=s['dtype'])
    else:
        out['k'], out['v'] = _plain_read(s)
    return out


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_rotary(s):
    c = s['case']
    f, m = _frequencies(c)
    f = torch.tensor(f, dtype=torch.float64, device=DEV)
    angle = (s['positions'].double().view(c['tokens'], c['axes'], 1) * f)[:, None]           # (T, 1, axes, pairs)
    half = f.numel()
    first = torch.arange(half, device=DEV) * (1 if c['layout'] == 'half' else 2)
    second = first + (half if c['layout'] == 'half' else 1)

    def turn(x, way):
        y = x.detach().double().clone()
        z = y[..., :c['part']].unflatten(-1, (c['axes'], 2 * half))                          # a view of y
        a, b = z[..., first].clone(), z[..., second].clone()
        z[..., first] = m * (a * torch.cos(angle) - b * torch.sin(way * angle))
        z[..., second] = m * (a * torch.sin(way * angle) + b * torch.cos(angle))
        return y

    out = dict(q=turn(s['q'], 1), k=turn(s['k'], 1))
    if c['grad']:
        out.update(dq=turn(s['dq'], -1), dk=turn(s['dk'], -1))
    return out


def _nearest_code(x, bits):
    """x (64 bits) rounded to the nearest code, ties to even: steps of 2^(e-3) from 2^-6 on, 2^-9 below, or whole numbers."""
    if bits == 'int8':
        return torch.round(x).clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    """Codes (64 bits) and factors after the call, block by block; each product that the definition rounds to 32 bits is."""
    c, bits = s['case'], s['case']['bits']
    held, new = _sizes(c)
    k = s['k'].float().double()
    v = s['v'].float().double().transpose(2, 3).contiguous()                                 # (blocks, H, 64, D)
    scales = s['scales'].double()
    pages, row = s['pages'].cpu().tolist(), 0

    def single(t):
        return t.float().double()

    for q, (h, n) in enumerate(zip(held, new)):
        for at in range(h - h % BLOCK, h + n, BLOCK) if n else ():
            lo, hi = max(at, h), min(at + BLOCK, h + n)
            p = pages[q][at // BLOCK]
            for w, (codes, src) in enumerate(((k, s['new_k']), (v, s['new_v']))):
                x = src[row + lo - h:row + hi - h].double().transpose(0, 1)                  # (H, tokens, D)
                amax = x.abs().amax((1, 2))
                if bits == 'int8':
                    fit = single(amax / 127).clamp(min=2.0 ** -60)
                else:
                    fit = torch.exp2(torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -60))))
                if lo > at:
                    before = scales[p, :, w].clone()
                    fit = torch.maximum(fit, before)
                    ratio = single(before / fit)[:, None, None]
                    part = codes[p, :, :lo - at]
                    codes[p, :, :lo - at] = torch.where(ratio < 1, _nearest_code(single(part * ratio), bits), part)
                scales[p, :, w] = fit
                codes[p, :, lo - at:hi - at] = _nearest_code(single(x * single(1 / fit)[:, None, None]), bits)
        row += n
    return k, v, scales


def _exact_read(s, k, v, scales):
    count = (s['back'][1:] - s['back'][:-1]).cpu().tolist()
    outs = ([], [])
    for q, (start, n) in enumerate(zip(s['back_from'].cpu().tolist(), count)):
        at = torch.arange(start, start + n, device=DEV)
        p, i = s['pages'][q].long()[at // BLOCK], at % BLOCK
        outs[0].append(k[p, :, i] * scales[p][..., 0:1])
        outs[1].append(v[p, :, i] * scales[p][..., 1:2])
    return torch.cat(outs[0]), torch.cat(outs[1])


def _exact_attend(s):
    c = s['case']
    held, new = _sizes(c)
    G, row, out = c['q_heads'] // c['k_heads'], 0, torch.zeros_like(s['q'], dtype=torch.float64)
    for q, (h, n) in enumerate(zip(held, new)):
        if n == 0:
            continue
        pages = s['pages'][q, :-(-(h + n) // BLOCK)].long()
        at = h + torch.arange(n, device=DEV)[:, None]
        j = torch.arange(h + n, device=DEV)
        hide = torch.zeros((n, h + n), dtype=torch.bool, device=DEV)
        if c['causal']:
            hide |= j > at
        if c['window']:
            hide |= j <= at - c['window']
        for head in range(c['k_heads']):
            sc = s['scales'][pages, head].double()
            k = (s['k'].view(torch.uint8)[pages, head].view(s['k'].dtype).double() * sc[:, 0, None, None])
            v = (s['v'].view(torch.uint8)[pages, head].view(s['v'].dtype).double() * sc[:, 1, None, None])
            k, v = k.flatten(0, 1)[:h + n], v.transpose(1, 2).flatten(0, 1)[:h + n]
            x = s['q'][row:row + n, head * G:(head + 1) * G].double().transpose(0, 1).reshape(G * n, -1)
            z = (x @ k.t() / math.sqrt(c['dim'])).masked_fill(hide.repeat(G, 1), -math.inf)
            z = torch.softmax(z, -1).nan_to_num(0.0) @ v
            out[row:row + n, head * G:(head + 1) * G] = z.view(G, n, -1).transpose(0, 1)
        row += n
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c['op'] == 'rotary':
        return _exact_rotary(s)
    if c['op'] == 'attend':
        return dict(o=_exact_attend(s))
    out = {}
    if c['op'] == 'write':
        k, v, scales = _exact_append(s)
        out['scales'] = scales
    else:
        k, v, scales = s['k'].float().double(), s['v'].float().double().transpose(2, 3), s['scales'].double()
    out['k'], out['v'] = _exact_read(s, k, v, scales)
    return out
