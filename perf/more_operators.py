"""The timed cases of what the 8-bit key/value cache offers beside writing, reading and plain attention: attention with
formed scores and masks, attention of a batch whose sequences begin with the same blocks, and the pages of the cache.

  attend  softmax(f(scale q.k)) v over the cached tokens of each sequence; the score z of a row at position p and a token j
          becomes cap tanh(z / cap), then less slope |p - j|; a row sees the tokens below its sequence's ``prefix``, and of
          the others those from its ``since`` and below its ``until``, causal and in the window.  With ``shared`` the first
          blocks of every list are the same.
  pages   block lists on the device: ``fork`` (children hold their parents' blocks), ``grow`` (blocks for new tokens, an own
          copy of a last block that others hold too), ``trim`` (tokens given back), ``compact`` (blocks moved together).
          Lowest free block first; sequences in their order.

A frame of 512 x 384 pixels in patches of 16 x 16 is 768 tokens, 12 blocks of 64.  With ``own`` false every operator is
computed in its plain form (torch, 32 bits).  Cache layout: ``k`` (n_blocks, heads, 64, dim), ``v`` (n_blocks, heads, dim,
64), one byte each, ``scales`` (n_blocks, heads, 2) in fp32; ``pages`` (n_seqs, most blocks), -1 where there is none.
"""
import math
import random

import torch

own = False

BLOCK = 64
FRAME = 768
DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
BITS = {'fp8': torch.float8_e4m3fn, 'int8': torch.int8}


# ------------------------------------------------------------------------------------------------ cases

def _attend(name, seqs, new, held, q_heads, k_heads, dim, bits, dtype='bf16', causal=True, window=0, cap=0.0, slopes=False,
            prefix=0, mask='none', spans=(0, 0), shared=0, salt=1):
    """new: (least, most) queries of a sequence; held: its own tokens before them, after ``shared`` blocks that all
    sequences begin with.  window, cap, prefix 0: none.  mask: 'documents' (a row sees its own document only; documents
    of ``spans`` tokens) or 'frames' (a row sees its whole frame and what is before it)."""
    c = dict(op='attend', seqs=seqs, new_lo=new[0], new_hi=new[1], held_lo=held[0], held_hi=held[1], q_heads=q_heads,
             k_heads=k_heads, dim=dim, bits=bits, dtype=dtype, causal=causal, window=window, cap=cap, slopes=slopes,
             prefix=prefix, mask=mask, span_lo=spans[0], span_hi=spans[1], shared=shared, salt=salt)
    return dict(c, name=name) if name else c


def _pages(name, op, seqs, held, new, heads, dim, bits, children=1, spare=0, salt=1):
    """held: (least, most) tokens of a sequence; new: most tokens it grows by; children: forks of each sequence; spare:
    free blocks beyond those that the call may need."""
    c = dict(op=op, seqs=seqs, held_lo=held[0], held_hi=held[1], new=new, heads=heads, dim=dim, bits=bits, children=children,
             spare=spare, salt=salt)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a query over the first frame, its scores capped: a launch
        _attend('capped token', 1, (1, 1), (776, 776), 16, 16, 64, 'fp8', cap=50.0),
        # a step of 48 sequences of many lengths with scores that fall with the distance, four query heads to a key head
        _attend('sloped tokens', 48, (1, 1), (0, 8191), 32, 8, 128, 'int8', slopes=True),
        # a step of 16 long sequences that see their first 64 tokens and the last 4096
        _attend('window after prefix', 16, (1, 1), (65000, 65535), 32, 8, 128, 'fp8', window=4096, prefix=64),
        # 8 frames at once after 8 kept ones: a token sees the frames up to its own
        _attend('frames', 1, (8 * FRAME, 8 * FRAME), (8 * FRAME, 8 * FRAME), 16, 16, 64, 'fp8', causal=False, mask='frames',
                spans=(FRAME, FRAME)),
        # documents of many lengths packed into one prompt
        _attend('documents', 1, (8192, 8192), (0, 0), 32, 8, 128, 'int8', dtype='fp16', mask='documents', spans=(50, 2000)),
        # a chunk of a long prompt for two sequences, scores capped
        _attend('capped chunk', 2, (2048, 2048), (14336, 14336), 32, 8, 128, 'int8', cap=30.0),
        # drafted tokens of 8 samples of a short prompt
        _attend('shared drafts', 8, (5, 5), (1, 40), 16, 16, 64, 'fp8', shared=16),
        # a step of 64 samples of one long prompt
        _attend('shared tokens', 64, (1, 1), (1, 512), 32, 8, 128, 'int8', shared=256),
        # six frames that are matched to the same 20 kept ones
        _attend('shared frames', 6, (FRAME, FRAME), (0, 0), 16, 16, 64, 'fp8', causal=False, shared=20 * FRAME // BLOCK),
        # 64 sequences give back the blocks of drafted tokens that were refused and take those of the next ones
        _pages('drafts undone', 'draft', 64, (1, 8192), 100, 8, 128, 'int8', spare=500),
        # 8 samples each of 16 prompts: lists forked, the last blocks copied, room for a token
        _pages('samples', 'fork', 16, (1, 8192), 1, 8, 128, 'int8', children=8, spare=1000),
        # a cache of many ended sequences moved together
        _pages('moved together', 'compact', 64, (1, 4096), 0, 16, 64, 'fp8', spare=3000),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    op = rng.choice(['attend', 'attend', 'shared', 'draft', 'fork', 'compact'])
    bits = rng.choice(['fp8', 'int8'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16'])
    salt = rng.randrange(1 << 20)
    dim = rng.choice([32, 64, 64, 96, 128, 128, 256])
    if op in ('draft', 'fork', 'compact'):
        heads = rng.choice([1, 2, 5, 8, 16])
        most = 500_000_000 // (2 * heads * dim)                    # tokens that the cache holds
        kids = rng.choice([1, 2, 5, 8]) if op == 'fork' else 1
        seqs = _log(rng, 1, 64)
        held = _log(rng, 1, min(8192, max(1, most // (2 * seqs * kids))))
        return _pages(None, op, seqs, (rng.choice([0, held]), held), rng.choice([1, 5, 64, 100, 700]), heads, dim, bits, kids,
                      _log(rng, 1, min(3000, most // BLOCK // 2)), salt)
    group = rng.choice([1, 2, 4, 8])
    heads = rng.choice([2, 5, 8])
    seqs = _log(rng, 1, 32)
    shared = _log(rng, 1, 256) if op == 'shared' else 0
    causal = rng.random() < 0.7
    window = rng.choice([0, 0, 0, 100, 1000])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    prefix = rng.choice([0, 0, 1, 70, 500])
    slopes = rng.random() < 0.3
    mask = rng.choice(['none', 'none', 'documents', 'frames'])
    spans = (rng.choice([1, 30]), _log(rng, 40, 2000))
    if rng.random() < 0.5:           # single tokens, or a few drafted ones
        new = rng.choice([1, 1, 2, 5])
        held = _log(rng, 1, min(100_000, 100_000_000 // (seqs * heads * dim)))
    else:                            # frames and chunks
        new = _log(rng, 6, 2048)
        held = _log(rng, 1, 16384)
    most = 200_000_000_000 // (4 * dim)
    while seqs > 1 and seqs * heads * group * new * (64 * shared + held + new) > most:
        seqs //= 2
    while held > 1 and seqs * heads * group * new * (64 * shared + held + new) > most:
        held //= 2
    while new > 6 and seqs * heads * group * new * (64 * shared + held + new) > most:
        new //= 2
    return _attend(None, seqs, (rng.choice([1, new]), new), (rng.choice([0, held]), held), heads * group, heads, dim, bits, dtype,
                   causal, window, cap, slopes, prefix, mask, spans, shared, salt)


def _some(n, lo, hi, salt):
    """n numbers from lo to hi, the largest among them."""
    r = random.Random(salt)
    got = [r.randint(lo, hi) for _ in range(n)]
    got[r.randrange(n)] = hi
    return got


def _sizes(c):
    """(tokens before the call, new tokens) of each sequence."""
    held = [BLOCK * c['shared'] + h for h in _some(c['seqs'], c['held_lo'], c['held_hi'], c['salt'])]
    return held, _some(c['seqs'], c['new_lo'], c['new_hi'], c['salt'] + 1)


def _spans(c, s, held, new):
    """(first token, end) of the document or frame of each of a sequence's new tokens."""
    r = random.Random(c['salt'] * 1009 + s)
    got, at = [], 0
    while at < held + new:
        end = at + r.randint(c['span_lo'], c['span_hi'])
        got += [(at, end)] * max(0, min(end, held + new) - max(at, held))
        at = end
    return got


def _seen(c, s, held, new):
    """Of each new token of sequence s: (prefix, first, end): it sees the tokens below prefix and from first to end."""
    n = held + new
    spans = _spans(c, s, held, new) if c['mask'] != 'none' else None
    got = []
    for i in range(new):
        p = held + i
        lo = max(0, p - c['window'] + 1) if c['window'] else 0
        hi = p + 1 if c['causal'] else n
        if c['mask'] == 'documents':
            lo = max(lo, spans[i][0])
        if c['mask'] == 'frames':
            hi = min(hi, spans[i][1])
        got.append((min(c['prefix'], n), lo, hi))
    return got


def _drop(c):
    """Which sequences have ended, of the compacted ones."""
    r = random.Random(c['salt'] + 7)
    return [r.random() < 0.45 for _ in range(c['seqs'])]


def work(c):
    if c['op'] == 'attend':
        held, new = _sizes(c)
        pairs = keys = 0
        first = BLOCK * c['shared']
        once = set()
        for s, (h, n) in enumerate(zip(held, new)):
            at = 0                                                 # tokens below it are counted
            rows = _seen(c, s, h, n)
            spans = sorted({(0, p) for p, _, _ in rows} | {(lo, hi) for _, lo, hi in rows})
            for lo, hi in spans:
                if first and lo < first:
                    once.add((lo, min(hi, first)))
                lo = max(lo, at, first)
                keys += max(0, hi - lo)
                at = max(at, hi)
            pairs += sum(max(0, hi - lo) + p - max(0, min(p, hi) - lo) if hi > lo else p for p, lo, hi in rows)
        at = 0
        for lo, hi in sorted(once):
            keys += max(0, hi - max(lo, at))
            at = max(at, hi)
        rows = sum(new)
        return dict(bytes=2 * keys * c['k_heads'] * c['dim'] + 4 * rows * c['q_heads'] * c['dim'], flops=4 * c['dim'] * c['q_heads'] * pairs)
    held = _some(c['seqs'], c['held_lo'], c['held_hi'], c['salt'])
    block = 2 * c['heads'] * BLOCK * c['dim'] + 8 * c['heads']
    lists = [-(-h // BLOCK) for h in held]
    if c['op'] == 'fork':            # parents' lists read, children's written, counts changed, open blocks copied
        opened = sum(h % BLOCK != 0 for h in held) * c['children']
        return dict(bytes=4 * sum(lists) * (1 + 3 * c['children']) + 2 * block * opened, flops=0)
    if c['op'] == 'draft':           # entries and counts of the new blocks, read and written twice
        return dict(bytes=sum(16 * (-(-(h + c['new']) // BLOCK) - b) + 16 for h, b in zip(held, lists)), flops=0)
    kept = sum(b for b, gone in zip(lists, _drop(c)) if not gone)
    n = sum(lists) + c['spare']
    return dict(bytes=4 * (2 * kept + n) + 2 * block * (kept * (n - kept) // n), flops=0)


# ------------------------------------------------------------------------------------------------ inputs

def _codes(gen, shape, bits):
    x = torch.randn(shape, device=DEV, generator=gen) * (100.0 if bits == 'fp8' else 40.0)
    return x.clamp_(-448, 448).to(BITS['fp8']) if bits == 'fp8' else x.round_().clamp_(-127, 127).to(torch.int8)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _lists(order, first, counts, most):
    """(n, most) block lists: counts[i] blocks of `order` from first[i] on, -1 after them."""
    slot = torch.arange(most, device=DEV)
    first, counts = torch.tensor(first, device=DEV), torch.tensor(counts, device=DEV)
    at = (first[:, None] + slot).clamp_(max=order.numel() - 1)
    return torch.where(slot < counts[:, None], order[at], -1).int().contiguous()


def _before(counts):
    return torch.tensor([0] + counts).cumsum(0).tolist()


def _cache(c, g, n_blocks, heads):
    k, v = _codes(g, (n_blocks, heads, BLOCK, c['dim']), c['bits']), _codes(g, (n_blocks, heads, c['dim'], BLOCK), c['bits'])
    u = torch.rand((n_blocks, heads, 2), device=DEV, generator=g)
    return dict(k=k, v=v, scales=torch.exp2(torch.floor(u * 3) - 8) if c['bits'] == 'fp8' else 0.015 + 0.015 * u)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c['op'] == 'attend':
        held, new = _sizes(c)
        blocks = [max(1, -(-(h + n) // BLOCK)) for h, n in zip(held, new)]
        own_blocks = [b - c['shared'] for b in blocks]
        n_blocks = c['shared'] + sum(own_blocks)
        order = torch.randperm(n_blocks, device=DEV, generator=g).int()              # blocks lie in no order
        s['pages'] = _lists(order, [c['shared'] + x for x in _before(own_blocks)[:-1]], own_blocks, max(own_blocks))
        if c['shared']:
            s['pages'] = torch.cat((order[:c['shared']].expand(c['seqs'], -1), s['pages']), 1).contiguous()
        s.update(_cache(c, g, n_blocks, c['k_heads']))
        s['q'] = (2.0 * torch.randn((sum(new), c['q_heads'], c['dim']), device=DEV, generator=g)).to(DTYPES[c['dtype']])
        s['lengths'], s['counts'], s['rows'] = _int([h + n for h, n in zip(held, new)]), _int(new), _int(_before(new))
        s['offsets'] = None if c['new_lo'] == c['new_hi'] else s['rows']
        s['most_new'] = max(new)
        heads = torch.arange(1, c['q_heads'] + 1, device=DEV)
        s['slopes'] = torch.exp2(-8.0 * heads / c['q_heads']).float() if c['slopes'] else None
        s['prefix'] = _int([c['prefix']] * c['seqs']) if c['prefix'] else None
        spans = [x for i, (h, n) in enumerate(zip(held, new)) for x in _spans(c, i, h, n)] if c['mask'] != 'none' else []
        s['since'] = _int([x[0] for x in spans]) if c['mask'] == 'documents' else None
        s['until'] = _int([x[1] for x in spans]) if c['mask'] == 'frames' else None
    else:
        held = _some(c['seqs'], c['held_lo'], c['held_hi'], c['salt'])
        lists = [-(-h // BLOCK) for h in held]
        grown = [-(-(h + c['new']) // BLOCK) for h in held]
        more = {'fork': c['children'] * (c['new'] // BLOCK + 2) * c['seqs'], 'draft': sum(grown) - sum(lists), 'compact': 0}[c['op']]
        n_blocks = sum(lists) + more + c['spare']
        order = torch.randperm(n_blocks, device=DEV, generator=g).int()
        if c['op'] == 'compact':
            lists = [0 if gone else b for b, gone in zip(lists, _drop(c))]
        s['pages'] = _lists(order, _before(lists)[:-1], lists, max(grown + [1]))
        s['lengths'] = _int(held)
        s['used'] = torch.zeros(n_blocks, dtype=torch.int32, device=DEV)             # lists that hold a block
        s['used'][order[:sum(lists)].long()] = 1
        s.update(_cache(c, g, n_blocks, c['heads']))
        if c['op'] == 'draft':
            s['new'] = torch.randint(1, c['new'] + 1, (c['seqs'],), device=DEV, generator=g).int()
        if c['op'] == 'fork':
            n = c['seqs'] * c['children']
            s['parents'] = torch.arange(c['seqs'], device=DEV).repeat(c['children']).int()
            s['children'] = torch.randperm(n, device=DEV, generator=g).int()
            s['child_pages'] = torch.full((n, s['pages'].shape[1]), -1, dtype=torch.int32, device=DEV)
            s['child_lengths'] = torch.zeros(n, dtype=torch.int32, device=DEV)
        if c['op'] == 'compact':
            s['table'] = s['pages'].clone()
    if own:
        from blast3r_amd.kv_cache import KVCache
        s['cache'] = KVCache.wrap(s['k'], s['v'], s['scales'])
        if c['op'] != 'attend':
            from blast3r_amd.kv_pool import BlockPool
            s['pool'] = BlockPool(s['used'].numel(), device=DEV)
            s['pool'].count(s['pages'])
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_attend(s):
    c = s['case']
    S, H, D, nq = c['seqs'], c['k_heads'], c['dim'], s['most_new']
    G = c['q_heads'] // H
    pages, kind, L = s['pages'].long().clamp(min=0), s['k'].dtype, s['pages'].shape[1] * BLOCK
    scale = s['scales'][pages]                                             # (S, P, H, 2)
    k = s['k'].view(torch.uint8)[pages].view(kind).float().mul_(scale[..., 0, None, None])
    v = s['v'].view(torch.uint8)[pages].view(kind).float().mul_(scale[..., 1, None, None])
    k = k.permute(0, 2, 1, 3, 4).reshape(S, H, L, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(S, H, L, D)
    rows = s['rows'].long()
    i = torch.arange(nq, device=DEV)
    row = (rows[:-1, None] + i).clamp(max=s['q'].shape[0] - 1)             # (S, nq)
    q = s['q'][row].float().view(S, nq, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * nq, D)
    z = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(S, H, G, nq, L)
    if c['cap']:
        z.div_(c['cap']).tanh_().mul_(c['cap'])
    at = (s['lengths'] - s['counts']).long()[:, None, None] + i[:, None]               # (S, nq, 1)
    j = torch.arange(L, device=DEV)
    if c['slopes']:
        z.sub_(s['slopes'].view(H, G, 1, 1) * (at - j).abs()[:, None, None].float())
    seen = (j < s['lengths'].long()[:, None, None]).expand(S, nq, L)
    if c['causal']:
        seen = seen & (j <= at)
    if c['window']:
        seen = seen & (j > at - c['window'])
    if s['since'] is not None:
        seen = seen & (j >= s['since'].long()[row][..., None])
    if s['until'] is not None:
        seen = seen & (j < s['until'].long()[row][..., None])
    if s['prefix'] is not None:
        seen = seen | (j < torch.minimum(s['prefix'], s['lengths']).long()[:, None, None])
    z.masked_fill_(~seen[:, None, None], -math.inf)
    z.sub_(z.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(S, H, G * nq, L), v).view(S, H, G, nq, D)
    o = torch.where(total > 0, o / total, 0.0).to(s['q'].dtype).permute(0, 3, 1, 2, 4).reshape(S, nq, H * G, D)
    t = torch.arange(s['q'].shape[0], device=DEV)
    seq = torch.searchsorted(rows[1:], t, right=True)
    return o[seq, t - rows[seq]]


def _dense(values, picked, size):
    """The picked values in their order in the first places of (size,) int32, -1 after them."""
    at = torch.where(picked, picked.cumsum(0) - 1, size)
    return torch.full((size + 1,), -1, dtype=torch.int32, device=DEV).scatter_(0, at, values.int())[:size]


def _add(used, blocks, there, n):
    used.add_(torch.zeros_like(used).scatter_add_(0, blocks.clamp(min=0).long().flatten(), (there.flatten() * n).int()))


def _plain_grow(used, pages, lengths, new):
    S, P = pages.shape
    n = used.numel()
    slot, seq = torch.arange(P, device=DEV), torch.arange(S, device=DEV)
    lengths, new = lengths.long(), new.long()
    filled, end = (lengths + BLOCK - 1) // BLOCK, (lengths + new + BLOCK - 1) // BLOCK
    last = (lengths // BLOCK).clamp(max=P - 1)
    page = pages.gather(1, last[:, None])[:, 0].long()
    p = page.clamp(min=0)
    several = (lengths % BLOCK > 0) & (new > 0) & (page >= 0) & (used[p] > 1)      # an open block that other lists hold
    wanted = torch.zeros(n, dtype=torch.int32, device=DEV).scatter_add_(0, p, several.int())
    final = torch.full((n,), -1, device=DEV).scatter_reduce_(0, p, torch.where(several, seq, -1), 'amax')
    copied = several & ~((wanted[p] == used[p]) & (final[p] == seq))               # the last of its holders keeps it
    free = used == 0
    blocks = _dense(torch.arange(n, device=DEV), free, n)
    want = (slot >= filled[:, None]) & (slot < end[:, None]) & (pages < 0) | copied[:, None] & (slot == last[:, None])
    rank = (want.flatten().cumsum(0) - 1).view(S, P)
    got = torch.where(rank < n, blocks[rank.clamp(0, n - 1)], -1)
    _add(used, p, copied, -1)
    _add(used, got, want & (got >= 0), 1)
    pages.copy_(torch.where(want, got, pages))
    to = pages.gather(1, last[:, None])[:, 0]
    done = copied & (to >= 0)
    return _dense(page, done, S), _dense(to, done, S), done.sum().int().view(1)


def _plain_fork(used, pages, lengths, parents, children, child_pages, child_lengths):
    parents, children = parents.long(), children.long()
    old = child_pages[children]
    _add(used, old, old >= 0, -1)
    rows = torch.where(torch.arange(pages.shape[1], device=DEV) < ((lengths[parents] + BLOCK - 1) // BLOCK)[:, None], pages[parents], -1)
    _add(used, rows, rows >= 0, 1)
    child_pages[children] = rows
    child_lengths[children] = lengths[parents]


def _plain_trim(used, pages, last):
    gone = (torch.arange(pages.shape[1], device=DEV) >= ((last + BLOCK - 1) // BLOCK)[:, None]) & (pages >= 0)
    _add(used, pages, gone, -1)
    pages.masked_fill_(gone, -1)


def _plain_compact(used, pages):
    n = used.numel()
    held = used > 0
    blocks = torch.arange(n, device=DEV)
    holes, tops = _dense(blocks, ~held, n), _dense(blocks.flip(0), held.flip(0), n)      # lowest first, highest first
    pair = (holes >= 0) & (holes < tops)
    src, dst = torch.where(pair, tops, -1)[:n // 2], torch.where(pair, holes, -1)[:n // 2]
    to = torch.cat((blocks, blocks[:1])).int().scatter_(0, torch.where(src >= 0, src, n).long(), dst)[:n]
    pages.copy_(torch.where(pages >= 0, to[pages.clamp(min=0).long()], -1))
    used.copy_(torch.zeros_like(used).scatter_add_(0, to.long(), used))
    return src, dst, pair.sum().int().view(1)


def _plain_copy(s, src, dst):
    same = torch.where(src[:1] >= 0, src[:1], 0)                           # in the place of no pair: a block onto itself
    src, dst = torch.where(src >= 0, src, same).long(), torch.where(dst >= 0, dst, same).long()
    s['k'].view(torch.uint8)[dst] = s['k'].view(torch.uint8)[src]
    s['v'].view(torch.uint8)[dst] = s['v'].view(torch.uint8)[src]
    s['scales'][dst] = s['scales'][src]


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    c = s['case']
    if c['op'] == 'attend':
        if not own:
            return dict(o=_plain_attend(s))
        return dict(o=s['cache'].attend(s['q'], s['pages'], s['lengths'], offsets=s['offsets'], max_new=s['most_new'],
                                        causal=c['causal'], window=c['window'] or None, cap=c['cap'] or None, slopes=s['slopes'],
                                        prefix=s['prefix'], since=s['since'], until=s['until'], shared=c['shared']))
    if c['op'] == 'draft':           # what earlier passes took is given back
        if own:
            s['pool'].trim(s['pages'], last=s['lengths'])
            src, dst, n = s['pool'].grow(s['pages'], s['lengths'], s['new'], max_new=c['new'])
        else:
            _plain_trim(s['used'], s['pages'], s['lengths'])
            src, dst, n = _plain_grow(s['used'], s['pages'], s['lengths'], s['new'])
        return dict(pages=s['pages'], used=s['pool'].counts if own else s['used'], src=src, dst=dst, n=n)
    out = dict(k=s['k'], v=s['v'], scales=s['scales'])
    if c['op'] == 'fork':            # the children of an earlier pass give back what they held
        pages, lengths = s['child_pages'], s['child_lengths']
        if own:
            s['pool'].fork(s['pages'], s['lengths'], s['parents'], s['children'], into=(pages, lengths))
            src, dst, n = s['pool'].grow(pages, lengths, c['new'])
        else:
            _plain_fork(s['used'], s['pages'], s['lengths'], s['parents'], s['children'], pages, lengths)
            src, dst, n = _plain_grow(s['used'], pages, lengths, torch.full_like(lengths, c['new']))
        out['lengths'] = lengths
    else:                            # lists as they were saved, counted and moved together
        pages = s['pages'].copy_(s['table'])
        if own:
            s['pool'].count(pages)
            src, dst, n = s['pool'].compact(pages)
        else:
            s['used'].zero_()
            _add(s['used'], pages, pages >= 0, 1)
            src, dst, n = _plain_compact(s['used'], pages)
    if own:
        s['cache'].copy(src, dst, n)
    else:
        _plain_copy(s, src, dst)
    return dict(out, pages=pages, used=s['pool'].counts if own else s['used'], src=src, dst=dst, n=n)


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_attend(s):
    c = s['case']
    held, new = _sizes(c)
    G, row, out = c['q_heads'] // c['k_heads'], 0, torch.zeros_like(s['q'], dtype=torch.float64)
    for q, (h, n) in enumerate(zip(held, new)):
        if n == 0:
            continue
        pages = s['pages'][q, :-(-(h + n) // BLOCK)].long()
        rows = torch.tensor(_seen(c, q, h, n), device=DEV)[:, :, None]
        j = torch.arange(h + n, device=DEV)
        hide = (j >= rows[:, 0]) & ((j < rows[:, 1]) | (j >= rows[:, 2]))
        far = (h + torch.arange(n, device=DEV)[:, None] - j).abs().double()
        for head in range(c['k_heads']):
            sc = s['scales'][pages, head].double()
            k = (s['k'].view(torch.uint8)[pages, head].view(s['k'].dtype).double() * sc[:, 0, None, None])
            v = (s['v'].view(torch.uint8)[pages, head].view(s['v'].dtype).double() * sc[:, 1, None, None])
            k, v = k.flatten(0, 1)[:h + n], v.transpose(1, 2).flatten(0, 1)[:h + n]
            for one in range(head * G, (head + 1) * G):
                z = s['q'][row:row + n, one].double() @ k.t() / math.sqrt(c['dim'])
                if c['cap']:
                    z = c['cap'] * torch.tanh(z / c['cap'])
                if c['slopes']:
                    z = z - 2.0 ** (-8.0 * (one + 1) / c['q_heads']) * far
                z = torch.softmax(z.masked_fill(hide, -math.inf), -1).nan_to_num(0.0)
                out[row:row + n, one] = z @ v
        row += n
    return out


def _exact_grow(used, pages, lengths, new):
    """One sequence after the other: the copies that have to be made."""
    free = [b for b, u in enumerate(used) if u == 0][::-1]
    moves = []
    for row, h, n in zip(pages, lengths, new):
        if n > 0 and h % BLOCK and row[h // BLOCK] >= 0 and used[row[h // BLOCK]] > 1:
            old, to = row[h // BLOCK], free.pop() if free else -1
            used[old] -= 1
            row[h // BLOCK] = to
            if to >= 0:
                used[to] = 1
                moves.append((old, to))
        for b in range(-(-h // BLOCK), min(len(row), -(-(h + n) // BLOCK))):
            if row[b] < 0 and free:
                row[b] = free.pop()
                used[row[b]] = 1
    return moves


def _exact_pages(s):
    c = s['case']
    used, pages, lengths = s['used'].tolist(), s['pages'].tolist(), s['lengths'].tolist()
    out = {}
    size = c['seqs']
    if c['op'] == 'draft':
        moves = _exact_grow(used, pages, lengths, s['new'].tolist())
    elif c['op'] == 'fork':
        kids, size = [None] * s['children'].numel(), s['children'].numel()
        far = [0] * size
        for p, k in zip(s['parents'].tolist(), s['children'].tolist()):
            kids[k] = [b if i * BLOCK < lengths[p] else -1 for i, b in enumerate(pages[p])]
            far[k] = lengths[p]
            for b in kids[k]:
                if b >= 0:
                    used[b] += 1
        pages = kids
        moves = _exact_grow(used, pages, far, [c['new']] * size)
        out['lengths'] = _int(far)
    else:
        moves, size, lo, hi = [], len(used) // 2, 0, len(used) - 1
        while True:
            while lo < len(used) and used[lo]:
                lo += 1
            while hi >= 0 and not used[hi]:
                hi -= 1
            if lo >= hi:
                break
            moves.append((hi, lo))
            used[lo], used[hi] = used[hi], 0
        to = dict(moves)
        pages = [[to.get(b, b) for b in row] for row in pages]
    out.update(pages=_int(pages), used=_int(used), n=_int([len(moves)]))
    for i, name in enumerate(('src', 'dst')):
        out[name] = _int([m[i] for m in moves] + [-1] * (size - len(moves)))
    if c['op'] != 'draft':
        for name in ('k', 'v', 'scales'):
            t = s[name].view(torch.uint8) if name != 'scales' else s[name]
            for a, b in moves:
                t[b] = t[a]
            out[name] = s[name].double() if s[name].is_floating_point() else s[name]
    return out


def exact(c, seed):
    s = prepare(c, seed)
    return dict(o=_exact_attend(s)) if c['op'] == 'attend' else _exact_pages(s)
