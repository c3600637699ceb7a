"""A key/value cache in 8 bits and attention over it, on the device (``ba_kv_*``, libba_hip.so).

What a transformer keeps of the tokens it has seen: online reconstruction keeps the tokens of earlier frames and looks
from a new frame at those of the retrieved ones, a sequence model keeps its context.  Tokens lie in blocks of 64 of a
head, with one factor for a block's keys and one for its values; a sequence is a list of blocks (``pages``), so a frame
of 768 tokens is 12 blocks, and which frames a query looks at is a choice of blocks::

    cache = KVCache(n_blocks, heads, head_dim, torch.float8_e4m3fn)
    cache.append(k, v, pages, lengths)                     # (n_tokens, heads, head_dim) each
    lengths += n
    o = cache.attend(q, pages, lengths, causal=False)      # (n_tokens, q_heads, head_dim)

Sequences of a call have the same number of rows each, or ``offsets`` (n_seqs + 1,) int32 gives their first rows; then
``max_new`` (a host number; default: all rows) bounds the rows of one of them, and a close bound saves launches' empty
workgroups.  Lengths, offsets and pages are device tensors, never read by the host: nothing here synchronises, and a
call can be captured in a graph.  What they say out of range is left out (include/ba_hip.h).
Rows of a result that no sequence has, or past ``max_new`` of one, are not written.
"""
import math

import torch

from ._lib import BaKvArgs, BaKvAttendArgs, BaKvCopyArgs, BaKvScoredArgs, dual_level, has_tangent, launch, lib, overlaps, written

__all__ = ['KVCache', 'BLOCK']

BLOCK = 64
HEAD_DIMS = (32, 64, 96, 128, 256)
BITS = {torch.float8_e4m3fn: 0, torch.int8: 1}
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _tensor(name):
    """A tensor of a cache; another one put in its place is checked, with the other two, by the next call."""
    def put(self, t):
        setattr(self, name, t)
        self._at = None
    return property(lambda self: getattr(self, name), put)


def _given(name):
    return property(lambda self: getattr(self, name))


class KVCache:
    """``n_blocks`` blocks of 64 tokens for ``heads`` heads of ``head_dim`` elements.

    k       (n_blocks, heads, 64, head_dim), torch.float8_e4m3fn or torch.int8
    v       (n_blocks, heads, head_dim, 64): transposed, as attention reads it
    scales  (n_blocks, heads, 2) fp32: a block's factors of keys and values, value = code * factor

    Other tensors may be put in the place of these three between calls (all of them for another number of blocks): the
    next call takes them.  A captured graph goes on with the memory that it was captured with.
    """

    k, v, scales = _tensor('_k'), _tensor('_v'), _tensor('_scales')
    # of the tensors that the last call used
    n_blocks, heads, head_dim = _given('_n_blocks'), _given('_heads'), _given('_head_dim')
    device, dtype = _given('_device'), _given('_dtype')

    def __init__(self, n_blocks, heads, head_dim, dtype=torch.float8_e4m3fn, device='cuda'):
        if n_blocks < 0 or heads < 1:
            raise ValueError(f'cache: bad sizes ({n_blocks} blocks, {heads} heads)')
        if dtype not in BITS:
            raise ValueError(f'cache: dtype must be torch.float8_e4m3fn or torch.int8, got {dtype}')
        if head_dim not in HEAD_DIMS:
            raise ValueError(f'cache: head_dim must be one of {HEAD_DIMS}, got {head_dim}')
        self._hold(torch.zeros((n_blocks, heads, BLOCK, head_dim), dtype=torch.uint8, device=device).view(dtype),
                   torch.zeros((n_blocks, heads, head_dim, BLOCK), dtype=torch.uint8, device=device).view(dtype),
                   torch.ones((n_blocks, heads, 2), dtype=torch.float32, device=device))

    @classmethod
    def wrap(cls, k, v, scales):
        """A cache over tensors that the caller holds.  e4m3 codes in them must not be NaN (a block is made NaN by its
        factor), and factors must lie in [2^-60, 2^60] or be NaN."""
        self = cls.__new__(cls)
        self._hold(k, v, scales)
        return self

    def _hold(self, k, v, scales):
        if k.dim() != 4 or k.shape[2] != BLOCK or k.dtype not in BITS:
            raise ValueError(f'cache: k must be (n_blocks, heads, {BLOCK}, head_dim) in float8_e4m3fn or int8')
        n, h, _, d = k.shape
        if d not in HEAD_DIMS:
            raise ValueError(f'cache: head_dim must be one of {HEAD_DIMS}, got {d}')
        if tuple(v.shape) != (n, h, d, BLOCK) or v.dtype != k.dtype:
            raise ValueError(f'cache: v must be {(n, h, d, BLOCK)} in {k.dtype}')
        if tuple(scales.shape) != (n, h, 2) or scales.dtype != torch.float32:
            raise ValueError(f'cache: scales must be {(n, h, 2)} in fp32')
        if not (k.is_contiguous() and v.is_contiguous() and scales.is_contiguous()):
            raise ValueError('cache: k, v and scales must be contiguous')
        if not k.is_cuda or v.device != k.device or scales.device != k.device:
            raise RuntimeError('cache: k, v and scales must be on one GPU (the cache runs in libba_hip.so)')
        self._k, self._v, self._scales = k, v, scales
        self._n_blocks, self._heads, self._head_dim = n, h, d
        self._device, self._dtype = k.device, k.dtype
        # the fields of every call
        self._at = k.data_ptr(), v.data_ptr(), scales.data_ptr()
        same = dict(zip(('k', 'v', 'scales'), self._at), n_blocks=n, heads=h, dim=d, bits=BITS[k.dtype])
        self._lib, self._args = lib(), BaKvArgs(**same)
        self._attend_args = BaKvAttendArgs(n_splits=1, scale=1.0 / math.sqrt(d), **same)
        self._scored_args = BaKvScoredArgs(n_splits=1, scale=1.0 / math.sqrt(d), **same)

    def _begin(self, x, y):
        """Every call starts with it: the fields of calls are those of the tensors held now, and what has a gradient or a
        tangent, which codes cannot carry on, is refused."""
        k, v, scales, at = self._k, self._v, self._scales, self._at
        if at is None or k.data_ptr() != at[0] or v.data_ptr() != at[1] or scales.data_ptr() != at[2]:
            self._at = None
            self._hold(k, v, scales)
        if (x.requires_grad or y.requires_grad or scales.requires_grad) and torch.is_grad_enabled():
            raise RuntimeError('cache: codes carry no gradient: call it under torch.no_grad()')
        if dual_level() and has_tangent(x, y, scales):
            raise RuntimeError('cache: codes carry no tangent of forward-mode differentiation')

    def _fill(self, a, pages, firsts, name, offsets, n_rows, max_rows):
        """The fields of a call that the arguments of every call give."""
        dev = self._device
        shape, stride = pages.shape, pages.stride()
        if (len(shape) != 2 or pages.dtype is not torch.int32 or pages.device != dev or
                stride[1] != 1 and shape[0] > 0 and shape[1] > 1):
            raise ValueError(f'cache: pages must be (n_seqs, blocks) int32 on {dev} with contiguous rows')
        S, a.n_pages = shape
        a.n_seqs, a.pages, a.pages_stride = S, pages.data_ptr(), stride[0]
        if firsts.dtype is not torch.int32 or firsts.device != dev or firsts.shape != (S,) or not firsts.is_contiguous():
            raise ValueError(f'cache: {name} must be a contiguous int32 tensor of shape {(S,)} on {dev}')
        a.n_rows = n_rows
        if offsets is not None:
            if offsets.dtype is not torch.int32 or offsets.device != dev or offsets.shape != (S + 1,) or not offsets.is_contiguous():
                raise ValueError(f'cache: offsets must be a contiguous int32 tensor of shape {(S + 1,)} on {dev}')
            a.offsets = offsets.data_ptr()
            most = n_rows if max_rows is None or max_rows > n_rows else int(max_rows)
            if most < 0:
                raise ValueError('cache: a negative bound on rows')
        else:
            if S == 0 and n_rows or S and n_rows % S:
                raise ValueError(f'cache: {n_rows} rows are not the same number for each of {S} sequences: give offsets')
            most = n_rows // S if S else 0
            a.rows_per_seq = most
        a.max_rows = most
        return most

    def _rows(self, t, name, heads):
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self._head_dim or t.device != self._device:
            raise ValueError(f'cache: {name} must be (tokens, {heads}, {self._head_dim}) on {self._device}, got '
                             f'{tuple(shape)} on {t.device}')
        st, sh, one = t.stride()
        if one != 1:
            raise ValueError(f'cache: the elements of a head of {name} must be contiguous')
        return st, sh

    def append(self, k, v, pages, lengths, offsets=None, max_new=None):
        """Write the rows of k and v (tokens, heads, head_dim; fp32, fp16 or bf16) after the first ``lengths`` (n_seqs,)
        int32 tokens of their sequences.  ``lengths`` stays as it is.  No two sequences of a call may append to the
        same block.

        A block that is filled by several calls has its codes made anew whenever a call outgrows its factor.  int8 codes
        are rounded again each time: after n such calls a value is within (n + 1) / 2 steps of the factor, up to 32 steps
        of 127 where each of 64 single tokens is a little larger than all before.  e4m3 factors at least double, which
        loses nothing but the lowest bits of the smallest codes."""
        self._begin(k, v)
        a = BaKvArgs.from_buffer_copy(self._args)
        a.rk_st, a.rk_sh = self._rows(k, 'k', self._heads)
        a.rv_st, a.rv_sh = self._rows(v, 'v', self._heads)
        n, dtype = k.shape[0], k.dtype
        code = DTYPES.get(dtype)
        if code is None or v.shape[0] != n or dtype is not v.dtype:
            raise ValueError(f'cache: k and v must be alike, in fp32, fp16 or bf16: got {tuple(k.shape)} {k.dtype} and '
                             f'{tuple(v.shape)} {v.dtype}')
        a.starts, a.dtype, a.rk, a.rv = lengths.data_ptr(), code, k.data_ptr(), v.data_ptr()
        if self._fill(a, pages, lengths, 'lengths', offsets, n, max_new):
            launch(self._lib.ba_kv_write, a, self._device)
            written((self._k, self._v, self._scales))

    def read(self, pages, starts, offsets, n_rows, max_count=None, dtype=torch.bfloat16):
        """(k, v) of tokens ``starts[s]`` and on, ``offsets[s + 1] - offsets[s]`` of each sequence (n_rows / n_seqs where
        offsets is None), as (n_rows, heads, head_dim) tensors of ``dtype``: code * factor, rounded once."""
        code = DTYPES.get(dtype)
        if code is None:
            raise ValueError(f'cache: fp32, fp16 or bf16 values, got {dtype}')
        if n_rows < 0:
            raise ValueError(f'cache: {n_rows} rows')
        self._begin(self._scales, self._scales)
        a = BaKvArgs.from_buffer_copy(self._args)
        shape = (n_rows, self._heads, self._head_dim)
        k = torch.empty(shape, dtype=dtype, device=self._device)
        v = torch.empty_like(k)
        a.rk_st = a.rv_st = self._heads * self._head_dim
        a.rk_sh = a.rv_sh = self._head_dim
        a.starts, a.dtype, a.rk, a.rv = starts.data_ptr(), code, k.data_ptr(), v.data_ptr()
        if self._fill(a, pages, starts, 'starts', offsets, n_rows, max_count):
            launch(self._lib.ba_kv_read, a, self._device)
        return k, v

    def copy(self, src, dst, count=None):
        """Copy blocks ``src`` to blocks ``dst`` ((n,) int32 each), codes and factors: the pairs that ``BlockPool.grow`` and
        ``BlockPool.compact`` give, for each cache that the pool's lists are about.  count: (1,) int32, the first so many
        pairs only.  Pairs with a number that is no block's (-1) are left out.  No block may be the destination of two pairs,
        or of one and the source of another."""
        self._begin(self._scales, self._scales)
        dev, n = self._device, src.shape[0] if src.dim() == 1 else -1
        for t, name, shape in ((src, 'src', (n,)), (dst, 'dst', (n,)), (count, 'count', (1,))):
            if t is None and name == 'count':
                continue
            if t.dtype is not torch.int32 or t.device != dev or t.shape != shape or not t.is_contiguous():
                raise ValueError(f'cache: {name} must be a contiguous int32 tensor of one dimension on {dev}, dst as long as '
                                 'src, count of one number')
        a = BaKvCopyArgs(k=self._at[0], v=self._at[1], scales=self._at[2], n_blocks=self._n_blocks, heads=self._heads,
                         dim=self._head_dim, src=src.data_ptr(), dst=dst.data_ptr(), n=n)
        if count is not None:
            a.count = count.data_ptr()
        if n and self._n_blocks:
            launch(self._lib.ba_kv_copy, a, dev)
            written((self._k, self._v, self._scales))

    def _per(self, t, name, dtype, n):
        if t.dtype is not dtype or t.device != self._device or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f'cache: {name} must be a contiguous {dtype} tensor of shape {(n,)} on {self._device}')
        return t.data_ptr()

    def attend(self, q, pages, lengths, offsets=None, max_new=None, causal=True, window=None, scale=None, out=None,
               return_lse=False, cap=None, slopes=None, prefix=None, since=None, until=None, shared=0):
        """Attention of the rows of q (tokens, q_heads, head_dim; fp16 or bf16) over the cached tokens of their
        sequences: softmax(scale q k^T) v.

        lengths   (n_seqs,) int32: tokens of each sequence in the cache, those of the queries among them; the n rows of
                  a sequence stand at its last n positions
        causal    a row sees the tokens up to its own position (else all)
        window    it sees only tokens later than its position less ``window``
        scale     default 1 / sqrt(head_dim)
        out       a tensor like q for the result (q itself, or one that does not overlap it)
        cap       scores z become cap tanh(z / cap), cap in [1e-3, 1e3]; off by 4e-7 cap at most
        slopes    (q_heads,) fp32, finite: then less slope |p - j| for the row's position p and token j
        since     (tokens,) int32: a row sees only tokens from its own number on (the first token of its document)
        until     (tokens,) int32: and only those below this one (the end of its frame, with causal=False)
        prefix    (n_seqs,) int32: the first so many tokens of a sequence are seen by all its rows, whatever causal, window,
                  since and until say (a prompt that is read in both directions, the first tokens beside a window)
        shared    the first so many blocks (a host number) of all lists are the same as far as their tokens go (none that was
                  given back is among them): they are read once for all sequences, where that is expected to be faster than
                  reading each list by itself
        A row that sees no token gives zeros.  q_heads is a multiple of the cache's heads; query head h reads cache
        head h // (q_heads // heads).  With ``return_lse`` also the logarithm of the sum of exp(score) over the tokens that a
        row sees (scale q k^T, capped and less its bias where these are given) as (tokens, q_heads) fp32, -inf where it sees
        none, with which results over different tokens can be joined."""
        self._begin(q, q if out is None else out)
        shape = q.shape
        if len(shape) != 3 or shape[1] % self._heads or shape[1] == 0:
            raise ValueError(f'cache: q must be (tokens, a multiple of {self._heads} heads, {self._head_dim}), got {tuple(shape)}')
        n_rows, q_heads, dim = shape
        scored = bool(shared) or cap is not None or not (slopes is prefix is since is until is None)
        a = BaKvScoredArgs.from_buffer_copy(self._scored_args) if scored else BaKvAttendArgs.from_buffer_copy(self._attend_args)
        a.q_st, a.q_sh = self._rows(q, 'q', q_heads)
        dtype, dev = q.dtype, self._device
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            raise ValueError(f'cache: queries must be fp16 or bf16, got {dtype}')
        if window is not None:
            if window < 1:
                raise ValueError(f'cache: window must be at least 1, got {window}')
            a.window = min(window, 1 << 40)       # (a field of 64 bits keeps the low ones of a longer number)
        if scale is not None:
            if not 0.0 < scale < 1e30:
                raise ValueError(f'cache: scale must be positive, got {scale}')
            a.scale = scale
        given = out is not None
        if not given:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=dtype, device=dev)    # 1.1, 2.2 us
            a.o_st, a.o_sh = q_heads * dim, dim
        else:
            if out.shape != shape or out.dtype is not dtype:
                raise ValueError('cache: out must be like q')
            if overlaps(out, q):
                raise ValueError('cache: out overlaps itself or, not in its place, q')
            a.o_st, a.o_sh = self._rows(out, 'out', q_heads)
        lse = None
        if return_lse:
            lse = torch.empty((n_rows, q_heads), dtype=torch.float32, device=dev)
            a.lse = lse.data_ptr()
        a.lengths, a.dtype, a.q, a.o = lengths.data_ptr(), DTYPES[dtype], q.data_ptr(), out.data_ptr()
        a.q_heads, a.causal = q_heads, 1 if causal else 0
        most = self._fill(a, pages, lengths, 'lengths', offsets, n_rows, max_new)
        if scored:
            if cap is not None:
                if not 1e-3 <= cap <= 1e3:
                    raise ValueError(f'cache: cap must be in [1e-3, 1e3], got {cap}')
                a.cap = cap
            if slopes is not None:
                a.slopes = self._per(slopes, 'slopes', torch.float32, q_heads)
                if slopes.requires_grad and torch.is_grad_enabled() or dual_level() and has_tangent(slopes):
                    raise RuntimeError('cache: slopes carry no gradient: call it under torch.no_grad()')
            if prefix is not None:
                a.prefix = self._per(prefix, 'prefix', torch.int32, a.n_seqs)
            if since is not None:
                a.since = self._per(since, 'since', torch.int32, n_rows)
            if until is not None:
                a.until = self._per(until, 'until', torch.int32, n_rows)
            if not 0 <= shared <= a.n_pages:
                raise ValueError(f'cache: {shared} shared blocks of lists of {a.n_pages}')
            a.shared = shared
        if most:
            L = self._lib
            if scored:
                call = L.ba_kv_attend_scored
                L.ba_kv_scored_plan(a)
                n = a.n_splits + a.shared_parts
            else:
                call = L.ba_kv_attend
                a.n_splits = n = L.ba_kv_attend_splits(a.n_seqs, self._heads, q_heads, dim, most, a.n_pages)
            if n > 1:                        # the partial sums live until the launches on this stream are done
                size = L.ba_kv_attend_workspace_bytes(n_rows, q_heads, dim, n)
                work = torch.empty(size, dtype=torch.uint8, device=dev)
                a.workspace, a.workspace_bytes = work.data_ptr(), size
            launch(call, a, dev)
            if given:
                written((out,))
        return (out, lse) if return_lse else out
