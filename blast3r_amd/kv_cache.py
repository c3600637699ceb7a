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
"""
import ctypes
import math

import torch

from ._lib import BaKvArgs, BaKvAttendArgs, check, lib, stream_ptr

__all__ = ['KVCache', 'BLOCK']

BLOCK = 64
HEAD_DIMS = (32, 64, 96, 128, 256)
BITS = {torch.float8_e4m3fn: 0, torch.int8: 1}
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class KVCache:
    """``n_blocks`` blocks of 64 tokens for ``heads`` heads of ``head_dim`` elements.

    k       (n_blocks, heads, 64, head_dim), torch.float8_e4m3fn or torch.int8
    v       (n_blocks, heads, head_dim, 64): transposed, as attention reads it
    scales  (n_blocks, heads, 2) fp32: a block's factors of keys and values, value = code * factor
    """

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
        self.k, self.v, self.scales = k, v, scales
        self.n_blocks, self.heads, self.head_dim = n, h, d
        self.device, self.dtype = k.device, k.dtype

    def _index(self, t, name, shape):
        if t.dtype != torch.int32 or t.device != self.device or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f'cache: {name} must be a contiguous int32 tensor of shape {shape} on {self.device}')
        return t.data_ptr()

    def _fill(self, a, pages, firsts, name, offsets, n_rows, max_rows):
        """The fields that every call has; returns the largest number of rows of a sequence."""
        if pages.dim() != 2 or pages.dtype != torch.int32 or pages.device != self.device or pages.stride(1) != 1:
            raise ValueError(f'cache: pages must be (n_seqs, blocks) int32 on {self.device} with contiguous rows')
        S = pages.shape[0]
        a.k, a.v, a.scales = self.k.data_ptr(), self.v.data_ptr(), self.scales.data_ptr()
        a.n_blocks, a.heads, a.dim, a.bits = self.n_blocks, self.heads, self.head_dim, BITS[self.dtype]
        a.n_seqs, a.pages, a.pages_stride, a.n_pages = S, pages.data_ptr(), pages.stride(0), pages.shape[1]
        firsts_at = self._index(firsts, name, (S,))
        a.n_rows = n_rows
        if offsets is not None:
            a.offsets = self._index(offsets, 'offsets', (S + 1,))
            most = n_rows if max_rows is None else min(int(max_rows), n_rows)
            if most < 0:
                raise ValueError('cache: a negative bound on rows')
        else:
            if S == 0 and n_rows or S and n_rows % S:
                raise ValueError(f'cache: {n_rows} rows are not the same number for each of {S} sequences: give offsets')
            most = n_rows // S if S else 0
            a.rows_per_seq = most
        a.max_rows = most
        return firsts_at, most

    def _rows(self, t, name, heads):
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.head_dim or t.device != self.device:
            raise ValueError(f'cache: {name} must be (tokens, {heads}, {self.head_dim}) on {self.device}, got '
                             f'{tuple(t.shape)} on {t.device}')
        if t.stride(2) != 1:
            raise ValueError(f'cache: the elements of a head of {name} must be contiguous')

    def append(self, k, v, pages, lengths, offsets=None, max_new=None):
        """Write the rows of k and v (tokens, heads, head_dim; fp32, fp16 or bf16) after the first ``lengths`` (n_seqs,)
        int32 tokens of their sequences.  ``lengths`` stays as it is.  No two sequences of a call may append to the
        same block."""
        self._rows(k, 'k', self.heads)
        self._rows(v, 'v', self.heads)
        if k.shape != v.shape or k.dtype != v.dtype or k.dtype not in DTYPES:
            raise ValueError(f'cache: k and v must be alike, in fp32, fp16 or bf16: got {tuple(k.shape)} {k.dtype} and '
                             f'{tuple(v.shape)} {v.dtype}')
        a = BaKvArgs()
        a.starts, most = self._fill(a, pages, lengths, 'lengths', offsets, k.shape[0], max_new)
        self._move(a, k, v, most, lib().ba_kv_write)

    def read(self, pages, starts, offsets, n_rows, max_count=None, dtype=torch.bfloat16):
        """(k, v) of tokens ``starts[s]`` and on, ``offsets[s + 1] - offsets[s]`` of each sequence (n_rows / n_seqs where
        offsets is None), as (n_rows, heads, head_dim) tensors of ``dtype``: code * factor, rounded once."""
        if dtype not in DTYPES:
            raise ValueError(f'cache: fp32, fp16 or bf16 values, got {dtype}')
        if n_rows < 0:
            raise ValueError(f'cache: {n_rows} rows')
        k = torch.empty((n_rows, self.heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        a = BaKvArgs()
        a.starts, most = self._fill(a, pages, starts, 'starts', offsets, n_rows, max_count)
        self._move(a, k, v, most, lib().ba_kv_read)
        return k, v

    def _move(self, a, k, v, most, call):
        a.dtype = DTYPES[k.dtype]
        a.rk, a.rv = k.data_ptr(), v.data_ptr()
        a.rk_st, a.rk_sh, _ = k.stride()
        a.rv_st, a.rv_sh, _ = v.stride()
        if a.n_rows > 0 and most > 0:
            with torch.cuda.device(self.device):
                check(call(ctypes.byref(a), stream_ptr(self.device)))

    def attend(self, q, pages, lengths, offsets=None, max_new=None, causal=True, window=None, scale=None, out=None,
               return_lse=False):
        """Attention of the rows of q (tokens, q_heads, head_dim; fp16 or bf16) over the cached tokens of their
        sequences: softmax(scale q k^T) v.

        lengths   (n_seqs,) int32: tokens of each sequence in the cache, those of the queries among them; the n rows of
                  a sequence stand at its last n positions
        causal    a row sees the tokens up to its own position (else all)
        window    it sees only tokens later than its position less ``window``
        scale     default 1 / sqrt(head_dim)
        out       a tensor like q for the result
        A row that sees no token gives zeros.  q_heads is a multiple of the cache's heads; query head h reads cache
        head h // (q_heads // heads).  With ``return_lse`` also log(sum(exp(scale q k^T))) as (tokens, q_heads) fp32,
        -inf where no token is seen, with which results over different tokens can be joined."""
        if q.dim() != 3 or q.shape[1] % self.heads or q.shape[1] == 0:
            raise ValueError(f'cache: q must be (tokens, a multiple of {self.heads} heads, {self.head_dim}), got {tuple(q.shape)}')
        n_rows, q_heads = q.shape[0], q.shape[1]
        self._rows(q, 'q', q_heads)
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f'cache: queries must be fp16 or bf16, got {q.dtype}')
        if window is not None and window < 1:
            raise ValueError(f'cache: window must be at least 1, got {window}')
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        if not 0.0 < scale < 1e30:
            raise ValueError(f'cache: scale must be positive, got {scale}')
        if out is None:
            out = torch.empty((n_rows, q_heads, self.head_dim), dtype=q.dtype, device=self.device)
        else:
            if out.shape != q.shape or out.dtype != q.dtype:
                raise ValueError('cache: out must be like q')
            self._rows(out, 'out', q_heads)
        lse = torch.empty((n_rows, q_heads), dtype=torch.float32, device=self.device) if return_lse else None
        a = BaKvAttendArgs()
        a.lengths, most = self._fill(a, pages, lengths, 'lengths', offsets, n_rows, max_new)
        if n_rows > 0 and most > 0:
            L = lib()
            a.dtype = DTYPES[q.dtype]
            a.q, a.o = q.data_ptr(), out.data_ptr()
            a.q_st, a.q_sh, _ = q.stride()
            a.o_st, a.o_sh, _ = out.stride()
            if lse is not None:
                a.lse = lse.data_ptr()
            a.q_heads, a.causal, a.window, a.scale = q_heads, bool(causal), window or 0, scale
            with torch.cuda.device(self.device):
                n = L.ba_kv_attend_splits(a.n_seqs, a.heads, q_heads, a.dim, most, a.n_pages)
                a.n_splits = n
                if n > 1:                    # the partial sums live until the launches on this stream are done
                    size = L.ba_kv_attend_workspace_bytes(n_rows, q_heads, a.dim, n)
                    work = torch.empty(size, dtype=torch.uint8, device=self.device)
                    a.workspace, a.workspace_bytes = work.data_ptr(), size
                check(L.ba_kv_attend(ctypes.byref(a), stream_ptr(self.device)))
        return (out, lse) if return_lse else out
