"""A key/value cache held in 8 bits, and attention over it.

Codes are e4m3 with one power-of-two scale per (page, head): a quarter of the bytes of an fp32 cache, which is what bounds a
decode step.  A page holds `page` tokens of every head; a sequence's pages are named by a block table, or lie one behind the
other.  The kernels and the rules of scales, masks and absent pages are described at tvae_kv8_* in include/tvae_kernels.h.
The reference has no counterpart (its greedy_decode keeps no cache, transvae/trans_models.py:418-434)."""
import ctypes as C
import math

import torch

from . import ops
from ._lib import BF16, F16, F32, TvaeError, call
from .ops import _ptr

_TYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
DK = (32, 64, 128, 256)


def _rows(t, name):
    """(t, strides of sequence, token and head): t as rows that the kernels take, dense in the last dimension, every row on a 16-byte
    border (copied only if it is not)"""
    if t.dim() != 4 or t.dtype not in _TYPES:
        raise TvaeError("%s must be a 4-dimensional float32, bfloat16 or float16 tensor (got %s %s)" % (name, tuple(t.shape), t.dtype))
    a, b, c, one = t.stride()
    if one != 1 or (t.data_ptr() | (a | b | c) * t.element_size()) & 15:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        _, T, h, dk = t.shape
        a, b, c = T * h * dk, h * dk, dk               # not t.stride(): a dimension of one element keeps any stride
    return t, a, b, c


class KV8Cache:
    """Keys and values of some sequences in 8 bits.  For serving: nothing here is differentiated.

    ``KV8Cache.empty(n_pages, heads, dk, page)`` makes a pool whose pages block tables hand out;
    ``KV8Cache.for_batch(n, max_len, heads, dk, page)`` one whose pages belong to `n` sequences in order (no tables).
    ``KV8Cache(k, v, k_exp, v_exp, n_seq)`` wraps buffers that exist: codes (n_pages, heads, page, dk) and exponents
    (n_pages, heads), uint8, contiguous."""

    __slots__ = ("k", "v", "k_exp", "v_exp", "n_seq", "n_pages", "heads", "page", "dk", "device")

    def __init__(self, k, v, k_exp, v_exp, n_seq=None):
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or k_exp.shape != (shape[0], shape[1]) or v_exp.shape != (shape[0], shape[1]):
            raise TvaeError("cache: codes must be (n_pages, heads, page, dk) and exponents (n_pages, heads), got %s %s %s %s"
                            % (tuple(k.shape), tuple(v.shape), tuple(k_exp.shape), tuple(v_exp.shape)))
        dev, u8 = k.device, torch.uint8
        if not (k.dtype is u8 and v.dtype is u8 and k_exp.dtype is u8 and v_exp.dtype is u8 and v.device == dev and k_exp.device == dev
                and v_exp.device == dev and k.is_contiguous() and v.is_contiguous() and k_exp.is_contiguous() and v_exp.is_contiguous()):
            raise TvaeError("cache: codes and exponents must be contiguous uint8 tensors of one device")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.n_pages, self.heads, self.page, self.dk = shape
        self.device = dev
        if self.dk not in DK or self.page < 16 or self.page > 256 or self.page & (self.page - 1):
            raise TvaeError("cache: dk must be one of %s and page a power of two in [16, 256] (got dk %d, page %d)" % (DK, self.dk, self.page))
        if n_seq is not None and (n_seq < 1 or self.n_pages % n_seq):
            raise TvaeError("cache: %d pages cannot be dealt to %s sequences" % (self.n_pages, n_seq))
        self.n_seq = n_seq

    @classmethod
    def empty(cls, n_pages, heads, dk, page=32, device="cuda", n_seq=None):
        "a pool of zeroed pages"
        k, v = (torch.zeros((n_pages, heads, page, dk), dtype=torch.uint8, device=device) for _ in range(2))
        ke, ve = (torch.full((n_pages, heads), 127, dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, ke, ve, n_seq)

    @classmethod
    def for_batch(cls, n, max_len, heads, dk, page=32, device="cuda"):
        "room for `max_len` tokens of `n` sequences, one sequence's pages behind the other's"
        if n < 1 or max_len < 1:
            raise TvaeError("cache: need n >= 1 and max_len >= 1 (got %s, %s)" % (n, max_len))
        return cls.empty(n * -(-max_len // page), heads, dk, page, device, n_seq=n)

    # ------------------------------------------------------------------------------------------ arguments
    def _on(self, t, what):
        if t.device != self.device:
            raise TvaeError("%s is on %s, the cache on %s" % (what, t.device, self.device))
        return t

    def _pages(self, table, n):
        "(address of the block table or 0, pages a sequence, sequences) for a call over n sequences (None: as many as there are)"
        if table is None:
            if self.n_seq is None:
                raise TvaeError("a cache without sequences of its own needs a block table")
            if n is not None and n != self.n_seq:
                raise TvaeError("%d sequences, but the cache belongs to %d" % (n, self.n_seq))
            return 0, self.n_pages // self.n_seq, self.n_seq
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.shape[1] < 1 or (n is not None and table.shape[0] != n):
            raise TvaeError("block table must be a contiguous int32 (sequences, pages) tensor%s, got %s %s"
                            % ("" if n is None else " of %d sequences" % n, table.dtype, tuple(table.shape)))
        return _ptr(self._on(table, "block table")), table.shape[1], table.shape[0]

    def _ints(self, x, n, name):
        "(address or 0, number): per-sequence int32 values, or one number for all of them"
        if x is None or not torch.is_tensor(x):
            x = 0 if x is None else int(x)
            if not -(1 << 31) <= x < 1 << 31:
                raise TvaeError("%s must fit 32 bits (got %d)" % (name, x))
            return 0, x
        if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != n or not x.is_contiguous():
            raise TvaeError("%s must be a number or a contiguous int32 tensor of %d values, got %s %s" % (name, n, x.dtype, tuple(x.shape)))
        return _ptr(self._on(x, name)), 0

    def _cache_args(self):
        return _ptr(self.k), _ptr(self.v), _ptr(self.k_exp), _ptr(self.v_exp), self.n_pages

    def _call(self, name, *args):
        "on the cache's device, whichever is current, and on that device's current stream"
        ops.call_on(self.device, name, *args)

    # ------------------------------------------------------------------------------------------ operators
    def store(self, k, v, start=0, count=None, table=None):
        """Rows t < count[b] (None: all) of k, v (n, T, heads, dk) become tokens start[b] + t of sequence b.  `start` and
        `count` are numbers or int32 (n,) tensors on the device.  Overwriting from the middle of a sequence leaves what
        stands behind it dead; no page may be written for two sequences in one call.  Rows past a sequence's last page are dropped
        (a number as `start` has to leave room for all T rows, unless `count` is a tensor), a negative start in a tensor stores nothing."""
        (k, *ks), (v, *vs) = _rows(k, "k"), _rows(v, "v")
        n, T = k.shape[:2]
        if v.shape != k.shape or v.dtype != k.dtype or tuple(k.shape[2:]) != (self.heads, self.dk):
            raise TvaeError("store: k and v must both be (n, T, %d, %d) of one type, got %s %s and %s %s"
                            % (self.heads, self.dk, tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
        self._on(k, "k"), self._on(v, "v")
        tab, per, _ = self._pages(table, n)
        if count is not None and not torch.is_tensor(count):
            T, count = min(T, max(0, int(count))), None
        sp, s0 = self._ints(start, n, "start")
        cp, _ = self._ints(count, n, "count")
        self._call("tvae_kv8_store", _ptr(k), *ks, _ptr(v), *vs, _TYPES[k.dtype], *self._cache_args(), tab, per,
                   sp, s0, cp, n, T, self.heads, self.dk, self.page)

    def load(self, T, start=0, count=None, table=None, dtype=torch.float32):
        """(k, v), each (n, T, heads, dk) of `dtype`: tokens start[b] .. start[b] + T - 1 of every sequence, zeros from
        count[b] on and where a sequence has no such token."""
        if dtype not in _TYPES:
            raise TvaeError("load: dtype must be float32, bfloat16 or float16 (got %s)" % dtype)
        tab, per, n = self._pages(table, None)
        sp, s0 = self._ints(start, n, "start")
        if count is not None and not torch.is_tensor(count):
            count = torch.full((n,), min(T, max(0, int(count))), dtype=torch.int32, device=self.device)
        cp, _ = self._ints(count, n, "count")
        k, v = (torch.empty((n, T, self.heads, self.dk), dtype=dtype, device=self.device) for _ in range(2))
        self._call("tvae_kv8_load", *self._cache_args(), tab, per, sp, s0, cp, _ptr(k), _ptr(v), _TYPES[dtype], n, T, self.heads, self.dk, self.page)
        return k, v

    def attend(self, q, lens, table=None, causal=True, key_mask=None, scale=None, out=None, splits=None):
        """softmax(scale q k^T) v: q (n, Lq, G * heads, dk), query head i over key head i // G, the first lens[b] tokens of
        every sequence (a number or an int32 (n,) tensor).  The Lq queries are the LAST tokens of what lens counts: with
        `causal` query i sees lens - (Lq - 1 - i) tokens.  key_mask (n, W) bool or uint8: only tokens j < W with a non-zero
        entry.  scale: 1 / sqrt(dk) by default.  A query that sees nothing gets zeros.  q's type is the result's; sums and
        softmax are fp32 (with several 16-bit queries a key head, Lq * G > 1, each weight is rounded to within 2^-17 where it meets
        the values; their sum is not).  splits: parts that a sequence's tokens are cut into (by a rule of the sizes if None).  A lens tensor's
        values count at most as many tokens as the pages hold.  `out` may be q itself, but overlap
        it in no other way.  Returns `out` (or a new tensor of q's shape)."""
        q, qa, qb, qc = _rows(q, "q")
        n, Lq, hq, dk = q.shape
        if dk != self.dk or hq % self.heads or hq == 0:
            raise TvaeError("attend: q must be (n, Lq, G * %d, %d), got %s" % (self.heads, self.dk, tuple(q.shape)))
        self._on(q, "q")
        tab, per, _ = self._pages(table, n)
        lp, l0 = self._ints(lens, n, "lens")
        mp, ldm, mw = 0, 0, 0
        if key_mask is not None:
            if key_mask.dim() != 2 or key_mask.shape[0] != n or key_mask.dtype not in (torch.bool, torch.uint8):
                raise TvaeError("attend: key_mask must be a bool or uint8 (n, W) tensor, got %s %s" % (key_mask.dtype, tuple(key_mask.shape)))
            mw = key_mask.shape[1]
            if (mw > 1 and key_mask.stride(1) != 1) or key_mask.stride(0) < mw:       # also an expanded row
                key_mask = key_mask.contiguous()
            ldm = max(key_mask.stride(0), mw)
            mp = _ptr(self._on(key_mask, "key_mask") if mw else self.k_exp)             # no column: nothing is visible, nothing is read
        if out is None:
            o = out = torch.empty_like(q, memory_format=torch.contiguous_format)
            oa, ob, oc = Lq * hq * dk, hq * dk, dk
        else:
            if out.shape != q.shape or out.dtype != q.dtype:
                raise TvaeError("attend: out must have q's shape and type, got %s %s" % (tuple(out.shape), out.dtype))
            if any(st == 0 and sz > 1 for st, sz in zip(out.stride(), out.shape)):
                raise TvaeError("attend: out has several elements at one address (strides %s)" % (out.stride(),))
            self._on(out, "out")
            o, oa, ob, oc = _rows(out, "out")
        if splits is None:
            splits = self._splits(n, hq // self.heads * Lq, per * self.page if lp else l0)
        ws = None
        if splits > 1:
            ws = torch.empty(n * Lq * hq * splits * (dk + 2), dtype=torch.float32, device=q.device)
        self._call("tvae_kv8_attn", _ptr(q), qa, qb, qc, _ptr(o), oa, ob, oc, _TYPES[q.dtype], *self._cache_args(), tab, per,
                   lp, l0, mp, ldm, mw, int(causal), n, self.heads, hq // self.heads, Lq, dk, self.page,
                   1.0 / math.sqrt(dk) if scale is None else float(scale), splits, _ptr(ws))
        if o is not out:
            with torch.no_grad():
                out.copy_(o)
        return out

    def _splits(self, n, rows, keys):
        "parts for n sequences whose every key head has `rows` query rows"
        units = max(1, n * self.heads * -(-rows // 16))            # a block of four waves each, and part
        # enough blocks for the 256 compute units with parts of 256 tokens and more, and up to 2048 with parts of 1024 and more,
        # so that sequences of different lengths even out (one of 131 k tokens, 2 key heads: 64 parts 29 us, 128 21 us, 256 24 us;
        # 48 ragged ones up to 8 k, 8 key heads: 1 part 191 us, 5 parts 96 us)
        # (one sequence and head reach 2048 only past a million tokens: 1024 is what one join takes)
        return max(1, min(-(-keys // 1024), 2048 // units, 1024), min(-(-keys // 256), 256 // units))
