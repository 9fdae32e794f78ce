"""Caches of many sequences in pages of one pool (``qw_paged_*`` of ``include/qwattn.h``).

A layer's keys and values lie in pages of ``page_size`` tokens of every KV head. The caller owns the
tables: ``table`` [B, W] int32 on the device gives the pool's page of each ``page_size`` tokens of each
sequence, anything outside the pool (-1) where it has none.
"""
from __future__ import annotations

import ctypes
import functools

from . import KVCacheMode, QwError, _check, _stream, _torch, lib


# (A decoding step is a few of these calls, each about as long on the host as on the device: attributes that cost a
# call are read once.)


def _ints(t, what: str, device, n: int):
    """A [n] int32 tensor on the device, contiguous."""
    if t.shape != (n,) or t.dtype is not _torch().int32 or t.device != device:
        raise QwError(1, f"{what} must be a [{n}] int32 tensor on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _table(t, device, what: str):
    """(tensor, B, W, row stride) of a table [B, W] int32 on the device."""
    shape = t.shape
    if len(shape) != 2 or t.dtype is not _torch().int32 or t.device != device:
        raise QwError(1, f"{what}: table must be a [B, W] int32 tensor on {device}")
    B, W = shape
    if t.is_contiguous():
        return t, B, W, W
    row, col = t.stride()
    if W > 1 and col != 1 or B > 1 and row < W:
        return t.contiguous(), B, W, W
    return t, B, W, row if B > 1 else W


@functools.lru_cache(maxsize=64)
def _axes(sections: tuple, interleaved: bool) -> bytes:
    """The axis of each pair: runs of the sections' lengths, or the axes in turn, each while it has pairs
    left, the first for the rest."""
    n = len(sections)
    if not 1 <= n <= 8 or any(int(s) != s or s < 0 for s in sections) or not 0 < sum(sections) <= 256:
        raise QwError(1, "rope_axes: 1 to 8 sections of pairs, none negative, 1 to 256 in all, expected")
    sections = tuple(int(s) for s in sections)
    if not interleaved:
        return bytes(a for a, s in enumerate(sections) for _ in range(s))
    return bytes(p % n if p < n * sections[p % n] else 0 for p in range(sum(sections)))


def _turned(qkv, positions, sections, width: int, what: str):
    """Checked (qkv, its tokens, positions, their stride)."""
    torch = _torch()
    if qkv.dim() != 2 or qkv.shape[1] != width or qkv.dtype is not torch.float16 or not qkv.is_cuda:
        raise QwError(1, f"{what}: qkv must be [n, {width}] fp16 on the device")
    n = qkv.shape[0]
    if positions.dim() != 2 or positions.shape != (len(sections), n) or positions.dtype is not torch.int32 or \
            positions.device != qkv.device:
        raise QwError(1, f"{what}: positions must be [{len(sections)}, {n}] int32 on {qkv.device}")
    if n > 1 and positions.stride(1) != 1 or len(sections) > 1 and positions.stride(0) < n:
        positions = positions.contiguous()
    qkv = qkv.contiguous()
    if qkv.data_ptr() % 16:
        qkv = qkv.clone()
    return qkv, n, positions, positions.stride(0) if len(sections) > 1 else n


def rope_axes(qkv, positions, sections, n_q_heads: int, n_kv_heads: int, head_dim: int, rope_base: float,
              rope_scale: float = 1.0, interleaved: bool = False, traditional: bool = False):
    """Rotary positions of several axes (time, height, width) out of the packed projection ``qkv``
    [n, (Hq + 2 Hkv) D] fp16: ``positions`` [axes, n] int32, ``sections`` the pairs of each axis
    (2 * their sum dims of a head turn), one run after another or, ``interleaved``, in turn. Returns
    (q [n, Hq, D], k [n, Hkv, D]), rotated; the values stay in ``qkv``."""
    axes = _axes(tuple(sections), bool(interleaved))
    x, n, pos, stride = _turned(qkv, positions, sections, (n_q_heads + 2 * n_kv_heads) * head_dim, "rope_axes")
    q, k = x.new_empty((n, n_q_heads, head_dim)), x.new_empty((n, n_kv_heads, head_dim))
    args = (x.data_ptr(), n, n_q_heads, n_kv_heads, head_dim, 2 * len(axes), int(traditional), float(rope_base),
            float(rope_scale), pos.data_ptr(), stride, len(sections), axes, q.data_ptr(), k.data_ptr(), _stream(x.device))
    cuda = _torch().cuda
    if x.get_device() == cuda.current_device():
        _check(lib().qw_rope_axes(*args))
    else:
        with cuda.device(x.device):
            _check(lib().qw_rope_axes(*args))
    return q, k


class PagedKVCache:
    """One layer's keys and values of many sequences, in pages (``qw_paged_create``). Modes
    ``"fp16"``, ``"affine8"``, ``"affine4"`` and ``"int8"``, with the codecs of :class:`KVCache`;
    head_dim 128 or 256; ``page_size`` 16, 32, 64, 128 or 256."""

    def __init__(self, mode: int | str, n_kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64,
                 group_size: int = 64, device=None):
        torch = _torch()
        if isinstance(mode, str):
            mode = KVCacheMode.from_str(mode)
        self.mode, self.n_kv_heads, self.head_dim = mode, n_kv_heads, head_dim
        self.n_pages, self.page_size = n_pages, page_size
        self.bits = KVCacheMode.BITS[mode]
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else
                                   torch.device(device).index or 0)
        self._row = (n_kv_heads, head_dim)
        self._h = None
        h = ctypes.c_void_p()
        _check(lib().qw_paged_create(mode, group_size, n_kv_heads, head_dim, n_pages, page_size,
                                     self.device.index, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().qw_paged_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def nbytes(self) -> int:
        v = ctypes.c_int64()
        _check(lib().qw_paged_nbytes(self._h, ctypes.byref(v)))
        return v.value

    # -- new tokens in, tokens back out
    def _seqs(self, n: int, table, starts, offsets, what: str):
        t, B, W, stride = _table(table, self.device, what)
        s = _ints(starts, f"{what}: starts", self.device, B)
        o = None if offsets is None else _ints(offsets, f"{what}: offsets", self.device, B + 1)
        if o is None and B and n % B:
            raise QwError(1, f"{what}: without offsets the tokens must be as many for each sequence")
        return (n, B, None if o is None else o.data_ptr(), s.data_ptr(), t.data_ptr(), stride, W), (t, s, o)

    def _rows(self, t, what: str):
        """New rows [n, Hkv, D] of any token and head strides: (tensor, n, token stride, head stride)."""
        torch, shape = _torch(), t.shape
        if len(shape) != 3 or shape[1:] != self._row or t.dtype is not torch.float16 or t.device != self.device:
            raise QwError(1, f"{what} must be [n, {self.n_kv_heads}, {self.head_dim}] fp16 on {self.device}")
        token, head, d = t.stride()
        if d != 1 or token % 4 or head % 4 or t.data_ptr() % 8:
            t = t.clone(memory_format=torch.contiguous_format)
            token, head, d = t.stride()
        return t, shape[0], token, head

    def update(self, keys, values, table, starts, offsets=None) -> None:
        """New tokens ``keys``, ``values`` [n, Hkv, D] fp16 into their pages: those of sequence b,
        ``offsets[b]`` .. ``offsets[b + 1]`` - 1 (int32 [B + 1]; None: n / B each), to positions
        ``starts[b]`` .. (int32 [B])."""
        k, n, kt, kh = self._rows(keys, "update: keys")
        v, nv, vt, vh = self._rows(values, "update: values")
        if nv != n:
            raise QwError(1, "update: keys and values must be as many")
        args, _keep = self._seqs(n, table, starts, offsets, "update")
        _check(lib().qw_paged_update(self._h, k.data_ptr(), v.data_ptr(), kt, kh, vt, vh, *args, _stream(self.device)))

    def gather(self, table, starts, n: int, offsets=None):
        """The tokens at those positions back: (keys, values) [n, Hkv, D] fp16, zeros where a
        position has no page."""
        if n < 0:
            raise QwError(1, "gather: n >= 0 expected")
        args, _keep = self._seqs(n, table, starts, offsets, "gather")
        k, v = _torch().empty((2, n, *self._row), dtype=_torch().float16, device=self.device).unbind()
        _check(lib().qw_paged_gather(self._h, k.data_ptr(), v.data_ptr(), *args, _stream(self.device)))
        return k, v

    def rope_update(self, qkv, positions, sections, n_q_heads: int, rope_base: float, table, starts, offsets=None,
                    rope_scale: float = 1.0, interleaved: bool = False, traditional: bool = False):
        """:func:`rope_axes` of the new tokens' projection ``qkv`` [n, (Hq + 2 Hkv) D], its rotated keys and
        values into their pages as :meth:`update` takes them. Returns q [n, Hq, D], rotated."""
        axes = _axes(tuple(sections), bool(interleaved))
        x, n, pos, stride = _turned(qkv, positions, sections, (n_q_heads + 2 * self.n_kv_heads) * self.head_dim, "rope_update")
        if x.device != self.device:
            raise QwError(1, f"rope_update: qkv must be on {self.device}")
        args, _keep = self._seqs(n, table, starts, offsets, "rope_update")
        q = x.new_empty((n, n_q_heads, self.head_dim))
        _check(lib().qw_paged_rope_update(self._h, x.data_ptr(), n_q_heads, 2 * len(axes), int(traditional),
                                          float(rope_base), float(rope_scale), pos.data_ptr(), stride, len(sections),
                                          axes, q.data_ptr(), *args, _stream(self.device)))
        return q

    # -- attention
    def _query(self, q, table, lengths, what: str):
        torch, shape = _torch(), q.shape
        if len(shape) != 4 or shape[3] != self.head_dim or q.dtype is not torch.float16 or q.device != self.device:
            raise QwError(1, f"{what}: q must be [B, Hq, L, {self.head_dim}] fp16 on {self.device}")
        seq, head, row, d = q.stride()
        if d != 1 or (seq | head | row) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            seq, head, row, d = q.stride()
        t, B, W, stride = _table(table, self.device, what)
        if shape[0] != B:
            raise QwError(1, f"{what}: q and table must have as many sequences")
        n = _ints(lengths, f"{what}: lengths", self.device, B)
        return (q.data_ptr(), seq, head, row, B, shape[1], shape[2], n.data_ptr(), t.data_ptr(), stride, W), (q, t, n)

    def attention(self, q, table, lengths, scale: float, picked=None):
        """Attention of each sequence's newest L tokens ``q`` [B, Hq, L, D] over its first
        ``lengths[b]`` keys (int32 [B], the newest among them), causal among the last L; ``picked``
        ([B, Hkv, n] int32, as :meth:`select_pages` gives): over those pages alone. Returns [B, Hq, L, D]."""
        torch = _torch()
        args, _keep = self._query(q, table, lengths, "attention")
        n, at = 0, None
        if picked is not None:
            shape = picked.shape
            if len(shape) != 3 or shape[0] != args[4] or shape[1] != self.n_kv_heads or shape[2] < 1 or \
                    picked.dtype is not torch.int32 or picked.device != self.device:
                raise QwError(1, f"attention: picked must be [B, {self.n_kv_heads}, n] int32 on {self.device}")
            picked = picked.contiguous()
            n, at = shape[2], picked.data_ptr()
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _check(lib().qw_paged_attention(self._h, *args, at, n, float(scale), out.data_ptr(), _stream(self.device)))
        return out

    def select_pages(self, q, table, lengths, budget: int, sink: int = 0, recent: int = 0):
        """The pages that each KV head should read for those queries: the first ``sink``, the last
        ``recent`` and, of the others, those whose keys' bounds promise the largest scores, ``budget`` in all.
        Returns [B, Hkv, budget] int32, ascending columns of the table, -1 behind the last."""
        args, _keep = self._query(q, table, lengths, "select_pages")
        budget, sink, recent = int(budget), int(sink), int(recent)
        if not 0 < budget < 2 ** 27 or min(sink, recent) < 0 or sink + recent > budget:  # (before any of them passes an int)
            raise QwError(1, "select_pages: 0 < budget < 2^27 and sink + recent <= budget, neither negative, expected")
        picked = _torch().empty((args[4], self.n_kv_heads, budget), dtype=_torch().int32, device=self.device)
        _check(lib().qw_paged_select(self._h, *args, budget, sink, recent, picked.data_ptr(), _stream(self.device)))
        return picked
