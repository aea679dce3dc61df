"""Paged key-value cache and the attention of one new token over it.

The generating side of an encoder-decoder whose encoder runs MonarchAttention
(the reference's BART pipeline, bart/model.py:67-152, whose decoder keeps
dense keys and values that grow with every token):

  * ``kv_cache_write``    stores new tokens' keys and values in pages, in 16 or
                          32 bits, or as e4m3 / int8 codes with one scale a
                          token and head
  * ``kv_cache_read``     gives sequences back as the dense (E, Hk, N, D)
                          tensors and (E, N) mask that ``monarch_attention`` takes
  * ``decode_attention``  attention of one new token a sequence
  * ``PagedKVCache``      owns pages, page table and lengths, and hands out pages

Everything runs on the current CUDA stream of the tensors' device, allocates
only its outputs, and never waits for the device; sequence lengths, page
tables and counts are device tensors.  A page id or length that does not fit
the cache is left out by the kernels and raises ``MonarchAttentionError``
(code MA_ERR_DEVICE) as in ``monarch_attention``: at the latest at the next
call, at once with ``check=True``.  These operators have no gradient.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading

import torch

from . import _lib
from . import monarch_attention as _ma

Tensor = torch.Tensor

_PAGE_DTYPES = {
    torch.float32: _lib.DTYPE_F32,
    torch.float16: _lib.DTYPE_F16,
    torch.bfloat16: _lib.DTYPE_BF16,
    torch.float8_e4m3fn: _lib.DTYPE_E4M3,
    torch.int8: _lib.DTYPE_I8,
}
_DENSE_DTYPES = {
    torch.float32: _lib.DTYPE_F32,
    torch.float16: _lib.DTYPE_F16,
    torch.bfloat16: _lib.DTYPE_BF16,
}
_CODED = (torch.float8_e4m3fn, torch.int8)

_CACHE_BYTES = ctypes.sizeof(_lib.MaKvCache)
_WRITE = struct.Struct(_lib.MaCacheWriteParams.FORMAT)
_READ = struct.Struct(_lib.MaCacheReadParams.FORMAT)
_DECODE = struct.Struct(_lib.MaDecodeParams.FORMAT)

_lock = threading.Lock()
_mirrors: dict[int, tuple] = {}     # device -> (status word, its address, mirror, mirror's address)
_workspaces: dict[tuple, Tensor] = {}  # (device, stream) -> ma_decode's workspace


def _status(device: torch.device, index: int) -> tuple[int, int]:
    """Addresses of the device's status word and its host mirror, after raising
    for a failure that an earlier call reported."""
    got = _mirrors.get(index)
    if got is None:
        word, host = _ma.status_word(device), _ma._status_mirror(device)
        got = (word.data_ptr(), host.data_ptr(), ctypes.c_uint32.from_address(host.data_ptr()))
        with _lock:
            _mirrors[index] = got
    if got[2].value:
        _ma._check_previous(device)
    return got[0], (0 if index in _ma._mirror_refused else got[1])


def _seq_arg(t: Tensor, name: str, E: int, index: int) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != E or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape (E,) = ({E},); "
                         f"got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the same device as the pages")
    return t.data_ptr()


def _cache_arg(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, scales: tuple | None) -> tuple:
    """The fields of an ma_kv_cache, and (device, its index, E, Hk, D)."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must both be (num_pages, heads, page_size, head_dim); "
                         f"got {tuple(shape)} and {tuple(v_pages.shape)}")
    dtype = k_pages.dtype
    code = _PAGE_DTYPES.get(dtype)
    if code is None or v_pages.dtype != dtype:
        raise TypeError(f"unsupported dtypes of the pages: {dtype}, {v_pages.dtype}")
    if not k_pages.is_cuda:
        raise RuntimeError("the key-value cache (B200) lives on CUDA devices only; "
                           f"got a tensor on {k_pages.device}")
    index = k_pages.get_device()
    num_pages, Hk, page_size, D = shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if D > 1 and (ks[3] != 1 or vs[3] != 1):
        raise ValueError("the head dimension of the pages must have stride 1")
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("page_table must be an int32 tensor of shape (E, max_pages); "
                         f"got {page_table.dtype} {tuple(page_table.shape)}")
    if v_pages.get_device() != index or page_table.get_device() != index:
        raise ValueError("pages and page table are on different devices")
    if dtype in _CODED:
        if scales is None:
            raise ValueError(f"{dtype} pages need scales=(k_scale, v_scale)")
        k_scale, v_scale = scales
        for t in scales:
            if t.dtype != torch.float32 or t.shape != shape[:3]:
                raise ValueError("scales must be float32 tensors of shape (num_pages, heads, page_size) "
                                 f"= {tuple(shape[:3])}; got {t.dtype} {tuple(t.shape)}")
            if t.get_device() != index:
                raise ValueError("scales must be on the same device as the pages")
        sp = (k_scale.data_ptr(), v_scale.data_ptr())
        ss = k_scale.stride() + v_scale.stride()
    else:
        if scales is not None:
            raise ValueError(f"{dtype} pages have no scales")
        sp, ss = (0, 0), (0, 0, 0, 0, 0, 0)
    E, max_pages = page_table.shape
    device = k_pages.device
    fields = (_CACHE_BYTES, code, k_pages.data_ptr(), v_pages.data_ptr(), *sp, *ks[:3], *vs[:3], *ss,
              page_table.data_ptr(), *page_table.stride(), E, Hk, D, num_pages, page_size, max_pages)
    return fields, device, index, E, Hk, D


def _no_grad(*tensors: Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the key-value cache operators have no gradient: call them "
                                   "under torch.no_grad() or detach their inputs")


def _call(fn, pack: struct.Struct, head: tuple, cache: tuple, tail: tuple, device: torch.device,
          index: int, stream: int, check: bool) -> None:
    word, host = _status(device, index)
    args = pack.pack(pack.size, *head, *cache, word, host, 0, 0, 0, 0, *tail)
    if torch.cuda.current_device() == index:
        rc = fn(args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(args, stream)
    if rc == _lib.MA_ERR_BAD_PARAMS and host and \
            b"status_host" in _lib.load().ma_last_error_detail():
        _ma._mirror_refused.add(index)
        return _call(fn, pack, head, cache, tail, device, index, stream, check)
    if rc:
        _lib.check(rc)
    if check:
        _ma.check_status(device)


def kv_cache_write(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor,
                   start: Tensor, *, scales: tuple | None = None, count: Tensor | None = None,
                   check: bool = False) -> None:
    """Store T new tokens a sequence in the pages, in place.

    k, v (E, Hk, T, D) in fp32 / fp16 / bf16, any strides (a view of the
    projection's (E, T, Hk * D) output needs no copy); pages (num_pages, Hk,
    page_size, D) in fp32 / fp16 / bf16, or float8_e4m3fn / int8 with
    ``scales=(k_scale, v_scale)``, float32 (num_pages, Hk, page_size);
    page_table (E, max_pages) int32.  Token t of sequence e goes to position
    ``start[e] + t``, i.e. page ``page_table[e, pos // page_size]``, slot
    ``pos % page_size``; ``count`` (E,) int32 limits the tokens that are taken
    of each sequence.  start, count, page_table are device tensors.

    Codes: ``scale = max(max|x|, 1e-12) * (1 / top)`` a token and head (top 448
    for e4m3, 127 for int8), ``code = x / scale`` rounded to the nearest, ties
    to even, in fp32.
    """
    cache, device, index, E, Hk, D = _cache_arg(k_pages, v_pages, page_table, scales)
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[0] != E or shape[1] != Hk or shape[3] != D:
        raise ValueError(f"k and v must be (E, Hk, T, D) = ({E}, {Hk}, T, {D}); "
                         f"got {tuple(shape)} and {tuple(v.shape)}")
    code = _DENSE_DTYPES.get(k.dtype)
    if code is None or v.dtype != k.dtype:
        raise TypeError(f"unsupported dtypes of k and v: {k.dtype}, {v.dtype}")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError("k and v must be on the same device as the pages")
    _no_grad(k, v)
    T = shape[2]
    sp = _seq_arg(start, "start", E, index)
    cp = _seq_arg(count, "count", E, index) if count is not None else 0
    if E == 0 or T == 0:
        return
    lib = _lib.load()
    _call(lib.ma_cache_write, _WRITE, (code,), cache,
          (k.data_ptr(), v.data_ptr(), *k.stride(), *v.stride(), sp, cp, T, 0, 0, 0, 0, 0),
          device, index, torch.cuda.current_stream(index).cuda_stream, check)


def kv_cache_read(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor,
                  max_len: int, *, scales: tuple | None = None, dtype: torch.dtype | None = None,
                  out: tuple | None = None, check: bool = False) -> tuple[Tensor, Tensor, Tensor]:
    """Sequences as dense tensors: k, v (E, Hk, max_len, D), zero at and behind
    each length, and the (E, max_len) bool mask of valid tokens.

    Arguments as for ``kv_cache_write``; lengths (E,) int32 on the device
    (longer ones are cut at max_len).  ``dtype`` of the result: the pages', or
    bf16 for e4m3 / int8 pages, unless given (fp32 / fp16 / bf16).
    ``out=(k, v)`` receives the result instead of new tensors, any strides.
    """
    cache, device, index, E, Hk, D = _cache_arg(k_pages, v_pages, page_table, scales)
    lp = _seq_arg(lengths, "lengths", E, index)
    N = int(max_len)
    if N < 0:
        raise ValueError("max_len must not be negative")
    if out is None:
        if dtype is None:
            dtype = torch.bfloat16 if k_pages.dtype in _CODED else k_pages.dtype
        k = torch.empty((E, Hk, N, D), dtype=dtype, device=device)
        v = torch.empty((E, Hk, N, D), dtype=dtype, device=device)
    else:
        k, v = out
        if k.shape != (E, Hk, N, D) or v.shape != k.shape:
            raise ValueError(f"out tensors must be (E, Hk, max_len, D) = {(E, Hk, N, D)}; "
                             f"got {tuple(k.shape)} and {tuple(v.shape)}")
        if v.dtype != k.dtype or (dtype is not None and k.dtype != dtype):
            raise TypeError(f"out dtypes {k.dtype}, {v.dtype} do not match")
        if k.get_device() != index or v.get_device() != index:
            raise ValueError("out tensors must be on the same device as the pages")
    code = _DENSE_DTYPES.get(k.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {k.dtype}")
    mask = torch.empty((E, N), dtype=torch.bool, device=device)
    if E > 0 and N > 0:
        lib = _lib.load()
        _call(lib.ma_cache_read, _READ, (code,), cache,
              (k.data_ptr(), v.data_ptr(), *k.stride(), *v.stride(), lp, mask.data_ptr(), N,
               0, 0, 0, 0, 0),
              device, index, torch.cuda.current_stream(index).cuda_stream, check)
    return k, v, mask


def _workspace(lib, device: torch.device, index: int, stream: int) -> Tensor:
    """ma_decode's workspace: one a stream, so that calls on different streams
    do not meet in it; it is zero at first and every call leaves it ready.  A
    call that is being captured gets one of its own, zeroed in the graph."""
    ws = _workspaces.get((index, stream))
    capturing = torch.cuda.is_current_stream_capturing()
    if ws is None or capturing:
        ws = torch.zeros(lib.ma_decode_workspace_bytes(), dtype=torch.uint8, device=device)
        if not capturing:
            with _lock:
                ws = _workspaces.setdefault((index, stream), ws)
    return ws


def decode_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor,
                     attention_mask: Tensor | None = None, *, scales: tuple | None = None,
                     sm_scale: float | None = None, out: Tensor | None = None,
                     return_lse: bool = False, check: bool = False):
    """Softmax attention of one new token a sequence over its cached tokens.

    q (E, H, 1, D), any strides; H is a multiple of the pages' Hk heads, and
    query heads h * (H / Hk) .. share kv head h.  The token attends to positions
    0 .. lengths[e] - 1 whose ``attention_mask`` (E, N) is nonzero (any mask
    dtype, as in ``monarch_attention``; positions at and behind N are out).
    Pages, table and scales as for ``kv_cache_write``; 16- and 32-bit pages
    have q's dtype, e4m3 / int8 pages go with any.  sm_scale: 1 / sqrt(D)
    unless given.

    Returns out (E, H, 1, D) in q's dtype, and with ``return_lse`` also the
    fp32 (E, H) logarithm of the sum of exponentials, by which results over
    parts of a sequence can be joined.  A row without a valid token gives
    out = 0 and lse = -inf; what a masked token's page holds does not matter.
    """
    cache, device, index, E, Hk, D = _cache_arg(k_pages, v_pages, page_table, scales)
    shape = q.shape
    if len(shape) != 4 or shape[0] != E or shape[2] != 1 or shape[3] != D:
        raise ValueError(f"q must be (E, H, 1, D) = ({E}, H, 1, {D}); got {tuple(shape)}")
    H = shape[1]
    if H == 0 or H % Hk:
        raise ValueError(f"the number of query heads {H} is not a multiple of the cache's {Hk}")
    code = _DENSE_DTYPES.get(q.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype of q: {q.dtype}")
    if scales is None and q.dtype != k_pages.dtype:
        raise TypeError(f"q is {q.dtype} but the pages are {k_pages.dtype}")
    if q.get_device() != index:
        raise ValueError("q must be on the same device as the pages")
    _no_grad(q)
    lp = _seq_arg(lengths, "lengths", E, index)
    mp, ms, mcode, keep, mlen = 0, (0, 0), _lib.MASK_NONE, None, 0
    if attention_mask is not None:
        if attention_mask.dim() != 2:
            raise ValueError("attention_mask must have shape (E, N); "
                             f"got {tuple(attention_mask.shape)}")
        mlen = attention_mask.shape[1]
        mp, ms, mcode, keep = _ma._mask_arg(attention_mask, E, mlen, device)
        if mlen == 0:  # nothing is valid; a pointer that is never read
            mp = lp
    if out is None:
        out = torch.empty((E, H, 1, D), dtype=q.dtype, device=device)
    else:
        if out.shape != shape:
            raise ValueError(f"out shape {tuple(out.shape)} != {tuple(shape)}")
        if out.dtype != q.dtype:
            raise TypeError(f"out dtype {out.dtype} != {q.dtype}")
        if out.get_device() != index:
            raise ValueError("out is on a different device than the inputs")
    lse = torch.empty((E, H), dtype=torch.float32, device=device) if return_lse else None
    if E > 0:
        lib = _lib.load()
        stream = torch.cuda.current_stream(index).cuda_stream
        ws = _workspace(lib, device, index, stream)
        qs, os = q.stride(), out.stride()
        _call(lib.ma_decode, _DECODE, (code,), cache,
              (q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
               qs[0], qs[1], qs[3], os[0], os[1], os[3], lp, mp, *ms, ws.data_ptr(), ws.numel(),
               1.0 / math.sqrt(D) if sm_scale is None else sm_scale, H, mcode, mlen, 0, 0, 0, 0),
              device, index, stream, check)
    del keep
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences in ``num_pages`` pages.

    ``append`` stores new tokens behind each sequence's last one (taking pages
    from the free ones as needed), ``attend`` runs ``decode_attention``,
    ``read`` gives the sequences back, ``free`` returns a sequence's pages.
    dtype: torch.float32 / float16 / bfloat16, or float8_e4m3fn / int8 codes
    with a scale a token and head.  ``page_table`` and ``lengths`` are device
    tensors; the host knows an upper bound of each length, so nothing waits for
    the kernels (only new pages cost a small copy to the device).
    """

    def __init__(self, num_pages: int, num_heads: int, head_dim: int, *, max_seqs: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in _PAGE_DTYPES:
            raise TypeError(f"unsupported dtype of the pages: {dtype}")
        if min(num_pages, num_heads, head_dim, max_seqs, max_len, page_size) < 1:
            raise ValueError("num_pages, num_heads, head_dim, max_seqs, max_len and page_size must "
                             "all be >= 1")
        if head_dim > 256:
            raise ValueError(f"head_dim must be at most 256; got {head_dim}")
        self.page_size, self.max_len = page_size, max_len
        # rows start on 16-byte boundaries whatever head_dim is
        pad = 16 // dtype.itemsize
        row = (head_dim + pad - 1) // pad * pad
        shape = (num_pages, num_heads, page_size)
        self.k_pages = torch.empty((*shape, row), dtype=dtype, device=device)[..., :head_dim]
        self.v_pages = torch.empty((*shape, row), dtype=dtype, device=device)[..., :head_dim]
        self.scales = None
        if dtype in _CODED:
            self.scales = (torch.empty(shape, dtype=torch.float32, device=device),
                           torch.empty(shape, dtype=torch.float32, device=device))
        max_pages = (max_len + page_size - 1) // page_size
        self.page_table = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self._free = list(range(num_pages))[::-1]
        self._pages: list[list[int]] = [[] for _ in range(max_seqs)]
        self._bound = [0] * max_seqs  # no sequence is longer than this

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, tokens: list[int]) -> None:
        """Pages for ``tokens[e]`` tokens in all of each sequence e."""
        if len(tokens) != len(self._pages):
            raise ValueError(f"tokens must have {len(self._pages)} entries; got {len(tokens)}")
        if max(tokens) > self.max_len:
            raise ValueError(f"a sequence of {max(tokens)} tokens exceeds max_len = {self.max_len}")
        need = [(n + self.page_size - 1) // self.page_size - len(p) for n, p in zip(tokens, self._pages)]
        want = sum(n for n in need if n > 0)
        if want > len(self._free):
            raise RuntimeError(f"the key-value cache is full: {want} pages wanted, "
                               f"{len(self._free)} free")
        if want == 0:
            return
        at, ids = [], []
        width = self.page_table.shape[1]
        for e, n in enumerate(need):
            for _ in range(n):
                at.append(e * width + len(self._pages[e]))
                self._pages[e].append(self._free.pop())
                ids.append(self._pages[e][-1])
        dev = self.page_table.device
        self.page_table.view(-1)[torch.tensor(at, device=dev)] = torch.tensor(
            ids, dtype=torch.int32, device=dev)

    def append(self, k: Tensor, v: Tensor, count: Tensor | None = None, check: bool = False) -> None:
        """Store k, v (max_seqs, heads, T, head_dim) behind the last tokens;
        count (max_seqs,) int32 limits the tokens taken of each sequence."""
        T = k.shape[2] if k.dim() == 4 else 0
        bound = [n + T for n in self._bound]
        self.reserve(bound)
        kv_cache_write(k, v, self.k_pages, self.v_pages, self.page_table, self.lengths,
                       scales=self.scales, count=count, check=check)
        self._bound = bound
        self.lengths += T if count is None else count.clamp(0, T)

    def read(self, max_len: int | None = None, dtype: torch.dtype | None = None,
             check: bool = False) -> tuple[Tensor, Tensor, Tensor]:
        """``kv_cache_read`` of all sequences, up to the longest one's bound."""
        return kv_cache_read(self.k_pages, self.v_pages, self.page_table, self.lengths,
                             max(self._bound) if max_len is None else max_len, scales=self.scales,
                             dtype=dtype, check=check)

    def attend(self, q: Tensor, attention_mask: Tensor | None = None, **kw):
        """``decode_attention`` of q (max_seqs, H, 1, head_dim)."""
        return decode_attention(q, self.k_pages, self.v_pages, self.page_table, self.lengths,
                                attention_mask, scales=self.scales, **kw)

    def free(self, seq: int) -> None:
        """Give sequence seq's pages back; it is empty after it."""
        self._free += self._pages[seq][::-1]
        self._pages[seq], self._bound[seq] = [], 0
        self.page_table[seq] = -1
        self.lengths[seq] = 0
