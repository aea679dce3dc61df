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
call, at once with ``check=True``.  These operators have no gradient:
tensors that require one or carry a tangent raise.
"""
from __future__ import annotations

import operator

import torch

from . import _lib
from . import monarch_attention as _ma

Tensor = torch.Tensor

_PAGE_DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int8)
_CODED = (torch.float8_e4m3fn, torch.int8)

# what the binding (csrc/ma_torch.cpp) returns in the place of a result
_FAILED_BEFORE, _NO_STATUS = -100, -101


_binding = None


def _load():
    global _binding
    _binding = _lib.load_torch_binding()
    return _binding


def _again(fn, args: tuple, rc: int):
    """The rare returns of a call: an unknown device's status word is made known,
    a failure of an earlier call and the library's refusals raise."""
    device = next(a for a in args if isinstance(a, Tensor)).device
    if rc == _NO_STATUS:
        _know_status(device)
    elif rc == _FAILED_BEFORE:
        _ma._check_previous(device)
    elif rc == _lib.MA_ERR_BAD_PARAMS and device.index not in _ma._mirror_refused and \
            b"status_host" in _lib.load().ma_last_error_detail():
        _ma._mirror_refused.add(device.index)
        _know_status(device)
    else:
        _lib.check(rc)
    got = fn(*args)
    return got if type(got) is not int or got == 0 else _again(fn, args, got)


def _know_status(device: torch.device) -> None:
    _load().set_status(
        device.index, _ma.status_word(device).data_ptr(), _ma._status_mirror(device).data_ptr(),
        device.index not in _ma._mirror_refused)


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
    fn = (_binding or _load()).write
    got = fn(k, v, k_pages, v_pages, page_table, start, scales, count)
    if got:
        _again(fn, (k, v, k_pages, v_pages, page_table, start, scales, count), got)
    if check:
        _ma.check_status(k_pages.device)


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
    fn = (_binding or _load()).read
    got = fn(k_pages, v_pages, page_table, lengths, max_len, scales, dtype, out)
    if type(got) is int:
        got = _again(fn, (k_pages, v_pages, page_table, lengths, max_len, scales, dtype, out), got)
    if check:
        _ma.check_status(k_pages.device)
    return got


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
    out = 0 and lse = -inf; what a masked token's page holds, and whether it is
    there, does not matter.  A NaN score of a valid token makes its row NaN.
    """
    fn = (_binding or _load()).decode
    got = fn(q, k_pages, v_pages, page_table, lengths, attention_mask, scales, sm_scale, out, return_lse)
    if type(got) is int:
        got = _again(fn, (q, k_pages, v_pages, page_table, lengths, attention_mask, scales, sm_scale,
                          out, return_lse), got)
    if check:
        _ma.check_status(q.device)
    return got


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences in ``num_pages`` pages.

    ``append`` stores new tokens behind each sequence's last one (taking pages
    from the free ones as needed), ``attend`` runs ``decode_attention``,
    ``read`` gives the sequences back, ``free`` returns a sequence's pages.
    dtype: torch.float32 / float16 / bfloat16, or float8_e4m3fn / int8 codes
    with a scale a token and head.  ``page_table`` and ``lengths`` are device
    tensors; the host knows an upper bound of each length, so nothing waits for
    the kernels: new pages cost a small copy to the device in stream order.  A
    captured graph cannot take pages: ``reserve`` them before.

    Where only the device knows how many tokens were taken (``append`` with
    ``count`` on the device, ``lengths`` changed by a captured graph), the bounds
    drift from the lengths.  ``tighten`` asks the device for them, which waits for
    it; ``append`` does so itself where its bounds would pass max_len or want
    more pages than are free.
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
        self._exact = True  # the bounds are the lengths
        self._reserved = [0] * max_seqs  # tokens that the caller reserved pages for

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, tokens: list[int]) -> None:
        """Pages for ``tokens[e]`` tokens in all of each sequence e; it keeps them until
        it is freed."""
        if len(tokens) != len(self._pages):
            raise ValueError(f"tokens must have {len(self._pages)} entries; got {len(tokens)}")
        self._take(tokens)
        self._reserved = [max(n, r) for n, r in zip(tokens, self._reserved)]

    def _need(self, tokens: list[int]) -> tuple[list[int], int]:
        """Pages that each sequence lacks (negative: has too many), and the sum of what lacks."""
        size = self.page_size
        need = [(n + size - 1) // size - len(p) for n, p in zip(tokens, self._pages)]
        return need, sum(n for n in need if n > 0)

    def _fits(self, tokens: list[int]) -> bool:
        return max(tokens) <= self.max_len and self._need(tokens)[1] <= len(self._free)

    def _take(self, tokens: list[int]) -> None:
        if max(tokens) > self.max_len:
            raise ValueError(f"a sequence of {max(tokens)} tokens exceeds max_len = {self.max_len}")
        need, want = self._need(tokens)
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
        new = self._send([at, ids], torch.int64)
        self.page_table.view(-1)[new[0]] = new[1].int()

    def _send(self, values: list, dtype: torch.dtype) -> Tensor:
        """Whole numbers on the device, in stream order: through page-locked memory,
        which torch's allocator gives out again only when the copy is done."""
        t = torch.tensor(values, dtype=dtype)
        device = self.page_table.device
        return t.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else t

    def tighten(self) -> None:
        """Ask the device for the lengths (and wait for it): the bounds become exact, and
        pages that appending took beyond them are free again; those reserved stay."""
        self._bound = [min(max(n, 0), self.max_len) for n in self.lengths.tolist()]
        self._exact = True
        for e, pages in enumerate(self._pages):
            keep = (max(self._bound[e], self._reserved[e]) + self.page_size - 1) // self.page_size
            if keep < len(pages):
                self.page_table[e, keep:] = -1
                self._free += pages[keep:][::-1]
                del pages[keep:]

    def append(self, k: Tensor, v: Tensor, count: Tensor | list[int] | None = None,
               check: bool = False) -> None:
        """Store k, v (max_seqs, heads, T, head_dim) behind the last tokens.

        ``count`` limits the tokens taken of each sequence: max_seqs whole numbers as
        a list or CPU tensor, from which the host knows the new lengths too, or an
        int32 tensor on the device, of which it knows only that no sequence takes
        more than T.  Sequences that take nothing (0) take no pages.
        """
        E, T = len(self._pages), k.shape[2] if k.dim() == 4 else 0
        took, add = [T] * E, T  # on the host (None: not known), on the device
        if count is None:
            pass
        elif isinstance(count, Tensor) and count.is_cuda:
            took, add = None, count.clamp(0, T)
        else:
            took = [min(max(operator.index(n), 0), T)
                    for n in (count.tolist() if isinstance(count, Tensor) else count)]
            if len(took) != E:
                raise ValueError(f"count must have {E} entries; got {len(took)}")
            count = add = self._send(took, torch.int32)
        bound = [n + t for n, t in zip(self._bound, took or [T] * E)]
        if not (self._exact and took) and not self._fits(bound):
            self.tighten()
            took = took or add.tolist()
            bound = [n + t for n, t in zip(self._bound, took)]
        self._take(bound)
        kv_cache_write(k, v, self.k_pages, self.v_pages, self.page_table, self.lengths,
                       scales=self.scales, count=count, check=check)
        self._bound, self._exact = bound, self._exact and took is not None
        self.lengths += add

    def read(self, max_len: int | None = None, dtype: torch.dtype | None = None,
             check: bool = False) -> tuple[Tensor, Tensor, Tensor]:
        """``kv_cache_read`` of all sequences, up to the longest one's bound (``tighten`` it
        where it has drifted)."""
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
        self._pages[seq], self._bound[seq], self._reserved[seq] = [], 0, 0
        self.page_table[seq] = -1
        self.lengths[seq] = 0
