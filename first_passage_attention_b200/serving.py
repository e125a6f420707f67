"""Serving a model with First Passage Attention: the paged cache, attention of the newest tokens over it, and the
verification of drafted tokens. Forward only (tensors that require grad are refused while gradients are recorded); every
call runs the native kernels of libfpa_b200 on the current stream, allocates its outputs only, never synchronises, and can
be captured in a CUDA graph.

``FPACache`` holds keys, values and the field of many sequences in pages of a common pool, as the model's fp16 or fp32
values or as int8 codes with a scale for each token and head. A sequence's position s lies in page
``block_table[b, s // page_size]``; block tables, lengths and start positions are int32 tensors on the device.

    cache = FPACache(n_pages, n_heads, head_dim, dtype=torch.float16, storage=torch.int8)
    cache.append(k, v, phi, psi, block_table, start)                    # k, v [B, H, n, D], phi, psi [B, H, n]
    o = first_passage_decode(q, cache, block_table, start + n, beta)    # q, o [B, H, n, D], n from 1 to 16

The walk of the field is cumulative, so phi and psi of new tokens go on from the walk's last value; the model keeps it
(``LMGenerator`` in ``lm.py`` does).
"""
import ctypes

import torch

from . import _lib
from .ops import LaunchStats, _on_device

MAX_NEW_TOKENS = 16
_PAGE_SIZES = (32, 64, 128, 256)
_HEAD_DIMS = (16, 32, 64, 128, 256)


# The current stream's handle by device index, without building a Stream object (which costs as much as the launch).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _refuse_grad(what):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} is forward only and no gradient would reach its inputs: call it under torch.no_grad() "
                           "or with detached tensors")


def _int32_on(name, x, index, n):
    if x.dtype != torch.int32 or x.get_device() != index:
        raise ValueError(f"{name} must be an int32 tensor on cuda:{index}")
    if x.dim() != 1 or x.numel() != n or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous with shape ({n},)")
    return x.data_ptr()


def _table_on(x, index, B):
    if x.dtype != torch.int32 or x.get_device() != index:
        raise ValueError(f"block_table must be an int32 tensor on cuda:{index}")
    shape, stride = x.shape, x.stride()
    if len(shape) != 2 or shape[0] != B or shape[1] < 1 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("block_table must have shape (B, pages) with contiguous rows")
    return x.data_ptr(), stride[0], shape[1]


def _call(fn, args, index):
    if _device() == index:
        rc = fn(ctypes.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(ctypes.byref(args), _raw_stream(index))
    if rc:
        _lib.check(rc)


def _empty(shape, dtype, device):
    B, H, n, D = shape
    return torch.empty_strided(shape, (H * n * D, n * D, D, 1), dtype=dtype, device=device)


class FPACache:
    """A pool of pages of keys, values and the field, for every head: k and v [n_pages, n_heads, page_size, head_dim],
    phi and psi [n_pages, n_heads, page_size]; with ``storage=torch.int8`` also k_scale and v_scale of phi's shape.
    phi_min [n_pages, n_heads] is the minimum of phi over each page (``append`` maintains it; decoding relies on it
    for pages that a sequence has filled).

    dtype: of k, v, q and o (float16 or float32). storage: None (as dtype) or torch.int8: scale = max|x| / 127 for each
    token and head (at least 2^-90), code = round(127 x / max|x|), the value is code * scale; the pool holds code + 128 as
    uint8. A row with a NaN or an infinity gets the scale NaN: it reads back as NaN, and so does what attends to it."""

    def __init__(self, n_pages, n_heads, head_dim, page_size=64, dtype=torch.float16, storage=None, device="cuda"):
        if dtype not in (torch.float16, torch.float32):
            raise ValueError("the cache's dtype must be float16 or float32")
        if storage not in (None, dtype, torch.int8):
            raise ValueError("the cache's storage must be its dtype or int8")
        if page_size not in _PAGE_SIZES:
            raise ValueError("the page size must be 32, 64, 128 or 256")
        if head_dim not in _HEAD_DIMS:
            raise ValueError("the head dimension must be 16, 32, 64, 128 or 256")
        if n_pages < 1 or n_heads < 1:
            raise ValueError("the cache needs at least one page and one head")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the cache needs a CUDA device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.n_pages, self.n_heads, self.head_dim, self.page_size = n_pages, n_heads, head_dim, page_size
        self.dtype, self.storage, self.device = dtype, storage or dtype, device
        slots = (n_pages, n_heads, page_size)
        self.k = torch.full((*slots, head_dim), 128, dtype=torch.uint8, device=device) if self.storage == torch.int8 else \
            torch.zeros(*slots, head_dim, dtype=self.storage, device=device)
        self.v = torch.zeros_like(self.k)
        self.phi, self.psi = torch.zeros(slots, device=device), torch.zeros(slots, device=device)
        self.phi_min = torch.zeros(slots[:2], device=device)
        self.k_scale = self.v_scale = None
        if self.storage == torch.int8:
            self.k_scale, self.v_scale = torch.zeros(slots, device=device), torch.zeros(slots, device=device)
        self._status = torch.zeros(64, dtype=torch.int32, device=device)
        self._struct = _lib.FpaCache(
            _lib.DTYPE_F16 if dtype == torch.float16 else _lib.DTYPE_F32,
            {torch.float16: _lib.STORE_F16, torch.float32: _lib.STORE_F32, torch.int8: _lib.STORE_I8}[self.storage],
            n_pages, n_heads, page_size, head_dim,
            *(None if x is None else x.data_ptr() for x in (self.k, self.v, self.k_scale, self.v_scale, self.phi,
                                                            self.psi, self.phi_min, self._status)))
        self._addr, self._index = ctypes.addressof(self._struct), device.index

    def append(self, k, v, phi, psi, block_table, start, counts=None):
        """Write the tokens k, v [B, H, n, D], phi, psi [B, H, n] (any strides) at positions start[b], start[b] + 1, ...
        of each sequence: counts[b] of them, or all n. They become the sequence's newest tokens: whatever it held from
        there on is gone (that is also how refused drafts are taken back)."""
        lib = _lib.load()
        H, D = self.n_heads, self.head_dim
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or shape[1] != H or shape[3] != D:
            raise ValueError(f"k and v must have shape (B, {H}, n, {D})")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise ValueError(f"k and v must be {self.dtype}")
        B, _, n, _ = shape
        if phi.shape != (B, H, n) or psi.shape != (B, H, n):
            raise ValueError(f"phi and psi must have shape (B, {H}, n)")
        if phi.dtype != torch.float32 or psi.dtype != torch.float32:
            raise ValueError("phi and psi must be float32")
        dev = self._index
        if k.get_device() != dev or v.get_device() != dev or phi.get_device() != dev or psi.get_device() != dev:
            raise ValueError(f"k, v, phi and psi must be on the cache's device cuda:{dev}")
        if k.requires_grad or v.requires_grad or phi.requires_grad or psi.requires_grad:
            _refuse_grad("FPACache.append")
        if B == 0 or n == 0:
            return
        a = _lib.FpaAppendArgs()
        _lib.APPEND_PACKER.pack_into(
            a, 0, self._addr, B, n, k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), phi.data_ptr(), *phi.stride(),
            psi.data_ptr(), *psi.stride(), *_table_on(block_table, dev, B),
            _int32_on("start", start, dev, B), 0 if counts is None else _int32_on("counts", counts, dev, B))
        _call(lib.fpa_cache_append, a, dev)
        LaunchStats.kernels += 1

    def read(self, block_table, start, n, lengths=None):
        """k, v [B, H, n, D] in the cache's dtype and phi, psi [B, H, n] at positions start[b] .. start[b] + n - 1 (from
        0 with start None); positions from lengths[b] on (or beyond the table) are zeros."""
        lib = _lib.load()
        B, H, D, dev = block_table.shape[0], self.n_heads, self.head_dim, self._index
        if n < 0:
            raise ValueError("n must not be negative")
        table = _table_on(block_table, dev, B)
        start = 0 if start is None else _int32_on("start", start, dev, B)
        lengths = 0 if lengths is None else _int32_on("lengths", lengths, dev, B)
        k = _empty((B, H, n, D), self.dtype, self.device)
        v = torch.empty_like(k)
        phi = torch.empty_strided((B, H, n), (H * n, n, 1), dtype=torch.float32, device=self.device)
        psi = torch.empty_like(phi)
        if B and n:
            a = _lib.FpaReadArgs()
            _lib.READ_PACKER.pack_into(a, 0, self._addr, B, n, *table, start, lengths, k.data_ptr(), v.data_ptr(),
                                       phi.data_ptr(), psi.data_ptr())
            _call(lib.fpa_cache_read, a, dev)
            LaunchStats.kernels += 1
        return k, v, phi, psi

    def check(self):
        """Synchronise, and raise if a call since the last check met a page id outside the pool, or a position or
        length outside a block table (such entries are skipped, never touched)."""
        lib = _lib.load()
        with _on_device(self.device):
            _lib.check(lib.fpa_workspace_status(self._status.data_ptr(), _raw_stream(self._index)))


def first_passage_decode(q, cache, block_table, lengths, beta, prefix_table=None, prefix_len=0):
    """o [B, H, n, D] of the newest n tokens (1 to 16) of each sequence, which ``cache.append`` has stored already.

    q: [B, H, n, D] in the cache's dtype (any strides). lengths[b] counts the sequence's tokens, the new ones included;
    row r stands at position lengths[b] - n + r, and rows before position 0 come out as zeros (length 0: an idle slot).
    beta: [H] float32. prefix_table (int32, [pages]) and prefix_len: tokens in the cache that come before the first
    token of every sequence, such as a system prompt; lengths do not count them, and they are read once for the whole
    batch. Equal to the last n rows of ``first_passage_attention`` over the whole sequence."""
    lib = _lib.load()
    H, D, dev = cache.n_heads, cache.head_dim, cache._index
    shape = q.shape
    if len(shape) != 4 or shape[1] != H or shape[3] != D:
        raise ValueError(f"q must have shape (B, {H}, n, {D})")
    B, _, n, _ = shape
    if not 1 <= n <= MAX_NEW_TOKENS:
        raise ValueError(f"between 1 and {MAX_NEW_TOKENS} new tokens per call")
    if q.dtype != cache.dtype or q.get_device() != dev:
        raise ValueError(f"q must be {cache.dtype} on {cache.device}")
    if beta.shape != (H,) or beta.dtype != torch.float32 or beta.get_device() != dev or not beta.is_contiguous():
        raise ValueError(f"beta must be a contiguous float32 tensor of shape ({H},) on {cache.device}")
    if q.requires_grad or beta.requires_grad:
        _refuse_grad("first_passage_decode")
    pages, ptable = 0, 0
    if prefix_len < 0 or (prefix_len > 0 and prefix_table is None):
        raise ValueError("prefix_len must not be negative, and needs a prefix_table")
    if prefix_len > 0:
        pages = prefix_table.numel()
        ptable = _int32_on("prefix_table", prefix_table, dev, pages)
        if pages * cache.page_size < prefix_len:
            raise ValueError("the prefix is longer than the pages of its table")
    o = torch.empty_like(q) if q.is_contiguous() else _empty((B, H, n, D), q.dtype, cache.device)
    if B == 0:
        return o
    table = _table_on(block_table, dev, B)
    lengths = _int32_on("lengths", lengths, dev, B)
    ws, ws_ptr, nbytes = None, 0, 0
    if prefix_len > 0:
        with _on_device(cache.device):
            nbytes = lib.fpa_decode_workspace_bytes(cache._struct, B, n, prefix_len)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=cache.device)
        ws_ptr = ws.data_ptr()
    a = _lib.FpaDecodeArgs()
    _lib.DECODE_PACKER.pack_into(a, 0, cache._addr, B, n, q.data_ptr(), *q.stride(), o.data_ptr(), *o.stride(),
                                 beta.data_ptr(), *table, lengths, ptable, pages, prefix_len, ws_ptr, nbytes, 0)
    _call(lib.fpa_decode, a, dev)
    LaunchStats.kernels += a.kernels_launched
    return o


def verify_draft(p, q, draft, u, noise, draft_lens=None):
    """Accept drafted tokens against the target's probabilities, from given random numbers.

    p [B, n + 1, V]: the target's probabilities after 0, 1, ... n drafted tokens; q [B, n, V]: those that the drafts were
    drawn from (both fp16 or both fp32); draft [B, n] int64; u [B, n] float32 from [0, 1); noise [B, V] float32 from the
    exponential distribution; draft_lens [B] int32: drafts of each sequence where they are fewer than n.

    Draft i is accepted while u_i q_i(x_i) < p_i(x_i). Returns accepted [B] int32 (drafts before the first refusal) and
    tokens [B, n + 1] int64: the accepted drafts, the next token, then -1. The next token is argmax_v max(p_a - q_a, 0) /
    noise (a draw from the normalised residual), or argmax_v p_a / noise where every draft was accepted or the residual
    is nowhere positive; ties go to the lowest index. The tokens then have the target's distribution."""
    lib = _lib.load()
    ps, qs = p.shape, q.shape
    if len(ps) != 3 or len(qs) != 3 or ps[0] != qs[0] or ps[1] != qs[1] + 1 or ps[2] != qs[2]:
        raise ValueError("p must have shape (B, n + 1, V) and q shape (B, n, V)")
    B, n, V = qs
    dt = p.dtype
    if dt not in (torch.float16, torch.float32) or q.dtype != dt:
        raise ValueError("p and q must both be fp16 or both fp32")
    if draft.shape != (B, n) or draft.dtype != torch.int64:
        raise ValueError("draft must be an int64 tensor of shape (B, n)")
    if u.shape != (B, n) or u.dtype != torch.float32:
        raise ValueError("u must be a float32 tensor of shape (B, n)")
    if noise.shape != (B, V) or noise.dtype != torch.float32:
        raise ValueError("noise must be a float32 tensor of shape (B, V)")
    if V < 1:
        raise ValueError("the vocabulary must not be empty")
    dev = p.get_device()
    if dev < 0 or q.get_device() != dev or draft.get_device() != dev or u.get_device() != dev or noise.get_device() != dev:
        raise ValueError("p, q, draft, u and noise must be on one CUDA device")
    sp, sq, sn = p.stride(), q.stride(), noise.stride()
    if sp[2] != 1 or sq[2] != 1 or sn[1] != 1:
        p, q, noise = (x if x.stride(-1) == 1 else x.contiguous() for x in (p, q, noise))
        sp, sq, sn = p.stride(), q.stride(), noise.stride()
    lens = 0 if draft_lens is None else _int32_on("draft_lens", draft_lens, dev, B)
    accepted = torch.empty_strided((B,), (1,), dtype=torch.int32, device=p.device)
    tokens = torch.empty_strided((B, n + 1), (n + 1, 1), dtype=torch.int64, device=p.device)
    if B == 0:
        return accepted, tokens
    a = _lib.FpaVerifyArgs()
    _lib.VERIFY_PACKER.pack_into(
        a, 0, _lib.DTYPE_F16 if dt == torch.float16 else _lib.DTYPE_F32, B, n, V, p.data_ptr(), sp[0], sp[1], q.data_ptr(),
        sq[0], sq[1], draft.data_ptr(), *draft.stride(), u.data_ptr(), *u.stride(), noise.data_ptr(), sn[0], lens,
        accepted.data_ptr(), tokens.data_ptr())
    _call(lib.fpa_verify, a, dev)
    LaunchStats.kernels += 1
    return accepted, tokens
