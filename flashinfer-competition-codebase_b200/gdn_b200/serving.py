"""The serving operators around the GDN decode step.

What a server of a stack with GDN layers runs beside ``gated_delta_rule_decode_pretranspose``
and its state pool; the reference has no counterpart:

* ``paged_attention_decode`` — the decode step of the stack's softmax-attention layers: one
  new token per sequence against a paged key-value cache, appended to it in the same call.
* ``beam_select`` — beam search's selection over beams and vocabulary.
* ``copy_pages``, ``fork_pages``, ``compact_pages``, ``alloc_pages``, ``free_pages`` — the
  upkeep of the caches: slots of a pooled state and pages of a key-value cache.

Like the entry points in ``ops.py``, each checks its tensors on the host and makes one call
into libgdn_b200.so on their device's current stream: no host synchronisation, no CPU
fallback.  The small calls are bound by that host work, so each first tries its twin in
``csrc/torch_entry.cpp``, which makes the same checks and the same library call from C++ and
declines whatever does not pass; what it declines is checked here, and refused in words or
called through ctypes.  Workspaces come from torch's caching allocator for each call, so calls on
different streams, and graphs captured from them, never share one.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .ops import _BF16, _F32, _check, _index_tensor, _ptr

_I32 = torch.int32
_BOOL = torch.bool
_DTYPE_CODES = {_BF16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, _F32: _lib.DTYPE_FP32}

Pools = Union[torch.Tensor, Sequence[torch.Tensor]]


class _Nothing:
    """Stands for the extension where it is not built: declines every call."""

    attend = select = copy = alloc = release = fork = compact = staticmethod(lambda *args: None)


_calls = None


def _torch_calls():
    global _calls
    _calls = _lib.torch_calls() or _Nothing
    return _calls


def _made(result, name: str) -> bool:
    """Whether the extension made the call; raises the library's error."""
    if result is None:
        return False
    if type(result) is int:
        raise _lib.GdnError(name, result, _lib.strerror(result))
    return True


# Through ctypes: the common case of each check is one chain of comparisons, and the stream
# and device come from torch's cheapest accessors (72 ns against 2.2 us for
# torch.cuda.current_stream).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """One library call on the device's current stream (the last argument)."""
    index = device.index
    if torch.cuda.current_device() == index:
        _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _raw_stream(index))


def _need(t, name: str, dtype: torch.dtype, shape, device) -> None:
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.device == device
            and (shape is None or t.shape == shape) and t.is_contiguous()):
        return
    _check(t, name, dtype, shape, device)


def _check_counter(bad_index_count, device) -> None:
    if bad_index_count is not None:
        _need(bad_index_count, "bad_index_count", _I32, (1,), device)


@lru_cache(maxsize=256)
def _int64s(*values):
    return (ctypes.c_int64 * len(values))(*values)


@lru_cache(maxsize=256)
def _workspace_bytes(name: str, *sizes) -> int:
    return int(getattr(_lib.load(), name)(*sizes))


def _check_cache(cache: torch.Tensor, name: str, dtype, HKV: int, D: int, device):
    if not isinstance(cache, torch.Tensor) or cache.dim() != 4:
        raise ValueError(f"{name} must be 4-D [num_pages, page_size, num_kv_heads, head_dim]")
    if cache.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {cache.dtype}")
    if not cache.is_cuda or cache.device != device:
        raise ValueError(f"{name} is on {cache.device}, expected {device}")
    shape, strides = cache.shape, cache.stride()
    if shape[2] != HKV or shape[3] != D:
        raise ValueError(f"{name} must end in ({HKV}, {D}), got {tuple(shape)}")
    if strides[3] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    strides = tuple(s if n > 1 else 0 for s, n in zip(strides[:3], shape))
    if any(s <= 0 and n > 1 for s, n in zip(strides, shape)):
        raise ValueError(f"{name} must not be expanded (a stride of 0)")
    if (strides[0] | strides[1] | strides[2]) % 8 or cache.data_ptr() % 16:
        raise ValueError(f"{name} needs 16-byte aligned rows (strides a multiple of 8 elements)")
    return strides


def paged_attention_decode(
    q, k_cache, v_cache, block_tables, seq_lens, k=None, v=None, scale=None, window: int = 0,
    num_sinks: int = 0, output=None, bad_index_count=None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention of one new token per sequence over a paged key-value cache.

    q [B,1,HQ,D] bf16 or fp16, D 64, 128 or 256; k_cache, v_cache [num_pages, page_size, HKV, D]
    of the same type, HQ a multiple of HKV, any strides with D contiguous and rows 16-byte
    aligned (so a [pages, HKV, tokens, D] buffer goes in transposed, and so do the halves of
    an interleaved one); block_tables [B, width] int32, rows contiguous; seq_lens [B] int32
    counts each sequence's tokens, the new one included.  With k, v [B,1,HKV,D] the new token's
    rows are attended to and stored into the cache at position ``seq_lens - 1``; without them
    they have to be there already.  ``window`` > 0 leaves the first ``num_sinks`` and the last
    ``window`` tokens visible.  ``scale`` None or 0 is 1/sqrt(D), as in the GDN entries.  Returns
    ``(output [B,1,HQ,D], lse [B,HQ] fp32)``.

    A row of length <= 0 is padding: zeros, lse -inf, nothing stored.  A table entry < 0
    hides its tokens; one >= num_pages does too and is counted in ``bad_index_count`` (an int32
    CUDA tensor of one element), like a length beyond the table, which is cut to it.  The new
    token is seen even when its page is bad, but not stored.  The page of a sequence's last
    token must not be shared, and ``output`` not overlap an input.

    Scores, maxima, sums and the output's sums are fp32; each softmax weight is rounded to the tensors'
    type where it is multiplied with its value (in fp16 times 2^15, so that small ones are not lost),
    and the output once more.  At most 65535 sequences, and B * HQ up to 2**31 // 256.  C entry:
    ``gdn_paged_attention_decode``.
    """
    made = (_calls or _torch_calls()).attend(q, k_cache, v_cache, block_tables, seq_lens, k, v, scale,
                                            window, num_sinks, output, bad_index_count)
    if _made(made, "gdn_paged_attention_decode"):
        return made
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[1] != 1:
        raise ValueError("q must be 4-D [B, 1, heads, head_dim]")
    B, _, HQ, D = q.shape
    dev, dt = q.device, q.dtype
    if dt not in (_BF16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {dt}")
    if D not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {D}")
    _need(q, "q", dt, None, dev)
    HKV = k_cache.shape[2] if isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 else 0
    if HKV < 1 or HQ < 1 or HQ % HKV != 0:
        raise ValueError(f"num heads ({HQ}) must be a multiple of num kv heads ({HKV})")
    ks = _check_cache(k_cache, "k_cache", dt, HKV, D, dev)
    vs = _check_cache(v_cache, "v_cache", dt, HKV, D, dev)
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    num_pages, page_size = k_cache.shape[:2]
    if num_pages < 1 or page_size < 1:
        raise ValueError("the cache must have pages")
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be 2-D [B, width]")
    if block_tables.dtype != _I32:
        raise TypeError(f"block_tables must be torch.int32, got {block_tables.dtype}")
    if block_tables.device != dev:
        raise ValueError(f"block_tables is on {block_tables.device}, expected {dev}")
    if block_tables.shape[0] != B:
        raise ValueError(f"block_tables must have {B} rows, got {block_tables.shape[0]}")
    width = block_tables.shape[1]
    if width > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables must have contiguous rows")
    if width * page_size > 2**31 - 2048:
        raise ValueError("block_tables hold more than 2**31 - 2048 tokens a row")
    _need(seq_lens, "seq_lens", _I32, (B,), dev)
    if (k is None) != (v is None):
        raise ValueError("k and v must be provided together")
    if k is not None:
        _need(k, "k", dt, (B, 1, HKV, D), dev)
        _need(v, "v", dt, (B, 1, HKV, D), dev)
    if window < 0 or num_sinks < 0 or max(window, num_sinks) > 2**30 - 1:
        raise ValueError("window and num_sinks must be between 0 and 2**30 - 1")
    if output is None:
        output = torch.empty_like(q)
    else:
        _need(output, "output", dt, (B, 1, HQ, D), dev)
    _check_counter(bad_index_count, dev)
    lse = q.new_empty((B, HQ), dtype=_F32)
    most = min(width * page_size, window + num_sinks) if window else width * page_size
    nbytes = _workspace_bytes("gdn_paged_attention_workspace_bytes", B, HQ, HKV, D, most)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(
        dev, "gdn_paged_attention_decode", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        block_tables.data_ptr(), seq_lens.data_ptr(), _ptr(k), _ptr(v),
        0.0 if scale is None else float(scale), int(window), int(num_sinks), output.data_ptr(),
        lse.data_ptr(), _ptr(ws), nbytes, _DTYPE_CODES[dt], B, HQ, HKV, D, num_pages, page_size,
        width, block_tables.stride(0) if B > 1 else width, _int64s(*ks), _int64s(*vs),
        _ptr(bad_index_count))
    return output, lse


def beam_select(
    logits, scores, num_selected: Optional[int] = None, finished=None, eos_token: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Beam search's selection: the ``num_selected`` (default: the number of beams) best of all
    beams' continuations of each request.

    logits [B,K,V] bf16, fp16 or fp32, V contiguous; scores [B,K] fp32, the beams' cumulative
    log-probabilities.  Candidate (beam i, token t) scores ``scores[i] + log_softmax(logits[i])[t]``;
    a beam marked in ``finished`` [B,K] bool has the one candidate ``eos_token`` with
    ``scores[i]``.  Returns ``(tokens, parents, new_scores)``, int32, int32 and fp32
    [B,num_selected], best first; equal scores: the lower beam, within a beam the lower token.
    Candidates without a finite score (tokens masked with -inf, beams at -inf, rows that hold
    a NaN or +inf) are never chosen; places left over get -1, -1, -inf.  At most 64 beams,
    64 selected, 2**26 tokens and 2**25 - 1 beams in all.  C entry: ``gdn_beam_select``.
    """
    made = (_calls or _torch_calls()).select(logits, scores, num_selected, finished, eos_token)
    if _made(made, "gdn_beam_select"):
        return made
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3:
        raise ValueError("logits must be 3-D [B, beams, vocab]")
    B, K, V = logits.shape
    dev = logits.device
    if logits.dtype not in _DTYPE_CODES:
        raise TypeError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (the B200 path has no CPU fallback)")
    if K < 1 or V < 1:
        raise ValueError("logits must have at least one beam and one token")
    if V > 1 and logits.stride(2) != 1:
        raise ValueError("logits must be contiguous in the vocabulary")
    n = K if num_selected is None else int(num_selected)
    if n < 1 or n > 64 or K > 64:
        raise ValueError(f"beam_select takes up to 64 beams and 1 to 64 selected, got {K} and {n}")
    _need(scores, "scores", _F32, (B, K), dev)
    if finished is not None:
        _need(finished, "finished", _BOOL, (B, K), dev)
        if not 0 <= eos_token < V:
            raise ValueError(f"eos_token must be a token of the vocabulary, got {eos_token}")
    new_scores = scores.new_empty((B, n))
    tokens = torch.empty_like(new_scores, dtype=_I32)
    parents = torch.empty_like(tokens)
    nbytes = _workspace_bytes("gdn_beam_select_workspace_bytes", B, K, V, n)
    ws = scores.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    stride_batch, stride_beam, _ = logits.stride()
    _call(dev, "gdn_beam_select", logits.data_ptr(), _DTYPE_CODES[logits.dtype], stride_batch,
          stride_beam, scores.data_ptr(), _ptr(finished), int(eos_token), B, K, V, n,
          tokens.data_ptr(), parents.data_ptr(), new_scores.data_ptr(), _ptr(ws), nbytes)
    return tokens, parents, new_scores


class _PoolArrays:
    """The pools of a call as the C arrays of pointers, page bytes and page pitches."""

    def __init__(self, pools: Pools, device=None, num_pages: Optional[int] = None):
        pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
        n = len(pools)
        if n > 32:
            raise ValueError(f"at most 32 pools go through one call, got {n}")
        nbytes, pitch = [], []
        for i, t in enumerate(pools):
            if not isinstance(t, torch.Tensor) or t.dim() < 2:
                raise ValueError(f"pool {i} must be a tensor [num_pages, ...]")
            if not t.is_cuda:
                raise ValueError(f"pool {i} must be a CUDA tensor (the B200 path has no CPU fallback)")
            if device is None:
                device = t.device
            if t.device != device:
                raise ValueError(f"pool {i} is on {t.device}, expected {device}")
            pages, numel = t.shape[0], t.numel()
            if num_pages is None:
                num_pages = pages
            if pages != num_pages or numel < 1:
                raise ValueError(f"pool {i} must have {num_pages} pages, got {tuple(t.shape)}")
            if not t.is_contiguous() and not t[0].is_contiguous():
                raise ValueError(f"pool {i} must be contiguous within a page")
            size = t.element_size()
            nbytes.append(numel // pages * size)
            pitch.append(t.stride(0) * size if pages > 1 else nbytes[i])
        self.device, self.num_pages, self.count = device, num_pages, n
        self.ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in pools]) if n else None
        self.bytes = _int64s(*nbytes) if n else None
        self.pitch = _int64s(*pitch) if n else None


def _check_refcounts(refcounts) -> Tuple[int, torch.device]:
    if not isinstance(refcounts, torch.Tensor) or refcounts.dim() != 1 or refcounts.numel() < 1:
        raise ValueError("refcounts must be a 1-D tensor [num_pages]")
    dev = refcounts.device
    _need(refcounts, "refcounts", _I32, None, dev)
    return refcounts.shape[0], dev


def copy_pages(pools: Pools, src, dst, bad_index_count=None) -> None:
    """``pool[dst[i]] = pool[src[i]]`` for all i at once, in every pool, in place.

    ``pools``: a tensor [num_pages, ...] or up to 32 of them with the same number of pages
    (a pooled state [slots,HV,128,128], the layers of a cache, keys and values), of any type,
    each page contiguous.  src, dst [n] int32 or int64, n <= 4096.  All sources are read as
    they were before the call, so reordering beams within their own slots (a permutation, one
    parent several times) needs no second pool; of equal dst the last pair wins.  A negative
    index skips its pair, one >= num_pages does too and is counted in ``bad_index_count``.
    C entry: ``gdn_copy_pages``.
    """
    made = (_calls or _torch_calls()).copy(pools, src, dst, bad_index_count)
    if _made(made, "gdn_copy_pages"):
        return
    p = _PoolArrays(pools)
    if p.count == 0:
        return
    n = src.shape[0] if isinstance(src, torch.Tensor) and src.dim() == 1 else 0
    src = _index_tensor(src, "src", n, p.device, p.num_pages)
    dst = _index_tensor(dst, "dst", n, p.device, p.num_pages)
    if n > 4096:
        raise ValueError(f"at most 4096 pages are copied by one call, got {n}")
    _check_counter(bad_index_count, p.device)
    _call(p.device, "gdn_copy_pages", p.ptrs, p.bytes, p.pitch, p.count, p.num_pages,
          src.data_ptr(), dst.data_ptr(), n, _ptr(bad_index_count))


def alloc_pages(refcounts, need) -> torch.Tensor:
    """A free page for each marked entry of ``need`` [n] bool: returns pages [n] int32, the
    lowest free pages of ``refcounts`` [num_pages] int32 in order (their count becomes 1);
    -1 where nothing is needed or no page is left.  A page is free when its count is <= 0.
    C entry: ``gdn_alloc_pages``."""
    made = (_calls or _torch_calls()).alloc(refcounts, need)
    if _made(made, "gdn_alloc_pages"):
        return made[0]
    P, dev = _check_refcounts(refcounts)
    if not isinstance(need, torch.Tensor) or need.dim() != 1:
        raise ValueError("need must be a 1-D bool tensor")
    _need(need, "need", _BOOL, None, dev)
    n = need.shape[0]
    pages = refcounts.new_empty(n)
    ws = torch.empty_like(pages)
    _call(dev, "gdn_alloc_pages", refcounts.data_ptr(), P, need.data_ptr(), n, pages.data_ptr(),
          ws.data_ptr(), 4 * n)
    return pages


def free_pages(refcounts, pages, bad_index_count=None) -> None:
    """One reference less in ``refcounts`` for every entry of ``pages`` (int32, any shape,
    contiguous: block-table rows go in as they are, negative entries are skipped).  Entries
    >= num_pages and entries of pages without a reference left are counted in
    ``bad_index_count`` and change nothing.  C entry: ``gdn_free_pages``."""
    made = (_calls or _torch_calls()).release(refcounts, pages, bad_index_count)
    if _made(made, "gdn_free_pages"):
        return
    P, dev = _check_refcounts(refcounts)
    _need(pages, "pages", _I32, None, dev)
    _check_counter(bad_index_count, dev)
    _call(dev, "gdn_free_pages", refcounts.data_ptr(), P, pages.data_ptr(), pages.numel(),
          _ptr(bad_index_count))


def fork_pages(block_tables, seq_lens, parents, refcounts, page_size: int, pools: Pools = (),
               bad_index_count=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Forks (and thereby reorders, multiplies and drops) the sequences of a paged cache.

    Row i of the returned ``(block_tables [n,width], seq_lens [n])`` continues row
    ``parents[i]`` (int32 or int64) of the given ones; rows without a child give their pages
    up.  Full pages are shared: ``refcounts`` [num_pages] int32 is updated in place.  A partly
    filled last page stays with its row's first child; every other child gets the lowest
    free page as a copy of it in all ``pools``.  A negative parent makes an empty row, one
    beyond the rows does too and is counted in ``bad_index_count``, as is a copy for which no
    page was left (its entry becomes -1).  Entries behind a row's tokens are -1.
    C entry: ``gdn_fork_pages``.
    """
    made = (_calls or _torch_calls()).fork(block_tables, seq_lens, parents, refcounts, page_size, pools,
                                          bad_index_count)
    if _made(made, "gdn_fork_pages"):
        return made
    P, dev = _check_refcounts(refcounts)
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be 2-D [rows, width]")
    rows, width = block_tables.shape
    _need(block_tables, "block_tables", _I32, None, dev)
    _need(seq_lens, "seq_lens", _I32, (rows,), dev)
    n = parents.shape[0] if isinstance(parents, torch.Tensor) and parents.dim() == 1 else 0
    parents = _index_tensor(parents, "parents", n, dev, rows)
    if page_size < 1 or width * page_size > 2**31 - 1:
        raise ValueError(f"page_size must be positive and a row below 2**31 tokens, got {page_size}")
    _check_counter(bad_index_count, dev)
    p = _PoolArrays(pools, dev, P)
    new_tables = refcounts.new_empty((n, width))
    new_lens = refcounts.new_empty(n)
    ws = refcounts.new_empty(3 * n)
    _call(
        dev, "gdn_fork_pages", block_tables.data_ptr(), width, seq_lens.data_ptr(),
        parents.data_ptr(), refcounts.data_ptr(), new_tables.data_ptr(), new_lens.data_ptr(),
        rows, n, width, P, int(page_size), p.ptrs, p.bytes, p.pitch, p.count, ws.data_ptr(),
        12 * n, _ptr(bad_index_count))
    return new_tables, new_lens


def compact_pages(refcounts, block_tables=None, pools: Pools = ()) -> Tuple[torch.Tensor, torch.Tensor]:
    """Closes the holes of a pool: afterwards the live pages are the first ``num_live``.

    The k-th live page at or behind ``num_live`` moves to the k-th free page before it, in all
    ``pools``; ``refcounts`` and ``block_tables`` (int32, any shape, contiguous, or None) are
    updated in place.  Returns ``(remap [num_pages] int32, num_live [1] int32)``: each live
    page's new number, -1 for a free one.  C entry: ``gdn_compact_pages``.
    """
    made = (_calls or _torch_calls()).compact(refcounts, block_tables, pools)
    if _made(made, "gdn_compact_pages"):
        return made
    P, dev = _check_refcounts(refcounts)
    entries = 0
    if block_tables is not None:
        _need(block_tables, "block_tables", _I32, None, dev)
        entries = block_tables.numel()
    p = _PoolArrays(pools, dev, P)
    remap = torch.empty_like(refcounts)
    live = refcounts.new_empty(1)
    nws = 2 * (P // 2 + 1) + 1
    ws = refcounts.new_empty(nws)
    _call(dev, "gdn_compact_pages", refcounts.data_ptr(), P,
          block_tables.data_ptr() if entries else None, entries, remap.data_ptr(),
          live.data_ptr(), p.ptrs, p.bytes, p.pitch, p.count, ws.data_ptr(), 4 * nws)
    return remap, live
