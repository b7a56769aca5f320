"""Torch-facing wrappers of the C ABI (CUDA tensors only; no CPU fallback).

Each function checks devices, dtypes and layouts, passes raw device pointers and element
strides to libsva_b200.so on the current CUDA stream, and maps error codes to exceptions.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Sequence

import torch

from . import _lib

_DTYPE_CODE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError as exc:
        raise TypeError(f"sva_b200 supports float32, bfloat16 and float16 tensors, got {dtype}") from exc


def _cuda(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"sva_b200 runs on CUDA devices only; {name} is on {t.device}")
    return t


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_host_ok: dict[int, bool] = {}


def _cuda_or_host(t: torch.Tensor, name: str) -> None:
    """A CUDA tensor, or a page-locked host tensor that device code can address (checked once
    per allocation through sva_host_buffer_device_accessible)."""
    if t.is_cuda:
        return
    if t.device.type == "cpu" and t.is_pinned():
        base = t.untyped_storage().data_ptr()
        ok = _host_ok.get(base)
        if ok is None:
            ok = bool(_lib.load().sva_host_buffer_device_accessible(ctypes.c_void_p(base)))
            _host_ok[base] = ok
        if ok:
            return
    raise ValueError(f"{name} must be a CUDA tensor or a pinned host tensor that the GPU can address")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class Workspace:
    """Grow-only device scratch buffer reused across calls (one per device and purpose)."""

    def __init__(self) -> None:
        self._buf: dict[torch.device, torch.Tensor] = {}

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor | None:
        if nbytes <= 0:
            return None
        buf = self._buf.get(device)
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            self._buf[device] = buf
        return buf


_decode_ws = Workspace()


def tensor_core_write_ok(keys: torch.Tensor, k_proj: torch.Tensor) -> bool:
    """Whether the tcgen05 write path applies: bf16 keys with 16-byte aligned rows, head_dim a
    multiple of 16 up to 128, rank a multiple of 16 up to 64, and a key projection whose values
    are bf16 numbers (so rounding it to bf16 changes nothing)."""
    head_dim, rank = int(keys.shape[-1]), int(k_proj.shape[-1])
    if keys.dtype != torch.bfloat16 or head_dim % 16 or head_dim > 128 or rank % 16 or rank > 64:
        return False
    if keys.data_ptr() % 16 or (keys.stride(-2) * 2) % 16 or (keys.stride(0) * 2) % 16:
        return False
    return bool(torch.equal(k_proj, k_proj.to(torch.bfloat16).to(k_proj.dtype)))


def catalog_encode(keys: torch.Tensor, k_proj: torch.Tensor, codebooks: torch.Tensor, start: int, count: int,
                   k_low: torch.Tensor | None, codes: torch.Tensor | None, n_heads: int | None = None,
                   tensor_cores: bool = False, status: torch.Tensor | None = None) -> None:
    """Write k_low / codes rows [start, start+count) of every query head.

    keys [Hkv, L, D] (rows contiguous), k_proj [H, D, R] fp32, codebooks [H, S, C, R/S] fp32,
    k_low [H, cap, R] fp32 (contiguous rows), codes [H, cap, S] uint8.  ``tensor_cores`` selects
    the tcgen05 projection (sva_catalog_encode_tc; see ``tensor_core_write_ok``) instead of the
    exact sequential-order CUDA-core projection; ``status`` (int32 device scalar) receives its
    timeout flag.
    """
    _cuda(keys, "keys")
    if keys.stride(-1) != 1:
        raise ValueError("keys rows must be contiguous")
    n_heads = int(k_proj.shape[0]) if n_heads is None else n_heads
    n_kv, _, head_dim = keys.shape
    rank = int(k_proj.shape[-1])
    subspaces, codewords = int(codebooks.shape[1]), int(codebooks.shape[2])
    k_proj = k_proj.contiguous()
    codebooks = codebooks.contiguous()
    for name, t in (("k_low", k_low), ("codes", codes)):
        if t is not None:
            _cuda(t, name)
            if not (t.stride(-1) == 1 and t.stride(-2) == t.shape[-1]):
                raise ValueError(f"{name} rows must be contiguous")
    lib = _lib.load()
    common = (keys.data_ptr(), dtype_code(keys.dtype), keys.stride(0), keys.stride(1), n_heads, n_kv, head_dim, rank,
              k_proj.data_ptr(), codebooks.data_ptr(), subspaces, codewords, int(start), int(count), _ptr(k_low),
              0 if k_low is None else k_low.stride(0), _ptr(codes), 0 if codes is None else codes.stride(0))
    if tensor_cores:
        rc = lib.sva_catalog_encode_tc(*common, _ptr(status), _stream(keys.device))
    else:
        rc = lib.sva_catalog_encode(*common, _stream(keys.device))
    _lib.check(rc)


def catalog_encode_at(keys: torch.Tensor, k_proj: torch.Tensor, codebooks: torch.Tensor, start: torch.Tensor,
                      count: int, limit: int, k_low: torch.Tensor, codes: torch.Tensor,
                      n_heads: int | None = None) -> None:
    """catalog_encode of rows [start, start + count) with ``start`` an int64 device scalar read by
    the kernel (sva_catalog_encode_at): capturable in a CUDA graph whose replays append at a moving
    position.  Rows at or beyond ``limit`` are skipped."""
    _cuda(keys, "keys")
    _cuda(start, "start")
    if start.dtype != torch.int64:
        raise TypeError("start must be an int64 tensor")
    if keys.stride(-1) != 1:
        raise ValueError("keys rows must be contiguous")
    n_heads = int(k_proj.shape[0]) if n_heads is None else n_heads
    n_kv, _, head_dim = keys.shape
    for name, t in (("k_low", k_low), ("codes", codes)):
        _cuda(t, name)
        if not (t.stride(-1) == 1 and t.stride(-2) == t.shape[-1]):
            raise ValueError(f"{name} rows must be contiguous")
    rc = _lib.load().sva_catalog_encode_at(
        keys.data_ptr(), dtype_code(keys.dtype), keys.stride(0), keys.stride(1), n_heads, n_kv, head_dim,
        int(k_proj.shape[-1]), k_proj.data_ptr(), codebooks.data_ptr(), int(codebooks.shape[1]),
        int(codebooks.shape[2]), start.data_ptr(), int(count), int(limit), k_low.data_ptr(), k_low.stride(0),
        codes.data_ptr(), codes.stride(0), _stream(keys.device))
    _lib.check(rc)


def assign_centroids(x: torch.Tensor, centroids: torch.Tensor) -> torch.Tensor:
    _cuda(x, "x")
    x = x.float()
    if x.stride(-1) != 1:
        x = x.contiguous()
    cent = centroids.float().contiguous()
    labels = torch.empty(x.shape[0], dtype=torch.int64, device=x.device)
    rc = _lib.load().sva_assign_centroids(x.data_ptr(), x.shape[0], x.shape[1], x.stride(0), cent.data_ptr(),
                                          cent.shape[0], labels.data_ptr(), _stream(x.device))
    _lib.check(rc)
    return labels


def pq_scores(q_low: torch.Tensor, codebooks: torch.Tensor, codes_u8: torch.Tensor, rank_dim: int) -> torch.Tensor:
    _cuda(q_low, "q_low")
    q_low = q_low.float().contiguous()
    codebooks = codebooks.float().contiguous()
    codes_u8 = codes_u8.contiguous()
    n_heads, n_q, _ = q_low.shape
    key_len = int(codes_u8.shape[1])
    out = torch.empty(n_heads, n_q, key_len, dtype=torch.float32, device=q_low.device)
    rc = _lib.load().sva_pq_scores(q_low.data_ptr(), n_heads, n_q, rank_dim, codebooks.data_ptr(),
                                   codebooks.shape[1], codebooks.shape[2], codes_u8.data_ptr(), key_len,
                                   out.data_ptr(), _stream(q_low.device))
    _lib.check(rc)
    return out


def decode_args(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor,
                codes: torch.Tensor, k_low: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, shortlist: int,
                budget: int, softmax_scale: float | None = None, logits_mode: int = 0,
                allowed_len: torch.Tensor | None = None, allowed_mask: torch.Tensor | None = None,
                lut_override: torch.Tensor | None = None, out: torch.Tensor | None = None,
                stats: torch.Tensor | None = None) -> tuple[_lib.DecodeArgs, torch.Tensor]:
    """Validated sva_decode_args for the tensors of a decode call, and the output tensor."""
    for name, t in (("codes", codes), ("k_low", k_low), ("keys", keys), ("values", values)):
        _cuda(t, name)
    dev = codes.device
    _cuda_or_host(q, "q")
    if out is not None:
        _cuda_or_host(out, "out")
    n_heads, n_q, head_dim = q.shape
    n_kv = int(keys.shape[0])
    key_len = int(codes.shape[1])
    rank = int(q_proj.shape[-1])
    if q.stride(-1) != 1 or keys.stride(-1) != 1 or values.stride(-1) != 1:
        raise ValueError("q, keys and values must have contiguous rows")
    if codes.dtype != torch.uint8 or codes.stride(-1) != 1 or codes.stride(-2) != codes.shape[-1]:
        raise ValueError("codes must be uint8 with contiguous [L, S] rows per head")
    if k_low.dtype != torch.float32 or k_low.stride(-1) != 1 or k_low.stride(-2) != rank:
        raise ValueError("k_low must be float32 with contiguous [L, R] rows per head")
    if keys.dtype != q.dtype or values.dtype != q.dtype:
        raise TypeError("q, keys and values must share a dtype")
    if out is None:
        out = torch.empty(n_heads, n_q, head_dim, dtype=q.dtype, device=dev)
    a = _lib.DecodeArgs()
    a.n_heads, a.n_kv_heads, a.n_queries, a.head_dim = n_heads, n_kv, n_q, head_dim
    a.rank_dim, a.subspaces, a.codewords = rank, int(codebooks.shape[1]), int(codebooks.shape[2])
    a.shortlist, a.budget = int(shortlist), int(budget)
    a.qkv_dtype = dtype_code(q.dtype)
    a.logits_mode = int(logits_mode)
    a.softmax_scale = float(head_dim ** -0.5 if softmax_scale is None else softmax_scale)
    a.key_len = key_len
    a.query, a.q_head_stride, a.q_row_stride = q.data_ptr(), q.stride(0), q.stride(1)
    a.q_proj = q_proj.data_ptr()
    a.scale = scale.data_ptr()
    a.codebooks = codebooks.data_ptr()
    a.lut_override = _ptr(lut_override)
    a.codes, a.codes_head_stride = codes.data_ptr(), codes.stride(0)
    a.k_low, a.k_low_head_stride = k_low.data_ptr(), k_low.stride(0)
    a.keys, a.k_head_stride, a.k_row_stride = keys.data_ptr(), keys.stride(0), keys.stride(1)
    a.values, a.v_head_stride, a.v_row_stride = values.data_ptr(), values.stride(0), values.stride(1)
    a.allowed_len = _ptr(allowed_len)
    a.allowed_mask = _ptr(allowed_mask)
    a.mask_row_stride = 0 if allowed_mask is None else allowed_mask.stride(0)
    a.out, a.out_head_stride, a.out_row_stride = out.data_ptr(), out.stride(0), out.stride(1)
    a.stats = _ptr(stats)
    return a, out


def decode(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor, codes: torch.Tensor,
           k_low: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, shortlist: int, budget: int,
           softmax_scale: float | None = None, logits_mode: int = 0, allowed_len: torch.Tensor | None = None,
           allowed_mask: torch.Tensor | None = None, lut_override: torch.Tensor | None = None,
           out: torch.Tensor | None = None, want_shortlist: bool = False, want_final: bool = False,
           stats: torch.Tensor | None = None):
    """Scan summon -> rescore -> verify for H heads x T tokens (see include/sva_b200.h).

    q [H, T, D]; codes [H, L, S] uint8 (rows contiguous); k_low [H, L, R] fp32 (rows
    contiguous); keys/values [Hkv, L, D].  Returns out [H, T, D] (and the shortlist / final
    index tensors when requested, [H, T, shortlist] / [H, T, budget] int32, ascending, -1 padded).
    q and out may be pinned host tensors: the kernels then read q from and write out to host
    memory directly, so a host caller needs no separate copies for them.  A new output is
    allocated on the device of the catalog.
    """
    a, out = decode_args(q, q_proj, scale, codebooks, codes, k_low, keys, values, shortlist, budget, softmax_scale,
                         logits_mode, allowed_len, allowed_mask, lut_override, out, stats)
    dev = codes.device
    n_heads, n_q, _ = q.shape
    sl_out = fin_out = None
    if want_shortlist:
        sl_out = torch.empty(n_heads, n_q, int(shortlist), dtype=torch.int32, device=dev)
        a.shortlist_out = sl_out.data_ptr()
    if want_final:
        fin_out = torch.empty(n_heads, n_q, int(budget), dtype=torch.int32, device=dev)
        a.final_out = fin_out.data_ptr()
    lib = _lib.load()
    ws_bytes = int(lib.sva_decode_workspace_size(ctypes.byref(a)))
    ws = _decode_ws.get(dev, ws_bytes)
    rc = lib.sva_decode(ctypes.byref(a), _ptr(ws), ws_bytes, _stream(dev))
    _lib.check(rc)
    if want_shortlist or want_final:
        return out, sl_out, fin_out
    return out


def batched_args(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor,
                 codes: torch.Tensor, k_low: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, shortlist: int,
                 budget: int, *, seq_lens: torch.Tensor | None = None, page_table: torch.Tensor | None = None,
                 max_len: int | None = None, softmax_scale: float | None = None, logits_mode: int = 0,
                 allowed_len: torch.Tensor | None = None, allowed_mask: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, stats: torch.Tensor | None = None):
    """Validated (sva_decode_args, sva_batch_layout, out) for the tensors of a batched call (see
    decode_batched for the layouts)."""
    for name, t in (("codes", codes), ("k_low", k_low), ("keys", keys), ("values", values)):
        _cuda(t, name)
    _cuda_or_host(q, "q")
    if out is not None:
        _cuda_or_host(out, "out")
    if q.dim() != 4 or codes.dim() != 4 or k_low.dim() != 4 or keys.dim() != 4 or values.dim() != 4:
        raise ValueError("decode_batched takes 4-d q, codes, k_low, keys and values")
    dev = codes.device
    n_seqs, n_heads, n_q, head_dim = q.shape
    n_kv = int(keys.shape[1])
    rank = int(q_proj.shape[-1])
    if q.stride(-1) != 1 or keys.stride(-1) != 1 or values.stride(-1) != 1:
        raise ValueError("q, keys and values must have contiguous rows")
    if codes.dtype != torch.uint8 or codes.stride(-1) != 1 or codes.stride(-2) != codes.shape[-1]:
        raise ValueError("codes must be uint8 with contiguous rows")
    if k_low.dtype != torch.float32 or k_low.stride(-1) != 1 or k_low.stride(-2) != rank:
        raise ValueError("k_low must be float32 with contiguous rows")
    if keys.dtype != q.dtype or values.dtype != q.dtype:
        raise TypeError("q, keys and values must share a dtype")
    paged = page_table is not None
    if paged:
        _cuda(page_table, "page_table")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(-1) != 1:
            raise ValueError("page_table must be an int32 [B, max_pages] tensor with contiguous rows")
        page_keys = int(codes.shape[2])
        if max_len is None:
            max_len = int(page_table.shape[1]) * page_keys
    else:
        page_keys = 0
        if max_len is None:
            max_len = int(codes.shape[2])
    if seq_lens is not None:
        _cuda(seq_lens, "seq_lens")
        if seq_lens.dtype != torch.int64 or seq_lens.numel() != n_seqs:
            raise ValueError("seq_lens must be an int64 tensor of B entries")
    if out is None:
        out = torch.empty(n_seqs, n_heads, n_q, head_dim, dtype=q.dtype, device=dev)
    a = _lib.DecodeArgs()
    a.n_heads, a.n_kv_heads, a.n_queries, a.head_dim = n_heads, n_kv, n_q, head_dim
    a.rank_dim, a.subspaces, a.codewords = rank, int(codebooks.shape[1]), int(codebooks.shape[2])
    a.shortlist, a.budget = int(shortlist), int(budget)
    a.qkv_dtype = dtype_code(q.dtype)
    a.logits_mode = int(logits_mode)
    a.softmax_scale = float(head_dim ** -0.5 if softmax_scale is None else softmax_scale)
    a.key_len = int(max_len)
    a.query, a.q_head_stride, a.q_row_stride = q.data_ptr(), q.stride(1), q.stride(2)
    a.q_proj, a.scale, a.codebooks = q_proj.data_ptr(), scale.data_ptr(), codebooks.data_ptr()
    a.codes, a.codes_head_stride = codes.data_ptr(), codes.stride(1)
    a.k_low, a.k_low_head_stride = k_low.data_ptr(), k_low.stride(1)
    a.keys, a.k_head_stride, a.k_row_stride = keys.data_ptr(), keys.stride(1), keys.stride(2)
    a.values, a.v_head_stride, a.v_row_stride = values.data_ptr(), values.stride(1), values.stride(2)
    a.allowed_len = _ptr(allowed_len)
    a.allowed_mask = _ptr(allowed_mask)
    a.mask_row_stride = 0 if allowed_mask is None else allowed_mask.stride(0)
    a.out, a.out_head_stride, a.out_row_stride = out.data_ptr(), out.stride(1), out.stride(2)
    a.stats = _ptr(stats)
    lay = _lib.BatchLayout()
    lay.n_seqs, lay.page_keys = n_seqs, page_keys
    lay.seq_lens = _ptr(seq_lens)
    lay.page_table = _ptr(page_table)
    lay.page_table_stride = 0 if page_table is None else page_table.stride(0)
    lay.q_seq_stride, lay.out_seq_stride = q.stride(0), out.stride(0)
    lay.codes_page_stride, lay.k_low_page_stride = codes.stride(0), k_low.stride(0)
    lay.k_page_stride, lay.v_page_stride = keys.stride(0), values.stride(0)
    return a, lay, out


def decode_batched(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor,
                   codes: torch.Tensor, k_low: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, shortlist: int,
                   budget: int, *, seq_lens: torch.Tensor | None = None, page_table: torch.Tensor | None = None,
                   max_len: int | None = None, softmax_scale: float | None = None, logits_mode: int = 0,
                   allowed_len: torch.Tensor | None = None, allowed_mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, want_shortlist: bool = False, want_final: bool = False,
                   stats: torch.Tensor | None = None):
    """Scan decode of B sequences in one call (sva_decode_batched, see include/sva_b200.h).

    q [B, H, T, D]; q_proj / scale / codebooks are shared by the sequences (one layer).
    Unpaged (``page_table`` None): codes [B, H, L, S], k_low [B, H, L, R], keys / values
    [B, Hkv, L, D], with L the longest sequence.  Paged: codes [pages, H, page_keys, S], k_low
    [pages, H, page_keys, R], keys / values [pages, Hkv, page_keys, D] page pools and page_table
    [B, max_pages] int32 (page of every page_keys-key block of each sequence).  ``seq_lens`` [B]
    int64 (device) gives each sequence's keys (None: all L, or all ``max_len``); ``max_len`` (host
    int) bounds them (default: L, or max_pages * page_keys).  ``allowed_len`` [B, T] int64 and
    ``allowed_mask`` [B * T, >= L] uint8 as for ``decode``.  Returns out [B, H, T, D] (and
    shortlist / final index tensors [B, H, T, shortlist] / [B, H, T, budget] when requested).
    As for ``decode``, q and out may be page-locked host tensors that the GPU can address.
    """
    a, lay, out = batched_args(q, q_proj, scale, codebooks, codes, k_low, keys, values, shortlist, budget,
                               seq_lens=seq_lens, page_table=page_table, max_len=max_len,
                               softmax_scale=softmax_scale, logits_mode=logits_mode, allowed_len=allowed_len,
                               allowed_mask=allowed_mask, out=out, stats=stats)
    dev = codes.device
    n_seqs, n_heads, n_q, _ = q.shape
    sl_out = fin_out = None
    if want_shortlist:
        sl_out = torch.empty(n_seqs, n_heads, n_q, int(shortlist), dtype=torch.int32, device=dev)
        a.shortlist_out = sl_out.data_ptr()
    if want_final:
        fin_out = torch.empty(n_seqs, n_heads, n_q, int(budget), dtype=torch.int32, device=dev)
        a.final_out = fin_out.data_ptr()
    lib = _lib.load()
    ws_bytes = int(lib.sva_decode_batched_workspace_size(ctypes.byref(a), ctypes.byref(lay)))
    ws = _decode_ws.get(dev, ws_bytes)
    rc = lib.sva_decode_batched(ctypes.byref(a), ctypes.byref(lay), _ptr(ws), ws_bytes, _stream(dev))
    _lib.check(rc)
    if want_shortlist or want_final:
        return out, sl_out, fin_out
    return out


def sva_scale(logit_scale: torch.Tensor) -> torch.Tensor:
    """clamp(exp(logit_scale), 0.01, 100) computed as the reference does (sva/llama.py:69-73)."""
    return logit_scale.detach().float().exp().clamp(0.01, 100.0)


def sqrt_rank(rank_dim: int) -> float:
    return math.sqrt(rank_dim)


_post_ws = Workspace()
_inv_ws = Workspace()


class Postings:
    """Device posting lists of one catalog: CSR (sva_postings_build) or, with ``cap``, the padded
    layout of sva_postings_append (cell c of every (head, subspace) owns ``cap`` id slots)."""

    def __init__(self, counts, offsets, ids, max_bucket, key_len: int, cap: int | None = None):
        self.counts, self.offsets, self.ids, self.max_bucket = counts, offsets, ids, max_bucket
        self.key_len = int(key_len)
        self.cap = cap
        self.overflow = None


def postings_build(codes: torch.Tensor, codewords: int, key_len: int | None = None) -> Postings:
    """Posting lists of keys [0, key_len) of codes [H, L, S] uint8 (reference sva/llama.py:626-657)."""
    _cuda(codes, "codes")
    if codes.dtype != torch.uint8 or codes.stride(-1) != 1 or codes.stride(-2) != codes.shape[-1]:
        raise ValueError("codes must be uint8 with contiguous [L, S] rows per head")
    n_heads, cap, subspaces = codes.shape
    key_len = cap if key_len is None else int(key_len)
    dev = codes.device
    counts = torch.empty(n_heads, subspaces, codewords, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_heads, subspaces, codewords + 1, dtype=torch.int32, device=dev)
    ids = torch.empty(n_heads, subspaces, max(key_len, 1), dtype=torch.int32, device=dev)
    max_bucket = torch.empty(1, dtype=torch.int32, device=dev)
    lib = _lib.load()
    ws_bytes = int(lib.sva_postings_workspace_size(n_heads, subspaces, codewords, key_len))
    ws = _post_ws.get(dev, ws_bytes)
    rc = lib.sva_postings_build(codes.data_ptr(), codes.stride(0), n_heads, subspaces, codewords, key_len,
                                counts.data_ptr(), offsets.data_ptr(), ids.data_ptr(), ids.shape[-1],
                                max_bucket.data_ptr(), _ptr(ws), ws_bytes, _stream(dev))
    _lib.check(rc)
    return Postings(counts, offsets, ids, max_bucket, key_len)


def postings_padded(codes: torch.Tensor, codewords: int, key_len: int, cap: int | None = None) -> Postings:
    """Posting lists of keys [0, key_len) in the padded layout with ``cap`` slots per cell (at least
    the largest list; None: twice the largest list, at least 64 more): the CSR build, then each
    list moved to its cell's slots.  Reads the largest list size on the host."""
    csr = postings_build(codes, codewords, key_len=key_len)
    largest = int(csr.max_bucket.item())
    if cap is None:
        cap = max(2 * largest, largest + 64)
    if largest > cap:
        raise ValueError(f"postings_padded: the largest list has {largest} keys, more than cap={cap}")
    n_heads, subspaces, _ = csr.counts.shape
    dev = codes.device
    offsets = (torch.arange(codewords + 1, device=dev, dtype=torch.int32) * cap).expand(n_heads, subspaces, -1)
    offsets = offsets.contiguous()
    ids = torch.zeros(n_heads, subspaces, codewords * cap, dtype=torch.int32, device=dev)
    if key_len > 0:
        pos = torch.arange(key_len, device=dev, dtype=torch.int32).expand(n_heads, subspaces, -1).contiguous()
        # cell of every CSR position, and its slot inside the cell
        cell = torch.searchsorted(csr.offsets[..., 1:].contiguous(), pos, right=True)
        slot = pos - torch.gather(csr.offsets, 2, cell)
        ids.scatter_(2, (cell * cap + slot).to(torch.int64), csr.ids[..., :key_len])
    out = Postings(csr.counts, offsets, ids, csr.max_bucket, key_len, cap=int(cap))
    out.overflow = torch.zeros(1, dtype=torch.int32, device=dev)
    out.largest_at_build = largest
    return out


def postings_append(codes: torch.Tensor, postings: Postings, start: int, count: int) -> None:
    """Appends keys [start, start + count) of codes [H, L, S] to padded posting lists in place
    (sva_postings_append; reference sva/llama.py:659-693)."""
    if postings.cap is None:
        raise ValueError("postings_append needs the padded layout (postings_padded)")
    n_heads, _, subspaces = codes.shape
    codewords = int(postings.counts.shape[-1])
    rc = _lib.load().sva_postings_append(codes.data_ptr(), codes.stride(0), n_heads, subspaces, codewords, int(start),
                                         int(count), postings.counts.data_ptr(), postings.offsets.data_ptr(),
                                         postings.ids.data_ptr(), postings.ids.shape[-1],
                                         postings.max_bucket.data_ptr(), postings.overflow.data_ptr(),
                                         _stream(codes.device))
    _lib.check(rc)
    postings.key_len = int(start + count)


def inverted_args(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor,
                  codes: torch.Tensor, postings: Postings, k_low: torch.Tensor, keys: torch.Tensor,
                  values: torch.Tensor, budget: int, cells: int, min_budget: int, mid_budget: int,
                  low_margin: float = 0.35, high_margin: float = 0.70, dynamic: bool = False, refill_factor: int = 2,
                  allowed_len: int | None = None, allowed_mask: torch.Tensor | None = None,
                  softmax_scale: float | None = None, out: torch.Tensor | None = None,
                  stats: torch.Tensor | None = None, max_bucket: torch.Tensor | None = None):
    """Validated (sva_inverted_args, out) for decode_inverted's tensors; ``max_bucket`` (device int32)
    overrides the postings' own largest bucket (the shards pass the global one)."""
    for name, t in (("q", q), ("codes", codes), ("k_low", k_low), ("keys", keys), ("values", values)):
        _cuda(t, name)
    dev = q.device
    n_heads, head_dim = q.shape
    key_len = int(k_low.shape[1])
    if out is None:
        out = torch.empty(n_heads, head_dim, dtype=q.dtype, device=dev)
    a = _lib.InvertedArgs()
    a.n_heads, a.n_kv_heads, a.head_dim = n_heads, int(keys.shape[0]), head_dim
    a.rank_dim, a.subspaces, a.codewords = int(q_proj.shape[-1]), int(codebooks.shape[1]), int(codebooks.shape[2])
    a.budget, a.cells, a.refill_factor, a.dynamic = int(budget), int(cells), int(refill_factor), int(bool(dynamic))
    a.min_budget, a.mid_budget = int(min_budget), int(mid_budget)
    a.qkv_dtype = dtype_code(q.dtype)
    a.low_margin, a.high_margin = float(low_margin), float(high_margin)
    a.softmax_scale = float(head_dim ** -0.5 if softmax_scale is None else softmax_scale)
    a.key_len = key_len
    a.postings_len = postings.key_len
    a.allowed_len = key_len if allowed_len is None else int(allowed_len)
    a.allowed_mask = _ptr(allowed_mask)
    a.query, a.q_head_stride = q.data_ptr(), q.stride(0)
    a.q_proj, a.scale, a.codebooks = q_proj.data_ptr(), scale.data_ptr(), codebooks.data_ptr()
    a.codes, a.codes_head_stride = codes.data_ptr(), codes.stride(0)
    a.post_counts, a.post_offsets = postings.counts.data_ptr(), postings.offsets.data_ptr()
    a.post_ids, a.post_ids_sub_stride = postings.ids.data_ptr(), postings.ids.shape[-1]
    a.max_bucket = (postings.max_bucket if max_bucket is None else max_bucket).data_ptr()
    a.k_low, a.k_low_head_stride = k_low.data_ptr(), k_low.stride(0)
    a.keys, a.k_head_stride, a.k_row_stride = keys.data_ptr(), keys.stride(0), keys.stride(1)
    a.values, a.v_head_stride, a.v_row_stride = values.data_ptr(), values.stride(0), values.stride(1)
    a.out, a.out_head_stride = out.data_ptr(), out.stride(0)
    a.stats = _ptr(stats)
    return a, out


def decode_inverted(q: torch.Tensor, q_proj: torch.Tensor, scale: torch.Tensor, codebooks: torch.Tensor,
                    codes: torch.Tensor, postings: Postings, k_low: torch.Tensor, keys: torch.Tensor,
                    values: torch.Tensor, budget: int, cells: int, min_budget: int, mid_budget: int,
                    low_margin: float = 0.35, high_margin: float = 0.70, dynamic: bool = False,
                    refill_factor: int = 2, allowed_len: int | None = None, allowed_mask: torch.Tensor | None = None,
                    softmax_scale: float | None = None,
                    out: torch.Tensor | None = None, want_selection: bool = False, stats: torch.Tensor | None = None):
    """Inverted-index decode of one token per head (reference sva/llama.py:427-576 / :330-425).

    q [H, D]; codes [H, >=postings_len, S]; k_low [H, L, R]; keys/values [Hkv, L, D].  ``budget``,
    ``min_budget`` and ``mid_budget`` are already clamped as the reference clamps them.
    """
    a, out = inverted_args(q, q_proj, scale, codebooks, codes, postings, k_low, keys, values, budget, cells,
                           min_budget, mid_budget, low_margin, high_margin, dynamic, refill_factor, allowed_len,
                           allowed_mask, softmax_scale, out, stats)
    dev = q.device
    n_heads = q.shape[0]
    sel = None
    if want_selection:
        sel = (torch.empty(n_heads, int(budget), dtype=torch.int32, device=dev),
               torch.empty(n_heads, int(budget), dtype=torch.uint8, device=dev),
               torch.empty(n_heads, int(budget), dtype=torch.float32, device=dev),
               torch.empty(n_heads, dtype=torch.int32, device=dev))
        a.sel_idx_out, a.sel_valid_out, a.sel_score_out, a.budget_out = (t.data_ptr() for t in sel)
    lib = _lib.load()
    ws_bytes = int(lib.sva_inverted_workspace_size(ctypes.byref(a)))
    if ws_bytes == 0:
        raise ValueError("sva_b200: invalid inverted decode arguments")
    ws = _inv_ws.get(dev, ws_bytes)
    rc = lib.sva_decode_inverted(ctypes.byref(a), _ptr(ws), ws_bytes, _stream(dev))
    _lib.check(rc)
    return (out, *sel) if want_selection else out


def top_unique(candidate_idx: torch.Tensor, candidate_scores: torch.Tensor, candidate_valid: torch.Tensor,
               budget: int, refill_factor: int = 2):
    """Refill-and-dedupe selection on explicit rows (reference sva/llama.py:83-116)."""
    for name, t in (("candidate_idx", candidate_idx), ("candidate_scores", candidate_scores),
                    ("candidate_valid", candidate_valid)):
        _cuda(t, name)
    dev = candidate_idx.device
    rows, width = candidate_idx.shape
    idx = candidate_idx.to(torch.int64).contiguous()
    scores = candidate_scores.to(torch.float32).contiguous()
    valid = candidate_valid.to(torch.uint8).contiguous()
    if width == 0 or budget <= 0:
        return candidate_idx[:, :0], candidate_scores[:, :0], candidate_valid[:, :0], 0
    refill = min(width, max(budget, budget * refill_factor))
    sel_count = min(budget, refill)
    sel_idx = torch.empty(rows, sel_count, dtype=torch.int64, device=dev)
    sel_scores = torch.empty(rows, sel_count, dtype=torch.float32, device=dev)
    sel_valid = torch.empty(rows, sel_count, dtype=torch.uint8, device=dev)
    refill_out = ctypes.c_int32(0)
    rc = _lib.load().sva_top_unique(idx.data_ptr(), scores.data_ptr(), valid.data_ptr(), rows, width, int(budget),
                                    int(refill_factor), sel_idx.data_ptr(), sel_scores.data_ptr(), sel_valid.data_ptr(),
                                    ctypes.byref(refill_out), _stream(dev))
    _lib.check(rc)
    return sel_idx, sel_scores.to(candidate_scores.dtype), sel_valid.bool(), int(refill_out.value)


# ------------------------------------------------------------------------------------------
# attention over every key: whole prompts, a 4-bit cache, eviction
# ------------------------------------------------------------------------------------------


def _same_device(dev: torch.device, **tensors: torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            if not t.is_cuda:
                _cuda(t, name)
            raise ValueError(f"{name} is on {t.device}, the call's other tensors on {dev}")


def _call(dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) with ``dev`` as the current device, on its current stream."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc)


def _scratch(dev: torch.device, nbytes: int) -> torch.Tensor | None:
    """Workspace of one call.  It comes from torch's allocator at every call, so that calls on two
    streams, and graphs captured apart, never share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None


def _int64(t: torch.Tensor, name: str, n: int) -> int:
    if t.dtype != torch.int64 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int64 tensor of {n} entries")
    return t.data_ptr()


def _page_table(t: torch.Tensor | None, n_seqs: int) -> tuple:
    """(pointer, row stride, columns) of a page table, or of none."""
    if t is None:
        return None, 0, 0
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != n_seqs or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"page_table must be an int32 [{n_seqs}, max_pages] tensor with contiguous rows")
    return t.data_ptr(), t.stride(0), t.shape[1]


def prompt_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     cu_seqlens_k: torch.Tensor | None = None, causal: bool = True, softmax_scale: float | None = None,
                     out: torch.Tensor | None = None, want_lse: bool = False, status: torch.Tensor | None = None):
    """Attention over whole prompts packed without padding (sva_prompt_attention).

    q [N, H, D]; keys / values [Nk, Hkv, D] (any strides with contiguous rows; H a multiple of Hkv, D <= 256);
    ``cu_seqlens`` [B + 1] int64 on the device: sequence b owns query rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1, and key rows likewise by ``cu_seqlens_k`` (None: the same).  With Lq query and Lk key
    rows, query i sees keys j <= i + Lk - Lq, so new tokens may follow a cached beginning; ``causal``
    False: all Lk.  A query that sees no key gets zeros; rows behind the last sequence are left as they
    were.  Returns out [N, H, D] (and the log-sum-exp [H, N] fp32 with ``want_lse``).  bf16 and fp16
    rows of D <= 128 channels, a multiple of 8, run on the tensor cores when every stride is a multiple of 16
    bytes; other calls on the CUDA cores in fp32.  ``status`` (int32 device scalar) receives a timeout flag.
    """
    _cuda(q, "q")
    dev = q.device
    _same_device(dev, keys=keys, values=values, cu_seqlens=cu_seqlens, cu_seqlens_k=cu_seqlens_k, out=out, status=status)
    if q.dim() != 3 or keys.dim() != 3 or values.shape != keys.shape or keys.shape[2] != q.shape[2]:
        raise ValueError("prompt_attention takes q [N, H, D] and keys / values [Nk, Hkv, D]")
    if keys.dtype != q.dtype or values.dtype != q.dtype:
        raise TypeError("q, keys and values must share a dtype")
    n, n_heads, head_dim = q.shape
    if head_dim > 1 and (q.stride(2) != 1 or keys.stride(2) != 1 or values.stride(2) != 1):
        raise ValueError("q, keys and values must have contiguous rows")
    n_seqs = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
    if n_seqs < 0:
        raise ValueError("cu_seqlens must be a [B + 1] tensor")
    if cu_seqlens_k is None and keys.shape[0] != n:
        raise ValueError("cu_seqlens_k is needed where queries and keys differ in number")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or (head_dim > 1 and out.stride(2) != 1):
        raise ValueError("out must have q's shape and dtype, with contiguous rows")
    lse = torch.full((n_heads, n), float("-inf"), dtype=torch.float32, device=dev) if want_lse else None
    a = _lib.PromptArgs(n_seqs, n_heads, keys.shape[1], head_dim, dtype_code(q.dtype), int(causal),
                        head_dim ** -0.5 if softmax_scale is None else softmax_scale, n, keys.shape[0],
                        q.data_ptr(), q.stride(0), q.stride(1), keys.data_ptr(), keys.stride(0), keys.stride(1),
                        values.data_ptr(), values.stride(0), values.stride(1),
                        _int64(cu_seqlens, "cu_seqlens", n_seqs + 1),
                        None if cu_seqlens_k is None else _int64(cu_seqlens_k, "cu_seqlens_k", n_seqs + 1),
                        out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), _ptr(status))
    lib = _lib.load()
    ref = ctypes.byref(a)
    nbytes = lib.sva_prompt_attention_workspace_size(ref)
    ws = _scratch(dev, nbytes)
    _call(dev, lib.sva_prompt_attention, ref, _ptr(ws), nbytes)
    return (out, lse) if want_lse else out


class Kv4Cache(NamedTuple):
    """A key/value cache in 4 bits (see include/sva_b200.h for the format): codes [pages, Hkv, rows, D / 2]
    uint8 and parameters [pages, Hkv, rows, D / 32, 2] bf16 (scale, minimum) of the keys and of the values.
    A page is a sequence when calls get no page table."""

    k_codes: torch.Tensor
    k_params: torch.Tensor
    v_codes: torch.Tensor
    v_params: torch.Tensor


def kv4_empty(pages: int, n_kv_heads: int, rows: int, head_dim: int, device="cuda") -> Kv4Cache:
    """An uninitialised 4-bit cache of ``pages`` pages (or sequences) of ``rows`` rows (a multiple of 64)."""
    if head_dim not in (64, 128):
        raise ValueError("a 4-bit cache takes head_dim 64 or 128")
    if rows <= 0 or rows % 64:
        raise ValueError("rows must be a positive multiple of 64")
    return Kv4Cache(*(torch.empty(pages, n_kv_heads, rows, *tail, dtype=dtype, device=device)
                      for tail, dtype in (((head_dim // 2,), torch.uint8), ((head_dim // 32, 2), torch.bfloat16)) * 2))


def _kv4_args(cache: Kv4Cache, n_seqs: int, page_table: torch.Tensor | None) -> _lib.Kv4CacheArgs:
    kc, kp, vc, vp = cache
    dev = _cuda(kc, "k_codes").device
    _same_device(dev, k_params=kp, v_codes=vc, v_params=vp, page_table=page_table)
    if kc.dim() != 4 or kc.dtype != torch.uint8 or vc.dtype != torch.uint8 or vc.shape != kc.shape:
        raise ValueError("codes must be uint8 [pages, Hkv, rows, D / 2]")
    pages, n_kv, rows, half = kc.shape
    tail = (pages, n_kv, rows, half // 16, 2)
    if kp.dtype != torch.bfloat16 or vp.dtype != torch.bfloat16 or kp.shape != tail or vp.shape != tail:
        raise ValueError("parameters must be bfloat16 [pages, Hkv, rows, D / 32, 2]")
    if not (kc.is_contiguous() and kp.is_contiguous() and vc.is_contiguous() and vp.is_contiguous()):
        raise ValueError("the cache's tensors must be contiguous")
    return _lib.Kv4CacheArgs(pages, rows, n_kv, half * 2, kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(),
                             *_page_table(page_table, n_seqs))


def kv4_write(keys: torch.Tensor, values: torch.Tensor, cache: Kv4Cache, start: torch.Tensor, *,
              page_table: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None) -> None:
    """Quantises rows into the 4-bit cache (sva_kv4_write).

    keys / values [B, Hkv, T, D]: token t of sequence b goes to position start[b] + t; or packed
    [N, Hkv, D] with ``cu_seqlens`` [B + 1]: row n of sequence b goes to start[b] + n - cu_seqlens[b], and rows of no
    sequence are skipped.  ``start`` [B] int64 on the device, so that a captured graph may append at a moving
    position.  Positions outside the cache are skipped.
    """
    _cuda(keys, "keys")
    packed = cu_seqlens is not None
    if keys.dim() != (3 if packed else 4) or values.shape != keys.shape:
        raise ValueError("kv4_write takes keys and values [B, Hkv, T, D], or [N, Hkv, D] with cu_seqlens")
    if values.dtype != keys.dtype:
        raise TypeError("keys and values must share a dtype")
    dev = keys.device
    _same_device(dev, values=values, start=start, cu_seqlens=cu_seqlens, k_codes=cache.k_codes)
    if keys.stride(-1) != 1 or values.stride(-1) != 1:
        raise ValueError("keys and values must have contiguous rows")
    n_seqs = start.shape[0] if start.dim() == 1 else -1
    c = _kv4_args(cache, n_seqs, page_table)
    if keys.shape[1] != c.n_kv_heads or keys.shape[-1] != c.head_dim or (not packed and keys.shape[0] != n_seqs):
        raise ValueError("keys do not match the cache's heads, head_dim or start's sequences")
    order = (lambda t: (0, t.stride(1), t.stride(0))) if packed else (lambda t: t.stride()[:3])
    if n_seqs == 0 or keys.numel() == 0:
        return
    _call(dev, _lib.load().sva_kv4_write, ctypes.byref(c), keys.data_ptr(), *order(keys), values.data_ptr(),
          *order(values), dtype_code(keys.dtype), n_seqs, keys.shape[0] if packed else keys.shape[2],
          _int64(start, "start", n_seqs), None if cu_seqlens is None else _int64(cu_seqlens, "cu_seqlens", n_seqs + 1))


def kv4_read(cache: Kv4Cache, start: torch.Tensor, count: int, *, dtype: torch.dtype = torch.bfloat16,
             page_table: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions start[b] .. start[b] + count - 1 of every sequence back in ``dtype`` (sva_kv4_read): keys and
    values [B, Hkv, count, D]; zeros where a position lies outside the cache.  ``start`` [B] int64, device."""
    dev = _cuda(cache.k_codes, "k_codes").device
    _same_device(dev, start=start)
    n_seqs = start.shape[0] if start.dim() == 1 else -1
    c = _kv4_args(cache, n_seqs, page_table)
    if count < 0:
        raise ValueError("count must not be negative")
    code = dtype_code(dtype)
    out = torch.empty(2, n_seqs, c.n_kv_heads, count, c.head_dim, dtype=dtype, device=dev)
    if out.numel() > 0:
        _call(dev, _lib.load().sva_kv4_read, ctypes.byref(c), out[0].data_ptr(), out[1].data_ptr(), code, n_seqs, count,
              _int64(start, "start", n_seqs))
    return out[0], out[1]


def kv4_decode(q: torch.Tensor, cache: Kv4Cache, *, seq_lens: torch.Tensor | None = None,
               page_table: torch.Tensor | None = None, max_len: int | None = None, softmax_scale: float | None = None,
               out: torch.Tensor | None = None, weights: torch.Tensor | None = None, want_lse: bool = False,
               status: torch.Tensor | None = None):
    """Attention of each sequence's newest T tokens over its whole 4-bit cache (sva_kv4_decode).

    q [B, H, T, D] (contiguous rows).  Sequence b holds ``seq_lens[b]`` keys, the T new ones among them ([B] int64
    on the device; None: ``max_len``), and its token t sees the first seq_lens[b] - T + t + 1.  ``max_len`` (host)
    bounds the lengths (default: the cache's capacity).  ``weights`` [B, Hkv, >= max_len] fp32: every key's softmax
    weight, summed over the tokens and the heads that share its kv head, is added in place (``cache_evict``
    goes by these sums).  Returns out [B, H, T, D] (and the log-sum-exp [B, H, T] fp32 with ``want_lse``).
    A token that sees no key gets zeros.
    """
    _cuda(q, "q")
    dev = q.device
    if q.dim() != 4:
        raise ValueError("kv4_decode takes q [B, H, T, D]")
    n_seqs, n_heads, n_tokens, head_dim = q.shape
    _same_device(dev, k_codes=cache.k_codes, seq_lens=seq_lens, out=out, weights=weights, status=status)
    c = _kv4_args(cache, n_seqs, page_table)
    if head_dim != c.head_dim or q.stride(3) != 1:
        raise ValueError("q must have contiguous rows of the cache's head_dim")
    if max_len is None:
        max_len = c.page_rows * (c.page_table_cols if page_table is not None else 1)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(3) != 1:
        raise ValueError("out must have q's shape and dtype, with contiguous rows")
    if weights is not None and (weights.dtype != torch.float32 or weights.dim() != 3 or weights.stride(2) != 1
                                or weights.shape[:2] != (n_seqs, c.n_kv_heads) or weights.shape[2] < max_len):
        raise ValueError("weights must be float32 [B, Hkv, >= max_len] with contiguous rows")
    lse = torch.empty(n_seqs, n_heads, n_tokens, dtype=torch.float32, device=dev) if want_lse else None
    a = _lib.Kv4DecodeArgs(n_seqs, n_heads, n_tokens, dtype_code(q.dtype), max_len,
                           head_dim ** -0.5 if softmax_scale is None else softmax_scale, q.data_ptr(), *q.stride()[:3],
                           None if seq_lens is None else _int64(seq_lens, "seq_lens", n_seqs), out.data_ptr(),
                           *out.stride()[:3], _ptr(lse), _ptr(weights),
                           *((0, 0) if weights is None else weights.stride()[:2]), _ptr(status))
    if q.numel() > 0:
        lib = _lib.load()
        refs = ctypes.byref(c), ctypes.byref(a)
        nbytes = lib.sva_kv4_decode_workspace_size(*refs)
        ws = _scratch(dev, nbytes)
        _call(dev, lib.sva_kv4_decode, *refs, _ptr(ws), nbytes)
    return (out, lse) if want_lse else out


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First byte of a tensor and the byte behind its last."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def cache_evict(rows: Sequence[torch.Tensor], weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, *,
                recent: int = 0, page_table: torch.Tensor | None = None, out: Sequence[torch.Tensor] | None = None,
                out_weights: torch.Tensor | None = None, out_page_table: torch.Tensor | None = None):
    """Cuts each sequence's cache down to ``keep`` rows a kv head by accumulated weight (sva_cache_evict).

    ``rows``: up to 8 tensors [pages, Hkv, page_rows, ...] (keys, values, or the members of a ``Kv4Cache``), rows
    contiguous; without a page table a page is a sequence.  ``weights`` [B, Hkv, >= longest] fp32 (as ``kv4_decode``
    sums them) and ``seq_lens`` [B] int64.  A sequence of at most ``keep`` rows keeps all of them; else the last
    ``recent`` rows stay and, of the others, those with the largest weights (ties: the first; NaN counts as
    the largest).  Rows that stay move together in their order, with their weights; weights behind them
    become 0.  In place, unless ``out`` (and then ``out_weights``, ``out_page_table``) name another cache; in place no
    page may belong to two sequences.  Returns (kept [B, Hkv, keep] int32: the old positions, ascending,
    -1 padded; lengths [B] int64).  Append new rows at the returned lengths, and keep the model's own position
    count for rotary embeddings: rows are not re-rotated.
    """
    _cuda(weights, "weights")
    dev = weights.device
    in_place = out is None
    if in_place and (out_weights is not None or out_page_table is not None):
        raise ValueError("out_weights and out_page_table go with out")
    if not in_place and out_weights is None:
        raise ValueError("out needs out_weights")
    src = list(rows)
    dst = src if in_place else list(out)
    if not 1 <= len(src) <= _lib.EVICT_MAX_ARRAYS or len(dst) != len(src):
        raise ValueError("cache_evict takes 1 to 8 row tensors, and as many outputs")
    dst_weights = weights if in_place else out_weights
    dst_table = page_table if in_place else out_page_table
    n_seqs = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    n_kv = src[0].shape[1] if src[0].dim() >= 3 else -1
    _same_device(dev, seq_lens=seq_lens, page_table=page_table, out_weights=dst_weights, out_page_table=dst_table)
    for name, w in (("weights", weights), ("out_weights", dst_weights)):
        if w.dtype != torch.float32 or w.dim() != 3 or w.shape[:2] != (n_seqs, n_kv) or w.stride(2) != 1:
            raise ValueError(f"{name} must be float32 [B, Hkv, width] with contiguous rows")
    arrays = (_lib.EvictArray * len(src))()
    for i, (s, d) in enumerate(zip(src, dst)):
        _same_device(dev, rows=s, out=d)
        for t, like in ((s, src[0]), (d, dst[0])):
            if t.dim() < 3 or t.shape[:3] != like.shape[:3] or t.shape[1] != n_kv or not t[0, 0].is_contiguous():
                raise ValueError("rows must be [pages, Hkv, page_rows, ...] tensors of one shape with contiguous rows")
        if s.dtype != d.dtype or s.shape[3:] != d.shape[3:]:
            raise ValueError("out must have rows of the same shape and dtype")
        if not in_place and (any(_overlap(d, t) for t in src) or any(_overlap(d, t) for t in dst[:i])):
            raise ValueError("out must not overlap rows or itself")
        size = s.element_size()
        arrays[i] = (s.data_ptr(), d.data_ptr(), math.prod(s.shape[3:]) * size, s.stride(0) * size, s.stride(1) * size,
                     d.stride(0) * size, d.stride(1) * size)
    if not in_place and _overlap(weights, dst_weights):
        raise ValueError("out_weights must not overlap weights")
    kept = torch.empty(n_seqs, n_kv, max(keep, 0), dtype=torch.int32, device=dev)
    lens = torch.empty(n_seqs, dtype=torch.int64, device=dev)
    rows_of = (lambda t, table: t.shape[2] * (table.shape[1] if table is not None else 1))
    a = _lib.EvictArgs(n_seqs, n_kv, len(src), int(in_place), min(weights.shape[2], rows_of(src[0], page_table)), keep, recent,
                       _int64(seq_lens, "seq_lens", n_seqs), weights.data_ptr(), weights.stride(0), weights.stride(1),
                       dst_weights.data_ptr(), dst_weights.stride(0), dst_weights.stride(1), dst_weights.shape[2],
                       src[0].shape[0], src[0].shape[2], dst[0].shape[0], dst[0].shape[2],
                       *_page_table(page_table, n_seqs), *_page_table(dst_table, n_seqs), kept.data_ptr(),
                       lens.data_ptr())
    if n_seqs > 0:
        lib = _lib.load()
        ref = ctypes.byref(a)
        nbytes = lib.sva_cache_evict_workspace_size(ref)
        ws = _scratch(dev, nbytes)
        _call(dev, lib.sva_cache_evict, ref, arrays, _ptr(ws), nbytes)
    return kept, lens
