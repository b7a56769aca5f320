"""Refusals of the exact-attention entry points that need no GPU: every call here ends in the host's checks,
before any CUDA call, so the pointers are never used."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch

from sva_b200 import _lib, kernels
from tests.test_capi import HEADER

P = 1 << 20  # a 16-byte aligned address that nothing reads


def _cache(**kw):
    c = _lib.Kv4CacheArgs(4, 256, 3, 64, P, P, P, P, None, 0, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _decode(**kw):
    a = _lib.Kv4DecodeArgs(2, 9, 1, _lib.DTYPE_BF16, 200, 0.125, P, 64, 64, 64, None, P, 64, 64, 64, None, None, 0, 0, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _prompt(**kw):
    a = _lib.PromptArgs(1, 9, 3, 64, _lib.DTYPE_BF16, 1, 0.125, 10, 10, P, 576, 64, P, 192, 64, P, 192, 64, P, None, P, 576,
                        64, None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _evict(**kw):
    a = _lib.EvictArgs(2, 3, 1, 0, 200, 100, 10, P, P, 600, 200, P + 4096, 300, 100, 100, 2, 200, 2, 100, None, 0, 0, None, 0,
                       0, P, P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _refused(rc, error, word):
    with pytest.raises(error, match=word):
        _lib.check(rc)


def test_struct_layouts_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for struct, cls in (("sva_prompt_args", _lib.PromptArgs), ("sva_kv4_cache", _lib.Kv4CacheArgs),
                        ("sva_kv4_decode_args", _lib.Kv4DecodeArgs), ("sva_evict_array", _lib.EvictArray),
                        ("sva_evict_args", _lib.EvictArgs)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\} " + struct + ";", text, flags=re.S).group(1)
        want = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
        fields = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind, names = re.match(r"(?:const )?(\w+)(.*)", decl, flags=re.S).groups()
            for name in names.split(","):
                pointer = "*" in names
                fields.append((name.strip(" *\n"), ctypes.c_void_p if pointer else want[kind]))
        assert list(cls._fields_) == fields, struct


@pytest.mark.parametrize("change, error, word", [
    (dict(head_dim=96), ValueError, "head_dim"),
    (dict(page_rows=100), ValueError, "64 rows"),
    (dict(page_rows=0), ValueError, "64 rows"),
    (dict(n_kv_heads=0), ValueError, "pages"),
    (dict(k_params=None), ValueError, "null"),
    (dict(v_codes=P + 8), ValueError, "aligned"),
    (dict(n_pages=1), ValueError, "fewer pages"),
    (dict(page_table=P, page_rows=192, page_table_cols=4), ValueError, "power of two"),
    (dict(page_table=P, page_table_cols=0), ValueError, "page table"),
])
def test_cache_refusals(change, error, word):
    lib, c = _lib.load(), _cache(**change)
    a = _decode(max_len=100)
    assert lib.sva_kv4_decode_workspace_size(ctypes.byref(c), ctypes.byref(a)) == 0
    _refused(lib.sva_kv4_decode(ctypes.byref(c), ctypes.byref(a), None, 0, None), error, word)
    _refused(lib.sva_kv4_read(ctypes.byref(c), P, P, 1, 2, 5, P, None), error, word)
    _refused(lib.sva_kv4_write(ctypes.byref(c), P, 64, 64, 64, P, 64, 64, 64, 1, 2, 5, P, None, None), error, word)


@pytest.mark.parametrize("change, error, word", [
    (dict(n_seqs=0), ValueError, "n_seqs"),
    (dict(n_seqs=70000), ValueError, "n_seqs"),
    (dict(n_heads=10), ValueError, "n_heads"),
    (dict(n_tokens=0), ValueError, "n_tokens"),
    (dict(max_len=257), ValueError, "max_len"),
    (dict(max_len=-1), ValueError, "max_len"),
    (dict(dtype=3), TypeError, "dtype"),
    (dict(query=None), ValueError, "null"),
    (dict(out=None), ValueError, "null"),
    (dict(weights=P), ValueError, "workspace"),
])
def test_decode_refusals(change, error, word):
    lib, c, a = _lib.load(), _cache(), _decode(**change)
    _refused(lib.sva_kv4_decode(ctypes.byref(c), ctypes.byref(a), None, 0, None), error, word)


def test_write_and_read_refusals():
    lib, c = _lib.load(), ctypes.byref(_cache())
    _refused(lib.sva_kv4_write(c, P, 64, 64, 64, P, 64, 64, 64, 7, 2, 5, P, None, None), TypeError, "dtype")
    _refused(lib.sva_kv4_write(c, P, 64, 64, 64, P, 64, 64, 64, 1, 2, -5, P, None, None), ValueError, "n_tokens")
    _refused(lib.sva_kv4_write(c, None, 64, 64, 64, P, 64, 64, 64, 1, 2, 5, P, None, None), ValueError, "null")
    _refused(lib.sva_kv4_read(c, P, P + 2, 1, 2, 5, P, None), ValueError, "aligned")
    _refused(lib.sva_kv4_read(c, P, P, 1, 2, 5, None, None), ValueError, "null")


@pytest.mark.parametrize("change, error, word", [
    (dict(n_heads=10), ValueError, "n_heads"),
    (dict(head_dim=257), ValueError, "head_dim"),
    (dict(head_dim=0), ValueError, "head_dim"),
    (dict(n_rows=1 << 31), ValueError, "row counts"),
    (dict(n_seqs=-1), ValueError, "n_seqs"),
    (dict(dtype=-1), TypeError, "dtype"),
    (dict(cu_seqlens=None), ValueError, "null"),
    (dict(values=None), ValueError, "null"),
])
def test_prompt_refusals(change, error, word):
    lib, a = _lib.load(), _prompt(**change)
    _refused(lib.sva_prompt_attention(ctypes.byref(a), None, 0, None), error, word)


@pytest.mark.parametrize("change, error, word", [
    (dict(n_seqs=0), ValueError, "n_seqs"),
    (dict(n_arrays=9), ValueError, "arrays"),
    (dict(keep=-1), ValueError, "keep"),
    (dict(recent=101), ValueError, "recent"),
    (dict(recent=-1), ValueError, "recent"),
    (dict(max_len=201), ValueError, "source rows"),
    (dict(dst_page_rows=99), ValueError, "destination"),
    (dict(src_pages=1), ValueError, "fewer pages"),
    (dict(dst_weights_width=99), ValueError, "narrower"),
    (dict(dst_weights=P), ValueError, "strides"),
    (dict(seq_lens=None), ValueError, "null"),
])
def test_evict_refusals(change, error, word):
    lib, a = _lib.load(), _evict(**change)
    rows = (_lib.EvictArray * 1)((P, 2 * P, 32, 6400, 3200, 3200, 1600))
    _refused(lib.sva_cache_evict(ctypes.byref(a), rows, P, 1 << 20, None), error, word)


@pytest.mark.parametrize("row, word", [
    ((None, 2 * P, 32, 6400, 3200, 3200, 1600), "null"),
    ((P, 2 * P, 31, 6400, 3200, 3200, 1600), "row_bytes"),
    ((P, 2 * P, 1 << 17, 6400, 3200, 3200, 1600), "row_bytes"),
    ((P + 1, 2 * P, 32, 6400, 3200, 3200, 1600), "aligned"),
    ((P, P, 32, 6400, 3200, 3200, 1600), "in_place"),
])
def test_evict_row_refusals(row, word):
    lib, a = _lib.load(), _evict()
    _refused(lib.sva_cache_evict(ctypes.byref(a), (_lib.EvictArray * 1)(row), P, 1 << 20, None), ValueError, word)
    _refused(lib.sva_cache_evict(ctypes.byref(a), (_lib.EvictArray * 1)((P, 2 * P, 32, 1, 1, 1, 1)), P, 8, None), ValueError,
             "workspace|aligned")


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4])
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.prompt_attention(q, q, q, cu)
    cache = kernels.kv4_empty(1, 2, 64, 64, device="cpu")
    start = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_write(q[None], q[None], cache, start)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_read(cache, start, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.kv4_decode(q[None], cache)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.cache_evict(cache, torch.zeros(1, 2, 64), start, 3)
    for pages, kv, rows, dim in ((1, 1, 63, 64), (1, 1, 0, 64), (1, 1, 64, 96)):
        with pytest.raises(ValueError):
            kernels.kv4_empty(pages, kv, rows, dim, device="cpu")
