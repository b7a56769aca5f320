"""The 4-bit cache and its attention where they can go wrong: groups without a scale, scales of very different size, values
that only some of the new tokens see, channels next to half steps, outputs and weights that overlap themselves.

The references and bounds are those of ``test_gpu_exact_attention``; what a test adds to them is derived beside it.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_exact_attention import DEV, HALF, _check, _check_decode, _decode_case, _fp32_share, _gen, _quantised, _randn, _reference

pytestmark = pytest.mark.gpu

TYPES16 = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
# query heads of one kv head: key tiles that share an accumulator, one column tile, two
HEADS = pytest.mark.parametrize("heads", [3, 8, 16])


def _filled(k, v):
    """A cache of k, v [B, Hkv, L, D]; the rows behind them hold NaN parameters."""
    from sva_b200 import kernels

    n, kv, rows, dim = k.shape
    cache = kernels.kv4_empty(n, kv, -(-rows // 64) * 64, dim)
    for t in cache:
        t.view(torch.uint8).fill_(0xFF)
    kernels.kv4_write(k, v, cache, torch.zeros(n, dtype=torch.int64, device=DEV))
    return cache


def _decode_and_check(q, k, v, check=_check_decode):
    """One sequence of all of k, v: output, log-sum-exp and weights; the output without weights is the same."""
    from sva_b200 import kernels

    cache, n = _filled(k, v), torch.tensor([k.shape[2]], device=DEV)
    weights = torch.zeros(1, k.shape[1], k.shape[2], device=DEV)
    out, lse = kernels.kv4_decode(q, cache, seq_lens=n, max_len=k.shape[2], want_lse=True, weights=weights)
    assert torch.equal(out, kernels.kv4_decode(q, cache, seq_lens=n, max_len=k.shape[2]))
    check(q, (k, v), n, out, lse, weights)
    return out


# ------------------------------------------------------------------------------------------
# groups whose channels are all one number have no scale
# ------------------------------------------------------------------------------------------
def _flat_values(kind, v):
    """v [1, 1, L, D] with rows of one number: everywhere, or in some 64-key tiles."""
    v, n = v.clone(), v.shape[2]
    if isinstance(kind, float):
        return torch.full_like(v, kind)
    tile = torch.arange(n, device=DEV) // 64
    flat = {"first": tile == 0, "last": tile == (n - 1) // 64, "second": tile % 4 == 1, "odd": tile % 2 == 1,
            "but the last key": torch.arange(n, device=DEV) < n - 1}[kind]
    v[:, :, flat] = 0.0
    if kind == "odd":
        v[:, :, flat & (tile % 4 == 1)] = 3.0
    return v


@TYPES16
@HEADS
@pytest.mark.parametrize("n", [1, 65, 300, 5000])
def test_kv4_decode_groups_without_a_scale(n, heads, dtype):
    g = _gen(n + heads)
    q = _randn(g, 1, heads, 1, 64, dtype=dtype)
    k, v = (_randn(g, 1, 1, n, 64, dtype=torch.bfloat16) for _ in range(2))
    for kind in (0.0, 1.0, 1.5, 3.0, -8.0, 1e4, "first", "last", "second", "odd", "but the last key"):
        _decode_and_check(q, k, _flat_values(kind, v))


def test_kv4_decode_of_a_zeroed_cache():
    """Rows that were never written read as zeros, and attending to them alone gives zeros and equal weights."""
    from sva_b200 import kernels

    cache = kernels.kv4_empty(1, 2, 256, 128)
    for t in cache:
        t.view(torch.uint8).zero_()
    q, n = _randn(_gen(3), 1, 8, 1, 128, dtype=torch.bfloat16), torch.tensor([200], device=DEV)
    weights = torch.zeros(1, 2, 256, device=DEV)
    out, lse = kernels.kv4_decode(q, cache, seq_lens=n, weights=weights, want_lse=True)
    assert bool((out == 0).all())
    assert bool(((lse - math.log(200)).abs() <= 2.0 ** -20).all())
    # four heads a kv head; an exponential, a sum and a quotient
    assert bool(((weights[..., :200] - 4 / 200).abs() <= 4 / 200 * 2.0 ** -20).all()) and bool((weights[..., 200:] == 0).all())
