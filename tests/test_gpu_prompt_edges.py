"""Values and weights of prompts at the ends of their ranges: infinities, and weights far below the largest."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_exact_attention import _check_prompt, _prompt_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens, lens_k, dim", [([300], [300], 64), ([300], [300], 128), ([300], [300], 40), ([5, 9], [5000, 9], 64),
                                               ([5, 9], [5000, 9], 128)])
def test_prompt_infinite_values(lens, lens_k, dim, dtype):
    """A row that sees +inf in a channel gets +inf there, -inf likewise, and NaN from both or from a NaN, whether all rows of its tile see
    the key or only some (every weight is far from 0 in the operand's type)."""
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case(lens, lens_k, 3, 1, dim, dtype, seed=3)
    want = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k)
    lq, lk = lens[0], lens_k[0]
    at = [lk - lq // 2 - 1, lk - 2, 1]  # seen by half of the first sequence's rows, by its last two (or one), by nearly all
    v[at[0], 0, 7], v[at[1], 0, 9], v[at[2], 0, 11] = math.inf, -math.inf, math.inf
    v[at[0], 0, 13], v[at[1], 0, 13] = math.inf, -math.inf
    v[at[1], 0, 15] = math.nan
    got = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k)
    expect = want.clone()
    last = torch.arange(lq, device=q.device) + lk - lq  # the last key of every row of the first sequence
    for channel, key, value in ((7, 0, math.inf), (9, 1, -math.inf), (11, 2, math.inf), (13, 0, math.inf), (13, 1, math.nan), (15, 1, math.nan)):
        expect[:lq][last >= at[key], :, channel] = value
    assert torch.equal(got.isnan(), expect.isnan())
    assert torch.equal(got.nan_to_num(0.0, math.inf, -math.inf), expect.nan_to_num(0.0, math.inf, -math.inf))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens, lens_k, dim", [([700], [700], 64), ([700], [700], 128), ([3, 2], [9000, 2], 64), ([3, 2], [9000, 2], 128)])
def test_prompt_small_weights_beside_a_large_one(lens, lens_k, dim, dtype):
    """The first key has values of zero and nearly all the weight; the others weigh 2^-20.5 of it each, and the output is theirs.
    The bounds are the general ones: half a step of the type for every weight, whatever its size."""
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case(lens, lens_k, 3, 1, dim, dtype, seed=6)
    q.fill_(1.0)
    k.zero_()
    v[1:] = v[1]
    for at in cu_k[:-1].tolist():
        k[at], v[at] = 20.5 * math.log(2) / math.sqrt(dim), 0.0
    out, lse = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, want_lse=True)
    _check_prompt(q, k, v, cu, cu_k, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens, lens_k", [([300, 1, 70], [300, 1, 70]), ([5, 9], [5000, 9])])
def test_prompt_output_in_the_place_of_the_queries(lens, lens_k, dtype):
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case(lens, lens_k, 6, 2, 64, dtype, seed=9)
    want = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k)
    assert kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, out=q) is q
    assert torch.equal(q, want)
