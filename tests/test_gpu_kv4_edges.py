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


# ------------------------------------------------------------------------------------------
# weights times scales in 16 bits
# ------------------------------------------------------------------------------------------
def _check_close(q, kv_rows, lens, out, lse=None, weights=None):
    """As _check_decode, with what 16-bit queries are held to: a weight times a scale is one fp16 number (half a step: 2^-11
    of it).  The largest of a group's products lies in [2^13, 2^15], so that the smallest fp16 numbers, half a step of which is 2^-25, add at
    most 2^-25 2^-13 8 = 2^-35 of the group's largest scale for each key (its code is within 8 of the centre)."""
    for b, n in enumerate(lens.tolist()):
        (k, _, _), (v, s, m) = (_quantised(x[b, :, :n]) for x in kv_rows)
        limit = (torch.arange(q.shape[2], device=DEV) + n - q.shape[2] + 1).clamp(min=0)
        centre, scale = (m + 8 * s).repeat_interleave(32, -1), q.shape[-1] ** -0.5
        spread = (v - centre).abs()
        ref, _, _, wide, size = _reference(q[b].double(), k, v, limit, scale, spread)
        _, _, _, whole, _ = _reference(q[b].double(), k, v, limit, scale, spread + centre.abs())
        floor = n * 2.0 ** -35 * s.amax(1, keepdim=True).repeat_interleave(32, -1).repeat_interleave(q.shape[1] // k.shape[0], 0)
        _check(out[b], ref, q.dtype, HALF[torch.float16], wide + floor / HALF[torch.float16],
               _fp32_share(n, q.shape[-1], 4 * size + 8), whole)
    _check_decode(q, kv_rows, lens, out, lse, weights)


@HEADS
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [65, 3000])
def test_kv4_decode_holds_fp16_outputs_to_their_type(n, dim, heads):
    g = _gen(n + dim + heads)
    k, v = (_randn(g, 1, 1, n, dim, dtype=torch.bfloat16) for _ in range(2))
    _decode_and_check(_randn(g, 1, heads, 1, dim, dtype=torch.float16), k, v, _check_close)


@TYPES16
@HEADS
@pytest.mark.parametrize("dim", [64, 128])
def test_kv4_decode_channel_groups_of_very_different_size(dim, heads, dtype):
    """A group of large channels takes nothing from the others."""
    g = _gen(dim + heads)
    n = 700
    k, v = (_randn(g, 1, 1, n, dim) for _ in range(2))
    for big, small in ((2.0 ** 10, 1.0), (8.0, 2.0 ** -10), (2.0 ** 60, 2.0 ** -60)):
        if dtype == torch.float16 and big > 2.0 ** 15:
            continue  # an output beyond the type
        size = torch.full((dim,), small, device=DEV)
        size[32:64] = big
        _decode_and_check(_randn(g, 1, heads, 1, dim, dtype=dtype), k.to(torch.bfloat16), (v * size).to(torch.bfloat16), _check_close)


@TYPES16
@pytest.mark.parametrize("heads", [1, 8, 16])
def test_kv4_decode_small_weights_beside_large_ones(heads, dtype):
    """Every 64th key has values of zero and nearly all the weight; the others weigh 2^-22 of it each, and the output is theirs."""
    n, dim = 4096, 64
    g = _gen(heads)
    q = torch.full((1, heads, 1, dim), 1.0, device=DEV).to(dtype)
    k = torch.zeros(1, 1, n, dim, dtype=torch.bfloat16, device=DEV)
    k[:, :, ::64] = 22 * math.log(2) / math.sqrt(dim)
    v = _randn(g, 1, 1, 1, dim, dtype=torch.bfloat16).repeat(1, 1, n, 1)
    v[:, :, ::64] = 0.0
    _decode_and_check(q, k, v, _check_close)


@TYPES16
def test_kv4_decode_scales_at_the_ends_of_the_range(dtype):
    """Values around 2^110 and 2^-110 (bf16 outputs hold them; fp16 ones overflow to infinity or vanish)."""
    from sva_b200 import kernels

    g = _gen(5)
    q = _randn(g, 1, 3, 1, 64, dtype=dtype)
    k, v = (_randn(g, 1, 1, 300, 64, dtype=torch.bfloat16) for _ in range(2))
    for factor in (2.0 ** 110, 2.0 ** -110):
        w = (v.float() * factor).to(torch.bfloat16)
        if dtype == torch.bfloat16:
            _decode_and_check(q, k, w)
        else:
            out = kernels.kv4_decode(q, _filled(k, w), max_len=300)
            assert not bool(out.isnan().any()) and (factor > 1 or bool((out == 0).all()))


# ------------------------------------------------------------------------------------------
# keys that only the later of the new tokens see
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n, tokens, heads, kv, dim", [(300, 3, 3, 3, 64), (65, 2, 2, 1, 128), (3, 3, 1, 1, 64), (5000, 4, 16, 2, 64),
                                                        (400, 150, 1, 1, 64), (256, 5, 8, 2, 128)])
def test_kv4_decode_non_finite_rows_reach_only_the_tokens_that_see_them(n, tokens, heads, kv, dim, dtype):
    from sva_b200 import kernels

    q, cache, _, lens, rows, longest = _decode_case([n], heads, kv, dim, tokens, dtype, 0, seed=n)
    want, want_lse = kernels.kv4_decode(q, cache, seq_lens=lens, max_len=longest, want_lse=True)
    k, v = (x.clone() for x in rows)
    first = n - tokens + max(1, tokens // 2)  # the first token that sees it, counted in keys
    v[0, kv - 1, first, 40], v[0, 0, n - 1, 3] = float("inf"), float("nan")
    start = torch.zeros(1, dtype=torch.int64, device=DEV)
    kernels.kv4_write(k, v, cache, start)
    got = kernels.kv4_decode(q, cache, seq_lens=lens, max_len=longest)
    position = n - tokens + torch.arange(tokens, device=DEV)  # of every token
    bad = torch.zeros_like(got, dtype=torch.bool)
    group = heads // kv
    bad[0, (kv - 1) * group:, :, 32:64] |= (position >= first)[:, None]
    bad[0, :group, :, :32] |= (position >= n - 1)[:, None]
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])
    # a key that is not a number: nothing is left of the rows that see it, the others are as they were
    k[0, 0, n - 1, 5] = float("nan")
    kernels.kv4_write(k, rows[1], cache, start)
    weights = torch.zeros(1, kv, n, device=DEV)
    got, lse = kernels.kv4_decode(q, cache, seq_lens=lens, max_len=longest, want_lse=True, weights=weights)
    assert bool(got[0, :group, -1].isnan().all()) and bool(lse[0, :group, -1].isnan().all())
    assert torch.equal(got[:, :, :-1], want[:, :, :-1]) and torch.equal(lse[:, :, :-1], want_lse[:, :, :-1])
    assert torch.equal(got[:, group:], want[:, group:]) and bool(weights[:, 1:].isfinite().all())


# ------------------------------------------------------------------------------------------
# codes next to half steps
# ------------------------------------------------------------------------------------------
def _codes(cache, rows):
    c = cache.k_codes[0, 0, :rows]
    return torch.stack([c & 15, c >> 4], -1).flatten(-2)


def _exact_codes(x):
    """Codes in 64 bits: every difference and product here has at most 53 bits, and a quotient that is no half step differs from
    one by more than 2^-50 of it."""
    g = x.double().unflatten(-1, (-1, 32))
    _, s, m = _quantised(x)
    return ((g - m[..., None]) / s[..., None]).round().flatten(-2).to(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_kv4_codes_are_the_exact_quotients_nearest(dtype):
    """Group minima from 1 down to 2^-24 of the step, of both signs; channels on half steps and one or two units beside them,
    and channels far below the minimum."""
    from sva_b200 import kernels

    r = torch.Generator().manual_seed(1)
    n = 4096
    e = torch.randint(0, 25 if dtype != torch.float16 else 12, (n,), generator=r)
    s = ((128 + torch.randint(0, 128, (n,), generator=r)) / 128.0).double()
    m = (128 + torch.randint(0, 128, (n,), generator=r)) / 128.0 * torch.ldexp(torch.ones(n), -e) * (1 - 2 * torch.randint(0, 2, (n,), generator=r))
    m = m.double()
    half = torch.randint(0, 15, (n, 32), generator=r) + 0.5
    x = (m[:, None] + half * s[:, None]).to(dtype)
    # a minimum below zero also has channels far below it, on either side of a half step's sum
    tiny = (128 + torch.randint(0, 128, (n, 32), generator=r)) / 128.0 * (1 - 2 * torch.randint(0, 2, (n, 32), generator=r))
    tiny = torch.ldexp(tiny.double(), -torch.randint(1, 31 if dtype != torch.float16 else 12, (n, 32), generator=r))
    pick = torch.randint(0, 7, (n, 32), generator=r)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    x = (x.view(bits) + (pick - 2).clamp(-2, 2).to(bits)).view(dtype)
    x = x.double().nan_to_num(0.0)  # the pattern below that of zero
    x = torch.where((pick == 6) & (m[:, None] < 0), tiny, x)
    x = torch.minimum(torch.maximum(x, m[:, None]), m[:, None] + 15 * s[:, None]).to(dtype)
    x = torch.where(x.double() < m[:, None], m[:, None].to(dtype), x)
    x[:, 0], x[:, 1] = m.to(dtype), (m + 14.97 * s).to(dtype)
    x = x.view(1, 1, n // 2, 64).to(DEV)
    cache = kernels.kv4_empty(1, 1, n // 2, 64)
    kernels.kv4_write(x, x, cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    got, want = _codes(cache, n // 2), _exact_codes(x)[0, 0]
    wrong = (got != want).nonzero()
    assert len(wrong) == 0, f"{len(wrong)} codes, first {wrong[0].tolist()}"


@pytest.mark.parametrize("dtype, minimum, scale, x, code", [
    (torch.float32, -2.0 ** -23, 1.0, 6.5, 7),
    (torch.float32, 2.0 ** -23, 1.0, 7.5, 7),
    (torch.float32, -2.0 ** -26, 1.0, 0.5, 1),
    (torch.float32, 2.0 ** -26, 1.0, 1.5, 1),
    (torch.float32, 0.0, 1.0, 6.5, 6),
    (torch.float32, 0.0, 1.0, 7.5, 8),
    (torch.float32, 5.5879354e-07, 0.35546875, 4.087891, 11),
    (torch.bfloat16, -1.0, 2.0, 2.0 ** -30, 1),
    (torch.bfloat16, -1.0, 2.0, -(2.0 ** -30), 0),
    (torch.bfloat16, -1.0, 2.0, 0.0, 0),
    (torch.bfloat16, -6.5, 1.0, 2.0 ** -30, 7),
    (torch.bfloat16, 2.0 ** -30, 1.0, 7.5, 7),
    (torch.float16, -6.5, 1.0, 2.0 ** -24, 7),
    (torch.float32, -0.5e31, 1e31, 1e-10, 1),
    (torch.float32, -0.5e31, 1e31, -1e-10, 0),
    (torch.float32, -2.0 ** -110, 2.0 ** -109, 2.0 ** -149, 1),
])
def test_kv4_codes_of_sums_that_fp32_rounds_to_half_steps(dtype, minimum, scale, x, code):
    from sva_b200 import kernels

    s = torch.tensor(scale).to(torch.bfloat16).float()
    m = torch.tensor(minimum).to(torch.bfloat16).float() if scale != 1e31 else -s / 2
    row = torch.full((64,), x, dtype=torch.float32)
    row[::32] = m
    row[1::32] = m + 14.97 * s
    row = row.to(dtype).to(DEV).expand(1, 1, 1, 64)
    cache = kernels.kv4_empty(1, 1, 64, 64)
    kernels.kv4_write(row, row, cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert cache.k_params[0, 0, 0, 0].tolist() == [float(s), float(m)]
    got = _codes(cache, 1)[0].tolist()
    assert got[2:32] == [code] * 30 and got[34:] == [code] * 30 and got[0] == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_kv4_decode_of_empty_sequences_with_weights(dtype):
    """Zeros, -inf, and weights as they were, complete when the next kernel of the stream reads them."""
    from sva_b200 import kernels

    q, cache, _, _, _, _ = _decode_case([300, 300], 4, 2, 64, 1, dtype, 0, seed=2)
    none = torch.zeros(2, dtype=torch.int64, device=DEV)
    for max_len in (0, 64, 300):
        for _ in range(20):
            weights, out = torch.full((2, 2, 300), 0.25, device=DEV), torch.full_like(q, 7.0)
            got, lse = kernels.kv4_decode(q, cache, seq_lens=none, max_len=max_len, weights=weights, want_lse=True, out=out)
            total = got.float().abs().sum() + (lse != -math.inf).sum() + (weights != 0.25).sum()
            assert float(total) == 0


def test_cache_evict_of_one_row_pages_moves_the_row_alone():
    from sva_b200 import kernels

    base = _randn(_gen(4), 1, 1, 640, 32, dtype=torch.bfloat16)
    before, w, n = base.clone(), torch.ones(1, 1, 1, device=DEV), torch.ones(1, dtype=torch.int64, device=DEV)
    room = torch.full((1, 1, 64, 32), 5.0, dtype=torch.bfloat16, device=DEV)
    for rows in (base[:, :, ::640], base.as_strided((1, 1, 1, 32), (7, 9, 11, 1))):
        kernels.cache_evict([rows], w, n, 1, out=[room[:, :, 3:4]], out_weights=torch.zeros(1, 1, 1, device=DEV))
        assert torch.equal(room[0, 0, 3], base[0, 0, 0]) and bool((room[0, 0, :3] == 5).all()) and bool((room[0, 0, 4:] == 5).all())
        room[0, 0, 3] = 5.0
        kernels.cache_evict([rows], w, n, 1)
        assert torch.equal(base, before)


# ------------------------------------------------------------------------------------------
# tensors that are written and overlap themselves; sequences without keys
# ------------------------------------------------------------------------------------------
def test_written_tensors_that_overlap_themselves_are_refused():
    from sva_b200 import kernels

    q, cache, _, n, rows, longest = _decode_case([70, 64], 4, 2, 64, 1, torch.bfloat16, 0, seed=1)
    sums = torch.zeros(2, 2, 200, device=DEV)
    kw = dict(seq_lens=n, max_len=longest)
    for weights in (sums[:1].expand(2, 2, 200), sums[:, :1].expand(2, 2, 200), sums.view(-1).as_strided((2, 2, 100), (150, 50, 1))):
        with pytest.raises(ValueError, match="overlap"):
            kernels.kv4_decode(q, cache, weights=weights, **kw)
    kernels.kv4_decode(q, cache, weights=sums.view(-1).as_strided((2, 2, 100), (100, 200, 1)), **kw)  # heads apart, sequences within
    for out in (q[:1].clone().expand(2, 4, 1, 64), q[:, :1].clone().expand(2, 4, 1, 64)):
        with pytest.raises(ValueError, match="overlap"):
            kernels.kv4_decode(q, cache, out=out, **kw)
    p, cu = _randn(_gen(1), 9, 4, 64, dtype=torch.bfloat16), torch.tensor([0, 9], device=DEV)
    for out in (p[:1].clone().expand(9, 4, 64), p[:, :1].clone().expand(9, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            kernels.prompt_attention(p, p, p, cu, out=out)
    for bad in (lambda: kernels.cache_evict([rows[0][:1].expand(2, 2, 70, 64)], sums, n, 16),
                lambda: kernels.cache_evict([rows[0][:, :1].expand(2, 2, 70, 64)], sums, n, 16),
                lambda: kernels.cache_evict([rows[0]], sums[:1].expand(2, 2, 200), n, 16),
                lambda: kernels.cache_evict([rows[0]], sums, n, 16, out=[rows[1]], out_weights=sums.clone()[:, :1].expand(2, 2, 200)),
                lambda: kernels.cache_evict([rows[0]], sums, n, 16, out=[rows[1][:1].expand(2, 2, 70, 64)], out_weights=sums.clone())):
        with pytest.raises(ValueError, match="overlap"):
            bad()
    # what is only read may
    kernels.cache_evict([rows[0][:1].expand(2, 2, 70, 64)], sums[:1].expand(2, 2, 200), n, 16, out=[rows[1]], out_weights=sums.clone())


@TYPES16
@HEADS
@pytest.mark.parametrize("dim", [64, 128])
def test_kv4_decode_query_channels_far_below_the_largest(dim, heads, dtype):
    """One query channel 2^20 times the others, on keys as much smaller there: the scores are the others'."""
    g = _gen(dim + heads)
    n = 500
    q = _randn(g, 1, heads, 1, dim) * 2.0 ** -6
    q[..., 0] = 2.0 ** 14
    k = _randn(g, 1, 1, n, dim) * 2.0 ** 7
    k[..., :32] *= 2.0 ** -23
    _decode_and_check(q.to(dtype), k.to(torch.bfloat16), _randn(g, 1, 1, n, dim, dtype=torch.bfloat16), _check_close)
