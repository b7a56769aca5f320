"""Attention over every key: packed prompts, the 4-bit cache and its attention, and eviction, against
plain implementations in 64 bits.

Tolerances count roundings (half a step of a type relative to the value: HALF).  An output sum_j p_j v_j is off
by its own rounding, by the rounding of every p_j to the kernel's operand type (at most HALF of sum_j p_j |v_j|,
times the scale's share for 4-bit rows), and by fp32 arithmetic: a logit of D products is off by at most
(D + 2) 2^-24 sum |q k| scale, which moves a weight by twice that, and a sum of n terms by n 2^-24 of its
absolute sum.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _reference(q, k, v, limit, scale, spread=None):
    """q [H, T, D], k / v [Hkv, L, D] in 64 bits; row t sees limit[t] keys.  Output, log-sum-exp, weights
    [H, T, L], sum p spread (spread: |v| unless given) and the largest sum |q k| scale of a row's keys."""
    h, t, _ = q.shape
    rep = h // k.shape[0]
    kk, vv = k.repeat_interleave(rep, 0), v.repeat_interleave(rep, 0)
    sp = (vv.abs() if spread is None else spread.repeat_interleave(rep, 0))
    x = q @ kk.transpose(1, 2) * scale
    seen = torch.arange(k.shape[1], device=q.device)[None, None, :] < limit[None, :, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True) if k.shape[1] else x.new_full((h, t, 1), -math.inf)
    top = top.masked_fill(top == -math.inf, 0.0)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    lse = (total.log() + top).squeeze(-1)
    zero = torch.zeros((), dtype=q.dtype, device=q.device)
    fine = torch.where(seen.any(1)[..., None], vv, zero)  # a value that no row sees may be anything
    size = ((q.abs() @ torch.nan_to_num(kk.abs()).transpose(1, 2)) * scale).masked_fill(~seen, 0.0)
    size = size.amax(-1, keepdim=True) if k.shape[1] else torch.zeros_like(top)
    return p @ fine, lse, p, p @ torch.where(seen.any(1)[..., None], sp, zero), size


def _fp32_share(n, d, size):
    """What fp32 arithmetic may add, relative to the absolute sum, for n keys of d channels."""
    return (n + 8) * 2.0 ** -24 + 2 * (d + 8) * 2.0 ** -24 * (size + 1)


def _check(got, ref, dtype, operand, spread, share, whole=None):
    """``share`` counts against the absolute sum of all terms that fp32 sums hold (``whole``; the spread unless
    given): a 4-bit row's term is z + s (c - 8), and with c = 8 its rounded part is 0 while z p is still summed."""
    off = (got.double() - ref).abs()
    terms = operand * spread + share * (spread if whole is None else whole)
    bound = HALF[dtype] * ref.abs() + (1 + HALF[dtype]) * terms + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of the smallest fp16 numbers
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} bounds"


# ------------------------------------------------------------------------------------------
# packed prompts
# ------------------------------------------------------------------------------------------
def _prompt_case(lens, lens_k, heads, kv, dim, dtype, seed=0, gap=0):
    g = _gen(seed)
    # `gap` unused rows stand before the first sequence and behind the last
    cu = torch.tensor([0, *lens]).cumsum(0) + gap
    cu_k = torch.tensor([0, *lens_k]).cumsum(0) + gap
    n, nk = int(cu[-1]) + gap, int(cu_k[-1]) + gap
    return (_randn(g, n, heads, dim, dtype=dtype), _randn(g, nk, kv, dim, dtype=dtype), _randn(g, nk, kv, dim, dtype=dtype),
            cu.to(DEV), cu_k.to(DEV))


def _check_prompt(q, k, v, cu, cu_k, out, lse=None, causal=True, scale=None):
    dtype, d = q.dtype, q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    # 16-bit prompts multiply weights rounded to their type; fp32 ones keep them
    operand = HALF[dtype] + 2.0 ** -20
    c, ck = cu.tolist(), cu_k.tolist()
    for b in range(len(c) - 1):
        lq, lk = c[b + 1] - c[b], ck[b + 1] - ck[b]
        limit = (torch.arange(lq, device=DEV) + lk - lq + 1).clamp(0, lk) if causal else torch.full((lq,), lk, device=DEV)
        qs, ks, vs = (x.double().transpose(0, 1) for x in (q[c[b]:c[b + 1]], k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]))
        ref, ref_lse, _, spread, size = _reference(qs, ks, vs, limit, scale)
        share = _fp32_share(lk, d, size)
        _check(out[c[b]:c[b + 1]].transpose(0, 1), ref, dtype, operand, spread, share)
        if lse is not None:
            got = lse[:, c[b]:c[b + 1]].double()
            empty = (limit == 0).expand_as(got)
            assert bool((got[empty] == -math.inf).all())
            bound = share.squeeze(-1) + 2.0 ** -20 + 2.0 ** -23 * torch.nan_to_num(ref_lse.abs(), posinf=0)
            assert bool(((got - ref_lse).abs()[~empty] <= bound[~empty]).all())


PROMPTS = [
    # lens, lens_k, heads, kv heads
    ([1], [1], 1, 1),
    ([2], [2], 3, 1),
    ([19], [19], 9, 3),
    ([127, 128, 129], [127, 128, 129], 9, 3),
    ([1, 0, 300, 5], [1, 0, 300, 5], 4, 4),
    ([42, 43, 84, 85, 86], [42, 43, 84, 85, 86], 3, 1),
    ([1, 7, 64], [513, 300, 1000], 8, 1),     # new tokens behind cached ones
    ([100, 3], [37, 3], 6, 2),                # the first queries see nothing
    ([5, 9], [0, 0], 2, 1),                   # no keys at all
    ([700], [700], 14, 2),
    ([3, 250], [256, 255], 40, 2),
    ([130], [130], 160, 1),                   # more heads a group than rows of a tile
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128, 80, 20, 200])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompt_matches_the_formula(case, dim, dtype):
    from sva_b200 import kernels

    lens, lens_k, heads, kv = PROMPTS[case]
    q, k, v, cu, cu_k = _prompt_case(lens, lens_k, heads, kv, dim, dtype, seed=case)
    out, lse = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, want_lse=True)
    _check_prompt(q, k, v, cu, cu_k, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_prompt_without_causal_mask_and_with_a_scale(dtype):
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case([200, 1, 33], [77, 300, 1], 6, 3, 64, dtype, seed=5)
    for scale in (0.37, 2.0, -0.2):
        out, lse = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, causal=False, softmax_scale=scale,
                                            want_lse=True)
        if scale > 0:
            _check_prompt(q, k, v, cu, cu_k, out, lse, causal=False, scale=scale)
        else:
            _check_prompt(-q, k, v, cu, cu_k, out, lse, causal=False, scale=-scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_prompt_leaves_other_rows_and_ignores_what_no_row_sees(dtype):
    from sva_b200 import kernels

    gap = 70
    q, k, v, cu, cu_k = _prompt_case([100, 31], [100, 31], 3, 1, 64, dtype, seed=2, gap=gap)
    want = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k)
    _check_prompt(q, k, v, cu, cu_k, want)
    # rows of no sequence hold NaN and infinities; so do the last key and value, seen by the last query alone
    for x in (q, k, v):
        x[:gap], x[-gap:] = float("nan"), float("inf")
    k[gap + 99], v[gap + 99, :, 3] = float("nan"), float("inf")
    v[gap + 99, :, 5] = float("nan")
    out = torch.full_like(q, 7.0)
    got = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, out=out)
    assert got is out
    assert bool((out[:gap] == 7).all()) and bool((out[-gap:] == 7).all())
    assert bool(out[gap + 99].isnan().all())
    rest = [i for i in range(gap, gap + 131) if i != gap + 99]
    assert torch.equal(out[rest], want[rest])


def test_prompt_non_finite_values_reach_the_rows_that_see_them():
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case([300], [300], 3, 1, 64, torch.bfloat16, seed=3)
    want = kernels.prompt_attention(q, k, v, cu)
    v[150, 0, 7], v[260, 0, 9] = float("inf"), float("nan")
    got = kernels.prompt_attention(q, k, v, cu)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[150:, :, 7] = True
    bad[260:, :, 9] = True
    assert torch.equal(got.isfinite(), ~bad)
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dim", [64, 72, 128])
def test_prompt_strides(dim):
    """Views into a fused projection, head-major tensors, odd offsets and a strided output."""
    from sva_b200 import kernels

    g = _gen(9)
    n, heads, kv = 150, 6, 2
    cu = torch.tensor([0, 60, 150], device=DEV)
    for pad, off in ((0, 0), (1, 0), (3, 1), (8, 8)):
        fused = _randn(g, n, (heads + 2 * kv) * dim + pad, dtype=torch.bfloat16)[:, off if off <= pad else 0:]
        q = fused[:, :heads * dim].unflatten(1, (heads, dim))
        k = fused[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        v = fused[:, (heads + kv) * dim:(heads + 2 * kv) * dim].unflatten(1, (kv, dim))
        out = torch.zeros(heads, n, dim + pad, dtype=torch.bfloat16, device=DEV).transpose(0, 1)[..., :dim]
        kernels.prompt_attention(q, k, v, cu, out=out)
        _check_prompt(q, k, v, cu, cu, out)
    hm = [_randn(g, h, n, dim, dtype=torch.float16).transpose(0, 1) for h in (heads, kv, kv)]
    _check_prompt(*hm, cu, cu, kernels.prompt_attention(*hm, cu))
    shared = _randn(g, n, 1, dim, dtype=torch.bfloat16).expand(n, kv, dim)  # one kv head for all, stride 0
    _check_prompt(q, shared, shared, cu, cu, kernels.prompt_attention(q, shared, shared, cu))


def test_prompt_large_logits_and_equal_logits():
    """Rows whose maximum jumps late, and rows of equal logits."""
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case([600], [600], 3, 1, 64, torch.bfloat16, seed=4)
    k[::97] *= 16
    q *= 4
    out = kernels.prompt_attention(q, k, v, cu)
    _check_prompt(q, k, v, cu, cu_k, out)
    k.zero_()
    out = kernels.prompt_attention(q, k, v, cu)
    _check_prompt(q, k, v, cu, cu_k, out)


def test_prompt_boundaries_are_clamped():
    from sva_b200 import kernels

    q, k, v, _, _ = _prompt_case([50], [50], 2, 1, 64, torch.bfloat16, seed=6)
    wild = torch.tensor([-5, 20, 10, 999], device=DEV)  # reads as sequences [0, 20), [], [10, 50)
    out = torch.zeros_like(q)
    kernels.prompt_attention(q, k, v, wild, out=out)
    # rows 10 .. 19 belong to two sequences and hold either one's output
    want = kernels.prompt_attention(q[10:], k[10:], v[10:], torch.tensor([0, 40], device=DEV))
    _check_prompt(q[10:], k[10:], v[10:], torch.tensor([0, 40]), torch.tensor([0, 40]), want)
    assert torch.equal(out[20:], want[10:])
    assert bool(out.isfinite().all())


# ------------------------------------------------------------------------------------------
# the 4-bit cache
# ------------------------------------------------------------------------------------------
def _down(x, up=False):
    """bf16 at or below (above) x, in 64 bits."""
    f, e = torch.frexp(x)
    return torch.ldexp((torch.ceil if up else torch.floor)(f * 256), e - 8)


def _quantised(x):
    """Values, scales and centres (m + 8 s) of rows in the 4-bit format, in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    m = _down(g.amin(-1))
    s = _down((g.amax(-1) - m) / 15, up=True)
    c = ((g - m[..., None]) / s.masked_fill(s == 0, 1)[..., None]).round()
    return (c * s[..., None] + m[..., None]).flatten(-2), s, m


def _paged(gen, lens, page, spare=1):
    need = [-(-int(n) // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return sum(need) + spare, table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [0, 64, 256])
@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_kv4_write_and_read(tokens, page, dim, dtype):
    from sva_b200 import kernels

    g = _gen(tokens + page + dim)
    n, kv = 3, 2
    start = torch.tensor([0, 63, 130], device=DEV)
    pages, table = (n, None) if not page else _paged(g, (start + tokens).tolist(), page)
    cache = kernels.kv4_empty(pages, kv, page or 384, dim)
    for t in cache:
        t.view(torch.uint8).fill_(0x5A)
    k = (_randn(g, n, kv, tokens, dim) * 3 + 2).to(dtype)
    v = _randn(g, n, tokens, kv, dim, dtype=dtype).transpose(1, 2)
    kernels.kv4_write(k, v, cache, start, page_table=table)
    got = kernels.kv4_read(cache, start, tokens, dtype=torch.float32, page_table=table)
    for x, y in zip((k, v), got):
        want, s, m = _quantised(x)
        # one rounding of m + s c to fp32
        assert torch.equal(y, want.float())
        assert bool(((y.double() - x.double()).unflatten(-1, (-1, 32)).abs() <= s[..., None] / 2 * (1 + 2.0 ** -20)
                     + y.double().abs().unflatten(-1, (-1, 32)) * 2.0 ** -23).all())
    low = kernels.kv4_read(cache, start, tokens, dtype=dtype, page_table=table)
    assert all(torch.equal(a, b.to(dtype)) for a, b in zip(low, got))
    # other rows are as they were
    before = kernels.kv4_read(cache, start - 1, 1, dtype=torch.float32, page_table=table)[0]
    assert bool((before[0] == 0).all())  # position -1
    untouched = kernels.kv4_empty(1, kv, 64, dim)
    for t in untouched:
        t.view(torch.uint8).fill_(0x5A)
    fill = kernels.kv4_read(untouched, torch.zeros(1, dtype=torch.int64, device=DEV), 1, dtype=torch.float32)[0]
    assert torch.equal(before[1:].nan_to_num(), fill.expand_as(before[1:]).nan_to_num())


def test_kv4_write_packed_equals_padded_and_skips_rows_of_no_sequence():
    from sva_b200 import kernels

    g = _gen(1)
    lens, kv, dim = [5, 0, 130, 1], 3, 64
    cu = torch.tensor([2, 7, 7, 137, 138], device=DEV)
    k, v = (_randn(g, 150, kv, dim, dtype=torch.bfloat16) for _ in range(2))
    start = torch.tensor([10, 0, 3, 200], device=DEV)
    a, b = kernels.kv4_empty(4, kv, 256, dim), kernels.kv4_empty(4, kv, 256, dim)
    for t in (*a, *b):
        t.view(torch.uint8).zero_()
    kernels.kv4_write(k, v, a, start, cu_seqlens=cu)
    for i, n in enumerate(lens):
        if n:
            c = kernels.Kv4Cache(*(t[i:i + 1] for t in b))
            rows = slice(int(cu[i]), int(cu[i]) + n)
            kernels.kv4_write(k[rows].transpose(0, 1)[None], v[rows].transpose(0, 1)[None], c, start[i:i + 1])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_kv4_write_awkward_values():
    """Constant groups, zeros, tiny and huge numbers, non-finite groups, exact halves."""
    from sva_b200 import kernels

    x = torch.zeros(1, 1, 12, 64, device=DEV)
    x[0, 0, 0] = 3.3
    x[0, 0, 1] = -3.3
    x[0, 0, 3] = torch.arange(64, device=DEV) * 1e-44
    x[0, 0, 4] = torch.linspace(-1e37, 1e37, 64, device=DEV)
    x[0, 0, 5] = torch.arange(64, device=DEV) / 4.0          # halves of a step
    x[0, 0, 6] = 1e4 + torch.arange(64, device=DEV) / 64.0   # far from zero
    x[0, 0, 7, 5] = float("nan")
    x[0, 0, 8, 40] = float("inf")
    x[0, 0, 9, 0], x[0, 0, 9, 1] = 3e38, -3e38
    x[0, 0, 10] = -torch.arange(64, device=DEV) * 2.0 ** -120
    x[0, 0, 11, 13] = -1e-30
    cache = kernels.kv4_empty(1, 1, 64, 64)
    start = torch.zeros(1, dtype=torch.int64, device=DEV)
    kernels.kv4_write(x, x, cache, start)
    y = kernels.kv4_read(cache, start, 12, dtype=torch.float32)[0]
    fine = [i for i in range(12) if i not in (3, 7, 8, 9)]
    want, s, _ = _quantised(x[:, :, fine])
    assert torch.equal(y[:, :, fine], want.float())
    # row 3 lies among the smallest numbers of bf16
    assert bool(((y[0, 0, 3].double() - x[0, 0, 3].double()).abs() <= 2.0 ** -133).all())
    assert torch.equal(y[0, 0, 7].isnan(), torch.arange(64, device=DEV) < 32)
    assert torch.equal(y[0, 0, 8].isnan(), torch.arange(64, device=DEV) >= 32)
    assert torch.equal(y[0, 0, 9].isnan(), torch.arange(64, device=DEV) < 32)


def test_kv4_positions_outside_the_cache():
    """Rows beyond the table, pages outside the pool: skipped by writes, zeros to reads, unseen by queries."""
    from sva_b200 import kernels

    g = _gen(12)
    table = torch.tensor([[1, -1, 7], [0, 2, 99]], dtype=torch.int32, device=DEV)
    cache = kernels.kv4_empty(3, 1, 64, 64)
    for t in cache:
        t.view(torch.uint8).zero_()
    k, v = (_randn(g, 2, 1, 250, 64, dtype=torch.bfloat16) for _ in range(2))
    start = torch.zeros(2, dtype=torch.int64, device=DEV)
    kernels.kv4_write(k, v, cache, start, page_table=table)
    rk, rv = kernels.kv4_read(cache, start, 250, dtype=torch.float32, page_table=table)
    assert bool((rk[0, :, 64:] == 0).all()) and bool((rk[1, :, 128:] == 0).all())
    assert bool((rk[1, :, :128] != 0).any(-1).all())
    q = _randn(g, 2, 3, 1, 64, dtype=torch.float32)
    weights = torch.zeros(2, 1, 192, device=DEV)
    out = kernels.kv4_decode(q, cache, page_table=table, weights=weights)
    for b, n in ((0, 64), (1, 128)):
        ref, _, p, spread, size = _reference(q[b].double(), rk[b, :, :n].double(), rv[b, :, :n].double(),
                                             torch.tensor([n], device=DEV), 64 ** -0.5)
        _check(out[b], ref, torch.float32, 2.0 ** -23, 4 * spread + 1e-3, _fp32_share(n, 64, size))
        assert bool((weights[b, 0, n:] == 0).all())
        assert torch.allclose(weights[b, 0, :n].double(), p.sum((0, 1)), rtol=1e-4, atol=0)


def _decode_case(lens, heads, kv, dim, tokens, dtype, page, seed):
    from sva_b200 import kernels

    g = _gen(seed)
    n, longest = len(lens), max(max(lens), 1)
    pages, table = (n, None) if not page else _paged(g, lens, page)
    rows = page or -(-longest // 64) * 64
    cache = kernels.kv4_empty(pages, kv, rows, dim)
    for t in cache:
        t.view(torch.uint8).fill_(0xFF)  # rows that no sequence holds: NaN parameters
    k = (_randn(g, n, kv, longest, dim) + _randn(g, dim) * 1.5).to(torch.bfloat16)
    v = _randn(g, n, kv, longest, dim, dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    for b, m in enumerate(lens):
        if m and page:
            kernels.kv4_write(k[b:b + 1, :, :m], v[b:b + 1, :, :m], cache, zero, page_table=table[b:b + 1])
        elif m:
            kernels.kv4_write(k[b:b + 1, :, :m], v[b:b + 1, :, :m], kernels.Kv4Cache(*(t[b:b + 1] for t in cache)), zero)
    q = _randn(g, n, heads, tokens, dim, dtype=dtype)
    return q, cache, table, torch.tensor(lens, device=DEV), (k, v), longest


def _check_decode(q, kv_rows, lens, out, lse=None, weights=None, scale=None):
    dtype, d, t = q.dtype, q.shape[-1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    operand = 2.0 ** -8 if dtype != torch.float32 else 2.0 ** -23
    for b, n in enumerate(lens.tolist()):
        (k, _, _), (v, s, m) = (_quantised(x[b, :, :n]) for x in kv_rows)
        limit = (torch.arange(t, device=DEV) + n - t + 1).clamp(min=0)
        centre = (m + 8 * s).repeat_interleave(32, -1)
        # weights times scales are rounded, the codes around 8 they multiply are exact; fp32 sums hold both terms
        spread = (v - centre).abs()
        ref, ref_lse, p, wide, size = _reference(q[b].double(), k, v, limit, scale, spread)
        _, _, _, whole, _ = _reference(q[b].double(), k, v, limit, scale, spread + centre.abs())
        # the logits' terms are s (q . (c - 8)) and z sum(q): their absolute sizes, not their sum's
        size = 4 * size + 8
        share = _fp32_share(n, d, size)
        _check(out[b], ref, dtype, operand, wide, share, whole)
        if lse is not None:
            empty = (limit == 0).expand_as(lse[b])
            assert bool((lse[b][empty] == -math.inf).all())
            bound = share.squeeze(-1) + 2.0 ** -20 + 2.0 ** -23 * torch.nan_to_num(ref_lse.abs(), posinf=0)
            assert bool(((lse[b].double() - ref_lse).abs()[~empty] <= bound[~empty]).all())
        if weights is not None:
            mass = p.unflatten(0, (k.shape[0], -1)).sum((1, 2))
            bound = (p * share).unflatten(0, (k.shape[0], -1)).sum((1, 2)) + 2.0 ** -22 * mass + 1e-37
            assert bool(((weights[b, :, :n].double() - mass).abs() <= bound).all())


DECODES = [
    # lens, heads, kv heads, tokens, page
    ([1], 1, 1, 1, 0),
    ([2, 1], 9, 3, 1, 0),
    ([63, 64, 65], 9, 3, 1, 64),
    ([301], 9, 3, 1, 0),
    ([0, 5, 700], 3, 1, 1, 256),              # an empty sequence
    ([3, 1, 260], 8, 1, 4, 64),               # the first token of the second sequence sees nothing
    ([5000], 16, 2, 1, 0),
    ([4097, 33, 1024], 14, 2, 1, 256),
    ([300], 7, 7, 5, 0),
    ([20000], 3, 1, 2, 64),
    ([257], 40, 2, 1, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_kv4_decode_matches_the_formula(case, dim, dtype):
    from sva_b200 import kernels

    lens, heads, kv, tokens, page = DECODES[case]
    q, cache, table, n, rows, longest = _decode_case(lens, heads, kv, dim, tokens, dtype, page, seed=case)
    out, lse = kernels.kv4_decode(q, cache, seq_lens=n, page_table=table, max_len=longest, want_lse=True)
    _check_decode(q, rows, n, out, lse)
    # with the weights: the same output, and sums that add up over calls; entries behind a sequence stay
    weights = torch.full((len(lens), kv, longest + 3), 0.5, device=DEV)
    again = kernels.kv4_decode(q, cache, seq_lens=n, page_table=table, max_len=longest, weights=weights)
    assert torch.equal(again, out)
    for b, m in enumerate(lens):
        assert bool((weights[b, :, m:] == 0.5).all())
    weights.zero_()
    kernels.kv4_decode(q, cache, seq_lens=n, page_table=table, max_len=longest, weights=weights)
    _check_decode(q, rows, n, out, weights=weights)


def test_kv4_decode_strides_scale_and_default_length():
    from sva_b200 import kernels

    q, cache, _, n, rows, longest = _decode_case([192, 192], 6, 2, 64, 3, torch.bfloat16, 0, seed=3)
    base = torch.zeros(2, 3, 6, 66, dtype=torch.bfloat16, device=DEV)
    base[..., 1:65] = q.transpose(1, 2)
    view = base[..., 1:65].transpose(1, 2)
    out = torch.zeros(2, 3, 6, 64, dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    kernels.kv4_decode(view, cache, softmax_scale=0.3, out=out)
    _check_decode(q, rows, n, out, scale=0.3)


def test_kv4_decode_lengths_are_clamped_and_shared_pages_are_read():
    from sva_b200 import kernels

    q, cache, table, _, rows, _ = _decode_case([128], 3, 1, 64, 1, torch.float32, 64, seed=4)
    q = q.expand(3, -1, -1, -1).contiguous()
    both = table.expand(3, -1).contiguous()  # three sequences in the same pages
    lens = torch.tensor([10 ** 12, 128, -4], device=DEV)
    out = kernels.kv4_decode(q, cache, seq_lens=lens, page_table=both)
    assert torch.equal(out[0], out[1]) and bool((out[2] == 0).all())
    _check_decode(q[:1], rows, torch.tensor([128]), out[:1])


def test_kv4_decode_sharp_softmax():
    """One key far above the rest, seen early and late."""
    from sva_b200 import kernels

    q, cache, table, n, rows, longest = _decode_case([3000], 3, 1, 64, 1, torch.float32, 0, seed=8)
    for at in (0, 1500, 2999):
        rows[0][0, 0, at] = q[0, 0, 0].to(torch.bfloat16) * 4
        kernels.kv4_write(rows[0][:, :, at:at + 1], rows[1][:, :, at:at + 1], cache, torch.tensor([at], device=DEV))
        out = kernels.kv4_decode(q * 3, cache, seq_lens=n, max_len=longest)
        _check_decode(q * 3, rows, n, out)


# ------------------------------------------------------------------------------------------
# eviction
# ------------------------------------------------------------------------------------------
def _kept(w, n, keep, recent):
    if n <= keep:
        return list(range(n))
    recent = min(recent, keep)
    old = n - recent
    key = [math.inf if x != x else x for x in w[:old].tolist()]
    nan = [x != x for x in w[:old].tolist()]
    best = sorted(range(old), key=lambda i: (not nan[i], -key[i], i))[:keep - recent]
    return sorted(best) + list(range(old, n))


def _evict_case(lens, kv, page, seed, ties):
    g = _gen(seed)
    longest = max(max(lens), 1)
    pages, table = (len(lens), None) if not page else _paged(g, lens, page)
    rows = page or longest + 5
    arrays = [torch.randint(0, 256, (pages, kv, rows, 32), generator=g, device=DEV).to(torch.uint8),
              _randn(g, pages, kv, rows, 2, 2, dtype=torch.bfloat16), _randn(g, pages, kv, rows, 80, dtype=torch.float32),
              _randn(g, pages, kv, rows, 3, dtype=torch.float16)]
    w = torch.rand(len(lens), kv, longest + 7, generator=g, device=DEV)
    if ties:
        w = (w * 4).floor()
    return arrays, w, table


def _rows_of(t, table, b, n):
    if table is None:
        return t[b, :, :n]
    return t[table[b].clamp(min=0).long()].transpose(0, 1).flatten(1, 2)[:, :n]


EVICTS = [
    # lens, kv heads, keep, recent, page
    ([1], 1, 1, 0, 0),
    ([2, 1, 0], 3, 1, 1, 0),
    ([300, 64, 65], 2, 64, 16, 0),
    ([1000, 5, 700], 3, 333, 0, 64),
    ([2304], 3, 2048, 256, 256),
    ([500], 2, 100, 100, 0),                 # the recent rows alone
    ([5000, 4999], 1, 4097, 1000, 0),
    ([40], 1, 0, 0, 0),                      # nothing stays
    ([70000], 1, 30000, 17, 0),
]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_cache_evict(case, in_place, ties):
    from sva_b200 import kernels

    lens, kv, keep, recent, page = EVICTS[case]
    arrays, w, table = _evict_case(lens, kv, page, case, ties)
    before = [a.clone() for a in arrays]
    w_before = w.clone()
    n = torch.tensor(lens, device=DEV)
    if in_place:
        kept, new = kernels.cache_evict(arrays, w, n, keep, recent=recent, page_table=table)
        got, got_w, got_table = arrays, w, table
    else:
        got = [torch.zeros(len(lens), kv, keep + 3, *a.shape[3:], dtype=a.dtype, device=DEV) for a in arrays]
        got_w, got_table = torch.full((len(lens), kv, keep + 2), 9.0, device=DEV), None
        kept, new = kernels.cache_evict(arrays, w, n, keep, recent=recent, page_table=table, out=got, out_weights=got_w)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(arrays, before))
        assert torch.equal(w, w_before)
    assert new.tolist() == [min(m, keep) for m in lens]
    for b, m in enumerate(lens):
        for h in range(kv):
            rows = _kept(w_before[b, h], m, keep, recent)
            assert kept[b, h].tolist() == rows + [-1] * (keep - len(rows))
            at = torch.tensor(rows, dtype=torch.int64, device=DEV)
            assert torch.equal(got_w[b, h, :len(rows)], w_before[b, h, at])
            assert bool((got_w[b, h, len(rows):] == 0).all())
            for a, o in zip(before, got):
                x, y = _rows_of(a, table, b, m)[h, at], _rows_of(o, got_table, b, len(rows))[h]
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            if in_place:
                for a, o in zip(before, got):
                    x, y = _rows_of(a, table, b, m)[h, len(rows):], _rows_of(o, table, b, m)[h, len(rows):]
                    assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_cache_evict_order_of_awkward_weights():
    from sva_b200 import kernels

    w = torch.tensor([0.0, -0.0, float("nan"), float("inf"), -1.0, 1e-40, -float("inf"), -float("nan"), 0.0, 5.0], device=DEV)
    w = w.expand(1, 1, -1).contiguous()
    rows = torch.arange(10, device=DEV, dtype=torch.int32).view(1, 1, 10, 1)
    for keep, want in ((1, [2]), (2, [2, 7]), (3, [2, 3, 7]), (4, [2, 3, 7, 9]), (5, [2, 3, 5, 7, 9]), (6, [0, 2, 3, 5, 7, 9]),
                       (7, [0, 1, 2, 3, 5, 7, 9]), (8, [0, 1, 2, 3, 5, 7, 8, 9])):
        out, ow = torch.zeros(1, 1, keep, 1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, keep, device=DEV)
        kept, _ = kernels.cache_evict([rows], w, torch.tensor([10], device=DEV), keep, out=[out], out_weights=ow)
        assert kept.flatten().tolist() == want
        assert out.flatten().tolist() == want


def test_cache_evict_keys_and_values_side_by_side():
    """Keys and values as views of one pool [pages, 2, Hkv, rows, D], and the refusal of arrays that do overlap."""
    from sva_b200 import kernels

    g = _gen(5)
    pool = _randn(g, 2, 2, 3, 64, 32, dtype=torch.bfloat16)
    before, w = pool.clone(), torch.rand(2, 3, 64, generator=g, device=DEV)
    n = torch.tensor([64, 40], device=DEV)
    w0 = w.clone()
    kept, lens = kernels.cache_evict([pool[:, 0], pool[:, 1]], w, n, 16, recent=4)
    for b in range(2):
        for h in range(3):
            at = torch.tensor(_kept(w0[b, h], int(n[b]), 16, 4), device=DEV)
            assert torch.equal(kept[b, h].long(), at)
            assert torch.equal(pool[b, :, h, :16], before[b, :, h, at])
            assert torch.equal(pool[b, :, h, 16:], before[b, :, h, 16:])
    out, ow = torch.zeros(2, 2, 3, 16, 32, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 3, 16, device=DEV)
    kernels.cache_evict([pool[:, 0], pool[:, 1]], w, n, 16, out=[out[:, 0], out[:, 1]], out_weights=ow)
    keys = pool[:, 0]
    for bad in (lambda: kernels.cache_evict([keys, keys], w, n, 16),
                lambda: kernels.cache_evict([keys[:, :, :40], keys[:, :, 8:48]], w, n, 16),
                lambda: kernels.cache_evict([keys], w, n, 16, out=[keys], out_weights=ow),
                lambda: kernels.cache_evict([keys], w, n, 16, out=[out[:, 0]], out_weights=w),
                lambda: kernels.cache_evict([keys, keys], w, n, 16, out=[out[:, 0], out[:, 0]], out_weights=ow)):
        with pytest.raises(ValueError, match="overlap"):
            bad()


@pytest.mark.parametrize("dim", [8, 24, 40, 56, 72, 104, 120])
def test_prompt_head_dims_that_fill_part_of_a_tile(dim):
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case([150, 1, 20], [150, 1, 300], 6, 2, dim, torch.bfloat16, seed=dim)
    _check_prompt(q, k, v, cu, cu_k, *kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, want_lse=True))


def test_prompt_split_over_a_long_axis():
    """Few rows over many keys: the keys are shared out and joined; rows that see nothing, and NaN, come through."""
    from sva_b200 import kernels

    q, k, v, cu, cu_k = _prompt_case([5, 9], [5000, 3], 8, 2, 64, torch.bfloat16, seed=8)
    out, lse = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k, want_lse=True)
    _check_prompt(q, k, v, cu, cu_k, out, lse)
    k[4000, 0] = float("nan")
    v[4998, 1, 3] = float("nan")  # seen by the last two queries of the first sequence
    got = kernels.prompt_attention(q, k, v, cu, cu_seqlens_k=cu_k)
    assert bool(got[:5, :4].isnan().all())
    bad = torch.zeros_like(got[:, 4:], dtype=torch.bool)
    bad[3:5, :, 3] = True
    assert torch.equal(got[:, 4:].isfinite(), ~bad)
    assert torch.equal(got[:, 4:][~bad], out[:, 4:][~bad])


def test_kv4_decode_scales_of_very_different_size():
    """Values whose scales span 2^40, in an order that makes the running bound grow, and tiny and huge queries."""
    from sva_b200 import kernels

    q, cache, _, n, rows, longest = _decode_case([700], 3, 1, 64, 1, torch.bfloat16, 0, seed=11)
    size = torch.ones(700, device=DEV)
    size[:256], size[256:512], size[600:] = 2.0 ** -30, 2.0 ** -10, 2.0 ** 10
    v = (rows[1].float() * size[:, None]).to(torch.bfloat16)
    kernels.kv4_write(rows[0], v, cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    for factor in (1.0, 2.0 ** -40, 2.0 ** 30):
        out = kernels.kv4_decode(q * factor, cache, seq_lens=n, max_len=longest, softmax_scale=0.125 / factor)
        _check_decode(q, (rows[0], v), n, out, scale=0.125)
    # a scale of zero weighs every key alike; a negative one is the positive one of -q
    assert torch.equal(kernels.kv4_decode(q, cache, seq_lens=n, max_len=longest, softmax_scale=-0.125),
                       kernels.kv4_decode(-q, cache, seq_lens=n, max_len=longest, softmax_scale=0.125))
    _check_decode(q * 0, (rows[0], v), n, kernels.kv4_decode(q, cache, seq_lens=n, max_len=longest, softmax_scale=0.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_kv4_decode_zero_queries_and_vanishing_scales(dtype):
    """Every key weighs the same, in a tile that the sequence ends in too."""
    from sva_b200 import kernels

    q, cache, _, n, rows, longest = _decode_case([300], 3, 1, 64, 1, dtype, 0, seed=14)
    zero = torch.zeros_like(q)
    for query, scale in ((zero, 0.125), (zero, 0.0), (zero, 1e-30), (q, 0.0), (q, 1e-38), (zero, -1e-30)):
        out = kernels.kv4_decode(query, cache, seq_lens=n, max_len=longest, softmax_scale=scale)
        _check_decode(zero, rows, n, out)


def test_kv4_decode_non_finite_groups_stay_in_their_channels():
    from sva_b200 import kernels

    q, cache, _, n, rows, longest = _decode_case([300], 3, 1, 64, 1, torch.bfloat16, 0, seed=13)
    want = kernels.kv4_decode(q, cache, seq_lens=n, max_len=longest)
    rows[1][0, 0, 250, 40] = float("inf")
    kernels.kv4_write(rows[0][:, :, 250:251], rows[1][:, :, 250:251], cache, torch.tensor([250], device=DEV))
    got = kernels.kv4_decode(q, cache, seq_lens=n, max_len=longest)
    assert bool(got[..., 32:].isnan().all()) and torch.equal(got[..., :32], want[..., :32])
    assert torch.equal(kernels.kv4_decode(q, cache, seq_lens=n - 50, max_len=longest),
                       kernels.kv4_decode(q, cache, seq_lens=n - 50, max_len=longest).nan_to_num(7.0))


def test_wrapper_refusals():
    from sva_b200 import kernels

    q, k, v, cu, _ = _prompt_case([10], [10], 4, 2, 64, torch.bfloat16)
    for call, error in ((lambda: kernels.prompt_attention(q[0], k, v, cu), ValueError),
                        (lambda: kernels.prompt_attention(q, k.half(), v, cu), TypeError),
                        (lambda: kernels.prompt_attention(q, k[:5], v[:5], cu), ValueError),
                        (lambda: kernels.prompt_attention(q, k[..., :32], v[..., :32], cu), ValueError),
                        (lambda: kernels.prompt_attention(q, k, v, cu.int()), ValueError),
                        (lambda: kernels.prompt_attention(q, k, v, cu.cpu()), RuntimeError),
                        (lambda: kernels.prompt_attention(q[:, :3], k, v, cu), ValueError),
                        (lambda: kernels.prompt_attention(q.double(), k.double(), v.double(), cu), TypeError),
                        (lambda: kernels.prompt_attention(q, k, v, cu, out=q[:5]), ValueError)):
        with pytest.raises(error):
            call()
    dq, cache, table, n, rows, longest = _decode_case([70, 64], 4, 2, 64, 1, torch.bfloat16, 64, seed=1)
    for call, error in ((lambda: kernels.kv4_decode(dq[0], cache), ValueError),
                        (lambda: kernels.kv4_decode(dq[..., :32], cache), ValueError),
                        (lambda: kernels.kv4_decode(dq[:, :3], cache, page_table=table), ValueError),
                        (lambda: kernels.kv4_decode(dq, cache, page_table=table[:1]), ValueError),
                        (lambda: kernels.kv4_decode(dq, cache, page_table=table.long()), ValueError),
                        (lambda: kernels.kv4_decode(dq, cache, page_table=table, max_len=129), ValueError),
                        (lambda: kernels.kv4_decode(dq, cache, page_table=table, seq_lens=n.int()), ValueError),
                        (lambda: kernels.kv4_decode(dq, cache, page_table=table, weights=torch.zeros(2, 2, 9, device=DEV)),
                         ValueError),
                        (lambda: kernels.kv4_write(rows[0], rows[1][:, :1], cache, n), ValueError),
                        (lambda: kernels.kv4_write(rows[0], rows[1].half(), cache, n), TypeError),
                        (lambda: kernels.kv4_write(rows[0], rows[1], cache, n[:1]), ValueError),
                        (lambda: kernels.kv4_read(cache, n, -1), ValueError),
                        (lambda: kernels.kv4_read(cache, n, 1, dtype=torch.int8), TypeError),
                        (lambda: kernels.cache_evict(cache, torch.zeros(2, 2, 128, device=DEV), n, -1, page_table=table),
                         ValueError),
                        (lambda: kernels.cache_evict(cache, torch.zeros(2, 2, 128, device=DEV), n, 9, recent=10,
                                                     page_table=table), ValueError),
                        (lambda: kernels.cache_evict([], torch.zeros(2, 2, 128, device=DEV), n, 9), ValueError)):
        with pytest.raises(error):
            call()


# ------------------------------------------------------------------------------------------
# all of them together, streams, graphs, large offsets
# ------------------------------------------------------------------------------------------
def test_prompt_then_cache_then_decode_then_evict():
    """A serving run: packed prompts, their rows into a paged 4-bit cache, decode steps that append and sum
    weights, an eviction, and more steps over what stayed."""
    from sva_b200 import kernels

    g = _gen(77)
    heads, kv, dim, page, dtype = 9, 3, 64, 64, torch.bfloat16
    lens = [150, 37, 201]
    cu = torch.tensor([0, *lens], device=DEV).cumsum(0)
    q, k, v = (_randn(g, sum(lens), h, dim, dtype=dtype) for h in (heads, kv, kv))
    _check_prompt(q, k, v, cu, cu, kernels.prompt_attention(q, k, v, cu))
    steps = 12
    pages, table = _paged(g, [n + steps for n in lens], page)
    cache = kernels.kv4_empty(pages, kv, page, dim)
    n = torch.zeros(3, dtype=torch.int64, device=DEV)
    kernels.kv4_write(k, v, cache, n, page_table=table, cu_seqlens=cu)
    n = torch.tensor(lens, device=DEV)
    rows = [[x[cu[b]:cu[b + 1]].transpose(0, 1) for b in range(3)] for x in (k, v)]
    most = max(lens) + steps
    weights, mass = torch.zeros(3, kv, most, device=DEV), torch.zeros(3, kv, most, dtype=torch.float64, device=DEV)
    for step in range(steps):
        qs, ks, vs = (_randn(g, 3, h, 1, dim, dtype=dtype) for h in (heads, kv, kv))
        kernels.kv4_write(ks, vs, cache, n, page_table=table)
        n = n + 1
        rows = [[torch.cat([r, x[b]], 1) for b, r in enumerate(y)] for x, y in zip((ks, vs), rows)]
        out = kernels.kv4_decode(qs, cache, seq_lens=n, page_table=table, max_len=most, weights=weights)
        for b in range(3):
            _check_decode(qs[b:b + 1], [r[b][None] for r in rows], n[b:b + 1], out[b:b + 1])
            kq = _quantised(rows[0][b])[0]
            p = (qs[b].double().unflatten(0, (kv, -1)) @ kq.transpose(1, 2).unsqueeze(1) / 8).softmax(-1)
            mass[b, :, :kq.shape[1]] += p.sum((1, 2))
        if step == 7:
            assert torch.allclose(weights.double(), mass, rtol=1e-3, atol=1e-7)
            kept, n = kernels.cache_evict(cache, weights, n, 100, recent=20, page_table=table)
            assert n.tolist() == [100, 45, 100]
            for b in range(3):
                at = kept[b, :, :int(n[b])].long()
                pick = at.unsqueeze(-1).expand(-1, -1, dim)
                for r in rows:
                    r[b] = torch.gather(r[b], 1, pick)
                m = torch.gather(mass[b], 1, at)
                mass[b].zero_()
                mass[b, :, :m.shape[1]] = m
    assert torch.allclose(weights.double(), mass, rtol=1e-3, atol=1e-7)


def test_streams_and_graphs():
    """Calls on a side stream, and two captured graphs that replay in turn, equal the eager calls."""
    from sva_b200 import kernels

    q, k, v, cu, _ = _prompt_case([200, 77], [200, 77], 9, 3, 64, torch.bfloat16, seed=21)
    dq, cache, table, n, _, longest = _decode_case([5000, 300], 9, 3, 64, 1, torch.bfloat16, 64, seed=22)
    dk, dv = (_randn(_gen(23), 2, 3, 1, 64, dtype=torch.bfloat16) for _ in range(2))
    weights = torch.zeros(2, 3, longest, device=DEV)
    out = [torch.zeros(2, 3, 128, *t.shape[3:], dtype=t.dtype, device=DEV) for t in cache]
    ow = torch.zeros(2, 3, 128, device=DEV)

    def work():
        kernels.kv4_write(dk, dv, cache, n - 1, page_table=table)
        weights.zero_()
        a = kernels.prompt_attention(q, k, v, cu)
        b = kernels.kv4_decode(dq, cache, seq_lens=n, page_table=table, max_len=longest, weights=weights)
        c = kernels.cache_evict(cache, weights, n, 128, recent=9, page_table=table, out=out, out_weights=ow)
        return (a, b, *c, weights, ow, *out)

    want = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in work()]
    side.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = work()
        graphs.append((graph, held))
    for graph, held in graphs + graphs:
        graph.replay()
        got = [t.clone() for t in held]
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # other inputs in the same places
    q.mul_(0.5)
    dq.mul_(0.5)
    want = [t.clone() for t in work()]
    for graph, held in graphs:
        graph.replay()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, want))


def test_offsets_beyond_32_bits():
    """A page pool of more than 2^32 code bytes: the last pages are written, read and attended to."""
    from sva_b200 import kernels

    rows, dim = 1 << 16, 128
    pages = (1 << 32) // (rows * dim // 2) + 2
    cache = kernels.kv4_empty(pages, 1, rows, dim)
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device=DEV)
    g = _gen(31)
    k, v = (_randn(g, 1, 1, 100, dim, dtype=torch.bfloat16) for _ in range(2))
    start = torch.tensor([rows - 50], device=DEV)
    for t in cache:
        t[pages - 1].view(torch.uint8).zero_()
        t[0].view(torch.uint8).zero_()
    kernels.kv4_write(k, v, cache, start, page_table=table)
    got = kernels.kv4_read(cache, start, 100, dtype=torch.float32, page_table=table)
    for x, y in zip((k, v), got):
        assert torch.equal(y, _quantised(x)[0].float())
    q = _randn(g, 1, 2, 1, dim, dtype=torch.float32)
    n = torch.tensor([rows + 50], device=DEV)
    whole = [torch.cat([torch.zeros(1, 1, rows - 50, dim, device=DEV, dtype=x.dtype), x], 2) for x in (k, v)]
    _check_decode(q, whole, n, kernels.kv4_decode(q, cache, seq_lens=n, page_table=table))
