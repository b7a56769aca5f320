"""Cases, plain forms and work counts of the exact-attention operators.

Four operators serve the layers and steps that attend to every key, next to the summon path:

* ``prompt``: causal attention over whole prompts, packed without padding, grouped heads;
* ``write``:  keys and values into a 4-bit cache (groups of 32 channels, a bf16 scale and minimum each),
  and the same rows read back;
* ``decode``: attention of the newest tokens over the 4-bit cache, optionally adding every key's softmax
  weight to a running sum;
* ``evict``:  the cache cut down to the keys with the largest accumulated weight and the most recent ones.

``own`` False computes the plain forms (elementary torch operations in 32 bits, in 64 where a border
decides), ``own`` True calls sva_b200.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 32


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # a chat turn's few tokens: latency
        dict(name="prompt_19", op="prompt", seqs=1, longest=19, shortest=19, cached=0, heads=9, kv=3, dim=64, dtype="bf16"),
        # the 8192-token prompt of the 30-layer decode benchmark, one layer of it
        dict(name="prompt_8192", op="prompt", seqs=1, longest=8192, shortest=8192, cached=0, heads=9, kv=3, dim=64,
             dtype="bf16"),
        # a server's batch of prompts of very different lengths, packed
        dict(name="prompt_packed", op="prompt", seqs=12, longest=4095, shortest=1, cached=0, heads=9, kv=3, dim=64,
             dtype="fp16"),
        # a chunk of new tokens behind a long cached conversation, wide heads
        dict(name="prompt_chunk", op="prompt", seqs=2, longest=61, shortest=61, cached=30011, heads=16, kv=2, dim=128,
             dtype="bf16"),
        # every decode step appends one row per sequence: latency
        dict(name="write_step", op="write", seqs=8, tokens=1, at=1000, page=256, kv=3, dim=64, dtype="bf16"),
        # a batch of 32k prompts goes into the cache
        dict(name="write_prompt", op="write", seqs=8, tokens=32768, at=0, page=0, kv=3, dim=64, dtype="bf16"),
        # one token over a short cache in 32 bits: latency
        dict(name="decode_301", op="decode", seqs=1, tokens=1, longest=301, shortest=301, page=0, weights=False, heads=9,
             kv=3, dim=64, dtype="fp32"),
        # one layer of the 32k, batch 8 decode benchmark
        dict(name="decode_8x32768", op="decode", seqs=8, tokens=1, longest=32768, shortest=32768, page=0, weights=False,
             heads=9, kv=3, dim=64, dtype="bf16"),
        # the benchmark's ragged batch of 64 sequences in pages of 256 keys
        dict(name="decode_ragged", op="decode", seqs=64, tokens=1, longest=131072, shortest=4096, page=256,
             weights=False, heads=9, kv=3, dim=64, dtype="bf16"),
        # a million-key cache, with the weights that an eviction goes by
        dict(name="decode_million", op="decode", seqs=1, tokens=1, longest=1048576, shortest=1048576, page=0,
             weights=True, heads=9, kv=3, dim=64, dtype="fp16"),
        # a 4-bit cache trimmed during decoding, every 256 tokens
        dict(name="evict_2304", op="evict", seqs=8, longest=2304, shortest=2304, keep=2048, recent=256, bits=4, kv=3,
             dim=64),
        # long prompts cut to a quarter, 16-bit rows
        dict(name="evict_16385", op="evict", seqs=16, longest=16385, shortest=9001, keep=4096, recent=511, bits=16,
             kv=8, dim=128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "write", "decode", "decode", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv, groups = rng.choice([(3, 3), (1, 1), (2, 5), (4, 2), (2, 8), (1, 7)])
    dim = rng.choice([64, 64, 128])
    if op == "prompt":
        dim = rng.choice([64, 64, 128, 80])
        cached = rng.choice([0, 0, _log(rng, 1, 8000)])
        seqs = _log(rng, 1, 9)
        # the padded plain form holds seqs x queries x keys scores a head
        room = 3.2e8 / (kv * groups * seqs)
        longest = max(1, min(_log(rng, 1, 4096), int((math.sqrt(cached * cached + 4 * room) - cached) / 2)))
        return dict(op=op, seqs=seqs, longest=longest, shortest=rng.choice([longest, 1]), cached=cached, heads=kv * groups,
                    kv=kv, dim=dim, dtype=dtype)
    if op == "write":
        seqs = _log(rng, 1, 16)
        tokens = max(1, min(_log(rng, 1, 32768), 700000 * 64 // (seqs * kv * dim)))
        return dict(op=op, seqs=seqs, tokens=tokens, at=_log(rng, 1, 5000) - 1, page=rng.choice([0, 64, 256]), kv=kv, dim=dim,
                    dtype=dtype)
    if op == "decode":
        seqs = _log(rng, 1, 32)
        longest = max(1, min(_log(rng, 1, 300000), 4000000 * 64 // (seqs * kv * dim)))
        tokens = min(longest, rng.choice([1, 1, 1, 2, 4]))
        return dict(op=op, seqs=seqs, tokens=tokens, longest=longest, shortest=rng.choice([longest, tokens]),
                    page=rng.choice([0, 64, 256]), weights=rng.choice([True, False]), heads=kv * groups, kv=kv, dim=dim,
                    dtype=dtype)
    seqs = _log(rng, 1, 16)
    longest = _log(rng, 2, 16000)
    keep = max(1, min(_log(rng, 1, 8000), longest))
    return dict(op=op, seqs=seqs, longest=longest, shortest=rng.choice([longest, 1]), keep=keep,
                recent=rng.randint(0, keep), bits=rng.choice([4, 16]), kv=kv, dim=dim)


def _lengths(case):
    """The sequences' lengths: the same for every seed, logarithmically between shortest and longest."""
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    r = np.random.RandomState(n * 1000003 + low * 1009 + high)
    lens = np.exp(r.uniform(math.log(low), math.log(high), n)).round().astype(np.int64)
    lens[r.randint(n)] = high
    return lens.clip(low, high)


def _up(n, to):
    return (n + to - 1) // to * to


# ------------------------------------------------------------------------------------------
# the 4-bit format: (scale, minimum) in bf16 for 32 channels, both rounded outwards so that every value lies
# within the sixteen steps; the codes are the exact quotients' nearest whole numbers, halves to even
# ------------------------------------------------------------------------------------------
def _next16(b, up):
    """The bf16 value above (up) or below ``b``, by its bits."""
    i = b.view(torch.int16).to(torch.int32) & 0xFFFF
    away = (i + 1) & 0xFFFF
    near = torch.where((i & 0x7FFF) == 0, torch.full_like(i, 0x0001 if up else 0x8001), i - 1)
    grows = (i < 0x8000) if up else (i > 0x8000)
    grows = grows | ((i & 0x7FFF) == 0) & (i == (0 if up else 0x8000))
    i = torch.where(grows, away, near)
    return torch.where(i >= 0x8000, i - 0x10000, i).to(torch.int16).view(torch.bfloat16)


def _quantise(x):
    """Codes (uint8 [..., D / 2]) and parameters (bf16 [..., D / 32, 2]) of rows x [..., D]."""
    g = x.double().unflatten(-1, (x.shape[-1] // GROUP, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    m = low.to(torch.bfloat16)
    m = torch.where(m.double() > low, _next16(m, False), m)
    step = (high - m.double()) / 15
    s = step.to(torch.bfloat16)
    s = torch.where(s.double() < step, _next16(s, True), s)
    sd = s.double().unsqueeze(-1)
    c = torch.where(sd > 0, (g - m.double().unsqueeze(-1)) / sd, torch.zeros_like(g)).round().clamp(0, 15)
    c = c.to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([s, m], -1)


def _values(codes, params):
    """The values (32 bits) that codes and parameters stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    c = c.unflatten(-1, (c.shape[-1] // GROUP, GROUP))
    return (c * params[..., 0].float().unsqueeze(-1) + params[..., 1].float().unsqueeze(-1)).flatten(-2)


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _rand(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _kv_rows(gen, *shape):
    """Keys as layers have them: some channels far from zero; values around zero."""
    off = torch.randn(shape[-1], generator=gen, device=DEV) * 1.5
    return torch.randn(*shape, generator=gen, device=DEV) + off


def _pool(case, gen, lens):
    """(pages, rows a page, page table or None) of a cache for sequences of these lengths."""
    n, page = case["seqs"], case["page"]
    if not page:
        return n, _up(max(lens), 64), None
    need = [-(-int(v) // page) for v in lens]
    order = torch.randperm(sum(need), generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(n, max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return sum(need), page, table


def _cache(gen, pages, kv, rows, dim):
    """A filled 4-bit cache, page by page so that the wide rows never exist at once."""
    k = [torch.empty(pages, kv, rows, dim // 2, dtype=torch.uint8, device=DEV) for _ in range(2)]
    p = [torch.empty(pages, kv, rows, dim // GROUP, 2, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    some = max(1, (1 << 25) // (kv * rows * dim))
    for a in range(0, pages, some):
        n = min(some, pages - a)
        for w in range(2):
            for r in range(0, rows, 1 << 17):
                e = min(rows, r + (1 << 17))
                x = _kv_rows(gen, n, kv, e - r, dim) if w == 0 else _rand(gen, n, kv, e - r, dim)
                k[w][a:a + n, :, r:e], p[w][a:a + n, :, r:e] = _quantise(x)
    return k[0], p[0], k[1], p[1]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, dim, kv = case["op"], case["dim"], case["kv"]
    s = dict(case=case)
    if op == "prompt":
        lens = _lengths(case)
        lk = lens + case["cached"]
        dt = TYPES[case["dtype"]]
        n, nk = int(lens.sum()), int(lk.sum())
        s["q"] = _rand(gen, n, case["heads"], dim, dtype=dt)
        s["keys"] = _rand(gen, nk, kv, dim, dtype=dt)
        s["values"] = _rand(gen, nk, kv, dim, dtype=dt)
        s["cu"] = torch.tensor(np.concatenate([[0], lens.cumsum()]), device=DEV)
        s["cu_k"] = torch.tensor(np.concatenate([[0], lk.cumsum()]), device=DEV)
        s["pad"] = int(lens.max()), int(lk.max())
    elif op == "write":
        n, t, dt = case["seqs"], case["tokens"], TYPES[case["dtype"]]
        pages, rows, s["table"] = _pool(case, gen, [case["at"] + t] * n)
        s["keys"] = _kv_rows(gen, n, kv, t, dim).to(dt)
        s["values"] = _rand(gen, n, kv, t, dim, dtype=dt)
        s["start"] = torch.full((n,), case["at"], dtype=torch.int64, device=DEV)
        s["cache"] = tuple(torch.zeros(pages, kv, rows, *tail, dtype=d, device=DEV)
                           for tail, d in (((dim // 2,), torch.uint8), ((dim // GROUP, 2), torch.bfloat16)) * 2)
    elif op == "decode":
        lens = _lengths(case)
        pages, rows, s["table"] = _pool(case, gen, lens)
        s["cache"] = _cache(gen, pages, kv, rows, dim)
        s["q"] = _rand(gen, case["seqs"], case["heads"], case["tokens"], dim, dtype=TYPES[case["dtype"]])
        s["lens"] = torch.tensor(lens, device=DEV)
        s["longest"] = int(lens.max())
        s["weights"] = (torch.zeros(case["seqs"], kv, s["longest"], device=DEV) if case["weights"] else None)
    else:
        lens = _lengths(case)
        n, longest = case["seqs"], case["longest"]
        s["lens"] = torch.tensor(lens, device=DEV)
        # accumulated softmax weights: a few keys hold most of the mass
        s["weights"] = torch.rand(n, kv, longest, generator=gen, device=DEV).pow(8)
        rows, out_rows = _up(longest, 64), _up(case["keep"], 64)
        if case["bits"] == 4:
            s["rows"] = _cache(gen, n, kv, rows, dim)
        else:
            s["rows"] = tuple(_rand(gen, n, kv, rows, dim, dtype=torch.bfloat16) for _ in range(2))
        s["out"] = tuple(torch.zeros(n, kv, out_rows, *r.shape[3:], dtype=r.dtype, device=DEV) for r in s["rows"])
        s["out_weights"] = torch.zeros(n, kv, out_rows, device=DEV)
    return s


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _softmax_parts(logits, seen):
    """(weights, rows that see nothing) of masked logits."""
    logits = logits.masked_fill(~seen, float("-inf"))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0)


def _prompt_plain(s):
    case = s["case"]
    q, k, v = s["q"].float(), s["keys"].float(), s["values"].float()
    cu, cu_k = s["cu"], s["cu_k"]
    tq, tk = torch.arange(s["pad"][0], device=DEV), torch.arange(s["pad"][1], device=DEV)
    lq, lk = cu.diff(), cu_k.diff()
    iq = (cu[:-1, None] + tq).clamp(max=q.shape[0] - 1)
    ik = (cu_k[:-1, None] + tk).clamp(max=k.shape[0] - 1)
    n, g = case["seqs"], case["heads"] // case["kv"]
    qp = q[iq].view(n, len(tq), case["kv"], g, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, g * Tq, D]
    kp, vp = k[ik].transpose(1, 2), v[ik].transpose(1, 2)
    logits = (qp @ kp.transpose(2, 3)) * case["dim"] ** -0.5
    seen = (tk <= (tq[:, None] + (lk - lq)[:, None, None])) & (tk < lk[:, None, None])  # [B, Tq, Tk]
    p = _softmax_parts(logits.view(n, case["kv"], g, len(tq), len(tk)), seen[:, None, None])
    o = (p.flatten(2, 3) @ vp).view(n, case["kv"], g, len(tq), -1).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[tq < lq[:, None]].to(s["q"].dtype)


def _row_index(s, pos):
    """(page, row) of positions pos [B, T] of every sequence."""
    if s["table"] is None:
        return torch.arange(pos.shape[0], device=DEV)[:, None].expand_as(pos), pos
    page = s["case"]["page"]
    col = (pos // page).clamp(max=s["table"].shape[1] - 1)
    return torch.gather(s["table"].long(), 1, col), pos % page


def _write_plain(s):
    dt = s["keys"].dtype
    pos = s["start"][:, None] + torch.arange(s["case"]["tokens"], device=DEV)
    page, row = _row_index(s, pos)
    got = []
    for x, codes, params in ((s["keys"], *s["cache"][:2]), (s["values"], *s["cache"][2:])):
        c, p = _quantise(x)
        codes[page, :, row] = c.transpose(1, 2)
        params[page, :, row] = p.transpose(1, 2)
        got.append(_values(codes[page, :, row], params[page, :, row]).transpose(1, 2).to(dt))
    return tuple(got)


def _decode_plain(s):
    case = s["case"]
    kc, kp, vc, vp = s["cache"]
    n, t, g = case["seqs"], case["tokens"], case["heads"] // case["kv"]
    pos = torch.arange(s["longest"], device=DEV).expand(n, -1)
    page, row = _row_index(s, pos)
    if s["table"] is None:
        pick = lambda x: x[:, :, :s["longest"]]  # noqa: E731
    else:
        pick = lambda x: x[page, :, row].transpose(1, 2)  # noqa: E731
    k, v = _values(pick(kc), pick(kp)), _values(pick(vc), pick(vp))
    live = (pos < s["lens"][:, None])[:, None, :, None]
    v = v.masked_fill(~live, 0.0)
    q = s["q"].float().view(n, case["kv"], g * t, case["dim"])
    logits = (q @ k.transpose(2, 3)) * case["dim"] ** -0.5
    last = s["lens"][:, None] - t + 1 + torch.arange(t, device=DEV)  # [B, T] keys seen
    seen = pos[:, None] < last[:, :, None]
    p = _softmax_parts(logits.view(n, case["kv"], g, t, -1), seen[:, None, None])
    out = (p.flatten(2, 3) @ v).view(n, case["heads"], t, -1).to(s["q"].dtype)
    if s["weights"] is None:
        return out
    s["weights"] += p.sum((2, 3))
    return out, s["weights"]


def _evict_plain(s):
    case = s["case"]
    n, kv, longest = s["weights"].shape
    lens, keep, recent = s["lens"][:, None, None], case["keep"], case["recent"]
    pos = torch.arange(longest, device=DEV)
    w = s["weights"].masked_fill((pos >= lens - recent) & (pos < lens), float("inf")).masked_fill(pos >= lens, -1.0)
    top = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    n_new = lens.clamp(max=keep)
    slot = torch.arange(top.shape[-1], device=DEV)
    kept = top.masked_fill(slot >= n_new, longest).sort(-1).values
    there = kept < longest
    at = kept.clamp(max=longest - 1)
    for src, dst in zip((*s["rows"], s["weights"]), (*s["out"], s["out_weights"])):
        tail = src.shape[3:]
        view = (n, kv, keep) + (1,) * len(tail)
        rows = torch.gather(src, 2, at.view(view).expand(n, kv, keep, *tail))
        dst[:, :, :keep] = torch.where(there.view(view), rows, dst[:, :, :keep])
    s["out_weights"].masked_fill_(torch.arange(s["out_weights"].shape[-1], device=DEV) >= n_new, 0.0)
    return (kept.masked_fill(~there, -1).to(torch.int32), n_new.flatten(), *s["out"], s["out_weights"])


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"prompt": _prompt_plain, "write": _write_plain, "decode": _decode_plain, "evict": _evict_plain}[op](s)
    from sva_b200 import kernels

    if op == "prompt":
        return kernels.prompt_attention(s["q"], s["keys"], s["values"], s["cu"], cu_seqlens_k=s["cu_k"])
    if op == "write":
        cache = kernels.Kv4Cache(*s["cache"])
        kernels.kv4_write(s["keys"], s["values"], cache, s["start"], page_table=s["table"])
        return kernels.kv4_read(cache, s["start"], s["case"]["tokens"], dtype=s["keys"].dtype, page_table=s["table"])
    if op == "decode":
        out = kernels.kv4_decode(s["q"], kernels.Kv4Cache(*s["cache"]), seq_lens=s["lens"], page_table=s["table"],
                                 max_len=s["longest"], weights=s["weights"])
        return out if s["weights"] is None else (out, s["weights"])
    kept, lens = kernels.cache_evict(s["rows"], s["weights"], s["lens"], s["case"]["keep"], recent=s["case"]["recent"],
                                     out=s["out"], out_weights=s["out_weights"])
    return (kept, lens, *s["out"], s["out_weights"])


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    op, dim, kv = case["op"], case["dim"], case["kv"]
    cell = dim // 2 + dim // GROUP * 4  # bytes of one 4-bit row with its parameters
    if op == "write":
        rows = case["seqs"] * kv * case["tokens"] * 2
        wide = torch.finfo(TYPES[case["dtype"]]).bits // 8 * dim
        return {"bytes": rows * (2 * wide + 2 * cell), "flops": rows * dim * 6}
    lens = _lengths(case)
    if op == "prompt":
        lk = lens + case["cached"]
        pairs = float((lens * lk - lens * (lens - 1) // 2).sum())
        size = torch.finfo(TYPES[case["dtype"]]).bits // 8
        return {"bytes": size * dim * float((2 * case["heads"] * lens + 2 * kv * lk).sum()),
                "flops": 4.0 * dim * case["heads"] * pairs}
    if op == "decode":
        size = torch.finfo(TYPES[case["dtype"]]).bits // 8
        total = float(lens.sum())
        flat = 2 * size * case["seqs"] * case["heads"] * case["tokens"] * dim
        return {"bytes": total * kv * (2 * cell + (8 if case["weights"] else 0)) + flat,
                "flops": 4.0 * dim * case["heads"] * case["tokens"] * total}
    row = 2 * cell if case["bits"] == 4 else 4 * dim
    kept = float(np.minimum(lens, case["keep"]).sum())
    return {"bytes": kv * (4 * float(lens.sum()) + kept * (2 * row + 4 + 4)), "flops": kv * float(lens.sum())}


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ------------------------------------------------------------------------------------------
def _attend64(q, k, v, first):
    """Rows q [H, T, D] over k, v [Hkv, L, D]: row t sees keys 0 .. first + t. Output and weights, a head at a time."""
    h, t, d = q.shape
    out = torch.zeros(h, t, d, dtype=torch.float64, device=DEV)
    mass = torch.zeros(k.shape[0], k.shape[1], dtype=torch.float64, device=DEV)
    allowed = torch.arange(k.shape[1], device=DEV)[None, :] <= first + torch.arange(t, device=DEV)[:, None]
    for i in range(h):
        j = i * k.shape[0] // h
        x = torch.where(allowed, (q[i] @ k[j].T) / math.sqrt(d), -math.inf)
        some = allowed.any(1)
        p = torch.softmax(x[some], 1)
        out[i, some] = p @ v[j]
        mass[j] += p.sum(0)
    return out, mass


def _rows64(s, which, b, upto):
    """Rows 0 .. upto of sequence b of the cache in 64 bits."""
    codes, params = s["cache"][2 * which], s["cache"][2 * which + 1]
    if s["table"] is None:
        codes, params = codes[b, :, :upto], params[b, :, :upto]
    else:
        pages = s["table"][b].long()[: -(-upto // codes.shape[2])]
        codes = codes[pages].transpose(0, 1).flatten(1, 2)[:, :upto]
        params = params[pages].transpose(0, 1).flatten(1, 2)[:, :upto]
    x = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=DEV)
    x[..., 0::2] = (codes % 16).double()
    x[..., 1::2] = (codes // 16).double()
    return x * params[..., 0].double().repeat_interleave(GROUP, -1) + params[..., 1].double().repeat_interleave(GROUP, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "prompt":
        cu, cu_k, got = s["cu"].tolist(), s["cu_k"].tolist(), []
        for a, b, c, d in zip(cu, cu[1:], cu_k, cu_k[1:]):
            o, _ = _attend64(s["q"][a:b].double().transpose(0, 1), s["keys"][c:d].double().transpose(0, 1),
                             s["values"][c:d].double().transpose(0, 1), (d - c) - (b - a))
            got.append(o.transpose(0, 1))
        return torch.cat(got)
    if op == "write":
        def nearest(x):
            g = x.double().unflatten(-1, (-1, GROUP))
            low, high = g.min(-1).values, g.max(-1).values
            # to 8 bits of mantissa, downwards and upwards
            f, e = torch.frexp(low)
            m = torch.ldexp(torch.floor(f * 256), e - 8)
            f, e = torch.frexp((high - m) / 15)
            w = torch.ldexp(torch.ceil(f * 256), e - 8).unsqueeze(-1)
            c = torch.round((g - m.unsqueeze(-1)) / w.masked_fill(w == 0, 1.0)).clip(0, 15)
            return (c * w + m.unsqueeze(-1)).flatten(-2)

        return nearest(s["keys"]), nearest(s["values"])
    if op == "decode":
        lens = s["lens"].tolist()
        out = torch.zeros(case["seqs"], case["heads"], case["tokens"], case["dim"], dtype=torch.float64, device=DEV)
        mass = torch.zeros(case["seqs"], case["kv"], s["longest"], dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            out[b], mass[b, :, :n] = _attend64(s["q"][b].double(), _rows64(s, 0, b, n), _rows64(s, 1, b, n),
                                               n - case["tokens"])
        return (out, mass) if case["weights"] else out
    w, lens, keep, recent = s["weights"].cpu().numpy(), s["lens"].tolist(), case["keep"], case["recent"]
    kept = np.full((case["seqs"], case["kv"], keep), -1, dtype=np.int32)
    out = [o.clone() for o in s["out"]]
    mass = torch.zeros_like(s["out_weights"])
    for b, n in enumerate(lens):
        for h in range(case["kv"]):
            old = max(0, n - recent)
            best = np.lexsort((np.arange(old), -w[b, h, :old].astype(np.float64)))[: max(0, min(n, keep) - (n - old))]
            rows = np.sort(np.concatenate([best, np.arange(old, n)]))[:min(n, keep)]
            kept[b, h, :len(rows)] = rows
            at = torch.from_numpy(rows).to(DEV)
            for src, dst in zip(s["rows"], out):
                dst[b, h, :len(rows)] = src[b, h, at]
            mass[b, h, :len(rows)] = s["weights"][b, h, at]
    return (torch.from_numpy(kept), torch.tensor([min(n, keep) for n in lens]), *out, mass.double())
