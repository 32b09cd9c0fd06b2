"""Workloads of the streaming-attention operators: rotary positions over several axes,
masked attention over packed documents, the quantised key/value cache and attention
over it.

`run` computes an operator either in its plain form (elementary torch operations in 32
bits, `own = False`) or through the framework's entry points (`own = True`); both take
the state that `prepare` makes from a case and a seed.
"""
import math

import numpy as np
import torch

own = False

HEAD_DIM = 64
VIEW = 866  # tokens of one 504 x 336 view: 1 + 1 special tokens and 36 x 24 patches

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ints(text):
    return [int(t) for t in text.split(",")] if text else []


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _offsets(lens):
    return [0] + [int(v) for v in np.cumsum(lens)]


# ---------------------------------------------------------------------------- cases
def _rope(name, **kw):
    return dict({"op": "rope", "name": name, "rows": 1, "heads": 12, "kv_heads": 12, "dtype": "bf16",
                 "sections": "16,24,24", "layout": "per_axis", "pairing": 0, "base": 100.0, "views": 12,
                 "head_dim": 64}, **kw)


def _attn(name, **kw):
    return dict({"op": "attention", "name": name, "q_lens": "1", "k_lens": "1", "heads": 12, "kv_heads": 12,
                 "dtype": "bf16", "causal": False, "frame": 1, "prefix": "", "bias": False, "cap": 0.0}, **kw)


def _cache(name, **kw):
    return dict({"op": "cache", "name": name, "new": "1", "held": "1", "capacity": 64, "kv_heads": 12,
                 "dtype": "bf16", "format": "int8"}, **kw)


def _cached(name, **kw):
    return dict({"op": "cached_attention", "name": name, "new": "1", "held": "1", "capacity": 64, "heads": 12,
                 "kv_heads": 12, "dtype": "bf16", "format": "int8", "causal": True, "frame": 1, "prefix": "",
                 "bias": False, "cap": 0.0}, **kw)


def listed():
    return [
        # One streaming step's two special tokens: nothing but latency.
        _rope("rope_two_tokens", rows=2),
        # The queries and keys of a 12-view window, as views of one packed projection.
        _rope("rope_window", rows=12 * VIEW),
        # A long clip in F32 with one shared frequency ladder, far time positions.
        _rope("rope_clip_f32", rows=32 * VIEW + 17, heads=16, kv_heads=4, dtype="f32", layout="shared", pairing=1,
              base=10000.0, views=32000),
        # One query token over the window held so far: latency and cache bandwidth.
        _attn("attn_one_token", q_lens="1", k_lens=str(12 * VIEW), causal=True, bias=True),
        # One new view attends to the views held so far and to itself, frame by frame.
        _attn("attn_new_view", q_lens=str(VIEW), k_lens=str(12 * VIEW), causal=True, frame=VIEW, prefix=str(VIEW),
              cap=50.0),
        # Four requests' windows of different sizes packed into one call.
        _attn("attn_packed", q_lens=_text([VIEW * 3, VIEW, VIEW * 5, 731]), k_lens=_text([VIEW * 3, VIEW, VIEW * 5, 731]),
              dtype="f16"),
        # Token-causal documents with a distance bias, shared key heads.
        _attn("attn_bias", q_lens="4097,255,2000,1", k_lens="4097,300,2000,77", heads=16, kv_heads=4, causal=True,
              bias=True),
        # The largest: a whole 12-view window, every token to every token, capped scores.
        _attn("attn_window", q_lens=str(12 * VIEW), k_lens=str(12 * VIEW), cap=30.0),
        # A new view's keys and values into the cache, the views held read back.
        _cache("cache_new_view", new=str(VIEW), held=str(3 * VIEW), capacity=12 * VIEW),
        # Whole windows of four requests written and read back.
        _cache("cache_windows", new=_text([12 * VIEW, 8 * VIEW, 1, 5001]), held=_text([12 * VIEW, 8 * VIEW, 9000, 5001]),
               capacity=12 * VIEW, dtype="f16", format="e4m3", kv_heads=16),
        # One token of one request over its cached window.
        _cached("cached_one_token", new="1", held=str(12 * VIEW), capacity=12 * VIEW),
        # Sixteen requests, one to four tokens each, shared key heads, every score term.
        _cached("cached_batch", new="1,1,2,1,4,1,0,1,1,3,1,1,1,2,1,1",
                held="32000,17,20011,8660,31999,1,0,12345,27712,866,30000,4097,25000,16000,128,22222",
                capacity=32000, heads=16, kv_heads=4, dtype="f16", format="e4m3", prefix=_text([0, 5] * 8),
                bias=True, cap=50.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "cache", "cached_attention"])
    dtype = rng.choice(["bf16", "f16"])
    heads, kv_heads = rng.choice([(12, 12), (16, 16), (16, 4), (12, 4), (6, 1), (8, 2), (10, 5), (3, 3)])
    if op == "rope":
        head_dim, sections = rng.choice([(64, "16,24,24"), (64, "32,32"), (64, "64"), (64, "20,22,22"), (64, "8,16,24"),
                                         (128, "32,48,48"), (96, "2,40,40")])
        case = _rope("", rows=_log_int(rng, 1, 20000), heads=heads, kv_heads=kv_heads,
                     dtype=rng.choice(["bf16", "f16", "f32"]), head_dim=head_dim, sections=sections,
                     layout=rng.choice(["per_axis", "shared"]), pairing=rng.choice([0, 1]),
                     base=rng.choice([100.0, 10000.0]), views=_log_int(rng, 1, 100000))
    elif op == "attention":
        docs = rng.randint(1, 6)
        q, k = [], []
        for _ in range(docs):
            kl = _log_int(rng, 1, 4000)
            kind = rng.choice(["same", "few", "tail", "longer"])
            ql = {"same": kl, "few": rng.randint(0, 5), "tail": rng.randint(1, kl), "longer": kl + rng.randint(1, 200)}[kind]
            q.append(ql)
            k.append(0 if rng.random() < 0.05 else kl)
        if sum(q) == 0:
            q[0] = 1
        if sum(k) == 0:
            k[0] = 1
        causal = rng.random() < 0.6
        case = _attn("", q_lens=_text(q), k_lens=_text(k), heads=heads, kv_heads=kv_heads, dtype=dtype, causal=causal,
                     frame=rng.choice([1, 1, _log_int(rng, 2, 900)]),
                     prefix=_text([rng.randint(0, v) if rng.random() < 0.5 else 0 for v in k]) if causal else "",
                     bias=rng.random() < 0.5, cap=rng.choice([0.0, 30.0, 50.0]))
    else:
        docs = rng.randint(1, 8)
        held = [_log_int(rng, 1, 9000) for _ in range(docs)]
        capacity = max(held) + rng.randint(0, 100)
        fmt = rng.choice(["int8", "e4m3"])
        if op == "cache":
            new = [rng.choice([0, 1, rng.randint(0, h), h]) for h in held]
            if sum(new) == 0:
                new[0] = 1
            case = _cache("", new=_text(new), held=_text(held), capacity=capacity, kv_heads=kv_heads,
                          dtype=rng.choice(["bf16", "f16", "f32"]), format=fmt)
        else:
            new = [min(h, rng.choice([0, 1, 1, 1, rng.randint(1, 9)])) for h in held]
            if sum(new) == 0:
                new[0] = 1
            case = _cached("", new=_text(new), held=_text(held), capacity=capacity, heads=heads, kv_heads=kv_heads,
                           dtype=dtype, format=fmt, causal=rng.random() < 0.8,
                           frame=rng.choice([1, 1, _log_int(rng, 2, 900)]),
                           prefix=_text([rng.randint(0, h) if rng.random() < 0.5 else 0 for h in held]),
                           bias=rng.random() < 0.5, cap=rng.choice([0.0, 30.0, 50.0]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------- state
def _context():
    import os
    import sys
    pkg = os.path.join(os.getcwd(), "vestra-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import vestra_attn as va
    return va, va.Context(va.default_config(max_rows=64), torch.cuda.current_device())


def _slopes(heads):
    """The geometric ladder of distance biases: 2^(-8 (h + 1) / heads)."""
    return np.array([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], np.float32)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _qkv(gen, q_rows, k_rows, heads, kv_heads, dtype):
    """Queries and keys as QK normalisation leaves them (unit variance, a gain of its own
    per head and a shared component that makes scores of a few units); values with a mean."""
    gain = 0.5 + 2.0 * torch.rand(1, heads, 1, generator=gen, device="cuda")
    common = _randn(gen, 1, 1, HEAD_DIM)
    q = ((_randn(gen, q_rows, heads, HEAD_DIM) + 0.3 * common) * gain).to(dtype)
    k = (_randn(gen, k_rows, kv_heads, HEAD_DIM) + 0.3 * common).to(dtype)
    v = (_randn(gen, k_rows, kv_heads, HEAD_DIM) + 0.5 * _randn(gen, 1, kv_heads, HEAD_DIM)).to(dtype)
    return q, k, v


def _quantise(x, fmt):
    """Codes and one scale per (row, head) of x [rows, heads, 64].  int8: scale = amax / 127,
    code = x / scale rounded half to even (in 64 bits: quotients next to a half step
    count); e4m3: the power of two that brings amax to at most 448."""
    x = x.double()
    amax = x.abs().amax(-1)
    if fmt == "int8":
        scale = (amax / 127.0).float().clamp_min(2.0 ** -126)
        codes = torch.round(x / scale.double()[..., None]).clamp(-127, 127).to(torch.int8)
    else:
        m, e = torch.frexp(amax / 448.0)  # amax / 448 = m 2^e, 0.5 <= m < 1
        e = torch.where(m == 0.5, e - 1, e).clamp_min(-126)
        scale = torch.ldexp(torch.ones_like(amax), e).float()
        codes = (x / scale.double()[..., None]).float().to(torch.float8_e4m3fn)
    return codes, scale


def _cache_buffers(gen, case):
    """A cache whose rows before the call's new ones are in place (other rows hold
    what an earlier request left)."""
    fmt, docs = case["format"], len(_ints(case["held"]))
    shape = (docs, case["kv_heads"], case["capacity"])
    out = {}
    for name in ("k", "v"):
        if fmt == "int8":
            codes = torch.randint(-127, 128, shape + (HEAD_DIM,), generator=gen, device="cuda", dtype=torch.int8)
            codes[..., 0] = 127
            scale = 0.02 + 0.01 * torch.rand(shape, generator=gen, device="cuda")
        else:
            codes = (torch.randn(shape + (HEAD_DIM,), generator=gen, device="cuda", dtype=torch.float16) * 64).clamp(
                -448, 448).to(torch.float8_e4m3fn)
            scale = torch.ldexp(torch.ones(shape, device="cuda"),
                                torch.randint(-8, -5, shape, generator=gen, device="cuda", dtype=torch.int32))
        out[name] = codes
        out[name + "_scale"] = scale.contiguous()
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    st = {"case": case}
    if own:
        va, st["ctx"] = _context()
    if op == "rope":
        rows, heads, kvh, d = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        packed = _randn(gen, rows, heads + 2 * kvh, d).to(dtype)
        st["q"], st["k"] = packed[:, :heads], packed[:, heads:heads + kvh]
        sections = _ints(case["sections"])
        pos = torch.randint(0, 40, (rows, len(sections)), generator=gen, device="cuda", dtype=torch.int32)
        pos[:, 0] = torch.randint(0, case["views"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
        st["positions"] = pos
        if own:
            st["rope"] = va.RopeAxes(sections, base=case["base"], layout=case["layout"], pairing=case["pairing"])
            st["q_out"] = torch.empty(rows, heads, d, device="cuda", dtype=dtype)
            st["k_out"] = torch.empty(rows, kvh, d, device="cuda", dtype=dtype)
        return st
    heads = case.get("heads", 0)
    if op == "attention":
        ql, kl = _ints(case["q_lens"]), _ints(case["k_lens"])
        st["q"], st["k"], st["v"] = _qkv(gen, sum(ql), sum(kl), heads, case["kv_heads"], dtype)
        st["slopes"] = torch.from_numpy(_slopes(heads)).cuda() if case["bias"] else None
        if own:
            st["plan"] = va.AttentionPlan(st["ctx"], heads, case["kv_heads"], _offsets(ql), _offsets(kl),
                                          causal=case["causal"], frame=case["frame"],
                                          prefix=_ints(case["prefix"]) or None,
                                          slopes=_slopes(heads) if case["bias"] else None, score_cap=case["cap"])
            st["out"] = torch.empty_like(st["q"])
        return st
    new, held = _ints(case["new"]), _ints(case["held"])
    st["buf"] = _cache_buffers(gen, case)
    st["offsets"] = torch.tensor(_offsets(new), device="cuda", dtype=torch.int32)
    st["lens"] = torch.tensor(held, device="cuda", dtype=torch.int32)
    if own:
        b = st["buf"]
        st["cache"] = va.KvCache(b["k"], b["v"], b["k_scale"], b["v_scale"])
    if op == "cache":
        _, st["k"], st["v"] = _qkv(gen, 0, sum(new), 1, case["kv_heads"], dtype)
        st["held_offsets"] = torch.tensor(_offsets(held), device="cuda", dtype=torch.int32)
        if own:
            st["k_out"] = torch.empty(sum(held), case["kv_heads"], HEAD_DIM, device="cuda", dtype=dtype)
            st["v_out"] = torch.empty_like(st["k_out"])
        return st
    st["q"], _, _ = _qkv(gen, sum(new), 0, heads, case["kv_heads"], dtype)
    pre = _ints(case["prefix"])
    st["prefix"] = torch.tensor(pre, device="cuda", dtype=torch.int32) if pre else None
    st["slopes"] = torch.from_numpy(_slopes(heads)).cuda() if case["bias"] else None
    if own:
        st["out"] = torch.empty_like(st["q"])
    return st


# ---------------------------------------------------------------------------- one pass
def run(st):
    return {"rope": _run_rope, "attention": _run_attention, "cache": _run_cache,
            "cached_attention": _run_cached}[st["case"]["op"]](st)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _pairs(sections, layout, pairing):
    """Per rotated pair: its two dims, its axis and its exponent 2 i / block."""
    first, second, axis, power = [], [], [], []
    start = 0
    total = sum(sections)
    shared = 0
    for a, s in enumerate(sections):
        for i in range(s // 2):
            j = shared if layout == "shared" else i
            block = total if layout == "shared" else s
            o = 0 if layout == "shared" else start
            first.append(o + (j if pairing == 0 else 2 * j))
            second.append(o + (j + block // 2 if pairing == 0 else 2 * j + 1))
            axis.append(a)
            power.append(2.0 * j / block)
            shared += 1
        start += s
    return first, second, axis, power


def _run_rope(st):
    case = st["case"]
    if own:
        # F32 operands turn in place, as in the plain form (where .float() is no copy).
        in_place = case["dtype"] == "f32"
        q_out, k_out = (st["q"], st["k"]) if in_place else (st["q_out"], st["k_out"])
        st["ctx"].rope_axes(st["rope"], st["positions"], st["q"], q_out, st["k"], k_out, stream=_stream())
        return q_out, k_out
    first, second, axis, power = _pairs(_ints(case["sections"]), case["layout"], case["pairing"])
    freq = torch.tensor([case["base"] ** -p for p in power], device="cuda", dtype=torch.float64)
    angle = st["positions"].double()[:, axis] * freq  # far positions: 64 bits
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    outs = []
    for x in (st["q"], st["k"]):
        y = x.float()
        x0, x1 = y[..., first], y[..., second]
        y[..., first], y[..., second] = x0 * c - x1 * s, x1 * c + x0 * s
        outs.append(y.to(x.dtype).contiguous())
    return tuple(outs)


def _limit(n_q, n_k, causal, frame, prefix, dev):
    """Keys each of the n_q rows (the last ones of n_k positions) sees: the first `limit`."""
    pos = torch.arange(n_q, device=dev) + (n_k - n_q)
    if not causal:
        return pos, torch.full_like(pos, n_k)
    end = (torch.div(pos, frame, rounding_mode="floor") + 1) * frame
    return pos, end.clamp_min(prefix).clamp(0, n_k)


def _attend(q, k, v, causal, frame, prefix, slopes, cap):
    """Plain attention of one document: q [n, H, 64], k and v [m, KV, 64], F32 out."""
    n, heads = q.shape[:2]
    m, kvh = k.shape[:2]
    out = torch.zeros(n, heads, HEAD_DIM, device=q.device, dtype=torch.float32)
    if n == 0 or m == 0:
        return out
    group = heads // kvh
    pos, limit = _limit(n, m, causal, frame, prefix, q.device)
    keys = torch.arange(m, device=q.device)
    hidden = keys[None, :] >= limit[:, None]
    empty = limit <= 0
    dist = None
    if slopes is not None:
        fq, fk = torch.div(pos, frame, rounding_mode="floor"), torch.div(keys, frame, rounding_mode="floor")
        dist = (fq[:, None] - fk[None, :]).abs().float()
    for h in range(heads):
        s = (q[:, h].float() @ k[:, h // group].float().T) * (1.0 / math.sqrt(HEAD_DIM))
        if cap > 0:
            s = cap * torch.tanh(s / cap)
        if dist is not None:
            s = s - slopes[h] * dist
        s = s.masked_fill(hidden, float("-inf"))
        s = s - s.amax(-1, keepdim=True).masked_fill(empty[:, None], 0.0)
        p = s.exp()
        o = (p @ v[:, h // group].float()) / p.sum(-1, keepdim=True).masked_fill(empty[:, None], 1.0)
        out[:, h] = o
    return out


def _run_attention(st):
    case = st["case"]
    if own:
        st["ctx"].masked_attention(st["plan"], st["q"], st["k"], st["v"], st["out"], stream=_stream())
        return st["out"]
    q, k, v = st["q"], st["k"], st["v"]
    qo, ko = _offsets(_ints(case["q_lens"])), _offsets(_ints(case["k_lens"]))
    pre = _ints(case["prefix"]) or [0] * (len(qo) - 1)
    outs = [_attend(q[qo[b]:qo[b + 1]], k[ko[b]:ko[b + 1]], v[ko[b]:ko[b + 1]], case["causal"], case["frame"], pre[b],
                    st["slopes"], case["cap"]) for b in range(len(qo) - 1)]
    return torch.cat(outs).to(q.dtype)


def _run_cache(st):
    case, b = st["case"], st["buf"]
    if own:
        st["ctx"].kv_cache_write(st["cache"], st["k"], st["v"], st["offsets"], st["lens"], stream=_stream())
        st["ctx"].kv_cache_read(st["cache"], st["held_offsets"], st["k_out"], st["v_out"], stream=_stream())
        return {"k": st["k_out"], "v": st["v_out"], "k_scale": b["k_scale"], "v_scale": b["v_scale"]}
    new, held = _ints(case["new"]), _ints(case["held"])
    off = _offsets(new)
    out = {}
    for name in ("k", "v"):
        x, codes, scales = st[name], b[name], b[name + "_scale"]
        c, s = _quantise(x, case["format"])
        parts = []
        top = torch.finfo(x.dtype).max
        for d, (n, h) in enumerate(zip(new, held)):
            if n:
                codes[d, :, h - n:h].view(torch.int8).copy_(
                    c[off[d]:off[d + 1]].transpose(0, 1).contiguous().view(torch.int8))
                scales[d, :, h - n:h] = s[off[d]:off[d + 1]].T
            val = codes[d, :, :h].float() * scales[d, :, :h, None]
            parts.append(val.clamp(-top, top).transpose(0, 1))
        out[name] = torch.cat(parts).to(x.dtype)
    return {"k": out["k"], "v": out["v"], "k_scale": b["k_scale"], "v_scale": b["v_scale"]}


def _run_cached(st):
    case = st["case"]
    if own:
        st["ctx"].cache_attention(st["cache"], st["q"], st["out"], st["offsets"], st["lens"],
                                  max_tokens=max(_ints(case["new"])), causal=case["causal"], frame=case["frame"],
                                  prefix=st["prefix"], slopes=st["slopes"], score_cap=case["cap"], stream=_stream())
        return st["out"]
    new, held, b, q = _ints(case["new"]), _ints(case["held"]), st["buf"], st["q"]
    off = _offsets(new)
    pre = _ints(case["prefix"]) or [0] * len(new)
    outs = []
    for d, (n, h) in enumerate(zip(new, held)):
        if n == 0:
            continue
        k = (b["k"][d, :, :h].float() * b["k_scale"][d, :, :h, None]).transpose(0, 1)
        v = (b["v"][d, :, :h].float() * b["v_scale"][d, :, :h, None]).transpose(0, 1)
        outs.append(_attend(q[off[d]:off[d + 1]], k, v, case["causal"], case["frame"], pre[d], st["slopes"],
                            case["cap"]))
    return torch.cat(outs).to(q.dtype)


# ---------------------------------------------------------------------------- cost
def _visible(n, m, causal, frame, prefix):
    """(row, key) pairs a document's attention looks at."""
    if n == 0 or m == 0:
        return 0
    if not causal:
        return n * m
    pos = np.arange(n, dtype=np.int64) + (m - n)
    end = np.clip(np.maximum((pos // frame + 1) * frame, prefix), 0, m)
    return int(end.sum())


def work(case):
    op = case["op"]
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if op == "rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * size + 4 * case["rows"] * len(_ints(case["sections"])), "flops": 3 * n}
    kvh = case["kv_heads"]
    if op == "attention":
        ql, kl = _ints(case["q_lens"]), _ints(case["k_lens"])
        pre = _ints(case["prefix"]) or [0] * len(ql)
        pairs = sum(_visible(n, m, case["causal"], case["frame"], p) for n, m, p in zip(ql, kl, pre))
        seen = sum(m for n, m in zip(ql, kl) if n)
        return {"bytes": HEAD_DIM * size * (2 * sum(ql) * case["heads"] + 2 * seen * kvh),
                "flops": 4 * HEAD_DIM * pairs * case["heads"]}
    new, held = _ints(case["new"]), _ints(case["held"])
    row = 2 * kvh * (HEAD_DIM + 4)  # codes and scales of K and V
    if op == "cache":
        wide = 2 * kvh * HEAD_DIM * size
        return {"bytes": sum(new) * (wide + row) + sum(held) * (wide + row),
                "flops": 4 * kvh * HEAD_DIM * (sum(new) + sum(held))}
    pre = _ints(case["prefix"]) or [0] * len(new)
    pairs = sum(_visible(n, m, case["causal"], case["frame"], p) for n, m, p in zip(new, held, pre))
    seen = sum(m for n, m in zip(new, held) if n)
    return {"bytes": seen * row + 2 * sum(new) * case["heads"] * HEAD_DIM * size,
            "flops": 4 * HEAD_DIM * pairs * case["heads"]}


# ---------------------------------------------------------------------------- definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return tuple(_exact_rope(x.double(), st["positions"].double(), case) for x in (st["q"], st["k"]))
    if op == "attention":
        qo, ko = _offsets(_ints(case["q_lens"])), _offsets(_ints(case["k_lens"]))
        res = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
        for b in range(len(qo) - 1):
            _exact_attention(res[qo[b]:qo[b + 1]], st["q"][qo[b]:qo[b + 1]].double(), st["k"][ko[b]:ko[b + 1]].double(),
                             st["v"][ko[b]:ko[b + 1]].double(), case, b)
        return res
    new, held, buf = _ints(case["new"]), _ints(case["held"]), st["buf"]
    if op == "cached_attention":
        res = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
        row = 0
        for b, (n, h) in enumerate(zip(new, held)):
            k = torch.einsum("hmd,hm->mhd", buf["k"][b, :, :h].double(), buf["k_scale"][b, :, :h].double())
            v = torch.einsum("hmd,hm->mhd", buf["v"][b, :, :h].double(), buf["v_scale"][b, :, :h].double())
            _exact_attention(res[row:row + n], st["q"][row:row + n].double(), k, v, case, b)
            row += n
        return res
    out = {}
    for name in ("k", "v"):
        values = [buf[name][b, :, :h].double() * buf[name + "_scale"][b, :, :h, None].double()
                  for b, h in enumerate(held)]
        scales = buf[name + "_scale"].double().clone()
        row = 0
        for b, (n, h) in enumerate(zip(new, held)):
            if n == 0:
                continue
            x = st[name][row:row + n].double().permute(1, 0, 2)  # [heads, n, 64]
            row += n
            top = x.abs().max(dim=-1).values
            if case["format"] == "int8":
                step = torch.clamp((top / 127).to(torch.float32).double(), min=2.0 ** -126)
                y = torch.round(x / step[..., None])
            else:
                step = torch.exp2(torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448)).clamp(min=-126))
                u = x / step[..., None]
                # spacing of e4m3 at |u|: 2^(floor(log2 |u|) - 3), at least 2^-9
                gap = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
                y = torch.round(u / gap) * gap
            values[b][:, h - n:h] = y * step[..., None]
            scales[b, :, h - n:h] = step
        limit = torch.finfo(DTYPES[case["dtype"]]).max
        out[name] = torch.cat([w.permute(1, 0, 2) for w in values]).clamp(-limit, limit)
        out[name + "_scale"] = scales
    return {"k": out["k"], "v": out["v"], "k_scale": out["k_scale"], "v_scale": out["v_scale"]}


def _exact_rope(x, pos, case):
    sections = _ints(case["sections"])
    y = x.clone()
    total = sum(sections)
    if case["layout"] == "shared":
        ids = torch.repeat_interleave(torch.arange(len(sections), device="cuda"),
                                      torch.tensor([s // 2 for s in sections], device="cuda"))
        blocks = [(0, total, pos[:, ids])]
    else:
        starts = np.cumsum([0] + sections)
        blocks = [(int(starts[a]), s, pos[:, a:a + 1].expand(-1, s // 2)) for a, s in enumerate(sections)]
    for start, size, p in blocks:
        i = torch.arange(size // 2, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones_like(p), p * torch.pow(torch.tensor(case["base"], dtype=torch.float64,
                                                                          device="cuda"), -2 * i / size))
        part = x[..., start:start + size]
        if case["pairing"] == 0:
            z = torch.complex(part[..., :size // 2].contiguous(), part[..., size // 2:].contiguous()) * turn[:, None]
            y[..., start:start + size] = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], size // 2, 2).contiguous()) * turn[:, None]
            y[..., start:start + size] = torch.view_as_real(z).reshape(part.shape)
    return y


def _exact_attention(res, q, k, v, case, b):
    """Fills res [n, H, 64] with the softmax over the visible keys, rows in blocks."""
    n, m = q.shape[0], k.shape[0]
    if n == 0 or m == 0:
        return
    frame, cap = case["frame"], case["cap"]
    pre = _ints(case["prefix"])
    kf = torch.arange(m, device="cuda") // frame
    share = case["heads"] // case["kv_heads"]
    for r0 in range(0, n, 2048):
        r1 = min(n, r0 + 2048)
        at = torch.arange(r0, r1, device="cuda") + (m - n)
        qf = torch.floor(at.double() / frame).long()
        seen = torch.ones(r1 - r0, m, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = (kf[None] <= qf[:, None]) | (torch.arange(m, device="cuda") < (pre[b] if pre else 0))[None]
        some = seen.any(1)
        for h in range(case["heads"]):
            x = torch.einsum("nd,md->nm", q[r0:r1, h], k[:, h // share]) / math.sqrt(HEAD_DIM)
            if cap:
                x = torch.tanh(x / cap) * cap
            if case["bias"]:
                x = x - float(_slopes(case["heads"])[h]) * (qf[:, None] - kf[None]).abs().double()
            x = torch.where(seen, x, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
            w = torch.softmax(x, dim=-1)
            o = torch.einsum("nm,md->nd", torch.where(some[:, None], w, torch.zeros_like(w)), v[:, h // share])
            res[r0:r1, h] = o
