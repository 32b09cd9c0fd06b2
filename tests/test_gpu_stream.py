"""Streaming-attention operators on the GPU against plain 64-bit implementations: rotary
positions over several axes, masked attention over packed documents, the quantised
key/value cache and attention over it.  Every call goes through the C ABI.

Tolerances count roundings.  A result rounded to a type t is off by at most u = eps(t) / 2
of its value (u = 2^-8 bf16, 2^-11 f16, 2^-24 f32).  The masked attention rounds each
probability to the operands' type (u again), so an output is off by at most
u * A + u * |out|, A = sum p |v| / sum p; scores, exponentials and sums are F32, whose
part is below 2^-12 * A for scores up to a few hundred.  The cache attention splits
probabilities in two bf16 parts (2^-16 of each)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

import vestra_attn as va  # noqa: E402

D = 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ctx():
    c = va.Context(va.default_config(max_rows=64), 0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def _no_device_error(ctx):
    yield
    torch.cuda.synchronize()
    ctx.check_device()


@pytest.fixture(autouse=True)
def _float32_by_default():
    """Other test modules make 64 bits torch's default."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(F32)
    yield
    torch.set_default_dtype(before)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


# ------------------------------------------------------------------------------- rope
def rope_ref(x, pos, sections, base, layout, pairing):
    y = x.double().clone()
    total, start, shared = sum(sections), 0, 0
    for a, s in enumerate(sections):
        for i in range(s // 2):
            block, origin, j = (total, 0, shared) if layout == "shared" else (s, start, i)
            c0 = origin + (2 * j if pairing else j)
            c1 = origin + (2 * j + 1 if pairing else j + block // 2)
            ang = pos[:, a].double() * base ** (-2.0 * j / block)
            c, sn = ang.cos()[:, None], ang.sin()[:, None]
            x0, x1 = x[..., c0].double(), x[..., c1].double()
            y[..., c0], y[..., c1] = x0 * c - x1 * sn, x1 * c + x0 * sn
            shared += 1
        start += s
    return y


def rope_tol(x, dtype):
    # result half step, plus F32 products, the sum, and cos / sin good to 2^-22
    return half_step(dtype) * 1.5 * x.double().abs().amax() + 2.0 ** -20 * x.double().abs().amax()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["per_axis", "shared"])
@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("d,sections", [(64, (16, 24, 24)), (64, (20, 22, 22)), (64, (32, 32)), (64, (64,)),
                                        (128, (32, 48, 48)), (96, (2, 40, 40)), (6, (2,)), (256, (64, 64, 64, 64))])
def test_rope_matches_64_bit(ctx, dtype, layout, pairing, d, sections):
    g = gen(d + pairing)
    rows = 37
    q, k = randn(g, rows, 3, d, dtype=dtype), randn(g, rows, 2, d, dtype=dtype)
    pos = torch.randint(-50, 50, (rows, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 2 ** 31 - 1  # far positions: the angle is reduced in 64 bits
    pos[1] = -(2 ** 31)
    pos[2] = 0
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ctx.rope_axes(va.RopeAxes(sections, 100.0, layout, pairing), pos, q, qo, k, ko)
    for x, y in ((q, qo), (k, ko)):
        ref = rope_ref(x, pos, sections, 100.0, layout, pairing)
        err = (y.double() - ref).abs()
        # far rows: base^p is rounded to 64 bits, 2^31 * 2^-52 of a turn more
        assert err.max() <= rope_tol(x, dtype) + 2.0 ** -17 * (err[:2].max() == err.max()).double()
        assert err[2:].max() <= rope_tol(x, dtype)
        assert torch.equal(y[2], x[2])  # position 0 turns nothing
        assert torch.equal(y[..., sum(sections):], x[..., sum(sections):])


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 1000])
def test_rope_in_place_strided_and_odd_alignment(ctx, rows):
    g = gen(rows)
    sections = (16, 24, 24)
    pos = torch.randint(0, 900, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
    rope = va.RopeAxes(sections)
    packed = randn(g, rows, 9, D, dtype=BF16)  # 4 query, 2 key, 2 value heads and a spare
    before = packed.clone()
    q, k = packed[:, :4], packed[:, 4:6]
    ctx.rope_axes(rope, pos, q, q, k, k)
    for x, y in ((before[:, :4], q), (before[:, 4:6], k)):
        assert (y.double() - rope_ref(x, pos, sections, 100.0, "per_axis", 0)).abs().max() <= rope_tol(x, BF16)
    assert torch.equal(packed[:, 6:], before[:, 6:])
    # one element off any vector boundary, head-major
    flat = randn(g, 3 * rows * D + 1, dtype=F16)
    x = flat[1:].view(3, rows, D).transpose(0, 1)
    out = torch.zeros(3 * rows * D + 3, device="cuda", dtype=F16)[3:].view(rows, 3, D)
    ctx.rope_axes(rope, pos, x, out)
    assert (out.double() - rope_ref(x, pos, sections, 100.0, "per_axis", 0)).abs().max() <= rope_tol(x, F16)


def test_rope_two_axes_is_the_layer_paths_rope(ctx):
    """Sections (32, 32), per axis, base 100: the (y, x) rotation of Op::Attention's restatement."""
    g = gen(7)
    n = 50
    x = randn(g, n, 2, D)
    pos = torch.randint(0, 40, (n, 2), generator=g, device="cuda", dtype=torch.int32)
    y = torch.empty_like(x)
    ctx.rope_axes(va.RopeAxes((32, 32)), pos, x, y)
    import oracle
    oracle.build()
    ref = oracle.rope2d(x.transpose(0, 1).contiguous().cpu().numpy(), pos.cpu().numpy().astype(np.float32), 100.0)
    assert np.abs(y.transpose(0, 1).cpu().numpy() - ref).max() <= 2e-6 * 4


# ------------------------------------------------------------------- masked attention
def attention_ref(q, k, v, causal, frame, prefix, slopes, cap, scale=0.125):
    """One document in 64 bits -> (out, A): q [n, H, 64], k, v [m, KV, 64]."""
    n, heads = q.shape[:2]
    m, kvh = k.shape[:2]
    out = torch.zeros(n, heads, D, device="cuda", dtype=torch.float64)
    a = torch.zeros_like(out)
    if n == 0 or m == 0:
        return out, a
    p = torch.arange(n, device="cuda") + (m - n)
    j = torch.arange(m, device="cuda")
    fp, fj = torch.div(p, frame, rounding_mode="floor"), torch.div(j, frame, rounding_mode="floor")
    seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
    if causal:
        seen = (fj[None] <= fp[:, None]) | (j < prefix)[None]
    for h in range(heads):
        kd, vd = k[:, h * kvh // heads].double(), v[:, h * kvh // heads].double()
        s = q[:, h].double() @ kd.T * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * (fp[:, None] - fj[None]).abs().double()
        s = s.masked_fill(~seen, -torch.inf)
        w = torch.softmax(s, -1).masked_fill(~seen.any(1, keepdim=True), 0.0)
        out[:, h], a[:, h] = w @ vd, w @ vd.abs()
    return out, a


def check_attention(got, ref, a, p_step=None):
    if got.numel() == 0:
        return
    u = half_step(got.dtype)
    tol = (u if p_step is None else p_step) * a + u * ref.abs() + 2.0 ** -12 * a + 1e-6
    bad = (got.double() - ref).abs() > tol
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, worst {worst:.2f} of the tolerance"
    assert torch.isfinite(got.float()).all()


def run_masked(ctx, ql, kl, heads, kvh, dtype, causal=False, frame=1, prefix=None, bias=False, cap=0.0, scale=0.0,
               seed=0, gain=1.5):
    g = gen(seed)
    q, k, v = (randn(g, sum(ql), heads, D, dtype=F32) * gain).to(dtype), randn(g, sum(kl), kvh, D, dtype=dtype), \
        randn(g, sum(kl), kvh, D, dtype=dtype)
    slopes = np.array([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], np.float32) if bias else None
    qo, ko = np.cumsum([0] + list(ql)), np.cumsum([0] + list(kl))
    plan = va.AttentionPlan(ctx, heads, kvh, qo, ko, causal, frame, prefix, slopes, cap, scale)
    out = torch.full_like(q, float("nan"))
    ctx.masked_attention(plan, q, k, v, out)
    torch.cuda.synchronize()
    ctx.check_device()
    for b in range(len(ql)):
        ref, a = attention_ref(q[qo[b]:qo[b + 1]], k[ko[b]:ko[b + 1]], v[ko[b]:ko[b + 1]], causal, frame,
                               prefix[b] if prefix else 0, slopes, cap, scale or 0.125)
        check_attention(out[qo[b]:qo[b + 1]], ref, a)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,m", [(1, 1), (1, 127), (1, 128), (1, 129), (128, 128), (129, 257), (255, 64), (300, 1000), (5, 2049)])
def test_masked_lengths(ctx, dtype, n, m):
    run_masked(ctx, [n], [m], 2, 2, dtype, seed=n + m)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (12, 4), (6, 1), (16, 2), (10, 2), (128, 1), (100, 1)])
def test_masked_shared_heads(ctx, dtype, heads, kvh):
    run_masked(ctx, [70, 3], [70, 150], heads, kvh, dtype, causal=True, bias=True, seed=heads)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("causal,frame,prefix", [(False, 1, None), (True, 1, None), (True, 1, [0, 100, 200, 5, 0, 10 ** 9]),
                                                 (True, 50, [130, 0, 0, 3, 1, 0]), (False, 7, None)])
def test_masked_terms(ctx, dtype, bias, cap, causal, frame, prefix):
    """Documents with more rows than keys (rows that see nothing), no keys, no rows."""
    run_masked(ctx, [300, 200, 0, 40, 1, 260], [300, 90, 50, 0, 500, 390], 4, 2, dtype, causal, frame, prefix, bias,
               cap, seed=frame)


@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_masked_cap_over_its_whole_range(ctx, cap):
    """Scores far past the cap (tanh saturates) and far below it."""
    run_masked(ctx, [200], [333], 2, 2, BF16, cap=cap, gain=40.0, seed=3)
    run_masked(ctx, [200], [333], 2, 2, F16, cap=cap, gain=0.01, seed=4)


@pytest.mark.parametrize("cap,scale", [(0.01, 100.0), (0.01, 0.0), (1000.0, 0.0), (1000.0, 30.0), (50.0, 1e-6)])
def test_masked_cap_and_scale_at_their_limits(ctx, cap, scale):
    """The ends of the ranges taken; scores up to several thousand at cap 1000."""
    for n in (2, 150):
        q, k, v = (randn(gen(40 + i), rows, 1, D, dtype=BF16) for i, rows in enumerate((n, 300, 300)))
        out = torch.empty_like(q)
        ctx.masked_attention(va.AttentionPlan(ctx, 1, 1, [0, n], [0, 300], score_cap=cap, scale=scale), q, k, v, out)
        ref, a = attention_ref(q, k, v, False, 1, 0, None, cap, scale or 0.125)
        # a capped score is off by up to 4e-7 of the cap, an F32 product by 64 * 2^-24 of the score
        check_attention(out, ref, a, p_step=half_step(BF16) + 2 * 4e-7 * cap + 2.0 ** -17 * min(cap, 60 * (scale or 0.125)))


@pytest.mark.parametrize("cap,gain", [(50.0, 1.5), (50.0, 60.0), (30.0, 8.0), (2.0, 1.5), (60.0, 30.0)])
def test_masked_cap_with_many_keys(ctx, cap, gain):
    """Rows that all see many keys (a constant exponent reference up to cap 50), scores from
    ordinary to saturated at both ends of the cap; one document, two, and split keys."""
    run_masked(ctx, [150], [1500], 2, 2, BF16, cap=cap, gain=gain, seed=11)
    run_masked(ctx, [70, 300], [1100, 2000], 4, 2, BF16, cap=cap, gain=gain, seed=12)
    # every key scores -cap: the smallest probabilities the reference allows
    g = gen(13)
    q = torch.ones(3, 1, D, device="cuda", dtype=BF16) * 30
    k = -torch.ones(1300, 1, D, device="cuda", dtype=BF16) * 30
    v = randn(g, 1300, 1, D, dtype=BF16)
    out = torch.empty_like(q)
    ctx.masked_attention(va.AttentionPlan(ctx, 1, 1, [0, 3], [0, 1300], score_cap=cap), q, k, v, out)
    check_attention(out, *attention_ref(q, k, v, False, 1, 0, None, cap))
    ctx.masked_attention(va.AttentionPlan(ctx, 1, 1, [0, 3], [0, 1300], score_cap=cap), q, -k, v, out)
    check_attention(out, *attention_ref(q, -k, v, False, 1, 0, None, cap))


def test_masked_scale_and_growing_scores(ctx):
    run_masked(ctx, [140], [900], 2, 1, BF16, scale=1.0, seed=5)   # near one-hot rows
    run_masked(ctx, [140], [900], 2, 1, F16, scale=0.001, seed=6)  # flat rows
    # scores that rise along the keys: the running maximum moves in every tile
    for dtype in (BF16, F16):
        g = gen(8)
        q = torch.ones(130, 1, D, device="cuda", dtype=dtype)
        k = (torch.arange(1500, device="cuda")[:, None, None] * torch.ones(1, 1, D, device="cuda") / 300).to(dtype)
        v = randn(g, 1500, 1, D, dtype=dtype)
        plan = va.AttentionPlan(ctx, 1, 1, [0, 130], [0, 1500])
        out = torch.empty_like(q)
        ctx.masked_attention(plan, q, k, v, out)
        check_attention(out, *attention_ref(q, k, v, False, 1, 0, None, 0.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (8, 1), (16, 2), (3, 3), (10, 2)])
@pytest.mark.parametrize("causal,frame,prefix,bias,cap", [(True, 1, None, False, 0.0), (True, 5, [3, 0, 900, 0, 1], True, 30.0),
                                                          (False, 1, None, True, 0.0), (False, 64, None, False, 50.0)])
def test_masked_few_rows(ctx, dtype, heads, kvh, causal, frame, prefix, bias, cap):
    """Every tile holds at most 16 rows (single tokens and their shared heads), long and short
    documents, more rows than keys, no keys; strided operands; keys cut over a cluster."""
    per = max(1, 16 * kvh // heads)
    ql = [1, per, 1, min(2, per), per]
    kl = [4097, 1, 1000, 0, 33]
    run_masked(ctx, ql, kl, heads, kvh, dtype, causal, frame, prefix, bias, cap, seed=heads)
    g = gen(21)
    packed = randn(g, 300, heads + 2 * kvh, D, dtype=dtype)
    q, k, v = packed[:, :heads], packed[:, heads:heads + kvh], packed[:, heads + kvh:]
    k[290:] = float("nan")  # past the documents
    v[290:] = float("inf")
    plan = va.AttentionPlan(ctx, heads, kvh, [5, 6, 6 + per], [9, 200, 290], causal=True)
    out = torch.full((heads, 300, D), 7.0, device="cuda", dtype=dtype).transpose(0, 1)
    ctx.masked_attention(plan, q, k, v, out)
    for ql0, ql1, kl0, kl1 in ((5, 6, 9, 200), (6, 6 + per, 200, 290)):
        check_attention(out[ql0:ql1], *attention_ref(q[ql0:ql1], k[kl0:kl1], v[kl0:kl1], True, 1, 0, None, 0.0))
    assert (out[:5] == 7).all() and (out[6 + per:] == 7).all()


def test_masked_split_tiles_match_the_definition(ctx):
    """Few tiles: the keys of one tile are cut over a cluster; some CTAs get no key."""
    for n, m, heads, kvh, causal in ((1, 10392, 12, 12, True), (3, 5000, 8, 2, True), (129, 4000, 2, 2, False),
                                     (300, 3000, 1, 1, True)):
        assert va.attention_plan_shape(heads, kvh, [0, n], [0, m], causal)["splits"] > 1
        run_masked(ctx, [n], [m], heads, kvh, BF16, causal=causal, seed=n)
    ql, kl = [1, 60, 2], [6000, 60, 0]
    assert va.attention_plan_shape(2, 2, np.cumsum([0] + ql), np.cumsum([0] + kl), True)["splits"] > 1
    run_masked(ctx, ql, kl, 2, 2, F16, causal=True, bias=True, seed=9)


def test_masked_ignores_rows_outside_documents(ctx):
    """NaN and infinities in rows of no document, and past a document's last key in its last
    tile, change nothing; rows of no document are left as they were."""
    g = gen(1)
    q, k, v = randn(g, 400, 2, D, dtype=BF16), randn(g, 500, 2, D, dtype=BF16), randn(g, 500, 2, D, dtype=BF16)
    qo, ko = [10, 150, 290], [20, 220, 333]
    plan = va.AttentionPlan(ctx, 2, 2, qo, ko, causal=True)
    clean = torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, clean)
    for x, lo, hi in ((q, 10, 290), (k, 20, 333), (v, 20, 333)):
        x[:lo] = float("nan")
        x[hi:] = float("inf")
    out = torch.full_like(q, 7.0)
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.equal(out[10:290], clean[10:290])
    assert (out[:10] == 7).all() and (out[290:] == 7).all()
    # keys of the other document are hidden too
    k[220:], v[220:] = float("nan"), float("inf")
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.equal(out[10:150], clean[10:150])


def test_masked_hidden_keys_may_be_infinite(ctx):
    """A hidden key row may hold anything (its scores are replaced, not added to)."""
    g = gen(2)
    q, k, v = randn(g, 100, 1, D, dtype=BF16), randn(g, 100, 1, D, dtype=BF16), randn(g, 100, 1, D, dtype=BF16)
    plan = va.AttentionPlan(ctx, 1, 1, [0, 100], [0, 100], causal=True)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, clean)
    k[60:] = torch.finfo(BF16).min
    k[80:] = float("nan")
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.equal(out[:60], clean[:60])


def test_masked_strided_views_streams_and_repeats(ctx):
    """q, k, v as views of one packed projection, a head-major output, another stream; the
    same bits on every run."""
    g = gen(3)
    rows = 700
    packed = randn(g, rows, 12, D, dtype=BF16)
    q, k, v = packed[:, :6], packed[:, 6:9], packed[:, 9:]
    plan = va.AttentionPlan(ctx, 6, 3, [0, 300, 700], [0, 300, 700], causal=True, frame=10, prefix=[4, 40])
    out = torch.empty(6, rows, D, device="cuda", dtype=BF16).transpose(0, 1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    ctx.masked_attention(plan, q, k, v, out, stream=st.cuda_stream)
    st.synchronize()
    for b, (lo, hi) in enumerate(((0, 300), (300, 700))):
        check_attention(out[lo:hi], *attention_ref(q[lo:hi], k[lo:hi], v[lo:hi], True, 10, [4, 40][b], None, 0.0))
    again = torch.empty_like(q)
    ctx.masked_attention(plan, q.contiguous(), k.contiguous(), v.contiguous(), again)
    assert torch.equal(again, out)
    q2 = q.contiguous()
    ctx.masked_attention(plan, q2, k, v, q2)  # out may be q
    assert torch.equal(q2, out)


# ------------------------------------------------------------------------------ cache
def quantise_ref(x, fmt):
    """(values, scale) of x [rows, heads, 64] in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1)
    if fmt == torch.int8:
        scale = (top / 127).float().double().clamp_min(2.0 ** -126)
        return torch.round(x / scale[..., None]), scale
    scale = torch.ones_like(top)
    e = torch.full_like(top, -126)
    for ex in range(-126, 128):
        e = torch.where(top > 448 * 2.0 ** (ex - 1), torch.full_like(e, ex), e) if ex > -126 else e
    scale = torch.exp2(e)
    return (x / scale[..., None]).float().to(torch.float8_e4m3fn).double(), scale


def new_cache(g, docs, heads, cap, fmt):
    codes = [torch.randint(0, 256, (docs, heads, cap, D), generator=g, device="cuda", dtype=torch.uint8).view(fmt)
             for _ in range(2)]
    scales = [torch.full((docs, heads, cap), float("nan"), device="cuda") for _ in range(2)]
    return va.KvCache(*codes, *scales), codes, scales


FORMATS = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_cache_write_and_read(ctx, fmt, dtype):
    g = gen(5)
    docs, heads, cap = 4, 3, 75
    new, lens = [33, 0, 1, 75], [40, 10, 75, 75]
    off = np.cumsum([0] + new)
    rows = int(off[-1])
    k, v = randn(g, rows + 5, heads, D, dtype=dtype), randn(g, rows + 5, heads, D, dtype=dtype)
    k[0] = 0
    k[1] *= 1e-4
    v[2, 0] *= 1000
    v[3, 0, 5] = 0.5
    cache, codes, scales = new_cache(g, docs, heads, cap, fmt)
    before = [c.view(torch.uint8).clone() for c in codes]
    ctx.kv_cache_write(cache, k, v, i32(off), i32(lens))
    for x, c, s, old in ((k, codes[0], scales[0], before[0]), (v, codes[1], scales[1], before[1])):
        val, sc = quantise_ref(x, fmt)
        for b in range(docs):
            lo = lens[b] - new[b]
            got = c[b, :, lo:lens[b]].float().double().transpose(0, 1)
            assert torch.equal(got, val[off[b]:off[b + 1]])
            assert torch.equal(s[b, :, lo:lens[b]].double().T, sc[off[b]:off[b + 1]])
            untouched = torch.ones(cap, dtype=torch.bool, device="cuda")
            untouched[lo:lens[b]] = False
            assert torch.equal(c.view(torch.uint8)[b][:, untouched], old[b][:, untouched])
            assert torch.isnan(s[b][:, untouched]).all()
    # read back a middle range of document 0, all of 3, none of 1, one of 2
    first, count = [10, 0, 74, 0], [30, 0, 1, 75]
    ro = np.cumsum([3] + count)
    ko = torch.full((int(ro[-1]) + 4, heads, D), 5.0, device="cuda", dtype=dtype)
    vo = ko.clone()
    ctx.kv_cache_read(cache, i32(ro), ko, vo, first=i32(first))
    for o, c, s in ((ko, codes[0], scales[0]), (vo, codes[1], scales[1])):
        assert (o[:3] == 5).all() and (o[int(ro[-1]):] == 5).all()
        for b in range(docs):
            sl = slice(first[b], first[b] + count[b])
            want = (c[b, :, sl].float() * s[b, :, sl, None]).to(dtype).transpose(0, 1)
            assert torch.equal(o[ro[b]:ro[b + 1]], want) or torch.allclose(
                o[ro[b]:ro[b + 1]].double(), want.double(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_cache_extreme_values(ctx, fmt):
    """Non-finite heads read as NaN; the largest and the smallest finite values survive;
    quotients on a half step round to even."""
    x = torch.zeros(6, 2, D, device="cuda")
    x[0, 0, 3] = float("nan")
    x[1, 0, 60] = float("-inf")
    x[2] = 3.389e38  # the largest bf16
    x[3] = 1e-40     # below F32's normal range
    x[4, 0, :] = torch.arange(D, device="cuda") * 0.5 + 95.5
    x[4, 0, 0] = 127.0  # scale 1: the others are half steps
    x[5, 1, :] = -x[4, 0, :]
    for dtype in (F32, BF16):
        y = x.to(dtype)
        cache, codes, scales = new_cache(gen(1), 1, 2, 6, fmt)
        ctx.kv_cache_write(cache, y, y, i32([0, 6]), i32([6]))
        val, sc = quantise_ref(torch.where(torch.isfinite(y), y, 0), fmt)
        assert torch.isnan(scales[0][0, 0, :2]).all() and torch.isfinite(scales[0][0, 1]).all()
        assert torch.equal(codes[0][0, :, 2:].float().double().transpose(0, 1), val[2:])
        assert torch.equal(scales[0][0, :, 2:].double().T, sc[2:])
        ko, vo = torch.empty_like(y), torch.empty_like(y)
        ctx.kv_cache_read(cache, i32([0, 6]), ko, vo)
        assert torch.isnan(ko[0, 0]).all() and torch.isnan(ko[1, 0]).all() and (ko[:2, 1] == 0).all()
        assert torch.isfinite(ko[2:].float()).all()
        step = 0.5 / 127 if fmt == torch.int8 else 2.0 ** -4
        assert ((ko[2].double() - y[2].double()).abs() <= (step + half_step(dtype)) * y[2].double().abs()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (12, 4), (16, 1), (5, 1), (128, 2)])
@pytest.mark.parametrize("bias,cap,frame,prefix,causal", [(False, 0.0, 1, False, True), (True, 30.0, 7, True, True),
                                                          (True, 0.0, 1, True, False)])
def test_cache_attention(ctx, fmt, dtype, heads, kvh, bias, cap, frame, prefix, causal):
    g = gen(heads)
    new, lens, cap_rows = [1, 3, 0, 17, 1, 2], [1, 33, 12, 1500, 4097, 2], 4100
    off = np.cumsum([2] + new)
    docs = len(new)
    cache, codes, scales = new_cache(g, docs, kvh, cap_rows, fmt)
    hist = np.cumsum([0] + lens)
    k, v = randn(g, int(hist[-1]), kvh, D, dtype=dtype), randn(g, int(hist[-1]), kvh, D, dtype=dtype)
    ctx.kv_cache_write(cache, k, v, i32(hist), i32(lens))
    q = (randn(g, int(off[-1]) + 3, heads, D) * 1.5).to(dtype)
    out = torch.full_like(q, 7.0)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], device="cuda") if bias else None
    pre = [0, 20, 5, 1490, 9, 100] if prefix else [0] * docs
    ctx.cache_attention(cache, q, out, i32(off), i32(lens), max_tokens=3, causal=causal, frame=frame,
                        prefix=i32(pre) if prefix else None, slopes=slopes, score_cap=cap)
    assert (out[:2] == 7).all() and (out[int(off[-1]):] == 7).all()
    for b in range(docs):
        kd = (codes[0][b, :, :lens[b]].double() * scales[0][b, :, :lens[b], None].double()).transpose(0, 1)
        vd = (codes[1][b, :, :lens[b]].double() * scales[1][b, :, :lens[b], None].double()).transpose(0, 1)
        check_attention(out[off[b]:off[b + 1]], *attention_ref(q[off[b]:off[b + 1]], kd, vd, causal, frame, pre[b], slopes,
                                                             cap), p_step=2.0 ** -15)


@pytest.mark.parametrize("fmt", FORMATS)
def test_cache_attention_more_rows_than_tokens_held(ctx, fmt):
    """Rows that stand before the first key see nothing (zeros), except a prefix."""
    g = gen(4)
    cache, codes, scales = new_cache(g, 2, 1, 64, fmt)
    k = randn(g, 8, 1, D, dtype=BF16)
    ctx.kv_cache_write(cache, k, k, i32([0, 4, 8]), i32([4, 4]))
    q = randn(g, 14, 2, D, dtype=BF16)
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 7, 14]), i32([4, 0]), max_tokens=1, frame=3)
    assert (out[7:] == 0).all() and (out[0] == 0).all()
    kd = (codes[0][0, :, :4].double() * scales[0][0, :, :4, None].double()).transpose(0, 1)
    vd = (codes[1][0, :, :4].double() * scales[1][0, :, :4, None].double()).transpose(0, 1)
    check_attention(out[:7], *attention_ref(q[:7], kd, vd, True, 3, 0, None, 0.0), p_step=2.0 ** -15)


SHARED = [(16, 4, 16), (10, 16, 16), (9, 8, 8), (150, 1, 5)]


def shared_lengths(docs, cap, kind):
    if kind == "equal":
        return [cap - 1] * docs
    if kind == "one":
        return [0] * (docs - 1) + [cap]
    r = np.random.default_rng(docs)
    lens = [0, 1, cap, 63, 64, 65, cap - 1, 257] + [int(2 ** r.uniform(0, 13)) for _ in range(docs - 8)]
    return [lens[i] for i in r.permutation(docs)]


@pytest.mark.parametrize("kind", ["mixed", "equal", "one"])
@pytest.mark.parametrize("docs,kvh,heads", SHARED)
def test_cache_attention_documents_sharing_a_cluster(ctx, docs, kvh, heads, kind):
    """Batches whose documents go two to a cluster: odd counts, empty documents, documents without rows and with more rows
    than max_tokens (more blocks of rows than their neighbour), a bad document among good ones."""
    fmt, dtype, cap = (torch.int8, BF16, 8192) if docs % 4 else (torch.float8_e4m3fn, F16, 8200)
    g = gen(docs + len(kind))
    lens = shared_lengths(docs, cap, kind)
    new = [(1, 2, 0, 1, 1, 19, 1, 3)[b % 8] if kind == "mixed" else 1 for b in range(docs)]
    cache, codes, scales = new_cache(g, docs, kvh, cap, fmt)
    hist = np.cumsum([0] + lens)
    k, v = randn(g, int(hist[-1]), kvh, D, dtype=dtype), randn(g, int(hist[-1]), kvh, D, dtype=dtype)
    ctx.kv_cache_write(cache, k, v, i32(hist), i32(lens))
    off = np.cumsum([1] + new)
    q = (randn(g, int(off[-1]) + 2, heads, D) * 1.5).to(dtype)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], device="cuda")

    def check(out, skip=()):
        assert (out[:1] == 7).all() and (out[int(off[-1]):] == 7).all()
        for b in range(docs):
            rows = slice(int(off[b]), int(off[b + 1]))
            if b in skip:
                assert (out[rows] == 7).all()
                continue
            kd = (codes[0][b, :, :lens[b]].double() * scales[0][b, :, :lens[b], None].double()).transpose(0, 1)
            vd = (codes[1][b, :, :lens[b]].double() * scales[1][b, :, :lens[b], None].double()).transpose(0, 1)
            check_attention(out[rows], *attention_ref(q[rows], kd, vd, True, 5, 0, slopes, 40.0), p_step=2.0 ** -15)

    def attend(out, offsets, held):
        ctx.cache_attention(cache, q, out, offsets, held, max_tokens=2, frame=5, slopes=slopes, score_cap=40.0)

    out = torch.full_like(q, 7.0)
    attend(out, i32(off), i32(lens))
    check(out)
    again = torch.full_like(q, 7.0)
    attend(again, i32(off), i32(lens))
    assert torch.equal(out, again)
    if kind == "mixed":
        bad = new.index(19)
        wrong = list(lens)
        wrong[bad] = cap + 1
        out = torch.full_like(q, 7.0)
        attend(out, i32(off), i32(wrong))
        torch.cuda.synchronize()
        with pytest.raises(va.VestraError) as e:
            ctx.check_device()
        assert e.value.code == va.VA_ERR_DEVICE and "lengths" in str(e.value)
        check(out, skip=(bad,))


def test_cache_attention_sharing_follows_the_lengths_in_a_graph(ctx):
    """A captured call whose lengths move on the device gives the eager call's bits at each of them."""
    docs, kvh, cap = 16, 4, 8192
    g = gen(3)
    cache, codes, scales = new_cache(g, docs, kvh, cap, torch.int8)
    k = randn(g, docs * cap, kvh, D, dtype=BF16)
    ctx.kv_cache_write(cache, k, k, i32([cap * b for b in range(docs + 1)]), i32([cap] * docs))
    q = randn(g, docs, 4 * kvh, D, dtype=BF16)
    offsets, lens, out = i32(list(range(docs + 1))), i32([cap] * docs), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.cache_attention(cache, q, out, offsets, lens, max_tokens=1, stream=torch.cuda.current_stream().cuda_stream)
    for kind in ("mixed", "one", "equal"):
        lens.copy_(i32(shared_lengths(docs, cap, kind)))
        out.fill_(7.0)
        graph.replay()
        eager = torch.empty_like(q)
        ctx.cache_attention(cache, q, eager, offsets, lens, max_tokens=1)
        assert torch.equal(out, eager)
    graph.reset()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("held", [3, 64, 130])
def test_cache_attention_hidden_non_finite_heads(ctx, fmt, held):
    """A token whose value (or key) head is not finite reaches the rows that see it, and no other."""
    g = gen(held)
    cache, codes, scales = new_cache(g, 1, 1, 256, fmt)
    k, v = randn(g, held, 1, D, dtype=BF16), randn(g, held, 1, D, dtype=BF16)
    v[held - 1, 0, 5] = float("nan")
    q = randn(g, 3, 1, D, dtype=BF16)
    for key_too in (False, True):
        if key_too:
            k[held - 1, 0, 7] = float("inf")
        ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
        out = torch.empty_like(q)
        ctx.cache_attention(cache, q, out, i32([0, 3]), i32([held]), max_tokens=3)
        kd = (codes[0][0, :, :held - 1].double() * scales[0][0, :, :held - 1, None].double()).transpose(0, 1)
        vd = (codes[1][0, :, :held - 1].double() * scales[1][0, :, :held - 1, None].double()).transpose(0, 1)
        check_attention(out[:2], *attention_ref(q[:2], kd, vd, True, 1, 0, None, 0.0), p_step=2.0 ** -15)
        assert torch.isnan(out[2]).all()


def test_bad_lengths_are_reported_and_skipped(ctx):
    """Offsets and lengths live on the device; a bad document is skipped by bounds checks in
    the kernels and reported by check_device."""
    g = gen(6)
    cache, codes, scales = new_cache(g, 3, 2, 16, torch.int8)
    old = codes[0].clone()
    k = randn(g, 9, 2, D, dtype=BF16)
    for off, lens in (([0, 3, 6, 9], [3, 17, 3]), ([0, 3, 6, 9], [3, 2, 3]), ([0, 3, 12, 9], [3, 12, 3]),
                      ([-2, 3, 6, 9], [5, 3, 3])):
        codes[0].copy_(old)
        ctx.kv_cache_write(cache, k, k, i32(off), i32(lens))
        torch.cuda.synchronize()
        with pytest.raises(va.VestraError) as e:
            ctx.check_device()
        assert e.value.code == va.VA_ERR_DEVICE and "lengths" in str(e.value)
        ctx.check_device()  # reported once
        bad = 1 if off[0] == 0 else 0
        assert torch.equal(codes[0][bad], old[bad])
    q = randn(g, 9, 2, D, dtype=BF16)
    ctx.kv_cache_write(cache, k, k, i32([0, 3, 6, 9]), i32([3, 3, 3]))
    ctx.check_device()
    for off, lens, b in (([0, 3, 6, 9], [3, 17, 3], 1), ([0, 3, 6, 9], [3, -1, 3], 1), ([0, 3, 6, 10], [3, 3, 4], 2)):
        out = torch.full_like(q, 7.0)
        ctx.cache_attention(cache, q, out, i32(off), i32(lens), max_tokens=3)
        torch.cuda.synchronize()
        with pytest.raises(va.VestraError):
            ctx.check_device()
        assert (out[3 * b:3 * b + 3] == 7).all() and not (out[:3] == 7).any()


# ---------------------------------------------------------------------------- together
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_streaming_window(ctx, fmt):
    """Rotate, attend within the prompt, cache, then single steps over the cache, as a captured
    graph whose lengths move on the device; every step against 64 bits over what the
    cache holds, and the whole against the masked attention of the whole sequence."""
    g = gen(9)
    heads, kvh, frame, prompt, steps = 4, 2, 6, [40, 25], 4
    total = [p + steps for p in prompt]
    rope = va.RopeAxes((16, 24, 24))
    qkv = [randn(g, t, heads + 2 * kvh, D, dtype=BF16) for t in total]
    pos = [torch.stack([torch.arange(t, device="cuda") // frame, torch.arange(t, device="cuda") % 3,
                        torch.arange(t, device="cuda") % 2], 1).int() for t in total]
    cache, codes, scales = new_cache(g, 2, kvh, 64, fmt)
    off = np.cumsum([0] + prompt)
    x = torch.cat([a[:p] for a, p in zip(qkv, prompt)])
    ctx.rope_axes(rope, torch.cat([a[:p] for a, p in zip(pos, prompt)]), x[:, :heads], x[:, :heads],
                  x[:, heads:heads + kvh], x[:, heads:heads + kvh])
    plan = va.AttentionPlan(ctx, heads, kvh, off, off, causal=True, frame=frame, score_cap=30.0)
    out = torch.empty(int(off[-1]), heads, D, device="cuda", dtype=BF16)
    ctx.masked_attention(plan, x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], out)
    ctx.kv_cache_write(cache, x[:, heads:heads + kvh], x[:, heads + kvh:], i32(off), i32(prompt))
    # one step of both documents: rotate in place, append, attend
    y = torch.empty(2, heads + 2 * kvh, D, device="cuda", dtype=BF16)
    p = torch.empty(2, 3, device="cuda", dtype=torch.int32)
    lens, offsets = i32(prompt), i32([0, 1, 2])
    o = torch.empty(2, heads, D, device="cuda", dtype=BF16)

    def step(stream):
        ctx.rope_axes(rope, p, y[:, :heads], y[:, :heads], y[:, heads:heads + kvh], y[:, heads:heads + kvh], stream=stream)
        ctx.kv_cache_write(cache, y[:, heads:heads + kvh], y[:, heads + kvh:], offsets, lens, stream=stream)
        ctx.cache_attention(cache, y[:, :heads], o, offsets, lens, max_tokens=1, frame=frame, score_cap=30.0,
                            stream=stream)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for s in range(steps):
        y.copy_(torch.stack([a[n + s] for a, n in zip(qkv, prompt)]))
        p.copy_(torch.stack([a[n + s] for a, n in zip(pos, prompt)]))
        lens += 1
        graph.replay()
        for b in range(2):
            n = prompt[b] + s + 1
            kd, vd = ((c[b, :, :n].double() * sc[b, :, :n, None].double()).transpose(0, 1)
                      for c, sc in zip(codes, scales))
            check_attention(o[b:b + 1], *attention_ref(y[b:b + 1, :heads], kd, vd, True, frame, 0, None, 30.0),
                            p_step=2.0 ** -15)
            whole = rope_ref(qkv[b][:n, :heads + kvh], pos[b][:n], (16, 24, 24), 100.0, "per_axis", 0)
            ref, a = attention_ref(whole[:, :heads], whole[:, heads:], qkv[b][:n, heads + kvh:], True, frame, 0, None, 30.0)
            # quantised keys move a score by at most |q| |k| 2^-4 / 8 (e4m3), 1/254 of the largest (int8)
            assert (o[b].double() - ref[-1]).abs().max() <= 0.35 * a[-1].max()
    # the cache read back equals what the steps left there
    ro = np.cumsum([0] + total)
    ko = torch.empty(int(ro[-1]), kvh, D, device="cuda", dtype=BF16)
    vo = torch.empty_like(ko)
    ctx.kv_cache_read(cache, i32(ro), ko, vo)
    for b in range(2):
        want = (codes[1][b, :, :total[b]].float() * scales[1][b, :, :total[b], None]).to(BF16).transpose(0, 1)
        assert torch.equal(vo[ro[b]:ro[b + 1]], want)


def test_two_graphs_at_once(ctx):
    """Two captured graphs over one plan and one cache, replayed at once on two streams with
    inputs of their own: no call has scratch memory that another could overwrite."""
    g = gen(31)
    n, m, heads, kvh = 200, 3000, 4, 2
    plans = [va.AttentionPlan(ctx, heads, kvh, [0, n], [0, m], causal=True, score_cap=30.0),
             va.AttentionPlan(ctx, heads, kvh, [0, 1], [0, m], causal=True)]
    assert va.attention_plan_shape(heads, kvh, [0, n], [0, m], True)["splits"] > 1
    cache, codes, scales = new_cache(g, 1, kvh, m, torch.int8)
    k, v = randn(g, m, kvh, D, dtype=BF16), randn(g, m, kvh, D, dtype=BF16)
    ctx.kv_cache_write(cache, k, v, i32([0, m]), i32([m]))
    off, lens = i32([0, 3]), i32([m])
    sides = []
    for i in range(2):
        q = randn(g, n, heads, D, dtype=BF16)
        outs = [torch.empty_like(q), torch.empty_like(q[:1]), torch.empty_like(q[:3])]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            s = torch.cuda.current_stream().cuda_stream
            for _ in range(10):
                ctx.masked_attention(plans[0], q, k, v, outs[0], stream=s)
                ctx.masked_attention(plans[1], q, k, v, outs[1], stream=s)
                ctx.cache_attention(cache, q[:3], outs[2], off, lens, max_tokens=3, stream=s)
        sides.append((q, outs, graph, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, _, graph, st in sides:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    kd, vd = ((c[0].double() * sc[0, :, :, None].double()).transpose(0, 1) for c, sc in zip(codes, scales))
    for q, outs, _, _ in sides:
        check_attention(outs[0], *attention_ref(q, k, v, True, 1, 0, None, 30.0))
        check_attention(outs[1], *attention_ref(q[:1], k, v, True, 1, 0, None, 0.0))
        check_attention(outs[2], *attention_ref(q[:3], kd, vd, True, 1, 0, None, 0.0), p_step=2.0 ** -15)


def test_addresses_past_32_bits(ctx):
    """A cache of more than 2^32 bytes and key rows more than 2^32 bytes apart."""
    g = gen(32)
    cap, n = 23_000_001, 150  # odd: the scales of a head start anywhere
    shape = (2, 2, cap)
    codes = [torch.empty(shape + (D,), device="cuda", dtype=torch.int8) for _ in range(2)]
    scales = [torch.empty(shape, device="cuda") for _ in range(2)]
    cache = va.KvCache(*codes, *scales)
    k, v = randn(g, 2 * n, 2, D, dtype=BF16), randn(g, 2 * n, 2, D, dtype=BF16)
    # document 1's tokens at the far end of the buffer
    ctx.kv_cache_write(cache, k, v, i32([0, n, 2 * n]), i32([n, cap]))
    val, sc = quantise_ref(v[n:], torch.int8)
    assert torch.equal(codes[1][1, :, cap - n:].double().transpose(0, 1), val)
    ko, vo = torch.zeros_like(k[:n]), torch.zeros_like(v[:n])
    ctx.kv_cache_read(cache, i32([0, 0, n]), ko, vo, first=i32([0, cap - n]))
    assert torch.equal(vo, (val * sc[..., None]).float().to(BF16))
    for c in codes:
        c[1, :, :n] = c[1, :, cap - n:]
    for x in scales:
        x[1, :, :n] = x[1, :, cap - n:]
    q = randn(g, 2, 4, D, dtype=BF16)
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 1, 2]), i32([n, n]), max_tokens=1)
    for b in range(2):
        kd, vd = ((c[b, :, :n].double() * x[b, :, :n, None].double()).transpose(0, 1) for c, x in zip(codes, scales))
        check_attention(out[b:b + 1], *attention_ref(q[b:b + 1], kd, vd, True, 1, 0, None, 0.0), p_step=2.0 ** -15)
    del cache, codes, scales, c, x
    rows, step = 1200, 2 ** 21
    big = torch.empty((rows - 1) * step + 2 * D, device="cuda", dtype=BF16)  # 5 GB
    far = big.as_strided((rows, 2, D), (step, D, 1))
    far.copy_(randn(g, rows, 2, D, dtype=BF16))
    for n in (1, 200):
        q = randn(g, n, 2, D, dtype=BF16)
        out = torch.empty_like(q)
        ctx.masked_attention(va.AttentionPlan(ctx, 2, 2, [0, n], [0, rows]), q, far, far, out)
        check_attention(out, *attention_ref(q, far, far, False, 1, 0, None, 0.0))
    pos = torch.randint(0, 100, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
    before = far.clone()
    ctx.rope_axes(va.RopeAxes((16, 24, 24)), pos, far, far)
    assert (far.double() - rope_ref(before, pos, (16, 24, 24), 100.0, "per_axis", 0)).abs().max() <= rope_tol(before, BF16)


def test_many_documents_and_widest_heads(ctx):
    g = gen(33)
    docs = 1500
    new = [int(x) for x in torch.randint(0, 3, (docs,), generator=torch.Generator().manual_seed(1))]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 20, (docs,), generator=torch.Generator().manual_seed(2)))]
    cache, codes, scales = new_cache(g, docs, 2, 24, torch.float8_e4m3fn)
    hist, off = np.cumsum([0] + lens), np.cumsum([0] + new)
    k, v = randn(g, int(hist[-1]), 2, D, dtype=F16), randn(g, int(hist[-1]), 2, D, dtype=F16)
    ctx.kv_cache_write(cache, k, v, i32(hist), i32(lens))
    q = randn(g, int(off[-1]), 4, D, dtype=F16)
    out, dense = torch.empty_like(q), torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32(off), i32(lens), max_tokens=2)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ctx.kv_cache_read(cache, i32(hist), ko, vo)
    ctx.masked_attention(va.AttentionPlan(ctx, 4, 2, off, hist, causal=True), q, ko, vo, dense)
    for b in list(range(0, docs, 97)) + [docs - 1]:
        if new[b]:
            kd, vd = ((c[b, :, :lens[b]].double() * x[b, :, :lens[b], None].double()).transpose(0, 1) for c, x in zip(codes, scales))
            ref, a = attention_ref(q[off[b]:off[b + 1]], kd, vd, True, 1, 0, None, 0.0)
            check_attention(out[off[b]:off[b + 1]], ref, a, p_step=2.0 ** -15)
            # the values read back carry one more f16 rounding
            check_attention(dense[off[b]:off[b + 1]], ref, a, p_step=2.0 ** -9)
    assert (out.float() - dense.float()).abs().max() <= 2.0 ** -7 * v.abs().max()
    run_masked(ctx, [3, 40], [30, 45], 128, 128, BF16, causal=True, bias=True, seed=34)
    run_masked(ctx, [1], [400], 128, 128, F16, causal=True, seed=35)


@pytest.mark.parametrize("frame", [2 ** 31 - 1, 2 ** 24, 127, 128, 129, 200, 3])
def test_masked_frames_at_their_edges(ctx, frame):
    """Frames longer than any document, and around the tile's 128 keys; rows before the first key."""
    run_masked(ctx, [300, 150], [500, 40], 2, 1, BF16, True, frame, [7, 30], True, 0.0, seed=frame % 1000)
    run_masked(ctx, [2, 1], [500, 40], 2, 1, F16, False, frame, None, True, 30.0, seed=frame % 1000)


# ---------------------------------------------------------------------------- refusals
def test_refusals(ctx):
    q = torch.zeros(8, 4, D, device="cuda", dtype=BF16)
    kv = torch.zeros(8, 2, D, device="cuda", dtype=BF16)
    pos = torch.zeros(8, 3, device="cuda", dtype=torch.int32)

    def refused(fn, code=va.VA_ERR_INVALID):
        with pytest.raises(va.VestraError) as e:
            fn()
        assert e.value.code == code

    rope = va.RopeAxes((16, 24, 24))
    for bad in (va.RopeAxes((16, 24, 26)), va.RopeAxes((15, 24)), va.RopeAxes((0, 24)), va.RopeAxes((16,), base=0.0),
                va.RopeAxes((16,), base=float("nan")), va.RopeAxes((16,), pairing=2)):
        refused(lambda bad=bad: ctx.rope_axes(bad, pos[:, :len(bad.c.section[:bad.c.axes])].contiguous(), q, q.clone()))
    refused(lambda: va.RopeAxes((16,), layout="other"))
    refused(lambda: ctx.rope_axes(rope, pos[:7].contiguous(), q, q))
    refused(lambda: ctx.rope_axes(rope, pos.cpu(), q, q))
    refused(lambda: ctx.rope_axes(rope, pos.long(), q, q))
    refused(lambda: ctx.rope_axes(rope, pos, q, q.float()))
    refused(lambda: ctx.rope_axes(rope, pos, q, q.view(-1).as_strided((8, 4, D), (D, 8 * D, 1))))  # on its input, other strides
    refused(lambda: ctx.rope_axes(rope, pos, q, q.clone()[:, :1].expand(8, 4, D)))  # heads on top of each other
    refused(lambda: ctx.rope_axes(rope, pos, q, q.clone(), kv))
    for kw in (dict(heads=4, kv_heads=3), dict(heads=0), dict(heads=129, kv_heads=1), dict(frame=0),
               dict(score_cap=-1.0), dict(score_cap=float("inf")), dict(scale=float("nan")), dict(score_cap=2000.0),
               dict(score_cap=1e-3), dict(scale=-0.1), dict(scale=1e3), dict(score_cap=float("nan")),
               dict(q_offsets=[0, 9, 8]), dict(q_offsets=[-1, 8]), dict(k_offsets=[0, 2 ** 24 + 1]),
               dict(k_offsets=[0, 2 ** 31 + 9]), dict(prefix=[-1]), dict(slopes=np.array([1, 2, np.nan, 0])),
               dict(slopes=np.ones(3)), dict(q_offsets=[0])):
        args = dict(heads=4, kv_heads=2, q_offsets=[0, 8], k_offsets=[0, 8])
        args.update(kw)
        if len(args["q_offsets"]) == 3:
            args["k_offsets"] = [0, 4, 8]
        refused(lambda args=args: va.AttentionPlan(ctx, **args))
    plan = va.AttentionPlan(ctx, 4, 2, [0, 8], [0, 8])
    out = torch.empty_like(q)
    refused(lambda: ctx.masked_attention(plan, q[:7], kv, kv, out))
    refused(lambda: ctx.masked_attention(plan, q, kv[:7], kv, out))
    refused(lambda: ctx.masked_attention(plan, q, q, kv, out))
    refused(lambda: ctx.masked_attention(plan, q, kv.half(), kv, out))
    refused(lambda: ctx.masked_attention(plan, q.float(), kv.float(), kv.float(), out.float()))
    refused(lambda: ctx.masked_attention(plan, q, kv, kv, out.cpu()))
    odd = torch.zeros(8 * 4 * D + 1, device="cuda", dtype=BF16)[1:].view(8, 4, D)
    refused(lambda: ctx.masked_attention(plan, odd, kv, kv, out))
    refused(lambda: ctx.masked_attention(plan, torch.zeros(8, 4, D + 1, device="cuda", dtype=BF16)[..., :D], kv, kv, out))
    plan.close()
    refused(lambda: ctx.masked_attention(plan, q, kv, kv, out), va.VA_ERR_STATE)
    cache, codes, scales = new_cache(gen(0), 1, 2, 16, torch.int8)
    refused(lambda: va.KvCache(codes[0], codes[1], scales[0], scales[1][..., :8]))
    refused(lambda: va.KvCache(codes[0].view(torch.uint8), codes[1], scales[0], scales[1]))
    refused(lambda: ctx.kv_cache_write(cache, kv, kv, i32([0]), i32([8])))
    refused(lambda: ctx.kv_cache_write(cache, kv, kv, i32([0, 8]), None))
    refused(lambda: ctx.kv_cache_write(cache, q, q, i32([0, 8]), i32([8])))
    refused(lambda: ctx.kv_cache_write(cache, kv, kv.half(), i32([0, 8]), i32([8])))
    refused(lambda: ctx.kv_cache_read(cache, i32([0, 8]).long(), kv, kv))
    refused(lambda: ctx.cache_attention(cache, q, out, i32([0, 8]), i32([8]), max_tokens=0))
    refused(lambda: ctx.cache_attention(cache, q[:, :3], out[:, :3], i32([0, 8]), i32([8]), max_tokens=8))
    refused(lambda: ctx.cache_attention(cache, q, out, i32([0, 8]), i32([8]), max_tokens=8, frame=0))
    refused(lambda: ctx.cache_attention(cache, q.float(), out.float(), i32([0, 8]), i32([8]), max_tokens=8))
    refused(lambda: ctx.cache_attention(cache, q, out, i32([0, 8]), i32([8]), max_tokens=8, slopes=torch.ones(3, device="cuda")))


def test_empty_calls(ctx):
    e = torch.zeros(0, 2, D, device="cuda", dtype=BF16)
    ctx.rope_axes(va.RopeAxes((64,)), torch.zeros(0, 1, device="cuda", dtype=torch.int32), e, e)
    ctx.masked_attention(va.AttentionPlan(ctx, 2, 2, [0, 0], [0, 5]), e, torch.zeros(5, 2, D, device="cuda", dtype=BF16),
                         torch.zeros(5, 2, D, device="cuda", dtype=BF16), e)
    q = torch.ones(3, 2, D, device="cuda", dtype=BF16)
    out = torch.full_like(q, 7.0)
    ctx.masked_attention(va.AttentionPlan(ctx, 2, 2, [0, 3], [0, 0]), q, e, e, out)  # rows without a key
    assert (out == 0).all()
    cache, _, _ = new_cache(gen(0), 1, 2, 16, torch.int8)
    ctx.kv_cache_write(cache, e, e, i32([0, 0]), i32([0]))
    ctx.kv_cache_read(cache, i32([0, 0]), e, e)
    ctx.cache_attention(cache, e, e, i32([0, 0]), i32([0]), max_tokens=1)
