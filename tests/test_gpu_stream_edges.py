"""Streaming-attention operators on the GPU, where one row, document or launch must not
reach another: rows past a tile, neighbouring documents, heads of very different size.

Tolerances count roundings, as in test_gpu_stream: u = eps / 2 of the type."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

import vestra_attn as va  # noqa: E402
from test_gpu_stream import (  # noqa: E402, F401  (ctx and the two autouse fixtures)
    _float32_by_default, _no_device_error, attention_ref, check_attention, ctx, gen, half_step, i32, new_cache, randn)

D = 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def slopes_of(heads):
    return np.array([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], np.float32)


# --------------------------------------------------------- capped scores: rows of the tile only
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("keys", [300, 1500])  # from 1024 keys on bf16 takes the constant reference
@pytest.mark.parametrize("huge", [1e4, float("inf")])
def test_capped_document_does_not_depend_on_its_neighbours_queries(ctx, dtype, bias, keys, huge):
    g = gen(keys)
    ql, heads = [100, 100, 37], 2
    qo, ko = np.cumsum([0] + ql), np.cumsum([0] + [keys] * 3)
    q, k, v = (randn(g, n, heads, D, dtype=dtype) for n in (int(qo[-1]) + 5, int(ko[-1]), int(ko[-1])))
    plan = va.AttentionPlan(ctx, heads, heads, qo, ko, slopes=slopes_of(heads) if bias else None, score_cap=50.0)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, clean)
    q[100:200] *= huge
    q[237:] = huge  # rows of no document, behind the last tile
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.equal(out[:100], clean[:100])
    assert torch.equal(out[200:237], clean[200:237])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh", [(12, 4), (6, 1), (10, 2)])
@pytest.mark.parametrize("keys", [200, 1300])
def test_capped_bits_do_not_depend_on_earlier_launches(ctx, dtype, heads, kvh, keys):
    """Heads that do not divide a tile of 128 rows: its last rows are never written."""
    g = gen(heads)
    rows = 1200
    q, k, v = (randn(g, n, h, D, dtype=dtype) for n, h in ((rows, heads), (keys, kvh), (keys, kvh)))
    plan = va.AttentionPlan(ctx, heads, kvh, [0, rows], [0, keys], score_cap=30.0)
    other = va.AttentionPlan(ctx, 2, 2, [0, 40000], [0, 128])
    first, out = torch.empty_like(q), torch.empty_like(q)
    for i, left in enumerate((0.0, 1.0, 1e4, float("inf"))):  # what other tiles leave in shared memory
        x = torch.full((40000, 2, D), left, device="cuda", dtype=dtype)
        y = torch.zeros(128, 2, D, device="cuda", dtype=dtype)
        ctx.masked_attention(other, x, y, y, torch.empty_like(x))
        ctx.masked_attention(plan, q, k, v, out if i else first)
        if i:
            assert torch.equal(out, first)


@pytest.mark.parametrize("heads,kvh", [(2, 2), (12, 4), (6, 1)])
@pytest.mark.parametrize("keys", [200, 1300])
def test_capped_output_over_its_queries(ctx, heads, kvh, keys):
    """out may be q: tiles that end inside their 128 rows lie before rows that another CTA writes."""
    g = gen(7)
    docs = 60
    ql = [1 + (37 * b) % 120 for b in range(docs)]
    qo, ko = np.cumsum([0] + ql), [0] + [keys] * docs
    ko = np.cumsum(ko)
    q = randn(g, int(qo[-1]), heads, D, dtype=BF16) * 4
    k, v = (randn(g, int(ko[-1]), kvh, D, dtype=BF16) for _ in range(2))
    v = v * 40  # outputs unlike the queries they replace
    plan = va.AttentionPlan(ctx, heads, kvh, qo, ko, score_cap=20.0)
    want = torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, want)
    for _ in range(20):
        x = q.clone()
        ctx.masked_attention(plan, x, k, v, x)
        assert torch.equal(x, want)


# ------------------------------------------------------------------------------- plans
def test_plans_used_at_once_on_a_stream_of_their_own(ctx):
    """A plan's first launch goes to a stream that does not wait for the legacy stream, right after create."""
    g = gen(11)
    st = torch.cuda.Stream()
    q, k, v = (randn(g, 900, 2, D, dtype=BF16) for _ in range(3))
    want, out = torch.empty_like(q), torch.empty_like(q)
    ends = [[0, 900], [0, 3, 500, 900], [0, 1], [0, 130, 131]]
    for i in range(60):
        e = ends[i % len(ends)]
        slopes = slopes_of(2) * (1 + i % 3)
        torch.cuda.synchronize()
        plan = va.AttentionPlan(ctx, 2, 2, e, e, causal=True, slopes=slopes)
        ctx.masked_attention(plan, q, k, v, out, stream=st.cuda_stream)
        torch.cuda.synchronize()
        ctx.masked_attention(plan, q, k, v, want)
        assert torch.equal(out[:e[-1]], want[:e[-1]])


# ------------------------------------------------------------------ values of unlike size
def close(got, ref, a, keys, p_step=2.0 ** -15):
    """As check_attention, with another absolute part: outputs here may be as small as 1e-30.  The row's weights
    p * scale are brought to a largest of 2^7 or more and held in two f16 parts, so each is off by at most 2^-25,
    2^-32 of the largest weight.  A code is at most twice its head's largest one, and the largest weight times that
    head's largest value is at most the largest A of the row."""
    tol = half_step(got.dtype) * ref.abs() + (p_step + 2.0 ** -12) * a + keys * 2.0 ** -31 * a.amax(-1, keepdim=True)
    assert ((got.double() - ref).abs() <= tol).all(), f"{((got.double() - ref).abs() / tol).max().item():.3g} of the tolerance"


def held_values(codes, scales, n):
    return [(c[0, :, :n].double() * s[0, :, :n, None].double()).transpose(0, 1) for c, s in zip(codes, scales)]


FORMATS = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("power", [20, 30, 45, -45])
@pytest.mark.parametrize("held", [2, 64, 65, 130])
def test_hidden_token_with_values_of_another_size(ctx, fmt, held, power):
    """The last token's values are 2^power times the others'; the earlier rows do not see it."""
    g = gen(held)
    cache, codes, scales = new_cache(g, 1, 1, 256, fmt)
    k, v = randn(g, held, 1, D), randn(g, held, 1, D)
    v[held - 1] *= 2.0 ** power
    ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
    q = randn(g, 2, 1, D, dtype=BF16)
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 2]), i32([held]), max_tokens=2)
    close(out, *attention_ref(q, *held_values(codes, scales, held), True, 1, 0, None, 0.0), held)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("at", [0, 100, 299])
@pytest.mark.parametrize("score,power", [(-40.0, 30), (-80.0, 60), (-300.0, 100), (40.0, -60), (-8.0, 45)])
def test_token_that_hardly_counts_with_values_of_another_size(ctx, fmt, at, score, power):
    """Every row sees the token, but its probability makes it count little (or, at -8, all)."""
    g = gen(at + 1)
    held = 300
    cache, codes, scales = new_cache(g, 1, 1, 512, fmt)
    q = torch.full((1, 2, D), 1.0, device="cuda", dtype=BF16)
    k, v = randn(g, held, 1, D) * 0.05, randn(g, held, 1, D)
    k[at] = score / 8  # q . k / sqrt(64) = score
    v[at] *= 2.0 ** power
    ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 1]), i32([held]), max_tokens=1)
    close(out, *attention_ref(q, *held_values(codes, scales, held), True, 1, 0, None, 0.0), held)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-28, 1e-4, 1e6, 1e30])
def test_values_of_one_size(ctx, fmt, size):
    """All values tiny or huge; scores that grow from chunk to chunk, so the sums are rescaled often."""
    g = gen(5)
    held = 1000
    cache, codes, scales = new_cache(g, 1, 2, 1024, fmt)
    k, v = randn(g, held, 2, D) * 0.1, randn(g, held, 2, D) * size
    k += torch.linspace(-2, 2, held, device="cuda")[:, None, None]
    v *= torch.exp2(torch.linspace(10, -10, held, device="cuda"))[:, None, None]
    ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
    q = torch.full((4, 4, D), 0.5, device="cuda", dtype=BF16)
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 4]), i32([held]), max_tokens=4)
    close(out, *attention_ref(q, *held_values(codes, scales, held), True, 1, 0, None, 0.0), held)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("held", [2, 64, 65, 130, 600])
def test_hidden_tokens_do_not_change_a_bit(ctx, fmt, held):
    """Rows that do not see the last two tokens, whatever those hold."""
    g = gen(held)
    cache, codes, scales = new_cache(g, 1, 2, 640, fmt)
    k, v = randn(g, held, 2, D), randn(g, held, 2, D) * torch.exp2(torch.randint(0, 6, (held, 1, 1), generator=g, device="cuda"))
    q = randn(g, 3, 4, D, dtype=BF16)
    outs = []
    for power in (0, 5, 45, 100, -100):
        x = v.clone()
        x[max(0, held - 2):] *= 2.0 ** power
        ctx.kv_cache_write(cache, k, x, i32([0, held]), i32([held]))
        outs.append(torch.empty_like(q))
        ctx.cache_attention(cache, q, outs[-1], i32([0, 3]), i32([held]), max_tokens=3)
    for out in outs[1:]:
        assert torch.equal(out[0], outs[0][0])


# ------------------------------------------------------------------ few rows over long documents
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("depth", [8.0, 14.0, 17.5, 20.0])
@pytest.mark.parametrize("docs", [1, 40])  # 40: a key head's keys stay with one CTA
def test_single_row_with_a_long_flat_tail(ctx, dtype, depth, docs):
    """One key `depth` nats above many equal ones whose values share a sign: every one of them is small, their
    sum is not.  The values of the equal keys are 1, the other key's 0, so the result is the tail's share.

    Tolerance: the output's rounding; two parts of a probability (2^-16 of it in bf16, 2^-22 or 2^-40 of the largest
    in f16); F32 sums in order: a lane adds n / lanes probabilities, each addition off by at most 2^-24 of the lane's
    sum, which for the lane with the largest key is at most its share of the tail, 1 / lanes; the products' sums
    likewise (16 keys an addition, truncated: 2^-23)."""
    n = 1 << 20 if docs == 1 else 1 << 18
    heads = 1 if docs == 1 else 12
    ends = [64 * i for i in range(docs)] + [64 * docs + n]  # the last document is long, the others short
    rows = list(range(docs + 1))
    splits = va.attention_plan_shape(heads, heads, rows, ends)["splits"]
    assert splits == (16 if docs == 1 else 1)
    long = ends[-2]
    n = ends[-1] - long
    k = torch.zeros(ends[-1], heads, D, device="cuda", dtype=dtype)
    v = torch.ones_like(k)
    k[long, :, 0] = depth
    v[long] = 0
    q = torch.zeros(docs, heads, D, device="cuda", dtype=dtype)
    q[..., 0] = 8.0
    out = torch.empty_like(q)
    ctx.masked_attention(va.AttentionPlan(ctx, heads, heads, rows, ends), q, k, v, out)
    score = float(k[long, 0, 0])  # as rounded to the type
    tail = (n - 1) * np.exp(-score)
    ref, lanes = tail / (1 + tail), 16 * splits
    parts = 2.0 ** -16 * ref if dtype == BF16 else 2.0 ** -22 * ref + n * 2.0 ** -40
    sums = ref * (tail / (1 + tail) / lanes + n / lanes * 2.0 ** -24 + n / (lanes / 4) / 16 * 2.0 ** -23)
    assert (out[-1].double() - ref).abs().max() <= half_step(dtype) * ref + parts + sums


# ------------------------------------------------------------------ constant exponent reference
@pytest.mark.parametrize("keys", [1100, 5000])
@pytest.mark.parametrize("power", [0, -20, -28, -30, 60, 78])
@pytest.mark.parametrize("sign", [1, -1])
def test_saturated_scores_with_small_and_large_values(ctx, keys, power, sign):
    """Every score at one end of the cap: the probabilities are the largest or the smallest the reference allows."""
    g = gen(keys)
    q = torch.full((20, 1, D), 30.0, device="cuda", dtype=BF16)
    k = torch.full((keys, 1, D), 30.0 * sign, device="cuda", dtype=BF16)
    v = (randn(g, keys, 1, D).double() * 2.0 ** power / 4).to(BF16)
    out = torch.empty_like(q)
    ctx.masked_attention(va.AttentionPlan(ctx, 1, 1, [0, 20], [0, keys], score_cap=50.0), q, k, v, out)
    ref, a = attention_ref(q, k, v, False, 1, 0, None, 50.0)
    u = half_step(BF16)
    # equal probabilities: one rounding of each, and the output's
    assert ((out.double() - ref).abs() <= u * ref.abs() + (u + 2.0 ** -12) * a).all()


# ------------------------------------------------------------------ slopes
@pytest.mark.parametrize("slope", [2.0 ** 96, -2.0 ** 96, 1e6])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("n,m", [(2, 40), (150, 300), (300, 150)])
def test_steep_slopes(ctx, slope, cap, n, m):
    """A bias that leaves every row one frame: the nearest, or with a negative slope the farthest.  Score and bias
    are one F32 sum, so a score beside a bias of 1e6 and more is lost (half an ulp of 1e6 is 2^-5); rows whose own
    frame holds keys have distance 0 there, and their scores count."""
    g = gen(n)
    q, k, v = (randn(g, r, 1, D, dtype=BF16) for r in (n, m, m))
    slopes = np.array([slope], np.float32)
    plan = va.AttentionPlan(ctx, 1, 1, [0, n], [0, m], causal=True, frame=5, prefix=[3], slopes=slopes, score_cap=cap)
    out = torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.isfinite(out.float()).all()
    if slope > 0:
        ref, a = attention_ref(q, k, v, True, 5, 3, np.array([1e6]), cap)
        rows = torch.arange(n, device="cuda") + m - n >= 0
        check_attention(out[rows], ref[rows], a[rows])


# ------------------------------------------------------------------ strides that are never stepped over
@pytest.mark.parametrize("token_stride", [64, 1, 0, 2 ** 40])
def test_one_row_of_any_token_stride(ctx, token_stride):
    """A view of one row keeps whatever stride its rows had."""
    g = gen(3)
    heads = 4
    wide = randn(g, heads, 7, D, dtype=BF16)  # head-major
    row = wide[:, 5:6].transpose(0, 1)
    x = row.as_strided((1, heads, D), (token_stride, 7 * D, 1), row.storage_offset())
    clean = row.contiguous()
    kv = randn(g, 300, heads, D, dtype=BF16)
    out, want = torch.empty_like(clean), torch.empty_like(clean)
    for n in (1, 300):  # one key row, too
        plan = va.AttentionPlan(ctx, heads, heads, [0, 1], [0, n])
        ctx.masked_attention(plan, x, x if n == 1 else kv, x if n == 1 else kv, out)
        ctx.masked_attention(plan, clean, clean if n == 1 else kv, clean if n == 1 else kv, want)
        assert torch.equal(out, want)
    one_key = va.AttentionPlan(ctx, heads, heads, [0, 300], [0, 1])  # the tensor maps' form
    o2, w2 = torch.empty_like(kv), torch.empty_like(kv)
    ctx.masked_attention(one_key, kv, x, x, o2)
    ctx.masked_attention(one_key, kv, clean, clean, w2)
    assert torch.equal(o2, w2) and torch.equal(o2, clean.expand_as(o2))
    pos = i32([[7]])
    ctx.rope_axes(va.RopeAxes((64,)), pos, x, out)
    ctx.rope_axes(va.RopeAxes((64,)), pos, clean, want)
    assert torch.equal(out, want)
    results = []
    for y in (x, clean):
        cache, codes, scales = new_cache(gen(1), 1, heads, 8, torch.int8)
        ctx.kv_cache_write(cache, y, y, i32([0, 1]), i32([1]))
        o = torch.empty_like(clean)
        ctx.cache_attention(cache, y, o, i32([0, 1]), i32([1]), max_tokens=1)
        results.append((codes[0][:, :, 0].clone(), o))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


# ------------------------------------------------------------------ many documents
def test_max_tokens_of_the_whole_batch_over_many_documents(ctx):
    """max_tokens is an estimate: taken as all rows of the batch it may not size a launch past the grid's limit."""
    docs, heads = 70000, 8
    g = gen(17)
    cache, codes, scales = new_cache(g, docs, 1, 2, torch.int8)
    k, v = randn(g, docs, 1, D, dtype=BF16), randn(g, docs, 1, D, dtype=BF16)
    ends = torch.arange(docs + 1, device="cuda", dtype=torch.int32)
    ctx.kv_cache_write(cache, k, v, ends, torch.ones(docs, device="cuda", dtype=torch.int32))
    q = randn(g, docs, heads, D, dtype=BF16)
    out, want = torch.empty_like(q), torch.empty_like(q)
    lens = torch.ones(docs, device="cuda", dtype=torch.int32)
    ctx.cache_attention(cache, q, out, ends, lens, max_tokens=docs)
    ctx.cache_attention(cache, q, want, ends, lens, max_tokens=1)
    assert torch.equal(out, want)
    # one token held: its value, from the codes
    value = codes[1][:, 0, 0].double() * scales[1][:, 0, :1].double()
    assert ((out.double() - value[:, None]).abs() <= (half_step(BF16) + 2.0 ** -18) * value[:, None].abs()).all()


# ------------------------------------------------------------------ what the tolerances tell apart
def weight_steps(w, dropped):
    """w [keys] as the kernel holds weights: two f16 parts of w * 2^k, the largest in [2^13, 2^14), or one (dropped)."""
    k = 14 - torch.floor(torch.log2(w.max())) - 1
    x = (w * torch.exp2(k)).float().double()
    hi = x.half().double()
    return (hi if dropped else hi + (x - hi).half().double()) * torch.exp2(-k)


@pytest.mark.parametrize("held", [1, 2, 40, 64, 200])
def test_both_parts_of_a_weight_count(ctx, held):
    """Queries of zeros: every probability is 1 exactly, so a weight is its int8 value scale and the result is off by
    half a step of f16 at its size, a weight's 2^-22 (two parts; 2^-38 of the largest at least), and F32 products and sums:
    held + 4 roundings of 2^-24.  A weight of one part, 2^-11, is told apart."""
    g = gen(held)
    heads = 16
    cache, codes, scales = new_cache(g, 1, heads, 256, torch.int8)
    v = (randn(g, held, heads, D).abs() * 30 + 20).clamp(max=120)
    v[..., 0] = 127 * (1 + 0.98 * 2.0 ** -11)  # every scale: 0.98 half steps of f16 past 1, and none cancels another
    ctx.kv_cache_write(cache, torch.zeros_like(v), v, i32([0, held]), i32([held]))
    q = torch.zeros(1, heads, D, device="cuda", dtype=F16)
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 1]), i32([held]), max_tokens=1)
    c, s = codes[1][0, :, :held].double(), scales[1][0, :, :held].double()
    ref = (c * s[..., None]).sum(1) / held
    tol = torch.exp2(torch.floor(torch.log2(ref.abs())) - 11) + (2.0 ** -22 + (held + 4) * 2.0 ** -24) * ref.abs()
    assert ((out[0].double() - ref).abs() <= tol).all()
    one = torch.stack([(c[h] * weight_steps(s[h], True)[:, None]).sum(0) / held for h in range(heads)])
    assert ((one.half().double() - ref).abs() > tol).any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["one channel", "wide"])
def test_scores_of_a_few_units_to_f32(ctx, fmt, kind):
    """Keys of one channel, so that a score is one product: probabilities are as good as F32's.  A score s is off by
    4 roundings of 2^-24 of s, the exponential by 2^-22 (and its argument by 2^-24 of s log2(e)), a weight by 2^-22,
    F32 sums by keys * 2^-24: with s up to 8 below 2^-18 a key, 2^-16 for numerator and denominator of 300 keys.
    wide: the channel that scores holds 2^-12 of the row's largest element, still exact."""
    g = gen(9)
    held, heads = 300, 16
    cache, codes, scales = new_cache(g, 1, heads, 512, fmt)
    s = torch.rand(held, heads, generator=g, device="cuda") * 8
    k = torch.zeros(held, heads, D, device="cuda")
    v = randn(g, held, heads, D).abs() + 0.5
    q = torch.zeros(1, heads, D, device="cuda", dtype=F16)
    at = 2.0 ** -12 * 1.1875 if kind == "wide" else 1.1875
    q[..., 7] = at
    if kind == "wide":
        q[..., 50] = 1.0
    k[..., 7] = s * 8 / at
    ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
    out = torch.empty_like(q)
    ctx.cache_attention(cache, q, out, i32([0, 1]), i32([held]), max_tokens=1)
    kd, vd = held_values(codes, scales, held)
    ref, a = attention_ref(q, kd, vd, True, 1, 0, None, 0.0)
    tol = torch.exp2(torch.floor(torch.log2(ref.abs())) - 11) + 2.0 ** -16 * a
    assert ((out.double() - ref).abs() <= tol).all()


# ------------------------------------------------------------------ rows that are not finite, operands head by head
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("n,m,splits", [(2, 5000, 16), (200, 5000, 2), (40000, 300, 1)])
def test_a_query_that_is_not_finite_reaches_its_own_row_only(ctx, dtype, cap, n, m, splits):
    """Its row is NaN in every form of the launch (few rows, keys cut over a cluster, one CTA a tile)."""
    g = gen(n)
    q, k, v = (randn(g, r, 1, D, dtype=dtype) for r in (n, m, m))
    shape = va.attention_plan_shape(1, 1, [0, n], [0, m])
    assert (shape["splits"] == 1) == (splits == 1)
    plan = va.AttentionPlan(ctx, 1, 1, [0, n], [0, m], score_cap=cap)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ctx.masked_attention(plan, q, k, v, clean)
    q[1] = float("nan")
    ctx.masked_attention(plan, q, k, v, out)
    assert torch.isnan(out[1]).all()
    others = torch.arange(n, device="cuda") != 1
    if cap == 0:
        assert torch.equal(out[others], clean[others])
    assert torch.isfinite(out[others].float()).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_cached_query_that_is_not_finite_reaches_its_own_row_only(ctx, fmt):
    g = gen(2)
    for held in (3, 3000):
        cache, codes, scales = new_cache(g, 1, 2, 3000, fmt)
        k, v = randn(g, held, 2, D), randn(g, held, 2, D)
        ctx.kv_cache_write(cache, k, v, i32([0, held]), i32([held]))
        q = randn(g, 3, 4, D, dtype=BF16)
        clean, out = torch.empty_like(q), torch.empty_like(q)
        ctx.cache_attention(cache, q, clean, i32([0, 3]), i32([held]), max_tokens=3)
        q[1, 2] = float("nan")
        ctx.cache_attention(cache, q, out, i32([0, 3]), i32([held]), max_tokens=3)
        assert torch.isnan(out[1, 2]).all()
        out[1, 2] = clean[1, 2]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("n,m,heads,kvh", [(1, 3000, 4, 2), (300, 700, 6, 2), (3, 40, 3, 3)])
def test_head_major_operands(ctx, n, m, heads, kvh):
    g = gen(m)
    q, k, v = (randn(g, h, r, D, dtype=BF16) for h, r in ((heads, n), (kvh, m), (kvh, m)))
    plan = va.AttentionPlan(ctx, heads, kvh, [0, n], [0, m], causal=True)
    want = torch.empty(n, heads, D, device="cuda", dtype=BF16)
    ctx.masked_attention(plan, *(x.transpose(0, 1).contiguous() for x in (q, k, v)), want)
    out = torch.empty(heads, n, D, device="cuda", dtype=BF16)
    ctx.masked_attention(plan, *(x.transpose(0, 1) for x in (q, k, v)), out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), want)
    results = []
    for a, b, c in ((k, v, q), tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v, q))):
        cache, codes, scales = new_cache(gen(1), 1, kvh, m, torch.int8)
        ctx.kv_cache_write(cache, a.transpose(0, 1), b.transpose(0, 1), i32([0, m]), i32([m]))
        o = torch.empty_like(c)
        ctx.cache_attention(cache, c.transpose(0, 1), o.transpose(0, 1), i32([0, n]), i32([m]), max_tokens=n)
        back = torch.empty_like(k)
        ctx.kv_cache_read(cache, i32([0, m]), back.transpose(0, 1), torch.empty_like(v).transpose(0, 1))
        results.append((o.clone(), back, codes[1].clone()))
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_first_calls_of_a_process_may_be_captured():
    """No call needs one before it: everything that a launch sets up can be set up during a capture."""
    import os
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch, vestra_attn as va
from test_gpu_stream import gen, i32, new_cache, randn
ctx, g, bf = va.Context(va.default_config(max_rows=64), 0), gen(0), torch.bfloat16
docs, cap = 16, 8192
cache, codes, scales = new_cache(g, docs, 4, cap, torch.int8)
q, k, v = randn(g, 64, 4, 64, dtype=bf), randn(g, 64, 4, 64, dtype=bf), randn(g, 64, 4, 64, dtype=bf)
plans = [va.AttentionPlan(ctx, 4, 4, [0, n], [0, 64]) for n in (64, 1)]
ends, lens, pos = i32([4 * b for b in range(docs + 1)]), i32([4] * docs), i32([[i] for i in range(64)])
outs = [torch.zeros_like(q) for _ in range(6)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def calls(outs, s):
    ctx.rope_axes(va.RopeAxes((64,)), pos, q, outs[0], stream=s)
    ctx.kv_cache_write(cache, k, v, ends, lens, stream=s)
    ctx.masked_attention(plans[0], q, k, v, outs[1], stream=s)
    ctx.masked_attention(plans[1], q, k, v, outs[2], stream=s)
    ctx.cache_attention(cache, q, outs[3], ends, lens, max_tokens=4, stream=s)
    ctx.kv_cache_read(cache, ends, outs[4], outs[5], stream=s)
with torch.cuda.graph(graph):
    calls(outs, torch.cuda.current_stream().cuda_stream)
graph.replay()
torch.cuda.synchronize()
again = [torch.zeros_like(q) for _ in range(6)]
calls(again, 0)
torch.cuda.synchronize()
ctx.check_device()
assert all(torch.equal(a, b) and b.any() for a, b in zip(outs, again))
graph.reset()
""" % (os.path.dirname(os.path.abspath(__file__)), os.path.dirname(va.__file__))
    assert subprocess.run([sys.executable, "-c", code], timeout=300).returncode == 0


# ------------------------------------------------------------------ rotary operands off every vector boundary
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("offset,pad,gap", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (3, 2, 5), (2, 0, 4), (4, 4, 0), (8, 8, 8)])
@pytest.mark.parametrize("sections,layout", [((2,), "per_axis"), ((20, 22, 22), "per_axis"), ((20, 22, 20), "shared"),
                                             ((16, 24, 24), "per_axis"), ((64,), "shared")])
def test_rope_at_any_offset_and_stride(ctx, dtype, pairing, offset, pad, gap, sections, layout):
    from test_gpu_stream import rope_ref, rope_tol
    g = gen(offset + 10 * pad)
    rows, heads, d = 9, 3, sum(sections) + 2
    flat = randn(g, offset + rows * (heads * (d + pad) + gap), dtype=dtype)
    x = flat.as_strided((rows, heads, d), (heads * (d + pad) + gap, d + pad, 1), offset)
    pos = torch.randint(-100, 100, (rows, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    rope = va.RopeAxes(sections, 100.0, layout, pairing)
    ref = rope_ref(x, pos, sections, 100.0, layout, pairing)
    out = torch.full_like(flat, 7.0).as_strided(x.shape, x.stride(), offset)
    ctx.rope_axes(rope, pos, x, out)
    assert (out.double() - ref).abs().max() <= rope_tol(x, dtype)
    outside = torch.ones_like(flat, dtype=torch.bool)
    outside.as_strided(x.shape, x.stride(), offset).fill_(False)
    keep = flat.clone()
    ctx.rope_axes(rope, pos, x, x)
    assert torch.equal(x, out) and torch.equal(flat[outside], keep[outside])


@pytest.mark.parametrize("docs,heads,kvh", [(3, 4, 2), (12, 4, 4), (40, 5, 1)])
def test_cache_attention_over_its_queries(ctx, docs, heads, kvh):
    """out may be q: every CTA of a cluster has read its rows before one is written."""
    g = gen(docs)
    cap = 8192 if docs >= 8 else 900
    new = [1 + (5 * b) % 9 for b in range(docs)]
    lens = [n + (997 * b) % (cap - 20) for b, n in enumerate(new)]
    cache, codes, scales = new_cache(g, docs, kvh, cap, torch.int8)
    k, v = randn(g, sum(lens), kvh, D), randn(g, sum(lens), kvh, D) * 40
    ctx.kv_cache_write(cache, k, v, i32(np.cumsum([0] + lens)), i32(lens))
    q = randn(g, sum(new), heads, D, dtype=BF16)
    off, held, want = i32(np.cumsum([0] + new)), i32(lens), torch.empty_like(q)
    ctx.cache_attention(cache, q, want, off, held, max_tokens=4)
    for _ in range(10):
        x = q.clone()
        ctx.cache_attention(cache, x, x, off, held, max_tokens=4)
        assert torch.equal(x, want)
