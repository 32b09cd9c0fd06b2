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
