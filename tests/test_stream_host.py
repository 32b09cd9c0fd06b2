"""Host side of the streaming-attention operators, no GPU: the plan of a masked-attention
layout (tiles, key ranges, refusals), argument structures, and the Python mirror's checks."""
import ctypes

import numpy as np
import pytest

import vestra_attn as va


def shape(q_lens, k_lens, heads=12, kv_heads=12, **kw):
    return va.attention_plan_shape(heads, kv_heads, np.cumsum([0] + list(q_lens)), np.cumsum([0] + list(k_lens)), **kw)


def test_structures_match_the_header():
    """Sizes of the C structures on this ABI (LP64)."""
    assert len(va._PACK_HEADS(1, 2, 3, 4, 0)) == 32
    assert ctypes.sizeof(va.VaRopeAxes) == 32
    assert ctypes.sizeof(va.VaAttnTerms) == 24
    assert ctypes.sizeof(va.VaKvCache) == 56


def test_tiles_pack_the_heads_that_share_a_key_head():
    for heads, kv, tokens in ((12, 12, 128), (12, 4, 42), (16, 1, 8), (128, 1, 1), (100, 1, 1), (10, 2, 25)):
        p = shape([256], [256], heads, kv)
        assert p["tile_tokens"] == tokens
        assert p["tiles"] == -(-256 // tokens) * kv
        assert p["ctas"] == p["tiles"] * p["splits"]


def test_causal_tiles_take_only_the_keys_their_last_row_sees():
    full = shape([1024], [1024], 1, 1)
    assert full["key_tiles"] == 8 * 8
    assert shape([1024], [1024], 1, 1, causal=True)["key_tiles"] == sum(range(1, 9))
    # frames of 512 tokens: the first four tiles see 512 keys, the others all
    assert shape([1024], [1024], 1, 1, causal=True, frame=512)["key_tiles"] == 4 * 4 + 4 * 8
    # a prefix is seen by every row
    assert shape([1024], [1024], 1, 1, causal=True, prefix=[300])["key_tiles"] == 3 + 3 + 3 + 4 + 5 + 6 + 7 + 8
    # new rows at the end of longer documents
    assert shape([128], [1024], 1, 1, causal=True)["key_tiles"] == 8
    # more rows than keys: the first rows see nothing
    assert shape([1024], [128], 1, 1, causal=True)["key_tiles"] == 1
    assert shape([0, 5], [7, 0], 1, 1, causal=True) == dict(tiles=1, splits=1, tile_tokens=128, key_tiles=0, ctas=1)


def test_few_tiles_are_cut_over_their_keys():
    assert shape([1], [10392], causal=True)["splits"] >= 8
    assert shape([128 * 296 // 12 * 12], [10392], 1, 1)["splits"] == 1  # whole waves of two CTAs per SM
    assert shape([64], [128])["splits"] == 1       # one key tile
    for n in (1, 100, 866, 2598):
        p = shape([n], [10392])
        assert 1 <= p["splits"] <= 16 and p["ctas"] <= 2 ** 31 - 1


@pytest.mark.parametrize("kw", [
    dict(heads=12, kv_heads=5), dict(heads=0), dict(heads=129, kv_heads=1), dict(kv_heads=0), dict(frame=0),
    dict(frame=-3), dict(q_offsets=[0, 5, 4], k_offsets=[0, 1, 2]), dict(k_offsets=[0, 5, 4], q_offsets=[0, 1, 2]),
    dict(q_offsets=[-1, 4]), dict(k_offsets=[-1, 4]), dict(k_offsets=[0, 2 ** 24 + 1]), dict(q_offsets=[0, 2 ** 24 + 1]),
    dict(k_offsets=[2 ** 31 - 2, 2 ** 31 + 5]), dict(prefix=[-1]), dict(q_offsets=[0]), dict(prefix=[1, 2]),
    dict(sms=0), dict(k_offsets=[0, 2 ** 62]), dict(q_offsets=[0, 4, 2 ** 62], k_offsets=[0, 4, 8])])
def test_bad_layouts_are_refused(kw):
    args = dict(heads=12, kv_heads=12, q_offsets=[0, 8], k_offsets=[0, 8])
    args.update(kw)
    with pytest.raises(va.VestraError) as e:
        va.attention_plan_shape(**args)
    assert e.value.code == va.VA_ERR_INVALID


def test_null_arguments_are_refused():
    lib = va.load_library()
    out = (ctypes.c_int64 * 5)()
    t = va.VaAttnTerms(4, 4, 0, 1, 0.0, 0.0)
    off = (ctypes.c_int64 * 2)(0, 4)
    assert lib.va_attn_plan_shape(None, 1, off, off, None, 148, out) == va.VA_ERR_INVALID
    assert lib.va_attn_plan_shape(ctypes.byref(t), 1, None, off, None, 148, out) == va.VA_ERR_INVALID
    assert lib.va_attn_plan_shape(ctypes.byref(t), 1, off, off, None, 148, None) == va.VA_ERR_INVALID
    assert lib.va_attn_plan_shape(ctypes.byref(t), 0, off, off, None, 148, out) == va.VA_ERR_INVALID
    h = ctypes.c_void_p()
    assert lib.va_attn_plan_create(None, ctypes.byref(t), 1, off, off, None, None, ctypes.byref(h)) == va.VA_ERR_INVALID
    assert lib.va_rope_axes_device(None, None, 0, 64, None, None, None, None, None, None) == va.VA_ERR_INVALID
    assert lib.va_masked_attention_device(None, None, None, None, None, None, None) == va.VA_ERR_INVALID
    assert lib.va_kv_cache_write_device(None, None, 0, None, None, None, None, None) == va.VA_ERR_INVALID
    assert lib.va_kv_cache_read_device(None, None, 0, None, None, None, None, None) == va.VA_ERR_INVALID
    assert lib.va_cache_attention_device(None, None, None, 0, None, None, 1, None, None, None, None, None) == \
        va.VA_ERR_INVALID
    lib.va_attn_plan_destroy(None)


def test_the_mirror_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(va.VestraError):
        va._heads(x, 0, "q", 64)
    with pytest.raises(va.VestraError):
        va._device_array(torch.zeros(3, dtype=torch.int32), 0, "offsets", va._INT32, 3)
    with pytest.raises(va.VestraError):
        va.RopeAxes((16, 16, 16, 8, 8))
    codes, scales = torch.zeros(1, 2, 8, 64, dtype=torch.int8), torch.zeros(1, 2, 8, dtype=torch.float32)
    cache = va.KvCache(codes, codes.clone(), scales, scales.clone())
    with pytest.raises(va.VestraError):
        cache.check_device(0)
    with pytest.raises(va.VestraError):
        va.KvCache(codes, codes, scales, scales[:, :, :4])
