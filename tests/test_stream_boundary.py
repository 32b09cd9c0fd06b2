"""C entry points of the streaming-attention operators without a GPU: va_stream.cu built against a stand-in
for the CUDA runtime and the launchers (fake_stream_runtime.cpp), which records what a launch was given."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import build as package_build
import vestra_attn as va

HERE = os.path.dirname(os.path.abspath(__file__))


class Seen(ctypes.Structure):
    _fields_ = [("launches", ctypes.c_int64), ("unfinished", ctypes.c_int64), ("items", ctypes.c_int64),
                ("most_keys", ctypes.c_int64), ("token_stride", ctypes.c_int64 * 2), ("head_stride", ctypes.c_int64 * 2),
                ("slope", ctypes.c_float * 4), ("rope_chunk", ctypes.c_int64), ("rope_pairs", ctypes.c_int64),
                ("rope_first", ctypes.c_uint8 * 128), ("rope_second", ctypes.c_uint8 * 128)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libstream.so")
    cuda = os.path.join(os.path.dirname(os.path.dirname(package_build.nvcc())), "include")
    gxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    # -Bsymbolic: the stand-ins, not a CUDA runtime that the process has loaded
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I" + cuda, "-I" + package_build.CSRC,
                    "-I" + os.path.join(package_build.ROOT, "include"), "-x", "c++",
                    os.path.join(package_build.CSRC, "va_stream.cu"), os.path.join(HERE, "fake_stream_runtime.cpp"),
                    "-o", so], check=True)
    fake = ctypes.CDLL(so)
    real = va.load_library()
    for name in ("va_rope_axes_device", "va_attn_plan_create", "va_attn_plan_destroy", "va_masked_attention_device",
                 "va_kv_cache_write_device", "va_kv_cache_read_device", "va_cache_attention_device"):
        getattr(fake, name).argtypes = getattr(real, name).argtypes
        getattr(fake, name).restype = getattr(real, name).restype
    fake.fake_context.restype = ctypes.c_void_p
    fake.fake_error.argtypes, fake.fake_error.restype = [ctypes.c_void_p], ctypes.c_char_p
    fake.fake_seen.restype = ctypes.POINTER(Seen)
    fake.ctx = fake.fake_context()
    return fake


@pytest.fixture(autouse=True)
def _fresh(lib):
    lib.fake_reset()


def heads_of(token_stride, head_stride, heads, dtype=va.VA_BF16, data=1 << 20):
    return va._PACK_HEADS(data, token_stride, head_stride, heads, dtype)


def create_plan(lib, q_offsets, k_offsets, heads=4, kv_heads=4, slopes=None, prefix=None):
    qo, ko = (np.asarray(x, np.int64) for x in (q_offsets, k_offsets))
    sl = None if slopes is None else np.asarray(slopes, np.float32)
    pre = None if prefix is None else np.asarray(prefix, np.int64)
    terms = va.VaAttnTerms(heads, kv_heads, 1, 1, 0.0, 0.0)
    plan = ctypes.c_void_p()
    rc = lib.va_attn_plan_create(lib.ctx, ctypes.byref(terms), qo.size - 1, va._ptr(qo), va._ptr(ko), va._ptr(pre),
                                 va._ptr(sl), ctypes.byref(plan))
    return rc, plan


# ------------------------------------------------------------------------------- plan
@pytest.mark.parametrize("slopes", [None, [0.5, 0.25, 0.125, 0.0625]])
@pytest.mark.parametrize("q_lens,k_lens", [([1], [900]), ([300, 40], [300, 500])])
def test_a_plan_is_on_the_device_when_create_returns(lib, slopes, q_lens, k_lens):
    """A copy from pageable memory may still be under way when it returns, and streams that do not wait for the
    legacy stream would read an unwritten work list."""
    rc, plan = create_plan(lib, np.cumsum([0] + q_lens), np.cumsum([0] + k_lens), slopes=slopes)
    assert rc == va.VA_OK
    assert lib.fake_pending() == 0
    q = heads_of(4 * 64, 64, 4)
    assert lib.va_masked_attention_device(lib.ctx, plan, q, q, q, q, 0x1234) == va.VA_OK
    seen = lib.fake_seen().contents
    assert seen.launches == 1 and seen.unfinished == 0
    assert seen.most_keys == max(k_lens)
    for h, s in enumerate(slopes or []):
        assert seen.slope[h] == pytest.approx(s * np.log2(np.e), rel=1e-6)
    lib.va_attn_plan_destroy(plan)


def test_a_layout_of_too_many_tiles_is_refused_before_it_is_built():
    """2^31 tiles of one token would be 60 GB of work list: refused by their number, in a process that may
    not allocate 2 GB more than it has."""
    code = """
import resource, sys
sys.path.insert(0, %r)
import numpy as np, vestra_attn as va
va.load_library()
with open('/proc/self/statm') as f:
    used = int(f.read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + 2 ** 31, used + 2 ** 31))
ends = np.minimum(np.arange(129, dtype=np.int64) * 2 ** 24, 2 ** 31 - 1)
try:
    va.attention_plan_shape(128, 1, ends, np.zeros(129, np.int64))
except va.VestraError as e:
    sys.exit(0 if e.code == va.VA_ERR_INVALID else 3)
sys.exit(4)
""" % os.path.dirname(va.__file__)
    assert subprocess.run([sys.executable, "-c", code], timeout=300).returncode == 0


# ------------------------------------------------------------------------------ slopes
@pytest.mark.parametrize("slope,ok", [(2.0 ** 96, True), (-2.0 ** 96, True), (2.0 ** 96 * 1.001, False), (3e38, False),
                                      (-3e38, False), (float("inf"), False), (float("nan"), False), (0.0, True)])
def test_slopes_whose_bias_would_leave_f32_are_refused(lib, slope, ok):
    """slope log2(e) times the largest distance has to stay finite: an infinite one times distance 0 is NaN."""
    rc, plan = create_plan(lib, [0, 3], [0, 3], slopes=[0.5, 0.5, slope, 0.5])
    assert rc == (va.VA_OK if ok else va.VA_ERR_INVALID)
    if ok:
        assert lib.va_masked_attention_device(lib.ctx, plan, *[heads_of(4 * 64, 64, 4)] * 4, 0) == va.VA_OK
        assert np.isfinite(np.float32(lib.fake_seen().contents.slope[2]) * np.float32(2.0 ** 30))
        lib.va_attn_plan_destroy(plan)
    else:
        assert b"slopes" in lib.fake_error(lib.ctx)


# ------------------------------------------------------------------------------ strides
PTR = 1 << 20


def cache_of(kv_heads, documents=1, capacity=64):
    return va.VaKvCache(documents, kv_heads, capacity, va.KV_INT8, 0, PTR, PTR, PTR, PTR)


def every_call(lib, h, rows, heads):
    """Return codes of the calls with all operands of these heads and rows."""
    cache, terms = cache_of(heads), va.VaAttnTerms(heads, heads, 1, 1, 0.0, 0.0)
    rope = va.VaRopeAxes(1, (ctypes.c_int32 * 4)(64), 0, 0, 100.0)
    out = [lib.va_rope_axes_device(lib.ctx, ctypes.byref(rope), rows, 64, PTR, h, h, h, h, 0),
           lib.va_kv_cache_write_device(lib.ctx, ctypes.byref(cache), rows, PTR, PTR, h, h, 0),
           lib.va_kv_cache_read_device(lib.ctx, ctypes.byref(cache), rows, PTR, PTR, h, h, 0),
           lib.va_cache_attention_device(lib.ctx, ctypes.byref(cache), ctypes.byref(terms), rows, PTR, PTR, 1, None,
                                         None, h, h, 0)]
    rc, plan = create_plan(lib, [0, rows], [0, rows], heads, heads)
    out += [rc, lib.va_masked_attention_device(lib.ctx, plan, h, h, h, h, 0)]
    lib.va_attn_plan_destroy(plan)
    return out


@pytest.mark.parametrize("rows,token_stride,head_stride", [
    (0, 64, 64), (0, 0, 0), (0, 256, 64),                                   # head-major and empty
    (1, 64, 64), (1, 0, 64), (1, 1, 64), (1, -8, 64), (1, 2 ** 40, 64),     # a stride that is never stepped over
    (1, 64, 2 ** 27), (1, 4 * 2 ** 27, 2 ** 27),                            # one row of a long head-major buffer
    (2, 256, 64), (2, 64, 128), (5, 64, 320), (5, 2 ** 30, 64)])
def test_strides_that_no_element_shares_are_taken(lib, rows, token_stride, head_stride):
    h = heads_of(token_stride, head_stride, 4)
    assert every_call(lib, h, rows, 4) == [va.VA_OK] * 6
    seen = lib.fake_seen().contents
    if seen.launches and rows == 1:
        assert seen.token_stride[0] % 8 == 0 and 0 < seen.token_stride[0] <= 2 ** 30
    if rows > 1:
        assert seen.token_stride[0] == token_stride and seen.head_stride[0] == head_stride


@pytest.mark.parametrize("rows,token_stride,head_stride", [
    (1, 64, 0), (1, 64, 63), (1, 64, -64), (1, 64, 2 ** 39), (2, 64, 64), (2, 0, 64), (2, -256, 64), (5, 64, 319),
    (5, 2 ** 30 + 8, 64), (5, 192, 64)])
def test_strides_that_overlap_are_refused(lib, rows, token_stride, head_stride):
    h = heads_of(token_stride, head_stride, 4)
    codes = every_call(lib, h, rows, 4)
    assert codes[4] == va.VA_OK and codes[:4] + codes[5:] == [va.VA_ERR_INVALID] * 5
    assert lib.fake_seen().contents.launches == 0


def view_on_device(x):
    """A meta tensor's numbers, as of a CUDA tensor."""
    class View:
        shape, dtype = x.shape, x.dtype
        get_device = staticmethod(lambda: 0)
        stride = staticmethod(x.stride)
        data_ptr = staticmethod(lambda: PTR)
    return View()


@pytest.mark.parametrize("rows", [0, 1, 2])
def test_a_few_rows_of_a_long_head_major_buffer(lib, rows):
    torch = pytest.importorskip("torch")
    x = torch.empty(16, 2 ** 22, 64, dtype=torch.bfloat16, device="meta")  # 2^28 elements a head
    packed, n, heads = va._heads(view_on_device(x[:, 5:5 + rows].transpose(0, 1)), 0, "q", 64)
    assert (n, heads) == (rows, 16)
    assert every_call(lib, packed, rows, 16) == [va.VA_OK] * 6


# ------------------------------------------------------------------------------ rotary vectors
@pytest.mark.parametrize("dtype,size", [(va.VA_BF16, 2), (va.VA_F16, 2), (va.VA_F32, 4)])
@pytest.mark.parametrize("pairing", [0, 1])
@pytest.mark.parametrize("layout", ["per_axis", "shared"])
def test_every_rotary_vector_is_aligned(lib, dtype, size, pairing, layout):
    """Random offsets, strides and sections: each vector that the chosen chunk loads or stores starts at a multiple
    of its size, and the chunk is as wide as that allows."""
    rng = np.random.default_rng(10 * pairing + size + len(layout))
    chunks = set()
    for _ in range(400):
        sections = [2 * int(rng.choice([1, 3, 4, 5, 8, 12, 16, 32])) for _ in range(int(rng.integers(1, 4)))]
        d, heads, rows = sum(sections) + 2 * int(rng.integers(0, 3)), int(rng.integers(1, 4)), int(rng.integers(1, 4))
        if d > 256:
            continue
        tensors = []
        for at in (PTR, 2 * PTR):  # input and output
            head = d + int(rng.choice([0, 0, 1, 2, 6, 8]))
            token = heads * head + int(rng.choice([0, 0, 0, 1, 4, 8]))
            tensors.append((at + size * int(rng.choice([0, 0, 0, 1, 2, 3, 4, 8])), token, head))
        rope = va.VaRopeAxes(len(sections), (ctypes.c_int32 * 4)(*sections), va.ROPE_LAYOUTS[layout], pairing, 100.0)
        packed = [heads_of(t, h, heads, dtype, p) for p, t, h in tensors]
        assert lib.va_rope_axes_device(lib.ctx, ctypes.byref(rope), rows, d, PTR, packed[0], packed[1], None, None, 0) == va.VA_OK
        seen = lib.fake_seen().contents
        v, pairs = seen.rope_chunk, seen.rope_pairs

        def aligned(v):
            if pairs % v:
                return False
            n = v * (2 if pairing else 1)
            starts = {0}
            for p, t, h in tensors:
                for r in range(rows):
                    for k in range(heads):
                        for at in range(0, pairs, v):
                            first, second = seen.rope_first[at], seen.rope_second[at]
                            # the chunk's pairs lie in a row
                            for e in range(v):
                                step = 2 * e if pairing else e
                                if (seen.rope_first[at + e], seen.rope_second[at + e]) != (first + step, second + step):
                                    return False
                            base = p + size * (r * t + k * h)
                            starts |= {(base + size * c) % (size * n) for c in ((first,) if pairing else (first, second))}
            return starts == {0}

        chunks.add(v)
        if v == 0:
            assert pairing == 1 and not aligned(1)  # element by element
            continue
        assert aligned(v)
        if 2 * v * (2 if pairing else 1) * size <= 16 and len(sections) == 1 and rows > 1 and heads > 1:
            assert not aligned(2 * v)
    assert chunks == ({0, 1, 2, 4} if pairing and size == 2 else {0, 1, 2} if pairing else {1, 2, 4, 8} if size == 2 else {1, 2, 4})


# ------------------------------------------------------------------------------ arrays read on the device
@pytest.mark.parametrize("which", ["positions", "offsets", "lens", "first", "prefix", "slopes"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_off_their_types_alignment_are_refused(lib, which, off):
    """An int32 or F32 array at an odd address would be a misaligned access in the kernel."""
    h = heads_of(256, 64, 4)
    cache, terms = cache_of(4), va.VaAttnTerms(4, 4, 1, 1, 0.0, 0.0)
    rope = va.VaRopeAxes(1, (ctypes.c_int32 * 4)(64), 0, 0, 100.0)
    at = {k: PTR + (off if k == which else 0) for k in ("positions", "offsets", "lens", "first", "prefix", "slopes")}
    calls = {
        "rope": lambda: lib.va_rope_axes_device(lib.ctx, ctypes.byref(rope), 3, 64, at["positions"], h, h, None, None, 0),
        "write": lambda: lib.va_kv_cache_write_device(lib.ctx, ctypes.byref(cache), 3, at["offsets"], at["lens"], h, h, 0),
        "read": lambda: lib.va_kv_cache_read_device(lib.ctx, ctypes.byref(cache), 3, at["offsets"], at["first"], h, h, 0),
        "attend": lambda: lib.va_cache_attention_device(lib.ctx, ctypes.byref(cache), ctypes.byref(terms), 3, at["offsets"],
                                                        at["lens"], 1, at["prefix"], at["slopes"], h, h, 0)}
    uses = {"positions": ["rope"], "offsets": ["write", "read", "attend"], "lens": ["write", "attend"], "first": ["read"],
            "prefix": ["attend"], "slopes": ["attend"]}[which]
    for name, call in calls.items():
        assert call() == (va.VA_ERR_INVALID if name in uses else va.VA_OK), name
