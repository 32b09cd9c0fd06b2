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
                ("slope", ctypes.c_float * 4)]


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
