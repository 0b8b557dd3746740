"""What the paged cache's C ABI refuses before anything runs, and its host helpers.  Needs no GPU."""
import ctypes
import math
import os
import re

import numpy as np
import pytest

from litenn_b200 import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20  # stands for an aligned device address: refused calls look at no memory


@pytest.fixture(scope="module", autouse=True)
def library(qmm_lib):
    return qmm_lib


def test_header_and_binding_agree(qmm_lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "litenn_kv.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(qmm_[a-z0-9_]+)\s*\(", text)))
    assert names and sorted(capi.KV_SYMBOLS) == names
    for name in names:
        assert hasattr(qmm_lib, name), name


def refused(call, code=capi.E_INVALID, text=""):
    with pytest.raises(capi.QmmError) as e:
        call()
    assert e.value.code == code and text in str(e.value), str(e.value)


def cache(fmt=1, kv_heads=2, hd=128, page=16, n_pages=8, pool=A):
    return capi.KVCache(fmt, kv_heads, hd, page, n_pages, pool)


def batch(n=2, width=4, table=A, length=A, begin=0, rows=2):
    return capi.KVBatch(n, width, table, length, begin, rows)


def attend(c=None, b=None, heads=4, q=A, q_type=0, q_stride=512, out=2 * A, out_type=0, out_stride=512, scale=1.0, window=0,
           workspace=A):
    (c or cache()).attend(b or batch(), heads, q, q_type, q_stride, out, out_type, out_stride, scale, window, workspace)


def append(c=None, b=None, rope=None, heads=4, kind=0, q=A, qs=512, k=2 * A, ks=256, v=3 * A, vs=256, q_out=4 * A, q_type=0, os=512):
    (c or cache()).append(b or batch(), rope, heads, kind, q, qs, k, ks, v, vs, q_out, q_type, os)


@pytest.mark.parametrize("call", [attend, append])
def test_caches(call):
    refused(lambda: call(cache(fmt=2)), capi.E_UNSUPPORTED)
    refused(lambda: call(cache(fmt=9)), capi.E_UNSUPPORTED)
    for hd in (0, 32, 80, 160, 512):
        refused(lambda: call(cache(hd=hd)), text="head_dim")
    for page in (0, 8, 24, -16, 65552):
        refused(lambda: call(cache(page=page)), text="page_tokens")
    refused(lambda: call(cache(kv_heads=0)), text="kv heads")
    refused(lambda: call(cache(n_pages=0)), text="pages")
    refused(lambda: call(cache(n_pages=1 << 40)), text="pages")
    refused(lambda: call(cache(kv_heads=65536, hd=256, page=65536, n_pages=2 ** 31 - 1)), text="larger than any memory")
    refused(lambda: call(cache(pool=0)), text="pool")
    refused(lambda: call(cache(pool=A + 8)), text="pool")


@pytest.mark.parametrize("call", [attend, append])
def test_batches(call):
    refused(lambda: call(b=batch(n=-1)))
    refused(lambda: call(b=batch(rows=-1)))
    refused(lambda: call(b=batch(width=-1)))
    refused(lambda: call(b=batch(table=0)), text="page_table")
    refused(lambda: call(b=batch(length=0)), text="kv_len")
    refused(lambda: call(b=batch(n=3, rows=2)), text="one row each")
    refused(lambda: call(b=batch(rows=1 << 31, begin=A)), text="2^30")
    refused(lambda: call(cache(page=65536), b=batch(width=1 << 15)), text="31 bits")


@pytest.mark.parametrize("call", [attend, append])
def test_arrays_of_whole_numbers_are_aligned(call):
    for off in (1, 2, 3):
        refused(lambda: call(b=batch(table=A + off)), text="4-byte aligned")
        refused(lambda: call(b=batch(length=A + off)), text="4-byte aligned")
        refused(lambda: call(b=batch(begin=A + off)), text="4-byte aligned")


def test_attention_arguments():
    refused(lambda: attend(heads=0))
    refused(lambda: attend(heads=5), text="divide")
    refused(lambda: attend(window=-1))
    for scale in (math.nan, math.inf):
        refused(lambda: attend(scale=scale))
    refused(lambda: attend(q=0), text="q is null")
    refused(lambda: attend(q=A + 4), text="aligned")
    refused(lambda: attend(out=2 * A + 8), text="aligned")
    refused(lambda: attend(q_type=2), text="type")
    refused(lambda: attend(out_type=-1), text="type")
    refused(lambda: attend(q_stride=508), text="stride")
    refused(lambda: attend(q_stride=514), text="stride")
    refused(lambda: attend(q_type=1, q_stride=516), text="stride")
    refused(lambda: attend(out_stride=-512), text="stride")
    refused(lambda: attend(out=A), text="overlaps")
    refused(lambda: attend(out=A + 512 * 4), text="overlaps")
    refused(lambda: attend(q_stride=1024, out=A + 1024, out_stride=1024), text="overlaps")
    refused(lambda: attend(workspace=0), text="workspace")
    refused(lambda: attend(workspace=A + 128), text="workspace")


def test_append_arguments():
    refused(lambda: append(heads=-1))
    refused(lambda: append(heads=0))            # q without heads
    refused(lambda: append(q=0))                # heads without q
    refused(lambda: append(kind=3), text="type")
    refused(lambda: append(k=0), text="k is null")
    refused(lambda: append(v=3 * A + 2), text="v is null or")
    refused(lambda: append(ks=128), text="stride")
    refused(lambda: append(q_out=0), text="q_out")
    refused(lambda: append(q_out=A, os=1024), text="overlaps q")
    refused(lambda: append(q_out=A, q_type=1), text="overlaps q")
    refused(lambda: append(q_out=A + 16), text="overlaps q")
    refused(lambda: append(q_out=2 * A), text="overlaps k or v")
    for dim, layout in ((3, 0), (130, 0), (-2, 0), (12, 1), (64, 2)):
        refused(lambda: append(rope=capi.Rope(dim, layout, A, 1.0)))
    refused(lambda: append(rope=capi.Rope(64, 0, 0, 1.0)), text="inv_freq")
    refused(lambda: append(rope=capi.Rope(64, 0, A + 4, 1.0)), text="inv_freq")


def test_read_arguments():
    def read(k=A, ks=256, v=2 * A, vs=256, kind=0):
        cache().read(batch(), k, ks, v, vs, kind)
    refused(lambda: read(k=0))
    refused(lambda: read(kind=2))
    refused(lambda: read(vs=255))
    refused(lambda: read(v=A + 64), text="overlaps")


def test_without_a_gpu_a_good_call_fails_loudly():
    if capi.device_count() > 0:
        pytest.skip("a GPU is present")
    for call in (attend, append, lambda: cache().read(batch(), A, 256, 2 * A, 256, 0)):
        refused(call, capi.E_CUDA)
    # columns of one tensor side by side do not overlap: this call gets as far as the device
    refused(lambda: attend(q_stride=1024, out=A + 2048, out_stride=1024), capi.E_CUDA)
    refused(lambda: append(q_out=A), capi.E_CUDA)


def test_pool_bytes():
    assert capi.kv_pool_bytes(1, 8, 128, 64, 10) == 10 * 64 * 8 * 144
    assert capi.kv_pool_bytes(5, 2, 64, 16, 3) == 3 * 16 * 2 * 136
    assert capi.kv_pool_bytes(0, 1, 96, 32, 1) == 32 * 96 * 4
    refused(lambda: capi.kv_pool_bytes(1, 8, 80, 64, 10))
    refused(lambda: capi.kv_pool_bytes(3, 8, 64, 64, 10), capi.E_UNSUPPORTED)


def test_rope_frequencies():
    f, gain = capi.rope_frequencies(128, 10000.0)
    i = np.arange(64)
    np.testing.assert_allclose(f, 10000.0 ** (-2 * i / 128), rtol=1e-14)
    assert gain == 1.0
    lin, gain = capi.rope_frequencies(128, 10000.0, scaling=capi.RopeScaling(capi.ROPE_SCALE_LINEAR, 4.0, 0, 0, 0))
    np.testing.assert_allclose(lin, f / 4, rtol=1e-14)
    fac = np.linspace(1, 8, 64).astype(np.float32)
    div, _ = capi.rope_frequencies(128, 10000.0, factors=fac)
    np.testing.assert_allclose(div, f / fac.astype(np.float64), rtol=1e-14)
    # YaRN: by the paper's ramp over the pairs
    y, gain = capi.rope_frequencies(128, 10000.0, scaling=capi.RopeScaling(capi.ROPE_SCALE_YARN, 8.0, 4096, 32, 1))
    pair = lambda beta: 128 * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    low, high = math.floor(pair(32)), math.ceil(pair(1))
    ramp = np.clip((i - low) / (high - low), 0, 1)
    np.testing.assert_allclose(y, f * (1 - ramp) + f / 8 * ramp, rtol=1e-14)
    assert y[0] == f[0] and abs(y[-1] * 8 / f[-1] - 1) < 1e-14 and abs(gain - (0.1 * math.log(8) + 1)) < 1e-15
    with pytest.raises(ValueError):
        capi.rope_frequencies(128, 10000.0, factors=fac[:5])
    for dim, theta in ((3, 1e4), (0, 1e4), (64, 0.0), (64, math.nan), (64, -1.0)):
        refused(lambda: capi.rope_frequencies(dim, theta))
    for s in ((3, 2, 0, 0, 0), (1, 0.5, 0, 0, 0), (1, math.nan, 0, 0, 0), (2, 2, 0, 32, 1), (2, 2, 4096, 1, 32), (2, 2, 4096, 32, 0)):
        refused(lambda: capi.rope_frequencies(64, 1e4, scaling=capi.RopeScaling(*s)))
    refused(lambda: capi.rope_frequencies(4, 1e4, factors=np.array([1, 0], dtype=np.float32)))


def test_null_structures():
    L = capi.load()
    assert L.qmm_kv_pool_bytes(None, ctypes.byref(ctypes.c_size_t())) == capi.E_INVALID
    assert L.qmm_kv_attention(0, None, None, 1, None, 0, 0, None, 0, 0, 1.0, 0, None, None) == capi.E_INVALID
    assert L.qmm_kv_append(0, cache().desc, None, None, 0, 0, None, 0, None, 0, None, 0, None, 0, 0, None) == capi.E_INVALID
    assert L.qmm_kv_read(0, None, None, None, 0, None, 0, 0, None) == capi.E_INVALID
    assert L.qmm_rope_frequencies(64, 1e4, None, None, None, None) == capi.E_INVALID


def test_decoder_entry_points_without_a_model():
    L = capi.load()
    assert L.qmm_llama_set_rope_scaling(None, None, None) == capi.E_INVALID
    assert L.qmm_llama_batch_create_paged(None, 1, 1, 1, 0, 1) == capi.E_INVALID
    assert L.qmm_llama_batch_create_paged(None, 1, 1, 1, 64, 1) == capi.E_INVALID
    assert L.qmm_llama_batch_free_pages(None, ctypes.byref(ctypes.c_int64())) == capi.E_INVALID
