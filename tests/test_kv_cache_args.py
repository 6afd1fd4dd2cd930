"""CPU: the key/value cache's entry points check their arguments before they
touch a device, and refuse without one."""
import ctypes

import pytest
import torch

from burn_image_b200 import KVCache
from burn_image_b200 import _lib as L
from burn_image_b200.q4 import Bq4Error

FAKE = 1 << 20  # an aligned address that nothing reads: every call below is refused on the host
S3 = (ctypes.c_int64 * 3)(1024, 1024, 128)


def cache(**kw):
    f = dict(data=FAKE, pages=4, page_size=16, kv_heads=2, head_dim=128, format=L.CACHE_Q8, device=0)
    f.update(kw)
    return L.Cache(**f)


def seqs(**kw):
    f = dict(page_table=FAKE, table_stride=4, table_width=4, lengths=FAKE, batch=2)
    f.update(kw)
    return L.CacheSequences(**f)


def append(c=None, s=None, k=FAKE, v=FAKE, dtype=L.DTYPE_F16, tokens=3, strides=S3):
    c, s = c or cache(), s or seqs()
    return L.lib().bq4_cache_append(ctypes.byref(c), ctypes.byref(s), k, strides, v, strides, dtype, tokens, None)


def read(c=None, s=None, out=FAKE, dtype=L.DTYPE_F32, count=3, starts=None):
    c, s = c or cache(), s or seqs()
    return L.lib().bq4_cache_read(ctypes.byref(c), ctypes.byref(s), starts, count, out, out, S3, dtype, None)


def attention(c=None, s=None, max_length=0, q=FAKE, tokens=1, q_heads=4, out=FAKE, scale=0.0):
    c, s = c or cache(), s or seqs()
    return L.lib().bq4_cache_attention(ctypes.byref(c), ctypes.byref(s), max_length, q, S3, tokens, q_heads, 1, scale,
                                       out, None, 0, None)


def prefix(c=None, s=None, pages=FAKE, width=2, length=FAKE):
    c, s = c or cache(), s or seqs()
    return L.lib().bq4_cache_prefix_attention(ctypes.byref(c), pages, width, length, ctypes.byref(s), 0, FAKE, S3, 1, 4,
                                              1, 0.0, FAKE, None, 0, None)


GEOMETRY = [(dict(format=3), L.EINVAL_ARG), (dict(format=-1), L.EINVAL_ARG), (dict(pages=0), L.EINVAL_SHAPE),
            (dict(pages=1 << 31), L.EINVAL_SHAPE), (dict(page_size=0), L.EINVAL_SHAPE),
            (dict(page_size=24), L.EINVAL_SHAPE), (dict(page_size=1 << 17), L.EINVAL_SHAPE),
            (dict(kv_heads=0), L.EINVAL_SHAPE), (dict(head_dim=0), L.EINVAL_SHAPE), (dict(head_dim=20), L.EINVAL_SHAPE),
            (dict(head_dim=136), L.EINVAL_SHAPE),
            (dict(pages=(1 << 31) - 1, page_size=65536, kv_heads=65535), L.EINVAL_SHAPE)]


@pytest.mark.parametrize("change,status", GEOMETRY)
def test_geometry_is_checked_by_every_call(change, status):
    c = cache(**change)
    a = ctypes.c_size_t()
    assert L.lib().bq4_cache_size(ctypes.byref(c), ctypes.byref(a)) == status
    assert append(c) == read(c) == attention(c) == prefix(c) == status
    assert L.lib().bq4_cache_attention_workspace_size(ctypes.byref(c), 1, 1, 4, 16, 0, ctypes.byref(a)) == status


def test_size():
    a = ctypes.c_size_t()
    for fmt, dim, row, scales in ((L.CACHE_F16, 120, 256, 0), (L.CACHE_Q8, 128, 128, 1), (L.CACHE_Q8, 64, 64, 1),
                                  (L.CACHE_Q4, 128, 64, 4), (L.CACHE_Q4, 72, 64, 4), (L.CACHE_Q4, 40, 32, 2)):
        c = cache(format=fmt, head_dim=dim, data=None)
        assert L.lib().bq4_cache_size(ctypes.byref(c), ctypes.byref(a)) == L.OK
        assert a.value == 4 * 2 * 2 * 16 * (row + 2 * scales)
    assert L.lib().bq4_cache_size(None, ctypes.byref(a)) == L.EINVAL_ARG
    assert L.lib().bq4_cache_size(ctypes.byref(c), None) == L.EINVAL_ARG
    # 2^34 rows: past 32 bits
    c = cache(pages=1 << 20, page_size=4096, kv_heads=4)
    assert L.lib().bq4_cache_size(ctypes.byref(c), ctypes.byref(a)) == L.OK
    assert a.value == (1 << 32) * 4 * 2 * 130


@pytest.mark.parametrize("call", [append, read, attention, prefix])
def test_buffers_and_sequences_are_checked(call):
    assert call(cache(data=None)) == L.EINVAL_ARG
    assert call(cache(data=FAKE + 16)) == L.EALIGN
    assert call(s=seqs(lengths=None)) == L.EINVAL_ARG
    assert call(s=seqs(page_table=None)) == L.EINVAL_ARG
    assert call(s=seqs(lengths=FAKE + 2)) == L.EALIGN
    assert call(s=seqs(batch=-1)) == L.EINVAL_SHAPE
    assert call(s=seqs(table_width=-1)) == L.EINVAL_SHAPE
    assert call(s=seqs(table_stride=-4)) == L.EINVAL_SHAPE
    assert call(s=seqs(table_width=(1 << 26) + 1)) == L.EINVAL_SHAPE
    assert call(s=seqs(batch=1 << 31)) == L.EINVAL_SHAPE
    assert call(s=seqs(batch=0, page_table=None, lengths=None)) == L.OK  # nothing to do
    if not torch.cuda.is_available():
        assert call() in (L.EINVAL_ARG, L.EUNSUPPORTED, L.ECUDA)  # no device: refused, never computed
    assert call(cache(device=99)) == L.EINVAL_ARG
    assert call(cache(device=-1)) == L.EINVAL_ARG


def test_append_arguments():
    assert append(dtype=2) == L.EINVAL_ARG
    assert append(tokens=-1) == L.EINVAL_SHAPE
    assert append(tokens=1 << 30) == L.EINVAL_SHAPE
    assert append(tokens=0, k=None, v=None) == L.OK
    assert append(k=None) == append(v=None) == append(strides=None) == L.EINVAL_ARG
    assert append(k=FAKE + 1) == L.EALIGN
    assert append(v=FAKE + 2, dtype=L.DTYPE_F32) == L.EALIGN


def test_read_arguments():
    assert read(dtype=2) == L.EINVAL_ARG
    assert read(count=-1) == L.EINVAL_SHAPE
    assert read(count=1 << 30) == L.EINVAL_SHAPE
    assert read(count=0, out=None) == L.OK
    assert read(out=None) == L.EINVAL_ARG
    assert read(out=FAKE + 2) == L.EALIGN
    assert read(starts=FAKE + 2) == L.EALIGN


def test_attention_arguments():
    assert attention(q_heads=3) == L.EINVAL_SHAPE
    assert attention(q_heads=0) == L.EINVAL_SHAPE
    assert attention(tokens=-1) == L.EINVAL_SHAPE
    assert attention(tokens=1 << 30) == L.EINVAL_SHAPE
    assert attention(max_length=-1) == L.EINVAL_SHAPE
    assert attention(tokens=0, q=None, out=None) == L.OK
    assert attention(q=None) == attention(out=None) == L.EINVAL_ARG
    assert attention(out=FAKE + 8) == L.EALIGN
    assert attention(q=FAKE + 1) == L.EALIGN
    assert attention(scale=float("nan")) == L.EINVAL_ARG
    assert prefix(length=None) == prefix(pages=None) == L.EINVAL_ARG
    assert prefix(width=-1) == prefix(width=(1 << 26) + 1) == L.EINVAL_SHAPE
    assert prefix(pages=FAKE + 2) == prefix(length=FAKE + 2) == L.EALIGN


def test_python_refuses_what_it_cannot_take():
    with pytest.raises(Bq4Error, match="format"):
        KVCache(4, 16, 2, 128, "q5")
    with pytest.raises(Bq4Error, match="page_size"):
        KVCache(4, 20, 2, 128)
    with pytest.raises(Bq4Error, match="CUDA device"):
        KVCache(4, 16, 2, 128, device="cpu")


def test_an_infinite_scale_is_refused():
    for scale in (float("inf"), 1e39):
        assert attention(scale=scale) == L.EINVAL_ARG
        assert b"scale" in L.lib().bq4_last_error_string()


@pytest.mark.parametrize("what", ["pages", "page_size", "kv_heads", "head_dim"])
def test_sizes_past_their_c_fields_are_refused(what):
    for size in (2 ** 64 + 16, 2 ** 32 + 16, 2 ** 31, 0, -16):
        sizes = dict(pages=4, page_size=16, kv_heads=2, head_dim=128)
        sizes[what] = size
        with pytest.raises(Bq4Error, match=what):
            KVCache(**sizes)


def test_workspace_size_arguments():
    n, c = ctypes.c_size_t(), cache()

    def size(batch=1, tokens=1, q_heads=4, max_length=64, max_prefix=0):
        return L.lib().bq4_cache_attention_workspace_size(ctypes.byref(c), batch, tokens, q_heads, max_length,
                                                          max_prefix, ctypes.byref(n))

    for bad in (dict(max_length=-2 ** 30 - 1), dict(max_length=-2 ** 63), dict(max_length=2 ** 30 + 1),
                dict(max_prefix=-1), dict(max_prefix=2 ** 30 + 1), dict(batch=-1), dict(tokens=-1), dict(q_heads=3),
                dict(tokens=2 ** 31)):
        assert size(**bad) == L.EINVAL_SHAPE, bad
    assert size(batch=0) == size(batch=0, max_length=-64) == size(tokens=0) == L.OK and n.value == 0
