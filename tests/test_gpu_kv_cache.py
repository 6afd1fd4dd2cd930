"""GPU: the paged key/value cache (KVCache) against plain 64-bit
implementations of its definitions.

- written rows read back exactly as q * scale rounded once, for every format,
  head size and source type, strided sources, pages of 16 to 128 rows;
- attention over the cache and with a shared prefix: formats, head layouts,
  one to many query tokens, ragged and zero lengths, causal or not, pages that
  end inside a tile, NaN behind a length;
- rows that no call names stay as they were; out-of-range pages and lengths
  are reported; caches past 4 GiB; streams and graphs; the calls in sequence.

Tolerance of an attention output (f16).  The kernels sum f16-rounded
probabilities (off by at most half a step, 2^-11 of each) in f32 and round the
result once (2^-11 of it), so with a = sum_j p_j |v_j|
    |out - exact| <= 2^-11 |exact| + 2^-11 a + a d + 2^-25,
where d covers the f32 score: an error of e in the exponent moves p by a
factor 1 + e.  A score is at most SCORE in size (asserted) with sums of |q k|
at most 8 SCORE, over at most 32 roundings of 2^-24: e <= 2^-16 SCORE for the
numerator, the same for the sum; plus 2^-14 for the exponential, the online
rescalings and f32 sums of up to 2^10 steps of 2^-24.
The kernels for many rows a kv head also round the widened v of an 8-bit cache to
f16 (at most half a step, 2^-11 of each value): where `staged` is given, another
2^-11 a.  BQ4_CACHE_TILE=1 takes them for every call, 0 for none.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import oracle as O
from burn_image_b200 import KVCache, q4
from burn_image_b200 import _lib as L
from burn_image_b200 import f16 as F
from burn_image_b200.q4 import Bq4Error
from conftest import gen_q4

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
QMAX = {"q8": 127.0, "q4": 7.0}


# --------------------------------------------------------------------- 64-bit definitions

def held(x, fmt):
    """What the cache stands for, of rows [..., D], in 64 bits."""
    if fmt == "f16":
        return x.float().half().double()
    parts = []
    for p in x.double().split(x.shape[-1] if fmt == "q8" else 32, -1):
        top = p.abs().amax(-1, keepdim=True)
        s = (top / QMAX[fmt]).float().bfloat16().double()
        q = (p / s).float().double().round().clamp(-QMAX[fmt], QMAX[fmt])
        w = torch.where(s > 0, q * s, torch.zeros_like(q))
        parts.append(torch.where(p.isfinite().all(-1, keepdim=True), w, torch.full_like(w, math.nan)))
    return torch.cat(parts, -1)


def attend(q, ks, vs, causal, pk=None, pv=None, scale=None):
    """q [B,S,Hq,D] (64-bit); ks, vs: per sequence [n,Hkv,D]; pk, pv: prefix rows or None.
    Returns out and sum p |v| (both [B,S,Hq,D]), and the largest |score|."""
    B, S, Hq, D = q.shape
    c = 1 / math.sqrt(D) if scale is None else scale
    out, mag, top = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for b in range(B):
        k, v = ks[b], vs[b]
        n0 = 0
        if pk is not None:
            k, v, n0 = torch.cat([pk, k]), torch.cat([pv, v]), pk.shape[0]
        n = k.shape[0]
        if n == 0:
            continue
        g = Hq // k.shape[1]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        s = torch.einsum("shd,nhd->hsn", q[b], k) * c
        top = max(top, s.abs().nan_to_num().max().item())
        if causal:
            see = n0 + (n - n0 - S + 1 + torch.arange(S, device=q.device)).clamp(min=0)  # the whole prefix, always
            s = s.masked_fill(torch.arange(n, device=q.device)[None, None] >= see[None, :, None], -math.inf)
        p = torch.softmax(s, -1).masked_fill((s == -math.inf).all(-1, keepdim=True), 0.0)
        out[b] = torch.einsum("hsn,nhd->shd", p, v)
        mag[b] = torch.einsum("hsn,nhd->shd", p, v.abs())
    return out, mag, top


def check(got, exact, mag, top, staged=False):
    q4.poll_device_error()
    rounded = 2.0 ** -10 if staged else 2.0 ** -11
    tol = 2.0 ** -11 * exact.abs() + (rounded + 2.0 ** -15 * top + 2.0 ** -14) * mag + 2.0 ** -25
    err = (got.double() - exact).abs()
    assert not got.isnan().any()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst} times the tolerance (max error {err.max().item()})"


class Book:
    """A cache whose pages are handed out in no order, beside the rows that went in."""

    def __init__(self, fmt, lengths, Hkv, D, page, prefix=0, seed=0, spare=3, poison=False):
        g = torch.Generator().manual_seed(seed + 77)
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        B = len(lengths)
        W = max(1, -(-max(lengths + [1]) // page))
        PW = -(-prefix // page)
        pages = B * W + PW + spare
        order = torch.randperm(pages, generator=g).int().to(DEV)
        self.table, self.ptable = order[:B * W].reshape(B, W), order[B * W:B * W + PW]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        self.plen = torch.tensor([prefix], dtype=torch.int32, device=DEV)
        self.cache = KVCache(pages, page, Hkv, D, fmt, DEV)
        if poison:  # NaN in every place that a length leaves out
            self.cache.data.fill_(0xFF)
        self.k, self.v = [], []
        for b, n in enumerate(lengths):
            k, v = self.rows(n, Hkv, D), self.rows(n, Hkv, D)
            if n:
                self.cache.append(k[None], v[None], self.table[b:b + 1], self.lengths[b:b + 1])
            self.k.append(held(k, fmt)), self.v.append(held(v, fmt))
        self.pk = self.pv = None
        if prefix:
            k, v = self.rows(prefix, Hkv, D), self.rows(prefix, Hkv, D)
            self.cache.append(k[None], v[None], self.ptable[None], self.plen)
            self.pk, self.pv = held(k, fmt), held(v, fmt)

    def rows(self, n, H, D):
        off = torch.randn((1, H, D), generator=self.g, device=DEV) * 0.5
        return (torch.randn((n, H, D), generator=self.g, device=DEV) + off).half()

    def query(self, S, Hq):
        return torch.randn((len(self.k), S, Hq, self.cache.head_dim), generator=self.g, device=DEV).half()


# --------------------------------------------------------------------- write and read

@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("D", [128, 120, 72, 64, 8])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_write_and_read_back(fmt, D, src):
    B, S, H, page = 3, 19, 3, 16
    g = torch.Generator(device=DEV).manual_seed(D)
    lengths = torch.tensor([40, 19, 7], dtype=torch.int32, device=DEV)  # the third: 12 rows fall below 0
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).int().to(DEV)[:9].reshape(3, 3)
    c = KVCache(12, page, H, D, fmt, DEV)
    size = torch.rand((B, S, H, 1), generator=g, device=DEV) * 3
    k = (torch.randn((B, S, H, D), generator=g, device=DEV) * size).to(src)
    v = torch.randn((B, S, H, D), generator=g, device=DEV).to(src)
    k[0, 3] = 0.0  # an all-zero row
    k[1, 2, 1, :8] *= 1e-4 if src == torch.float16 else 1e-30
    c.append(k, v, table, lengths)
    for dtype in (torch.float32, torch.float16):
        got = c.read(table, lengths, S + 5, starts=lengths - S, dtype=dtype)
        for x, y in zip((k, v), got):
            want = torch.zeros((B, H, S + 5, D), dtype=torch.float64, device=DEV)
            want[:, :, :S] = held(x, fmt).transpose(1, 2)
            want[2, :, :12] = 0.0  # positions below 0
            assert torch.equal(y, want.float().to(dtype))
    q4.poll_device_error()


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
def test_extreme_values(fmt):
    c = KVCache(2, 16, 1, 64, fmt, DEV)
    x = torch.zeros((1, 8, 1, 64), device=DEV)
    x[0, 0] = 1e-42            # under the smallest scale
    x[0, 1] = 3e38             # near the largest float32
    x[0, 2, 0, 5] = math.inf
    x[0, 3, 0, 40] = math.nan
    x[0, 4] = torch.linspace(-6e4, 6e4, 64, device=DEV)
    x[0, 5] = torch.linspace(-1.0, 1.0, 64, device=DEV) * 2.0 ** -120
    x[0, 6, 0, 0] = -7.0       # whole numbers are exact
    x[0, 7, 0, 33] = -math.inf
    table = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    n = torch.tensor([8], dtype=torch.int32, device=DEV)
    c.append(x, -x, table, n)
    k, v = c.read(table, n, 8, dtype=torch.float32)
    q4.poll_device_error()
    for y, z in ((k, x), (v, -x)):
        want = held(z[0], fmt).float()[:, 0]
        assert torch.equal(y[0, 0].nan_to_num(123.0), want.nan_to_num(123.0))
        assert torch.equal(y[0, 0].isnan(), want.isnan())


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_many_values_and_ties(fmt):
    # 2^23 values of rows from 2^-140 to 2^100, and rows of exact halves of their scale
    g = torch.Generator(device=DEV).manual_seed(17)
    c = KVCache(64, 256, 4, 128, fmt, DEV)
    x = torch.randn((64, 256, 4, 128), generator=g, device=DEV)
    x *= 2.0 ** torch.randint(-140, 101, (64, 256, 4, 1), generator=g, device=DEV).double().float()
    s = 2.0 ** torch.randint(-20, 20, (8, 256, 4, 1), generator=g, device=DEV).float()
    top = int(QMAX[fmt])
    x[:8] = (torch.randint(-top, top, (8, 256, 4, 128), generator=g, device=DEV) + 0.5) * s
    x[:8, :, :, ::32] = QMAX[fmt] * s  # the largest of every block: the scale is s
    table = torch.arange(64, dtype=torch.int32, device=DEV)[:, None]
    n = torch.full((64,), 256, dtype=torch.int32, device=DEV)
    for v in (x, x.clamp(-6e4, 6e4).half()):
        c.append(v, v, table, n)
        for y in c.read(table, n, 256, dtype=torch.float32):
            assert torch.equal(y, held(v, fmt).float().transpose(1, 2))
    q4.poll_device_error()


@pytest.mark.parametrize("fmt", ["q8", "q4", "f16"])
def test_strided_sources_and_untouched_rows(fmt):
    # k and v as sections of one projection output, head-major views, an odd offset (scalar loads)
    B, S, H, D = 2, 5, 2, 128
    g = torch.Generator(device=DEV).manual_seed(4)
    proj = torch.randn((B, S, 4 * H * D), generator=g, device=DEV).half()
    k = proj[:, :, 2 * H * D:3 * H * D].unflatten(-1, (H, D))
    v = proj[:, :, 3 * H * D:].unflatten(-1, (H, D))
    table = torch.tensor([[5, 0], [3, 1]], dtype=torch.int32, device=DEV)
    n = torch.tensor([18, 5], dtype=torch.int32, device=DEV)
    plain = KVCache(6, 16, H, D, fmt, DEV)
    plain.data.fill_(0x5A)
    before = plain.read(torch.arange(6, dtype=torch.int32, device=DEV)[:, None], torch.full((6,), 16, dtype=torch.int32,
                                                                                           device=DEV), 16)
    plain.append(k.contiguous(), v.contiguous(), table, n)
    odd = torch.empty(B * S * H * D + 1, dtype=torch.float16, device=DEV)[1:].view(B, S, H, D).copy_(k)
    turned = v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    for kk, vv in ((k, v), (odd, turned), (k.transpose(-1, -2).contiguous().transpose(-1, -2), v)):
        c = KVCache(6, 16, H, D, fmt, DEV)
        c.data.fill_(0x5A)
        c.append(kk, vv, table, n)
        assert torch.equal(c.data, plain.data)
    after = plain.read(torch.arange(6, dtype=torch.int32, device=DEV)[:, None], torch.full((6,), 16, dtype=torch.int32,
                                                                                          device=DEV), 16)
    touched = torch.zeros((6, 16), dtype=torch.bool, device=DEV)
    for b, length in ((0, 18), (1, 5)):
        for p in range(length - S, length):
            touched[table[b, p // 16].long(), p % 16] = True
    for x, y in zip(before, after):
        keep = ~touched[:, None, :, None].expand_as(x)
        assert torch.equal(x[keep].nan_to_num(9.0), y[keep].nan_to_num(9.0))
    # an output dtype and starts past the length read zeros
    k0, v0 = plain.read(table, n, 4, starts=torch.tensor([17, -2], dtype=torch.int32, device=DEV))
    assert k0[0, :, 1:].abs().sum() == 0 and k0[1, :, :2].abs().sum() == 0 and v0[1, :, 2:].abs().sum() > 0
    q4.poll_device_error()


# --------------------------------------------------------------------- attention

def run_attention(book, S, Hq, causal=True, scale=None, staged=False):
    q = book.query(S, Hq)
    got = book.cache.attention(q, book.table, book.lengths, causal=causal, scale=scale)
    check(got, *attend(q.double(), book.k, book.v, causal, scale=scale), staged=staged)
    return q, got


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (28, 7, 120), (3, 3, 64), (6, 1, 72), (16, 1, 128), (40, 2, 96),
                                      (2, 1, 8)])
def test_decode(fmt, Hq, Hkv, D):
    book = Book(fmt, [0, 1, 15, 16, 17, 63, 64, 129, 500], Hkv, D, 16, seed=Hq + D, poison=True)
    run_attention(book, 1, Hq)


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("S,causal", [(2, True), (3, False), (5, True), (8, True), (17, True), (33, False), (70, True)])
def test_several_query_tokens(fmt, S, causal):
    # lengths below S leave the first rows without a key
    book = Book(fmt, [S + 200, S, max(0, S - 2), 1, S + 31], 2, 128, 48, seed=S, poison=True)
    run_attention(book, S, 8, causal)


@pytest.mark.parametrize("fmt", ["q8", "q4", "f16"])
def test_one_long_context(fmt):
    book = Book(fmt, [9001], 2, 128, 64, seed=3)
    run_attention(book, 1, 8)
    run_attention(book, 4, 16)


@pytest.fixture(params=["0", "1"], ids=["split", "tile"])
def path(request, monkeypatch):
    monkeypatch.setenv("BQ4_CACHE_TILE", request.param)
    return request.param


def test_many_query_tokens(path):
    for fmt, S, n, D, causal in (("q8", 300, 1111, 128, True), ("q4", 129, 129, 64, True),
                                 ("f16", 256, 700, 120, False), ("q8", 513, 2000, 120, True)):
        run_attention(Book(fmt, [n, max(0, n - 130), 40], 2, D, 32, seed=S, poison=True), S, 8, causal, staged=True)


def test_scale_and_running_maximum():
    # scores that grow along the keys: the running maximum moves all the way
    for fmt in ("f16", "q8", "q4"):
        book = Book(fmt, [700], 1, 128, 16, seed=8)
        ramp = torch.linspace(0.05, 4.0, 700, device=DEV)[:, None, None]
        k = (book.rows(700, 1, 128).abs() * ramp).half()
        book.cache.append(k[None], k[None].flip(1), book.table, book.lengths)
        book.k, book.v = [held(k, fmt)], [held(k.flip(0), fmt)]
        q = book.query(2, 4).abs()
        for scale in (0.02, 0.2):
            got = book.cache.attention(q, book.table, book.lengths, scale=scale)
            check(got, *attend(q.double(), book.k, book.v, True, scale=scale))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_values_of_very_different_size(fmt):
    # v rows from 2^-12 to 2^12: their scales must not leave a probability's range.  Small rows
    # beside large ones: the tolerance's a is the large ones' share.
    book = Book(fmt, [300, 77], 2, 128, 16, seed=5)
    for b, n in enumerate((300, 77)):
        size = 2.0 ** torch.randint(-12, 13, (n, 1, 1), generator=book.g, device=DEV).float()
        v = (book.rows(n, 2, 128).float() * size)
        k = book.rows(n, 2, 128).float()
        book.cache.append(k[None], v[None], book.table[b:b + 1], book.lengths[b:b + 1])
        book.k[b], book.v[b] = held(k, fmt), held(v, fmt)
    run_attention(book, 3, 8)


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("S,Hq,Hkv,D,prefix", [(1, 8, 2, 128, 700), (1, 28, 7, 120, 17), (4, 8, 8, 64, 333),
                                               (3, 8, 1, 128, 1), (40, 8, 2, 128, 260)])
def test_shared_prefix(fmt, S, Hq, Hkv, D, prefix, path):
    book = Book(fmt, [0, 1, 100, 37, 64, S], Hkv, D, 16, prefix=prefix, seed=S + D, poison=True)
    q = book.query(S, Hq)
    for causal in (True, False):
        got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths, causal=causal)
        exact = attend(q.double(), book.k, book.v, causal, book.pk, book.pv)
        check(got, *exact, staged=True)
    # an empty prefix is plain attention; an empty table is the prefix alone
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = book.cache.prefix_attention(q, book.ptable, none, book.table, book.lengths)
    check(got, *attend(q.double(), book.k, book.v, True), staged=True)
    got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table[:, :0], torch.zeros_like(book.lengths))
    empty = [x[:0] for x in book.k]
    check(got, *attend(q.double(), empty, empty, False, book.pk, book.pv), staged=True)


def test_shared_prefix_of_a_large_batch():
    B, prefix = 70, 1500
    book = Book("q8", [i % 90 for i in range(B)], 2, 128, 64, prefix=prefix, seed=2)
    q = book.query(2, 16)
    got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths, max_length=100)
    check(got, *attend(q.double(), book.k, book.v, True, book.pk, book.pv))


def test_strided_queries_and_out():
    book = Book("q8", [100, 33], 2, 128, 16, seed=6)
    q = book.query(3, 8)
    want = book.cache.attention(q, book.table, book.lengths)
    turned = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    wide = torch.zeros((2, 3, 9, 130), dtype=torch.float16, device=DEV)
    wide[:, :, 1:, 1:129] = q
    out = torch.empty_like(q)
    for x in (turned, wide[:, :, 1:, 1:129]):
        assert torch.equal(book.cache.attention(x, book.table, book.lengths, out=out), want)
        assert torch.equal(out, want)
    # the bound of the lengths changes the split, not the result's meaning
    check(book.cache.attention(q, book.table, book.lengths, max_length=100),
          *attend(q.double(), book.k, book.v, True))
    q4.poll_device_error()


def test_masked_nan_and_held_nan():
    book = Book("f16", [20, 20], 1, 64, 16, seed=9, poison=True)
    k = torch.ones((1, 1, 1, 64), device=DEV).half()
    v = torch.full((1, 1, 1, 64), math.nan, device=DEV).half()
    book.cache.append(k, v, book.table[:1], book.lengths[:1])  # the last row of sequence 0
    q = book.query(2, 2)
    out = book.cache.attention(q, book.table, book.lengths)
    q4.poll_device_error()
    assert out[0, 1].isnan().all()      # sees it
    assert not out[1].isnan().any()
    exact = attend(q.double()[:, :1], [x[:19] for x in book.k], [x[:19] for x in book.v], True)
    check(out[:, :1], *exact)           # query 0 sees 19 rows


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("page", [16, 48, 4096])
def test_prefix_and_own_keys_both_long(fmt, page, path):
    # 160 rows of each sequence and 480 of the batch on hundreds of keys
    book = Book(fmt, [700, 263, 39], 2, 128, page, prefix=600, seed=page, poison=True)
    q = book.query(40, 8)
    for causal in (True, False):
        got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths, causal=causal)
        check(got, *attend(q.double(), book.k, book.v, causal, book.pk, book.pv), staged=True)
    got = book.cache.attention(q, book.table, book.lengths)
    check(got, *attend(q.double(), book.k, book.v, True), staged=True)
    for _ in range(3):
        assert torch.equal(got, book.cache.attention(q, book.table, book.lengths))
    odd = torch.zeros((3, 40, 8, 129), dtype=torch.float16, device=DEV)[..., 1:]
    odd.copy_(q)  # rows on no 16-byte boundary
    assert torch.equal(got, book.cache.attention(odd, book.table, book.lengths))


@pytest.mark.parametrize("fmt", ["q8", "q4", "f16"])
def test_many_rows_with_rows_of_any_size(fmt, path):
    # k from 2^-30 to 2^4 and v from 2^-12 to 2^17 (f32 rows; f16 caches hold up to 2^15): the
    # widened tiles keep them in f16's range by factors of two
    n, S = 600, 20
    book = Book(fmt, [n], 1, 128, 64, seed=21)
    g = book.g
    k = torch.randn((n, 1, 128), generator=g, device=DEV)
    k *= 2.0 ** torch.randint(-30, 3, (n, 1, 1), generator=g, device=DEV)
    hi = 15 if fmt == "f16" else 18
    v = torch.randn((n, 1, 128), generator=g, device=DEV).clamp(-1.9, 1.9)
    v *= 2.0 ** torch.randint(-12, hi - 1, (n, 1, 1), generator=g, device=DEV)
    book.cache.append(k[None], v[None], book.table, book.lengths)
    hk, hv = held(k, fmt), held(v, fmt)
    for Hq in (4, 1):  # 80 rows, then 20
        q = torch.randn((1, S, Hq, 128), generator=g, device=DEV).half()
        got = book.cache.attention(q, book.table, book.lengths)
        exact, mag, top = attend(q.double(), [hk], [hv], True)
        fits = exact.abs() < 65504
        assert fits.float().mean() > 0.9
        zero = torch.zeros((), dtype=torch.float64, device=DEV)
        # rows a factor 2^20 below the block's largest are rounded to steps of 2^-25 of 2^15
        check(torch.where(fits, got.double(), zero), torch.where(fits, exact, zero), mag, top, staged=True)


def test_many_rows_with_nan_and_bad_pages(path):
    n, S = 400, 30
    for fmt in ("f16", "q8", "q4"):
        book = Book(fmt, [n, n], 1, 128, 16, seed=31, poison=True)
        q = book.query(S, 4)
        want = book.cache.attention(q, book.table, book.lengths)
        # the newest row but 9 gets a NaN v: queries before it do not see it
        x = torch.ones((1, 1, 1, 128), device=DEV).half()
        bad = x.clone()
        bad[0, 0, 0, 77] = math.nan
        at = torch.tensor([n - 9], dtype=torch.int32, device=DEV)
        book.cache.append(x, bad, book.table[:1], at)
        got = book.cache.attention(q, book.table, book.lengths)
        q4.poll_device_error()
        assert torch.equal(got[1], want[1]) and torch.equal(got[0, :S - 10], want[0, :S - 10])
        assert got[0, S - 10:, :, 77].isnan().all()  # (the many-row kernels give the whole row NaN)
        # a page outside the cache holds nothing: the rest is as without its rows
        table = book.table.clone()
        table[1, 3] = 10 ** 6
        got = book.cache.attention(q[1:], table[1:], book.lengths[1:])
        reported()
        keep = [i for i in range(n) if i // 16 != 3]
        k, v = book.k[1][keep], book.v[1][keep]
        check(got, *attend(q[1:].double(), [k], [v], True), staged=True)


def test_more_sequences_than_threads(path):
    # 300 sequences, most of them empty or short, in one line of work
    lengths = [(7 * i) % 90 if i % 3 else 0 for i in range(300)]
    book = Book("q8", [max(lengths)], 2, 64, 16, seed=41)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    table = book.table.expand(300, -1)  # every sequence reads the same pages, to its own length
    q = torch.randn((300, 1, 4, 64), generator=book.g, device=DEV).half()
    got = book.cache.attention(q, table, n)
    ks, vs = [book.k[0][:x] for x in lengths], [book.v[0][:x] for x in lengths]
    check(got, *attend(q.double(), ks, vs, True))
    q = torch.randn((300, 33, 4, 64), generator=book.g, device=DEV).half()
    got = book.cache.attention(q, table, n)
    check(got, *attend(q.double(), ks, vs, True), staged=True)
    assert torch.equal(got, book.cache.attention(q, table, n))


# --------------------------------------------------------------------- bad pages, long caches

def reported():
    with pytest.raises(Bq4Error, match="EINVAL_ARG|device error"):
        q4.poll_device_error()


def test_bad_pages_and_lengths_are_reported():
    c = KVCache(4, 16, 2, 128, "q8", DEV)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    x = torch.ones((2, 2, 2, 128), device=DEV).half()
    q = torch.ones((2, 1, 4, 128), device=DEV).half()
    good = i32([0, 1], [2, 3])
    ones = torch.ones((2, 32, 2, 128), device=DEV).half()
    c.append(ones, ones, good, i32(32, 32))
    q4.poll_device_error()
    before = c.data.clone()
    for bad in (i32([4, 4], [-1, -1]), i32([2 ** 31 - 1, -2 ** 31], [4, 5])):
        c.append(x, x, bad, i32(20, 20))
        reported()
        k, v = c.read(bad, i32(32, 32), 32)
        reported()
        assert k.abs().sum() == 0 and v.abs().sum() == 0
        out = c.attention(q, bad, i32(32, 32))
        reported()
        assert out.abs().sum() == 0
        out = c.prefix_attention(q, bad[0], i32(32), good, i32(0, 32))
        reported()
        assert out[0].abs().sum() == 0 and torch.equal(out[1], torch.ones_like(out[1]))
    assert torch.equal(c.data, before)
    for n in (i32(33, 2), i32(-1, 2), i32(2 ** 31 - 1, 2)):
        c.read(good, n, 8)
        reported()
        c.attention(q, good, n)
        reported()
        c.prefix_attention(q, good[0], n[:1], good, i32(1, 1))
        reported()
    c.attention(q, good, i32(20, 32), max_length=16)  # above the caller's own bound
    reported()
    q4.poll_device_error()


def test_cache_past_four_gib(path):
    # 5 GiB of pages: offsets of the last ones pass 32 bits
    pages, page, H, D = 20480, 64, 16, 128
    c = KVCache(pages, page, H, D, "q8", DEV)
    assert c.data.numel() >= 2 ** 32 + 2 ** 30
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=DEV)
    n = torch.tensor([150], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    k = torch.randn((1, 150, H, D), generator=g, device=DEV).half()
    v = torch.randn((1, 150, H, D), generator=g, device=DEV).half()
    c.append(k, v, table, n)
    got = c.read(table, n, 150, dtype=torch.float32)
    assert torch.equal(got[0][0], held(k[0], "q8").float().transpose(0, 1))
    q = torch.randn((1, 2, H, D), generator=g, device=DEV).half()
    out = c.attention(q, table, n)
    check(out, *attend(q.double(), [held(k[0], "q8")], [held(v[0], "q8")], True))
    out = c.prefix_attention(q, table[0], n, table[:, :0], n * 0)
    check(out, *attend(q.double(), [held(k[0], "q8")[:0]], [held(v[0], "q8")[:0]], False, held(k[0], "q8"),
                       held(v[0], "q8")))
    assert int(c.data.view(pages, -1).any(1).sum()) == 3  # nothing went to another page


# --------------------------------------------------------------------- in use

def test_refusals():
    c = KVCache(4, 16, 2, 128, "q8", DEV)
    t = torch.zeros((1, 2), dtype=torch.int32, device=DEV)
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    x = torch.zeros((1, 1, 2, 128), device=DEV).half()
    q = torch.zeros((1, 1, 4, 128), device=DEV).half()
    for bad in (lambda: c.append(x.cpu(), x, t, n), lambda: c.append(x.double(), x.double(), t, n),
                lambda: c.append(x[..., :64], x[..., :64], t, n), lambda: c.append(x, x.float(), t, n),
                lambda: c.append(x, x, t.long(), n), lambda: c.append(x, x, t, n.cpu()),
                lambda: c.append(x, x, t[0], n),
                lambda: c.append(x, x, t, torch.cat([n, n])), lambda: c.append(x[:, :, :1], x[:, :, :1], t, n),
                lambda: c.read(t, n, -1), lambda: c.read(t, n, 1, dtype=torch.bfloat16),
                lambda: c.read(t, n, 1, starts=t[0]), lambda: c.attention(q.float(), t, n),
                lambda: c.attention(q[:, :, :3], t, n), lambda: c.attention(q, t, n, max_length=-1),
                lambda: c.attention(q, t, n, scale=math.nan), lambda: c.attention(q, t, n, out=q.float()),
                lambda: c.prefix_attention(q, t, n, t, n), lambda: c.prefix_attention(q, t[0], t[0], t, n)):
        with pytest.raises(Bq4Error):
            bad()
    e = torch.zeros((0, 2), dtype=torch.int32, device=DEV)  # empty batches and no tokens do nothing
    c.append(x[:0], x[:0], e, n[:0])
    assert c.read(e, n[:0], 3)[0].shape == (0, 2, 3, 128)
    assert c.read(t, n, 0)[0].numel() == 0
    assert c.attention(q[:0], e, n[:0]).shape == (0, 1, 4, 128)
    assert c.attention(q[:, :0], t, n).shape == (1, 0, 4, 128)
    q4.poll_device_error()


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
def test_prompt_then_decode_matches_contiguous_attention(fmt):
    # a prompt enters in two chunks, tokens follow one by one: each step's output is that of
    # f16.attention on rows read back (f32 output, so f16's half step and both kernels' errors)
    B, Hq, Hkv, D, page = 2, 8, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(1)
    c = KVCache(2 * 6, page, Hkv, D, fmt, DEV)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(2)).int().to(DEV).reshape(2, 6)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for S in (30, 21, 1, 1, 1, 3):
        lengths = lengths + S
        new = torch.randn((B, S, Hq + 2 * Hkv, D), generator=g, device=DEV).half()
        q, k, v = new.split([Hq, Hkv, Hkv], 2)
        c.append(k, v, table, lengths)
        out = c.attention(q, table, lengths)
        total = int(lengths[0])
        kk, vv = c.read(table, lengths, total, dtype=torch.float16)
        want = F.attention(q[:, -1:].transpose(1, 2), kk, vv).transpose(1, 2)
        # both round probabilities to f16 (2^-11 of a <= max |v|), K and V to f16 once more when
        # read (2^-11 of a score of at most 8, 2^-11 of v), the result here to f16
        bound = (2 ** -11 * (3 + 2 * 8) + 2 ** -9) * vv.abs().max().item()
        assert (out[:, -1:].float() - want).abs().max().item() <= bound
    q4.poll_device_error()


def test_streams_and_graphs():
    book = Book("q8", [300, 150, 40, 9], 2, 128, 16, prefix=200, seed=11)
    c = book.cache
    q = book.query(1, 8)
    new_k, new_v = book.rows(4, 2, 128)[:, None], book.rows(4, 2, 128)[:, None]
    lengths = book.lengths.clone()
    want0 = c.attention(q, book.table, lengths)
    # another stream than the current one's tensors, and two calls in flight on two streams
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = c.attention(q, book.table, lengths)
    with torch.cuda.stream(s2):
        b = c.prefix_attention(q, book.ptable, book.plen, book.table, lengths)
    torch.cuda.synchronize()
    assert torch.equal(a, want0)
    assert torch.equal(b, c.prefix_attention(q, book.ptable, book.plen, book.table, lengths))
    # captured: write the new row, then attend; replayed with lengths changed in place
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append(new_k, new_v, book.table, lengths)
        out = c.attention(q, book.table, lengths, max_length=19 * 16)
    with torch.cuda.graph(other):
        out2 = c.prefix_attention(q, book.ptable, book.plen, book.table, lengths, max_length=19 * 16)
    for step in (1, 2):
        lengths.copy_(book.lengths + step)
        graph.replay()
        torch.cuda.synchronize()
        ks = [torch.cat([x] + [held(new_k[i], "q8")] * step) for i, x in enumerate(book.k)]
        vs = [torch.cat([x] + [held(new_v[i], "q8")] * step) for i, x in enumerate(book.v)]
        check(out, *attend(q.double(), ks, vs, True))
        want = out.clone()
        # both graphs in flight at once: neither uses the other's workspace
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graph.replay()
        with torch.cuda.stream(s2):
            other.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out2, *attend(q.double(), ks, vs, True, book.pk, book.pv))
    q4.poll_device_error()


def test_many_rows_in_a_graph(path):
    book = Book("q4", [500, 300], 2, 128, 16, prefix=400, seed=13)
    c, S = book.cache, 24
    q = book.query(S, 8)
    lengths = book.lengths.clone()
    c.prefix_attention(q, book.ptable, book.plen, book.table, lengths)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = c.prefix_attention(q, book.ptable, book.plen, book.table, lengths)
        own = c.attention(q, book.table, lengths)
    for less in (0, 111, 300):
        lengths.copy_(book.lengths - less)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        ks = [x[:x.shape[0] - less] for x in book.k]
        vs = [x[:x.shape[0] - less] for x in book.v]
        check(out, *attend(q.double(), ks, vs, True, book.pk, book.pv), staged=True)
        check(own, *attend(q.double(), ks, vs, True), staged=True)


def test_same_bits_every_time():
    book = Book("q4", [1000, 5000, 20], 4, 128, 64, prefix=900, seed=12)
    q = book.query(1, 16)
    one = book.cache.attention(q, book.table, book.lengths)
    two = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths)
    for _ in range(5):
        assert torch.equal(one, book.cache.attention(q, book.table, book.lengths))
        assert torch.equal(two, book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths))


def test_more_tokens_than_a_cache_holds():
    # 2^31 - 8 rows given (one row, expanded), of which the cache keeps the last 5
    c = KVCache(2, 16, 1, 8, "f16", DEV)
    c.data.fill_(0x5A)
    before = c.data.clone()
    x = torch.randn((1, 1, 1, 8), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    many = x.expand(1, 2 ** 31 - 8, 1, 8)
    table = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    c.append(many, -many, table, torch.tensor([5], dtype=torch.int32, device=DEV))
    q4.poll_device_error()
    for got, want in zip(c.read(table, torch.tensor([5], dtype=torch.int32, device=DEV), 5), (x, -x)):
        assert torch.equal(got, want.half().expand(1, 1, 5, 8))
    half = c.data.numel() // 2
    assert torch.equal(c.data[:half], before[:half])  # page 0 stayed as it was


def test_more_warps_than_32_bits_of_threads():
    # one row of each of 2^26 + 8 sequences, k and v: 2^27 + 16 warps.  All but the last sequence are empty.
    B = 2 ** 26 + 8
    c = KVCache(2, 16, 1, 8, "f16", DEV)
    x = torch.randn((1, 1, 1, 8), generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).half()
    table = torch.ones((1, 1), dtype=torch.int32, device=DEV).expand(B, 1)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    lengths[-1] = 1
    c.append(x.expand(B, 1, 1, 8), -x.expand(B, 1, 1, 8), table, lengths)
    k, v = c.read(table[:1], lengths[-1:], 1)
    assert torch.equal(k[0, 0, 0], x[0, 0, 0]) and torch.equal(v[0, 0, 0], -x[0, 0, 0])
    outs = c.read(table, lengths, 1)
    q4.poll_device_error()
    for got, want in zip(outs, (x, -x)):
        assert torch.equal(got[-1, 0, 0], want[0, 0, 0])
        assert not got[:-1].any()


def test_many_keys_with_values_of_zero():
    # 40 million keys of k = v = 0 (rows that nothing wrote) and one with a value: the sum of their
    # probabilities, as large as a v scale of 0 lets them be, stays in f32
    n, page = 40_000_000, 65536
    c = KVCache(-(-n // page), page, 1, 8, "q8", DEV)
    table = torch.arange(c.pages, dtype=torch.int32, device=DEV)[None]
    length = torch.tensor([n], dtype=torch.int32, device=DEV)
    v = torch.linspace(-6e4, 6e4, 8, device=DEV)[None, None, None]
    c.append(torch.zeros_like(v), v, table, length)
    q = torch.ones((1, 1, 2, 8), device=DEV).half()
    exact = (held(v, "q8") / n).expand(1, 1, 2, 8)
    check(c.attention(q, table, length), exact, exact.abs(), 0.0)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_large_values_that_a_query_does_not_see(fmt, path):
    # f32 rows: the v of one of the newest tokens is far beyond f16, the others' are not.  Queries before it
    # do not see it; to the others it is there with the weight that its score gives it.
    n, S, late = 400, 64, 10
    book = Book(fmt, [n, n], 1, 128, 32, seed=51)
    for size in (1e12, 3e30):
        v = book.v[0].clone()
        x = torch.randn((1, 1, 1, 128), generator=book.g, device=DEV)
        big = x * size
        book.cache.append(x, big, book.table[:1], book.lengths[:1] - late + 1)
        k = book.k[0].clone()
        k[n - late], v[n - late] = held(x[0, 0], fmt), held(big[0, 0], fmt)
        q = book.query(S, 4)
        got = book.cache.attention(q, book.table, book.lengths)
        q4.poll_device_error()
        exact, mag, top = attend(q.double(), [k, book.k[1]], [v, book.v[1]], True)
        check(got[:, :S - late], exact[:, :S - late], mag[:, :S - late], top, staged=True)
        check(got[1:], exact[1:], mag[1:], top, staged=True)
        assert not got[0, S - late:].isfinite().all()
    # seen, with a weight of 2^-43: 2^40 in its place adds 2^-3 to every output
    k = torch.zeros((1, 1, 1, 128), device=DEV)
    k[..., 0] = -30 * 128 ** 0.5
    v = torch.full((1, 1, 1, 128), 2.0 ** 40, device=DEV)
    book.cache.append(k, v, book.table[:1], book.lengths[:1] - late + 1)
    k0, v0 = book.k[0].clone(), book.v[0].clone()
    k0[n - late], v0[n - late] = held(k[0, 0], fmt), held(v[0, 0], fmt)
    q = torch.zeros_like(book.query(S, 4))
    q[..., 0] = 1.0
    got = book.cache.attention(q, book.table, book.lengths)
    check(got, *attend(q.double(), [k0, book.k[1]], [v0, book.v[1]], True), staged=True)


def test_scales_that_are_refused():
    book = Book("q8", [20], 2, 128, 16)
    q = book.query(1, 4)
    for scale in (0.0, -0.0, -1.0, math.inf, -math.inf, math.nan, 1e39, 1e-60):
        with pytest.raises(Bq4Error, match="scale"):
            book.cache.attention(q, book.table, book.lengths, scale=scale)
        with pytest.raises(Bq4Error, match="scale"):
            book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths, scale=scale)
    run_attention(book, 1, 4, scale=1)


def test_a_bound_past_64_bits_is_the_page_tables():
    book = Book("q8", [40, 20], 2, 128, 16)
    q = book.query(1, 4)
    want = book.cache.attention(q, book.table, book.lengths)
    for bound in (2 ** 64 + 5, 2 ** 63, 2 ** 31):
        assert torch.equal(book.cache.attention(q, book.table, book.lengths, max_length=bound), want)
    q4.poll_device_error()


def test_a_short_prefix_keeps_the_row_tile():
    # 128 single tokens: the 512 rows that share 16 keys do not make the sequences' own 4 rows run in
    # tiles of 24, whose partial results the workspace would have to hold
    c = KVCache(4, 16, 8, 128, "q4", DEV)
    n = ctypes.c_size_t()

    def size(prefix):
        L.check(L.lib().bq4_cache_attention_workspace_size(ctypes.byref(c._c), 128, 1, 32, 2000, prefix, ctypes.byref(n)))
        return n.value

    assert size(16) < 1.5 * size(0)


def launches(call):
    before = L.lib().bq4_launch_count()
    out = call()
    return out, L.lib().bq4_launch_count() - before


def test_a_short_prefix_leaves_long_own_keys_to_the_many_row_kernels():
    book = Book("q8", [3000], 8, 128, 16, prefix=16, seed=61)
    q = book.query(200, 32)
    got, alone = launches(lambda: book.cache.attention(q, book.table, book.lengths))
    assert alone >= 2  # widening and products (the split kernel's call: itself and the join)
    check(got, *attend(q.double(), book.k, book.v, True), staged=True)
    got, n = launches(lambda: book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths))
    assert n == 5  # both for the prefix, both for the own keys, the join
    check(got, *attend(q.double(), book.k, book.v, True, book.pk, book.pv), staged=True)


def test_a_prefix_takes_no_launches_that_it_does_not_gain():
    book = Book("q8", [8] * 72, 8, 128, 16, prefix=16, seed=62)
    q = book.query(5, 32)
    got, n = launches(lambda: book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths))
    assert n == 2  # the split kernel and the join
    check(got, *attend(q.double(), book.k, book.v, True, book.pk, book.pv))


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("S,page", [(1, 16), (7, 48), (40, 64)])
def test_prefix_by_the_many_row_kernels_and_own_keys_by_the_split_kernel(fmt, S, page, monkeypatch):
    # the two run beside each other; the join takes both
    monkeypatch.setenv("BQ4_CACHE_TILE", "p")
    book = Book(fmt, [0, 1, 500, S, 77, 263], 2, 128, page, prefix=700, seed=S, poison=True)
    q = book.query(S, 8)
    for causal in (True, False):
        got, n = launches(lambda: book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths,
                                                              causal=causal))
        assert n == 4
        check(got, *attend(q.double(), book.k, book.v, causal, book.pk, book.pv), staged=True)
        assert torch.equal(got, book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths,
                                                            causal=causal))


@pytest.mark.parametrize("prefix", [0, 200])
def test_a_batch_of_prompts_in_slices(prefix, monkeypatch):
    # 37 sequences of 40 tokens on up to 8192 rows (the same pages, other lengths): their widened keys pass
    # the workspace that one run may have, so that the batch runs in slices, the last of another size
    monkeypatch.setenv("BQ4_CACHE_TILE", "1")
    B, S, H, n = 37, 40, 8, 8192
    book = Book("q8", [n], H, 128, 64, prefix=prefix, seed=71)
    lengths = [n - 211 * i for i in range(B - 2)] + [0, 17]
    table, t = book.table.expand(B, -1), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.randn((B, S, 2 * H, 128), generator=book.g, device=DEV).half()
    q = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # not contiguous

    def call():
        if prefix:
            return book.cache.prefix_attention(q, book.ptable, book.plen, table, t)
        return book.cache.attention(q, table, t)

    got, count = launches(call)
    slices = (count - (2 if prefix else 0)) // 3
    assert slices > 1 and B % slices and count == 3 * slices + (2 if prefix else 0)
    assert torch.equal(got, call())
    at = sorted({i for s in range(1, slices) for i in (s * -(-B // slices) - 1, s * -(-B // slices))} | {0, B - 2, B - 1})
    ks, vs = ([x[0][:lengths[i]] for i in at] for x in (book.k, book.v))
    check(got[at], *attend(q[at].double(), ks, vs, True, book.pk, book.pv), staged=True)


@pytest.mark.parametrize("S,B,Hkv,longest,prefix", [(128, 1, 8, 8192, 0), (64, 1, 8, 2432, 0), (1, 20, 2, 4000, 0),
                                                    (40, 3, 8, 3000, 0), (1, 60, 8, 2000, 16), (9, 12, 2, 1500, 700),
                                                    (200, 1, 8, 3000, 16)])
def test_a_workspace_serves_every_smaller_bound(S, B, Hkv, longest, prefix):
    # one workspace, sized for the largest bound, and calls with bounds below it (the lengths follow)
    book = Book("q8", [longest], Hkv, 128, 16, prefix=prefix, seed=S + B)
    c, lib, group = book.cache, L.lib(), 4
    q = torch.randn((B, S, group * Hkv, 128), generator=book.g, device=DEV).half()
    out = torch.empty_like(q)
    n = ctypes.c_size_t()
    L.check(lib.bq4_cache_attention_workspace_size(c._ref, B, S, group * Hkv, longest, prefix, ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device=DEV)
    strides = (ctypes.c_int64 * 3)(*q.stride()[:3])
    stream = torch.cuda.current_stream().cuda_stream
    bounds = sorted({max(1, longest * i // 97) for i in range(98)} | {longest - 128, longest - 1, 1, 127, 128, 129})
    for bound in bounds:
        lengths = torch.full((B,), bound, dtype=torch.int32, device=DEV)
        # the bound given, or all that a table of so many rows holds
        for width, given in ((book.table.shape[1], bound), (-(-bound // 16), 0)):
            if given == 0 and width * 16 > longest:
                continue
            seqs = L.CacheSequences(book.table.data_ptr(), 0, width, lengths.data_ptr(), B)
            tail = (q.data_ptr(), strides, S, group * Hkv, 1, 0.0, out.data_ptr(), ws.data_ptr(), n.value, stream)
            out.zero_()
            if prefix:
                L.check(lib.bq4_cache_prefix_attention(c._ref, book.ptable.data_ptr(), -(-prefix // 16),
                                                       book.plen.data_ptr(), ctypes.byref(seqs), given, *tail))
            else:
                L.check(lib.bq4_cache_attention(c._ref, ctypes.byref(seqs), given, *tail))
            if bound in (1, bounds[len(bounds) // 2], bounds[-1]):
                ks, vs = [book.k[0][:bound]] * B, [book.v[0][:bound]] * B
                check(out, *attend(q.double(), ks, vs, True, book.pk, book.pv), staged=True)
    q4.poll_device_error()
    with pytest.raises(Bq4Error, match="workspace"):  # a workspace that holds no plan is refused
        L.check(lib.bq4_cache_attention(c._ref, ctypes.byref(seqs), 0, *tail[:-2], 256, stream))


def test_the_environment_may_change_between_calls(monkeypatch):
    book = Book("q8", [700, 300], 2, 128, 16, prefix=100, seed=81)
    q = book.query(24, 8)
    for setting in ("0", "1", "p", "1", "0"):
        monkeypatch.setenv("BQ4_CACHE_TILE", setting)
        check(book.cache.attention(q, book.table, book.lengths), *attend(q.double(), book.k, book.v, True), staged=True)
        got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths)
        check(got, *attend(q.double(), book.k, book.v, True, book.pk, book.pv), staged=True)


def test_a_wide_table_without_a_bound():
    # 16 sequences of up to 40 rows in tables of 65536: neither the kernels for many rows of keys that
    # are not there, nor their workspace
    book = Book("q8", [40, 9, 31, 40] * 4, 8, 128, 16, seed=91)
    table = torch.zeros((16, 4096), dtype=torch.int32, device=DEV)
    table[:, :book.table.shape[1]] = book.table
    q = book.query(32, 32)
    torch.cuda.reset_peak_memory_stats()
    held_before = torch.cuda.memory_allocated()
    got, n = launches(lambda: book.cache.attention(q, table, book.lengths))
    assert n == 2 and torch.cuda.max_memory_allocated() - held_before < 2 ** 28
    check(got, *attend(q.double(), book.k, book.v, True))


# --------------------------------------------------------------------- calls of many rows, the whole chain

@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("D", [128, 120, 72, 64, 40])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_many_rows_written_and_read_back(fmt, D, src):
    # above the 16384 rows from which warps take several at a time; positions that begin inside their groups
    B, S, H, page = 3, 431, 7, 48
    g = torch.Generator(device=DEV).manual_seed(D)
    lengths = torch.tensor([S + 13, S, 100], dtype=torch.int32, device=DEV)  # the third: 331 rows fall below 0
    W = -(-(S + 13) // page)
    table = torch.randperm(3 * W + 2, generator=torch.Generator().manual_seed(1)).int().to(DEV)[:3 * W].reshape(3, W)
    c = KVCache(3 * W + 2, page, H, D, fmt, DEV)
    c.data.fill_(0x5A)
    k = (torch.randn((B, S, H, D), generator=g, device=DEV) * 3).to(src)
    v = torch.randn((B, H, S, D), generator=g, device=DEV).to(src).transpose(1, 2)
    c.append(k, v, table, lengths)
    odd = [torch.empty(B * S * H * D + 1, dtype=src, device=DEV)[1:].view(B, S, H, D).copy_(x) for x in (k, v)]
    d = KVCache(3 * W + 2, page, H, D, fmt, DEV)
    d.data.fill_(0x5A)
    d.append(*odd, table, lengths)  # rows on no 16-byte boundary
    assert torch.equal(c.data, d.data)
    for dtype in (torch.float32, torch.float16):
        for extra in (0, 5):  # starts of whole and of broken groups, some below 0
            got = c.read(table, lengths, S + 2 * extra, starts=lengths - S - extra, dtype=dtype)
            for x, y in zip((k, v), got):
                want = torch.zeros((B, H, S + 2 * extra, D), dtype=torch.float64, device=DEV)
                want[:, :, extra:extra + S] = held(x, fmt).transpose(1, 2)
                want[2, :, :S - 100 + extra] = 0.0  # positions below 0
                if extra:  # rows before the first written one hold anything
                    y[0, :, :extra] = 0.0
                assert torch.equal(y, want.float().to(dtype))
    got = c.read(table, lengths, S + 13, dtype=torch.float16)
    assert torch.equal(got[0][1, :, :S], held(k[1], fmt).transpose(0, 1).float().half())
    assert not got[1][1:, :, S:].any() and not got[1][2, :, 100:].any()
    q4.poll_device_error()


@pytest.mark.parametrize("fmt,D", [("q8", 128), ("q4", 128), ("f16", 120)])
def test_projection_cache_attention_and_next_linear(fmt, D, rng):
    # as a decoder layer runs them: projection with QK-norm and RoPE, k and v into the cache, attention of
    # the newest tokens, the next linear; a prompt, then tokens one by one, the last of them from a graph.
    # Each step is held to its own inputs in 64 bits: attention as above, linears to the library's 5e-3.
    B, Hq, Hkv, K = 2, 8, 2, 256
    N = (Hq + 2 * Hkv) * D
    w, s = gen_q4(K, N, 128, O.LAYOUT_ROW, rng)
    w2, s2 = gen_q4(1024, K, 128, O.LAYOUT_ROW, rng)
    dev = lambda a: torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(DEV)  # noqa: E731
    qkv_w = q4.PreparedQ4Weight(dev(w), dev(s), K, N, 128, O.LAYOUT_ROW, DEV)
    out_w = q4.PreparedQ4Weight(dev(w2), dev(s2), 1024, K, 128, O.LAYOUT_ROW, DEV)
    wide = O.unpack(w2, s2, 1024, K, 128, O.LAYOUT_ROW)
    gamma = torch.rand(D, device=DEV) + 0.5
    angle = torch.arange(128, device=DEV)[:, None] * (100.0 ** (-torch.arange(0, D, 2, device=DEV) / D))[None]
    cos, sin = (f(angle).repeat_interleave(2, 1).contiguous() for f in (torch.cos, torch.sin))
    c = KVCache(2 * 8, 16, Hkv, D, fmt, DEV)
    table = torch.randperm(16, generator=torch.Generator().manual_seed(2)).int().to(DEV).reshape(2, 8)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    ks, vs = [torch.zeros((0, Hkv, D), dtype=torch.float64, device=DEV)] * B, [torch.zeros((0, Hkv, D),
                                                                                      dtype=torch.float64, device=DEV)] * B

    def layer(x, cos, sin, S):
        y = qkv_w.linear_qk_norm_rope(x, Hq, Hkv, D, gamma_q=gamma, gamma_k=gamma, cos=cos, sin=sin,
                                      out_dtype=torch.float16)
        q, k, v = y.view(B, S, Hq + 2 * Hkv, D).split([Hq, Hkv, Hkv], 2)
        c.append(k, v, table, lengths)
        a = c.attention(q, table, lengths)
        padded = torch.nn.functional.pad(a.view(B * S, Hq * D), (0, 1024 - Hq * D))
        return q, k, v, a, out_w.linear_ex(padded, out_dtype=torch.float32)

    def verify(q, k, v, a, z):
        for b in range(B):
            ks[b], vs[b] = torch.cat([ks[b], held(k[b], fmt)]), torch.cat([vs[b], held(v[b], fmt)])
        check(a, *attend(q.double(), ks, vs, True), staged=True)
        flat = torch.nn.functional.pad(a.reshape(-1, Hq * D), (0, 1024 - Hq * D)).double().cpu().numpy()
        assert O.rel_frobenius(z.cpu().numpy(), flat @ wide) <= 5e-3

    at = 0
    for S in (37, 1, 5, 1):
        lengths += S
        x = torch.randn((B * S, K), device=DEV)
        verify(*layer(x, cos[at:at + S].repeat(B, 1), sin[at:at + S].repeat(B, 1), S))
        at += S
    x, ct, st = torch.randn((B, K), device=DEV), cos[:B].clone(), sin[:B].clone()
    lengths += 1
    layer(x, ct, st, 1)  # warm-up at the next position; the replays below write it again
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x, ct, st, 1)
    for step in range(3):
        lengths.fill_(at + step + 1)
        x.copy_(torch.randn((B, K), device=DEV))
        ct.copy_(cos[at + step].expand(B, -1)), st.copy_(sin[at + step].expand(B, -1))
        graph.replay()
        torch.cuda.synchronize()
        verify(*got)
    q4.poll_device_error()


@pytest.mark.parametrize("fmt", ["f16", "q4", "q8"])
def test_a_value_that_is_not_finite_stays_where_it_is(fmt, path):
    # one v value of NaN or infinity: what holds it (the value, a 4-bit block, an 8-bit row) reaches the
    # outputs of the queries that see it, there only, whichever kernels run; with keys on other CTAs,
    # a shared prefix, and D short of the padded head
    D, S, n, prefix = 120, 40, 900, 300
    book = Book(fmt, [n, 50], 2, D, 16, prefix=prefix, seed=101, poison=True)
    q = book.query(S, 8)
    for bad, d, at in ((math.nan, 77, n - 9), (math.inf, 3, n - 30), (-math.inf, 119, 200), (math.nan, 64, -50)):
        x, y = book.rows(1, 2, D)[None], book.rows(1, 2, D)[None].clone()
        y[0, 0, 1, d] = bad  # kv head 1
        if at < 0:           # a row of the prefix, which every query sees
            book.cache.append(x, y, book.ptable[None], book.plen + at + 1)
            at += prefix
            book.pk[at], book.pv[at] = held(x[0, 0], fmt), held(y[0, 0], fmt)
        else:
            book.cache.append(x, y, book.table[:1], book.lengths[:1] - n + at + 1)
            book.k[0][at], book.v[0][at] = held(x[0, 0], fmt), held(y[0, 0], fmt)
        for pre in (False, True):
            if pre:
                got = book.cache.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths)
            else:
                got = book.cache.attention(q, book.table, book.lengths)
            q4.poll_device_error()
            exact, mag, top = attend(q.double(), book.k, book.v, True, *((book.pk, book.pv) if pre else ()))
            # the formula's 0 * NaN of keys that a query does not see is not meant: recompute those
            for i in range(S):
                seen = [x[:len(x) - S + i + 1] for x in book.k], [x[:len(x) - S + i + 1] for x in book.v]
                e, m, _ = attend(q.double()[:, i:i + 1], *seen, False, *((book.pk, book.pv) if pre else ()))
                exact[:, i:i + 1], mag[:, i:i + 1] = e, m
            fine = exact.isfinite()
            assert torch.equal(got.isfinite(), fine)
            if fmt == "f16":
                assert torch.equal(got.isposinf(), exact.isposinf()) and torch.equal(got.isneginf(), exact.isneginf())
            zero = torch.zeros((), dtype=torch.float64, device=DEV)
            check(torch.where(fine, got.double(), zero), torch.where(fine, exact, zero), mag.nan_to_num(0, 0, 0), top,
                  staged=True)


def test_many_calls_at_once_on_several_streams(monkeypatch):
    # every plan, on four streams: the results of calls one by one
    book = Book("q8", [900, 300, 41], 2, 128, 16, prefix=500, seed=111)
    c, big, one = book.cache, book.query(60, 8), book.query(1, 8)
    calls = []
    for setting in ("0", "1", "p"):
        for q in (big, one):
            calls.append((setting, lambda q=q: c.attention(q, book.table, book.lengths)))
            calls.append((setting, lambda q=q: c.prefix_attention(q, book.ptable, book.plen, book.table, book.lengths)))
    want = []
    for setting, call in calls:
        monkeypatch.setenv("BQ4_CACHE_TILE", setting)
        want.append(call())
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for i, (setting, call) in enumerate(calls):
            monkeypatch.setenv("BQ4_CACHE_TILE", setting)
            with torch.cuda.stream(streams[(i + turn) % 4]):
                got.append((i, call()))
    torch.cuda.synchronize()
    q4.poll_device_error()
    for i, out in got:
        assert torch.equal(out, want[i])
