"""GPU tests of the low-bit operators against their 64-bit restatement (oracle/microscaled.py).

Quantised values are compared exactly: the scaling is a power of two and the one rounding is the
element's, so there is nothing to be near to.  Products and attention come with bounds counted
from the arithmetic, written at each helper."""
import math

import numpy as np
import pytest
import torch

from vdit import _lib
from vdit import fast_kernels as fk

from oracle import microscaled as mxo

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_error(clear=True) == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def host(t):
    return t.detach().cpu().double().numpy()


def same(a, b):
    """Equal values, NaN where the other has NaN."""
    return np.array_equal(a, b, equal_nan=True)


def rows(g, m, k, dtype=BF16, spread=3.0):
    """Normal rows whose blocks differ in size by powers of two."""
    x = torch.randn(m, k, generator=g, device=DEV)
    s = torch.exp2(torch.randn(m, k // 32, generator=g, device=DEV) * spread).repeat_interleave(32, 1)
    return (x * s).to(dtype)


# ----------------------------------------------------------------------------- 4-bit matrices

@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 1536), (2, 96), (33, 128), (127, 160), (129, 288), (300, 2080)])
def test_quantized_values_are_exact(m, k, dtype):
    x = rows(gen(m * 10007 + k), m, k, dtype)
    q = fk.quantize_mxfp4(x)
    want = mxo.values(host(x), 4)
    assert same(host(fk.dequantize_mxfp4(q, torch.float32)), want)
    assert same(host(fk.dequantize_mxfp4(q)), want)
    with np.errstate(over="ignore"):
        assert same(host(fk.dequantize_mxfp4(q, torch.float16)), want.astype(np.float16).astype(np.float64))
    code, neg, scale = mxo.quantize(host(x), 4)
    c = q.codes.cpu().numpy()
    got = np.stack([c & 15, c >> 4], -1).reshape(m, k)
    assert np.array_equal(got & 7, code) and np.array_equal((got >> 3).astype(bool), neg)
    # the scales in the block-scaled MMA's order, zero past the matrix
    s = q.scales.cpu().numpy().reshape(-(-m // 128), -(-k // 128), 32, 4, 4).transpose(0, 3, 2, 1, 4)
    s = s.reshape(-(-m // 128) * 128, -1)
    assert np.array_equal(s[:m, :k // 32], scale)
    assert not s[m:].any() and not s[:, k // 32:].any()


def test_quantize_special_blocks():
    """Zeros, subnormals, the largest numbers, halves between elements, NaN and infinities."""
    big = torch.finfo(torch.float32).max
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 0.2499999, 0.2500001, -0.25, -5, -7, -0.0])
    x = torch.zeros(12, 64)
    x[1, :32] = torch.arange(32) * 2.0 ** -149                       # subnormal fp32
    x[2, :32] = 2.0 ** -126 * torch.linspace(0, 1, 32)
    x[3, :32] = big * torch.linspace(-1, 1, 32)
    x[4, :16], x[4, 16:32] = grid, -grid
    x[5, :32] = torch.cat([grid, -grid]) * 2.0 ** 100
    x[6, 5], x[6, 40] = math.nan, 3.0
    x[7, 31], x[7, 33] = math.inf, -1.0
    x[8, 0], x[8, 63] = -math.inf, math.nan
    x[9] = 1e-3
    x[10, ::2] = -0.0
    x[11, :32] = 2.0 ** torch.arange(-16, 16).float()
    got = host(fk.dequantize_mxfp4(fk.quantize_mxfp4(x.to(DEV)), torch.float32))
    want = mxo.values(x.double().numpy(), 4)
    assert same(got, want)
    assert np.isnan(got[6, :32]).all() and (got[6, 32:] != 0).sum() == 1
    assert not got[0].any()


def test_quantize_strided_rows_and_empty():
    g = gen(5)
    wide = rows(g, 70, 512)
    for v in (wide[:, 128:288], wide[::3, 64:96], wide[5:6, 8:40], wide[7:8].expand(1, 512)):
        q = fk.quantize_mxfp4(v)
        assert same(host(fk.dequantize_mxfp4(q)), mxo.values(host(v), 4))
    with pytest.raises(RuntimeError, match="aligned"):
        fk.quantize_mxfp4(wide[:, 4:36])
    with pytest.raises(RuntimeError, match="aligned"):
        fk.quantize_mxfp4(torch.zeros(4, 36, dtype=BF16, device=DEV)[:, :32])
    e = fk.quantize_mxfp4(wide[:0])
    assert e.shape == (0, 512) and fk.dequantize_mxfp4(e).shape == (0, 512)
    assert fk.linear_mxfp4(e, fk.quantize_mxfp4(wide[:8])).shape == (0, 8)


# ----------------------------------------------------------------------------- linear

def check_linear(got, x, w, bias):
    """fp32 sums of k exact products in some order, each addition off by at most 2^-23 of the sum
    of magnitudes (a rounded one by 2^-24; the matrix units may truncate), then one rounding to
    bf16 (2^-8 of the value)."""
    want, mag = mxo.linear(host(x), host(w), None if bias is None else host(bias))
    acc = (x.shape[1] + 2) * 2.0 ** -23 * mag
    err = np.abs(host(got) - want)
    assert np.isfinite(host(got)).all()
    assert (err <= acc + 2.0 ** -8 * (np.abs(want) + acc) + 1e-38).all(), (err - acc).max()


@pytest.mark.parametrize("m,n,k", [
    (1, 8, 32), (1, 1536, 1536), (1, 200, 3840), (2, 264, 96), (5, 1000, 160), (7, 64, 2080), (8, 136, 352),
    (4, 136, 352), (3, 48, 16384), (5, 24, 13088), (1, 16, 70016), (9, 136, 352), (16, 1536, 256), (17, 72, 64), (33, 200, 1280), (127, 128, 128), (128, 192, 256), (129, 200, 288),
    (250, 1536, 1536), (300, 392, 1280), (1000, 776, 3840), (257, 7680, 160), (4101, 1536, 512), (20000, 384, 64)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear_matches_64_bits(m, n, k, with_bias):
    g = gen(m * 131 + n * 17 + k)
    x, w = rows(g, m, k, spread=1.0), rows(g, n, k, spread=1.0)
    bias = torch.randn(n, generator=g, device=DEV).to(BF16) if with_bias else None
    wq = fk.quantize_mxfp4(w)
    got = fk.linear_mxfp4(x, wq, bias)
    assert got.shape == (m, n) and got.dtype == BF16
    check_linear(got, x, w, bias)
    # quantised by the caller, or again: the same operands in the same order
    xq = fk.quantize_mxfp4(x)
    a = fk.linear_mxfp4(xq, wq, bias)
    check_linear(a, x, w, bias)
    assert torch.equal(a, fk.linear_mxfp4(xq, wq, bias)) and torch.equal(got, fk.linear_mxfp4(x, wq, bias))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m", [1, 6, 140])
def test_linear_takes_other_types(m, dtype):
    g = gen(m)
    x, w = rows(g, m, 320, dtype, spread=1.0), rows(g, 208, 320, dtype, spread=1.0)
    check_linear(fk.linear_mxfp4(x, fk.quantize_mxfp4(w)), x, w, None)


@pytest.mark.parametrize("m", [1, 4, 8, 40, 200])
def test_linear_spreads_nan_over_its_row_and_column_only(m):
    g = gen(90 + m)
    x, w = rows(g, m, 256, spread=1.0), rows(g, 136, 256, spread=1.0)
    x[m // 2, 70], w[11, 200], w[100, 3] = math.nan, math.inf, math.nan
    got = host(fk.linear_mxfp4(x, fk.quantize_mxfp4(w)))
    bad = np.zeros((m, 136), dtype=bool)
    bad[m // 2], bad[:, 11], bad[:, 100] = True, True, True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("m", [3, 150])
def test_linear_writes_its_part_of_out_only(m):
    g = gen(m)
    x, w = rows(g, m, 128, spread=1.0), rows(g, 72, 128, spread=1.0)
    wq = fk.quantize_mxfp4(w)
    out = torch.full((m + 3, 160), 7.0, dtype=BF16, device=DEV)
    view = out[1:, 16:]
    assert fk.linear_mxfp4(x, wq, out=view) is view
    assert torch.equal(out[1:m + 1, 16:88], fk.linear_mxfp4(x, wq))
    out[1:m + 1, 16:88] = 7
    assert (out == 7).all()


@pytest.mark.parametrize("m", [2, 130])
def test_linear_over_the_range_of_scales(m):
    """Blocks near both ends of the scale's range: large times small comes out in between."""
    x = torch.full((m, 96), 2.0 ** 100, dtype=BF16, device=DEV)
    w = torch.full((8, 96), -1.5 * 2.0 ** -98, dtype=BF16, device=DEV)
    x[:, 32:64], w[:, 64:] = 2.0 ** -120, 0
    want = -1.5 * 4 * 32                                     # the second block adds nothing that bf16 holds
    assert (fk.linear_mxfp4(x, fk.quantize_mxfp4(w)).float() == want).all()


@pytest.mark.parametrize("x_exp,w_exp", [(-120, 124), (124, -120), (-60, 62), (3, -3)])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 130])
def test_linear_of_large_weights_and_small_rows(m, x_exp, w_exp):
    """Ordinary products of operands near both ends of the range, and blocks of zeros between them."""
    g = gen(m + x_exp)
    x = (torch.randn(m, 160, generator=g, device=DEV).double() * 2.0 ** x_exp).to(BF16)
    w = (torch.randn(72, 160, generator=g, device=DEV).double() * 2.0 ** w_exp).to(BF16)
    x[:, 32:64], w[:, 64:96] = 0, 0
    check_linear(fk.linear_mxfp4(x, fk.quantize_mxfp4(w)), x, w, None)


# ----------------------------------------------------------------------------- cache

def filled(g, pages, page, heads, hd, bits):
    """A cache whose every slot is written, and the rows that went in."""
    c = fk.MxKvCache(pages, page, heads, hd, bits=bits, device=DEV)
    k, v = (torch.randn(c.slots, c.width, generator=g, device=DEV).to(BF16) for _ in range(2))
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    return c, k, v


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,hd,page", [(1, 32, 16), (3, 64, 16), (5, 96, 32), (12, 128, 64), (2, 128, 1024)])
def test_cache_holds_what_was_written(heads, hd, page, bits):
    g = gen(heads * 1000 + hd + page + bits)
    c = fk.MxKvCache(3, page, heads, hd, bits=bits, device=DEV)
    n = max(1, c.slots // 2)
    both = rows(g, n, 2 * c.width)                            # keys and values as halves of one matrix
    k, v = both[:, :c.width], both[:, c.width:]
    slots = torch.randperm(c.slots, generator=g, device=DEV)[:n]
    skip = torch.arange(n, device=DEV) % 5 == 3
    fk.kv_cache_write(c, k, v, torch.where(skip, -1 - slots, slots))
    want = [np.zeros((c.slots, c.width)) for _ in range(2)]
    at = slots[~skip].cpu().numpy()
    for w, t in zip(want, (k, v)):
        w[at] = mxo.values(host(t), bits)[~skip.cpu().numpy()]
    back = torch.randperm(c.slots, generator=g, device=DEV)
    for dtype in (BF16, torch.float32):
        got = fk.kv_cache_read(c, back, dtype)
        for a, b in zip(got, want):
            assert a.dtype == dtype and same(host(a), b[back.cpu().numpy()])   # untouched slots are zeros still
    back[::2] = -7
    for a in fk.kv_cache_read(c, back):
        assert not a[::2].any()
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    fk.kv_cache_write(c, k[:0], v[:0], none)
    assert fk.kv_cache_read(c, none)[0].shape == (0, c.width)


@pytest.mark.parametrize("bits", [4, 8])
def test_cache_special_blocks(bits):
    c = fk.MxKvCache(1, 16, 1, 64, bits=bits, device=DEV)
    x = torch.zeros(4, 64)
    x[0, 3], x[0, 40] = math.nan, 1.0
    x[1, 33], x[2, 0] = -math.inf, 2.0 ** -130
    x[3] = torch.cat([torch.linspace(440, 511, 32), torch.linspace(0.0, 0.05, 32)])
    x = x.to(BF16)
    fk.kv_cache_write(c, x.to(DEV), -x.to(DEV), torch.arange(4, device=DEV))
    k, v = fk.kv_cache_read(c, torch.arange(4, device=DEV), torch.float32)
    assert same(host(k), mxo.values(host(x), bits)) and same(host(v), mxo.values(host(-x), bits))


def test_slots_outside_the_cache_are_left_out_and_recorded():
    g = gen(1)
    c, k, v = filled(g, 2, 16, 2, 32, 8)
    before = [t.clone() for t in (c.k, c.v, c.k_scales, c.v_scales)]
    slots = torch.tensor([32, 1 << 40, -1], device=DEV)
    fk.kv_cache_write(c, k[:3], v[:3], slots)
    assert _lib.device_error(clear=True) == 0x4B56
    assert all(torch.equal(a, b) for a, b in zip(before, (c.k, c.v, c.k_scales, c.v_scales)))
    a, b = fk.kv_cache_read(c, torch.tensor([32, 3], device=DEV))
    assert _lib.device_error(clear=True) == 0x4B56
    assert not a[0].any() and not b[0].any() and same(host(a[1]), mxo.values(host(k[3:4]), 8)[0])


# ----------------------------------------------------------------------------- attention over the cache

def check_attend(got, q, c, k, v, table, lengths, bits, scale=None):
    """Scores are fp32 sums of head_dim products (each addition off by 2^-24 of the magnitudes'
    sum, the query's scaling by another), so a weight is off by e^d - 1 with d that error in
    natural units, and by 2^-21 of itself through two base-2 exponentials (2 ulp each and the
    rescaling); sums over n keys and their quotient add (n + 8) 2^-24.  The error of the weights
    counts twice, above and below the fraction; above it each weight is also rounded to f16
    (2^-11 of itself).  Then one rounding to bf16."""
    hk, hd, page = c.kv_heads, c.head_dim, c.page_size
    h = q.shape[1] // hd
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    kv, vv = (mxo.values(host(t), bits).reshape(c.slots, hk, hd) for t in (k, v))
    t, out = table.cpu().numpy(), host(got)
    for b, n in enumerate(lengths):
        at = np.arange(n)
        r = t[b][at // page].astype(np.int64) * page + at % page if n else at
        want, mag, unit = mxo.attend(host(q[b]).reshape(h, hd), kv[r], vv[r], scale)
        d = (hd + 4) * 2.0 ** -24 * unit
        rel = 2 * (np.expm1(d) + 2.0 ** -21) + 2.0 ** -11 + (n + 8) * 2.0 ** -24
        e = rel[:, None] * mag
        err = np.abs(out[b].reshape(h, hd) - want)
        assert (err <= e + 2.0 ** -8 * (np.abs(want) + e)).all(), (b, n, err.max())


def paged(g, c, lengths, spare=0):
    """A table of pages in no order, -1 past each sequence's last page."""
    need = [-(-n // c.page_size) for n in lengths]
    order = torch.randperm(c.pages, generator=g, device=DEV).to(torch.int32)
    assert sum(need) <= c.pages
    t = torch.full((len(lengths), max(max(need), 1) + spare), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t


def i32(vals):
    return torch.tensor(vals, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hk,grp,hd,page", [(2, 1, 32, 16), (3, 2, 64, 16), (5, 1, 96, 32), (12, 1, 128, 64),
                                            (2, 3, 128, 16), (1, 4, 96, 128), (2, 5, 64, 32), (1, 9, 128, 16),
                                            (4, 4, 96, 16)])
def test_attention_over_ragged_pages(hk, grp, hd, page, bits):
    g = gen(hk * 100 + grp * 10 + hd + page + bits)
    lengths = [1, 0, page, page + 1, 3 * page - 1, 130, 517]
    c, k, v = filled(g, sum(-(-n // page) for n in lengths) + 2, page, hk, hd, bits)
    q = (torch.randn(len(lengths), hk * grp * hd, generator=g, device=DEV) * 2).to(BF16)
    t = paged(g, c, lengths, spare=2)
    got = fk.attention_1q_cached(q, c, t, i32(lengths))
    assert not got[1].any()
    check_attend(got, q, c, k, v, t, lengths, bits)
    assert torch.equal(got, fk.attention_1q_cached(q, c, t, i32(lengths)))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch,n,hk,grp,hd,page", [(1, 4101, 12, 1, 128, 64), (1, 20000, 2, 1, 96, 128),
                                                    (40, 300, 3, 2, 64, 16), (300, 33, 2, 1, 32, 32)])
def test_attention_splits_and_batches(batch, n, hk, grp, hd, page, bits):
    g = gen(n + batch)
    lengths = [max(0, n - (i * 37) % (n + 1)) for i in range(batch)]
    c, k, v = filled(g, sum(-(-m // page) for m in lengths) + 1, page, hk, hd, bits)
    wide = torch.randn(batch, hk * grp * hd + 64, generator=g, device=DEV).to(BF16)
    q = wide[:, 64:]                                          # a strided view
    t = paged(g, c, lengths)
    check_attend(fk.attention_1q_cached(q, c, t, i32(lengths)), q, c, k, v, t, lengths, bits)


def test_attention_peaked_scores_and_scale():
    """Scores hundreds apart, growing along the keys (the running maximum moves all the time) and
    falling; a given softmax scale, also a negative one."""
    g = gen(3)
    c = fk.MxKvCache(40, 16, 1, 64, bits=8, device=DEV)
    ramp = torch.linspace(-4, 4, c.slots, device=DEV)[:, None]
    v = torch.randn(c.slots, 64, generator=g, device=DEV).to(BF16)
    k = (ramp * torch.ones(1, 64, device=DEV)).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    q = torch.ones(1, 64, device=DEV, dtype=BF16) * 4
    t = torch.arange(40, dtype=torch.int32, device=DEV)[None]
    for scale in (None, 1.0, -1.0, 0.0):
        for table in (t, t.flip(1)):
            got = fk.attention_1q_cached(q, c, table.contiguous(), i32([c.slots]), scale)
            check_attend(got, q, c, k, v, table, [c.slots], 8, scale)


def test_attention_nan_stays_in_its_sequence_and_head():
    g = gen(4)
    c, k, v = filled(g, 8, 16, 2, 64, 8)
    k[20, 70], v[100, 3] = math.nan, math.inf                 # head 1 of page 1, head 0 of page 6
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    q = torch.randn(4, 128, generator=g, device=DEV).to(BF16)
    t = i32([[0, 1], [2, 3], [6, 7], [1, 0]])
    got = host(fk.attention_1q_cached(q, c, t, i32([32, 32, 32, 4]))).reshape(4, 2, 64)
    bad = np.isnan(got)
    assert bad[0, 1].all() and not bad[0, 0].any() and not bad[1].any()
    assert bad[2, 0, :32].all() and not bad[2, 0, 32:].any() and not bad[2, 1].any()
    assert not bad[3].any()                                   # the NaN lies past this length


def test_attention_with_infinities_in_queries():
    """Scores of +-inf and NaN as a softmax has them: one at -inf weighs nothing, all at -inf or any
    at +inf or NaN give NaN; other queries of the same key head are untouched."""
    g = gen(8)
    c = fk.MxKvCache(4, 16, 1, 32, bits=8, device=DEV)
    k = torch.randn(64, 32, generator=g, device=DEV).to(BF16)
    k[:, 0] = 1.0
    k[5, 0] = -1.0
    v = torch.randn(64, 32, generator=g, device=DEV).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(64, device=DEV))
    q = torch.randn(4, 32, generator=g, device=DEV).to(BF16)
    q[:3, 1:] = 0                                             # 0 * finite: the score is the first channel's
    q[0, 0], q[1, 0], q[2, 0] = math.inf, -math.inf, math.nan
    t = i32([[0, 1, 2, 3]])
    got = fk.attention_1q_cached(q.reshape(1, 128), c, t, i32([64]))
    o = host(got).reshape(4, 32)
    assert np.isnan(o[:3]).all() and not np.isnan(o[3]).any()
    # key 5 alone is at -inf for +inf and the other way round: 63 keys at +inf, then one at +inf
    q2 = q.clone()
    q2[0, 0], q2[1, 0] = -math.inf, -math.inf
    k[:, 0] = 1.0
    fk.kv_cache_write(c, k, v, torch.arange(64, device=DEV))  # every score -inf
    o = host(fk.attention_1q_cached(q2.reshape(1, 128), c, t, i32([64]))).reshape(4, 32)
    assert np.isnan(o[:3]).all() and not np.isnan(o[3]).any()
    check_attend(got[:, 96:], q[3:], c, _first_key_negative(k), v, t, [64], 8)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [32, 128])
def test_attention_weights_have_the_accuracy_of_32_bits(hd, bits):
    """Two kinds of keys whose values cancel: what is left of the output shows the weights' own error,
    which the output's rounding hides elsewhere.  32 sequences of 64 keys, the weight of the first kind
    another one in each; a last key takes the rest of the sum, as near as its few bits allow.  The bound
    is that of ``check_attend`` with weights off by 2^-21 of themselves, not by f16's 2^-11."""
    n, b = 64, 32
    c = fk.MxKvCache(b * n // 16, 16, 1, hd, bits=bits, device=DEV)
    x = torch.linspace(-2.5, -0.05, b).to(BF16)
    q = torch.zeros(b, hd, dtype=BF16)
    q[:, 0] = x
    k, v = (torch.zeros(b, n, hd, dtype=BF16) for _ in range(2))
    w = torch.exp(x.double())
    first = (n / (1 + w)).round().long().clamp(1, n - 2)      # keys of the first kind: first * w ~ n - first
    for i in range(b):
        k[i, :first[i], 0] = 1.0
        v[i, :first[i]], v[i, first[i]:] = 1.0, -1.0
        v[i, n - 1] = float(n - 1 - first[i] - first[i] * w[i])
    k, v = (t.reshape(c.slots, hd).to(DEV) for t in (k, v))
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    t = torch.arange(b * n // 16, dtype=torch.int32, device=DEV).view(b, n // 16)
    got = host(fk.attention_1q_cached(q.to(DEV), c, t, i32([n] * b), 1.0))
    kv, vv = (mxo.values(host(t), bits).reshape(b, n, 1, hd) for t in (k, v))
    for i in range(b):
        want, mag, unit = mxo.attend(host(q[i]).reshape(1, hd), kv[i], vv[i], 1.0)
        assert np.abs(want).max() < 0.05 * mag.max()
        rel = 2 * (np.expm1((hd + 4) * 2.0 ** -24 * unit) + 2.0 ** -21) + 2.0 ** -21 + (n + 8) * 2.0 ** -24
        e = rel[:, None] * mag
        err = np.abs(got[i].reshape(1, hd) - want)
        assert (err <= e + 2.0 ** -8 * (np.abs(want) + e)).all(), (i, err.max(), e.max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("key_exp,query_exp", [(110, -108), (-118, 119), (118, -118), (60, -58), (0, 0)])
@pytest.mark.parametrize("grp", [1, 5])
def test_attention_over_the_range_of_keys_and_queries(grp, key_exp, query_exp, bits):
    """Ordinary scores from keys and queries near both ends of the range."""
    g = gen(grp + bits + key_exp)
    c = fk.MxKvCache(20, 16, 2, 64, bits=bits, device=DEV)
    k = (torch.randn(c.slots, 128, generator=g, device=DEV).double() * 2.0 ** key_exp).to(BF16)
    v = torch.randn(c.slots, 128, generator=g, device=DEV).to(BF16)
    q = (torch.randn(2, grp * 128, generator=g, device=DEV).double() * 2.0 ** query_exp).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    t = torch.randperm(20, generator=g, device=DEV).to(torch.int32).view(1, 20).expand(2, 20)
    got = fk.attention_1q_cached(q, c, t, i32([c.slots, 77]))
    assert torch.isfinite(got).all()
    check_attend(got, q, c, k, v, t, [c.slots, 77], bits)


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_scores_up_to_the_range_of_32_bits(bits):
    """Queries of ones over keys of 2^110: products of a key pass 2^117, the largest score takes all."""
    g = gen(bits)
    c = fk.MxKvCache(8, 16, 1, 128, bits=bits, device=DEV)
    k = (torch.randn(c.slots, 128, generator=g, device=DEV).double() * 2.0 ** 110).to(BF16)
    v = torch.randn(c.slots, 128, generator=g, device=DEV).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    got = host(fk.attention_1q_cached(torch.ones(1, 128, device=DEV, dtype=BF16), c, i32([list(range(8))]), i32([c.slots])))
    score = np.sort(mxo.values(host(k), bits).sum(1))
    best = mxo.values(host(k), bits).sum(1).argmax()
    assert score[-1] - score[-2] > 1e-3 * score[-1]           # far more than fp32 sums are off by
    want = mxo.values(host(v), bits)[best]                    # 8-bit and 4-bit values are bf16 values
    assert np.array_equal(got[0], want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch,n,grp", [(1, 4, 1), (1, 200, 5), (1, 4101, 1), (1, 20000, 2), (300, 130, 1)])
def test_attention_sums_of_values_past_the_range(batch, n, grp, bits):
    """Values of one sign near bf16's largest: their sum over the keys is out of range, their mean is not.
    One warp, one CTA, a cluster and the second kernel join the parts."""
    g = gen(n + grp + bits)
    c = fk.MxKvCache(-(-n // 16), 16, 2, 64, bits=bits, device=DEV)
    k = torch.randn(c.slots, 128, generator=g, device=DEV).to(BF16)
    v = ((torch.rand(c.slots, 128, generator=g, device=DEV) * 0.7 + 1).double() * 2.0 ** 126).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(c.slots, device=DEV))
    q = torch.randn(batch, grp * 128, generator=g, device=DEV).to(BF16)
    t = torch.randperm(c.pages, generator=g, device=DEV).to(torch.int32)[None].expand(batch, c.pages)
    got = fk.attention_1q_cached(q, c, t, i32([n] * batch))
    assert torch.isfinite(got).all()
    for b in {0, batch - 1}:
        check_attend(got[b:b + 1], q[b:b + 1], c, k, v, t[b:b + 1], [n], bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("order", ["first", "last", "each group"])
def test_attention_huge_values_without_weight(order, bits):
    """Values 2^90 times the others at keys whose weight is nothing beside the others': they must not
    take the others' precision, whether they come first (with the largest score so far), last or
    once in every group of keys; 300 sequences, so that a warp has several groups."""
    g = gen(15 + bits)
    c = fk.MxKvCache(125, 16, 2, 64, bits=bits, device=DEV)
    n = c.slots
    k = torch.randn(n, 128, generator=g, device=DEV).to(BF16)
    v = torch.randn(n, 128, generator=g, device=DEV).to(BF16)
    at = {"first": slice(0, 40), "last": slice(n - 40, n), "each group": slice(7, n, 32)}[order]
    score = 700.0 if order == "each group" else torch.linspace(0, 700, n, device=DEV)[:, None]
    k[:, ::64] = torch.as_tensor(score, device=DEV).to(BF16).expand(n, 2) if order != "last" else 700.0
    k[at, ::64] = 0.0
    v[at] = (v[at].float() * 2.0 ** 90).to(BF16)
    fk.kv_cache_write(c, k, v, torch.arange(n, device=DEV))
    q = torch.randn(300, 128, generator=g, device=DEV).to(BF16)
    q[:, ::64] = 8.0                                          # scores up to 700 apart (scale 1/8)
    t = torch.arange(125, dtype=torch.int32, device=DEV)[None].expand(300, 125)
    got = fk.attention_1q_cached(q, c, t, i32([n] * 300))
    for b in (0, 150, 299):
        check_attend(got[b:b + 1], q[b:b + 1], c, k, v, t[b:b + 1], [n], bits)


def _first_key_negative(k):
    k = k.clone()
    k[5, 0] = -1.0
    return k


def test_attention_one_table_for_all_and_bad_pages():
    g = gen(6)
    c, k, v = filled(g, 6, 32, 3, 96, 4)
    q = torch.randn(5, 3 * 96, generator=g, device=DEV).to(BF16)
    shared = i32([[4, 1, 5]]).expand(5, 3)                    # row stride 0: one prefix for all
    lengths = [96, 40, 1, 0, 64]
    check_attend(fk.attention_1q_cached(q, c, shared, i32(lengths)), q, c, k, v, shared, lengths, 4)
    # a page that is not there: its keys are left out; lengths past the table end with it
    t = i32([[4, 6, 5], [4, -1, 5], [4, 1, 5], [4, 1, 5], [6, -2, 3]])
    got = fk.attention_1q_cached(q, c, t, i32([96, 96, 1000, -3, 64]))
    assert _lib.device_error(clear=True) == 0x4B56
    two, three = i32([[4, 5]] * 5), i32([[4, 1, 5]] * 5)
    check_attend(got[:2], q[:2], c, k, v, two, [64, 64], 4)
    check_attend(got[2:3], q[2:3], c, k, v, three, [96], 4)
    assert not got[3:].any()


# ----------------------------------------------------------------------------- past 2^32

def test_cache_past_four_gigabytes():
    """Keys and values of 4.9 GB each: slots and pages at the end are where they should be."""
    g = gen(13)
    c = fk.MxKvCache(25000, 128, 12, 128, bits=8, device=DEV)
    assert c.k.numel() > 2 ** 32
    n = 300
    slots = c.slots - 1 - torch.randperm(n, generator=g, device=DEV)
    k, v = (torch.randn(n, c.width, generator=g, device=DEV).to(BF16) for _ in range(2))
    fk.kv_cache_write(c, k, v, slots)
    back = fk.kv_cache_read(c, slots)
    assert same(host(back[0]), mxo.values(host(k), 8)) and same(host(back[1]), mxo.values(host(v), 8))
    assert not c.k[:c.pages // 2].any() and not c.k[c.pages // 2:-3].any()
    q = torch.randn(1, c.width, generator=g, device=DEV).to(BF16)
    t = i32([[24998, 24999]])                                 # the last 256 slots, in order
    tail = torch.arange(c.slots - 256, c.slots, device=DEV)
    place = torch.empty(n, dtype=torch.int64, device=DEV)
    place[c.slots - 1 - slots] = torch.arange(n, device=DEV)
    rows_in = place[c.slots - 1 - tail]
    small = fk.MxKvCache(2, 128, 12, 128, bits=8, device=DEV)
    fk.kv_cache_write(small, k[rows_in], v[rows_in], torch.arange(256, device=DEV))
    assert torch.equal(fk.attention_1q_cached(q, c, t, i32([256])),
                       fk.attention_1q_cached(q, small, i32([[0, 1]]), i32([256])))


def test_matrices_past_two_gigaelements():
    g = gen(14)
    m, k = 70000, 32768
    x = torch.zeros(m, k, dtype=BF16, device=DEV)
    tail = rows(g, 130, k)
    x[-130:] = tail
    q = fk.quantize_mxfp4(x)
    del x
    y = fk.dequantize_mxfp4(q)
    assert same(host(y[-130:]), mxo.values(host(tail), 4)) and not y[:-130].any()
    del y, q
    m, n = 300000, 7680
    x, w = rows(g, m, 32, spread=1.0), rows(g, n, 32, spread=1.0)
    out = fk.linear_mxfp4(x, fk.quantize_mxfp4(w))
    assert out.numel() > 2 ** 31
    check_linear(out[-200:], x[-200:], w, None)
    check_linear(out[:200], x[:200], w, None)


# ----------------------------------------------------------------------------- together

def test_a_served_block_step_by_step():
    """What a server of one block's attention does: the K/V linear in 4 bits, its rows written into the
    cache as they come, one query per sequence over them, the output linear; and the cached rows
    read back for the many-query attention."""
    g = gen(11)
    heads, hd, page = 4, 64, 16
    d = heads * hd
    wkv, wo = (torch.randn(n, d, generator=g, device=DEV).to(BF16) * 0.05 for n in (2 * d, d))
    qkv, qo = fk.quantize_mxfp4(wkv), fk.quantize_mxfp4(wo)
    c = fk.MxKvCache(12, page, heads, hd, bits=8, device=DEV)
    table = torch.randperm(12, generator=g, device=DEV).to(torch.int32).view(3, 4)
    lengths = [0, 0, 0]
    k_in, v_in = (torch.zeros(c.slots, d, dtype=BF16, device=DEV) for _ in range(2))
    for step in range(3):
        new = [17, 1, 20] if step == 0 else [1, 1, 1]
        if step == 2:
            new = [1, 0, 1]                                   # one sequence pauses
        x = torch.randn(sum(new), d, generator=g, device=DEV).to(BF16)
        kv = fk.linear_mxfp4(x, qkv)
        at = [(b, lengths[b] + i) for b in range(3) for i in range(new[b])]
        slots = torch.tensor([int(table[b, i // page]) * page + i % page for b, i in at], device=DEV)
        fk.kv_cache_write(c, kv[:, :d], kv[:, d:], slots)
        k_in[slots], v_in[slots] = kv[:, :d], kv[:, d:]
        lengths = [a + b for a, b in zip(lengths, new)]
        q = torch.randn(3, d, generator=g, device=DEV).to(BF16)
        o = fk.attention_1q_cached(q, c, table, i32(lengths))
        check_attend(o, q, c, k_in, v_in, table, lengths, 8)
        y = fk.linear_mxfp4(o, qo)
        check_linear(y, o, wo, None)
    # the same sequence through the many-query attention, which takes bf16 rows
    n = lengths[0]
    r = torch.tensor([int(table[0, i // page]) * page + i % page for i in range(n)], device=DEV)
    k, v = fk.kv_cache_read(c, r)
    assert same(host(k), mxo.values(host(k_in[r]), 8)) and same(host(v), mxo.values(host(v_in[r]), 8))


def test_captured_and_on_another_stream():
    """One graph of the whole step replayed on new inputs, beside a second graph of the same calls
    and eager calls on another stream: each has its own workspace."""
    g = gen(12)
    heads, hd, page, d = 3, 128, 16, 384
    wq = fk.quantize_mxfp4(torch.randn(d, d, generator=g, device=DEV).to(BF16) * 0.05)

    def step(s):
        fk.kv_cache_write(s["c"], s["k"], s["v"], s["slots"])
        o = fk.attention_1q_cached(s["q"], s["c"], s["t"], s["n"])
        return o, fk.linear_mxfp4(o, wq), fk.kv_cache_read(s["c"], s["slots"])[0]

    def state(seed):
        gg = gen(seed)
        s = {n: torch.randn(r, d, generator=gg, device=DEV).to(BF16) for n, r in (("k", 60), ("v", 60), ("q", 2))}
        s["c"] = fk.MxKvCache(80, page, heads, hd, device=DEV)
        s["slots"] = torch.randperm(60, generator=gg, device=DEV)
        s["t"] = torch.arange(80, dtype=torch.int32, device=DEV).view(2, 40)
        s["n"] = i32([60, 7])
        return s

    states, graphs = [state(1), state(2)], []
    step(states[0])
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    side = torch.cuda.Stream()
    for seed in (21, 22, 23):
        fresh = [state(seed), state(seed + 100)]
        for s, f in zip(states, fresh):
            f["n"] = i32([60 - seed % 20, 7 * seed])           # past the last written slot: zeros
            for n in ("k", "v", "q", "slots", "n"):
                s[n].copy_(f[n])
            s["c"].k.zero_()
            s["c"].v.zero_()
            s["c"].k_scales.zero_()
            s["c"].v_scales.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = [step(f) for f in fresh]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_workspaces_of_calls_in_flight_at_once():
    """Two captured graphs replayed on two streams beside eager calls on a third, at sizes where the attention's
    splits and the linear's quantised rows go through workspaces: none sees another's."""
    from vdit import microscaled
    heads, hd, page, pages, d = 2, 128, 64, 320, 256
    assert microscaled._attend_workspace(2, 2 * heads, heads, hd, pages, page) > 0     # a second kernel joins
    assert microscaled._dense_workspace(300, d) > 0                                    # rows quantised, then multiplied

    def state(seed):
        g = gen(seed)
        c, _, _ = filled(g, pages, page, heads, hd, 8)
        return {"c": c, "q": torch.randn(2, 2 * d, generator=g, device=DEV).to(BF16),
                "t": torch.stack([torch.randperm(pages, generator=g, device=DEV) for _ in range(2)]).to(torch.int32),
                "n": i32([pages * page - seed, 9000 + seed]), "x": torch.randn(300, d, generator=g, device=DEV).to(BF16),
                "w": fk.quantize_mxfp4(torch.randn(512, d, generator=g, device=DEV).to(BF16))}

    def step(s):
        out = []
        for _ in range(6):
            out.append(fk.attention_1q_cached(s["q"], s["c"], s["t"], s["n"]))
            out.append(fk.linear_mxfp4(s["x"], s["w"]))
            out.append(fk.linear_mxfp4(out[-1][:, d:], s["w"]))
        return out

    states = [state(1), state(2), state(3)]
    want = [[t.clone() for t in step(s)[:3]] for s in states]
    torch.cuda.synchronize()
    graphs = []
    for s in states[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for _, out in graphs:
            for t in out:
                t.zero_()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [graphs[0][1], graphs[1][1], None]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        with torch.cuda.stream(streams[2]):
            got[2] = step(states[2])
        torch.cuda.synchronize()
        for out, w in zip(got, want):
            assert all(torch.equal(t, w[i % 3]) for i, t in enumerate(out))


@pytest.mark.parametrize("rows", [3, 700, 9000])
def test_each_call_waits_for_the_one_before(rows):
    """Every call reads what the call before it wrote (a kernel, a copy or another stream's kernel), in
    place and on the same buffers each time, eagerly and captured: as with a wait on the host between."""
    g = gen(31)
    heads, hd, page, d = 2, 64, 64, 128
    xs = torch.randn(6, rows, d, generator=g, device=DEV).to(BF16)
    wq = fk.quantize_mxfp4(torch.randn(256, d, generator=g, device=DEV).to(BF16))
    perm = torch.randperm(rows, generator=g, device=DEV)
    pages = -(-rows // page)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).flip(0).contiguous()[None]
    side = torch.cuda.Stream()

    def chain(b, bias, sync):
        out = []
        for i in range(xs.shape[0]):
            wait = torch.cuda.synchronize if sync else (lambda: None)
            b["x"].copy_(xs[i])
            wait()
            r = fk.dequantize_mxfp4(fk.quantize_mxfp4(b["x"]), dtype=BF16)
            wait()
            fk.kv_cache_write(b["c"], r, b["x"], b["slots"])
            wait()
            k, v = fk.kv_cache_read(b["c"], b["slots"])
            wait()
            b["slots"].copy_(perm[b["slots"]])               # the next write goes elsewhere
            wait()
            fk.kv_cache_write(b["c"], v, k, b["slots"])
            wait()
            o = fk.attention_1q_cached(k[:1], b["c"], table, b["n"])
            wait()
            fork = torch.cuda.current_stream()
            side.wait_stream(fork)
            with torch.cuda.stream(side):
                y = fk.linear_mxfp4(v, wq, bias)
            fork.wait_stream(side)
            wait()
            b["x"].copy_(y[:, :d])
            wait()
            q = fk.quantize_mxfp4(b["x"])
            wait()
            z = fk.linear_mxfp4(q, wq, y[0])                 # its bias is a product's row
            wait()
            rows_q = fk.quantize_mxfp4(y)
            wait()
            row = fk.dequantize_mxfp4(rows_q, dtype=BF16)[0]
            wait()
            u = fk.linear_mxfp4(b["x"], wq, row)             # its bias is the last call's
            wait()
            b["n"].sub_(1).clamp_(min=1)
            out += [r, k, v, o, y, z, u]
        return out

    def fresh():
        return {"x": torch.empty(rows, d, dtype=BF16, device=DEV), "slots": torch.arange(rows, device=DEV),
                "c": fk.MxKvCache(pages, page, heads, hd, device=DEV), "n": i32([rows])}

    bias = torch.randn(256, generator=g, device=DEV).to(BF16)
    want = chain(fresh(), bias, True)
    torch.cuda.synchronize()
    for _ in range(5):
        got = chain(fresh(), bias, False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))
    b, graph = fresh(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(b, bias, False)
    for _ in range(5):
        start = fresh()
        b["slots"].copy_(start["slots"])
        b["n"].copy_(start["n"])
        for name in ("k", "v", "k_scales", "v_scales"):
            getattr(b["c"], name).copy_(getattr(start["c"], name))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


# ----------------------------------------------------------------------------- on the model's path

def _model(dim=256, depth=3, cond_depth=2, n=700, side=8):
    from oracle import model as om
    from tests.golden.make_golden import shell_voxels
    from vdit.model import LatDitModel
    cfg = om.ModelConfig(dim=dim, head_dim=128, depth=depth, cond_depth=cond_depth, res=64, patch_size=256)
    p = om.init_params(cfg, 5, weight_std=0.03, bias_std=0.02, scale_jitter=0.1)
    mc = {"dim": dim, "head_dim": 128, "depth": depth, "cond_depth": cond_depth, "res": 64, "patch_size": 256,
          "latent_scale": cfg.latent_scale}
    gg = torch.Generator().manual_seed(6)
    vox = shell_voxels(n, 64, 22.0, 6)
    return (LatDitModel.from_state_dict(p, mc), torch.from_numpy(vox).to(DEV),
            torch.randn(5 + side * side, dim, generator=gg).to(DEV, BF16), torch.randn(n, 16, generator=gg).to(DEV))


def test_runner_runs_the_named_linears_in_four_bits(monkeypatch):
    """Every voxel-side linear that is named goes through linear_mxfp4 on its own weight, in both
    branches, and no other; each result is the one of that call's operands."""
    from vdit.fast_flow import MXFP4_LINEARS, OptimizedLatDitRunner
    from vdit.fast_sampler import SolverConfig
    model, vox, ctx, xt = _model()
    r = OptimizedLatDitRunner(model, SolverConfig(), device=torch.device(DEV), mxfp4_linears=MXFP4_LINEARS)
    of = {id(w[n]): (b, n) for b, w in enumerate(r.blocks) for n in MXFP4_LINEARS if n in w}
    assert len(of) == 3 * 4 + 2 + 1                           # two context blocks, one plain block
    for (b, n), q in ((of[id(w[n])], w[n]) for w in r.blocks for n in MXFP4_LINEARS if n in w):
        want = model.state[f"flow.blocks.{b}.{n}.weight"].to(BF16)
        if n == "ffn0" and r.ffn_interleaved:
            want = want[r.ffn_perm.cpu()]
        assert same(host(fk.dequantize_mxfp4(q)), mxo.values(host(want), 4))
    calls, real = [], fk.linear_mxfp4

    def record(a, w, bias=None, out=None):
        got = real(a, w, bias, out)
        calls.append((of[id(w)], a.clone(), w, bias, got.clone()))
        return got

    monkeypatch.setattr(fk, "linear_mxfp4", record)
    geom = r._prepare_sample_geometry([vox], ctx)
    pos = r.forward_flow_fast(xt, 0.75, ctx, None, geom)
    names = sorted(c[0] for c in calls)
    assert names == sorted(of.values())
    neg = r.forward_flow_fast(xt, 0.75, None, None, geom, uncond=True)
    assert torch.isfinite(pos).all() and torch.isfinite(neg).all()
    # the 1-token branch has constant cross-attention outputs, and shares block 0's self-attention
    assert sorted(c[0] for c in calls[len(names):]) == sorted(
        [(b, n) for b in range(3) for n in ("ffn0", "ffn1")] + [(b, "to_out") for b in (1, 2)])
    torch.cuda.synchronize()
    for (b, n), a, w, bias, got in calls[::4]:
        check_linear(got, a, fk.dequantize_mxfp4(w), bias)


def test_runner_in_four_bits_captured():
    from vdit.fast_flow import OptimizedLatDitRunner
    from vdit.fast_sampler import SolverConfig
    model, vox, ctx, xt = _model()
    r = OptimizedLatDitRunner(model, SolverConfig(), device=torch.device(DEV), mxfp4_linears=("ffn0", "ffn1"))
    eager = r.sample_with_context(vox, ctx, noise=xt)
    graphed = [r.sample_with_context(vox, ctx, noise=xt, cuda_graph=True) for _ in range(2)]
    assert torch.isfinite(eager).all()
    assert torch.equal(graphed[0], graphed[1]) and torch.equal(graphed[0], eager)


def test_runner_takes_a_name_given_twice_once():
    from vdit.fast_flow import OptimizedLatDitRunner
    from vdit.fast_sampler import SolverConfig
    model, vox, ctx, xt = _model(depth=2, cond_depth=1)
    once, twice = (OptimizedLatDitRunner(model, SolverConfig(), device=torch.device(DEV), mxfp4_linears=names)
                   for names in (("ffn0", "ffn1"), ["ffn0", "ffn1", "ffn0"]))
    assert twice.mxfp4_linears == ("ffn0", "ffn1")
    for a, b in zip(once.blocks, twice.blocks):
        for n in ("ffn0", "ffn1"):
            assert torch.equal(a[n].codes, b[n].codes) and torch.equal(a[n].scales, b[n].scales)
