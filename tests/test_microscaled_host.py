"""CPU tests of the low-bit operators: the 64-bit restatement itself, the refusals of the wrappers
and of the C entry points, and the addresses the cache kernels form."""
import ctypes

import numpy as np
import pytest
import torch

from vdit import _lib
from vdit import fast_kernels as fk

from oracle import microscaled as mxo

BF16 = torch.bfloat16


def test_oracle_rounds_to_the_nearest_and_ties_to_even():
    x = np.zeros((1, 32))
    x[0, :16] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 0.2500001, 4.9, 5.1, -0.3, 7.9, -7.9, 0]
    x[0, 16] = 4                                             # max 7.9: scale 1
    v = mxo.values(x, 4)[0]
    assert v[:16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -4, 0.5, 4, 6, -0.5, 6, -6, 0]
    y = torch.randn(64, 256, generator=torch.Generator().manual_seed(0))
    s = torch.ldexp(torch.ones(64, 8), torch.frexp(y.view(64, 8, 32).abs().amax(-1)).exponent - 9)
    e4 = ((y.view(64, 8, 32) / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s[..., None]).view(64, 256)
    assert np.array_equal(mxo.values(y.numpy(), 8), e4.double().numpy())


def test_wrappers_refuse_what_they_cannot_take():
    x = torch.zeros(4, 64, dtype=BF16)
    q = fk.Mxfp4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 4, 64)
    for bad in (x[:, ::2], x.double(), x[0], torch.zeros(4, 48, dtype=BF16), torch.zeros(4, 0, dtype=BF16),
                x[:1].expand(4, 64)):
        with pytest.raises(ValueError):
            fk.quantize_mxfp4(bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        fk.quantize_mxfp4(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fk.dequantize_mxfp4(q)
    with pytest.raises(ValueError, match="dtype"):
        fk.dequantize_mxfp4(q, torch.float64)
    with pytest.raises(ValueError, match="Mxfp4Tensor"):
        fk.linear_mxfp4(x, x)
    with pytest.raises(ValueError, match="columns"):
        fk.linear_mxfp4(torch.zeros(4, 96, dtype=BF16), q)
    with pytest.raises(ValueError, match="bias"):
        fk.linear_mxfp4(x, q, torch.zeros(5, dtype=BF16))
    with pytest.raises(ValueError, match="out"):
        fk.linear_mxfp4(x, q, out=torch.zeros(3, 8, dtype=BF16))
    with pytest.raises(ValueError, match="scale bytes"):
        fk.linear_mxfp4(x, fk.Mxfp4Tensor(q.codes, q.scales[:256], 4, 64))


def test_cache_refusals():
    for kw in (dict(bits=6), dict(head_dim=80), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(pages=0),
               dict(kv_heads=0)):
        a = dict(pages=2, page_size=16, kv_heads=2, head_dim=64, bits=8, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError, match="MxKvCache"):
            fk.MxKvCache(**a)
    c = fk.MxKvCache(2, 16, 2, 64, bits=4, device="cpu")
    assert c.slots == 32 and c.width == 128 and c.k.shape == (2, 2, 16, 32) and c.k_scales.shape == (2, 2, 16, 2)
    rows, slots = torch.zeros(3, 128, dtype=BF16), torch.arange(3)
    for k, v, s in ((rows, rows, slots.int()), (rows, rows[:2], slots), (rows.float(), rows, slots),
                    (rows[:, :64], rows, slots), (rows, rows, torch.arange(6)[::2])):
        with pytest.raises(ValueError, match="kv_cache_write"):
            fk.kv_cache_write(c, k, v, s)
    with pytest.raises(ValueError, match="dtype"):
        fk.kv_cache_read(c, slots, torch.float16)
    table, lengths = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for q, t, n in ((rows[:, :64], table, lengths), (rows, table.long(), lengths), (rows, table[:2], lengths),
                    (rows, table, lengths.long()), (rows, table, lengths[:2]), (rows, table[:, :0], lengths),
                    (rows.float(), table, lengths)):
        with pytest.raises(ValueError, match="attention_1q_cached"):
            fk.attention_1q_cached(q, c, t, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        fk.attention_1q_cached(rows, c, table, lengths)


def test_c_entry_points_check_before_any_launch():
    lib = _lib.load()
    assert lib.vdit_mxfp4_scale_bytes(1, 32) == 512 and lib.vdit_mxfp4_scale_bytes(129, 160) == 4 * 512
    assert lib.vdit_mxfp4_scale_bytes(0, 32) == 0
    assert lib.vdit_mxfp4_quantize(None, 0, 64, 4, 64, None, None, None) == -1
    assert lib.vdit_mxfp4_quantize(16, 3, 64, 4, 64, 16, 16, None) == -1            # no such type
    assert lib.vdit_mxfp4_quantize(16, 0, 32, 4, 64, 16, 16, None) == -1            # rows overlap
    assert lib.vdit_mxfp4_quantize(16, 0, 64, 4, 48, 16, 16, None) == -4            # half a block
    assert lib.vdit_mxfp4_quantize(8, 0, 64, 4, 64, 16, 16, None) == -2
    assert lib.vdit_mxfp4_quantize(16, 0, 68, 4, 64, 16, 16, None) == -2
    assert lib.vdit_mxfp4_quantize(16, 0, 64, 0, 64, 16, 16, None) == 0
    assert lib.vdit_mxfp4_dequantize(16, 16, 4, 64, 16, 7, 64, None) == -1
    assert lib.vdit_linear_mxfp4(16, 16, 16, 16, None, 16, 64, 4, 64, 48, None) == -4
    assert lib.vdit_linear_mxfp4(16, 16, 16, 16, None, 16, 64, 4, 60, 64, None) == -4
    assert lib.vdit_linear_mxfp4(16, 16, 16, 16, None, 16, 56, 4, 64, 64, None) == -1
    assert lib.vdit_linear_mxfp4(16, 16, 8, 16, None, 16, 64, 4, 64, 64, None) == -2
    assert lib.vdit_linear_mxfp4(16, 16, 16, 16, None, 16, 64, 0, 64, 64, None) == 0

    assert lib.vdit_linear_mxfp4_dense_workspace_bytes(4, 1536) == 0
    nb = lib.vdit_linear_mxfp4_dense_workspace_bytes(129, 160)
    assert nb == 129 * 80 + 4 * 512
    dense = [16, 0, 160, 16, 16, None, 16, 64, 129, 64, 160, 16, nb, None]
    for at, value, rc in ((1, 5, -1), (2, 152, -1), (2, 164, -2), (9, 60, -4), (10, 144, -4), (7, 56, -1), (0, 8, -2),
                          (11, None, -5), (12, nb - 1, -5), (8, 0, 0)):
        a = list(dense)
        a[at] = value
        assert lib.vdit_linear_mxfp4_dense(*a) == rc, (at, value)

    def cache(**kw):
        a = dict(k=16, v=16, k_scales=16, v_scales=16, pages=2, page_size=16, heads=2, head_dim=64, bits=8)
        a.update(kw)
        return ctypes.byref(_lib.KvCacheStruct(**a))

    for kw, rc in ((dict(page_size=24), -4), (dict(page_size=8), -4), (dict(head_dim=48), -4), (dict(bits=5), -4),
                   (dict(k=None), -1), (dict(pages=0), -1), (dict(v_scales=8), -2), (dict(v=24), -2)):
        assert lib.vdit_kv_cache_write(16, 128, 16, 128, 16, 3, cache(**kw), None) == rc, kw
        assert lib.vdit_kv_cache_read(cache(**kw), 16, 3, 16, 128, 16, 128, 0, None) == rc, kw
    assert lib.vdit_kv_cache_write(16, 120, 16, 128, 16, 3, cache(), None) == -1
    assert lib.vdit_kv_cache_write(16, 132, 16, 128, 16, 3, cache(), None) == -2
    assert lib.vdit_kv_cache_write(16, 128, 16, 128, 16, 0, cache(), None) == 0
    assert lib.vdit_kv_cache_write(16, 128, 16, 128, 16, 0, None, None) == -1
    assert lib.vdit_kv_cache_read(cache(), 16, 3, 16, 128, 16, 128, 1, None) == -1
    args = [16, 128, cache(), 16, 4, 4, 16, 1, 2, 0.125, 16, 128, None, 0, None]
    need = lib.vdit_attention_1q_cached_workspace_bytes(1, 2, 2, 64, 512, 16)
    assert need > 0
    for at, value, rc in ((8, 3, -1), (1, 120, -1), (4, -1, -1), (5, 1 << 30, -4), (2, cache(head_dim=80), -4),
                          (2, None, -1), (0, 8, -2), (7, 0, 0)):
        a = list(args)
        a[at] = value
        assert lib.vdit_attention_1q_cached(*a) == rc, (at, value)
    a = list(args)
    a[5], a[12], a[13] = 512, 16, need - 1
    assert lib.vdit_attention_1q_cached(*a) == -5


def test_which_rows_are_quantised_on_the_way():
    """No workspace for one and two rows of up to 65536 elements in all, and for three and four of up to 2048."""
    need = _lib.load().vdit_linear_mxfp4_dense_workspace_bytes
    for m, k, none in ((1, 65536, True), (1, 65568, False), (2, 32768, True), (2, 32800, False), (3, 2048, True),
                       (4, 2048, True), (3, 2080, False), (4, 2080, False), (5, 32, False)):
        assert (need(m, k) == 0) == none, (m, k)
        if not none:
            assert need(m, k) == m * k // 2 + -(-m // 128) * -(-k // 128) * 512


@pytest.mark.parametrize("pages,page,heads,hd,bits", [(3, 16, 5, 96, 4), (7, 16, 2, 32, 8), (2, 1024, 3, 128, 8),
                                                       (70000, 128, 12, 128, 8)])
def test_cache_addresses_stay_inside_and_apart(pages, page, heads, hd, bits):
    """The kernels' address arithmetic, ((page * heads + head) * page_size + offset) * width + the byte of
    the channels with its 16-byte piece exchanged: the last slot ends where the buffer ends (past 2^32
    bytes in the last case), no two pieces share bytes, and the 16 keys of a copy are consecutive and
    16-byte aligned."""
    width, nb = hd * bits // 8, pages * heads * page * (hd * bits // 8)
    pieces = width // 16

    def swap(row):
        return {8: row & 7, 4: row >> 1 & 3, 6: row >> 2 & 1, 2: row >> 2 & 1}.get(pieces, row & 0)

    last = ((np.int64(pages - 1) * heads + heads - 1) * page + page - 1) * width
    assert last + width == nb
    row, p = np.meshgrid(np.arange(16), np.arange(pieces), indexing="ij")
    at = row * width + ((p * 16) ^ (swap(row) * 16))
    assert np.array_equal(np.sort(at.ravel()), np.arange(16 * pieces) * 16)     # a permutation within the copy
    assert all(set(at[r] // width) == {r} for r in range(16))                   # and within each row
    # eight neighbouring rows have the same piece in 8 of the 128 bytes' 16-byte columns, or all they can
    for q in range(pieces):
        assert len(set(at[:8, q] // 16 % 8)) == 8
    if pages < 100:
        pg, h, o = np.meshgrid(np.arange(pages), np.arange(heads), np.arange(0, page, 16), indexing="ij")
        start = ((pg * heads + h) * page + o) * width
        assert len(np.unique(start)) == start.size and (start % 16 == 0).all() and start.max() + 16 * width == nb


def test_runner_refuses_unknown_four_bit_linears():
    from vdit.fast_flow import OptimizedLatDitRunner
    with pytest.raises(ValueError, match="to_qkv"):
        OptimizedLatDitRunner(None, mxfp4_linears=("ffn0", "to_qkv"))
