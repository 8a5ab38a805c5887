"""What the native operators refuse, without a GPU: argument checks of the C ABI
that come before any device work, and of the Python layer."""
import ctypes

import numpy as np
import pytest
import torch

import drift_b200 as d
from drift_b200 import _lib

LIB = _lib.load()


@pytest.mark.parametrize("rows,cols,codes,scales", [
    (1, 1, 16, 1024), (128, 32, 2048, 1024), (129, 257, 129 * 144, 4096), (0, 64, 0, 0),
    (5, 0, 0, 0), (2048, 2048, 2048 * 1024, 16 * 16 * 512)])
def test_packed_sizes(rows, cols, codes, scales):
    a, b = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(LIB.drift_mx4_sizes(rows, cols, ctypes.byref(a), ctypes.byref(b)))
    assert (a.value, b.value) == (codes, scales)


@pytest.mark.parametrize("rows,cols", [(-1, 4), (4, -1), (1 << 31, 4), (4, 1 << 31)])
def test_packed_sizes_refuse(rows, cols):
    assert LIB.drift_mx4_sizes(rows, cols, None, None) == _lib.EINVAL


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("tokens,depth,vocab", [(0, 1, 1), (0, 64, 300), (1, 1, 1), (1, 8, 1 << 24),
                                                (1 << 22, 8, 3), (100, 4096, 131072)])
def test_cross_entropy_workspace_of_any_shape(mode, tokens, depth, vocab):
    op = _lib.DriftXent(tokens=tokens, depth=depth, vocab=vocab)
    out = ctypes.c_int64()
    _lib.check(LIB.drift_linear_xent_workspace(ctypes.byref(op), mode, ctypes.byref(out)))
    assert 0 < out.value < 1 << 36
    assert LIB.drift_linear_xent_workspace(ctypes.byref(op), 3, ctypes.byref(out)) == _lib.EINVAL


@pytest.mark.parametrize("tokens,depth,vocab", [
    (-1, 8, 8), (4, 0, 8), (4, 8, 0), (1 << 31, 8, 8), (4, 1 << 31, 8), (4, 8, 1 << 31),
    (1 << 24, 1 << 24, 8), (4, 1 << 24, 1 << 24), ((1 << 31) - 1, (1 << 31) - 1, 8)])
def test_cross_entropy_workspace_refuses_what_no_memory_holds(tokens, depth, vocab):
    op = _lib.DriftXent(tokens=tokens, depth=depth, vocab=vocab)
    out = ctypes.c_int64()
    for mode in range(3):
        assert LIB.drift_linear_xent_workspace(ctypes.byref(op), mode,
                                               ctypes.byref(out)) == _lib.EINVAL


@pytest.mark.parametrize("tokens,depth,vocab", [(1 << 24, 1, 1 << 24), (1 << 24, 1 << 16, 256),
                                                ((1 << 31) - 1, 512, (1 << 31) - 1)])
def test_cross_entropy_workspace_of_the_longest_sides(tokens, depth, vocab):
    """Their tiles, 65536 a side, are past 32 bits in number."""
    op = _lib.DriftXent(tokens=tokens, depth=depth, vocab=vocab)
    out = ctypes.c_int64()
    for mode in range(3):
        _lib.check(LIB.drift_linear_xent_workspace(ctypes.byref(op), mode, ctypes.byref(out)))
        assert out.value >= 16 * tokens


def test_a_null_context_is_refused():
    q, x, h = _lib.DriftMx4(), _lib.DriftXent(), _lib.DriftAdamW()
    p = d.policies.by_name("mxfp4").to_c()
    assert LIB.drift_mx4_quantize_dev(None, ctypes.byref(p), 0, 1, None, 1, 1, 1, None, None, None,
                                      None, None, None, None, None) == _lib.EINVAL
    assert LIB.drift_mx4_dequantize_dev(None, ctypes.byref(q), 1, None, 1, None) == _lib.EINVAL
    assert LIB.drift_mx4_gemm_dev(None, ctypes.byref(q), ctypes.byref(q), None, 1, None, 1,
                                  None) == _lib.EINVAL
    assert LIB.drift_linear_xent_dev(None, ctypes.byref(x), None, None, None, None, 0,
                                     None) == _lib.EINVAL
    assert LIB.drift_linear_xent_grad_dev(None, ctypes.byref(x), None, None, 0, None, 0, None, 0,
                                          None, None, 0, None) == _lib.EINVAL
    assert LIB.drift_adamw_dev(None, ctypes.byref(h), None, 0, None, None, None, None, None,
                               None) == _lib.EINVAL


def test_host_tensors_are_refused():
    p = d.policies.by_name("mxfp4")
    x, w, t = torch.zeros(4, 32), torch.zeros(8, 32), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError):
        d.mx4_quantize_dev(p, x)
    with pytest.raises(TypeError):
        d.linear_xent_dev(x.bfloat16(), w.bfloat16(), t)
    with pytest.raises(TypeError):
        d.linear_xent_mean_dev(x.bfloat16(), w.bfloat16(), t)
    with pytest.raises(TypeError):
        d.AdamW([x])


@pytest.mark.parametrize("name", ["fp8-mx", "fp32", "bf16", "fp8"])
def test_only_e2m1_blocks_are_packed(name):
    with pytest.raises(ValueError):
        d.mx4_quantize_dev(d.policies.by_name(name), torch.zeros(4, 32))


def test_other_block_lengths_and_axes_are_refused():
    p = d.policies.by_name("mxfp4")
    with pytest.raises(ValueError):
        d.mx4_quantize_dev(p.to_builder("b16").scale_block(16).build(), torch.zeros(4, 32))
    with pytest.raises(ValueError):
        d.mx4_quantize_dev(p, torch.zeros(4, 32), axis=2)
    with pytest.raises(ValueError):
        d.mx4_quantize_dev(p, torch.zeros(4, 32, 1))


@pytest.mark.parametrize("kw", [dict(state_bits=16), dict(rounding=d.Rounding.TRUNCATE),
                                dict(rounding=d.Rounding.STOCHASTIC),
                                dict(rounding=d.Rounding.STOCHASTIC, state_bits=8)])
def test_adamw_settings_refused(kw):
    with pytest.raises(ValueError):
        d.AdamW([torch.zeros(4)], **kw)


def test_an_empty_parameter_list_is_refused():
    with pytest.raises(ValueError):
        d.AdamW([])


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (130, 256), (128, 257), (300, 1000)])
def test_plain_arrays_round_trip_through_the_tiled_scales(rows, cols):
    """from_parts lays scale (r, b) at byte (r % 32) * 16 + (r / 32) * 4 + b of its
    128 x 4 tile and pads with 127; to_parts undoes it."""
    rs = np.random.default_rng(rows * 1000 + cols)
    blocks = (cols + 31) // 32
    codes = rs.integers(0, 256, (rows, blocks * 16), dtype=np.uint8)
    nib = np.stack((codes & 15, codes >> 4), -1).reshape(rows, -1)
    nib[:, cols:] = 0
    dirty, codes = torch.from_numpy(codes), torch.from_numpy(nib[:, 0::2] | nib[:, 1::2] << 4)
    scales = torch.from_numpy(rs.integers(0, 255, (rows, blocks), dtype=np.uint8))
    q = d.Mx4.from_parts(dirty, scales, cols)  # padding codes are dropped
    k_tiles = (cols + 255) // 256 * 2
    want = np.full((rows + 127) // 128 * k_tiles * 512, 127, dtype=np.uint8)
    for r in range(rows):
        for b in range(blocks):
            want[((r // 128) * k_tiles + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] \
                = scales[r, b]
    assert (q.scales.numpy() == want).all()
    c2, s2 = q.to_parts()
    assert torch.equal(c2, codes) and torch.equal(s2, scales) and q.shape == (rows, cols)


def test_parts_that_do_not_match_are_refused():
    u8 = torch.uint8
    with pytest.raises(ValueError):
        d.Mx4.from_parts(torch.zeros(4, 16, dtype=u8), torch.zeros(4, 1, dtype=u8), 33)
    with pytest.raises(ValueError):
        d.Mx4.from_parts(torch.zeros(4, 15, dtype=u8), torch.zeros(4, 1, dtype=u8), 32)
    with pytest.raises(TypeError):
        d.Mx4.from_parts(torch.zeros(4, 16), torch.zeros(4, 1), 32)
    with pytest.raises(ValueError):
        d.Mx4(torch.zeros(64, dtype=u8), torch.zeros(100, dtype=u8), 4, 32)
