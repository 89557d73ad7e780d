"""MXFP4: the format's oracle against hand-computed values, and the refusals that need no GPU."""
import ctypes

import pytest
import torch

from firefly_b200 import (
    MXFP4SwiGLU,
    MXFP4Tensor,
    _capi,
    mxfp4_linear,
    mxfp4_matmul,
    mxfp4_swiglu,
    quantize_fp_to_mxfp4,
)
from oracle import mxfp4_oracle as O


def test_oracle_on_values_worked_out_by_hand():
    x = torch.zeros(3, 40)
    x[0, :4] = torch.tensor([6.0, -2.4, 0.25, 0.26])   # A = 6: scale 1
    x[0, 32] = 7.9                                     # A = 7.9: scale 1, saturates at 6
    x[1, 0] = 9.0                                      # A = 9: scale 2, 4.5 -> 4
    x[2, 3] = 2.0 ** -140
    v = O.values(x)
    assert v[0, :4].tolist() == [6.0, -2.0, 0.0, 0.5] and v[0, 32] == 6.0 and v[1, 0] == 8.0
    assert O.scale_exponents(x).tolist() == [[127, 127], [128, 0], [0, 0]]
    assert v[2, 3] == 0.0  # 2^-140 / 2^-127 rounds to 0


def _held(r, c):
    return MXFP4Tensor(torch.zeros(r, (c + 31) // 32 * 16, dtype=torch.uint8),
                       torch.zeros(_capi.lib().ff_mxfp4_scale_bytes(r, c), dtype=torch.uint8), (r, c))


def test_scale_sizes_and_order():
    lib = _capi.lib()
    assert lib.ff_mxfp4_scale_bytes(1, 1) == 1024
    assert lib.ff_mxfp4_scale_bytes(129, 257) == 2 * 4 * 512
    assert lib.ff_mxfp4_scale_bytes(0, 64) == 0
    q = _held(130, 300)
    s = q.scales
    # byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 of chunk (row / 128) * chunks + block / 4
    for row, blk in ((0, 0), (5, 3), (33, 4), (127, 9), (128, 0), (129, 8)):
        s.zero_()
        s[((row // 128) * 4 + blk // 4) * 512 + row % 32 * 16 + row // 32 % 4 * 4 + blk % 4] = 7
        got = q.scale_bytes()
        assert got[row, blk] == 7 and int(got.sum()) == 7


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        quantize_fp_to_mxfp4(torch.zeros(2, 32))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mxfp4_linear(torch.zeros(2, 32), torch.zeros(4, 32))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _held(4, 64).dequantize()


def test_shapes_and_types_are_refused():
    with pytest.raises(ValueError):
        quantize_fp_to_mxfp4(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError, match="contraction"):
        mxfp4_matmul(_held(4, 64), _held(4, 96))
    with pytest.raises(ValueError):
        mxfp4_matmul(torch.zeros(4, 64), _held(4, 64))
    with pytest.raises(ValueError, match="last dim"):
        mxfp4_linear(torch.zeros(2, 31), torch.zeros(4, 32))
    with pytest.raises(ValueError):
        mxfp4_linear(torch.zeros(2, 32, dtype=torch.int32), torch.zeros(4, 32))
    with pytest.raises(ValueError):
        mxfp4_linear(torch.zeros(2, 32), torch.zeros(4, 32, dtype=torch.int8))
    for f in (48, 33):  # hidden sizes that are no multiple of 32
        with pytest.raises(ValueError, match="multiple of 32"):
            mxfp4_swiglu(torch.zeros(2, 32), torch.zeros(2 * f, 32), torch.zeros(32, f))
    with pytest.raises(ValueError):
        mxfp4_swiglu(torch.zeros(2, 32), torch.zeros(64, 32), torch.zeros(32, 64))
    with pytest.raises(ValueError):
        MXFP4SwiGLU(torch.zeros(64, 32), torch.zeros(32, 64))


def test_held_tensors_are_checked():
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)
    MXFP4Tensor(codes, scales, (4, 64))
    for bad in ((codes, scales, (4, 65)), (codes.int(), scales, (4, 64)), (codes, scales[:-1], (4, 64)),
                (codes, scales, (5, 64)), (torch.zeros(32, 4, dtype=torch.uint8).t(), scales, (4, 64)),
                (codes, scales.int(), (4, 64))):
        with pytest.raises(ValueError):
            MXFP4Tensor(*bad)
    with pytest.raises(ValueError, match="transposed"):
        MXFP4Tensor(codes, scales, (4, 64), _held(4, 64))


def test_c_entries_refuse_before_any_launch():
    lib, bad, uns = _capi.lib(), _capi.FF_ERR_INVALID_ARG, _capi.FF_ERR_UNSUPPORTED
    p = ctypes.c_void_p(4096)  # an aligned address that is never read
    n = None
    q = lib.ff_mxfp4_quant
    assert q(p, 7, 4, 64, 64, p, 32, p, n, 0, n, n, n, n) == bad             # type
    assert q(p, 1, 4, 64, 63, p, 32, p, n, 0, n, n, n, n) == bad             # leading dimension
    assert q(p, 1, -1, 64, 64, p, 32, p, n, 0, n, n, n, n) == bad
    assert q(p, 1, 4, 0, 64, p, 32, p, n, 0, n, n, n, n) == bad
    assert q(p, 1, 4, 64, 64, p, 16, p, n, 0, n, n, n, n) == bad             # rows too short for the codes
    assert q(p, 1, 4, 64, 64, p, 40, p, n, 0, n, n, n, n) == bad             # no multiple of 16
    assert q(p, 1, 4, 64, 64, p, 32, n, n, 0, n, n, n, n) == bad             # codes without scales
    assert q(p, 1, 4, 64, 64, p, 32, p, n, 0, n, p, p, n) == bad             # sums without column codes
    assert q(n, 1, 4, 64, 64, p, 32, p, n, 0, n, n, n, n) == bad
    assert q(n, 1, 0, 64, 64, p, 32, p, n, 0, n, n, n, n) == _capi.FF_OK     # nothing to do
    assert lib.ff_mxfp4_dequant(p, 32, p, 4, 64, p, 9, 64, n) == bad
    assert lib.ff_mxfp4_dequant(p, 32, p, 4, 64, p, 1, 63, n) == bad
    s = lib.ff_mxfp4_swiglu_quant
    assert s(p, 96, 4, 48, p, 32, p, n, 0, n, n) == uns                      # no multiple of 32
    assert s(p, 65, 4, 32, p, 16, p, n, 0, n, n) == uns                      # rows not 16-byte aligned
    assert lib.ff_mxfp4_swiglu_bwd_quant(p, 31, p, 64, 4, 32, p, 32, p, n, 0, n, n) == uns
    g = lib.ff_mxfp4_gemm
    assert g(p, 32, p, p, 32, p, n, p, 8, _capi.FF_OUT_S32, 4, 8, 64, n) == bad
    assert g(p, 16, p, p, 32, p, n, p, 8, 2, 4, 8, 64, n) == bad             # lda
    assert g(p, 32, p, p, 32, p, n, p, 7, 2, 4, 8, 64, n) == bad             # ldd
    assert g(p, 32, n, p, 32, p, n, p, 8, 2, 4, 8, 64, n) == bad
    assert g(p, 32, p, p, 32, p, n, p, 8, 2, 4, 8, 0, n) == bad
    assert g(p, 32, p, p, 32, p, n, p, 1 << 23, 2, 4, 1 << 22, 64, n) == uns
    assert g(n, 32, n, n, 32, n, n, n, 8, 2, 0, 8, 64, n) == _capi.FF_OK
    assert lib.ff_mxfp4_swiglu_gemm(p, 32, p, p, 32, p, p, 16, p, 4, 96, 64, n) == uns


def test_serving_entries_refuse_before_any_launch():
    lib, bad, uns = _capi.lib(), _capi.FF_ERR_INVALID_ARG, _capi.FF_ERR_UNSUPPORTED
    p, n = ctypes.c_void_p(4096), None
    need = lib.ff_mxfp4_linear_ws_bytes(3, 64)
    assert need == 1024 + 1024 and lib.ff_mxfp4_linear_ws_bytes(0, 64) == 0
    f = lib.ff_mxfp4_linear
    assert f(p, 1, 64, p, 32, p, n, p, 8, 2, 3, 8, 64, p, need - 1, n) == bad    # workspace
    assert f(p, 1, 64, p, 32, p, n, p, 8, 2, 3, 8, 64, n, need, n) == bad
    assert f(p, 1, 64, p, 16, p, n, p, 8, 2, 3, 8, 64, p, need, n) == bad        # ldw
    assert f(p, 1, 64, n, 32, p, n, p, 8, 2, 3, 8, 64, p, need, n) == bad
    assert f(p, 1, 64, p, 32, p, n, p, 7, 2, 3, 8, 64, p, need, n) == bad        # ldd
    assert f(p, 1, 64, p, 32, p, n, p, 8, 0, 3, 8, 64, p, need, n) == bad        # int32 output
    assert f(p, 5, 64, p, 32, p, n, p, 8, 2, 3, 8, 64, p, need, n) == bad        # type
    assert f(p, 1, 63, p, 32, p, n, p, 8, 2, 3, 8, 64, p, need, n) == bad        # ldx
    assert f(p, 1, 64, p, 32, p, n, p, 8, 2, 3, 8, 0, p, need, n) == bad
    assert f(n, 1, 64, n, 32, n, n, n, 8, 2, 0, 8, 64, n, 0, n) == _capi.FF_OK
    need = lib.ff_mxfp4_swiglu_mlp_ws_bytes(3, 64, 128)
    g = lib.ff_mxfp4_swiglu_mlp
    assert g(p, 1, 64, p, 32, p, p, 64, p, p, 8, 2, 3, 64, 96, 8, p, 1 << 20, n) == uns     # F
    assert g(p, 1, 64, p, 32, p, p, 64, p, p, 8, 2, 3, 64, 128, 8, p, need - 1, n) == bad
    assert g(p, 1, 64, p, 16, p, p, 64, p, p, 8, 2, 3, 64, 128, 8, p, need, n) == bad
    assert g(p, 1, 64, p, 32, p, p, 48, p, p, 8, 2, 3, 64, 128, 8, p, need, n) == bad
    assert g(p, 1, 64, p, 32, p, p, 64, p, p, 7, 2, 3, 64, 128, 8, p, need, n) == bad


def test_pointers_that_are_not_aligned_to_their_elements_are_refused():
    lib, bad = _capi.lib(), _capi.FF_ERR_INVALID_ARG
    p, n, odd, two = ctypes.c_void_p(4096), None, ctypes.c_void_p(4097), ctypes.c_void_p(4098)
    q = lib.ff_mxfp4_quant
    assert q(odd, 1, 4, 64, 64, p, 32, p, n, 0, n, n, n, n) == bad
    assert q(two, 0, 4, 64, 64, p, 32, p, n, 0, n, n, n, n) == bad
    assert q(p, 1, 4, 64, 64, p, 32, p, p, 16, p, two, p, n) == bad          # sums
    assert q(p, 1, 4, 64, 64, p, 32, p, p, 16, p, p, two, n) == bad
    assert lib.ff_mxfp4_dequant(p, 32, p, 4, 64, odd, 1, 64, n) == bad
    assert lib.ff_mxfp4_dequant(p, 32, p, 4, 64, two, 0, 64, n) == bad
    for d, kind, bias in ((odd, 2, n), (two, 1, n), (p, 2, two)):
        assert lib.ff_mxfp4_gemm(p, 32, p, p, 32, p, bias, d, 8, kind, 4, 8, 64, n) == bad
        assert lib.ff_mxfp4_linear(p, 1, 64, p, 32, p, bias, d, 8, kind, 3, 8, 64, p, 1 << 20, n) == bad
    assert lib.ff_mxfp4_swiglu_mlp(p, 1, 64, p, 32, p, p, 64, p, odd, 8, 2, 3, 64, 128, 8, p, 1 << 20, n) == bad
    big = 1 << 24
    f = lib.ff_mxfp4_linear_train
    assert f(p, 1, 64, p, 1, 64, n, odd, 3, 8, 64, 1, 1, p, big, p, big, n) == bad
    assert f(p, 1, 64, p, 1, 64, two, p, 3, 8, 64, 1, 1, p, big, p, big, n) == bad
    b = lib.ff_mxfp4_linear_bwd
    for dx, dw, db in ((odd, p, p), (p, odd, p), (p, p, two)):
        assert b(p, 1, 8, p, big, 1, 1, dx, 2, dw, 2, db, 3, 8, 64, p, big, n) == bad
    assert lib.ff_mxfp4_swiglu_train(p, 1, 64, p, 1, 64, p, 1, 128, p, odd, 3, 64, 128, 8, 1, 1, 1, p, big, p, big, n) == bad
    assert lib.ff_mxfp4_swiglu_train(p, 1, 64, p, 1, 64, p, 1, 128, two, p, 3, 64, 128, 8, 1, 1, 1, p, big, p, big, n) == bad
    g = lib.ff_mxfp4_swiglu_bwd
    for gu, dh in ((two, p), (p, two)):
        assert g(p, 1, 8, gu, dh, p, big, 1, 1, 1, p, 2, p, 2, p, 2, 3, 64, 128, 8, p, big, n) == bad
    for dx, dgu, dd in ((odd, p, p), (p, odd, p), (p, p, odd)):
        assert g(p, 1, 8, p, p, p, big, 1, 1, 1, dx, 2, dgu, 2, dd, 2, 3, 64, 128, 8, p, big, n) == bad
