"""Refusals of the 4-bit layers' entry points, on the host: nothing here launches (no GPU needed). Pointers are
made-up aligned addresses that a refused call never reads."""

import ctypes
import os

import pytest

torch = pytest.importorskip("torch")
from strata_mlx_b200 import _lib, affine  # noqa: E402

EKIND, ESHAPE, EDTYPE, EARG, EWORKSPACE = 1, 2, 3, 4, 5
A = 1 << 20  # an aligned address


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from strata_mlx_b200 import _build

        _build.build()
    return _lib.lib()


def test_sizes_of_the_layout(lib):
    # strips of 16 rows, tiles of 128 columns: 1024 bytes of codes and 64 bytes for each group of a tile
    assert lib.smoe_q4_bytes(1, 16, 128, 128) == 1024 + 64
    assert lib.smoe_q4_bytes(1, 16, 128, 64) == 1024 + 128
    assert lib.smoe_q4_bytes(3, 17, 160, 32) == 3 * 2 * 2 * (1024 + 256)
    for bad in ((1, 16, 100, 64), (1, 16, 128, 16), (1, 0, 128, 64), (-1, 16, 128, 64), (1, 16, 96, 64),
                (1, 2**31, 128, 64), (1, 2**20, 2**21, 128), (2**20 + 1, 16, 128, 64)):
        assert lib.smoe_q4_bytes(*bad) == 0, bad


@pytest.mark.parametrize("rows, cols, group, code", [(4, 128, 48, ESHAPE), (4, 100, 32, ESHAPE), (4, 96, 64, ESHAPE),
                                                     (-1, 128, 64, ESHAPE), (4, 0, 64, ESHAPE),
                                                     (2**20, 2**21, 128, ESHAPE), (4, 2**31, 32, ESHAPE)])
def test_matrices_that_do_not_divide_are_refused(lib, rows, cols, group, code):
    assert lib.smoe_q4_quantize(A, 1, rows, cols, group, A, A, A, None) == code
    assert lib.smoe_q4_dequant(A, A, A, rows, cols, group, A, 1, None) == code
    assert lib.smoe_q4_pack(A, A, A, 2, rows, cols, group, A, None) == code
    assert lib.smoe_q4_unpack(A, 2, rows, cols, group, A, 1, None) == code
    assert lib.smoe_q4_linear(A, rows, cols, group, A, 3, A, 1, None) == code
    assert lib.smoe_last_error()


def test_pointers_and_types_are_checked(lib):
    assert lib.smoe_q4_quantize(None, 1, 4, 128, 64, A, A, A, None) == EARG
    assert lib.smoe_q4_quantize(A + 8, 1, 4, 128, 64, A, A, A, None) == EARG
    assert lib.smoe_q4_quantize(A, 7, 4, 128, 64, A, A, A, None) == EDTYPE
    assert lib.smoe_q4_dequant(A, A, None, 4, 128, 64, A, 1, None) == EARG
    assert lib.smoe_q4_dequant(A, A, A, 4, 128, 64, A, 2, None) == EDTYPE
    assert lib.smoe_q4_pack(A, A, A, -1, 4, 128, 64, A, None) == ESHAPE
    assert lib.smoe_q4_pack(A, A, A, 2**20 + 1, 4, 128, 64, A, None) == ESHAPE
    assert lib.smoe_q4_unpack(A, 2**20 + 1, 4, 128, 64, A, 1, None) == ESHAPE
    assert lib.smoe_q4_pack(A, A, A, 1, 4, 128, 64, None, None) == EARG
    assert lib.smoe_q4_unpack(None, 1, 4, 128, 64, A, 1, None) == EARG
    assert lib.smoe_q4_linear(A, 4, 128, 64, A + 4, 3, A, 1, None) == EARG  # activations off a 16-byte boundary
    assert lib.smoe_q4_linear(A + 8, 4, 128, 64, A, 3, A, 1, None) == EARG
    assert lib.smoe_q4_linear(A, 4, 128, 64, A, 3, None, 1, None) == EARG
    assert lib.smoe_q4_linear(A, 4, 128, 64, A, 3, A, 5, None) == EDTYPE
    assert lib.smoe_q4_linear(A, 4, 128, 64, A, -1, A, 1, None) == EARG
    assert lib.smoe_q4_product(None, None) == EARG
    assert lib.smoe_q4_moe(None, None, 0, None) == EARG


def test_tile_products_check_their_arguments(lib):
    def plan(te=A, tiles=3, experts=4, plan=A, nbytes=64):
        return lib.smoe_q4_tile_plan(te, tiles, experts, plan, nbytes, None)

    def product(w=A, experts=4, rows=16, cols=128, group=64, a=A, tiles=3, plan=A, slot=A, out_rows=9, out=A, dtype=1):
        return lib.smoe_q4_tile_matmul(w, experts, rows, cols, group, a, tiles, plan, slot, out_rows, out, dtype, None)

    assert lib.smoe_q4_tile_plan_size(3) == 64 and lib.smoe_q4_tile_plan_size(0) == 0
    assert plan(tiles=0) == 0 and product(tiles=0) == 0 and product(out_rows=0) == 0
    assert plan(te=None) == EARG and plan(tiles=-1) == ESHAPE and plan(experts=0) == ESHAPE and plan(tiles=2**24 + 1) == ESHAPE
    assert plan(plan=None) == EWORKSPACE and plan(nbytes=63) == EWORKSPACE and plan(plan=A + 8) == EWORKSPACE
    for bad in (dict(w=None), dict(a=None), dict(plan=None), dict(out=None), dict(w=A + 8), dict(a=A + 2), dict(out_rows=-1)):
        assert product(**bad) == EARG, bad
    for bad in (dict(tiles=-1), dict(experts=0), dict(cols=96), dict(group=16), dict(rows=0), dict(tiles=2**24, rows=2**20)):
        assert product(**bad) == ESHAPE, bad
    assert product(dtype=3) == EDTYPE


def test_empty_calls_do_nothing(lib):
    assert lib.smoe_q4_quantize(A, 1, 0, 128, 64, A, A, A, None) == 0
    assert lib.smoe_q4_linear(A, 4, 128, 64, A, 0, A, 1, None) == 0
    assert lib.smoe_q4_product(ctypes.byref(_lib.SmoeQ4Product(dtype=1)), None) == 0
    assert lib.smoe_q4_moe(ctypes.byref(_lib.SmoeQ4Moe(dtype=1)), None, 0, None) == 0


def _product(**kw):
    base = dict(dtype=1, group=64, x=A, cols=128, stack=A, rows=16, experts=4, idx=A, pairs=6, share=3, out=A)
    base.update(kw)
    return ctypes.byref(_lib.SmoeQ4Product(**base))


@pytest.mark.parametrize("kw, code", [
    (dict(share=4), EARG), (dict(share=0), EARG), (dict(experts=0), ESHAPE), (dict(experts=2049), ESHAPE),
    (dict(pairs=2049, share=1), ESHAPE), (dict(pairs=-3), EARG), (dict(idx=None), EARG), (dict(out=None), EARG),
    (dict(stack=None), EARG), (dict(x=None), EARG), (dict(weights=A), EARG), (dict(group=60), ESHAPE),
    (dict(stack2=A, dense=A, dense_rows=16, dense_tokens=2, dense_out=A), EARG),
    (dict(dense=A, dense_rows=16, dense_tokens=2, dense_out=A, dense_gate=A), EARG),
    (dict(dense=A, dense_rows=16, dense_tokens=2, dense_out=None), EARG), (dict(dtype=3), EDTYPE)])
def test_pair_products_check_their_arguments(lib, kw, code):
    assert lib.smoe_q4_product(_product(**kw), None) == code


def _moe(**kw):
    base = dict(dtype=1, group=64, down_group=64, tokens=2, hidden=128, experts=4, k=2, ffn=64, shared_ffn=64, x=A, idx=A,
                weights=A, shared_gate=A, gate=A, up=A, down=A, sgate=A, sup=A, sdown=A, out=A)
    base.update(kw)
    return ctypes.byref(_lib.SmoeQ4Moe(**base))


@pytest.mark.parametrize("kw, code", [
    (dict(tokens=65), ESHAPE), (dict(tokens=-1), EARG), (dict(experts=2049), ESHAPE), (dict(experts=0), ESHAPE),
    (dict(k=0), ESHAPE), (dict(k=33), ESHAPE), (dict(ffn=96), ESHAPE), (dict(hidden=96), ESHAPE),
    (dict(shared_ffn=96), ESHAPE), (dict(shared_ffn=-64), ESHAPE), (dict(sup=None), EARG), (dict(weights=None), EARG),
    (dict(down=A + 8), EARG), (dict(out=None), EARG), (dict(dtype=2), EDTYPE), (dict(down_group=20), ESHAPE)])
def test_the_moe_block_checks_its_arguments(lib, kw, code):
    assert lib.smoe_q4_moe(_moe(**kw), A, 1 << 20, None) == code


def test_the_moe_block_checks_its_workspace(lib):
    need = lib.smoe_q4_moe_workspace_size(2, 2, 128, 64, 64)
    assert need >= (4 + 2) * 64 * 2
    assert lib.smoe_q4_moe(_moe(), None, need, None) == EWORKSPACE
    assert lib.smoe_q4_moe(_moe(), A, need - 1, None) == EWORKSPACE
    assert lib.smoe_q4_moe(_moe(), A + 4, need, None) == EWORKSPACE
    assert lib.smoe_q4_moe_workspace_size(0, 2, 128, 64, 64) == 0


def test_the_route_of_a_window_checks_its_arguments(lib):
    def call(w=A, gw=A, x=A, tokens=2, experts=8, hidden=64, k=2, g=A, counter=A):
        return lib.smoe_route_window(w, gw, x, tokens, experts, hidden, k, A, A, A, g, counter, None)

    assert call(tokens=0) == 0
    assert call(tokens=65) == ESHAPE and call(hidden=48) == ESHAPE and call(experts=2049) == ESHAPE
    assert call(k=9) == ESHAPE and call(k=0) == ESHAPE and call(experts=64, k=33) == ESHAPE
    assert call(w=None) == EARG and call(counter=None) == EARG and call(g=None) == EARG and call(gw=None) == EARG
    assert call(x=A + 8) == EARG and call(w=A + 2) == EARG and call(tokens=-1) == EARG


def test_there_is_no_cpu_path():
    w = torch.zeros(4, 128)
    parts = torch.zeros(4, 16, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.float16), torch.zeros(4, 2, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        affine.quantize(w)
    with pytest.raises(ValueError, match="CUDA"):
        affine.dequantize(*parts)
    with pytest.raises(ValueError, match="CUDA"):
        affine.QuantizedLinear(*parts)


def test_group_sizes_and_bits_are_checked_first():
    w = torch.zeros(4, 128)
    with pytest.raises(ValueError, match="groups"):
        affine.quantize(w, group_size=16)
    with pytest.raises(ValueError, match="bits"):
        affine.quantize(w, bits=8)
    with pytest.raises(ValueError, match="bits"):
        affine.dequantize(w, w, w, bits=2)
    with pytest.raises(ValueError, match="codes"):
        affine.QuantizedLinear(torch.zeros(2, 4, 16), w, w)
    with pytest.raises(ValueError, match="codes"):
        affine.QuantizedSwitchLinear(torch.zeros(4, 16), w, w)
