"""Refusals of the 4-bit layers' entry points that test_affine.py does not make, on the host: nothing here launches."""

import os

import pytest

torch = pytest.importorskip("torch")
from strata_mlx_b200 import _lib  # noqa: E402
from test_affine import EARG, EDTYPE, ESHAPE, A  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from strata_mlx_b200 import _build

        _build.build()
    return _lib.lib()


def test_the_prompts_kernel_checks_its_arguments(lib):
    def call(w=A, rows=64, cols=128, group=64, x=A, tokens=40, out=A, dtype=0):
        return lib.smoe_q4_prompt(w, rows, cols, group, x, tokens, out, dtype, None)

    assert call(tokens=0) == 0
    for bad in (dict(w=None), dict(x=None), dict(out=None), dict(w=A + 8), dict(x=A + 2), dict(tokens=-1)):
        assert call(**bad) == EARG, bad
    for bad in (dict(rows=0), dict(cols=96), dict(group=16), dict(rows=2**30, cols=2**11), dict(tokens=2**31)):
        assert call(**bad) == ESHAPE, bad
    assert call(dtype=7) == EDTYPE


def test_which_counts_of_tokens_take_the_prompts_kernel(lib):
    takes = lib.smoe_q4_is_prompt
    assert takes(1180, 4096, 4096) == 1 and takes(4096, 1536, 4096) == 1
    assert all(takes(t, 64007, 2560) == 0 for t in (-1, 0, 1, 16))  # a window never does
    assert takes(17, 16, 2**20) == 0 and takes(40, 0, 128) == 0 and takes(40, 128, -1) == 0


def test_the_route_with_a_float32_gate_checks_its_arguments(lib):
    def call(w=A, gw=A, x=A, tokens=2, experts=8, hidden=64, k=2, g=A, counter=A):
        return lib.smoe_route_window_f32(w, gw, x, tokens, experts, hidden, k, A, A, A, g, counter, None)

    assert call(tokens=0) == 0
    for bad in (dict(tokens=65), dict(hidden=48), dict(experts=2049), dict(k=9), dict(k=0), dict(experts=64, k=33)):
        assert call(**bad) == ESHAPE, bad
    for bad in (dict(w=None), dict(counter=None), dict(g=None), dict(gw=None), dict(x=A + 8), dict(w=A + 2), dict(tokens=-1)):
        assert call(**bad) == EARG, bad
