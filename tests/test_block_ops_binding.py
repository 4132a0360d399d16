"""Lib.rope_axes, the Python form of the rotation plan. No device."""
import os

import numpy as np
import pytest
import torch

import __graft_entry__ as ge


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(os.path.join(ge.PKG_DIR, "libiris_b200.so")):
        ge.build()
    lib = ge.load_package().load()
    yield lib
    lib.iris_b200_clear_error()


def same(a, b):
    return (a.n, a.head_dim, list(a.turn), list(a.axis)) == (b.n, b.head_dim, list(b.turn), list(b.axis))


@pytest.mark.parametrize("scales", [(1.0,), (1.0, 2.0), (1.0, 2.0, 3.0, 4.0)])
def test_one_scale_for_every_axis(lib, scales):
    """A scale that is missing would turn its axis by nothing, one too many would be dropped."""
    with pytest.raises(ValueError):
        lib.rope_axes((32, 48, 48), scales, 256.0, False, 128)


@pytest.mark.parametrize("make", [tuple, list, np.array, torch.tensor])
def test_sequences_of_any_kind(lib, make):
    want = lib.rope_axes((32, 48, 48), (2.5, 1.0, 0.5), 256.0, False, 128)
    assert any(want.turn)
    assert same(lib.rope_axes(make([32, 48, 48]), make([2.5, 1.0, 0.5]), 256.0, False, 128), want)
    assert same(lib.rope_axes(make([32, 48, 48]), make([1, 1, 1]), 256.0, True, 128), lib.rope_axes((32, 48, 48), None, 256.0, True, 128))


def test_refusals_name_the_library_s_reason(lib):
    from iris_c_b200.binding import IrisB200Error
    for dims, hd in (((33,), 128), ((64, 66), 128), ((), 128), ((2,) * 9, 128), ((64,), 63)):
        with pytest.raises(IrisB200Error):
            lib.rope_axes(dims, None, 256.0, False, hd)
        lib.iris_b200_clear_error()
