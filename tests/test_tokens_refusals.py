"""What the operators on columns of tokens refuse, beside test_oracle_tokens.py: the same matrix in two places of a call.  Handles only, no
memory is touched."""
import ctypes as ct

import pytest

from test_oracle_tokens import UNSUPPORTED, Space, handle


@pytest.fixture
def lib():
    from deepnet_amd import cudamat
    return cudamat._cudamat


@pytest.fixture
def new():
    from deepnet_amd import cudamat
    return Space(cudamat)


def test_dot_gated_keeps_its_halves_apart_from_what_it_reads(lib, new):
    """pre where an operand of the same shape is: the very same handle, another one of its memory, a part of it."""
    f = 6
    at = lambda m: ct.addressof(m.contents.data_device.contents)
    w, x, b, y = new(2 * f, 2 * f, trans=1), new(2 * f, 3), new(2 * f, 1), new(f, 3)
    for pre in (x, handle(new.cm, 2 * f, 3, at(x)), handle(new.cm, 2 * f, 3, at(x) + 16), handle(new.cm, 2 * f, 3, at(w) + 64)):
        assert lib.dot_gated(w, x, b, y, pre, 4) == UNSUPPORTED
    # one column: the bias has the shape of pre too; weights of as many columns as cases
    x, y = new(2 * f, 1), new(f, 1)
    assert lib.dot_gated(w, x, b, y, b, 4) == UNSUPPORTED
    w, x, y = new(2 * f, 2 * f), new(2 * f, 2 * f), new(f, 2 * f)
    assert lib.dot_gated(w, x, b, y, w, 4) == UNSUPPORTED


def test_a_grid_that_no_launch_takes_is_refused(lib, new):
    """2^24 workgroups of 256 lanes: the calls that do not split such a grid say so, where a part of it would run."""
    w = 1 << 26
    x, y, row = new(4, w), new(4, w), new(1, w)
    apart = handle(new.cm, 4, w, 1 << 40)
    assert lib.normlimit_by_axis(x, apart, 0, ct.c_float(1.0)) == UNSUPPORTED
    assert lib.max_by_axis(x, row, 0) == UNSUPPORTED


def test_layer_norm_of_columns_that_it_cannot_count_is_refused(lib, new):
    h = 1 << 30
    x, y, dy = (handle(new.cm, h, 1, (i + 1) << 40) for i in range(3))
    assert lib.layer_norm(x, None, None, y, 1e-5) == UNSUPPORTED
    assert lib.layer_norm_grad(dy, x, None, y, None, None, 1e-5, 0.0, 1.0) == UNSUPPORTED
