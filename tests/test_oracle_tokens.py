"""CPU-only: the float64 restatements of the operators on columns of tokens against differences, published vectors and
other ways to the same numbers; and what the library refuses before it touches a device."""
import ctypes as ct

import numpy as np
import pytest

from oracle import token_oracle as tok

ACTS = [None, 'sigmoid', 'relu', 'tanh', 'silu', 'gelu']


def differences(f, x, step=1e-5):
    """Central differences of a scalar function by every entry."""
    g = np.empty_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + step; up = f(x)
        x[i] = keep - step; down = f(x)
        x[i] = keep
        g[i] = (up - down) / (2 * step)
    return g


def close(a, b, tol=2e-8):
    assert np.max(np.abs(a - b)) <= tol * max(1.0, np.max(np.abs(b))), np.max(np.abs(a - b))


def test_philox_known_answers():
    """The vectors that its authors publish with the generator."""
    def words(counter, key):
        return ['%08x' % v for v in tok.philox4x32(np.array([counter], dtype=np.uint64), key)[0]]
    ones = 0xFFFFFFFF
    assert words([0] * 4, [0, 0]) == ['6627e8d5', 'e169c58d', 'bc57ac4c', '9b00dbd8']
    assert words([ones] * 4, [ones, ones]) == ['408f276d', '41c83b0e', 'a20bc7c6', '6d5451fd']
    assert words([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == ['d16cfe09', '94fdcceb', '5001e420', '24126ea1']


def test_dropout_keeps_the_share_and_counts_from_any_entry():
    keep = tok.dropout_keep((301, 997), 0.3, 0x123456789abcdef0, stream=5, step=17.0)
    n = keep.size
    assert abs(keep.mean() - 0.7) < 5 * np.sqrt(0.21 / n)
    flat = keep.reshape(-1, order='F')
    for first in (0, 1, 2, 3, 4, 1001):
        assert np.array_equal(tok.dropout_keep((301, 997), 0.3, 0x123456789abcdef0, 5, 17.0, first, 50), flat[first:first + 50])
    for other in (dict(stream=6, step=17.0), dict(stream=5, step=18.0)):
        assert abs(np.mean(tok.dropout_keep((301, 997), 0.3, 0x123456789abcdef0, **other) == keep) - 0.58) < 0.01


@pytest.mark.parametrize("eps", [1e-5, 0.1])
def test_layer_norm_gradient_against_differences(eps):
    rng = np.random.default_rng(3)
    x, dy, gain, bias = rng.standard_normal((7, 4)), rng.standard_normal((7, 4)), rng.standard_normal((7, 1)), rng.standard_normal((7, 1))
    dx, dgain, dbias = tok.layer_norm_grad(dy, x, gain, eps)
    close(dx, differences(lambda v: np.sum(dy * tok.layer_norm(v, gain, bias, eps)), x))
    close(dgain, differences(lambda v: np.sum(dy * tok.layer_norm(x, v, bias, eps)), gain))
    close(dbias, differences(lambda v: np.sum(dy * tok.layer_norm(x, gain, v, eps)), bias))


@pytest.mark.parametrize("act", ACTS)
def test_gated_gradients_against_differences(act):
    rng = np.random.default_rng(4)
    w, x, b, dy = (rng.standard_normal(s) for s in ((5, 8), (5, 3), (8, 1), (4, 3)))
    f = lambda w, x, b: np.sum(dy * tok.dot_gated(w.T, x, b, act)[0])
    d = tok.gate_grad(dy, tok.dot_gated(w.T, x, b, act)[1], act)
    close(x @ d.T, differences(lambda v: f(v, x, b), w))
    close(w @ d, differences(lambda v: f(w, v, b), x))
    close(d.sum(axis=1, keepdims=True), differences(lambda v: f(w, x, v), b))


def test_log_prob_gradients_against_differences():
    rng = np.random.default_rng(5)
    x = 2 * rng.standard_normal((6, 5))
    labels, lw, ew = np.array([[0, 5, -1, 2, 6]]), rng.standard_normal((1, 5)), rng.standard_normal((1, 5))
    def f(v):
        o = tok.log_probs(v, labels)
        return np.sum(lw * o['logp']) + np.sum(ew * o['entropy'])
    o = tok.log_probs(x, labels)
    close(tok.log_probs_grad(x, labels, o['log_z'], lw, o['entropy'], ew), differences(f, x))


def test_log_probs_of_special_columns():
    inf, nan = np.inf, np.nan
    x = np.array([[1, -inf, 0, inf], [1, -inf, nan, 0], [-inf, -inf, 3, 0], [0, -inf, 3, inf]])
    o = tok.log_probs(x, [[2, 0, 1, -1]], top=4)
    assert o['logp'][0, 0] == -inf and o['logp'][0, 1] == -inf and np.isnan(o['logp'][0, 2]) and o['logp'][0, 3] == 0
    assert o['entropy'][0, 1] == 0 and o['log_z'][0, 1] == -inf and np.isnan(o['entropy'][0, 2:]).all()
    assert o['top_labels'].T.tolist() == [[0, 1, 3, 2], [0, 1, 2, 3], [2, 3, 0, 1], [0, 3, 1, 2]]
    assert not tok.log_probs_grad(x[:, 1:2], [[0]], [[-inf]], None, [[0.0]], [[1.0]])[1:].any()


# ---- what the library refuses

def handle(cm, rows, cols, base=0x100000, on_device=1, trans=0):
    m = cm.cudamat()
    m.data_device = ct.cast(base, type(m.data_device))
    m.on_device, m.size[0], m.size[1], m.is_trans = on_device, rows, cols, trans
    return ct.pointer(m)


class Space(object):
    """Handles of matrices at addresses apart from each other (never dereferenced)."""

    def __init__(self, cm):
        self.cm, self.at = cm, 1 << 30

    def __call__(self, rows, cols, **kw):
        m = handle(self.cm, rows, cols, self.at, **kw)
        self.at += 1 << 24
        return m


@pytest.fixture
def cm():
    from deepnet_amd import cudamat
    return cudamat


INCOMPATIBLE, TRANSPOSED, NOT_ON_DEVICE, UNSUPPORTED = -1, -5, -8, -9


def test_layer_norm_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    x, y, g, b = new(8, 4), new(8, 4), new(8, 1), new(8, 1)
    call = lambda *a, eps=1e-5: lib.layer_norm(*a, eps)
    assert call(new(8, 4, on_device=0), g, b, y) == NOT_ON_DEVICE and call(x, new(8, 1, on_device=0), b, y) == NOT_ON_DEVICE
    assert call(x, g, b, new(8, 4, trans=1)) == TRANSPOSED and call(new(8, 4, trans=1), g, b, y) == TRANSPOSED
    assert call(x, g, new(8, 1, trans=1), y) == TRANSPOSED
    for bad in (new(1, 8), new(7, 1), new(8, 2)):
        assert call(x, bad, b, y) == INCOMPATIBLE and call(x, g, bad, y) == INCOMPATIBLE
    assert call(x, g, b, new(8, 5)) == INCOMPATIBLE and call(x, g, b, new(4, 8)) == INCOMPATIBLE
    assert call(x, g, b, y, eps=-1e-5) == UNSUPPORTED and call(x, g, b, y, eps=float('nan')) == UNSUPPORTED
    base = ct.addressof(x.contents.data_device.contents)
    assert call(x, g, b, handle(cm, 8, 4, base + 4)) == UNSUPPORTED            # overlaps, and is not the same matrix
    assert call(x, g, b, handle(cm, 8, 4, ct.addressof(g.contents.data_device.contents) - 64)) == UNSUPPORTED
    grad = lambda dy, x, g, t, gg, bg, eps=1e-5: lib.layer_norm_grad(dy, x, g, t, gg, bg, eps, 0.0, 1.0)
    dy, gg, bg = new(8, 4), new(8, 1), new(8, 1)
    assert grad(new(8, 4, on_device=0), x, g, y, gg, bg) == NOT_ON_DEVICE and grad(dy, x, g, y, gg, new(8, 1, on_device=0)) == NOT_ON_DEVICE
    assert grad(dy, new(8, 4, trans=1), g, y, gg, bg) == TRANSPOSED
    assert grad(dy, new(8, 3), g, y, gg, bg) == INCOMPATIBLE and grad(dy, x, g, y, new(1, 8), bg) == INCOMPATIBLE
    assert grad(dy, x, g, y, gg, gg) == UNSUPPORTED and grad(dy, x, g, y, g, bg) == UNSUPPORTED
    assert grad(dy, x, g, handle(cm, 8, 4, base + 128 - 4), gg, bg) == UNSUPPORTED
    assert grad(dy, x, g, y, gg, bg, eps=-1.0) == UNSUPPORTED


def test_dot_gated_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    w, x, b, y, pre = new(5, 12, trans=1), new(5, 3), new(12, 1), new(6, 3), new(12, 3)
    call = lambda w, x, b, y, pre, act=4: lib.dot_gated(w, x, b, y, pre, act)
    assert call(w, new(5, 3, on_device=0), b, y, pre) == NOT_ON_DEVICE and call(w, x, b, y, new(12, 3, on_device=0)) == NOT_ON_DEVICE
    assert call(w, x, b, new(6, 3, trans=1), pre) == TRANSPOSED and call(w, x, b, y, new(12, 3, trans=1)) == TRANSPOSED
    assert call(new(5, 13, trans=1), x, b, y, pre) == INCOMPATIBLE and call(new(5, 12), x, b, y, pre) == INCOMPATIBLE
    assert call(w, new(4, 3), b, y, pre) == INCOMPATIBLE and call(w, x, new(6, 1), y, pre) == INCOMPATIBLE
    assert call(w, x, b, y, new(6, 3)) == INCOMPATIBLE and call(w, x, b, new(12, 3), pre) == INCOMPATIBLE
    assert call(w, x, b, y, pre, act=6) == UNSUPPORTED and call(w, x, b, y, pre, act=-1) == UNSUPPORTED
    assert call(w, x, b, handle(cm, 6, 3, ct.addressof(x.contents.data_device.contents) + 8), pre) == UNSUPPORTED
    assert call(w, x, b, handle(cm, 6, 3, ct.addressof(pre.contents.data_device.contents)), pre) == UNSUPPORTED
    with pytest.raises(ValueError):
        m = cm.CUDAMatrix(np.zeros((2, 2)), copy_to_device=False)
        cm.dot_gated(m, m, act='softplus', target=m)
    dy, t, dw, dx, db = new(6, 3), new(12, 3), new(5, 12), new(5, 3), new(12, 1)
    grad = lambda dy, w, x, pre, t, dw, dx, db, act=4: lib.dot_gated_grad(dy, w, x, pre, t, dw, dx, db, act, 0.0, 1.0)
    assert grad(dy, w, x, pre, t, new(5, 12, on_device=0), dx, db) == NOT_ON_DEVICE
    assert grad(dy, w, x, new(12, 3, trans=1), t, dw, dx, db) == TRANSPOSED and grad(dy, w, x, pre, t, new(12, 5, trans=1), dx, db) == TRANSPOSED
    assert grad(dy, w, x, pre, t, new(12, 5), dx, db) == INCOMPATIBLE and grad(dy, w, x, pre, t, dw, new(3, 5), db) == INCOMPATIBLE
    assert grad(new(12, 3), w, x, pre, t, dw, dx, db) == INCOMPATIBLE and grad(dy, w, x, pre, t, dw, dx, new(6, 1)) == INCOMPATIBLE
    assert grad(dy, w, x, pre, t, dw, x, db) == UNSUPPORTED and grad(dy, w, x, pre, t, dw, dx, db, act=9) == UNSUPPORTED
    assert grad(dy, w, x, pre, t, handle(cm, 5, 12, ct.addressof(w.contents.data_device.contents)), dx, db) == UNSUPPORTED


def test_counter_dropout_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    x, y, r, s = new(6, 3), new(6, 3), new(6, 3), new(1, 1)
    call = lambda x, r, y, s, p=0.5: lib.counter_dropout(x, r, y, s, p, 2.0, 1, 2, 3)
    assert call(new(6, 3, on_device=0), r, y, s) == NOT_ON_DEVICE and call(x, r, y, new(1, 1, on_device=0)) == NOT_ON_DEVICE
    assert call(x, new(6, 3, trans=1), y, s) == TRANSPOSED
    assert call(x, new(3, 6), y, s) == INCOMPATIBLE and call(x, r, y, new(2, 1)) == INCOMPATIBLE and call(x, r, new(6, 4), s) == INCOMPATIBLE
    for p in (-0.1, 1.1, float('nan')):
        assert call(x, r, y, s, p) == UNSUPPORTED
    at = lambda m: ct.addressof(m.contents.data_device.contents)
    assert call(x, r, handle(cm, 6, 3, at(x) + 4), s) == UNSUPPORTED and call(x, r, handle(cm, 6, 3, at(r) - 4), s) == UNSUPPORTED
    assert call(x, r, y, handle(cm, 1, 1, at(y) + 8)) == UNSUPPORTED
    m = cm.CUDAMatrix(np.zeros((2, 2)), copy_to_device=False)
    for bad in (dict(dropprob=1.5, seed=1), dict(dropprob=float('nan'), seed=1), dict(dropprob=0.5, seed=-1), dict(dropprob=0.5, seed=1 << 64),
                dict(dropprob=0.5, seed=1, stream=1 << 32)):
        with pytest.raises(ValueError):
            cm.counter_dropout(m, **bad)


def test_log_probs_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    x, l, a, b, c, t, tl = new(9, 3), new(1, 3), new(1, 3), new(1, 3), new(1, 3), new(2, 3), new(2, 3)
    call = lib.log_probs
    assert call(new(9, 3, on_device=0), l, a, b, c, t, tl) == NOT_ON_DEVICE and call(x, l, a, b, new(1, 3, on_device=0), t, tl) == NOT_ON_DEVICE
    assert call(new(9, 3, trans=1), l, a, b, c, t, tl) == TRANSPOSED and call(x, l, new(1, 3, trans=1), b, c, t, tl) == TRANSPOSED
    assert call(x, None, a, b, c, t, tl) == INCOMPATIBLE and call(x, new(3, 1), a, b, c, t, tl) == INCOMPATIBLE
    assert call(x, l, a, new(1, 4), c, t, tl) == INCOMPATIBLE and call(x, l, a, b, c, t, new(3, 3)) == INCOMPATIBLE
    assert call(x, l, a, b, c, new(10, 3), new(10, 3)) == INCOMPATIBLE
    assert call(new(100, 3), l, a, b, c, new(65, 3), new(65, 3)) == UNSUPPORTED and call(new((1 << 24) + 1, 3), l, a, b, c, t, tl) == UNSUPPORTED
    assert call(x, l, a, a, c, t, tl) == UNSUPPORTED and call(x, l, l, b, c, t, tl) == UNSUPPORTED
    assert call(x, l, a, b, c, t, handle(cm, 2, 3, ct.addressof(x.contents.data_device.contents) + 8)) == UNSUPPORTED
    grad, y = lib.log_probs_grad, new(9, 3)
    assert grad(x, l, new(1, 3, on_device=0), a, b, c, y) == NOT_ON_DEVICE and grad(x, l, new(1, 3), a, b, c, new(9, 3, trans=1)) == TRANSPOSED
    assert grad(x, None, new(1, 3), a, b, c, y) == INCOMPATIBLE and grad(x, l, new(1, 3), a, b, None, y) == INCOMPATIBLE
    assert grad(x, l, new(1, 3), a, None, c, y) == INCOMPATIBLE and grad(x, l, new(1, 2), a, b, c, y) == INCOMPATIBLE
    assert grad(x, l, new(1, 3), a, b, c, new(3, 9)) == INCOMPATIBLE
    assert grad(x, l, new(1, 3), a, b, c, handle(cm, 9, 3, ct.addressof(x.contents.data_device.contents) + 4)) == UNSUPPORTED
