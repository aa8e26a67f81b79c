"""CPU-only: the float64 restatements of embeddings, gated recurrences and sampling against differences and other ways to the same
numbers; and what the library refuses before it touches a device."""
import ctypes as ct

import numpy as np
import pytest

from oracle import sequence_oracle as seq
from test_oracle_tokens import INCOMPATIBLE, NOT_ON_DEVICE, TRANSPOSED, UNSUPPORTED, Space, close, differences, handle


@pytest.fixture
def cm():
    from deepnet_amd import cudamat
    return cudamat


def test_embed_gradient_against_differences():
    rng = np.random.default_rng(1)
    e, dy, labels = rng.standard_normal((3, 5)), rng.standard_normal((3, 7)), [4, 0, -1, 0, 5, 2.0, np.nan]
    g, _, n = seq.embed_grad(dy, labels, 5, 1.5)
    close(g, differences(lambda v: np.sum(dy * seq.embed(v, labels, 1.5)), e))
    assert n.tolist() == [2, 0, 1, 0, 1] and not seq.embed(e, labels)[:, [2, 4, 6]].any()


@pytest.mark.parametrize("offsets", [None, [0, 3, 3, 8], [1, 2, 6, 7]])
def test_gated_scan_gradients_against_differences(offsets):
    rng = np.random.default_rng(2)
    f, w, n = 3, 9, 3
    at = seq.borders(w, offsets, n)
    pre, state, dy, dlast = (rng.standard_normal(s) for s in ((2 * f, w), (f, n), (f, w), (f, n)))
    def value(p, s0):
        y, last = seq.gated_scan(p, at, s0)[:2]
        return np.nansum(dy * y) + np.sum(dlast * last)
    dpre, dstate = seq.gated_scan_grad(dy, pre, seq.gated_scan(pre, at, state)[0], at, state, dlast)[:2]
    close(np.nan_to_num(dpre), differences(lambda v: value(v, state), pre))
    close(dstate, differences(lambda v: value(pre, v), state))


def test_gated_scan_is_the_weighted_sum_that_it_unrolls_to():
    rng = np.random.default_rng(3)
    pre, h0 = rng.standard_normal((4, 6)), rng.standard_normal((2, 1))
    a, s, u = seq.gates(pre)
    y = seq.gated_scan(pre, [0, 6], h0)[0]
    for t in range(6):
        close(y[:, t], np.prod(a[:, :t + 1], axis=1) * h0[:, 0] + sum(np.prod(a[:, j + 1:t + 1], axis=1) * s[:, j] * u[:, j] for j in range(t + 1)))


def test_sample_token_by_hand():
    x = np.log([0.1, 0.4, 0.2, 0.3])
    assert [seq.sample_token(x, u)[0] for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.999, 1.0)] == [0, 0, 1, 1, 2, 2, 3, 3, 3]
    assert seq.sample_token(x, 0.5, top_k=2)[2] == [1, 3] and seq.sample_token(x, 0.5, top_p=0.65)[2] == [1, 3]
    assert seq.sample_token(x, 0.5, top_p=0.71)[2] == [1, 2, 3] and seq.sample_token(x, 0.5, top_p=0.0)[2] == [1]
    assert seq.sample_token(x, 0.5, min_p=0.49)[2] == [1, 2, 3] and seq.sample_token(x, 0.5, min_p=7.0)[2] == [1]
    assert seq.sample_token(x, 0.5, top_k=3, top_p=0.75)[2] == [1, 3] and seq.sample_token(x, 0.5, temperature=0.0)[:2] == (1, 0.0)
    token, logp, _ = seq.sample_token(x, 0.99, top_k=2)
    assert token == 3 and abs(logp - np.log(3 / 7)) < 1e-6
    assert seq.sample_token([0, 0, 0, 0], 0.3, top_p=0.5)[2] == [0, 1] and seq.sample_token([-np.inf] * 3, 0.5)[0] == -1
    # the shares of many draws
    rng = np.random.default_rng(4)
    draws = [seq.sample_token(x, u, temperature=2.0)[0] for u in rng.random(20000)]
    p = np.sqrt([0.1, 0.4, 0.2, 0.3])
    assert np.max(np.abs(np.bincount(draws, minlength=4) / 20000 - p / p.sum())) < 5 * np.sqrt(0.25 / 20000)


# ---- what the library refuses

def at(m):
    return ct.addressof(m.contents.data_device.contents)


def test_embed_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    e, l, y = new(6, 9), new(1, 4), new(6, 4)
    call = lambda e, l, y: lib.embed(e, l, y, 1.0)
    for i, m in enumerate((new(6, 9, on_device=0), new(1, 4, on_device=0), new(6, 4, on_device=0))):
        a = [e, l, y]; a[i] = m
        assert call(*a) == NOT_ON_DEVICE
    for i, m in enumerate((new(6, 9, trans=1), new(1, 4, trans=1), new(6, 4, trans=1))):
        a = [e, l, y]; a[i] = m
        assert call(*a) == TRANSPOSED
    assert call(e, new(4, 1), y) == INCOMPATIBLE and call(e, l, new(6, 5)) == INCOMPATIBLE and call(e, l, new(5, 4)) == INCOMPATIBLE
    assert call(e, l, handle(cm, 6, 4, at(e) + 8)) == UNSUPPORTED and call(e, l, handle(cm, 6, 4, at(l) - 8)) == UNSUPPORTED
    assert call(new(6, (1 << 24) + 1), l, y) == UNSUPPORTED
    grad = lambda dy, l, g: lib.embed_grad(dy, l, g, 0.0, 1.0)
    dy, g = new(6, 4), new(6, 9)
    assert grad(new(6, 4, on_device=0), l, g) == NOT_ON_DEVICE and grad(dy, l, new(6, 9, trans=1)) == TRANSPOSED
    assert grad(dy, new(1, 5), g) == INCOMPATIBLE and grad(dy, l, new(5, 9)) == INCOMPATIBLE
    assert grad(dy, l, handle(cm, 6, 9, at(dy) - 16)) == UNSUPPORTED and grad(dy, l, handle(cm, 6, 9, at(l))) == UNSUPPORTED
    assert grad(dy, l, handle(cm, 6, (1 << 24) + 1, 1 << 44)) == UNSUPPORTED


def test_gated_scan_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    f, w, n = 5, 12, 3
    pre, y, o, s, t = new(2 * f, w), new(f, w), new(1, n + 1), new(f, n), new(f, n)
    call = lambda pre, o, s, y, t, k=0: lib.gated_scan(pre, o, s, y, t, k)
    good = [pre, o, s, y, t]
    for i, shape in enumerate(((2 * f, w), (1, n + 1), (f, n), (f, w), (f, n))):
        a = list(good); a[i] = new(*shape, on_device=0)
        assert call(*a) == NOT_ON_DEVICE
        a[i] = new(*shape, trans=1)
        assert call(*a) == TRANSPOSED
        a[i] = new(shape[0], shape[1] + 1)
        assert call(*a, 3) == INCOMPATIBLE
        a[i] = new(shape[0] + 1, shape[1])
        assert call(*a, 3) == INCOMPATIBLE
    assert call(pre, o, None, y, None, 2) == INCOMPATIBLE and call(pre, None, s, y, None, 2) == INCOMPATIBLE
    assert call(pre, None, None, y, None, 5) == INCOMPATIBLE and call(pre, None, None, y, None, -1) == INCOMPATIBLE
    assert call(pre, new(1, 1), None, y, None) == INCOMPATIBLE
    assert call(pre, o, s, handle(cm, f, w, at(pre)), t) == UNSUPPORTED and call(pre, o, s, y, handle(cm, f, n, at(s) + 4)) == UNSUPPORTED
    assert call(pre, o, s, y, handle(cm, f, n, at(y) + 16)) == UNSUPPORTED and call(pre, o, handle(cm, f, n, at(y)), y, None) == UNSUPPORTED
    assert call(pre, handle(cm, 1, n + 1, at(y) + 4), s, y, t) == UNSUPPORTED and call(pre, handle(cm, 1, n + 1, at(t)), s, y, t) == UNSUPPORTED
    big = (1 << 24) + 1
    assert call(handle(cm, 2, big, 1 << 42), o, None, handle(cm, 1, big, 1 << 43), None) == UNSUPPORTED
    dy, out, dp, dl, ds = new(f, w), new(f, w), new(2 * f, w), new(f, n), new(f, n)
    grad = lambda dy, pre, out, o, s, dl, dp, ds, k=0: lib.gated_scan_grad(dy, pre, out, o, s, dl, dp, ds, k)
    good = [dy, pre, out, o, s, dl, dp, ds]
    for i, shape in enumerate(((f, w), (2 * f, w), (f, w), (1, n + 1), (f, n), (f, n), (2 * f, w), (f, n))):
        a = list(good); a[i] = new(*shape, on_device=0)
        assert grad(*a) == NOT_ON_DEVICE
        a[i] = new(*shape, trans=1)
        assert grad(*a) == TRANSPOSED
        a[i] = new(shape[0], shape[1] + 1)
        assert grad(*a, 3) == INCOMPATIBLE
    for i in (0, 2, 3, 4, 5):
        a = list(good); a[6] = handle(cm, 2 * f, w, at(a[i]) - 4)
        assert grad(*a) == UNSUPPORTED
    for i in (0, 1, 2, 3, 4, 6):
        a = list(good); a[7] = handle(cm, f, n, at(a[i]))
        assert grad(*a) == UNSUPPORTED
    a = list(good); a[6] = handle(cm, 2 * f, w, at(pre) + 4)
    assert grad(*a) == UNSUPPORTED
    a = list(good); a[7] = handle(cm, f, n, at(dl) + 4)
    assert grad(*a) == UNSUPPORTED


def test_gated_scan_refuses_more_sequences_than_it_counts(cm):
    """Of 2^30 sequences every number that the kernels step through them by stays below 2^31."""
    lib, new, n = cm._cudamat, Space(cm), (1 << 30) + 1
    pre, y, o = new(2, 12), new(1, 12), handle(cm, 1, n + 1, 1 << 42)
    assert lib.gated_scan(pre, o, None, y, None, 0) == UNSUPPORTED and lib.gated_scan(pre, o, None, y, handle(cm, 1, n, 1 << 43), n) == UNSUPPORTED
    assert lib.gated_scan_grad(new(1, 12), pre, y, o, None, None, new(2, 12), None, 0) == UNSUPPORTED


def test_sample_tokens_refusals(cm):
    lib, new = cm._cudamat, Space(cm)
    shapes = [(9, 3)] + [(1, 3)] * 7
    good = [new(*s) for s in shapes]
    call = lambda a: lib.sample_tokens(*a, 1.0, 0.0, 1.0, 0.0)
    for i, s in enumerate(shapes):
        a = list(good); a[i] = new(*s, on_device=0)
        assert call(a) == NOT_ON_DEVICE
        a[i] = new(*s, trans=1)
        assert call(a) == TRANSPOSED
        a[i] = new(s[0], s[1] + 1)
        assert call(a) == INCOMPATIBLE
        if i:
            a[i] = new(3, 1)
            assert call(a) == INCOMPATIBLE
            a[i] = good[0] if i < 6 else good[1]
            assert call(a) == (INCOMPATIBLE if i < 6 else UNSUPPORTED)
    for i in (6, 7):
        for k in range(6):
            a = list(good); a[i] = handle(cm, 1, 3, at(good[k]) + 4)
            assert call(a) == UNSUPPORTED
    a = list(good); a[7] = a[6]
    assert call(a) == UNSUPPORTED
    a = list(good); a[0] = handle(cm, (1 << 24) + 1, 3, 1 << 42)
    assert call(a) == UNSUPPORTED
    for i in (1, 6):
        a = list(good); a[i] = None
        assert call(a) == INCOMPATIBLE


def test_calls_without_columns_queue_nothing(cm):
    lib, new = cm._cudamat, Space(cm)
    assert lib.embed(new(6, 9), new(1, 0), new(6, 0), 1.0) == 0 and lib.embed(new(0, 9), new(1, 4), new(0, 4), 1.0) == 0
    assert lib.embed_grad(new(6, 4), new(1, 4), new(6, 0), 0.0, 1.0) == 0
    assert lib.gated_scan(new(10, 0), None, None, new(5, 0), None, 1) == 0 and lib.gated_scan(new(0, 4), None, None, new(0, 4), None, 1) == 0
    assert lib.sample_tokens(*[new(9, 0)] + [new(1, 0)] * 5 + [new(1, 0), new(1, 0)], 1.0, 0.0, 1.0, 0.0) == 0
