"""What layer normalisation, dropout by key and log probabilities refuse.  The checks come before anything touches a device, so
they are tested without one, on handles that name no memory."""
import ctypes as ct

import pytest

from deepnet_b200 import b200mat as cm

DIMENSIONS, TRANSPOSED, NOT_ON_DEVICE, UNSUPPORTED = -1, -5, -8, -9


_place = [1 << 20]


def mat(rows, cols, on_device=1, trans=0, at=None):
    """A handle of memory that nobody has, each somewhere else (or `at` an address)."""
    m = cm.cudamat()
    m.size[0], m.size[1], m.on_device, m.is_trans = rows, cols, on_device, trans
    m.data_device = ct.cast(_place[0] if at is None else at, ct.POINTER(ct.c_float))
    _place[0] += (4 * rows * cols + 255) // 256 * 256
    return ct.pointer(m)


def norm(x, gain, bias, y, stats, eps=1e-5):
    return cm._lib.layer_norm(x, gain, bias, y, stats, ct.c_float(eps))


def test_layer_norm_refuses():
    x = lambda **k: mat(8, 5, **k)
    assert norm(x(), None, None, mat(8, 4), None) == DIMENSIONS
    assert norm(x(), mat(7, 1), None, x(), None) == DIMENSIONS
    assert norm(x(), mat(4, 2), None, x(), None) == DIMENSIONS          # eight values, but no vector
    assert norm(x(), None, mat(1, 9), x(), None) == DIMENSIONS
    assert norm(x(), None, None, x(), mat(5, 2)) == DIMENSIONS
    assert norm(x(trans=1), None, None, x(), None) == TRANSPOSED
    assert norm(x(), None, None, x(trans=1), None) == TRANSPOSED
    assert norm(x(on_device=0), None, None, x(), None) == NOT_ON_DEVICE
    assert norm(x(), mat(8, 1, on_device=0), None, x(), None) == NOT_ON_DEVICE
    for eps in (-1e-5, float("nan")):
        assert norm(x(), None, None, x(), None, eps) == UNSUPPORTED
    assert norm(mat(0, 5), None, None, mat(0, 5), None) == 0 and norm(mat(8, 0), None, None, mat(8, 0), mat(2, 0)) == 0


def test_layer_norm_deriv_refuses():
    f = cm._lib.layer_norm_deriv
    x, st = (lambda **k: mat(8, 5, **k)), (lambda **k: mat(2, 5, **k))
    assert f(mat(8, 4), x(), st(), None, x(), None, None) == DIMENSIONS
    assert f(x(), x(), mat(1, 5), None, x(), None, None) == DIMENSIONS
    assert f(x(), x(), st(), None, mat(5, 8), None, None) == DIMENSIONS
    assert f(x(), x(), st(), mat(5, 1), x(), None, None) == DIMENSIONS
    assert f(x(), x(), st(), None, x(), mat(9, 1), None) == DIMENSIONS
    assert f(x(), x(), st(), None, x(), None, mat(1, 7)) == DIMENSIONS
    assert f(x(trans=1), x(), st(), None, x(), None, None) == TRANSPOSED
    assert f(x(), x(), st(on_device=0), None, x(), None, None) == NOT_ON_DEVICE


def test_dropout_scaled_refuses_and_draws_nothing():
    def f(x, add, y, p=0.5):
        state = cm.rnd_struct(3, 7)
        err = cm._lib.dropout_scaled(ct.byref(state), x, add, y, ct.c_float(p))
        assert (state.seed, state.calls) == (3, 8 if err == 0 else 7)
        return err
    assert f(mat(4, 3), None, mat(3, 4)) == DIMENSIONS
    assert f(mat(4, 3), mat(4, 2), mat(4, 3)) == DIMENSIONS
    assert f(mat(4, 3, trans=1), None, mat(4, 3)) == TRANSPOSED
    assert f(mat(4, 3), mat(4, 3, trans=1), mat(4, 3)) == TRANSPOSED
    assert f(mat(4, 3), None, mat(4, 3, on_device=0)) == NOT_ON_DEVICE
    for p in (-0.1, 1.5, float("nan")):
        assert f(mat(4, 3), None, mat(4, 3), p) == UNSUPPORTED
    assert f(mat(0, 3), None, mat(0, 3)) == 0


def test_log_prob_refuses():
    f = cm._lib.log_prob
    z, row = (lambda **k: mat(10, 6, **k)), (lambda **k: mat(1, 6, **k))
    assert f(z(), mat(1, 5), row(), None, None, None, None) == DIMENSIONS
    assert f(z(), mat(6, 1), row(), None, None, None, None) == DIMENSIONS
    assert f(z(), row(), None, None, None, None, None) == DIMENSIONS               # a token without a place for its result
    assert f(z(), None, row(), None, None, None, None) == DIMENSIONS
    assert f(z(), row(), row(), mat(1, 7), None, None, None) == DIMENSIONS
    assert f(z(), row(), row(), None, mat(6, 2), None, None) == DIMENSIONS
    assert f(z(), row(), row(), None, None, mat(3, 6), None) == DIMENSIONS
    assert f(z(), row(), row(), None, None, mat(3, 6), mat(2, 6)) == DIMENSIONS
    assert f(z(), row(), row(), None, None, mat(11, 6), mat(11, 6)) == DIMENSIONS  # more of them than tokens
    assert f(mat(40, 6), None, None, None, None, mat(33, 6), mat(33, 6)) == UNSUPPORTED
    assert f(mat(0, 6), row(), row(), None, None, None, None) == UNSUPPORTED
    assert f(mat((1 << 24) + 1, 6), row(), row(), None, None, None, None) == UNSUPPORTED
    assert f(z(trans=1), row(), row(), None, None, None, None) == TRANSPOSED
    assert f(z(on_device=0), row(), row(), None, None, None, None) == NOT_ON_DEVICE
    assert f(z(), row(on_device=0), row(), None, None, None, None) == NOT_ON_DEVICE
    assert f(mat(10, 0), mat(1, 0), mat(1, 0), None, None, None, None) == 0


def test_log_prob_deriv_refuses():
    f = cm._lib.log_prob_deriv
    z, row, st = (lambda **k: mat(10, 6, **k)), (lambda: mat(1, 6)), (lambda: mat(2, 6))
    assert f(z(), row(), st(), row(), None, None, mat(10, 5)) == DIMENSIONS
    assert f(z(), row(), mat(2, 5), row(), None, None, z()) == DIMENSIONS
    assert f(z(), None, st(), row(), None, None, z()) == DIMENSIONS                # a gradient of log probabilities of no tokens
    assert f(z(), row(), st(), row(), None, row(), z()) == DIMENSIONS              # a gradient of entropies that are not given
    assert f(z(trans=1), row(), st(), row(), None, None, z()) == TRANSPOSED
    assert f(z(), row(), st(), row(), None, None, z(on_device=0)) == NOT_ON_DEVICE
    long = lambda: mat((1 << 24) + 1, 6)
    assert f(long(), row(), st(), row(), None, None, long()) == UNSUPPORTED


def test_gated_product_refuses():
    def f(wg, wu, x, bg=None, bu=None, act=1, gate=None, up=None, y=None, planes=(None,) * 3):
        return cm._lib.gated_product(wg, wu, x, bg, bu, ct.c_int(act), *planes, gate, up, y if y is not None else mat(7, 5))
    w, x = (lambda **k: mat(9, 7, **k)), (lambda **k: mat(9, 5, **k))
    assert f(w(), mat(9, 6), x()) == DIMENSIONS
    assert f(w(), w(), mat(8, 5)) == DIMENSIONS
    assert f(w(), w(), x(), y=mat(7, 4)) == DIMENSIONS
    assert f(w(), w(), x(), bg=mat(9, 1)) == DIMENSIONS
    assert f(w(), w(), x(), bu=mat(7, 2)) == DIMENSIONS
    assert f(w(), w(), x(), gate=mat(7, 5)) == DIMENSIONS               # one of the two sums
    assert f(w(), w(), x(), gate=mat(7, 5), up=mat(5, 7)) == DIMENSIONS
    assert f(w(trans=1), w(), x()) == TRANSPOSED and f(w(), w(), x(trans=1)) == TRANSPOSED
    assert f(w(), w(on_device=0), x()) == NOT_ON_DEVICE and f(w(), w(), x(), y=mat(7, 5, on_device=0)) == NOT_ON_DEVICE
    assert f(w(), w(), x(), act=-1) == UNSUPPORTED and f(w(), w(), x(), act=5) == UNSUPPORTED
    assert f(w(), w(), mat(9, 0), y=mat(7, 0)) == 0
    # planes: all three, of the weights' shapes, on 16 bytes
    good = lambda: [mat(16, 7), mat(16, 7), mat(2, 7)]
    fill = lambda planes: cm._lib.gated_planes(w(), w(), *planes)
    for i, bad, err in ((0, None, DIMENSIONS), (1, mat(9, 7), DIMENSIONS), (2, mat(7, 2), DIMENSIONS), (1, mat(16, 7, on_device=0), NOT_ON_DEVICE),
                        (0, mat(16, 7, trans=1), TRANSPOSED)):
        planes = good()
        planes[i] = bad
        assert f(w(), w(), x(), planes=planes) == err and (fill(planes) == err)
    planes = good()
    planes[1] = mat(16, 7, at=(1 << 40) + 8)
    assert f(w(), w(), x(), planes=planes) == UNSUPPORTED and fill(planes) == UNSUPPORTED
    with pytest.raises(cm.CUDAMatException):
        cm._gated_activation("softmax")


def test_gated_product_deriv_refuses():
    def f(dy=None, gate=None, up=None, wg=None, wu=None, x=None, act=1, out=(None,) * 5):
        d = lambda m, r, c: m if m is not None else mat(r, c)
        return cm._lib.gated_product_deriv(d(dy, 7, 5), d(gate, 7, 5), d(up, 7, 5), d(wg, 9, 7), d(wu, 9, 7), d(x, 9, 5), ct.c_int(act),
                                          None, None, None, *out)
    assert f(dy=mat(7, 4)) == DIMENSIONS and f(up=mat(5, 7)) == DIMENSIONS and f(wu=mat(7, 9)) == DIMENSIONS
    assert f(out=(mat(9, 4), None, None, None, None)) == DIMENSIONS
    assert f(out=(None, mat(7, 9), None, None, None)) == DIMENSIONS
    assert f(out=(None, None, None, mat(9, 1), None)) == DIMENSIONS
    assert f(gate=mat(7, 5, trans=1)) == TRANSPOSED and f(out=(None, None, mat(9, 7, trans=1), None, None)) == TRANSPOSED
    assert f(x=mat(9, 5, on_device=0)) == NOT_ON_DEVICE and f(out=(None, None, None, None, mat(7, 1, on_device=0))) == NOT_ON_DEVICE
    assert f(act=9) == UNSUPPORTED


def test_results_may_not_lie_over_other_arguments():
    """Square shapes, where every matrix could stand for every other; one byte in common is enough."""
    sq = lambda at: mat(8, 8, at=at)
    names = ["wg", "wu", "x", "gate", "up", "y"]
    for i, a in enumerate(names):
        for b in names[:i]:
            if a in ("wg", "wu", "x") and b in ("wg", "wu", "x"):
                continue
            place = {n: (1 << 30) + 4096 * k for k, n in enumerate(names)}
            place[a] = place[b] + 252
            m = {n: sq(p) for n, p in place.items()}
            assert cm._lib.gated_product(m["wg"], m["wu"], m["x"], None, None, ct.c_int(1), None, None, None, m["gate"], m["up"],
                                         m["y"]) == UNSUPPORTED, (a, b)
    names = ["dy", "wg", "wu", "x", "gate", "up", "dx", "dwg", "dwu"]
    for i, a in enumerate(names):
        for b in names[:i]:
            if i < 4:
                continue
            place = {n: (1 << 30) + 4096 * k for k, n in enumerate(names)}
            place[a] = place[b] - 252
            m = {n: sq(p) for n, p in place.items()}
            assert cm._lib.gated_product_deriv(m["dy"], m["gate"], m["up"], m["wg"], m["wu"], m["x"], ct.c_int(1), None, None, None, m["dx"],
                                               m["dwg"], m["dwu"], None, None) == UNSUPPORTED, (a, b)


def test_results_lie_over_an_argument_in_place_or_not_at_all():
    """A byte in common is enough, but for the places that the documentation gives; what is refused draws nothing."""
    lib, at = cm._lib, 1 << 30
    h, w = 16, 8
    x = lambda off=0, rows=h, cols=w: mat(rows, cols, at=at + off)
    far = lambda rows=h, cols=w: mat(rows, cols)
    for off in (4, -4, 4 * h, 4 * h * w - 4, 4 - 4 * h * w):
        assert norm(x(), None, None, x(off), None) == UNSUPPORTED
        assert lib.layer_norm_deriv(x(), far(), far(2), None, x(off), None, None) == UNSUPPORTED
        assert lib.layer_norm_deriv(far(), x(), far(2), None, x(off), None, None) == UNSUPPORTED
        assert lib.log_prob_deriv(x(), far(1), far(2), far(1), None, None, x(off)) == UNSUPPORTED
        for m, add in ((x(), None), (far(), x())):
            state = cm.rnd_struct(3, 7)
            assert lib.dropout_scaled(ct.byref(state), m, add, x(off), ct.c_float(0.5)) == UNSUPPORTED and state.calls == 7
    inside = 4 * (h * w - 1)
    assert norm(x(), None, None, far(), x(inside, 2)) == UNSUPPORTED and norm(x(), None, None, x(), x(inside, 2)) == UNSUPPORTED
    assert norm(far(), x(inside, h, 1), None, x(), None) == UNSUPPORTED and norm(far(), None, x(inside, 1, h), x(), None) == UNSUPPORTED
    deriv = lambda *a: lib.layer_norm_deriv(*a)
    assert deriv(far(), far(), x(inside, 2), None, x(), None, None) == UNSUPPORTED
    assert deriv(far(), far(), far(2), x(inside, h, 1), x(), None, None) == UNSUPPORTED
    assert deriv(x(), far(), far(2), None, far(), x(inside, h, 1), None) == UNSUPPORTED
    assert deriv(far(), x(), far(2), None, far(), None, x(inside, h, 1)) == UNSUPPORTED
    assert deriv(far(), far(), far(2), None, far(), x(0, h, 1), x(60, h, 1)) == UNSUPPORTED
    assert deriv(far(), far(), far(2), x(0, h, 1), far(), x(4, h, 1), None) == UNSUPPORTED
    row = lambda off: x(off, 1)
    score = lambda z, t, *out: lib.log_prob(z, t, *out)
    none = [None] * 5
    for i, rows in enumerate((1, 1, 2, 3, 3)):
        out = [far(1)] + none[1:]
        out[i] = x(inside, rows)
        if i > 2:
            out[7 - i] = far(3)
        assert score(x(), far(1), *out) == UNSUPPORTED
        for j in range(i):
            two = [far(1), far(1), far(2), far(3), far(3)]
            two[i], two[j] = x(0, rows), x(4, (1, 1, 2, 3, 3)[j])
            assert score(far(), far(1), *two) == UNSUPPORTED
    assert score(far(), row(0), row(4), *none[1:]) == UNSUPPORTED
    for i in range(5):
        args = [far(1), far(2), far(1), far(1), far(1)]
        args[i] = x(inside, 2 if i == 1 else 1)
        assert lib.log_prob_deriv(far(), *args, x()) == UNSUPPORTED
