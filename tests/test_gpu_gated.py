"""Gated layers on the device against their definition in 64 bits.

Tolerances count roundings, u = 2^-24 the most that one to float32 is off.  A product of K terms a_k b_k is off by at most
c |a| . |b| (the vectors of magnitudes' product): full float32 multiply-adds round K times, c = (K + 1) u; operands split into two
parts keep each to 2^-21 of its column's largest magnitude or of itself, whichever is more, and leave out the product of the
small parts, c = 2^-19 with the largest magnitudes in the vectors' place, and what the tensor core's accumulation loses, chunks of
128 products at up to 2^-22 each product of the chunk's partial sum: the bound takes the larger form, K u + 2^-18."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["linear", "logistic", "relu", "silu", "gelu"]


def get(m):
    return np.array(m.asarray(), copy=True)


def within(got, want, bound):
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape and np.isfinite(got).all()
    off = np.abs(got - want) - np.broadcast_to(bound, want.shape)
    assert (off <= 0).all(), (float(off.max()), float(np.abs(got - want).max()))


def erf(x):
    return torch.erf(torch.from_numpy(np.ascontiguousarray(x))).numpy()


def act_exact(name, g):
    """act, slope, and bounds on how much either changes with g (their steepest slopes)."""
    if name == "linear":
        return g, np.ones_like(g), 1.0, 0.0
    if name == "relu":
        return np.maximum(g, 0), (g > 0).astype(np.float64), 1.0, None
    p = 0.5 * (1 + np.tanh(0.5 * g))
    if name == "logistic":
        return p, p * (1 - p), 0.25, 0.1
    if name == "silu":
        return g * p, p * (1 + g * (1 - p)), 1.1, 0.5
    cdf = 0.5 * (1 + erf(g / np.sqrt(2)))
    pdf = np.exp(-0.5 * g * g) / np.sqrt(2 * np.pi)
    return g * cdf, cdf + g * pdf, 1.13, 0.8


def act_off(name, a, g):
    """How far the device's act(g) may be off.  The logistic: within 6 roundings' worth, and flushed to 0 below 2^-126.  erfcf: within
    4 units in the last place (8 u); its argument -g / sqrt(2) carries two roundings (the constant's and the product's), and erfc's
    value changes by (2 t^2 + 1) times its argument's relative change (|t erfc'(t) / erfc(t)| = 2 t exp(-t^2) / (sqrt(pi) erfc(t)) is
    at most 2 t^2 + 1 for t > 0, as erfc(t) >= 2 t exp(-t^2) / (sqrt(pi) (2 t^2 + 1)), and less than 1 below), 2 t^2 = g^2."""
    return (12 + (2 * (g * g + 1) if name == "gelu" else 0)) * U * (np.abs(a) + np.abs(g) * 2.0 ** -20)


def product_bound(a, b, k):
    """How far op(a) . op(b) may be off: a is M x K, b K x N.  Magnitudes of each row of a and column of b at the largest."""
    big = np.abs(a).max(1, keepdims=True) * np.abs(b).max(0, keepdims=True)
    return (k + 2) * U * (np.abs(a) @ np.abs(b)) + 2.0 ** -18 * (np.abs(a) @ np.abs(b)) + 2.0 ** -30 * k * big


SHAPES = [(1, 1, 1), (5, 3, 2), (17, 33, 1), (64, 64, 64), (65, 130, 67), (100, 40, 9), (128, 256, 128), (300, 200, 8), (301, 203, 17),
          (784, 500, 100), (1357, 601, 203), (512, 1024, 300), (1000, 257, 129), (96, 2000, 5), (2048, 640, 1), (260, 388, 1028)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_gated_product_and_its_derivative(cm, shape, act):
    V, H, N = shape
    rng = np.random.default_rng(V + 3 * H + 7 * N + len(act))
    wg, wu = ((rng.standard_normal((V, H)) / np.sqrt(V)).astype(np.float32) for _ in range(2))
    x = (rng.standard_normal((V, N)) * (0.2 + rng.random((1, N)))).astype(np.float32)
    biased = (V + H + N) % 3 > 0
    bg, bu = ((0.5 * rng.standard_normal((H, 1))).astype(np.float32) if biased else None for _ in range(2))
    dy = rng.standard_normal((H, N)).astype(np.float32)
    G, X = cm.CUDAMatrix, x.astype(np.float64)
    A, B = wg.astype(np.float64), wu.astype(np.float64)
    g = A.T @ X + (bg if biased else 0)
    u = B.T @ X + (bu if biased else 0)
    eg, eu = product_bound(A.T, X, V) + U * np.abs(g), product_bound(B.T, X, V) + U * np.abs(u)
    a, slope, steep, bend = act_exact(act, g)
    y = a * u
    gm, um, out = cm.empty((H, N)), cm.empty((H, N)), cm.empty((H, N))
    bias = dict(gate_bias=G(bg), up_bias=G(bu)) if biased else {}
    ga, gb, gx = G(wg), G(wu), G(x)
    cm.gated_product(ga, gb, gx, out, activation=act, gate=gm, up=um, **bias)
    within(get(gm), g, eg)
    within(get(um), u, eu)
    ea = steep * eg + act_off(act, a, g)
    within(get(out), y, ea * np.abs(u) + np.abs(a) * eu + ea * eu + U * np.abs(y) + 1e-37)
    again = cm.gated_product(ga, gb, gx, activation=act, **bias)          # without the sums: the same bits
    assert np.array_equal(get(again), get(out))
    # the derivative, of the sums as they are on the device
    g32, u32 = get(gm).astype(np.float64), get(um).astype(np.float64)
    a, slope, _, _ = act_exact(act, g32)
    d = dy.astype(np.float64)
    dg, du = d * u32 * slope, d * a
    e_slope = 20 * U * (1 + np.abs(g32))
    edg, edu = np.abs(d * u32) * e_slope + 3 * U * np.abs(dg), np.abs(d) * act_off(act, a, g32) + 2 * U * np.abs(du)
    dx, dwg, dwu = cm.empty((V, N)), cm.empty((V, H)), cm.empty((V, H))
    dbg, dbu = (G(np.full((H, 1), 9.0)) for _ in range(2))
    cm.gated_product_deriv(G(dy), gm, um, ga, gb, gx, activation=act, grad_x=dx, grad_gate_w=dwg, grad_up_w=dwu, grad_gate_bias=dbg,
                           grad_up_bias=dbu)
    within(get(gm), dg, edg + 1e-37)
    within(get(um), du, edu + 1e-37)
    within(get(dwg), X @ dg.T, product_bound(X, dg.T, N) + np.abs(X) @ edg.T + 1e-30)
    within(get(dwu), X @ du.T, product_bound(X, du.T, N) + np.abs(X) @ edu.T + 1e-30)
    within(get(dx), A @ dg + B @ du, product_bound(A, dg, H) + product_bound(B, du, H) + np.abs(A) @ edg + np.abs(B) @ edu +
           2 * U * np.abs(A @ dg) + 1e-30)
    within(get(dbg), dg.sum(1, keepdims=True), (N + 8) * U * np.abs(dg).sum(1, keepdims=True) + edg.sum(1, keepdims=True) + 1e-37)
    within(get(dbu), du.sum(1, keepdims=True), (N + 8) * U * np.abs(du).sum(1, keepdims=True) + edu.sum(1, keepdims=True) + 1e-37)
    assert np.array_equal(get(gx), x) and np.array_equal(get(ga), wg) and np.array_equal(get(gb), wu)
    assert cm.read_status() == 0


def test_gradient_against_differences(cm):
    rng = np.random.default_rng(11)
    V, H, N = 24, 20, 6
    wg, wu, x, dy = (rng.standard_normal(s).astype(np.float32) for s in ((V, H), (V, H), (V, N), (H, N)))
    for act in ACTS:
        gm, um = cm.empty((H, N)), cm.empty((H, N))
        cm.gated_product(cm.CUDAMatrix(wg), cm.CUDAMatrix(wu), cm.CUDAMatrix(x), activation=act, gate=gm, up=um)
        dx, dw = cm.empty((V, N)), cm.empty((V, H))
        cm.gated_product_deriv(cm.CUDAMatrix(dy), gm, um, cm.CUDAMatrix(wg), cm.CUDAMatrix(wu), cm.CUDAMatrix(x), activation=act, grad_x=dx,
                               grad_gate_w=dw)

        def f(a, v):
            return (act_exact(act, a.T @ v)[0] * (wu.astype(np.float64).T @ v) * dy).sum()
        a64, x64, d = wg.astype(np.float64), x.astype(np.float64), 1e-6
        for r, c in ((0, 0), (23, 5), (7, 3)):
            e, s = np.zeros_like(x64), np.zeros_like(a64)
            e[r, c] = s[r, c] = d
            size = np.abs(get(dx)).max()
            assert abs((f(a64, x64 + e) - f(a64, x64 - e)) / (2 * d) - get(dx)[r, c]) < 1e-5 * size
            assert abs((f(a64 + s, x64) - f(a64 - s, x64)) / (2 * d) - get(dw)[r, c]) < 1e-5 * np.abs(get(dw)).max()


def test_gradients_over_no_cases_are_zero(cm):
    w, x, h = cm.CUDAMatrix(np.ones((6, 4))), cm.empty((6, 0)), cm.empty((4, 0))
    dw, db = cm.CUDAMatrix(np.ones((6, 4))), cm.CUDAMatrix(np.ones((4, 1)))
    cm.gated_product_deriv(h, h, h, w, w, x, grad_gate_w=dw, grad_up_bias=db)
    assert (get(dw) == 0).all() and (get(db) == 0).all()


def test_infinities_and_nan_stay_in_their_case(cm):
    rng = np.random.default_rng(12)
    for V, H, N in ((40, 30, 5), (512, 300, 200)):
        wg, wu, x = (rng.standard_normal(s).astype(np.float32) for s in ((V, H), (V, H), (V, N)))
        clean = get(cm.gated_product(cm.CUDAMatrix(wg), cm.CUDAMatrix(wu), cm.CUDAMatrix(x), activation="silu"))
        x[3, 1], x[4, 3] = np.nan, np.inf
        got = get(cm.gated_product(cm.CUDAMatrix(wg), cm.CUDAMatrix(wu), cm.CUDAMatrix(x), activation="silu"))
        keep = [c for c in range(N) if c not in (1, 3)]
        assert np.array_equal(got[:, keep], clean[:, keep])
        assert np.isnan(got[:, 1]).all() and not np.isfinite(got[:, 3]).all()
