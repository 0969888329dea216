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


def on_path(cm, path, call):
    cm.set_gemm_path(path)
    try:
        return call()
    finally:
        cm.set_gemm_path(0)


def columns_bound(w, x, k):
    """`product_bound` for operands with a power of two a column: the magnitudes of w's and x's columns, whatever the others'."""
    aw, ax = np.abs(w), np.abs(x)
    return (k * U + 2.0 ** -18) * (aw.T @ ax) + 2.0 ** -30 * k * aw.max(0)[:, None] * ax.max(0)[None]


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("shape", SHAPES + [(64, 128, 256), (65, 129, 257), (40, 600, 33), (4096, 300, 70), (130, 5000, 600), (1000, 9, 3000)])
def test_tensor_cores_and_cuda_cores_give_the_products(cm, shape, path):
    """Either kernel at every size, over columns whose magnitudes lie up to 2^80 apart, with and without planes kept by the caller."""
    V, H, N = shape
    rng = np.random.default_rng(V * 5 + H * 3 + N)
    wg, wu = (np.ldexp(rng.standard_normal((V, H)), rng.integers(-30, 10, (1, H))).astype(np.float32) for _ in range(2))
    x = np.ldexp(rng.standard_normal((V, N)), rng.integers(-30, 10, (1, N))).astype(np.float32)
    x[:, N // 2] = 0
    wg[:, H // 3] = 0
    ga, gb, gx = cm.CUDAMatrix(wg), cm.CUDAMatrix(wu), cm.CUDAMatrix(x)
    gm, um, y, y2 = (cm.empty((H, N)) for _ in range(4))
    on_path(cm, path, lambda: cm.gated_product(ga, gb, gx, y, activation="linear", gate=gm, up=um))
    A, B, X = (v.astype(np.float64) for v in (wg, wu, x))
    within(get(gm), A.T @ X, columns_bound(A, X, V) + 1e-37)
    within(get(um), B.T @ X, columns_bound(B, X, V) + 1e-37)
    within(get(y), get(gm).astype(np.float64) * get(um), U * np.abs(get(gm).astype(np.float64) * get(um)) + 1e-37)
    planes = cm.GatedPlanes(ga, gb)
    on_path(cm, path, lambda: cm.gated_product(ga, gb, gx, y2, activation="linear", planes=planes))
    assert np.array_equal(get(y2), get(y))
    other = cm.CUDAMatrix(wg[:, ::-1])                                      # filled again
    planes.fill(other, gb)
    on_path(cm, path, lambda: cm.gated_product(other, gb, gx, y2, activation="linear", gate=um, up=cm.empty((H, N)), planes=planes))
    assert np.array_equal(get(um), get(gm)[::-1])
    assert cm.read_status() == 0


def test_extreme_magnitudes_on_tensor_cores(cm):
    """Powers of two whose product is no normal number, and results at the ends of the range."""
    rng = np.random.default_rng(21)
    V, H, N = 200, 140, 40
    w, x = rng.standard_normal((V, H)), rng.standard_normal((V, N))
    for ew, ex in ((-70, -70), (60, 50), (-100, 100), (90, -110)):
        a, b = np.ldexp(w, ew).astype(np.float32), np.ldexp(x, ex).astype(np.float32)
        gm, um = cm.empty((H, N)), cm.empty((H, N))
        on_path(cm, 1, lambda: cm.gated_product(cm.CUDAMatrix(a), cm.CUDAMatrix(a), cm.CUDAMatrix(b), activation="linear", gate=gm, up=um))
        A, X = a.astype(np.float64), b.astype(np.float64)
        within(get(gm), A.T @ X, columns_bound(A, X, V) + 2.0 ** -126)
        assert np.array_equal(get(gm), get(um))
    assert cm.read_status() == 0


@pytest.mark.parametrize("off", [1, 2, 3])
def test_matrices_that_start_anywhere(cm, off):
    rng = np.random.default_rng(off)

    def at(a):
        big = cm.CUDAMatrix(np.concatenate([np.zeros(off, np.float32), np.asarray(a, np.float32).ravel(order="F")]).reshape(-1, 1))
        v = big.slice(off, off + a.size)
        v.reshape(a.shape)
        return v
    V, H, N = 256, 128, 96
    wg, wu, x, dy = (rng.standard_normal(s).astype(np.float32) for s in ((V, H), (V, H), (V, N), (H, N)))
    got = []
    for place in (cm.CUDAMatrix, at):
        m = [place(v) for v in (wg, wu, x, dy)]
        gm, um, y, dx, dw = (place(np.zeros(s, np.float32)) for s in ((H, N), (H, N), (H, N), (V, N), (V, H)))
        cm.gated_product(m[0], m[1], m[2], y, activation="silu", gate=gm, up=um)
        first = [get(v) for v in (y, gm, um)]
        cm.gated_product_deriv(m[3], gm, um, m[0], m[1], m[2], activation="silu", grad_x=dx, grad_up_w=dw)
        got.append(first + [get(dx), get(dw)])
    for a, b in zip(*got):          # the same sums by another kernel at most
        size = np.abs(a).max()
        np.testing.assert_allclose(a, b, rtol=0, atol=size * 2 * (256 * U + 2.0 ** -18) * 30)


def test_a_wait_that_cannot_end_is_reported(cm):
    """A product that is told to expect more bytes than its copies bring: the wait runs into its limit, the kernel returns, the status
    word says so, and the next product works."""
    rng = np.random.default_rng(4)
    w, x = cm.CUDAMatrix(rng.standard_normal((512, 512)).astype(np.float32)), cm.CUDAMatrix(rng.standard_normal((512, 512)).astype(np.float32))
    want = get(on_path(cm, 1, lambda: cm.gated_product(w, w, x)))
    assert cm.read_status() == 0
    cm.set_wait_limit(20000)                   # milliseconds
    try:
        cm._lib.b200_test_inject_stage_bytes(64)
        on_path(cm, 1, lambda: cm.gated_product(w, w, x))
        assert 31 <= cm.read_status() <= 34    # (waits until the kernel has returned)
        assert cm.read_status() == 0
    finally:
        cm.set_wait_limit(0)
    assert np.array_equal(get(on_path(cm, 1, lambda: cm.gated_product(w, w, x))), want)
    assert cm.read_status() == 0


class _On(object):
    """The library's calls on a stream of torch's; with a graph, recorded."""

    def __init__(self, cm, graph=None):
        self.cm, self.stream, self.graph = cm, torch.cuda.Stream(), graph

    def __enter__(self):
        torch.cuda.synchronize()
        self.cm._check(self.cm._lib.b200_set_stream(self.stream.cuda_stream))
        if self.graph is not None:
            self.ctx = torch.cuda.graph(self.graph, stream=self.stream)
            self.ctx.__enter__()
        return self

    def __exit__(self, *e):
        try:
            if self.graph is not None:
                self.ctx.__exit__(*e)
        finally:
            self.cm._lib.b200_set_stream(None)
        torch.cuda.synchronize()


def test_two_recorded_forward_passes_share_no_scratch(cm):
    rng = np.random.default_rng(8)
    torch.zeros(1, device="cuda")
    sets, streams, graphs = [], [], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for V, H, N in ((700, 900, 300), (1300, 500, 200)):
        s = [cm.CUDAMatrix(rng.standard_normal(shape).astype(np.float32)) for shape in ((V, H), (V, H), (V, N))] + [cm.empty((H, N))]
        sets.append(s)
    for s, graph in zip(sets, graphs):
        with _On(cm, graph) as on:
            cm.gated_product(*s, activation="gelu")
        streams.append(on.stream)
    want = []
    for s in sets:
        cm.gated_product(*s, activation="gelu")
        want.append(get(s[3]))
        s[3].assign(0)
    cm.cuda_sync_threads()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert np.array_equal(get(s[3]), w)
    assert cm.read_status() == 0


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("shape", SHAPES + [(64, 128, 256), (65, 129, 257), (40, 600, 33), (700, 300, 70), (130, 1000, 600), (257, 9, 1300), (520, 513, 127)])
def test_derivative_on_tensor_cores_and_cuda_cores(cm, shape, path):
    """Gradients of units, cases and weights whose magnitudes lie far apart: none costs another its bits."""
    V, H, N = shape
    rng = np.random.default_rng(V * 5 + H * 3 + N)
    wg, wu = (np.ldexp(rng.standard_normal((V, H)), rng.integers(-20, 5, (1, H))).astype(np.float32) for _ in range(2))
    x = np.ldexp(rng.standard_normal((V, N)), rng.integers(-20, 5, (1, N))).astype(np.float32)
    gate, up = (rng.standard_normal((H, N)).astype(np.float32) for _ in range(2))
    dy = np.ldexp(rng.standard_normal((H, N)), rng.integers(-25, 5, (H, 1)) + rng.integers(-25, 5, (1, N))).astype(np.float32)
    dy[:, N // 2] = 0                          # a case without weight
    G = cm.CUDAMatrix
    ga, gb, gx = G(wg), G(wu), G(x)
    dx, dwg, dwu, dbg, dbu = cm.empty((V, N)), cm.empty((V, H)), cm.empty((V, H)), cm.empty((H, 1)), cm.empty((1, H))
    gm, um = G(gate), G(up)
    out = dict(grad_x=dx, grad_gate_w=dwg, grad_up_w=dwu, grad_gate_bias=dbg, grad_up_bias=dbu)
    on_path(cm, path, lambda: cm.gated_product_deriv(G(dy), gm, um, ga, gb, gx, activation="relu", **out))
    dg, du = dy * up * (gate > 0), dy * np.maximum(gate, 0)      # one rounding a product
    assert np.array_equal(get(gm), dg) and np.array_equal(get(um), du)
    A, B, X, D, E = (v.astype(np.float64) for v in (wg, wu, x, dg, du))
    of_case = np.maximum((np.abs(A).max(0)[:, None] * np.abs(D)).max(0), (np.abs(B).max(0)[:, None] * np.abs(E)).max(0))
    size = np.abs(A) @ np.abs(D) + np.abs(B) @ np.abs(E)
    within(get(dx), A @ D + B @ E, ((2 * H + 4) * U + 2.0 ** -18) * size + 2.0 ** -30 * 2 * H * of_case[None] + 1e-37)
    assert (get(dx)[:, N // 2] == 0).all()
    for got, d in ((dwg, D), (dwu, E)):
        of_unit = (np.abs(d) * np.abs(X).max(0)[None]).max(1)
        within(get(got), X @ d.T, ((N + 4) * U + 2.0 ** -18) * (np.abs(X) @ np.abs(d).T) + 2.0 ** -30 * N * of_unit[None] + 1e-37)
    within(get(dbg)[:, 0], D.sum(1), (N + 8) * U * np.abs(D).sum(1) + 1e-37)
    within(get(dbu)[0], E.sum(1), (N + 8) * U * np.abs(E).sum(1) + 1e-37)
    want = {k: get(v) for k, v in out.items()}
    # each gradient alone, and with the weights' planes: the same bits
    planes = cm.GatedPlanes(ga, gb)
    for names in (["grad_x"], ["grad_gate_w"], ["grad_up_w", "grad_x"], ["grad_up_bias"], []):
        for name in names:
            out[name].assign(3.0)
        on_path(cm, path, lambda: cm.gated_product_deriv(G(dy), G(gate), G(up), ga, gb, gx, activation="relu", planes=planes,
                                                         **{k: out[k] for k in names}))
        for name in names:
            assert np.array_equal(get(out[name]), want[name]), name
    assert cm.read_status() == 0


def test_two_recorded_derivatives_share_no_scratch(cm):
    rng = np.random.default_rng(18)
    torch.zeros(1, device="cuda")
    sets, streams, graphs = [], [], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for V, H, N in ((700, 900, 300), (1300, 500, 200)):
        r = lambda *s: cm.CUDAMatrix(rng.standard_normal(s).astype(np.float32))
        s = dict(w=(r(V, H), r(V, H)), x=r(V, N), dy=r(H, N), gate=r(H, N), up=r(H, N), g=cm.empty((H, N)), u=cm.empty((H, N)),
                 out=dict(grad_x=cm.empty((V, N)), grad_gate_w=cm.empty((V, H)), grad_up_w=cm.empty((V, H)), grad_up_bias=cm.empty((H, 1))))
        sets.append(s)

    def step(s):
        s["g"].assign(s["gate"])
        s["u"].assign(s["up"])
        cm.gated_product_deriv(s["dy"], s["g"], s["u"], *s["w"], s["x"], activation="gelu", **s["out"])
    for s, graph in zip(sets, graphs):
        with _On(cm, graph) as on:
            on_path(cm, 1, lambda: step(s))
        streams.append(on.stream)
    want = []
    for s in sets:
        on_path(cm, 1, lambda: step(s))
        want.append({k: get(v) for k, v in s["out"].items()})
        for v in s["out"].values():
            v.assign(0)
    cm.cuda_sync_threads()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        for k, v in s["out"].items():
            assert np.array_equal(get(v), w[k]), k
    assert cm.read_status() == 0


def test_results_of_more_than_2_to_31_elements(cm):
    rng = np.random.default_rng(6)
    V, H, N = 64, 65536, 32800
    wg, wu = (cm.CUDAMatrix((rng.standard_normal((V, H)) / 8).astype(np.float32)) for _ in range(2))
    last = rng.standard_normal((V, 300)).astype(np.float32)
    x, y = cm.empty((V, N)), cm.empty((H, N))
    x.slice(N - 300, N).assign(cm.CUDAMatrix(last))
    cm.gated_product(wg, wu, x, y, activation="relu")
    want = cm.gated_product(wg, wu, cm.CUDAMatrix(last), activation="relu")
    assert np.array_equal(get(y.slice(N - 300, N)), get(want))            # a case's sums do not depend on the others
    assert (get(y.slice(0, 2)) == 0).all()
    y.free_device_memory()
    assert cm.read_status() == 0


def by_terms(a, b):
    """How far a . b may be off by its own terms alone, whatever else a row or column holds: operands are exact sums of three parts
    of eight bits, products of parts below 2^-26 of |a_k||b_k| are left out, a sum of 64 terms lies in the tensor core for four
    instructions at its full size and twenty at 2^-8 of it, each of which drops up to 2^-22 of it (4.2 x 2^-22), and the sums of 64
    are added in float32; full float32 multiply-adds round K times.  2^-19 + (K + 2) u covers either."""
    return ((a.shape[1] + 2) * U + 2.0 ** -19) * (np.abs(a) @ np.abs(b))


def gradients(cm, path, dy, gate, up, wg, wu, x):
    """dg, du, dx, dwg, dwu of the layer with relu."""
    G = cm.CUDAMatrix
    gm, um = G(gate), G(up)
    out = [cm.empty(s) for s in (x.shape, wg.shape, wu.shape)]
    on_path(cm, path, lambda: cm.gated_product_deriv(G(dy), gm, um, G(wg), G(wu), G(x), activation="relu", grad_x=out[0],
                                                     grad_gate_w=out[1], grad_up_w=out[2]))
    return [get(m) for m in [gm, um] + out]


def check_both_ways(cm, path, wg, wu, x, gate, up, dy, least=1e-36):
    V, H = wg.shape
    N = x.shape[1]
    gm, um = cm.empty((H, N)), cm.empty((H, N))
    G = cm.CUDAMatrix
    on_path(cm, path, lambda: cm.gated_product(G(wg), G(wu), G(x), activation="linear", gate=gm, up=um))
    A, B, X = (v.astype(np.float64) for v in (wg, wu, x))
    within(get(gm), A.T @ X, by_terms(A.T, X) + least)
    within(get(um), B.T @ X, by_terms(B.T, X) + least)
    dg, du, dx, dwg, dwu = gradients(cm, path, dy, gate, up, wg, wu, x)
    assert np.array_equal(dg, dy * up * (gate > 0)) and np.array_equal(du, dy * np.maximum(gate, 0))
    D, E = dg.astype(np.float64), du.astype(np.float64)
    AB, DE = np.concatenate([A, B], 1), np.concatenate([D, E], 0)
    within(dx, AB @ DE, by_terms(AB, DE) + least)
    within(dwg, X @ D.T, by_terms(X, D.T) + least)
    within(dwu, X @ E.T, by_terms(X, E.T) + least)
    assert cm.read_status() == 0


SPREAD_SHAPES = [(784, 64, 64), (300, 200, 40), (257, 129, 130), (2048, 256, 33)]


@pytest.mark.parametrize("path", [0, 1, 2])
@pytest.mark.parametrize("spread", [0, 13, 20, 27, 40, 50])
@pytest.mark.parametrize("shape", SPREAD_SHAPES)
def test_small_entries_beside_large_ones_of_their_column(cm, shape, spread, path):
    """A feature 2^spread above the others whose weights are as far below theirs, features all over that range, and the same of the
    units' gradients: every sum is held to its own terms."""
    V, H, N = shape
    rng = np.random.default_rng(V + H + N + spread)
    normal = lambda *s: rng.standard_normal(s)
    e = rng.integers(-spread // 2, spread // 2 + 1, (V, 1))
    e[:4] = spread
    e[4:V // 2] = 0
    wg, wu = (np.ldexp(normal(V, H), -e).astype(np.float32) for _ in range(2))
    x = np.ldexp(normal(V, N), e).astype(np.float32)
    f = rng.integers(-spread // 2, spread // 2 + 1, (H, 1))
    f[:3], f[3:H // 2] = spread, 0
    c = rng.integers(-8, 9, (1, N))               # (2^50 2^50 2^8 and what the sums add: every result is a normal number)
    dy = np.ldexp(normal(H, N), f + c).astype(np.float32)
    check_both_ways(cm, path, wg, wu, x, normal(H, N).astype(np.float32), normal(H, N).astype(np.float32), dy)


@pytest.mark.parametrize("path", [0, 1, 2])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 1e-8, 1e-12])
def test_a_unit_and_a_case_of_zeros_cost_the_others_nothing(cm, size, path):
    rng = np.random.default_rng(5)
    V, H, N = 300, 200, 64
    normal = lambda *s: rng.standard_normal(s).astype(np.float32)
    wg, wu, x = (size * normal(*s) for s in ((V, H), (V, H), (V, N)))
    wg[:, 7] = 0
    wu[:, [7, 11]] = 0
    x[:, 9] = 0
    check_both_ways(cm, path, wg, wu, x, np.abs(normal(H, N)), normal(H, N), normal(H, N))


@pytest.mark.parametrize("path", [0, 1, 2])
@pytest.mark.parametrize("ends", [(120, -100, -20), (-100, 20, 90), (124, -90, -40), (-90, 100, -80), (60, 60, -60), (100, -100, -100)])
def test_magnitudes_at_both_ends_of_the_range(cm, ends, path):
    """Weights, inputs and gradients about 2^ends: no power of two is out of reach where the result is a normal number."""
    rng = np.random.default_rng(6)
    V, H, N = 200, 140, 40
    normal = lambda *s: rng.standard_normal(s)
    wg, wu, x, dy = (np.ldexp(normal(*s), e).astype(np.float32) for s, e in zip(((V, H), (V, H), (V, N), (H, N)), (ends[0],) + ends))
    check_both_ways(cm, path, wg, wu, x, np.abs(normal(H, N)).astype(np.float32), normal(H, N).astype(np.float32), dy, least=2.0 ** -118)


def test_the_largest_number_there_is(cm):
    """It is above the largest of eight bits: its parts still add up to it."""
    V, H, N = 300, 128, 64
    top = np.finfo(np.float32).max
    x = np.zeros((V, N), np.float32)
    x[np.arange(N), np.arange(N)] = top
    x[np.arange(N), (np.arange(N) + 1) % N] = -top
    w = np.ldexp(np.random.default_rng(7).standard_normal((V, H)), -20).astype(np.float32)
    gm, um = cm.empty((H, N)), cm.empty((H, N))
    on_path(cm, 1, lambda: cm.gated_product(cm.CUDAMatrix(w), cm.CUDAMatrix(-w), cm.CUDAMatrix(x), activation="linear", gate=gm, up=um))
    A, X = w.astype(np.float64), x.astype(np.float64)
    within(get(gm), A.T @ X, by_terms(A.T, X))
    assert np.array_equal(get(um), -get(gm))


@pytest.mark.parametrize("shape", [(2048, 2048, 40), (2048, 2304, 9), (40, 30, 20), (300, 200, 100)])
def test_derivatives_recorded_before_they_ever_ran(cm, shape):
    """Two graphs of one stream, of layers large and small over few cases and many, recorded without a call before them and replayed on
    streams that nobody orders: each gives what the calls give."""
    V, H, N = shape
    rng = np.random.default_rng(V + N)
    torch.zeros(1, device="cuda")
    sets, graphs, streams = [], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in graphs:
        r = lambda *s: cm.CUDAMatrix(rng.standard_normal(s).astype(np.float32))
        sets.append(dict(w=(r(V, H), r(V, H)), x=r(V, N), dy=r(H, N), y=cm.empty((H, N)), gate=cm.empty((H, N)), up=cm.empty((H, N)),
                         out=dict(grad_x=cm.empty((V, N)), grad_gate_w=cm.empty((V, H)), grad_up_w=cm.empty((V, H)), grad_up_bias=cm.empty((H, 1)))))

    def step(s):
        cm.gated_product(*s["w"], s["x"], s["y"], activation="silu", gate=s["gate"], up=s["up"])
        cm.gated_product_deriv(s["dy"], s["gate"], s["up"], *s["w"], s["x"], activation="silu", **s["out"])
    capture = torch.cuda.Stream()
    torch.cuda.synchronize()
    cm._check(cm._lib.b200_set_stream(capture.cuda_stream))
    try:
        for s, graph in zip(sets, graphs):
            with torch.cuda.graph(graph, stream=capture):
                step(s)
    finally:
        cm._lib.b200_set_stream(None)
    want = []
    for s in sets:
        step(s)
        want.append([get(v) for v in [s["y"]] + list(s["out"].values())])
        for v in [s["y"]] + list(s["out"].values()):
            v.assign(0)
    cm.cuda_sync_threads()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        for v, x in zip([s["y"]] + list(s["out"].values()), w):
            assert np.array_equal(get(v), x)
    assert cm.read_status() == 0
