"""Layer normalisation, dropout by key and log probabilities of tokens on the device against their definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is the most one rounding to float32 is off, relative to the value; a sum of n terms that
every partial sum of which is rounded is off by at most n u times the sum of the terms' magnitudes (to first order), and a term
passes at most as many roundings as additions lie between it and the result."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def get(m):
    return np.array(m.asarray(), copy=True)


def odd_start(cm, a, off):
    """`a` on the device, its first element `off` floats behind an allocation's start."""
    big = cm.CUDAMatrix(np.concatenate([np.zeros(off, np.float32), np.asarray(a, np.float32).ravel(order="F")]).reshape(-1, 1))
    view = big.slice(off, off + a.size)
    view.reshape(a.shape)
    return view


def within(got, want, bound):
    got, want = got.astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    off = np.abs(got - want) - np.broadcast_to(bound, want.shape)
    assert (off <= 0).all(), (float(off.max()), float(np.abs(got - want).max()))


# -- layer normalisation ------------------------------------------------------------------------
def norm_exact(x, gain, bias, eps):
    x = x.astype(np.float64)
    h = x.shape[0]
    m = x.mean(0)
    rs = 1.0 / np.sqrt(((x - m) ** 2).mean(0) + eps)
    xh = (x - m) * rs
    g = np.ones((h, 1)) if gain is None else gain.astype(np.float64)
    b = np.zeros((h, 1)) if bias is None else bias.astype(np.float64)
    # a thread adds at most 32 values (long columns: one of 1024), then ten more additions join the threads'; with the division
    # and the rounding of eps
    n = max(32, -(-h // 1024)) + 12
    dm = n * U * np.abs(x).mean(0)
    dr = (n + 3) * U / 2 + 3 * U              # relative: the variance's sum, half of it behind the square root, its and 1 / .'s roundings
    # the mean's error adds its square to the variance
    dr = dr + 0.5 * (dm * rs) ** 2
    dxh = (dm + U * np.abs(x - m)) * rs + np.abs(xh) * (dr + 2 * U)
    return xh * g + b, xh, m, rs, dm, dr, dxh, g, b, n


SHAPES = [(1, 1), (1, 7), (3, 5), (31, 9), (32, 1), (33, 2), (64, 17), (100, 100), (128, 3), (257, 31), (500, 8), (512, 40), (513, 12),
          (784, 100), (510, 700), (1023, 900), (2047, 1300), (8190, 700), (1024, 33), (1028, 5), (1357, 203), (2048, 64), (4096, 50), (4100, 3), (4099, 20), (8192, 9), (8195, 4),
          (16384, 3), (20000, 5), (32772, 2), (40001, 3), (500, 3001), (16, 4096)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("params", ["both", "none", "gain"])
def test_layer_norm_and_its_derivative(cm, shape, params):
    h, w = shape
    rng = np.random.default_rng(h * 31 + w)
    x = (rng.standard_normal(shape) * (0.1 + rng.random((1, w)) * 5) + rng.standard_normal((h, 1))).astype(np.float32)
    dy = (rng.standard_normal(shape) * rng.random((1, w))).astype(np.float32)
    gain = (1 + 0.3 * rng.standard_normal((h, 1))).astype(np.float32) if params != "none" else None
    bias = rng.standard_normal((h, 1)).astype(np.float32) if params == "both" else None
    eps = 1e-5
    y, xh, m, rs, dm, dr, dxh, g, b, n = norm_exact(x, gain, bias, eps)
    gx, gd = cm.CUDAMatrix(x), cm.CUDAMatrix(dy)
    gg, gb = (cm.CUDAMatrix(v) if v is not None else None for v in (gain, bias))
    out, stats = cm.empty(shape), cm.empty((2, w))
    gx.layer_norm(gg, gb, eps=eps, target=out, stats=stats)
    assert np.array_equal(get(gx), x)
    within(get(out), y, np.abs(g) * dxh + 2 * U * (np.abs(xh * g) + np.abs(y)) + 1e-37)
    within(get(stats)[0:1], m[None], (dm + U * np.abs(m))[None] + 1e-37)
    within(get(stats)[1:2], rs[None], (rs * dr)[None])
    # without statistics, in place: the same bits
    again = cm.CUDAMatrix(x)
    again.layer_norm(gg, gb, eps=eps)
    assert np.array_equal(get(again), get(out))
    # back
    d = dy.astype(np.float64)
    a = d * g
    ma, mx = a.mean(0), (a * xh).mean(0)
    dx, dgain, dbias = rs * (a - ma - xh * mx), (d * xh).sum(1, keepdims=True), d.sum(1, keepdims=True)
    dxh = dxh + U * np.abs(xh)
    e_ma = (n + 2) * U * np.abs(a).mean(0)
    e_mx = (n + 4) * U * np.abs(a * xh).mean(0) + (np.abs(a) * dxh).mean(0)
    e_dx = rs * (U * np.abs(a) + e_ma + np.abs(xh) * e_mx + dxh * np.abs(mx) + 3 * U * (np.abs(a) + np.abs(ma) + np.abs(xh * mx)))
    e_dx = e_dx + (dr + U) * np.abs(dx)
    terms = w + 16                            # columns one after another, eight warps, then the blocks' shares
    e_g = terms * U * np.abs(d * xh).sum(1, keepdims=True) + (np.abs(d) * dxh).sum(1, keepdims=True)
    e_b = terms * U * np.abs(d).sum(1, keepdims=True)
    gdx, ggain, gbias = cm.empty(shape), cm.CUDAMatrix(np.full((h, 1), 7.0)), cm.CUDAMatrix(np.full((h, 1), 7.0))
    gd.layer_norm_deriv(gx, stats, gg, target=gdx, grad_gain=ggain, grad_bias=gbias)
    within(get(gdx), dx, 1.01 * e_dx + 1e-37)
    within(get(ggain), dgain, 1.01 * e_g + 1e-37)
    within(get(gbias), dbias, 1.01 * e_b + 1e-37)
    assert np.array_equal(get(gx), x) and np.array_equal(get(gd), dy)
    # over the gradient itself, one parameter's gradient or none: the same bits
    only = cm.CUDAMatrix(np.full((h, 1), 7.0))
    over = cm.CUDAMatrix(dy)
    over.layer_norm_deriv(gx, stats, gg, grad_gain=only)
    assert np.array_equal(get(over), get(gdx)) and np.array_equal(get(only), get(ggain))
    over = cm.CUDAMatrix(dy)
    over.layer_norm_deriv(gx, stats, gg)
    assert np.array_equal(get(over), get(gdx))
    over_x = cm.CUDAMatrix(x)
    gd.layer_norm_deriv(over_x, stats, gg, target=over_x, grad_gain=only, grad_bias=gbias)
    assert np.array_equal(get(over_x), get(gdx)) and np.array_equal(get(only), get(ggain))


@pytest.mark.parametrize("off", [1, 2, 3])
def test_layer_norm_of_matrices_that_start_anywhere(cm, off):
    rng = np.random.default_rng(off)
    x, dy = (rng.standard_normal((256, 21)).astype(np.float32) for _ in range(2))
    gain = rng.standard_normal((256, 1)).astype(np.float32)
    want, wdx, wst, wg = cm.empty((256, 21)), cm.empty((256, 21)), cm.empty((2, 21)), cm.empty((256, 1))
    cm.CUDAMatrix(x).layer_norm(cm.CUDAMatrix(gain), target=want, stats=wst)
    cm.CUDAMatrix(dy).layer_norm_deriv(cm.CUDAMatrix(x), wst, cm.CUDAMatrix(gain), target=wdx, grad_gain=wg)
    z = np.zeros_like(x)
    gx, out, dx = odd_start(cm, x, off), odd_start(cm, z, off), odd_start(cm, z, off)
    st, gg = cm.empty((2, 21)), cm.empty((256, 1))
    gx.layer_norm(odd_start(cm, gain, off), target=out, stats=st)
    odd_start(cm, dy, off).layer_norm_deriv(gx, st, odd_start(cm, gain, off), target=dx, grad_gain=gg)
    # (other groupings of the same sums: each within 45 roundings of the 64-bit value, values of size 1)
    for a, b in ((out, want), (dx, wdx)):
        np.testing.assert_allclose(get(a), get(b), rtol=0, atol=2 * 45 * U * 20)
    np.testing.assert_allclose(get(gg), get(wg), rtol=0, atol=2 * (45 + 37) * U * 21 * 20)


@pytest.mark.parametrize("shape", [(37, 50), (1001, 23), (1024, 30), (9001, 3)])
def test_layer_norm_of_matrices_that_lie_differently(cm, shape):
    """Inputs, gradients and results at different distances from 16 bytes."""
    h, w = shape
    rng = np.random.default_rng(h)
    x, dy = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    z = np.zeros_like(x)
    want, wdx, wst, wg = cm.empty(shape), cm.empty(shape), cm.empty((2, w)), cm.empty((h, 1))
    cm.CUDAMatrix(x).layer_norm(target=want, stats=wst)
    cm.CUDAMatrix(dy).layer_norm_deriv(cm.CUDAMatrix(x), wst, target=wdx, grad_gain=wg)
    for a, b, c in ((1, 0, 0), (0, 2, 0), (0, 0, 3), (1, 2, 3)):
        gx, out, dx = odd_start(cm, x, a), odd_start(cm, z, b), odd_start(cm, z, c)
        st, gg = cm.empty((2, w)), cm.empty((h, 1))
        gx.layer_norm(target=out, stats=st)
        odd_start(cm, dy, b).layer_norm_deriv(gx, st, target=dx, grad_gain=gg)
        n = max(32, -(-h // 1024)) + 12          # as in norm_exact, twice: two groupings of sums of values up to 6
        np.testing.assert_allclose(get(out), get(want), rtol=0, atol=2 * n * U * 20)
        np.testing.assert_allclose(get(dx), get(wdx), rtol=0, atol=2 * n * U * 20)
        np.testing.assert_allclose(get(gg), get(wg), rtol=0, atol=2 * (n + w + 16) * U * w * 20)


def test_layer_norm_of_constant_and_extreme_columns(cm):
    x = np.zeros((300, 5), np.float32)
    x[:, 1] = 4.0                              # exact in any order
    x[:, 2] = np.arange(300) % 2 * 2 - 1       # mean 0, variance 1
    x[7, 3], x[9, 4] = np.nan, np.inf
    out, st = cm.empty(x.shape), cm.empty((2, 5))
    cm.CUDAMatrix(x).layer_norm(eps=0.25, target=out, stats=st)
    y, s = get(out), get(st)
    assert (y[:, 0] == 0).all() and (y[:, 1] == 0).all() and s[1, 0] == 2 and s[1, 1] == 2 and s[0, 1] == 4
    np.testing.assert_allclose(y[:, 2], x[:, 2] / np.sqrt(1.25), rtol=4 * U)
    assert np.isnan(y[:, 3]).all() and np.isnan(y[:, 4]).any()


def test_layer_norm_gradients_of_no_columns_are_zero(cm):
    x, st = cm.empty((6, 0)), cm.empty((2, 0))
    g, b = cm.CUDAMatrix(np.ones((6, 1))), cm.CUDAMatrix(np.ones((6, 1)))
    x.layer_norm_deriv(x, st, target=x, grad_gain=g, grad_bias=b)
    assert (get(g) == 0).all() and (get(b) == 0).all()


def test_layer_norm_gradient_against_differences(cm):
    rng = np.random.default_rng(5)
    x, dy, gain = (rng.standard_normal(s).astype(np.float32) for s in ((40, 6), (40, 6), (40, 1)))
    st, dx, dg = cm.empty((2, 6)), cm.empty((40, 6)), cm.empty((40, 1))
    gx = cm.CUDAMatrix(x)
    gx.layer_norm(cm.CUDAMatrix(gain), target=cm.empty((40, 6)), stats=st)
    cm.CUDAMatrix(dy).layer_norm_deriv(gx, st, cm.CUDAMatrix(gain), target=dx, grad_gain=dg)
    f = lambda x, g: (norm_exact(x, g, None, 1e-5)[0] * dy).sum()
    x64, g64, d = x.astype(np.float64), gain.astype(np.float64), 1e-6
    for r, c in ((0, 0), (39, 5), (17, 3)):
        e = np.zeros_like(x64)
        e[r, c] = d
        assert abs((f(x64 + e, g64) - f(x64 - e, g64)) / (2 * d) - get(dx)[r, c]) < 1e-5
        e = np.zeros_like(g64)
        e[r, 0] = d
        assert abs((f(x64, g64 + e) - f(x64, g64 - e)) / (2 * d) - get(dg)[r, 0]) < 1e-5


# -- dropout by key -----------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (100, 3), (4, 1), (64, 33), (1000, 37), (257, 130), (2048, 19)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_dropout_by_key_keeps_what_the_uniforms_say(cm, shape, p):
    rng = np.random.default_rng(3)
    x, res = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    x[0, 0] = np.inf                           # dropped or kept, never 0 * inf
    cm.CUDAMatrix.init_random(91)
    before = cm.CUDAMatrix.rnd_state.calls
    u = cm.empty(shape)
    u.fill_with_rand()
    keep = get(u) > np.float32(p)
    cm.CUDAMatrix.rnd_state.calls = before     # the same call's numbers
    gx, out = cm.CUDAMatrix(x), cm.empty(shape)
    key = gx.dropout_scaled(p, target=out)
    assert key == (91, before) and cm.CUDAMatrix.rnd_state.calls == before + 1
    scale = np.float32(1 / (1 - float(np.float32(p)))) if p < 1 else np.float32(0)
    with np.errstate(invalid="ignore"):
        want = np.where(keep, x * scale, np.float32(0))
    assert np.array_equal(get(out), want) and np.array_equal(get(gx), x)
    # the key again: the same mask on another matrix, the random state left alone; the residual joins with one or two roundings
    g2 = cm.CUDAMatrix(res)
    assert g2.dropout_scaled(p, key=key) == key and cm.CUDAMatrix.rnd_state.calls == before + 1
    assert np.array_equal(get(g2), np.where(keep, res * scale, np.float32(0)))
    joined = cm.CUDAMatrix(res)
    gx.dropout_scaled(p, target=joined, add=joined, key=key)
    kept = np.where(keep, x.astype(np.float64) * scale, 0.0)
    fine = np.isfinite(kept)
    assert (np.abs(get(joined)[fine] - (res + kept)[fine]) <= U * (np.abs(kept) + np.abs(res + kept))[fine] * 1.01).all()
    assert not keep[0, 0] or np.isinf(get(joined)[0, 0])


@pytest.mark.parametrize("off", [1, 2, 3])
def test_dropout_of_matrices_that_start_anywhere_and_of_a_shard(cm, off):
    x = np.random.default_rng(4).standard_normal((64, 40)).astype(np.float32)
    whole = cm.empty(x.shape)
    cm.CUDAMatrix(x).dropout_scaled(0.3, target=whole, key=(5, 6))
    out = odd_start(cm, np.zeros_like(x), off)
    odd_start(cm, x, off).dropout_scaled(0.3, target=out, key=(5, 6))
    assert np.array_equal(get(out), get(whole))
    cm.set_rng_column_offset(10 + off)
    try:                                       # a process's share of the columns draws those columns' numbers
        part = cm.CUDAMatrix(x[:, 10 + off:31])
        part.dropout_scaled(0.3, key=(5, 6))
        assert np.array_equal(get(part), get(whole)[:, 10 + off:31])
    finally:
        cm.set_rng_column_offset(0)


# -- log probabilities --------------------------------------------------------------------------
def words_exact(z):
    z = z.astype(np.float64)
    m = z.max(0)
    d = z - m
    e = np.exp(d)
    s = e.sum(0)
    lp = d - np.log(s)
    p = e / s
    with np.errstate(invalid="ignore"):
        ent = -np.where(p > 0, p * lp, 0.0).sum(0)
    return lp, p, ent, d, s


def words_bounds(z, lp, p, ent, d, s):
    """How far log-sum, entropy may be off.  A thread of one warp a column adds h / 32 terms and joins ten times; whenever its maximum
    grows (at most once a batch of eight) and in every join the sums are scaled by an exponential (4 u with its argument's
    rounding, which weighs no more than u, the product's u, and t's three)."""
    h = z.shape[0]
    n = h / 32 + 8 + 10 + 6 * (h / 256 + 11) + 6
    finite = np.where(p > 0, d, 0.0)
    weighed = (p * np.abs(finite)).sum(0)
    rel_s = (n + weighed) * U                  # exp(d) with d rounded: |d| u relative
    dls = rel_s + 2 * U * np.abs(np.log(s))
    dent = dls + (n + 4) * U * 2 * weighed + (p * finite ** 2).sum(0) * U + 2 * U * np.abs(ent)
    return dls, dent


WORDS = [(1, 1), (2, 3), (7, 5), (32, 4), (33, 1), (100, 64), (255, 30), (256, 1), (1000, 2), (1001, 5), (10000, 1), (10000, 37), (4099, 301),
         (50021, 6), (100000, 1), (64, 6000), (600001, 2)]


def ranked(z, k):
    """Lower numbers first among equals."""
    return np.argsort(-z.astype(np.float64), axis=0, kind="stable")[:k]


@pytest.mark.parametrize("shape", WORDS)
@pytest.mark.parametrize("kind", ["normal", "steps", "peaked", "masked", "rising"])
def test_log_probabilities_entropy_likeliest_and_gradient(cm, shape, kind):
    h, w = shape
    rng = np.random.default_rng(h + 7 * w)
    z = (3 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "steps":
        z = np.round(z * 2) / 2                # many equal logits
    if kind == "peaked":
        z = z + 60                             # far from 0, one word with nearly everything
        z[rng.integers(0, h, w), np.arange(w)] += 50
    if kind == "masked":
        z[rng.random(shape) < 0.6] = -np.inf
        z[rng.integers(0, h, w), np.arange(w)] = 1.5       # (no column is without a word)
        z[rng.random(shape) < 0.2] = np.finfo(np.float32).min
        z[0, :] = np.where(np.isneginf(z).all(0), 1.5, z[0, :])
    if kind == "rising":
        z = np.sort(z, axis=0)                 # every word likelier than those before it
    z = z.astype(np.float32)
    t = rng.integers(0, h, w)
    given = t - h * (rng.random(w) < 0.3)      # counted from the end
    k = min(h, [1, 5, 20, 32][(h + w) % 4])
    gz, gt = cm.CUDAMatrix(z), cm.CUDAMatrix(given[None].astype(np.float32))
    out, ent, st, top, tops = cm.empty((1, w)), cm.empty((1, w)), cm.empty((2, w)), cm.empty((k, w)), cm.empty((k, w))
    assert gz.log_prob(gt, target=out, entropy=ent, stats=st, top=top, top_tokens=tops) is out
    lp, p, H, d, s = words_exact(z)
    dls, dent = words_bounds(z, lp, p, H, d, s)

    def close(got, want, bound):
        gone = np.isneginf(want)
        assert np.array_equal(np.isneginf(got), gone)
        within(np.where(gone, 0, got), np.where(gone, 0, want), bound)
    lt = lp[t, np.arange(w)]
    dt = np.where(np.isneginf(lt), 0, np.abs(d[t, np.arange(w)]))
    # (d of the type's lowest value is infinite in float32 where the maximum is above 0 by more than half a step: it is not here)
    close(get(out)[0], lt, dls + 2 * U * (dt + np.abs(np.where(np.isneginf(lt), 0, lt))))
    within(get(ent)[0], H, dent)
    order = ranked(z, k)
    assert np.array_equal(get(tops), order.astype(np.float32))
    lo = np.take_along_axis(lp, order, 0)
    mag = np.where(np.isneginf(lo), 0, np.abs(lo) + np.abs(np.take_along_axis(d, order, 0)))
    close(get(top), lo, dls + 2 * U * mag)
    # without the likeliest words, and with them alone
    out2 = gz.log_prob(gt)
    assert np.array_equal(get(out2), get(out))
    top2, tops2 = cm.empty((k, w)), cm.empty((k, w))
    assert gz.log_prob(top=top2, top_tokens=tops2) is None
    assert np.array_equal(get(top2), get(top)) and np.array_equal(get(tops2), get(tops))
    # gradient
    g = (rng.standard_normal(w) * (rng.random(w) < 0.8)).astype(np.float32)
    q = (rng.standard_normal(w) * (rng.random(w) < 0.5)).astype(np.float32)
    flp = np.where(p > 0, lp, 0.0)
    want = -p * (g + q * (flp + H)) * (p > 0)
    want[t, np.arange(w)] += g
    rel = (6 + np.abs(flp) * 2 + np.abs(np.where(p > 0, d, 0.0))) * U + dls
    bound = p * (np.abs(g) + np.abs(q) * np.abs(flp + H)) * (rel + 5 * U) + p * np.abs(q) * (dls + dent + U * (np.abs(flp) * 2 + H)) + U * np.abs(want)
    bound[t, np.arange(w)] += U * np.abs(g)
    bound = bound + 1e-37                      # (products below the smallest normal)
    grad = cm.empty(shape)
    row = lambda v: cm.CUDAMatrix(v[None])
    gz.log_prob_deriv(gt, st, row(g), entropy=ent, grad_entropy=row(q), target=grad)
    within(get(grad), want, 1.01 * bound)
    assert (get(grad)[:, (g == 0) & (q == 0)] == 0).all() and np.array_equal(get(gz), z)
    over = cm.CUDAMatrix(z)                    # over the logits: the same bits
    over.log_prob_deriv(gt, st, row(g), entropy=ent, grad_entropy=row(q))
    assert np.array_equal(get(over), get(grad))
    # either gradient alone
    over = cm.CUDAMatrix(z)
    over.log_prob_deriv(gt, st, row(g))
    want = -p * g
    want[t, np.arange(w)] += g
    within(get(over), want, 1.01 * (p * np.abs(g) * (rel + 4 * U) + U * np.abs(want) + 1e-37 + U * np.abs(g)))
    over = cm.CUDAMatrix(z)
    over.log_prob_deriv(None, st, None, entropy=ent, grad_entropy=row(q))
    within(get(over), -p * q * (flp + H) * (p > 0), 1.01 * bound)


@pytest.mark.parametrize("k", [5, 20, 32])
@pytest.mark.parametrize("h", [300, 512, 5000, 30000])
@pytest.mark.parametrize("w", [260, 131, 67, 33])
def test_likeliest_words_of_columns_that_share_a_block(cm, h, w, k):
    """Columns that find their words in one look beside columns that need sorted lists (equal logits, fewer words than are asked for,
    words in order), in any order: none may touch what another still reads.  On eight SMs these numbers of columns are read by one
    warp each, by two, by four and by eight, where a column is long enough."""
    rng = np.random.default_rng(h + 7 * w + k)
    z = (3 * rng.standard_normal((h, w))).astype(np.float32)
    kind = rng.integers(0, 5, w)
    z[:, kind == 1] = 1.0                                           # all equal
    some = np.flatnonzero(kind == 2)
    z[:, some] = -np.inf
    for c in some:
        z[rng.integers(0, h, 3), c] = rng.standard_normal(3)        # at most three words left
    z[:, kind == 3] = np.sort(z[:, kind == 3], axis=0)
    z[:, kind == 4] = np.round(z[:, kind == 4])
    want = ranked(z, k).astype(np.float32)
    gz, top, tops = cm.CUDAMatrix(z), cm.empty((k, w)), cm.empty((k, w))
    cm.set_sm_limit(8)
    try:
        for _ in range(5):
            tops.assign(-1)
            gz.log_prob(top=top, top_tokens=tops)
            assert np.array_equal(get(tops), want)
    finally:
        cm.set_sm_limit(0)
    best = np.take_along_axis(z, want.astype(np.int64), 0)
    fell = np.isneginf(best)
    assert np.array_equal(np.isneginf(get(top)), fell)
    # log p differs from column to column by one number alone: differences of logits, each off by a few roundings of values up to 40
    got = np.where(fell, 0, get(top) - get(top)[:1])
    np.testing.assert_allclose(got, np.where(fell, 0, best - best[:1]), rtol=0, atol=4 * 40 * U)


def test_columns_without_a_distribution(cm):
    h = 300
    z = np.random.default_rng(2).standard_normal((h, 8)).astype(np.float32)
    z[:, 1] = -np.inf                          # nothing left
    z[:, 2] = np.finfo(np.float32).min         # equal, and as low as the type goes
    z[5, 3], z[6, 4] = np.nan, np.inf
    z[:, 5] = -np.inf
    z[11, 5] = -3.0                            # one word left
    z[:, 6], z[7, 6] = -np.inf, np.nan
    t = np.array([[0, 4, -1, 5, 6, 11, 7, h]], np.float32)     # the last out of range
    gz, gt = cm.CUDAMatrix(z), cm.CUDAMatrix(t)
    out, ent, st, top, tops = (cm.empty((n, 8)) for n in (1, 1, 2, 3, 3))
    gz.log_prob(gt, target=out, entropy=ent, stats=st, top=top, top_tokens=tops)
    o, e, tp, ti = get(out)[0], get(ent)[0], get(top), get(tops)
    assert np.isneginf(o[1]) and e[1] == 0 and np.isneginf(tp[:, 1]).all() and ti[:, 1].tolist() == [0, 1, 2]
    assert abs(o[2] + np.log(h)) < 1e-5 and abs(e[2] - np.log(h)) < 1e-5 and ti[:, 2].tolist() == [0, 1, 2]
    for c in (3, 4, 6):
        assert np.isnan(o[c]) and np.isnan(e[c]) and np.isnan(tp[:, c]).all() and ti[:, c].tolist() == [0, 1, 2]
    assert o[5] == 0 and e[5] == 0 and ti[:, 5].tolist() == [11, 0, 1] and tp[0, 5] == 0 and np.isneginf(tp[1:, 5]).all()
    assert np.isnan(o[7]) and np.isfinite(e[7]) and np.isfinite(tp[:, 7]).all()
    g = np.ones((1, 8), np.float32)
    grad = cm.empty(z.shape)
    gz.log_prob_deriv(gt, st, cm.CUDAMatrix(g), target=grad)
    d = get(grad)
    assert (d[:, 1] == 0).all() and (d[:, 5] == 0).all() and abs(d[h - 1, 2] - (1 - 1 / h)) < 1e-6
    assert all(np.isnan(d[:, c]).any() for c in (3, 4, 6)) and np.isnan(d[:, 7]).all()
    gz.log_prob_deriv(gt, st, cm.CUDAMatrix(0 * g), entropy=ent, grad_entropy=cm.CUDAMatrix(0 * g), target=grad)
    assert (get(grad) == 0).all()
    for bad in (np.nan, 1e10, -h - 1, np.inf):
        assert np.isnan(get(gz.log_prob(cm.CUDAMatrix(np.full((1, 8), bad))))).all()


@pytest.mark.parametrize("h", [5, 40, 700, 5000])
def test_both_zeros_are_one_logit(cm, h):
    """Of equal logits the lower number, and 0 and -0 are equal."""
    z = np.full((h, 3), -1.0, np.float32)
    z[[0, h // 2, h - 1], 0] = [-0.0, 0.0, -0.0]
    z[[1, h // 2, h - 1], 1] = [0.0, -0.0, 0.0]
    z[h - 2:, 2] = -0.0
    z[0, 2] = 0.0
    top, tops = cm.empty((3, 3)), cm.empty((3, 3))
    cm.CUDAMatrix(z).log_prob(top=top, top_tokens=tops)
    assert np.array_equal(get(tops), np.array([[0, h // 2, h - 1], [1, h // 2, h - 1], [0, h - 2, h - 1]], np.float32).T)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_logits_that_start_anywhere(cm, off):
    rng = np.random.default_rng(off)
    z = rng.standard_normal((1024, 9)).astype(np.float32)
    t, g = cm.CUDAMatrix(rng.integers(0, 1024, (1, 9)).astype(np.float32)), cm.CUDAMatrix(rng.standard_normal((1, 9)))
    a, b = cm.CUDAMatrix(z), odd_start(cm, z, off)
    got = []
    for m in (a, b):
        st, top, tops = cm.empty((2, 9)), cm.empty((6, 9)), cm.empty((6, 9))
        lp = m.log_prob(t, stats=st, top=top, top_tokens=tops)
        m.log_prob_deriv(t, st, g)
        got.append([get(x) for x in (lp, top, tops, m)])
    assert np.array_equal(got[0][2], got[1][2])
    for x, y in zip(*got):                     # the same sums in another grouping: 2 x 60 roundings of values up to 12
        np.testing.assert_allclose(x, y, rtol=0, atol=2 * 60 * U * 12)


@pytest.mark.parametrize("h", [7, 300, 2049])
def test_logits_and_gradient_that_lie_differently(cm, h):
    rng = np.random.default_rng(h)
    z = rng.standard_normal((h, 11)).astype(np.float32)
    gz, t, g = cm.CUDAMatrix(z), cm.CUDAMatrix(rng.integers(0, h, (1, 11)).astype(np.float32)), cm.CUDAMatrix(rng.standard_normal((1, 11)))
    st, want = cm.empty((2, 11)), cm.empty((h, 11))
    gz.log_prob(t, stats=st)
    gz.log_prob_deriv(t, st, g, target=want)
    for off in (1, 2, 3):                      # elementwise: the same bits
        got = odd_start(cm, np.zeros_like(z), off)
        gz.log_prob_deriv(t, st, g, target=got)
        assert np.array_equal(get(got), get(want))


# -- streams and graphs -------------------------------------------------------------------------
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


def test_two_recorded_passes_share_no_scratch(cm):
    """Two graphs recorded before the calls ever ran on their streams, of matrices of other sizes, replayed side by side: each gives
    what it gives alone (the sums of the parameters' gradients need scratch)."""
    rng = np.random.default_rng(8)
    torch.zeros(1, device="cuda")
    sets, graphs, streams = [], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for h, w in ((700, 900), (1300, 500)):
        x, dy = (cm.CUDAMatrix(rng.standard_normal((h, w)).astype(np.float32)) for _ in range(2))
        z, t = cm.CUDAMatrix(rng.standard_normal((h, w)).astype(np.float32)), cm.CUDAMatrix(rng.integers(0, h, (1, w)).astype(np.float32))
        s = dict(x=x, dy=dy, z=z, t=t, g=cm.CUDAMatrix(rng.standard_normal((1, w))), y=cm.empty((h, w)), st=cm.empty((2, w)), dx=cm.empty((h, w)),
                 dg=cm.empty((h, 1)), db=cm.empty((h, 1)), lp=cm.empty((1, w)), zst=cm.empty((2, w)), dz=cm.empty((h, w)), dr=cm.empty((h, w)))
        sets.append(s)

    def step(s):
        s["x"].layer_norm(target=s["y"], stats=s["st"])
        s["dy"].layer_norm_deriv(s["x"], s["st"], target=s["dx"], grad_gain=s["dg"], grad_bias=s["db"])
        s["z"].log_prob(s["t"], target=s["lp"], stats=s["zst"])
        s["z"].log_prob_deriv(s["t"], s["zst"], s["g"], target=s["dz"])
        s["y"].dropout_scaled(0.25, target=s["dr"], add=s["x"], key=(4, 5))
    names = ("y", "dx", "dg", "db", "lp", "dz", "dr")
    for s, graph in zip(sets, graphs):
        with _On(cm, graph) as on:
            step(s)
        streams.append(on.stream)
    want = []
    for s in sets:
        step(s)
        want.append([get(s[n]) for n in names])
        for n in names:
            s[n].assign(0)
    cm.cuda_sync_threads()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        for n, v in zip(names, w):
            assert np.array_equal(get(s[n]), v), n


def test_matrices_of_more_than_2_to_31_elements(cm):
    """Their last columns as their own matrices give them."""
    h, w = 65536, 32800
    big = cm.empty((h, w))
    rng = np.random.default_rng(1)
    last = rng.standard_normal((h, 2)).astype(np.float32)

    def refill():
        big.slice(w - 2, w).assign(cm.CUDAMatrix(last))
    refill()
    lp, st, top, tops, t = cm.empty((1, w)), cm.empty((2, w)), cm.empty((4, w)), cm.empty((4, w)), cm.CUDAMatrix(np.full((1, w), 7.0))
    big.log_prob(t, target=lp, stats=st, top=top, top_tokens=tops)
    small, s1, p1, i1, t1 = cm.CUDAMatrix(last), cm.empty((2, 2)), cm.empty((4, 2)), cm.empty((4, 2)), cm.CUDAMatrix(np.full((1, 2), 7.0))
    l1 = small.log_prob(t1, stats=s1, top=p1, top_tokens=i1)
    # (sums in another grouping: within 2 (h / 32 + 100) roundings of values of some 12)
    tol = dict(rtol=0, atol=2 * (h / 32 + 100) * U * 12)
    np.testing.assert_allclose(get(lp)[:, -2:], get(l1), **tol)
    assert np.array_equal(get(tops)[:, -2:], get(i1)) and abs(get(lp)[0, 0] + np.log(h)) < 1e-4
    g = cm.CUDAMatrix(np.ones((1, w)))
    big.log_prob_deriv(t, st, g)
    small.log_prob_deriv(t1, s1, cm.CUDAMatrix(np.ones((1, 2))))
    np.testing.assert_allclose(get(big.slice(w - 2, w)), get(small), **tol)
    refill()
    small = cm.CUDAMatrix(last)
    big.dropout_scaled(0.5, key=(3, 4))
    cm.set_rng_column_offset(w - 2)
    try:
        small.dropout_scaled(0.5, key=(3, 4))
    finally:
        cm.set_rng_column_offset(0)
    assert np.array_equal(get(big.slice(w - 2, w)), get(small))
    refill()
    small = cm.CUDAMatrix(last)
    st1, gain = cm.empty((2, 2)), cm.empty((h, 1))
    big.layer_norm(stats=st)
    small.layer_norm(stats=st1)
    assert np.array_equal(get(big.slice(w - 2, w)), get(small)) and np.array_equal(get(st)[:, -2:], get(st1))
    big.layer_norm_deriv(big, st, grad_gain=gain)       # (any gradient will do: the normalised values themselves)
    small.layer_norm_deriv(small, st1)
    assert np.array_equal(get(big.slice(w - 2, w)), get(small))
    big.free_device_memory()


def test_calls_on_another_stream(cm):
    rng = np.random.default_rng(9)
    x, dy = (cm.CUDAMatrix(rng.standard_normal((513, 77)).astype(np.float32)) for _ in range(2))
    got = []
    for other in (False, True):
        y, st, dx, dg = cm.empty((513, 77)), cm.empty((2, 77)), cm.empty((513, 77)), cm.empty((513, 1))
        cm.cuda_sync_threads()

        def step():
            x.layer_norm(target=y, stats=st)
            dy.layer_norm_deriv(x, st, target=dx, grad_gain=dg)
        if other:
            with _On(cm):
                step()
        else:
            step()
        got.append([get(m) for m in (y, st, dx, dg)])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    assert cm.read_status() == 0
