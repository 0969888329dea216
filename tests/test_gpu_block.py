"""A layer over words built of the gradient-trained operators, forward and back, as a training loop calls them:
   n = layer_norm(x);  y = gated(n);  r = x + dropout(Wd' y);  z = Wo' r;  loss = -sum_j weight_j log softmax(z_j)[t_j]
against the same in 64 bits by automatic differentiation, and a few steps of descent on its own gradients."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def get(m):
    return np.array(m.asarray(), copy=True)


class Block(object):
    def __init__(self, cm, V, H, words, N, p, rng, act="silu"):
        f = lambda *s, scale=1.0: (rng.standard_normal(s) * scale).astype(np.float32)
        self.cm, self.p, self.act, self.shape = cm, p, act, (V, H, words, N)
        self.host = dict(gain=1 + f(V, 1, scale=0.1), bias=f(V, 1, scale=0.1), wg=f(V, H, scale=V ** -0.5), wu=f(V, H, scale=V ** -0.5),
                         bg=f(H, 1, scale=0.1), wd=f(H, V, scale=H ** -0.5), wo=f(V, words, scale=V ** -0.5))
        self.par = {k: cm.CUDAMatrix(v) for k, v in self.host.items()}
        self.grad = {k: cm.empty(v.shape) for k, v in self.host.items()}
        e = cm.empty
        self.n, self.st, self.gate, self.up, self.y = e((V, N)), e((2, N)), e((H, N)), e((H, N)), e((H, N))
        self.r, self.z, self.lp, self.zst, self.down = e((V, N)), e((words, N)), e((1, N)), e((2, N)), e((V, N))
        self.dr, self.dd, self.dy, self.dn, self.dx = e((V, N)), e((V, N)), e((H, N)), e((V, N)), e((V, N))

    def forward(self, x, tokens, key=None):
        cm, w = self.cm, self.par
        x.layer_norm(w["gain"], w["bias"], target=self.n, stats=self.st)
        cm.gated_product(w["wg"], w["wu"], self.n, self.y, activation=self.act, gate_bias=w["bg"], gate=self.gate, up=self.up)
        cm.dot(w["wd"].T, self.y, target=self.down)
        key = self.down.dropout_scaled(self.p, target=self.r, add=x, key=key)
        cm.dot(w["wo"].T, self.r, target=self.z)
        self.z.log_prob(tokens, target=self.lp, stats=self.zst)
        return key

    def back(self, x, tokens, weight, key):
        cm, w, g = self.cm, self.par, self.grad
        self.z.log_prob_deriv(tokens, self.zst, weight)                       # over the logits
        cm.dot(self.r, self.z.T, target=g["wo"])
        cm.dot(w["wo"], self.z, target=self.dr)
        self.dr.dropout_scaled(self.p, target=self.dd, key=key)
        cm.dot(self.y, self.dd.T, target=g["wd"])
        cm.dot(w["wd"], self.dd, target=self.dy)
        cm.gated_product_deriv(self.dy, self.gate, self.up, w["wg"], w["wu"], self.n, activation=self.act, grad_x=self.dn,
                               grad_gate_w=g["wg"], grad_up_w=g["wu"], grad_gate_bias=g["bg"])
        self.dn.layer_norm_deriv(x, self.st, w["gain"], target=self.dx, grad_gain=g["gain"], grad_bias=g["bias"])
        self.dx.add(self.dr)                                                  # the residual's way


@pytest.mark.parametrize("sizes", [(96, 160, 500, 40, 0.1), (131, 77, 301, 23, 0.5), (512, 1024, 2000, 256, 0.2), (64, 64, 100, 1, 0.0)])
def test_a_block_forward_and_back(cm, sizes):
    V, H, words, N, p = sizes
    rng = np.random.default_rng(V)
    b = Block(cm, V, H, words, N, p, rng)
    x, t = rng.standard_normal((V, N)).astype(np.float32), rng.integers(0, words, N)
    weight = ((rng.random(N) < 0.9) * (-1.0 / N)).astype(np.float32)
    gx, gt, gw = cm.CUDAMatrix(x), cm.CUDAMatrix(t[None].astype(np.float32)), cm.CUDAMatrix(weight[None])
    cm.CUDAMatrix.init_random(17)
    key = b.forward(gx, gt)
    ones = cm.CUDAMatrix(np.ones((V, N)))
    ones.dropout_scaled(p, key=key)
    mask = torch.from_numpy(get(ones).astype(np.float64))
    lp = get(b.lp)
    b.back(gx, gt, gw, key)
    # the same in 64 bits
    P = {k: torch.from_numpy(v.astype(np.float64)).requires_grad_() for k, v in b.host.items()}
    X = torch.from_numpy(x.astype(np.float64)).requires_grad_()
    m = X.mean(0)
    n = (X - m) / ((X - m).pow(2).mean(0) + 1e-5).sqrt() * P["gain"] + P["bias"]
    y = torch.nn.functional.silu(P["wg"].T @ n + P["bg"]) * (P["wu"].T @ n)
    z = P["wo"].T @ (X + mask * (P["wd"].T @ y))
    want = torch.log_softmax(z, 0)[torch.from_numpy(t), torch.arange(N)]
    (want * torch.from_numpy(weight.astype(np.float64))).sum().backward()
    # A product is off by 2^-18 of its magnitudes' product at most, a value by some 2^-20 elsewhere; on the way to a gradient lie at
    # most eight products and eight other steps, each of which takes an error on with a factor of 2 or less in the norm (weights of
    # norm 2 at most, a normalisation, slopes up to 1.1): 2^-18 x 8 x 1.25 on average paths, times 2 x 2 for the two that cross the
    # gate: 1.6e-4 of the largest entry.
    assert np.abs(lp[0] - want.detach().numpy()).max() < 1.6e-4 * np.abs(want.detach().numpy()).max()
    for name, got, grad in [("x", b.dx, X.grad)] + [(k, b.grad[k], P[k].grad) for k in b.grad]:
        w = grad.numpy()
        assert np.abs(get(got) - w).max() < 1.6e-4 * np.abs(w).max(), name
    assert cm.read_status() == 0


def test_descent_on_its_gradients(cm):
    """Runs, and the gradients stay finite; a captured and replayed step gives what the calls give one by one."""
    rng = np.random.default_rng(3)
    b = Block(cm, 96, 128, 300, 64, 0.1, rng, act="gelu")
    x, t = cm.CUDAMatrix(rng.standard_normal((96, 64)).astype(np.float32)), cm.CUDAMatrix(rng.integers(0, 300, (1, 64)).astype(np.float32))
    weight = cm.CUDAMatrix(np.full((1, 64), -1 / 64))
    cm.CUDAMatrix.init_random(5)
    for step in range(3):
        key = b.forward(x, t)
        b.back(x, t, weight, key)
        for k in b.par:
            b.par[k].add_mult(b.grad[k], -0.5)
    b.forward(x, t, key=(5, 99))
    lp = get(b.lp)
    b.back(x, t, weight, (5, 99))
    want = {k: get(v) for k, v in b.grad.items()}
    assert np.isfinite(lp).all() and all(np.isfinite(v).all() for v in want.values())
    torch.zeros(1, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    cm._check(cm._lib.b200_set_stream(stream.cuda_stream))
    try:
        b.forward(x, t, key=(5, 99))           # (the products' own scratch is taken before a capture)
        b.back(x, t, weight, (5, 99))
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            b.forward(x, t, key=(5, 99))
            b.back(x, t, weight, (5, 99))
    finally:
        cm._lib.b200_set_stream(None)
    for v in b.grad.values():
        v.assign(0)
    cm.cuda_sync_threads()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(get(b.lp), lp)
    for k, v in b.grad.items():
        assert np.array_equal(get(v), want[k]), k
    assert cm.read_status() == 0
