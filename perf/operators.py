"""The operators of a feed-forward layer over words, as cases that can be timed and compared.

A case is one pass through an operator as a user's program calls it: a forward call as it is made to serve,
or a forward call and its derivative as they are made to train.  The kinds:

  layer_norm   `CUDAMatrix.layer_norm`, `layer_norm_deriv`: every column normalised; gradients of input, gain and bias
  gated        `gated_product`, `gated_product_deriv`: act(Wg'x + bg) * (Wu'x + bu); gradients of all five
  dropout      `CUDAMatrix.dropout_scaled`: a mask drawn from (seed, call), scaled, joined to a residual; the same mask on the gradient
  log_prob     `CUDAMatrix.log_prob`, `log_prob_deriv`: log probability of a given word a column, entropy, likeliest words; gradient

Matrices are float32 and hold one case (word, token) a column, columns one after another in memory: a torch
tensor of cases x dims is the same memory.  `own` false computes the plain forms in elementary torch operations.
"""
import ctypes as ct
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # one minibatch of the features that a small layer is fed with, to be normalised before it
        dict(name="norm_784x100", kind="layer_norm", V=784, N=100, train=False),
        # odd feature count, more cases than a minibatch usually has: a training step's forward and backward pass
        dict(name="norm_train_1357x2003", kind="layer_norm", V=1357, N=2003, train=True),
        # a wide layer over the tokens of a large step
        dict(name="norm_train_4096x8192", kind="layer_norm", V=4096, N=8192, train=True),
        # one token at a time, as text is written: bound by the weights' bytes
        dict(name="gated_2048x8192x1", kind="gated", V=2048, H=8192, N=1, act="silu", bias=False, train=False),
        # a layer of odd sizes run over a held-out minibatch
        dict(name="gated_1357x601x203", kind="gated", V=1357, H=601, N=203, act="gelu", bias=True, train=False),
        # the layer sizes of the small models here, a training step
        dict(name="gated_train_784x500x100", kind="gated", V=784, H=500, N=100, act="logistic", bias=True, train=True),
        # a wide layer, a training step: bound by the products
        dict(name="gated_train_2048x8192x4096", kind="gated", V=2048, H=8192, N=4096, act="silu", bias=False, train=True),
        # hidden units of a small layer dropped
        dict(name="dropout_500x100", kind="dropout", V=500, N=100, p=0.5, residual=False, train=False),
        # a layer's output dropped and joined to its input, and the gradient that comes back through it
        dict(name="dropout_train_4096x8192", kind="dropout", V=4096, N=8192, p=0.1, residual=True, train=True),
        # the next word's candidates over a 10 000 word vocabulary
        dict(name="words_10000x1", kind="log_prob", V=10000, N=1, top=8, train=False),
        # held-out text scored, with the words the model would rather have had
        dict(name="words_50021x777", kind="log_prob", V=50021, N=777, top=20, train=False),
        # a training step over 10 000 words, some columns without weight
        dict(name="words_train_10000x4096", kind="log_prob", V=10000, N=4096, top=0, train=True),
    ]


def draw(rng):
    """One more case of the same kinds and ranges."""
    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice([1, 1, 1, 4, 10, 64])
        return max(lo, min(hi, n // step * step))

    kind = rng.choice(["layer_norm", "gated", "gated", "dropout", "log_prob", "log_prob"])
    train = rng.random() < 0.6
    if kind == "layer_norm":
        V = size(16, 16384)
        return dict(kind=kind, V=V, N=size(1, max(1, min(8192, (4096 * 8192) // V))), train=train)
    if kind == "gated":
        V, H = size(64, 4096), size(64, 8192)
        return dict(kind=kind, V=V, H=H, N=size(1, max(1, min(4096, (2048 * 8192 * 4096) // (V * H)))),
                    act=rng.choice(["silu", "gelu", "logistic", "relu", "linear"]), bias=rng.random() < 0.5, train=train)
    if kind == "dropout":
        V = size(16, 8192)
        return dict(kind=kind, V=V, N=size(1, max(1, min(8192, (4096 * 8192) // V))), p=rng.choice([0.05, 0.1, 0.2, 0.5, 0.8]),
                    residual=rng.random() < 0.5, train=train)
    V = size(64, 100000)
    return dict(kind=kind, V=V, N=size(1, max(1, min(4096, (10000 * 4096) // V))), top=rng.choice([0, 1, 5, 20]),
                train=train)


# -- inputs ---------------------------------------------------------------------------------
def _inputs(case, seed):
    """What goes into a case, from its seed: tensors of cases x dims (weights: units x inputs)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind, V, N, train = case["kind"], case["V"], case["N"], case["train"]
    x = {}
    if kind == "layer_norm":
        # features of different scales and offsets, cases of different size
        x["x"] = (normal(N, V) * (0.5 + normal(V).abs()) + 0.5 * normal(V)) * (0.25 + normal(N, 1).abs())
        x["gain"], x["bias"] = 1.0 + 0.2 * normal(V), 0.2 * normal(V)
        if train:
            x["dy"] = normal(N, V) / N
    elif kind == "gated":
        H = case["H"]
        x["x"] = normal(N, V)
        x["wg"], x["wu"] = normal(H, V) / math.sqrt(V), normal(H, V) / math.sqrt(V)
        if case["bias"]:
            x["bg"], x["bu"] = 0.3 * normal(H), 0.3 * normal(H)
        if train:
            x["dy"] = normal(N, H) / N
    elif kind == "dropout":
        x["x"] = normal(N, V)
        if case["residual"]:
            x["add"] = normal(N, V)
        if train:
            x["dy"] = normal(N, V) / N
        x["key"] = (seed & 0x7FFFFFFF, 1 + seed % 1000)
    else:
        # words by Zipf(1.07) over a shuffled vocabulary, each column with its own preferences
        place = torch.randperm(V, generator=g, device="cuda").float()
        x["z"] = normal(N, V).mul_(2.0).add_(-1.07 * torch.log(place + 1.0))
        # words that came up, likely and unlikely ones
        likely = (x["z"][:, : max(1, V // 16)]).argmax(1)
        other = torch.randint(0, V, (N,), generator=g, device="cuda")
        x["t"] = torch.where(torch.rand(N, generator=g, device="cuda") < 0.7, likely, other).float()
        if train:
            weight = (torch.rand(N, generator=g, device="cuda") < 0.95).float()      # padded columns weigh nothing
            x["g"], x["h"] = -weight / N, 0.01 * weight / N
    return x


def _over(cm, x, rows=None):
    """The memory of the (cases x dims) tensor x as a matrix with one case a column; a vector is a column."""
    mat = cm.cudamat()
    mat.data_device = ct.cast(x.data_ptr(), ct.POINTER(ct.c_float))
    mat.on_device = 1
    mat.size[0], mat.size[1] = (x.shape[1], x.shape[0]) if x.dim() == 2 else (x.shape[0], 1) if rows is None else (rows, x.numel() // rows)
    m = cm.CUDAMatrix._from_mat(mat)
    m.tensor = x
    return m


def prepare(case, seed):
    x = _inputs(case, seed)
    s = dict(case=case, x=x)
    if own:
        from deepnet_b200 import b200mat as cm
        cm.cublas_init()
        kind, V, N, train = case["kind"], case["V"], case["N"], case["train"]
        row = ("t", "g", "h")
        m = {k: _over(cm, v, 1 if k in row else None) for k, v in x.items() if k != "key"}

        def room(name, *shape):
            s["out"][name] = torch.empty(*shape, device="cuda")
            m[name] = _over(cm, s["out"][name])

        s.update(cm=cm, m=m, out={})
        if kind == "layer_norm":
            room("y", N, V)
            if train:
                room("stats", N, 2), room("dx", N, V), room("dgain", V), room("dbias", V)
        elif kind == "gated":
            H = case["H"]
            room("y", N, H)
            if train:
                for name, shape in (("gate", (N, H)), ("up", (N, H)), ("dx", (N, V)), ("dwg", (H, V)), ("dwu", (H, V))):
                    room(name, *shape)
                if case["bias"]:
                    room("dbg", H), room("dbu", H)
            else:
                # weights that stay as they are keep their layout for the tensor cores
                s["planes"] = cm.GatedPlanes(m["wg"], m["wu"])
        elif kind == "dropout":
            room("y", N, V)
            if train:
                room("dx", N, V)
        else:
            room("logp", N, 1), room("entropy", N, 1)
            if case["top"]:
                room("top", N, case["top"]), room("words", N, case["top"])
            if train:
                room("stats", N, 2), room("dz", N, V)
        torch.cuda.synchronize()
        cm.cuda_sync_threads()
    return s


# -- one pass -------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"layer_norm": _own_norm, "gated": _own_gated, "dropout": _own_dropout, "log_prob": _own_words}[kind](s["case"], s["m"], s)
    return {"layer_norm": _norm, "gated": _gated, "dropout": _dropout, "log_prob": _words}[kind](s["case"], s["x"])


def _own_norm(case, m, s):
    out = s["out"]
    if not case["train"]:
        m["x"].layer_norm(m["gain"], m["bias"], eps=EPS, target=m["y"])
        return [out["y"]]
    m["x"].layer_norm(m["gain"], m["bias"], eps=EPS, target=m["y"], stats=m["stats"])
    m["dy"].layer_norm_deriv(m["x"], m["stats"], m["gain"], target=m["dx"], grad_gain=m["dgain"], grad_bias=m["dbias"])
    return [out[k] for k in ("y", "dx", "dgain", "dbias")]


def _norm(case, x):
    centred = x["x"] - x["x"].mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xh = centred * rs
    y = xh * x["gain"] + x["bias"]
    if not case["train"]:
        return [y]
    a = x["dy"] * x["gain"]
    dx = rs * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return [y, dx, (x["dy"] * xh).sum(0), x["dy"].sum(0)]


def _own_gated(case, m, s):
    cm, out = s["cm"], s["out"]
    bias = dict(gate_bias=m["bg"], up_bias=m["bu"]) if case["bias"] else {}
    if not case["train"]:
        cm.gated_product(m["wg"], m["wu"], m["x"], m["y"], activation=case["act"], planes=s["planes"], **bias)
        return [out["y"]]
    cm.gated_product(m["wg"], m["wu"], m["x"], m["y"], activation=case["act"], gate=m["gate"], up=m["up"], **bias)
    grads = dict(grad_gate_bias=m["dbg"], grad_up_bias=m["dbu"]) if case["bias"] else {}
    cm.gated_product_deriv(m["dy"], m["gate"], m["up"], m["wg"], m["wu"], m["x"], activation=case["act"], grad_x=m["dx"],
                           grad_gate_w=m["dwg"], grad_up_w=m["dwu"], **grads)
    return [out[k] for k in ("y", "dx", "dwg", "dwu", "dbg", "dbu") if k in out]


def _activation(name, g):
    """act(g) and its derivative."""
    if name == "linear":
        return g, torch.ones_like(g)
    if name == "relu":
        return g * (g > 0), (g > 0).to(g.dtype)
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * math.sqrt(0.5 / math.pi)
    p = 1.0 / (1.0 + torch.exp(-g))
    return (p, p * (1.0 - p)) if name == "logistic" else (g * p, p * (1.0 + g * (1.0 - p)))


def _gated(case, x):
    gate, up = x["x"] @ x["wg"].T, x["x"] @ x["wu"].T
    if case["bias"]:
        gate, up = gate + x["bg"], up + x["bu"]
    a, slope = _activation(case["act"], gate)
    y = a * up
    if not case["train"]:
        return [y]
    dgate, dup = x["dy"] * up * slope, x["dy"] * a
    out = [y, dgate @ x["wg"] + dup @ x["wu"], dgate.T @ x["x"], dup.T @ x["x"]]
    return out + [dgate.sum(0), dup.sum(0)] if case["bias"] else out


def _own_dropout(case, m, s):
    out, p, key = s["out"], case["p"], s["x"]["key"]
    m["x"].dropout_scaled(p, target=m["y"], add=m.get("add"), key=key)
    if not case["train"]:
        return [out["y"]]
    m["dy"].dropout_scaled(p, target=m["dx"], key=key)
    return [out["y"], out["dx"]]


def _uniforms(V, N, key):
    """Uniforms in (0, 1]: element (row r, column c) is word c & 3 of Philox4x32-10 at counter {r, c >> 2, call, 0}, key {seed, 0}."""
    low = 0xFFFFFFFF
    c0 = torch.arange(V, device="cuda").repeat((N + 3) // 4, 1)
    c1 = torch.arange((N + 3) // 4, device="cuda")[:, None].expand_as(c0)
    c2, c3 = torch.full_like(c0, key[1]), torch.zeros_like(c0)
    k0, k1 = key[0], 0

    def product(a, c):
        """High and low words of a c, both below 2^32 (in halves of c: 64-bit integers have a sign)."""
        t = a * (c & 0xFFFF)
        u = a * (c >> 16) + (t >> 16)
        return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)

    for _ in range(10):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1).reshape(-1, V)[:N]
    return (words.float() + 1.0) * 2.3283064365386963e-10


def _dropout(case, x):
    keep = _uniforms(case["V"], case["N"], x["key"]) > case["p"]
    scaled = keep.float() * (1.0 / (1.0 - case["p"]))
    y = x["x"] * scaled
    if case["residual"]:
        y = y + x["add"]
    return [y, x["dy"] * scaled] if case["train"] else [y]


def _own_words(case, m, s):
    out = s["out"]
    m["z"].log_prob(m["t"], target=m["logp"], entropy=m["entropy"], stats=m.get("stats"), top=m.get("top"), top_tokens=m.get("words"))
    got = [out["logp"], out["entropy"]] + ([out["top"], out["words"]] if case["top"] else [])
    if case["train"]:
        m["z"].log_prob_deriv(m["t"], m["stats"], m["g"], entropy=m["entropy"], grad_entropy=m["h"], target=m["dz"])
        got.append(out["dz"])
    return got


def _words(case, x):
    z, N = x["z"], case["N"]
    t = x["t"].long()
    d = z - z.max(1, keepdim=True).values
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logs = d - torch.log(total)
    p = e / total
    logp = logs.gather(1, t[:, None])
    entropy = -(p * logs).sum(1, keepdim=True)
    out = [logp, entropy]
    if case["top"]:
        # ordered as whole numbers, a word's place below its logit: equal logits go by the lower word
        bits = z.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        words = torch.topk((order << 24) - torch.arange(z.shape[1], device="cuda"), case["top"], dim=1).indices
        out += [logs.gather(1, words), words.float()]
    if case["train"]:
        dz = -(p * (x["g"][:, None] + x["h"][:, None] * (logs + entropy)))
        dz[torch.arange(N, device="cuda"), t] += x["g"]
        out.append(dz)
    return out


# -- what a pass cannot do without ------------------------------------------------------------
def work(case):
    kind, V, N, train = case["kind"], case["V"], case["N"], case["train"]
    if kind == "layer_norm":
        # input in, output out, gain and bias; back: gradient in, gradients out (the input is read once for both)
        return dict(bytes=4.0 * (2 * V * N + 2 * V + (2 * V * N + 2 * V if train else 0)), flops=(18.0 if train else 7.0) * V * N)
    if kind == "gated":
        H, biases = case["H"], 2 * case["H"] if case["bias"] else 0
        if train:
            return dict(bytes=4.0 * (4 * V * H + 2 * V * N + 2 * H * N + 2 * biases), flops=12.0 * V * H * N)
        return dict(bytes=4.0 * (2 * V * H + V * N + H * N + biases), flops=4.0 * V * H * N)
    if kind == "dropout":
        return dict(bytes=4.0 * V * N * (2 + bool(case["residual"]) + (2 if train else 0)), flops=2.0 * V * N)
    return dict(bytes=4.0 * (V * N + 3 * N + 2 * case["top"] * N + (V * N + 2 * N if train else 0)), flops=(10.0 if train else 5.0) * V * N)


# -- the same in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    """What `run` returns, from the definitions, in 64 bits."""
    kind, N = case["kind"], case["N"]
    raw = _inputs(case, seed)
    x = {k: v.double() for k, v in raw.items() if k != "key"}
    if kind == "layer_norm":
        x["x"].requires_grad_(case["train"]), x["gain"].requires_grad_(case["train"]), x["bias"].requires_grad_(case["train"])
        var, mean = torch.var_mean(x["x"], 1, unbiased=False, keepdim=True)
        y = (x["x"] - mean) / (var + EPS).sqrt() * x["gain"] + x["bias"]
        if not case["train"]:
            return [y]
        y.backward(x["dy"])
        return [y.detach(), x["x"].grad, x["gain"].grad, x["bias"].grad]
    if kind == "gated":
        leaves = [x[k].requires_grad_(case["train"]) for k in ("x", "wg", "wu", "bg", "bu") if k in x]
        act = {"linear": lambda v: v, "relu": torch.relu, "logistic": torch.sigmoid, "silu": torch.nn.functional.silu,
               "gelu": torch.nn.functional.gelu}[case["act"]]
        y = act(torch.addmm(x.get("bg", x["x"].new_zeros(case["H"])), x["x"], x["wg"].T)) * torch.addmm(
            x.get("bu", x["x"].new_zeros(case["H"])), x["x"], x["wu"].T)
        if not case["train"]:
            return [y]
        y.backward(x["dy"])
        return [y.detach()] + [v.grad for v in leaves]
    if kind == "dropout":
        keep = _uniforms_exactly(case["V"], N, raw["key"]) > torch.tensor(case["p"], dtype=torch.float32).item()
        y = torch.where(keep, x["x"] / (1.0 - case["p"]), 0.0) + (x["add"] if case["residual"] else 0.0)
        return [y, torch.where(keep, x["dy"] / (1.0 - case["p"]), 0.0)] if case["train"] else [y]
    z = x["z"].requires_grad_(case["train"])
    logs = torch.log_softmax(z, 1)
    logp = logs.gather(1, raw["t"].long().view(N, 1))
    entropy = -torch.special.xlogy(logs.exp(), logs.exp()).sum(1, keepdim=True)
    out = [logp.detach(), entropy.detach()]
    if case["top"]:
        ranked = torch.sort(raw["z"], dim=1, descending=True, stable=True).indices[:, : case["top"]]
        out += [logs.detach().gather(1, ranked), ranked.double()]
    if case["train"]:
        ((logp[:, 0] * x["g"]).sum() + (entropy[:, 0] * x["h"]).sum()).backward()
        out.append(z.grad)
    return out


def _uniforms_exactly(V, N, key):
    """The uniforms of `_uniforms` with the products' words taken from 64-bit arithmetic on numpy's unsigned integers."""
    import numpy as np
    u32, u64 = np.uint32, np.uint64
    c, r = np.meshgrid(np.arange((N + 3) // 4, dtype=u32), np.arange(V, dtype=u32), indexing="ij")
    a = [r, c, np.full_like(r, key[1]), np.zeros_like(r)]
    k = [key[0] & 0xFFFFFFFF, key[0] >> 32]
    for i in range(10):
        p, q = u64(0xD2511F53) * a[0].astype(u64), u64(0xCD9E8D57) * a[2].astype(u64)
        a = [(q >> u64(32)).astype(u32) ^ a[1] ^ u32((k[0] + i * 0x9E3779B9) & 0xFFFFFFFF), q.astype(u32),
             (p >> u64(32)).astype(u32) ^ a[3] ^ u32((k[1] + i * 0xBB67AE85) & 0xFFFFFFFF), p.astype(u32)]
    words = np.stack(a, 1).reshape(-1, V)[:N]
    uniform = (words.astype(np.float32) + np.float32(1.0)) * np.float32(2.3283064365386963e-10)
    return torch.from_numpy(uniform).cuda()
