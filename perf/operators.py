"""Cases for timing the row operators: layer_norm and linear_act.

layer_norm  y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension.
linear_act  y = act(weight_gain * x @ weight^T + bias) * gain + residual.

A case is one call of one operator, without gradients (serving) or with the gradients of all its
inputs (training). `own` false computes it from elementary operations in 32 bits, `own` true calls
the package's operators.
"""

import math

import torch

own = False

EPS = 1e-5
SQRT2 = math.sqrt(2.0)
GAIN = {"linear": 1.0, "lrelu": SQRT2, "tanh": 1.0, "gelu": 1.0, "silu": 1.0}


def _ln(name, rows, n, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "n": n, "dtype": dtype, "train": train}


def _lin(name, rows, k, n, dtype, act, residual, train):
    return {"name": name, "op": "linear_act", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def listed():
    return [
        # the 17 latents (16 components and the global one) of one image, generated alone
        _ln("norm of one image's latents", 17, 512, "float32", False),
        # the latents of a training batch of 32 images
        _ln("norm of a batch's latents", 544, 512, "float32", True),
        # the tokens of 16 feature maps of 128x128 with 256 channels, generation
        _ln("norm of 128x128 tokens", 262144, 256, "bfloat16", False),
        # the tokens of 32 feature maps of 64x64 with 512 channels, training
        _ln("norm of 64x64 tokens", 131072, 512, "bfloat16", True),
        # a number of rows and of channels that no vector width divides
        _ln("norm of odd rows", 4099, 1021, "bfloat16", True),
        # one layer of the mapping network with its residual, one image
        _lin("mapping layer of one image", 17, 512, 512, "float32", "lrelu", True, False),
        # one single row against a wide layer: the weights are all there is to read
        _lin("one token", 1, 1024, 4096, "bfloat16", "gelu", False, False),
        # one layer of the mapping network in training, a batch of 32 images
        _lin("mapping layer of a batch", 544, 512, 512, "float32", "silu", True, True),
        # the query projection of 16 feature maps of 128x128, with a residual
        _lin("projection of 128x128 tokens", 262144, 256, 256, "bfloat16", "linear", True, False),
        # the widening layer of a feed-forward over 16 feature maps of 64x64, training
        _lin("feed-forward of 64x64 tokens", 65536, 512, 2048, "bfloat16", "gelu", False, True),
        # a matrix product that arithmetic bounds
        _lin("wide layer", 8192, 4096, 4096, "bfloat16", "gelu", True, False),
        # sizes that no tile and no vector width divides
        _lin("ragged layer", 1037, 515, 771, "bfloat16", "tanh", True, True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16"])
    train = rng.random() < 0.5
    if rng.random() < 0.4:
        n = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(262144, (1 << 26) // n))
        return {"op": "layer_norm", "rows": rows, "n": n, "dtype": dtype, "train": train}
    while True:
        n, k = _log(rng, 32, 4096), _log(rng, 32, 8192)
        rows = _log(rng, 1, 262144)
        if rng.random() < 0.5:
            n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
        if rows * n * k <= (1 << 36) // (4 if dtype == "float32" else 1) and rows * max(n, k) <= 1 << 27:
            break
    act = rng.choice(["linear", "tanh", "gelu", "silu"] + ([] if train else ["lrelu"]))
    return {"op": "linear_act", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act,
            "residual": rng.random() < 0.5, "train": train}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    rows, n, train = case["rows"], case["n"], case["train"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"op": case["op"], "train": train}
    if case["op"] == "layer_norm":
        # rows of different size and with a mean of their own, as activations have
        s["x"] = (randn(rows, n) * (0.5 + randn(rows, 1).abs()) + randn(rows, 1)).to(dtype)
        s["weight"] = 1.0 + 0.1 * randn(n)
        s["bias"] = 0.1 * randn(n)
        leaves = ["x", "weight", "bias"]
    else:
        k = case["k"]
        s["x"] = randn(rows, k).to(dtype)
        s["weight"] = randn(n, k).to(dtype)  # unit weights, scaled at run time
        s["bias"] = 0.1 * randn(n)
        s["residual"] = randn(rows, n).to(dtype) if case["residual"] else None
        s["act"], s["weight_gain"] = case["act"], 1.0 / math.sqrt(k)
        leaves = ["x", "weight", "bias"] + (["residual"] if case["residual"] else [])
    if train:
        s["dy"] = randn(rows, n).to(dtype)
        for name in leaves:
            s[name].requires_grad_()
    s["leaves"] = leaves
    return s


def _act(z, act):
    """The activation of z and its slope there."""
    if act == "lrelu":
        return torch.where(z > 0, z, 0.2 * z), torch.where(z > 0, 1.0, 0.2)
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / SQRT2))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _plain_layer_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = (xc.square().mean(1, keepdim=True) + EPS).rsqrt()
    h = xc * rstd
    out = {"y": (h * w + b).to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        out |= {"x": dx.to(s["x"].dtype), "weight": (dy * h).sum(0).to(s["weight"].dtype),
                "bias": dy.sum(0).to(s["bias"].dtype)}
    return out


def _plain_linear_act(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    z = (x @ w.t()) * s["weight_gain"] + b
    a, slope = _act(z, s["act"])
    y = a * GAIN[s["act"]]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(s["x"].dtype)}
    if s["train"]:
        dz = s["dy"].float() * (slope * GAIN[s["act"]])
        out |= {"x": (dz @ w * s["weight_gain"]).to(s["x"].dtype),
                "weight": (dz.t() @ x * s["weight_gain"]).to(s["weight"].dtype),
                "bias": dz.sum(0).to(s["bias"].dtype)}
        if s["residual"] is not None:
            out["residual"] = s["dy"]
    return out


def run(s):
    if not own:
        with torch.no_grad():
            return _plain_layer_norm(s) if s["op"] == "layer_norm" else _plain_linear_act(s)
    from gansformer_amd import ops
    with torch.set_grad_enabled(s["train"]):
        if s["op"] == "layer_norm":
            y = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        else:
            y = ops.linear_act(s["x"], s["weight"], s["bias"], act=s["act"], residual=s["residual"],
                               weight_gain=s["weight_gain"])
        if not s["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [s[name] for name in s["leaves"]], s["dy"])
    return {"y": y, **dict(zip(s["leaves"], grads))}


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    rows, n, train = case["rows"], case["n"], case["train"]
    if case["op"] == "layer_norm":
        # x and y, then dy and dx; the two parameters and their gradients
        return {"bytes": (4 if train else 2) * rows * n * e + (16 if train else 8) * n,
                "flops": (22 if train else 8) * rows * n}
    k = case["k"]
    inputs = rows * k + n * k + (rows * n if case["residual"] else 0)
    nbytes = (inputs + rows * n) * e + 4 * n
    if train:
        # dy is read, and the gradients of x, weight and bias are written; the residual's is dy
        nbytes += (rows * n + rows * k + n * k) * e + 4 * n
    return {"bytes": nbytes, "flops": (6 if train else 2) * rows * n * k}


def exact(case, seed):
    """The operators' definitions in 64 bits, with the gradients from automatic differentiation."""
    s = prepare(case, seed)
    wide = {name: s[name].detach().double().requires_grad_(s["train"]) for name in s["leaves"]}
    x, w, b = wide["x"], wide["weight"], wide["bias"]
    if s["op"] == "layer_norm":
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        y = torch.addcmul(b, (x - mean) / torch.sqrt(var + EPS), w)
    else:
        z = b + s["weight_gain"] * torch.matmul(x, w.transpose(0, 1))
        y = {"linear": lambda: z,
             "lrelu": lambda: torch.maximum(z, 0.2 * z),
             "tanh": lambda: torch.tanh(z),
             "gelu": lambda: z * torch.special.ndtr(z),
             "silu": lambda: z * torch.sigmoid(z)}[s["act"]]() * GAIN[s["act"]]
        if "residual" in wide:
            y = y + wide["residual"]
    out = {"y": y.detach()}
    if s["train"]:
        out |= dict(zip(s["leaves"], torch.autograd.grad(y, list(wide.values()), s["dy"].double())))
    return out
