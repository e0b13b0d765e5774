"""The operators of a transformer's feed-forward layer, as cases that can be timed.

A case is a dict of plain values.  `kind` names the operator:

  fc         Engine.fullConnect          Y = act(X W^T + b) + R                  X [rows][IC], W [OC][IC]
  fc_delta   Engine.fullConnect_delta    deltaX, deltaW, deltaB of it from deltaY and the saved Z = X W^T + b
  glu        Engine.fullConnect_glu      Y = act(g) u, g and u the halves of X W^T + b     W [2 OC][IC]
  glu_delta  Engine.fullConnect_glu_delta
  clip       Engine.clip_grad_norm       the norm of all gradients of a step, and the gradients scaled down to max_norm

With `own` false `run` computes them in elementary torch operations, in 32 bits (norms in 64), rounded once at the end; with `own`
true through the library.  Inputs N(0, 1), weights N(0, 1 / IC), so that sums are N(0, 1) too; output gradients N(0, 1).
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SLOPE = 0.2          # of leakyRelu


def _case(name, kind, **values):
    return dict(name=name, kind=kind, **values)


def listed():
    return [
        # one token of a serving program: the projection back to the model's width, added to the residual stream
        _case("fc_token", "fc", dtype="bf16", rows=1, IC=11008, OC=4096, act="none", bias=False, residual=True, save=False),
        # a ragged batch through a layer whose sizes are multiples of nothing, training (Z is kept)
        _case("fc_ragged_f16", "fc", dtype="f16", rows=777, IC=1001, OC=1507, act="gelu", bias=True, residual=True, save=True),
        # a classifier's FullConnect layer with its activation in fp32, as the rest of the engine runs it
        _case("fc_1000_f32", "fc", dtype="f32", rows=512, IC=4096, OC=1000, act="leakyRelu", bias=True, residual=False, save=False),
        # training: the gradients of a wide biased layer
        _case("fc_delta_bf16", "fc_delta", dtype="bf16", rows=4096, IC=4096, OC=16384, act="gelu_tanh", bias=True),
        # the classifier's gradients
        _case("fc_delta_1000_f32", "fc_delta", dtype="f32", rows=512, IC=4096, OC=1000, act="leakyRelu", bias=True),
        # four sequences decoding one token each through a gated block
        _case("glu_token", "glu", dtype="bf16", rows=4, IC=4096, OC=11008, act="silu", bias=False, save=False),
        # training: the gated block over 8192 tokens, both projections kept for the backward pass
        _case("glu_train_bf16", "glu", dtype="bf16", rows=8192, IC=4096, OC=11008, act="silu", bias=False, save=True),
        # a smaller gated block in fp32
        _case("glu_f32", "glu", dtype="f32", rows=1000, IC=1024, OC=2752, act="gelu", bias=True, save=False),
        # training: the gradients of the gated block (the largest case)
        _case("glu_delta_bf16", "glu_delta", dtype="bf16", rows=8192, IC=4096, OC=11008, act="silu", bias=False),
        # the gradients of a gated block of odd sizes over a ragged batch
        _case("glu_delta_ragged_f16", "glu_delta", dtype="f16", rows=1237, IC=770, OC=2050, act="sigmoid", bias=True),
        # the gradients of the CIFAR-10 ResNet-18's convolutions, fp32
        _case("clip_resnet18", "clip", dtype="f32", out="f32", model="resnet18", scale=1e-3, max_norm=1.0),
        # the gradients of four transformer layers, 0.8 billion elements in bf16
        _case("clip_layers_bf16", "clip", dtype="bf16", out="bf16", model="layers", layers=4, D=4096, H=11008, scale=1e-3, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("fc", "fc", "fc_delta", "glu", "glu", "glu_delta", "clip"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "clip":
        return dict(kind=kind, dtype=dtype, out=rng.choice((dtype, "f32")), model="ragged", tensors=_log(rng, 1, 60), most=_log(rng, 1000, 2000000),
                    sizes=rng.randrange(1 << 30), scale=math.exp(rng.uniform(math.log(1e-4), math.log(1.0))), max_norm=math.exp(rng.uniform(-2.0, 4.0)))
    while True:
        # half of the widths are multiples of 64, half are whatever the log scale gives
        IC, OC = [_log(rng, 20, 12000) if rng.random() < 0.5 else 64 * _log(rng, 1, 180) for _ in range(2)]
        rows = _log(rng, 1, 8192)
        flops = 2.0 * rows * IC * OC * (2 if "glu" in kind else 1) * (2 if "delta" in kind else 1)
        if 1e5 <= flops <= (2.5e11 if dtype == "f32" else 2e12) and max(IC, rows) * OC <= 9e7:
            break
    c = dict(kind=kind, dtype=dtype, rows=rows, IC=IC, OC=OC, bias=rng.random() < 0.5,
             act=rng.choice(("sigmoid", "silu", "gelu", "gelu_tanh", "leakyRelu") + (("none",) if "glu" not in kind else ())))
    if kind == "fc":
        c["residual"] = rng.random() < 0.5
    if "delta" not in kind:
        c["save"] = rng.random() < 0.5
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------

def _grad_shapes(case):
    if case["model"] == "layers":
        D, H = case["D"], case["H"]
        return [s for _ in range(case["layers"]) for s in ((D, D), (D, D), (D, D), (D, D), (2 * H, D), (D, H), (D,), (D,))]
    if case["model"] == "ragged":
        rng = random.Random(case["sizes"])
        return [(_log(rng, 1, case["most"]),) for _ in range(case["tensors"])]
    shapes, cin = [(64, 7, 7, 4)], 64
    for cout, blocks in ((64, 2), (128, 2), (256, 2), (512, 2)):
        for b in range(blocks):
            shapes += [(cout, 3, 3, cin), (cout, 3, 3, cout)] + ([(cout, 3, 3, cin)] if cin != cout else [])
            cin = cout
    return shapes


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, device=dev, generator=g).mul_(scale).to(t)

    if case["kind"] == "clip":
        return dict(grads=[normal(*s, scale=case["scale"]) for s in _grad_shapes(case)])
    rows, IC, OC = case["rows"], case["IC"], case["OC"]
    wide = 2 * OC if "glu" in case["kind"] else OC
    x = dict(X=normal(rows, IC), W=normal(wide, IC, scale=1.0 / math.sqrt(IC)))
    if "delta" in case["kind"]:
        x["dY"] = normal(rows, OC)
        x["Z"] = normal(rows, wide)
    else:
        if case["bias"]:
            x["B"] = normal(wide, scale=0.1)
        if case.get("residual"):
            x["R"] = normal(rows, OC)
    return x


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        from __graft_entry__ import submodule
        st["eng"] = submodule("engine").Engine()
    if case["kind"] == "clip":
        st["out"] = [torch.empty_like(a, dtype=_TYPES[case["out"]]) for a in st["grads"]]   # what the optimizer reads
    return st


# ---- the plain form ---------------------------------------------------------------------------------------------

def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _act(z, name):
    if name == "none":
        return z
    if name == "leakyRelu":
        return torch.where(z > 0, z, _SLOPE * z)
    if name == "sigmoid":
        return _sigmoid(z)
    if name == "silu":
        return z * _sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_slope(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "leakyRelu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, _SLOPE))
    if name == "sigmoid":
        s = _sigmoid(z)
        return s * (1.0 - s)
    if name == "silu":
        s = _sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    a = math.sqrt(2.0 / math.pi)
    th = torch.tanh(a * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * a * (1.0 + 3 * 0.044715 * z * z)


def _plain(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "clip":
        norm = torch.sqrt(sum(torch.sum(a.double() * a.double()) for a in st["grads"]))
        scale = torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0).float()
        for o, a in zip(st["out"], st["grads"]):
            o.copy_(a.float() * scale)
        return [norm.float()] + st["out"]
    t, OC, act = _TYPES[c["dtype"]], c["OC"], c["act"]
    X, W = st["X"].float(), st["W"].float()
    if "delta" not in kind:
        z = X @ W.t()
        if "B" in st:
            z = z + st["B"].float()
        y = _act(z, act) if kind == "fc" else _act(z[:, :OC], act) * z[:, OC:]
        if "R" in st:
            y = y + st["R"].float()
        return (y.to(t), z.to(t)) if c["save"] else y.to(t)
    dY, Z = st["dY"].float(), st["Z"].float()
    if kind == "fc_delta":
        dZ = dY * _act_slope(Z, act)
    else:
        G, U = Z[:, :OC], Z[:, OC:]
        dZ = torch.cat((dY * U * _act_slope(G, act), dY * _act(G, act)), dim=1)
    out = [(dZ @ W).to(t), (dZ.t() @ X).to(t)]
    return out + [dZ.sum(0).to(t)] if c["bias"] else out


def run(state):
    if not own:
        return _plain(state)
    c, eng = state["case"], state["eng"]
    kind = c["kind"]
    if kind == "clip":
        norm = eng.clip_grad_norm(state["grads"], c["max_norm"], Out=state["out"])
        return [norm] + state["out"]
    if kind == "fc":
        return eng.fullConnect(state["X"], state["W"], state.get("B"), act=c["act"], k=_SLOPE, Residual=state.get("R"), save=c["save"])
    if kind == "glu":
        return eng.fullConnect_glu(state["X"], state["W"], state.get("B"), act=c["act"], k=_SLOPE, save=c["save"])
    delta = eng.fullConnect_delta if kind == "fc_delta" else eng.fullConnect_glu_delta
    out = delta(state["dY"], state["X"], state["W"], state["Z"], act=c["act"], k=_SLOPE, bias=c["bias"])
    return list(out) if c["bias"] else list(out[:2])


# ---- what the operators cannot do without ------------------------------------------------------------------------

def work(case):
    size = torch.finfo(_TYPES[case["dtype"]]).bits // 8
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _grad_shapes(case))
        return {"bytes": float(n * (size + torch.finfo(_TYPES[case["out"]]).bits // 8)), "flops": 3.0 * n}
    rows, IC, OC = case["rows"], case["IC"], case["OC"]
    wide = 2 * OC if "glu" in case["kind"] else OC
    x, w, y, z = rows * IC, wide * IC, rows * OC, rows * wide
    b = wide if case["bias"] else 0
    if "delta" in case["kind"]:
        needs_z = z if case["act"] != "none" else 0
        return {"bytes": float(size * (2 * x + 2 * w + y + needs_z + b)), "flops": 4.0 * rows * IC * wide}
    return {"bytes": float(size * (x + w + b + y * (2 if case.get("residual") else 1) + (z if case["save"] else 0))), "flops": 2.0 * rows * IC * wide}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _f64(z, name):
    """Value and slope of an activation, from its definition."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "leakyRelu":
        s = torch.where(z > 0, 1.0, torch.full_like(z, _SLOPE))
        return s * z, s
    if name in ("sigmoid", "silu"):
        e = torch.exp(-z.abs())
        s = torch.where(z >= 0, 1 / (1 + e), e / (1 + e))
        ds = e / (1 + e) ** 2
        return (s, ds) if name == "sigmoid" else (z * s, s + z * ds)
    if name == "gelu":                       # z times the normal distribution function
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    th = torch.tanh(u)
    return z * (1 + th) / 2, (1 + th) / 2 + z / 2 * (1 - th ** 2) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)


def exact(case, seed):
    x = {k: ([a.double() for a in v] if k == "grads" else v.double()) for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(a) for a in x["grads"]]))
        scale = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return [norm] + [a.mul_(scale) for a in x["grads"]]
    OC, act = case["OC"], case["act"]
    if kind in ("fc", "glu"):
        z = torch.mm(x["X"], x["W"].T)
        z += x.get("B", 0.0)
        y = _f64(z, act)[0] if kind == "fc" else _f64(z[:, :OC], act)[0] * z[:, OC:]
        y = y + x.get("R", 0.0)
        return (y, z) if case["save"] else y
    if kind == "fc_delta":
        dZ = x["dY"] * _f64(x["Z"], act)[1]
    else:
        value, slope = _f64(x["Z"][:, :OC], act)
        dZ = torch.cat([x["dY"] * x["Z"][:, OC:] * slope, x["dY"] * value], dim=1)
    out = [torch.mm(dZ, x["W"]), torch.mm(dZ.T, x["X"])]
    return out + [dZ.sum(dim=0)] if case["bias"] else out
