"""The operators around a network's convolutions and FullConnect layers in a training step, as cases that can be timed: the normalisation between layers,
the loss over a vocabulary or a set of classes, and the optimizer's update.

A case is a dict of plain values.  `kind` names the operator:

  norm        Engine.groupNorm          Y = act((X - mean) rstd gamma + beta) over groups of channels of X [N][H][W][C]
  norm_delta  Engine.groupNorm_delta    deltaX, deltaGamma, deltaBeta of it from deltaY, X and the saved mean and rstd
  loss        Engine.fullConnect_softmax_crossEntropy        logsumexp(z) - z[label] for every row of z = X W^T + b, which is not kept
  loss_delta  Engine.fullConnect_softmax_crossEntropy_delta  deltaX, deltaW, deltaB of it from the saved logsumexp
  adamw       Engine.adamW              a step over many tensors, moments in 32 bits or in 8 (e4m3 with a power of two for each 32 elements, rounded
              up or down at random: the random bits come from a seed, the step and an element's place)

With `own` false `run` computes them in elementary torch operations, in 32 bits, rounded once at the end; with `own` true through the library.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SLOPE = 0.2          # of leakyRelu
_BETA1, _BETA2, _EPS, _LR, _DECAY = 0.9, 0.999, 1e-8, 1e-3, 0.01
_BLOCK = 32           # elements of an 8-bit moment that share a scale


def _case(name, kind, **values):
    return dict(name=name, kind=kind, **values)


def listed():
    return [
        # four drafted or candidate tokens scored over a vocabulary: W is read once
        _case("loss_tokens", "loss", dtype="bf16", rows=4, IC=4096, OC=128000, bias=False, ignored=0.0),
        # training a language model's head: the loss of 4096 tokens
        _case("loss_train_bf16", "loss", dtype="bf16", rows=4096, IC=4096, OC=128000, bias=False, ignored=0.05),
        # its gradients (the largest case)
        _case("loss_delta_bf16", "loss_delta", dtype="bf16", rows=4096, IC=4096, OC=128000, bias=False, ignored=0.05),
        # the gradients of a ragged batch over a vocabulary that is a multiple of nothing, a fifth of it padding
        _case("loss_delta_ragged_f16", "loss_delta", dtype="f16", rows=777, IC=1001, OC=30011, bias=True, ignored=0.2),
        # a classifier's gradients in fp32, as the rest of the engine runs it
        _case("loss_delta_1000_f32", "loss_delta", dtype="f32", rows=512, IC=4096, OC=1000, bias=True, ignored=0.0),
        # one small picture of an inference program
        _case("norm_small_bf16", "norm", dtype="bf16", N=1, H=16, W=16, C=320, groups=32, act="silu", save=False),
        # the first stage of a CIFAR-10 ResNet in fp32, batch 512, training
        _case("norm_32x32x64_f32", "norm", dtype="f32", N=512, H=32, W=32, C=64, groups=32, act="leakyRelu", save=True),
        # one large picture, whose groups fit no SM
        _case("norm_large_bf16", "norm", dtype="bf16", N=1, H=512, W=512, C=256, groups=32, act="silu", save=False),
        # gradients of 56x56x64 in fp32
        _case("norm_delta_56x56x64_f32", "norm_delta", dtype="f32", N=128, H=56, W=56, C=64, groups=16, act="leakyRelu"),
        # gradients in bf16
        _case("norm_delta_bf16", "norm_delta", dtype="bf16", N=8, H=64, W=64, C=640, groups=32, act="silu"),
        # the CIFAR-10 ResNet-18's convolutions, all in fp32
        _case("adamw_resnet18_f32", "adamw", dtype="f32", grad="f32", out="", bits=32, model="resnet18", max_norm=0.0, step=100),
        # four transformer layers, 0.8 billion elements: fp32 weights with bf16 copies, bf16 gradients, clipped, moments in 8 bits
        _case("adamw_layers_8bit", "adamw", dtype="f32", grad="bf16", out="bf16", bits=8, model="layers", layers=4, D=4096, H=11008, max_norm=1.0, step=100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("loss", "loss", "loss_delta", "loss_delta", "norm", "norm", "norm_delta", "norm_delta", "adamw", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "adamw":
        param = rng.choice(("f32", "f32", dtype))
        return dict(kind=kind, dtype=param, grad=rng.choice((param, dtype)), out=rng.choice(("", dtype)) if param == "f32" else "", bits=rng.choice((8, 32)), model="ragged",
                    tensors=_log(rng, 1, 60), most=_log(rng, 1000, 4000000), sizes=rng.randrange(1 << 30), max_norm=rng.choice((0.0, 0.5, 2.0)), step=_log(rng, 1, 10000))
    if kind.startswith("norm"):
        while True:
            groups = rng.choice((1, 2, 4, 8, 16, 32, _log(rng, 1, 64)))
            C = groups * _log(rng, 1, 40)
            N, H = _log(rng, 1, 256), _log(rng, 1, 256)
            W = H if rng.random() < 0.5 else _log(rng, 1, 256)
            if 2 <= N * H * W * C <= 33000000 and H * W * (C // groups) >= 8:
                break
        return dict(kind=kind, dtype=dtype, N=N, H=H, W=W, C=C, groups=groups, act=rng.choice(("none", "silu", "leakyRelu", "gelu", "gelu_tanh", "sigmoid")),
                    **({} if "delta" in kind else {"save": rng.random() < 0.5}))
    while True:
        # half of the widths are multiples of 64, half are whatever the log scale gives
        IC = _log(rng, 20, 5000) if rng.random() < 0.5 else 64 * _log(rng, 1, 80)
        OC = _log(rng, 10, 130000) if rng.random() < 0.5 else 64 * _log(rng, 1, 2000)
        rows = _log(rng, 1, 4096)
        flops = 2.0 * rows * IC * OC * (3 if "delta" in kind else 1)
        if 1e5 <= flops <= (2.5e11 if dtype == "f32" else 4e12):
            break
    return dict(kind=kind, dtype=dtype, rows=rows, IC=IC, OC=OC, bias=rng.random() < 0.5, ignored=rng.choice((0.0, 0.1, 0.5)) if rows > 8 else 0.0)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _shapes(case):
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


def _views(flat, sizes, shapes=None):
    """The tensors that lie one after the other in a flat buffer, each from a multiple of 64 elements on."""
    at, out = 0, []
    for i, n in enumerate(sizes):
        t = flat[at:at + n]
        out.append(t if shapes is None else t.view(shapes[i]))
        at += (n + 63) // 64 * 64
    return out


def _flat(case, unit=1):
    """Elements of the flat buffer of all tensors, or of their blocks of `unit` elements."""
    return sum(((math.prod(s) + unit - 1) // unit + 63) // 64 * 64 for s in _shapes(case))


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0, t=None):
        return torch.randn(shape, device=dev, generator=g).mul_(scale).to(t or _TYPES[case["dtype"]])

    if case["kind"] == "adamw":
        n = _flat(case)
        x = dict(p=normal(n, scale=0.02), g=normal(n, scale=1e-3, t=_TYPES[case["grad"]]))
        if case["bits"] == 32:
            x["m"] = normal(n, scale=3e-4, t=torch.float32)
            x["v"] = normal(n, scale=1e-3, t=torch.float32).square_()
        else:
            s = _flat(case, _BLOCK)
            x["m"] = normal(n, scale=60.0, t=torch.float32).clamp_(-400.0, 400.0).to(torch.float8_e4m3fn)
            x["v"] = normal(n, scale=8.0, t=torch.float32).square_().clamp_(0.002, 440.0).to(torch.float8_e4m3fn)
            x["ms"] = torch.randint(127 - 18, 127 - 15, (s,), device=dev, generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
            x["vs"] = torch.randint(127 - 28, 127 - 25, (s,), device=dev, generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        return x
    if case["kind"].startswith("norm"):
        N, H, W, C = case["N"], case["H"], case["W"], case["C"]
        # channels of different means and scales, as a convolution with a bias leaves them
        X = torch.randn((N, H, W, C), device=dev, generator=g).mul_(torch.rand(C, device=dev, generator=g) + 0.5).add_(normal(C, t=torch.float32)).to(_TYPES[case["dtype"]])
        x = dict(X=X, gamma=normal(C, scale=0.2).add_(1.0), beta=normal(C, scale=0.2))
        if "delta" in case["kind"]:
            x["dY"] = normal(N, H, W, C)
        return x
    rows, IC, OC = case["rows"], case["IC"], case["OC"]
    # logits of a half-trained layer: 2.5 N(0, 1), those of the labels up to 15 above
    x = dict(W=normal(OC, IC, scale=2.5 / math.sqrt(IC)))
    label = torch.randint(0, OC, (rows,), device=dev, generator=g)
    towards = torch.rand((rows, 1), device=dev, generator=g).mul_(2.4) * x["W"][label].float()
    x["X"] = torch.randn((rows, IC), device=dev, generator=g).add_(towards).to(_TYPES[case["dtype"]])
    label[torch.rand(rows, device=dev, generator=g) < case["ignored"]] = -1
    x["label"] = label
    if case["bias"]:
        x["B"] = normal(OC, scale=0.1)
    if "delta" in case["kind"]:
        # of the mean over the rows that count
        x["dL"] = 1.0 / (label >= 0).sum().clamp(min=1).float()
    return x


def _saved(case, x):
    """What the forward pass leaves for the backward pass, from 64 bits."""
    if case["kind"] == "norm_delta":
        N, C, G = case["N"], case["C"], case["groups"]
        each = [t.double().reshape(-1, G, C // G) for t in x["X"]]
        x["mean"] = torch.stack([t.mean((0, 2)) for t in each])
        x["rstd"] = torch.stack([1.0 / torch.sqrt((t - m[:, None]).square().mean((0, 2)) + 1e-5) for t, m in zip(each, x["mean"])]).float()
        x["mean"] = x["mean"].float()
    elif case["kind"] == "loss_delta":
        W, b = x["W"].float(), x["B"].double() if case["bias"] else 0.0
        x["lse"] = torch.cat([torch.logsumexp((X.float() @ W.t()).double() + b, 1) for X in x["X"].split(512)]).float()


def prepare(case, seed):
    st = _inputs(case, seed)
    _saved(case, st)
    st["case"] = case
    if own:
        from __graft_entry__ import submodule
        st["eng"] = submodule("engine").Engine()
    if case["kind"] == "adamw":
        shapes = _shapes(case)
        sizes, blocks = [math.prod(s) for s in shapes], [-(-math.prod(s) // _BLOCK) for s in shapes]
        if case["out"]:
            st["out"] = torch.zeros(st["p"].shape, dtype=_TYPES[case["out"]], device=st["p"].device)
            st["outs"] = _views(st["out"], sizes, shapes)
        st["step"] = case["step"]
        st["lists"] = {k: _views(st[k], sizes, shapes) for k in ("p", "g", "m", "v")}
        if case["bits"] == 8:
            st["lists"].update({k: _views(st[k], blocks) for k in ("ms", "vs")})
        if own:
            engine = submodule("engine")
            st["state"] = engine.AdamWState(*(st["lists"].get(k) for k in ("m", "v", "ms", "vs")))
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


def _plain_norm(st):
    c = st["case"]
    t, N, C, G = st["X"].dtype, c["N"], c["C"], c["groups"]
    x = st["X"].float().reshape(N, -1, G, C // G)
    gamma, beta = (st[k].float().reshape(1, 1, G, C // G) for k in ("gamma", "beta"))
    if c["kind"] == "norm":
        mean = x.mean((1, 3), keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
        y = _act(d * rstd * gamma + beta, c["act"]).reshape(st["X"].shape).to(t)
        return [y, mean.reshape(N, G), rstd.reshape(N, G)] if c["save"] else y
    mean, rstd = (st[k].reshape(N, 1, G, 1) for k in ("mean", "rstd"))
    xh = (x - mean) * rstd
    dz = st["dY"].float().reshape(x.shape) * _act_slope(xh * gamma + beta, c["act"])
    dxh = dz * gamma
    dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return [dx.reshape(st["X"].shape).to(t), (dz * xh).sum((0, 1)).reshape(C).to(t), dz.sum((0, 1)).reshape(C).to(t)]


def _plain_loss(st):
    c, label = st["case"], st["label"]
    X, W, t = st["X"].float(), st["W"].float(), st["X"].dtype
    z = X @ W.t()
    if c["bias"]:
        z = z + st["B"].float()
    counts = label >= 0
    at = label.clamp(min=0)[:, None]
    if c["kind"] == "loss":
        most = z.max(1, keepdim=True).values
        lse = (most + torch.log(torch.exp(z - most).sum(1, keepdim=True)))[:, 0]
        return [torch.where(counts, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse)), lse]
    dz = torch.exp(z - st["lse"][:, None])
    dz.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    dz = dz * torch.where(counts, st["dL"], torch.zeros_like(st["dL"]))[:, None]
    out = [(dz @ W).to(t), (dz.t() @ X).to(t)]
    return out + [dz.sum(0).to(t)] if c["bias"] else out


def _mix(x):
    """32 scrambled bits of each 32-bit number, held in int64."""
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(n, tensor, step, device):
    """The random bits of each element of a tensor's moments."""
    key = torch.tensor([0x243F6A88 ^ (step & 0xFFFFFFFF)], dtype=torch.int64, device=device)      # (seed 0)
    key = _mix(_mix(key) ^ tensor)
    return _mix(torch.arange(n, dtype=torch.int64, device=device) ^ key)


def _decode(codes, scales):
    return codes.reshape(-1).float() * scales.float().repeat_interleave(_BLOCK)[: codes.numel()]


def _encode(x, dither, codes, scales, floor):
    """x as e4m3 codes with a power of two for each block: the smallest with which no element is above 448.  Rounded up or down by 16 random bits."""
    n = x.numel()
    pad = -n % _BLOCK
    most = torch.nn.functional.pad(x.abs(), (0, pad)).reshape(-1, _BLOCK).max(1).values
    bits = most.view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    scales.copy_(e.to(torch.uint8).view(torch.float8_e8m0fnu))
    back = ((254 - e) << 23).view(torch.float32).repeat_interleave(_BLOCK)[:n]
    y = x * back
    a = y.abs()
    small = a < 2.0 ** -6
    a = torch.where(small, a + 2.0 ** -6, a)             # steps of 2^-9 there
    a = ((a.view(torch.int32) + (dither << 4).int()) & ~0xFFFFF).view(torch.float32)
    a = torch.where(small, a - 2.0 ** -6, a)
    if floor:
        a = torch.where(y > 0, a.clamp(min=2.0 ** -9), a)
    codes.copy_(torch.copysign(a, y).to(torch.float8_e4m3fn).view(codes.shape))


def _plain_adamw(st):
    c, L = st["case"], st["lists"]
    st["step"] += 1
    step = st["step"]
    size = _LR / (1.0 - _BETA1 ** step)
    root = 1.0 / math.sqrt(1.0 - _BETA2 ** step)
    norm, scale = None, 1.0
    if c["max_norm"]:
        norm = torch.sqrt(sum(torch.sum(a.double() * a.double()) for a in L["g"])).float()
        scale = torch.clamp(c["max_norm"] / (norm.double() + 1e-6), max=1.0).float()
    for i, (p, g, m, v) in enumerate(zip(L["p"], L["g"], L["m"], L["v"])):
        g = (g.float() * scale).reshape(-1)
        old_m, old_v = (m.reshape(-1), v.reshape(-1)) if c["bits"] == 32 else (_decode(m, L["ms"][i]), _decode(v, L["vs"][i]))
        m1 = old_m * _BETA1 + g * (1.0 - _BETA1)
        v1 = old_v * _BETA2 + (g * g) * (1.0 - _BETA2)
        q = p.float().reshape(-1) * (1.0 - _LR * _DECAY) - m1 / (torch.sqrt(v1) * root + _EPS) * size
        p.copy_(q.view(p.shape))
        if c["out"]:
            st["outs"][i].copy_(q.view(p.shape))
        if c["bits"] == 32:
            m.copy_(m1.view(m.shape))
            v.copy_(v1.view(v.shape))
        else:
            r = _dither(m1.numel(), i, step, m1.device)
            _encode(m1, r & 0xFFFF, m, L["ms"][i], False)
            _encode(v1, r >> 16, v, L["vs"][i], True)
    return _adamw_outputs(st, norm)


def _adamw_outputs(st, norm):
    return {k: st[k] for k in ("p", "m", "v", "ms", "vs", "out") if k in st} | ({} if norm is None else {"norm": norm})


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        return _plain_adamw(state) if kind == "adamw" else _plain_norm(state) if kind.startswith("norm") else _plain_loss(state)
    eng = state["eng"]
    if kind == "norm":
        out = eng.groupNorm(state["X"], c["groups"], state["gamma"], state["beta"], act=c["act"], k=_SLOPE, save=c["save"])
        return list(out) if c["save"] else out
    if kind == "norm_delta":
        return list(eng.groupNorm_delta(state["dY"], state["X"], state["mean"], state["rstd"], state["gamma"], state["beta"], act=c["act"], k=_SLOPE))
    if kind == "loss":
        return list(eng.fullConnect_softmax_crossEntropy(state["X"], state["W"], state["label"], state.get("B"), save=True))
    if kind == "loss_delta":
        out = eng.fullConnect_softmax_crossEntropy_delta(state["dL"], state["X"], state["W"], state["label"], state["lse"], state.get("B"))
        return list(out) if c["bias"] else list(out[:2])
    state["step"] += 1
    norm = eng.adamW(state["lists"]["p"], state["lists"]["g"], state["state"], state["step"], _LR, beta1=_BETA1, beta2=_BETA2, eps=_EPS, weight_decay=_DECAY,
                     max_norm=c["max_norm"] or None, Out=state.get("outs"))
    return _adamw_outputs(state, norm)


# ---- what the operators cannot do without ------------------------------------------------------------------------

def _size(name):
    return torch.finfo(_TYPES[name]).bits // 8 if name else 0


def work(case):
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16.0 if case["bits"] == 32 else 4.0 + 4.0 / _BLOCK
        return {"bytes": n * (2.0 * _size(case["dtype"]) + _size(case["grad"]) + _size(case["out"]) + moments), "flops": 15.0 * n}
    if case["kind"].startswith("norm"):
        n, C, G = case["N"] * case["H"] * case["W"] * case["C"], case["C"], case["groups"]
        if "delta" in case["kind"]:
            return {"bytes": float(_size(case["dtype"]) * (3 * n + 4 * C) + 8 * case["N"] * G), "flops": 20.0 * n}
        return {"bytes": float(_size(case["dtype"]) * (2 * n + 2 * C) + (8 * case["N"] * G if case["save"] else 0)), "flops": 10.0 * n}
    rows, IC, OC, size = case["rows"], case["IC"], case["OC"], _size(case["dtype"])
    tensors = rows * IC + OC * IC + (OC if case["bias"] else 0)
    if "delta" in case["kind"]:
        return {"bytes": float(size * 2 * tensors + 12 * rows), "flops": 6.0 * rows * IC * OC}
    return {"bytes": float(size * tensors + 16 * rows), "flops": 2.0 * rows * IC * OC}


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


def _exact_norm(case, x):
    G, C, out, db, dg = case["groups"], case["C"], [], 0.0, 0.0
    gamma, beta = x["gamma"].double(), x["beta"].double()
    wide = lambda s: s.repeat_interleave(C // G)       # noqa: E731
    for i, X in enumerate(x["X"]):
        X = X.double().reshape(-1, C)
        if case["kind"] == "norm":
            groups = X.reshape(-1, G, C // G).transpose(0, 1).reshape(G, -1)
            mean, rstd = groups.mean(1), (groups.var(1, correction=0) + 1e-5) ** -0.5
            out.append((_f64((X - wide(mean)) * wide(rstd) * gamma + beta, case["act"])[0], mean, rstd))
            continue
        mean, rstd = x["mean"][i].double(), x["rstd"][i].double()
        xh = (X - wide(mean)) * wide(rstd)
        dz = x["dY"][i].double().reshape(-1, C) * _f64(xh * gamma + beta, case["act"])[1]
        dg, db = dg + (dz * xh).sum(0), db + dz.sum(0)
        count = X.shape[0] * (C // G)
        s1, s2 = (wide((t * gamma).sum(0).reshape(G, -1).sum(1) / count) for t in (dz, dz * xh))
        out.append((wide(rstd) * (dz * gamma - s1 - xh * s2),))
    parts = [torch.stack(t) for t in zip(*out)]
    parts[0] = parts[0].reshape(x["X"].shape)
    if case["kind"] == "norm_delta":
        return [parts[0], dg, db]
    return parts if case["save"] else parts[0]


def _exact_loss(case, x):
    W, B = x["W"].double(), x["B"].double() if case["bias"] else 0.0
    lse, loss, dX, dW, dB = [], [], [], 0.0, 0.0
    for X, label, saved in zip(x["X"].split(1024), x["label"].split(1024), x.get("lse", x["label"]).split(1024)):
        X = X.double()
        z = torch.addmm(B * torch.ones(W.shape[0], dtype=torch.float64, device=X.device), X, W.T)
        rows = (label >= 0).nonzero()[:, 0]
        if case["kind"] == "loss":
            s = torch.logsumexp(z, 1)
            each = torch.zeros_like(s)
            each[rows] = s[rows] - z[rows, label[rows]]
            lse.append(s)
            loss.append(each)
            continue
        z = (z - saved.double()[:, None]).exp_()
        z[rows, label[rows]] -= 1.0
        z *= ((label >= 0).double() * x["dL"].double())[:, None]
        dX.append(z @ W)
        dW, dB = dW + z.T @ X, dB + z.sum(0)
    if case["kind"] == "loss":
        return [torch.cat(loss), torch.cat(lse)]
    return [torch.cat(dX), dW] + ([dB] if case["bias"] else [])


def _exact_adamw(case, x):
    shapes = _shapes(case)
    sizes, blocks = [math.prod(s) for s in shapes], [-(-math.prod(s) // _BLOCK) for s in shapes]
    step, eight = case["step"] + 1, case["bits"] == 8
    lists = {k: _views(x[k], blocks if k in ("ms", "vs") else sizes) for k in x}
    squares = sum(float(t.double().square().sum()) for t in lists["g"])
    c = min(1.0, case["max_norm"] / (math.sqrt(squares) + 1e-6)) if case["max_norm"] else 1.0
    flat = {k: x[k].double() for k in (("p",) if eight else ("p", "m", "v"))}
    for i, (p, *rest) in enumerate(zip(*(_views(flat[k], sizes) for k in flat))):
        g = lists["g"][i].double() * c
        if eight:
            m, v = (lists[k][i].double() * lists[s][i].double().repeat_interleave(_BLOCK)[: g.numel()] for k, s in (("m", "ms"), ("v", "vs")))
        else:
            m, v = rest
        m.mul_(_BETA1).add_(g, alpha=1 - _BETA1)
        v.mul_(_BETA2).add_(g.square(), alpha=1 - _BETA2)
        p.mul_(1 - _LR * _DECAY).sub_(_LR * (m / (1 - _BETA1 ** step)) / ((v / (1 - _BETA2 ** step)).sqrt_() + _EPS))
    out = {"p": flat["p"], "m": flat.get("m"), "v": flat.get("v")}
    if eight:
        out.update(ms=None, vs=None)
    if case["out"]:
        out["out"] = torch.zeros_like(flat["p"])
        for o, p in zip(_views(out["out"], sizes), _views(flat["p"], sizes)):
            o.copy_(p)
    if case["max_norm"]:
        out["norm"] = torch.tensor(math.sqrt(squares), dtype=torch.float64)
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(case, x)
    _saved(case, x)
    return _exact_norm(case, x) if case["kind"].startswith("norm") else _exact_loss(case, x)
