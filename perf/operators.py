"""What the framework's operators of the text towers are measured on: ``lsdm_amd.ops.linear`` (matrix product with bias, activation and
residual), ``lsdm_amd.ops.layer_norm`` and the 8-bit activation checkpoints ``lsdm_amd.ops.checkpoint8``, forward and training.

``own`` selects what ``run`` does: the plain form (elementary torch operations in 32 bits, rounded once at the end) or the calls a user makes
of the operators.  ``exact`` is the definition in 64 bits.  A case is one dict: ``op`` ("linear", "layer_norm", "checkpoint8"), the sizes, the type,
and ``train`` (forward and gradients) / ``checkpoint8`` (what the backward pass reads is kept in 8 bits)."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def _linear(name, M, K, N, dtype, activation, bias=True, residual=False, train=False, checkpoint8=False):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "activation": activation, "bias": bias, "residual": residual,
            "train": train, "checkpoint8": checkpoint8}


def _norm(name, M, K, dtype, affine="same", train=False, checkpoint8=False):
    return {"name": name, "op": "layer_norm", "M": M, "K": K, "dtype": dtype, "affine": affine, "train": train, "checkpoint8": checkpoint8}


def _pack(name, M, K, dtype):
    return {"name": name, "op": "checkpoint8", "M": M, "K": K, "dtype": dtype}


def listed():
    return [
        # the first layer of the conditioning text MLP for a single prompt: one row, fp32, nothing but latency
        _linear("prompt_f32", 1, 512, 256, "f32", "gelu"),
        # the MLP of a 512-wide text tower over 64 prompts of 77 tokens in half precision: its widening product ...
        _linear("tower_up_f16", 4928, 512, 2048, "f16", "quick_gelu"),
        # ... and its narrowing one, which adds the residual stream
        _linear("tower_down_f16", 4928, 2048, 512, "f16", "none", residual=True),
        # a per-point layer of the denoiser's kind trained in fp32: a batch of 6 clouds of 1024 points
        _linear("points_train_f32", 6144, 256, 192, "f32", "sigmoid", train=True),
        # fine-tuning on packed prompts without their padding, sizes that no vector load divides
        _linear("ragged_train_bf16", 1357, 515, 771, "bf16", "relu", residual=True, train=True),
        # the widening product of a large tower in training: the largest work
        _linear("large_train_bf16", 16384, 2048, 8192, "bf16", "gelu", train=True),
        # the norm in front of one prompt's block in half precision with fp32 weights: latency again
        _norm("norm_prompt_f16", 77, 512, "f16", affine="f32"),
        # the norms of a large tower in training
        _norm("norm_train_bf16", 32768, 2048, "bf16", train=True),
        # rows of an odd width in fp32
        _norm("norm_odd_train_f32", 4928, 771, "f32", train=True),
        # a residual stream stored in 8 bits and read back
        _pack("pack_bf16", 32768, 2048, "bf16"),
        # a widening product whose input and derivative are kept in 8 bits for the backward pass
        _linear("linear_8bit_train_bf16", 8192, 1024, 4096, "bf16", "gelu", train=True, checkpoint8=True),
        # a norm that keeps its normalised rows in 8 bits
        _norm("norm_8bit_train_f16", 16384, 1024, "f16", train=True, checkpoint8=True),
    ]


def _log_int(rng, lo, hi, multiple):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:                     # half of the sizes are what configurations hold, half are anything
        v = max(multiple, v // multiple * multiple) if v >= multiple else v
    return max(lo, min(hi, v))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    op = rng.choice(["linear", "linear", "linear", "layer_norm", "layer_norm", "checkpoint8"])
    if op == "linear":
        train = rng.random() < 0.6
        # an fp32 product costs up to 16 times a 16-bit one: its sizes end earlier
        top = 3.0e10 if dtype == "f32" else 2.7e11
        while True:
            M, K, N = _log_int(rng, 1, 16384, 64), _log_int(rng, 16, 8192, 64), _log_int(rng, 16, 8192, 64)
            if M * K * N <= top:
                break
        act = rng.choice(["none", "relu", "gelu", "quick_gelu", "silu", "sigmoid", "tanh"])
        return {"op": op, "M": M, "K": K, "N": N, "dtype": dtype, "activation": act, "bias": rng.random() < 0.8, "residual": rng.random() < 0.5,
                "train": train, "checkpoint8": train and rng.random() < 0.35}
    while True:
        M, K = _log_int(rng, 1, 65536, 64), _log_int(rng, 16, 8192, 64)
        if M * K <= 32768 * 2048:
            break
    if op == "checkpoint8":
        return {"op": op, "M": M, "K": K, "dtype": dtype}
    train = rng.random() < 0.6
    return {"op": op, "M": M, "K": K, "dtype": dtype, "affine": rng.choice(["same", "f32", "none"]), "train": train,
            "checkpoint8": train and dtype != "f32" and rng.random() < 0.35}


def prepare(case, seed):
    dev, t = torch.device("cuda"), TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    M, K = case["M"], case["K"]
    s = dict(case)
    if case["op"] == "checkpoint8":
        # a residual stream: a few channels far above the others, some entries exactly zero
        x = rand(M, K) * torch.where(rand(K) > 2.0, 20.0, 1.0)
        s["x"] = torch.where(rand(M, K) > 1.5, 0.0, x).to(t)
        return s
    if case["op"] == "linear":
        N = case["N"]
        s["x"] = rand(M, K).to(t)
        s["w"] = (rand(N, K) / math.sqrt(K)).to(t)
        s["b"] = (0.1 * rand(N)).to(t) if case["bias"] else None
        s["r"] = rand(M, N).to(t) if case["residual"] else None
        out = (M, N)
    else:
        s["x"] = (rand(M, K) * (0.5 + rand(M, 1).abs()) + 0.3 * rand(M, 1)).to(t)
        wt = torch.float32 if case["affine"] == "f32" else t
        s["w"] = (1.0 + 0.1 * rand(K)).to(wt) if case["affine"] != "none" else None
        s["b"] = (0.1 * rand(K)).to(wt) if case["affine"] != "none" else None
        out = (M, K)
    if case["train"]:
        s["dy"] = (0.25 * rand(*out)).to(t)
        for k in ("x", "w", "b", "r"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _act(name, z):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "quick_gelu":
        return z / (1.0 + torch.exp(-1.702 * z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name in ("quick_gelu", "silu"):
        c = 1.702 if name == "quick_gelu" else 1.0
        s = 1.0 / (1.0 + torch.exp(-c * z))
        return s * (1.0 + c * z * (1.0 - s))
    if name == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 - s)
    if name == "tanh":
        s = torch.tanh(z)
        return 1.0 - s * s
    return torch.ones_like(z)


def _through_8_bits(x):
    """(rows, K) in 32 bits -> the values its 8-bit checkpoint stands for: groups of 32 along a row, a power-of-two step for each."""
    M, K = x.shape
    G = (K + 31) // 32
    g = torch.nn.functional.pad(x, (0, G * 32 - K)).view(M, G, 32)
    _, e = torch.frexp(g.abs().amax(dim=2, keepdim=True))
    e = (e - 7).clamp(min=-126)
    q = torch.round(torch.ldexp(g, -e)).clamp(-127, 127)
    return torch.ldexp(q, e).view(M, G * 32)[:, :K]


def _plain_linear(s):
    t = s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y = _act(s["activation"], z)
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    if not s["train"]:
        return y.to(t)
    d = _act_grad(s["activation"], z)
    if s["checkpoint8"]:
        x = _through_8_bits(x)
        if t != torch.float32:                 # in fp32 the derivative keeps its 32 bits
            d = torch.round(192.0 * d) / 192.0
    dz = s["dy"].float() * d
    out = [y.to(t), (dz @ w).to(t), (dz.t() @ x).to(t)]
    if s["b"] is not None:
        out.append(dz.sum(0).to(s["b"].dtype))
    if s["r"] is not None:
        out.append(s["dy"])
    return out


def _plain_norm(s):
    t = s["x"].dtype
    x = s["x"].detach().float()
    mu = x.mean(1, keepdim=True)
    c = x - mu
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    h = c * rstd
    w = s["w"].detach().float() if s["w"] is not None else None
    y = h * w + s["b"].detach().float() if w is not None else h
    if not s["train"]:
        return y.to(t)
    if s["checkpoint8"]:
        h = _through_8_bits(h)
    dy = s["dy"].float()
    g = dy * w if w is not None else dy
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    out = [y.to(t), dx.to(t)]
    if w is not None:
        out += [(dy * h).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)]
    return out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if not own:
        if s["op"] == "linear":
            return _plain_linear(s)
        if s["op"] == "layer_norm":
            return _plain_norm(s)
        return _through_8_bits(s["x"].float()).to(s["x"].dtype)
    from lsdm_amd import ops
    if s["op"] == "checkpoint8":
        return ops.checkpoint8(s["x"]).restore()
    # a forward pass alone is inference: its inputs ask for no gradients
    if s["op"] == "linear":
        y = ops.linear(s["x"], s["w"], s["b"], s["activation"], s["r"], checkpoint8=s["checkpoint8"])
    else:
        y = ops.layer_norm(s["x"], s["w"], s["b"], EPS, checkpoint8=s["checkpoint8"])
    if not s["train"]:
        return y
    leaves = [s[k] for k in ("x", "w", "b", "r") if s.get(k) is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    val = lambda k: s[k].detach().double() if s.get(k) is not None else None
    x, w, b = val("x"), val("w"), val("b")

    def stored(v):
        out = torch.empty_like(v)
        for lo in range(0, v.shape[1], 32):
            part = v[:, lo:lo + 32]
            top = part.abs().max(dim=1, keepdim=True)[0]
            # floor(log2 top), put right where the logarithm rounded across a power of two
            f = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
            f = torch.where(torch.exp2(f) > top, f - 1, f)
            f = torch.where(torch.exp2(f + 1) <= top, f + 1, f)
            step = torch.exp2(torch.clamp(f - 6, min=-126.0))
            out[:, lo:lo + 32] = torch.clamp(torch.round(part / step), -127, 127) * step
        return out

    if case["op"] == "checkpoint8":
        return stored(x)
    if case["op"] == "linear":
        z = torch.mm(x, w.T)
        z = z if b is None else z.add_(b)
        a = case["activation"]
        sig = lambda v: torch.special.expit(v)
        phi = lambda v: torch.special.ndtr(v)
        f = {"none": lambda v: v.clone(), "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * phi(v), "quick_gelu": lambda v: v * sig(1.702 * v),
             "silu": lambda v: v * sig(v), "sigmoid": sig, "tanh": torch.tanh}[a]
        y = f(z)
        if s["r"] is not None:
            y += val("r")
        if not case["train"]:
            return y
        df = {"none": lambda v: torch.ones_like(v), "relu": lambda v: (v > 0).double(),
              "gelu": lambda v: phi(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi),
              "quick_gelu": lambda v: sig(1.702 * v) * (1 + 1.702 * v * sig(-1.702 * v)), "silu": lambda v: sig(v) * (1 + v * sig(-v)),
              "sigmoid": lambda v: sig(v) * sig(-v), "tanh": lambda v: 1 / torch.cosh(v) ** 2}[a]
        d = df(z)
        if case["checkpoint8"]:
            x = stored(x)
            d = torch.round(d * 192) / 192 if case["dtype"] != "f32" else d
        dy = s["dy"].double()
        d *= dy
        out = [y, torch.mm(d, w), torch.mm(d.T, x)]
        if b is not None:
            out.append(d.sum(dim=0))
        if s["r"] is not None:
            out.append(dy)
        return out
    v, m = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(v + EPS)
    h = (x - m) / sd
    y = h if w is None else torch.addcmul(b, h, w)
    if not case["train"]:
        return y
    if case["checkpoint8"]:
        h = stored(h)
    dy = s["dy"].double()
    g = dy if w is None else dy * w
    K = x.shape[1]
    dx = (g - g.sum(dim=1, keepdim=True) / K - h * ((g * h).sum(dim=1, keepdim=True) / K)) / sd
    return [y, dx] if w is None else [y, dx, torch.sum(dy * h, dim=0), torch.sum(dy, dim=0)]


# ------------------------------------------------------------------------------------------------ what one pass cannot do without
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    M, K = case["M"], case["K"]
    if case["op"] == "checkpoint8":
        codes = M * K + M * ((K + 31) // 32)
        return {"bytes": 2 * M * K * size + 2 * codes, "flops": 4 * M * K}
    if case["op"] == "linear":
        N = case["N"]
        tensors = M * K + N * K + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)
        flops = 2 * M * N * K
        if case["train"]:
            tensors += M * N + M * K + N * K + (N if case["bias"] else 0)      # dy; dx, dw, db (the residual's gradient is dy itself)
            flops *= 3
        return {"bytes": tensors * size, "flops": flops}
    wsize = {"same": size, "f32": 4, "none": 0}[case["affine"]]
    if case["train"]:
        return {"bytes": 4 * M * K * size + 4 * K * wsize, "flops": 24 * M * K}
    return {"bytes": 2 * M * K * size + 2 * K * wsize, "flops": 8 * M * K}
