"""The dense-layer and group-norm operators of the learned mel inversion: cases, inputs, plain forms, definitions.

A learned inversion takes log-mel frames (batch, frames, n_mels) to linear magnitudes (batch, frames, n_fft / 2 + 1):
dense layers (a matrix product with bias, activation and residual) with group norms between them, channels last, both
with their gradients.  ``run`` computes one operator on the inputs of ``prepare``: in plain torch operations where
``own`` is false, through ``tacotron2_amd.inversion`` where it is true.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5

# 641 frames: one utterance at n_fft 1024, hop 275; 64 x 861 frames: the batch of 64 ten-second utterances at n_fft 2048,
# hop 256; 51 680 frames: one utterance of ten minutes.  80 bands, 513 / 1025 bins; 256, 512 and 1024 channels, hidden
# layers four times as wide.
_BATCH = 64 * 861


def _dense(name, rows, inputs, outputs, dtype, activation, bias=True, residual=False, out="same", preactivation=False):
    return {"name": name, "op": "dense", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual, "out": out, "preactivation": preactivation}


def _dense_back(name, rows, inputs, outputs, dtype, activation, out="same"):
    return {"name": name, "op": "dense_backward", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "activation": activation, "out": out}


def _norm(name, op, batch, frames, channels, groups, dtype, activation, ragged, stats=False):
    c = {"name": name, "op": op, "batch": batch, "frames": frames, "channels": channels, "groups": groups,
         "dtype": dtype, "activation": activation, "ragged": ragged}
    if op == "group_norm":
        c["stats"] = stats
    return c


def listed():
    return [
        # one frame as a decoder emits it, hidden channels to 1025 magnitudes: latency
        _dense("frame_out", 1, 512, 1025, "bf16", "exp", out="f32"),
        # one utterance's 80 log-mel bands into the hidden channels
        _dense("utterance_in", 641, 80, 512, "f32", "silu"),
        # the wide hidden layer over the batch of 64 utterances
        _dense("batch_expand", _BATCH, 512, 2048, "bf16", "gelu"),
        # the same batch's last layer: 1025 magnitudes in the 32 bits that the reconstruction loop reads
        _dense("batch_out", _BATCH, 512, 1025, "bf16", "exp", out="f32"),
        # a batch of 8 utterances in full precision, back onto the residual stream
        _dense("batch_project_f32", 8 * 861, 1024, 1024, "f32", "none", residual=True),
        # gradients of the input layer for one utterance
        _dense_back("utterance_in_back", 641, 80, 512, "f32", "silu"),
        # gradients of the wide hidden layer over the batch
        _dense_back("batch_expand_back", _BATCH, 512, 2048, "bf16", "gelu"),
        # the norm in front of a layer, one utterance
        _norm("utterance_norm", "group_norm", 1, 641, 512, 32, "bf16", "silu", False),
        # the same over the batch with every utterance's own length, statistics kept for the gradients
        _norm("batch_norm", "group_norm", 64, 861, 512, 32, "bf16", "silu", True, stats=True),
        # ten minutes in one piece in full precision: few, long groups
        _norm("long_norm", "group_norm", 1, 51680, 256, 8, "f32", "silu", False),
        # gradients over the ragged batch
        _norm("batch_norm_back", "group_norm_backward", 64, 861, 512, 32, "bf16", "silu", True),
        # gradients of one long piece in half precision
        _norm("long_norm_back", "group_norm_backward", 1, 51680, 256, 8, "f16", "silu", False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    activation = rng.choice(["none", "relu", "silu", "gelu", "tanh", "exp"])
    if rng.random() < 0.55:
        back = rng.random() < 0.4
        rows = _log_int(rng, 1, _BATCH)
        inputs, outputs = _log_int(rng, 16, 2048), _log_int(rng, 16, 2049)
        if rng.random() < 0.6:                                # most layers' widths are whole multiples of 64
            inputs, outputs = max(64, inputs // 64 * 64), max(64, outputs // 64 * 64)
        most = (8 * 861 * 1024 * 1024 if dtype == "f32" else _BATCH * 512 * 2048) // (2 if back else 1)
        rows = max(1, min(rows, most // (inputs * outputs)))
        out = "f32" if dtype != "f32" and rng.random() < 0.25 else "same"
        if back:
            return {k: v for k, v in _dense_back("", rows, inputs, outputs, dtype, activation, out).items() if k != "name"}
        c = _dense("", rows, inputs, outputs, dtype, activation, rng.random() < 0.8, rng.random() < 0.4, out,
                   rng.random() < 0.3)
        return {k: v for k, v in c.items() if k != "name"}
    op = rng.choice(["group_norm", "group_norm_backward"])
    groups = rng.choice([1, 2, 4, 8, 16, 32])
    channels = groups * _log_int(rng, 1, 1024 // groups)
    if rng.random() < 0.6:
        channels = max(groups, 32) * max(1, channels // max(groups, 32))
    batch = _log_int(rng, 1, 64)
    frames = max(1, min(_log_int(rng, 1, 51680), _BATCH * 512 // 2 // (batch * channels)))
    c = _norm("", op, batch, frames, channels, groups, dtype, activation, batch > 1 and frames > 3 and rng.random() < 0.5,
              rng.random() < 0.5)
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(case):
    """Lengths of a ragged batch, longest first: evenly spread from the full length down to a third of it."""
    B, T = case["batch"], case["frames"]
    if not case["ragged"]:
        return [T] * B
    return [T - (T - T // 3) * b // max(1, B - 1) for b in range(B)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, to=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(to)

    s = {"case": case}
    if case["op"].startswith("dense"):
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        wide = torch.float32 if case["out"] == "f32" else dtype
        s["x"] = normal(M, K)
        s["weight"] = normal(N, K, scale=K ** -0.5)
        s["bias"] = normal(N, scale=0.1) if case.get("bias", True) else None
        if case["op"] == "dense":
            s["residual"] = normal(M, N, to=wide) if case["residual"] else None
        else:
            z = s["x"].float() @ s["weight"].float().t() + s["bias"].float()
            s["preactivation"] = z.to(wide) if case["activation"] != "none" else None
            s["dy"] = normal(M, N, scale=0.1, to=wide)
        return s
    B, T, C, G = case["batch"], case["frames"], case["channels"], case["groups"]
    level = torch.randn((1, 1, C), generator=g, device="cuda")   # channels differ in their mean, as activations do
    s["x"] = (torch.randn((B, T, C), generator=g, device="cuda") + level).to(dtype)
    s["gamma"] = normal(C, scale=0.2, mean=1.0)
    s["beta"] = normal(C, scale=0.2)
    s["lengths"] = None
    if case["ragged"]:
        order = torch.randperm(B, generator=g, device="cuda")
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order].contiguous()
    if case["op"] == "group_norm_backward":
        s["dy"] = normal(B, T, C, scale=0.1)
        s["stats"] = _plain_stats(s["x"].double(), s["lengths"], G)[2].float()
    return s


# -- plain forms -----------------------------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * (0.5 ** 0.5)))
    if name == "tanh":
        return torch.tanh(z)
    if name == "exp":
        return torch.exp(z)
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * (0.5 ** 0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    if name == "exp":
        return torch.exp(z)
    return torch.ones_like(z)


def _valid(x, lengths):
    """(B, T, 1) true where a frame lies inside its utterance."""
    B, T = x.shape[:2]
    if lengths is None:
        return torch.ones((B, T, 1), dtype=torch.bool, device=x.device)
    return (torch.arange(T, device=x.device)[None, :] < lengths[:, None])[:, :, None]


def _plain_stats(x, lengths, groups):
    """(normalised x, frame mask, (B, groups, 2) mean and 1 / standard deviation) of x (B, T, C) in x's type."""
    B, T, C = x.shape
    valid = _valid(x, lengths)
    count = valid.sum(1).to(x.dtype)[:, :, None] * (C // groups)                 # (B, 1, 1)
    xg = torch.where(valid, x, 0).reshape(B, T, groups, C // groups)
    mean = xg.sum((1, 3))[:, :, None] / count                                    # (B, G, 1)
    d = torch.where(valid[:, :, :, None], xg - mean[:, None], 0)
    rstd = torch.rsqrt((d * d).sum((1, 3))[:, :, None] / count + _EPS)
    return (d * rstd[:, None]).reshape(B, T, C), valid, torch.cat([mean, rstd], 2)


def _plain(s):
    c = s["case"]
    dtype = _TYPES[c["dtype"]]
    name = c["activation"]
    if c["op"] == "dense":
        wide = torch.float32 if c["out"] == "f32" else dtype
        z = s["x"].float() @ s["weight"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, name)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(wide), z.to(wide)) if c["preactivation"] else y.to(wide)
    if c["op"] == "dense_backward":
        dz = s["dy"].float()
        if name != "none":
            dz = dz * _act_grad(s["preactivation"].float(), name)
        return {"dx": (dz @ s["weight"].float()).to(dtype), "dweight": (dz.t() @ s["x"].float()).to(dtype),
                "dbias": dz.sum(0).to(dtype)}
    G = c["groups"]
    gamma, beta = s["gamma"].float(), s["beta"].float()
    if c["op"] == "group_norm":
        xh, valid, stats = _plain_stats(s["x"].float(), s["lengths"], G)
        y = torch.where(valid, _act(xh * gamma + beta, name), 0).to(dtype)
        return (y, stats) if c["stats"] else y
    x = s["x"].float()
    B, T, C = x.shape
    valid = _valid(x, s["lengths"])
    mean, rstd = s["stats"][:, None, :, :1], s["stats"][:, None, :, 1:]           # (B, 1, G, 1)
    xh = torch.where(valid, ((x.reshape(B, T, G, C // G) - mean) * rstd).reshape(B, T, C), 0)
    du = torch.where(valid, s["dy"].float() * _act_grad(xh * gamma + beta, name), 0)
    dgamma, dbeta = (du * xh).sum((0, 1)), du.sum((0, 1))
    count = valid.sum(1).float()[:, :, None, None] * (C // G)
    v, xg = (du * gamma).reshape(B, T, G, C // G), xh.reshape(B, T, G, C // G)
    p = v.sum((1, 3), keepdim=True) / count
    q = (v * xg).sum((1, 3), keepdim=True) / count
    dx = torch.where(valid, (rstd * (v - p - xg * q)).reshape(B, T, C), 0)
    return {"dx": dx.to(dtype), "dgamma": dgamma.to(dtype), "dbeta": dbeta.to(dtype)}


# -- the framework's operators ---------------------------------------------------------------------------------
def _framework(s):
    from tacotron2_amd import inversion
    c = s["case"]
    dtype = _TYPES[c["dtype"]]
    name = None if c["activation"] == "none" else c["activation"]
    if c["op"] == "dense":
        wide = torch.float32 if c["out"] == "f32" else dtype
        z = None
        if c["preactivation"]:
            z = torch.empty((c["rows"], c["outputs"]), dtype=wide, device=s["x"].device)
        y = inversion.dense(s["x"], s["weight"], s["bias"], activation=name, residual=s["residual"], out_dtype=wide,
                            preactivation=z)
        return (y, z) if c["preactivation"] else y
    if c["op"] == "dense_backward":
        dx, dw, db = inversion.dense_backward(s["dy"], s["x"], s["weight"], s["preactivation"], activation=name)
        return {"dx": dx, "dweight": dw, "dbias": db}
    if c["op"] == "group_norm":
        stats = None
        if c["stats"]:
            stats = torch.empty((c["batch"], c["groups"], 2), dtype=torch.float32, device=s["x"].device)
        y = inversion.group_norm(s["x"], c["groups"], s["gamma"], s["beta"], eps=_EPS, activation=name,
                                 lengths=s["lengths"], stats=stats)
        return (y, stats) if c["stats"] else y
    dx, dgamma, dbeta = inversion.group_norm_backward(s["dy"], s["x"], c["groups"], s["stats"], s["gamma"], s["beta"],
                                                      activation=name, lengths=s["lengths"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("dense"):
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        wide = 4 if case["out"] == "f32" else size
        if case["op"] == "dense":
            extra = N * size * case["bias"] + M * N * wide * (case["residual"] + case["preactivation"])
            return {"bytes": (M * K + N * K) * size + M * N * wide + extra, "flops": 2 * M * K * N}
        inputs = (M * K + N * K) * size + M * N * wide * (1 + (case["activation"] != "none"))
        return {"bytes": inputs + (M * K + N * K + N) * size, "flops": 4 * M * K * N}
    B, T, C, G = case["batch"], case["frames"], case["channels"], case["groups"]
    live = sum(_lengths(case)) * C
    if case["op"] == "group_norm":
        return {"bytes": (live + B * T * C + 2 * C) * size + 8 * B * G * case["stats"], "flops": 10 * live}
    return {"bytes": (2 * live + B * T * C + 4 * C) * size + 8 * B * G, "flops": 20 * live}


# -- the definitions in 64 bits --------------------------------------------------------------------------------
def _phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _curve(z, name):
    """(activation, its derivative) at z."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).double()
        return z * on, on
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == "gelu":
        return z * _phi(z), _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "tanh":
        return torch.tanh(z), torch.cosh(z) ** -2
    e = torch.exp(z)
    return e, e


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    name = case["activation"]
    if case["op"] == "dense":
        z = torch.mm(d["x"], d["weight"].t().contiguous())
        if d["bias"] is not None:
            z += d["bias"][None, :]
        y = _curve(z, name)[0]
        if d["residual"] is not None:
            y = y + d["residual"]
        return (y, z) if case["preactivation"] else y
    if case["op"] == "dense_backward":
        dz = d["dy"] if name == "none" else _curve(d["preactivation"], name)[1] * d["dy"]
        return {"dx": torch.mm(dz, d["weight"]), "dweight": torch.mm(dz.t().contiguous(), d["x"]),
                "dbias": torch.mv(dz.t(), torch.ones(dz.shape[0], dtype=dz.dtype, device=dz.device))}
    B, T, C, G = case["batch"], case["frames"], case["channels"], case["groups"]
    n = C // G
    ends = [T] * B if d["lengths"] is None else d["lengths"].tolist()
    first, stats = torch.zeros_like(d["x"]), torch.zeros((B, G, 2), dtype=torch.float64, device=d["x"].device)
    dgamma, dbeta = torch.zeros_like(d["gamma"]), torch.zeros_like(d["beta"])
    for b, end in enumerate(ends):
        rows = d["x"][b, :end].reshape(end, G, n).transpose(0, 1).reshape(G, end * n)
        if case["op"] == "group_norm":
            var, mean = torch.var_mean(rows, 1, unbiased=False)
            stats[b, :, 0], stats[b, :, 1] = mean, 1 / torch.sqrt(var + _EPS)
        else:
            stats[b] = d["stats"][b]
        h = (rows - stats[b, :, :1]) * stats[b, :, 1:]
        h = h.reshape(G, end, n).transpose(0, 1).reshape(end, C)
        y, slope = _curve(h * d["gamma"] + d["beta"], name)
        if case["op"] == "group_norm":
            first[b, :end] = y
            continue
        du = d["dy"][b, :end] * slope
        dgamma += (du * h).sum(0)
        dbeta += du.sum(0)
        v = (du * d["gamma"]).reshape(end, G, n)
        hg = h.reshape(end, G, n)
        inner = v - v.mean((0, 2), keepdim=True) - hg * (v * hg).mean((0, 2), keepdim=True)
        first[b, :end] = (inner * stats[b, :, 1][None, :, None]).reshape(end, C)
    if case["op"] == "group_norm":
        return (first, stats) if case["stats"] else first
    return {"dx": first, "dgamma": dgamma, "dbeta": dbeta}
