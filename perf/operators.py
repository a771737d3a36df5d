"""Workloads of the dense operators around the sampling op, in plain torch and through ``opus_amd.opus_dense``.

Three operators, each forward and (``train``) backward:

  linear          z = x W^T + b;  y = residual + D(act(z))
  residual_norm   r = scale * x + gate * D(post(block));  y = norm(r)      -> y, r
  dropout         y = residual + D(x)

``D`` is dropout from a counter-based generator, Philox 4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel
random numbers: as easy as 1, 2, 3", 2011).  For element (row, col) of a tensor seen as [rows, last
dimension] the counter is (col // 8, row mod 2^32, row div 2^32, offset), the key is the 64-bit seed, and the
element's 16 random bits are bits 16 * (col % 2) .. of word (col % 8) // 2.  With ``drop`` = p and
k = round(65536 p), an element is kept iff its bits are >= k and is then scaled by 65536 / (65536 - k).

``run`` computes the plain forms unless ``own`` is true.  Both read and return the same tensors.
"""
import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5


def _linear(dtype, rows, k, n, act="none", bias=True, residual=False, drop=0.0, train=False, **name):
    return dict(name, op="linear", dtype=dtype, rows=rows, k=k, n=n, act=act, bias=bias, residual=residual,
                drop=drop, train=train)


def _norm(dtype, batch, tokens, width, kind="layer", post=False, gate="none", scale=1.0, drop=0.0, train=False,
          **name):
    return dict(name, op="residual_norm", dtype=dtype, batch=batch, tokens=tokens, width=width, kind=kind, post=post,
                gate=gate, scale=scale, drop=drop, train=train)


def _dropout(dtype, rows, cols, drop, residual=False, train=False, **name):
    return dict(name, op="dropout", dtype=dtype, rows=rows, cols=cols, drop=drop, residual=residual, train=train)


def listed():
    return [
        # one token through a feed-forward layer's first product: bound by latency and the weights' bytes
        _linear("bf16", 1, 1024, 4096, act="gelu_tanh", name="linear-token"),
        # the sampling offsets of 600 queries (G * P * 3 = 48 outputs): a small product of an inference frame
        _linear("fp32", 600, 256, 48, name="linear-offsets"),
        # what leaves the mixing of 4800 queries (G * 32 * 64 inputs) back into the query stream, a training step
        _linear("fp32", 4800, 8192, 256, residual=True, drop=0.1, train=True, name="linear-mix-out"),
        # the mixing parameters of 4800 queries, G * (64 * 64 + 32 * 16) outputs, a training step in bf16
        _linear("bf16", 4800, 256, 18432, train=True, name="linear-mix-params"),
        # a wide feed-forward product over a long prompt
        _linear("bf16", 8192, 4096, 4096, act="silu", residual=True, name="linear-prompt"),
        # nothing a multiple of anything: rows that start at odd addresses, every part of the epilogue, both directions
        _linear("fp16", 1237, 333, 777, act="gelu", residual=True, drop=0.1, train=True, name="linear-odd"),
        # one token between two blocks of a sandwich-norm decoder
        _norm("bf16", 1, 1, 4096, kind="rms", post=True, gate="channel", name="norm-token"),
        # the norm after a block of the query decoder: 8 samples of 4800 queries, dropout on the block, a training step
        _norm("fp32", 8, 4800, 256, drop=0.1, train=True, name="norm-queries"),
        # a wide sandwich norm with one gate per sample, a training step
        _norm("bf16", 4, 2048, 8192, kind="rms", post=True, gate="sample", scale=0.5, train=True, name="norm-wide"),
        # odd widths, a gate per token, every part of the operator in both directions
        _norm("fp16", 3, 601, 1003, post=True, gate="token", drop=0.25, train=True, name="norm-odd"),
        # a block's output dropped and added to the query stream, with its gradient
        _dropout("fp32", 38400, 256, 0.1, residual=True, train=True, name="dropout-queries"),
        # activations of a long batch, both directions
        _dropout("bf16", 65536, 2048, 0.5, train=True, name="dropout-long"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.6
    op = rng.choice(["linear", "linear", "residual_norm", "dropout"])
    if op == "linear":
        passes = 3 if train else 1
        while True:
            rows, k, n = _log(rng, 1, 8192), _log(rng, 24, 8192), _log(rng, 24, 18432)
            if rng.random() < 0.5:
                k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
            if rows * k * n * passes <= 2 ** 36:
                break
        # relu's gradient hangs on the sign of z, which 32 bits do not settle where z is within about 2^-26 sqrt(k) of
        # zero: in a training step it is drawn where hardly any of the rows * n values is
        smooth = train and rows * n * k ** 0.5 > 2 ** 22
        return _linear(dtype, rows, k, n, act=rng.choice(["none", "silu" if smooth else "relu", "gelu", "gelu_tanh", "silu"]),
                       bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                       drop=rng.choice([0.0, 0.0, 0.1, 0.3]), train=train)
    if op == "residual_norm":
        while True:
            batch, tokens, width = _log(rng, 1, 16), _log(rng, 1, 8192), _log(rng, 24, 8192)
            if rng.random() < 0.5:
                width = (width + 7) // 8 * 8
            if batch * tokens * width <= 2 ** 26:
                break
        return _norm(dtype, batch, tokens, width, kind=rng.choice(["layer", "rms"]), post=rng.random() < 0.5,
                     gate=rng.choice(["none", "channel", "sample", "token"]), scale=rng.choice([1.0, 0.5, 1.25]),
                     drop=rng.choice([0.0, 0.1, 0.25]), train=train)
    while True:
        rows, cols = _log(rng, 1, 65536), _log(rng, 1, 8192)
        if rows * cols <= 2 ** 27:
            break
    return _dropout(dtype, rows, cols, rng.choice([0.05, 0.1, 0.5]), residual=rng.random() < 0.5, train=train)


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=gen, device=device).mul_(std).add_(mean).to(dtype)

    s = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 63, "offset": seed % 1000}
    op = case["op"]
    if op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = normal(rows, k)
        s["weight"] = normal(n, k, std=k ** -0.5)
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(rows, n) if case["residual"] else None
        leaves, out = ["x", "weight", "bias", "residual"], (rows, n)
    elif op == "residual_norm":
        batch, tokens, width = case["batch"], case["tokens"], case["width"]
        s["x"] = normal(batch, tokens, width)
        s["block"] = normal(batch, tokens, width, mean=0.1, std=1.5)
        s["weight"] = normal(width, mean=1.0, std=0.1)
        s["bias"] = normal(width, std=0.1) if case["kind"] == "layer" else None
        s["post_weight"] = normal(width, mean=1.0, std=0.1) if case["post"] else None
        s["post_bias"] = normal(width, std=0.1) if case["post"] and case["kind"] == "layer" else None
        shape = {"none": None, "channel": (width,), "sample": (batch, width), "token": (batch, tokens, width)}
        shape = shape[case["gate"]]
        s["gate"] = normal(*shape, mean=0.5, std=0.3) if shape else None
        leaves = ["x", "block", "weight", "bias", "post_weight", "post_bias", "gate"]
        out = (batch, tokens, width)
    else:
        s["x"] = normal(case["rows"], case["cols"])
        s["residual"] = normal(case["rows"], case["cols"]) if case["residual"] else None
        leaves, out = ["x", "residual"], (case["rows"], case["cols"])
    if case["train"]:
        s["grad"] = normal(*out)
        if op == "residual_norm":
            s["grad_stream"] = normal(*out)
        s["leaves"] = [name for name in leaves if s[name] is not None]
        for name in s["leaves"]:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _kept(case, s, rows, cols):
    """1 / (1 - p) where an element is kept, 0 where it is dropped: fp32 [rows, cols] (None without dropout)."""
    k = int(round(case["drop"] * 65536))
    if k == 0:
        return None
    device = s["x"].device
    blocks = (cols + 7) // 8
    mask = 0xFFFFFFFF
    row = torch.arange(rows, device=device)[:, None]
    c0 = torch.arange(blocks, device=device)[None, :].expand(rows, blocks)
    c1, c2 = (row & mask).expand(rows, blocks), (row >> 32).expand(rows, blocks)
    c3 = torch.full_like(c0, s["offset"])
    k0, k1 = s["seed"] & mask, s["seed"] >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57                # (the low 64 bits, as a signed number)
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([c0, c1, c2, c3], -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, blocks * 8)[:, :cols]
    return (bits >= k).float() * (65536.0 / (65536 - k))


def _act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).float()
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    t = torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s, case):
    x, w = s["x"].float(), s["weight"].float()
    z = torch.matmul(x, w.t())
    if case["bias"]:
        z = z + s["bias"].float()
    kept = _kept(case, s, case["rows"], case["n"])
    y = _act(z, case["act"])
    if kept is not None:
        y = y * kept
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y}
    if case["train"]:
        g = s["grad"].float()
        dz = g if kept is None else g * kept
        if case["act"] != "none":
            dz = dz * _act_slope(z, case["act"])
        out["dx"] = torch.matmul(dz, w)
        out["dweight"] = torch.matmul(dz.t(), x)
        if case["bias"]:
            out["dbias"] = dz.sum(0)
        if case["residual"]:
            out["dresidual"] = g
    return out


def _stats(r, kind):
    mean = r.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(r[..., :1])
    c = r - mean
    rstd = (c.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    return c * rstd, rstd


def _stats_back(g, xhat, rstd, kind):
    m = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (g - m - xhat * (g * xhat).mean(-1, keepdim=True))


def _plain_norm(s, case):
    kind = case["kind"]
    get = lambda name: None if s[name] is None else s[name].float()          # noqa: E731
    x, h, w, b, pw, pb = (get(name) for name in ("x", "block", "weight", "bias", "post_weight", "post_bias"))
    gate = get("gate")
    if case["gate"] == "sample":
        gate = gate[:, None, :]
    batch, tokens, width = x.shape
    u = h
    if pw is not None:
        hhat, hrstd = _stats(h, kind)
        u = hhat * pw if pb is None else hhat * pw + pb
    kept = _kept(case, s, batch * tokens, width)
    if kept is not None:
        kept = kept.view(batch, tokens, width)
        u = u * kept
    r = x * case["scale"] + (u if gate is None else u * gate)
    xhat, rstd = _stats(r, kind)
    y = xhat * w if b is None else xhat * w + b
    out = {"y": y, "stream": r}
    if case["train"]:
        g = s["grad"].float()
        dr = s["grad_stream"].float() + _stats_back(g * w, xhat, rstd, kind)
        out["dx"] = dr * case["scale"]
        du = dr if gate is None else dr * gate
        if kept is not None:
            du = du * kept
        out["dblock"] = du if pw is None else _stats_back(du * pw, hhat, hrstd, kind)
        out["dweight"] = (g * xhat).sum((0, 1))
        if b is not None:
            out["dbias"] = g.sum((0, 1))
        if pw is not None:
            out["dpost_weight"] = (du * hhat).sum((0, 1))
            if pb is not None:
                out["dpost_bias"] = du.sum((0, 1))
        if gate is not None:
            dgate = dr * u
            axes = {"channel": (0, 1), "sample": (1,), "token": None}[case["gate"]]
            out["dgate"] = dgate if axes is None else dgate.sum(axes)
    return out


def _plain_dropout(s, case):
    kept = _kept(case, s, case["rows"], case["cols"])
    y = s["x"].float() * kept
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y}
    if case["train"]:
        g = s["grad"].float()
        out["dx"] = g * kept
        if case["residual"]:
            out["dresidual"] = g
    return out


# ------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------
def _own(s, case):
    from opus_amd import opus_dense
    op = case["op"]
    random = {"dropout_p": case["drop"], "seed": s["seed"], "offset": s["offset"]} if case["drop"] else {}
    if op == "linear":
        outs = [opus_dense.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"],
                                  **random)]
        names = ["y"]
    elif op == "residual_norm":
        outs = opus_dense.residual_norm(s["x"], s["block"], s["weight"], s["bias"], kind=case["kind"], eps=_EPS,
                                        post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                                        residual_scale=case["scale"], return_stream=True, **random)
        names = ["y", "stream"]
    else:
        outs = [opus_dense.dropout(s["x"], case["drop"], s["seed"], offset=s["offset"], residual=s["residual"])]
        names = ["y"]
    out = dict(zip(names, outs))
    if case["train"]:
        grads = [s["grad"], s["grad_stream"]] if op == "residual_norm" else [s["grad"]]
        found = torch.autograd.grad(list(outs), [s[name] for name in s["leaves"]], grads)
        out.update(("d" + name, g) for name, g in zip(s["leaves"], found))
    return out


def run(state):
    case = state["case"]
    if own:
        return {name: t.detach() for name, t in _own(state, case).items()}
    plain = {"linear": _plain_linear, "residual_norm": _plain_norm, "dropout": _plain_dropout}[case["op"]]
    dtype = _TYPES[case["dtype"]]
    with torch.no_grad():
        return _ordered({name: t.to(dtype) for name, t in plain(state, case).items()}, state)


def _ordered(out, state):
    """The outputs in the order in which the framework's call returns them."""
    names = ["y"] + (["stream"] if "stream" in out else [])
    names += ["d" + name for name in state.get("leaves", [])]
    return {name: out[name] for name in names}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    size, train = _SIZES[case["dtype"]], case["train"]
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        vector = n if case["bias"] else 0
        elements = rows * k + n * k + vector + rows * n * (2 if case["residual"] else 1)
        if train:
            elements += rows * n + rows * k + n * k + vector
        return {"bytes": elements * size, "flops": 2 * rows * k * n * (3 if train else 1)}
    if case["op"] == "residual_norm":
        total, width = case["batch"] * case["tokens"] * case["width"], case["width"]
        gate = {"none": 0, "channel": width, "sample": case["batch"] * width, "token": total}[case["gate"]]
        params = width * ((2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1)) + gate
        elements = 4 * total + params
        if train:
            elements += 4 * total + params
        return {"bytes": elements * size, "flops": total * (40 if train else 12)}
    total = case["rows"] * case["cols"]
    elements = (3 if case["residual"] else 2) * total + (2 * total if train else 0)
    return {"bytes": elements * size, "flops": total * (4 if train else 2)}


def _kept64(case, s, rows, cols):
    """The generator on the host in unsigned 64-bit words."""
    k = int(round(case["drop"] * 65536))
    if k == 0:
        return 1.0
    device = s["x"].device
    out = torch.empty((rows, cols), dtype=torch.float64, device=device)
    blocks = -(-cols // 8)
    step = max(1, (1 << 21) // blocks)
    low, m0, m1, by32 = np.uint64(0xFFFFFFFF), np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(32)
    for first in range(0, rows, step):
        n = min(step, rows - first)
        row = np.arange(first, first + n, dtype=np.uint64)[:, None]
        ctr = [np.broadcast_to(v, (n, blocks)) for v in
               (np.arange(blocks, dtype=np.uint64)[None, :], row & low, row >> by32, np.uint64(s["offset"]))]
        key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
        for r in range(10):
            a, b = m0 * ctr[0], m1 * ctr[2]
            kr = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
            ctr = [(b >> by32) ^ ctr[1] ^ kr[0], b & low, (a >> by32) ^ ctr[3] ^ kr[1], a & low]
        bits = np.empty((n, blocks, 8), dtype=np.uint16)
        for j in range(4):
            bits[..., 2 * j] = (ctr[j] & np.uint64(0xFFFF)).astype(np.uint16)
            bits[..., 2 * j + 1] = (ctr[j] >> np.uint64(16)).astype(np.uint16)
        kept = torch.from_numpy((bits.reshape(n, blocks * 8)[:, :cols] >= k).astype(np.uint8))
        out[first:first + n] = kept.to(device).double() * (65536 / (65536 - k))
    return out


def _act64(z, name):
    """(value, derivative) of the activation."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).double()
        return z * on, on
    if name == "silu":
        e = torch.sigmoid(z)
        return z * e, e + z * e * (1 - e)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * z * (1 + 0.044715 * z * z))
    return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * c * (1 + 0.134145 * z * z)


def _norm64(r, kind, gain, shift):
    """(output, function from the output's gradient to (input's, gain's, shift's) gradients)."""
    centred = r - r.mean(-1, keepdim=True) if kind == "layer" else r
    sigma = torch.sqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    unit = centred / sigma
    y = unit * gain + (0.0 if shift is None else shift)

    def back(g):
        t = g * gain / sigma
        d = t - unit * (t * unit).mean(-1, keepdim=True)
        if kind == "layer":
            d = d - t.mean(-1, keepdim=True)
        return d, (g * unit).flatten(0, -2).sum(0), g.flatten(0, -2).sum(0)
    return y, back


def exact(case, seed):
    with torch.no_grad():
        return _exact(case, seed)


def _exact(case, seed):
    s = prepare(case, seed)
    v = {name: t.detach().double() for name, t in s.items() if isinstance(t, torch.Tensor)}
    out = {}
    if case["op"] == "linear":
        z = v["x"] @ v["weight"].T
        if case["bias"]:
            z += v["bias"]
        kept = _kept64(case, s, case["rows"], case["n"])
        value, slope = _act64(z, case["act"])
        out["y"] = value * kept + (v["residual"] if case["residual"] else 0.0)
        if case["train"]:
            dz = v["grad"] * kept * slope
            out.update(dx=dz @ v["weight"], dweight=dz.T @ v["x"], dbias=dz.sum(0), dresidual=v["grad"])
    elif case["op"] == "residual_norm":
        shape = v["x"].shape
        kept = _kept64(case, s, shape[0] * shape[1], shape[2])
        if case["drop"]:
            kept = kept.view(shape)
        h, post_back = v["block"], None
        if case["post"]:
            h, post_back = _norm64(h, case["kind"], v["post_weight"], v.get("post_bias"))
        gate = v.get("gate", 1.0)
        if case["gate"] == "sample":
            gate = gate.unsqueeze(1)
        out["stream"] = case["scale"] * v["x"] + gate * kept * h
        out["y"], back = _norm64(out["stream"], case["kind"], v["weight"], v.get("bias"))
        if case["train"]:
            dr, out["dweight"], out["dbias"] = back(v["grad"])
            dr = dr + v["grad_stream"]
            out["dx"] = case["scale"] * dr
            full = dr * kept * h
            out["dgate"] = {"none": lambda: None, "channel": lambda: full.sum((0, 1)), "sample": lambda: full.sum(1),
                            "token": lambda: full}[case["gate"]]()
            out["dblock"] = dr * kept * gate
            if post_back is not None:
                out["dblock"], out["dpost_weight"], out["dpost_bias"] = post_back(out["dblock"])
    else:
        kept = _kept64(case, s, case["rows"], case["cols"])
        out["y"] = v["x"] * kept + (v["residual"] if case["residual"] else 0.0)
        if case["train"]:
            out.update(dx=v["grad"] * kept, dresidual=v["grad"])
    return _ordered(out, s)
