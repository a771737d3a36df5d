"""The dense operators on the GPU against oracle/dense_oracle.py (numpy, 64 bits).

Tolerances are bounds, element by element, from the arithmetic: U[t] = eps / 2 of the output's type for its one
rounding (plus half the smallest subnormal), and 2^-23 a step of an fp32 sum (a rounding of 2^-24, and as much again
for what a matrix instruction may drop inside) times the sum of the terms' magnitudes."""
import functools
import math
import types

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from oracle import dense_oracle as do

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
STEP = 2.0 ** -23
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def od():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from opus_amd import opus_dense
    return opus_dense


def make(rng, dtype, *shape, mean=0.0, std=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * std + mean).to(dtype).cuda()


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def check(got, want, bound, what):
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.isfinite(got).all(), f"{what}: non-finite values"
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), f"{what}: off by {np.abs(got - want).flat[over.argmax()]:.3e} where {bound.flat[over.argmax()]:.3e} is allowed"


def rounded(want, dtype):
    """what rounding `want` once to dtype may cost"""
    return U[dtype] * np.abs(want) + TINY[dtype]


# ------------------------------------------------------------------------------------------------
# linear
# ------------------------------------------------------------------------------------------------
def linear_bounds(x, w, b, r, dy, name, kept, dtype):
    """(y, z, bounds of y, dx, dw, db): ez is z's error before any rounding; the backward sees z rounded to dtype
    (slope'' of the smooth activations is at most 0.8) and rounds dz to it."""
    K, (M, N) = x.shape[1], (x.shape[0], w.shape[0])
    y, z = do.linear(x, w, b, name, r, kept)
    ez = (K + 2) * STEP * (np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b)))
    value, slope = do.act(z, name)
    # the activation's own arithmetic: a few ulps of value and argument
    ey = kept * (1.2 * ez + 16 * STEP * (np.abs(value) + np.abs(z) * (name != "none")))
    by = ey * (1 + U[dtype]) + 2 * STEP * (np.abs(y) + np.abs(0 if r is None else r)) + rounded(y, dtype)
    if dy is None:
        return y, by
    _, _, _, dz = do.linear_backward(dy, x, w, z, name, kept)
    if name == "none":
        eslope = np.zeros_like(z)
    elif name == "relu":
        eslope = (np.abs(z) <= ez).astype(float)                 # the sign is open there
    else:
        eslope = 0.8 * (U[dtype] * np.abs(z) + TINY[dtype] + ez) + 32 * STEP * (1 + np.abs(z))
    edz = np.abs(dy) * kept * (eslope + 4 * STEP)
    if name != "none" or not np.isscalar(kept):
        edz = edz + rounded(np.abs(dz) + edz, dtype)
    dx, dw, db, _ = do.linear_backward(dy, x, w, z, name, kept)
    a = np.abs(dz) + edz
    bx = edz @ np.abs(w) + (N + 2) * STEP * (a @ np.abs(w))
    bw = edz.T @ np.abs(x) + (M + 2) * STEP * (a.T @ np.abs(x))
    bb = edz.sum(0) + (M + 2) * STEP * a.sum(0)
    return y, by, (dx, bx + rounded(dx, dtype) + bx * U[dtype]), (dw, bw + rounded(dw, dtype) + bw * U[dtype]), \
        (db, bb + rounded(db, dtype) + bb * U[dtype])


def run_linear(od, seed, dtype, M, K, N, name="none", bias=True, residual=True, p=0.0, train=True, leave=()):
    rng = np.random.default_rng(seed)
    x, w = make(rng, dtype, M, K), make(rng, dtype, N, K, std=max(K, 1) ** -0.5)
    b = make(rng, dtype, N) if bias else None
    r = make(rng, dtype, M, N) if residual else None
    dy = make(rng, dtype, M, N) if train else None
    kept = do.keep(M, N, p, 77, 5) if p else 1.0
    inputs = [("x", x), ("w", w), ("b", b), ("r", r)]
    if train:
        for n, t in inputs:
            if t is not None and n not in leave:
                t.requires_grad_(True)
    y = od.linear(x, w, b, activation=name, residual=r, dropout_p=p, seed=77, offset=5)
    assert y.dtype == dtype and y.shape == (M, N)
    want = linear_bounds(f64(x), f64(w), f64(b), f64(r), f64(dy), name, kept, dtype)
    what = f"{dtype} M{M} K{K} N{N} {name} p{p}"
    check(y, want[0], want[1], what + " y")
    if train:
        leaves = [(n, t) for n, t in inputs if t is not None and t.requires_grad]
        grads = dict(zip([n for n, _ in leaves], torch.autograd.grad(y, [t for _, t in leaves], dy)))
        for n, (g, bound) in zip("xwb", want[2:]):
            if n in grads:
                assert grads[n].dtype == dtype
                check(grads[n], g, bound, f"{what} d{n}")
        if "r" in grads:
            assert torch.equal(grads["r"], dy)


SIZES = [(1, 8, 8), (1, 1, 1), (3, 1, 5), (1, 1024, 96), (2, 333, 40), (16, 256, 72), (17, 64, 64), (33, 96, 50),
         (5, 33, 7), (64, 128, 48), (65, 256, 130), (130, 96, 257), (200, 520, 72), (257, 129, 333), (600, 256, 48),
         (40, 4096, 64), (300, 1000, 520), (129, 2050, 31)]


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("i", range(len(SIZES)), ids=["x".join(map(str, s)) for s in SIZES])
def test_linear(od, dtype, i):
    M, K, N = SIZES[i]
    run_linear(od, i, TYPES[dtype], M, K, N, name=ACTS[i % 5], bias=i % 3 != 1, residual=i % 2 == 0, p=0.0 if i % 4 else 0.3)


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("name", ACTS)
def test_linear_activations_with_dropout(od, dtype, name):
    run_linear(od, 50, TYPES[dtype], 70, 72, 88, name=name, p=0.25)
    run_linear(od, 51, TYPES[dtype], 3, 40, 264, name=name, p=0.0, train=False)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_activation_and_slope_at_every_magnitude(od, dtype, name):
    """z = x 1 is exact, so only the activation and the rounding of its result are off: every finite 16-bit number (every
    65521st fp32 one).  a, the exponent's argument, carries a few roundings: 2^-21 |a| of the value; beyond |a| = 100 the
    exponential is 0 or its term all that counts, and below -87 the value left, under 128 x 2^-126, may become 0.  erf's
    error is absolute: 2^-21 |z| until it is 1 (|z| < 8).  The oracle's 1 + tanh in 64 bits is itself off by up to 2^-52
    (tanh by an ulp below 1, and the sum's rounding) and so its value by |z| / 2 times that, until both are 0 or 2: at
    |z| >= 8 what it loses is under |z| exp(-49).  The slopes' as in linear_bounds."""
    if dtype == torch.float32:
        x = torch.arange(-2 ** 31, 2 ** 31, 65521).to(torch.int32).view(dtype)
    else:
        x = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)].reshape(-1, 1).cuda().requires_grad_()
    z = f64(x)
    with np.errstate(over="ignore"):
        value, slope = do.act(z, name)
    y = od.linear(x, torch.ones(1, 1, dtype=dtype, device="cuda"), activation=name)
    y.backward(torch.ones_like(y))
    a = {"gelu": 0, "silu": z, "gelu_tanh": 1.6 * (z + 0.044715 * z ** 3)}[name]
    off = 2.0 ** -21 * (np.abs(value) * (1 + np.minimum(np.abs(a), 100)) + (name == "gelu") * np.minimum(np.abs(z), 8))
    off += 2.0 ** -53 * (name == "gelu_tanh") * np.minimum(np.abs(z), 8)
    check(y, value, off * (1 + U[dtype]) + rounded(value, dtype) + 2.0 ** -119, f"{name} value")
    off = 32 * STEP * (1 + np.minimum(np.abs(z), 128))
    check(x.grad, slope, off * (1 + U[dtype]) + 2 * rounded(slope, dtype), f"{name} slope")


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_linear_few_rows(od, dtype):
    """Up to 16 rows of x go through a kernel of their own: both its widths, whole and odd lengths, every row count."""
    for i, M in enumerate(range(1, 18)):
        run_linear(od, 100 + i, TYPES[dtype], M, 64 * (i + 1) + (0, 1, 8)[i % 3], 33 + 17 * i, name=ACTS[i % 5], p=0.2, train=i % 4 == 0)
    run_linear(od, 120, TYPES[dtype], 1, 8200, 4096, name="silu", train=False)
    run_linear(od, 121, TYPES[dtype], 3, 4099, 57, train=False)
    run_linear(od, 122, TYPES[dtype], 16, 2048, 9001, train=False)
    run_linear(od, 123, TYPES[dtype], 2, 8192, 40, train=False)                # few columns over long rows: tiles in fp32
    run_linear(od, 124, TYPES[dtype], 9, 4104, 8200, train=False)              # nine rows over a large W: tiles in 16 bits


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_linear_many_tiles(od, dtype):
    """Whole and partial tiles of the wide variants, more than one band of tile rows, all three products."""
    run_linear(od, 60, TYPES[dtype], 1100, 192, 1300, bias=True, residual=False)
    run_linear(od, 61, TYPES[dtype], 2049, 136, 776, name="silu", p=0.1)
    run_linear(od, 62, TYPES[dtype], 1031, 131, 1029, name="gelu")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,wants", [(512, 264, (True, True)), (300, 7, (True, True)), (512, 264, (False, False)), (77, 1003, (True, False)),
                                       (4097, 40, (False, True)), (1, 24, (True, True))])
def test_bias_gradient_is_summed_before_dz_is_rounded(od, dtype, m, n, wants):
    """dy = 1 and a scale half a step from a 16-bit number: rounded first, dz and its sum would be off by half a step in
    every column, beside the sum's own rounding.  Sums in fp32: m roundings at most."""
    dtype = TYPES[dtype]
    k = round(65536 * U[dtype]) - (dtype == torch.bfloat16)            # scale 1 + U, just below
    x = torch.ones(m, 16, dtype=dtype, device="cuda", requires_grad=wants[0])
    w = torch.ones(n, 16, dtype=dtype, device="cuda", requires_grad=wants[1])
    b = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    y = od.linear(x, w, b, dropout_p=k / 65536, seed=9, offset=3)
    y.backward(torch.ones_like(y))
    want = do.keep(m, n, k / 65536, 9, 3).sum(0)
    check(b.grad, want, rounded(want, dtype) + (m + 2) * 2.0 ** -24 * want, "dbias")


@pytest.mark.parametrize("leave", ["x", "w", "b", "xw", "xb", "wb", "xwr"])
def test_linear_gradients_asked_for_one_by_one(od, leave):
    run_linear(od, 70, torch.bfloat16, 150, 136, 72, name="silu", leave=tuple(leave))
    run_linear(od, 71, torch.float32, 150, 136, 72, leave=tuple(leave))


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_linear_sizes_of_zero(od, dtype):
    for M, K, N in ((0, 16, 8), (4, 0, 8), (4, 16, 0), (0, 0, 0)):
        run_linear(od, 80, TYPES[dtype], M, K, N)
        run_linear(od, 81, TYPES[dtype], M, K, N, name="gelu", p=0.5)


def test_linear_orders_strides_and_addresses(od):
    rng = np.random.default_rng(90)
    for dtype in TYPES.values():
        buf = make(rng, dtype, 4000)
        for shift in (0, 1, 3):
            x = buf[shift:shift + 30 * 40].view(5, 6, 40)
            w = make(rng, dtype, 40, 24, std=0.1).t()                   # [24, 40], columns first
            b = make(rng, dtype, 48)[::2]
            r = make(rng, dtype, 6, 5, 24).transpose(0, 1)
            y = od.linear(x, w, b, residual=r, activation="silu")
            want, bound = linear_bounds(f64(x).reshape(30, 40), f64(w), f64(b), f64(r).reshape(30, 24), None, "silu", 1.0, dtype)
            assert y.is_contiguous()
            check(y.view(30, 24), want, bound, f"{dtype} shift {shift}")
        xe = make(rng, dtype, 1, 40).expand(9, 40).detach().requires_grad_(True)
        y = od.linear(xe, w)
        g, = torch.autograd.grad(y, xe, torch.ones((), device="cuda", dtype=dtype).expand(9, 24))
        want, bound = linear_bounds(f64(xe), f64(w), None, None, np.ones((9, 24)), "none", 1.0, dtype)[2]
        check(g, want, bound, "expanded")


def test_linear_non_finite_rows_stay_in_their_rows(od):
    rng = np.random.default_rng(91)
    for dtype in TYPES.values():
        for M, K, N in ((3, 64, 40), (40, 100, 70), (300, 192, 260)):
            x, w = make(rng, dtype, M, K), make(rng, dtype, N, K)
            clean = od.linear(x, w)
            x[1, 5], x[M - 1, K - 1] = float("inf"), float("nan")
            y = od.linear(x, w)
            keep = torch.ones(M, dtype=torch.bool)
            keep[[1, M - 1]] = False
            assert torch.equal(y[keep], clean[keep])
            assert not torch.isfinite(y[1]).any() and torch.isnan(y[M - 1]).all()
            z = w[:, 5].float() != 0
            assert (torch.isinf(y[1]) == z).all()                       # inf * w, no NaN made of it


def test_linear_repeats_bit_for_bit_and_in_place_residual(od):
    rng = np.random.default_rng(92)
    x, w, r = (make(rng, torch.float32, *s) for s in ((200, 4096), (64, 4096), (200, 64)))
    a = od.linear(x, w, residual=r, activation="gelu")
    for _ in range(3):
        assert torch.equal(a, od.linear(x, w, residual=r, activation="gelu"))


# ------------------------------------------------------------------------------------------------
# residual_norm
# ------------------------------------------------------------------------------------------------
def run_norm(od, seed, dtype, B, T, D, kind="layer", post=True, gate="sample", affine=True, p=0.0, scale=1.0, train=True,
             want_stream=True, what="", x_scale=1.0):
    rng = np.random.default_rng(seed)
    t = {"x": make(rng, dtype, B, T, D, std=x_scale), "block": make(rng, dtype, B, T, D, mean=0.2, std=1.5 * x_scale)}
    if affine:
        t["weight"], t["bias"] = make(rng, dtype, D, mean=1, std=0.2), make(rng, dtype, D)
    if post:
        t["post_weight"] = make(rng, dtype, D, mean=1, std=0.2)
        if affine:
            t["post_bias"] = make(rng, dtype, D)
    shape = {"none": None, "channel": (D,), "sample": (B, D), "ones": (B, 1, D), "token": (B, T, D)}[gate]
    if shape:
        t["gate"] = make(rng, dtype, *shape, mean=0.5)
    dy, ds = make(rng, dtype, B, T, D), make(rng, dtype, B, T, D)
    M = B * T
    if train:
        for v in t.values():
            v.requires_grad_(True)
    kept = do.keep(M, D, p, 31, 2) if p else 1.0
    res = od.residual_norm(**t, kind=kind, residual_scale=scale, dropout_p=p, seed=31, offset=2, return_stream=want_stream)
    y, stream = res if want_stream else (res, None)

    a = {n: f64(v) for n, v in t.items()}
    a["x"], a["block"] = a["x"].reshape(M, D), a["block"].reshape(M, D)
    if shape:
        a["gate"] = np.broadcast_to(a["gate"].reshape(B, 1, D) if gate == "sample" else a["gate"], (B, T, D)).reshape(M, D)
    n64 = dict(dy=f64(dy).reshape(M, D), dstream=f64(ds).reshape(M, D) if want_stream else None) if train else {}
    want = do.residual_norm(**a, kind=kind, scale=scale, kept=kept, **n64)

    # A row sum in fp32 takes at most 16 + 6 + 16 steps in sequence (a thread's values, the lanes, the waves); a
    # statistic is off by that, relative to the terms' magnitudes, and enters every element of its row.  C counts those
    # steps, the few operations around them and the chain of up to four such sums (post mean, post variance, mean,
    # variance); `size` is the largest magnitude an element's terms have in the row.
    C = 8 * 40 * STEP
    one = lambda v, d: np.full(D, d) if v is None else v                        # noqa: E731
    u_size = np.abs(a["block"])
    if post:
        h = a["block"]
        rs = 1 / np.sqrt((h.var(-1) if kind == "layer" else (h * h).mean(-1)) + 1e-5)[:, None]
        u_size = (rs * np.abs(h).max(-1, keepdims=True)) * np.abs(one(a.get("post_weight"), 1.0)) + np.abs(one(a.get("post_bias"), 0.0))
    g = np.abs(a["gate"]) if shape else 1.0
    r_size = abs(scale) * np.abs(a["x"]) + g * kept * u_size
    er = C * r_size.max(-1, keepdims=True)
    r = want["stream"]
    rstd = 1 / np.sqrt((r.var(-1) if kind == "layer" else (r * r).mean(-1)) + 1e-5)[:, None]
    hat = (want["y"] - one(a.get("bias"), 0.0)) / one(a.get("weight"), 1.0)
    w = np.abs(one(a.get("weight"), 1.0))
    hat_max = np.abs(hat).max(-1, keepdims=True)
    ehat = rstd * er * (1 + hat_max) + C * hat_max                              # r's own error, and rstd's
    ey = w * ehat + 4 * STEP * np.abs(one(a.get("bias"), 0.0))
    what = f"{what}{dtype} {B}x{T}x{D} {kind} post{post} gate {gate} p{p}"
    check(y.reshape(M, D), want["y"], ey + rounded(want["y"], dtype), what + " y")
    if want_stream:
        check(stream.reshape(M, D), r, er + rounded(r, dtype), what + " stream")
    if not train:
        return
    outs, grads = ([y, stream], [dy, ds]) if want_stream else ([y], [dy])
    got = dict(zip(t, torch.autograd.grad(outs, list(t.values()), grads)))

    def back_error(gin, egin, hat, ehat, rstd):
        """error of rstd (g - mean g - hat mean(g hat)) for a g off by egin and a hat off by ehat"""
        gm, hm = np.abs(gin).max(-1, keepdims=True), np.abs(hat).max(-1, keepdims=True)
        eg, eh = np.max(egin, -1, keepdims=True) + 0 * gm, np.max(ehat, -1, keepdims=True) + 0 * gm
        dot = np.abs(gin * hat).mean(-1, keepdims=True)
        edot = eg * np.abs(hat).mean(-1, keepdims=True) + eh * np.abs(gin).mean(-1, keepdims=True) + C * dot
        return rstd * (2 * eg + C * gm + eh * dot + hm * edot) + (C + ehat / np.maximum(hm, 1)) * rstd * (2 * gm + hm * dot)

    n64dy = f64(dy).reshape(M, D)
    edr = back_error(n64dy * w, 2 * STEP * np.abs(n64dy) * w, hat, ehat, rstd)
    ds_size = np.abs(f64(ds).reshape(M, D)) if want_stream else 0.0
    dr = want["dx"] / scale
    edr = edr + 4 * STEP * (np.abs(dr) + ds_size)
    bounds = {"x": abs(scale) * edr}
    du, edu = dr * (a["gate"] if shape else 1.0) * kept, edr * g * kept
    edu = edu + 4 * STEP * np.abs(du)
    u = want["dgate"] / np.where(dr == 0, 1, dr)
    if post:
        pw = np.abs(a["post_weight"])
        hhat = (a["block"] - (a["block"].mean(-1, keepdims=True) if kind == "layer" else 0)) * rs
        ehh = C * (1 + np.abs(hhat).max(-1, keepdims=True)) ** 2 * (1 + rs * np.abs(a["block"]).max(-1, keepdims=True))
        bounds["block"] = back_error(du * a["post_weight"], edu * pw, hhat, ehh, rs)
        eu = kept * (pw * ehh + C * u_size)
    else:
        bounds["block"] = edu
        eu = kept * C * u_size
    steps = (min(M, 4096) + 64) * STEP
    total = lambda v, e: e.sum(0) + steps * (np.abs(v) + e).sum(0)              # noqa: E731
    if affine:
        bounds["weight"], bounds["bias"] = total(n64dy * hat, np.abs(n64dy) * ehat), total(n64dy, 0 * n64dy)
    if post:
        bounds["post_weight"] = total(du * hhat, edu * np.abs(hhat) + np.abs(du) * ehh)
        if affine:
            bounds["post_bias"] = total(du, edu)
    if shape:
        dg, eg = want["dgate"], edr * np.abs(u) + np.abs(dr) * eu + edr * eu
        eg = eg + 4 * STEP * np.abs(dg)
        if gate == "token":
            bounds["gate"] = eg
        else:
            axes = (0, 1) if gate == "channel" else (1,)
            fold = lambda v: v.reshape(B, T, D).sum(axes)                       # noqa: E731
            bounds["gate"] = fold(eg) + steps * fold(np.abs(dg) + eg)
            want["dgate"] = fold(dg)
    for n in t:
        ref = want["d" + n]
        bound = np.broadcast_to(bounds[n], ref.shape) if n in ("x", "block") else bounds[n].reshape(ref.shape)
        check(got[n].reshape(ref.shape), ref, bound + rounded(ref, dtype), f"{what} d{n}")


WIDTHS = [1, 3, 8, 64, 100, 255, 256, 257, 512, 777, 1024, 1025, 2048, 2500, 4096, 5003, 8192, 10001, 16384]


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("i", range(len(WIDTHS)), ids=[str(w) for w in WIDTHS])
def test_norm_widths(od, dtype, i):
    run_norm(od, i, TYPES[dtype], 2, 3, WIDTHS[i], kind="layer" if i % 2 else "rms", post=i % 3 != 0,
             gate=["sample", "none", "token", "channel", "ones"][i % 5], p=0.25 if i % 4 == 1 else 0.0, scale=0.5 + 0.25 * (i % 3))


@pytest.mark.parametrize("gate", ["none", "channel", "sample", "ones", "token"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
def test_norm_gates(od, gate, kind, post):
    """Gate rows of many, a few and one row each; whole gate rows by a workgroup, and several workgroups a gate row."""
    run_norm(od, 40, torch.float32, 5, 61, 72, kind=kind, post=post, gate=gate, p=0.1)
    run_norm(od, 41, torch.bfloat16, 700, 3, 40, kind=kind, post=post, gate=gate)
    run_norm(od, 42, torch.float16, 1, 1, 264, kind=kind, post=post, gate=gate, p=0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_norm_many_rows(od, dtype):
    run_norm(od, 43, TYPES[dtype], 3, 1501, 48, gate="sample", p=0.1)
    run_norm(od, 44, TYPES[dtype], 2, 1400, 264, kind="rms", gate="channel")
    run_norm(od, 45, TYPES[dtype], 1, 700, 2056, kind="layer", post=False, gate="none")


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_norm_without_affine_gradients_or_stream(od, dtype):
    run_norm(od, 46, TYPES[dtype], 2, 9, 136, affine=False)
    run_norm(od, 47, TYPES[dtype], 2, 9, 136, want_stream=False, p=0.3)
    run_norm(od, 48, TYPES[dtype], 2, 9, 136, train=False, p=0.3)
    run_norm(od, 49, TYPES[dtype], 1, 1, 4096, kind="rms", train=False, want_stream=False)


def test_norm_large_offsets_and_constant_rows(od):
    """The variance is of deviations from the mean: an offset of 10^4 costs what it must, a constant row gives its bias."""
    x = torch.full((3, 300), 1e4, device="cuda") + torch.randn(3, 300, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    z = torch.zeros_like(x)
    y = od.residual_norm(x, z)
    want = do.residual_norm(f64(x), f64(z))["y"]
    # an element of 10^4 is off by 0 here (it is the input); its mean by 40 steps
    assert np.abs(f64(y) - want).max() < 40 * STEP * 1e4 * 2
    b = torch.randn(300, device="cuda")
    assert torch.equal(od.residual_norm(torch.full_like(x, 3.0), z, None, b), b.expand(3, 300))
    assert torch.equal(od.residual_norm(z, z, None, b, kind="rms"), b.expand(3, 300))


def test_norm_gradients_asked_for_one_by_one_and_one_result_used(od):
    rng = np.random.default_rng(5)
    names = ["x", "block", "weight", "bias", "post_weight", "post_bias", "gate"]
    shapes = [(6, 11, 72), (6, 11, 72), (72,), (72,), (72,), (72,), (6, 72)]
    vals = [make(rng, torch.float32, *s) for s in shapes]
    dy = make(rng, torch.float32, 6, 11, 72)

    def grads(only, which):
        t = dict(zip(names, [v.clone().requires_grad_(n in only) for n, v in zip(names, vals)]))
        out = od.residual_norm(**t, return_stream=True)[which]
        return dict(zip(only, torch.autograd.grad(out, [t[n] for n in only], dy, allow_unused=True)))

    for which in (0, 1):
        whole = grads(names, which)
        for n in names:
            if whole[n] is not None:
                assert torch.equal(grads([n], which)[n], whole[n]), (which, n)
    assert grads(names, 1)["weight"] is not None and not grads(names, 1)["weight"].any()


def test_norm_no_rows(od):
    for gate in (None, (0, 16), (16,), (0, 5, 16)):
        t = {"x": torch.zeros(0, 5, 16, device="cuda"), "block": torch.zeros(0, 5, 16, device="cuda"),
             "weight": torch.ones(16, device="cuda")}
        if gate:
            t["gate"] = torch.ones(gate, device="cuda")
        for v in t.values():
            v.requires_grad_(True)
        y = od.residual_norm(**t)
        got = dict(zip(t, torch.autograd.grad(y, list(t.values()), torch.zeros_like(y))))
        assert y.shape == (0, 5, 16) and not got["weight"].any() and all(got[n].shape == t[n].shape for n in t)
        assert not any(torch.isnan(v).any() for v in got.values())
    t = {"x": torch.zeros(3, 0, 16, device="cuda", requires_grad=True), "block": torch.zeros(3, 0, 16, device="cuda"),
         "gate": torch.ones(3, 16, device="cuda", requires_grad=True)}
    y = od.residual_norm(**t)
    assert not torch.autograd.grad(y, t["gate"], torch.zeros_like(y))[0].any()


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 1), (1, 8), (5, 3), (33, 20), (100, 256), (3, 4097), (300, 1003), (1, 70001)])
def test_dropout(od, dtype, rows, cols):
    dtype = TYPES[dtype]
    rng = np.random.default_rng(rows + cols)
    for p, residual in ((0.1, True), (0.5, False), (1.0, True), (0.0, True)):
        x = make(rng, dtype, rows, cols).requires_grad_(True)
        r = make(rng, dtype, rows, cols).requires_grad_(True) if residual else None
        dy = make(rng, dtype, rows, cols)
        y = od.dropout(x, p, 2 ** 63 + 11, offset=9, residual=r)
        k = do.keep(rows, cols, p, 2 ** 63 + 11, 9)
        want = f64(x) * k + (f64(r) if residual else 0.0)
        check(y, want, rounded(want, dtype) + 4 * STEP * (np.abs(f64(x) * k) + np.abs(want)), f"p {p}")
        if p == 1.0:
            assert torch.equal(y, r)
        g = torch.autograd.grad(y, [x] + ([r] if residual else []), dy)
        check(g[0], f64(dy) * k, rounded(f64(dy) * k, dtype) + 4 * STEP * np.abs(f64(dy) * k), "dx")
        if residual:
            assert torch.equal(g[1], dy)


def test_one_mask_whatever_the_operator_type_and_shape(od):
    rows, cols, p = 70, 100, 0.3
    k = do.keep(rows, cols, p, 123, 4) != 0
    eye = torch.eye(cols, device="cuda")
    for dtype in TYPES.values():
        one = torch.ones(rows, cols, device="cuda", dtype=dtype)
        assert np.array_equal(f64(od.dropout(one, p, 123, 4)) != 0, k)
        assert np.array_equal(f64(od.dropout(one.view(7, 10, cols), p, 123, 4)).reshape(rows, cols) != 0, k)
        assert np.array_equal(f64(od.linear(one, eye.to(dtype), dropout_p=p, seed=123, offset=4)) != 0, k)
        stream = od.residual_norm(torch.zeros_like(one), one, dropout_p=p, seed=123, offset=4, return_stream=True)[1]
        assert np.array_equal(f64(stream) != 0, k)
    seed = torch.tensor(123, device="cuda")
    assert np.array_equal(f64(od.dropout(one, p, seed, 4)) != 0, k)
    assert np.array_equal(f64(od.dropout(one, p, 123 - 2 ** 64, 4)) != 0, k)


def test_dropped_values_are_zero_whatever_they_were(od):
    x = torch.full((64, 64), float("nan"), device="cuda")
    y = od.dropout(x, 0.5, 1)
    k = do.keep(64, 64, 0.5, 1) != 0
    assert np.array_equal(np.isnan(f64(y)), k) and not f64(y)[~k].any()


def test_as_many_rows_as_a_launch_takes(od):
    """2^31 rows of two columns (8 GiB), both ends; 2^32 rows would be more threads than a launch counts: refused."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    x = torch.ones(2 ** 32, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="too large"):
        od.dropout(x, 0.5, 3)
    y = od.dropout(x.view(2 ** 31, 2), 0.5, 3)
    for first in (0, 2 ** 31 - 64):
        want = do.keep(64, 2, 0.5, 3, first_row=first)
        assert np.array_equal(f64(y[first:first + 64]), want)


# ------------------------------------------------------------------------------------------------
# streams, graphs, devices, seeds, refusals
# ------------------------------------------------------------------------------------------------
def layer(od, t, seed, offset=0):
    """What follows the sampling in a decoder layer: way back into the stream, norm, feed-forward block, norm."""
    h = od.linear(t["sampled"], t["w0"], t["b0"])
    q = od.residual_norm(t["query"], h, t["g0"], t["h0"], dropout_p=0.1, seed=seed, offset=offset)
    f = od.linear(q, t["w1"], t["b1"], activation="relu", dropout_p=0.1, seed=seed, offset=offset + 1)
    s = od.linear(f, t["w2"], t["b2"], dropout_p=0.1, seed=seed, offset=offset + 2, residual=q)
    return od.residual_norm(torch.zeros_like(s), s, t["g1"], t["h1"])


def layer_tensors(dtype=torch.float32, Q=150, E=64, S=512, F=128):
    gen = torch.Generator("cuda").manual_seed(3)
    n = lambda *s, std=1.0: (torch.randn(s, generator=gen, device="cuda") * std).to(dtype)        # noqa: E731
    return {"sampled": n(2, Q, S), "query": n(2, Q, E), "w0": n(E, S, std=S ** -0.5), "b0": n(E), "g0": 1 + n(E, std=0.1),
            "h0": n(E), "w1": n(F, E, std=E ** -0.5), "b1": n(F), "w2": n(E, F, std=F ** -0.5), "b2": n(E),
            "g1": 1 + n(E, std=0.1), "h1": n(E)}


def test_operators_together_with_the_sampling(od):
    """A decoder layer's sampling and what follows it, forward and backward, against the same in torch, fp64 on the CPU,
    from the sampled features on."""
    from opus_amd import opus_sampling
    from helpers import sampling4d_case, TINY_LEVELS
    B, Q, T, G, P, N, E = 1, 60, 2, 4, 2, 6, 256
    _, _, occ2img = sampling4d_case(5, B, Q, T, G, P, N=N)
    gen = torch.Generator("cuda").manual_seed(9)
    n = lambda *s, std=1.0: torch.randn(s, generator=gen, device="cuda") * std                    # noqa: E731
    feats = [n(B * T * G, N, h, w, 64).requires_grad_(True) for h, w in TINY_LEVELS]
    query = n(B, Q, E).requires_grad_(True)
    points = torch.rand((B, Q, 8, 3), generator=gen, device="cuda")
    ow, ob, sw, sb = n(G * P * 3, E, std=0.06), n(G * P * 3), n(G * P * 4, E, std=0.06), n(G * P * 4)
    rng = [-40.0, -40.0, -1.0, 40.0, 40.0, 5.4]
    inputs = (points, query, ow, ob, sw, sb, T, G, P, 4, rng)
    sp, scales = opus_sampling.sampling_inputs(*inputs, fused=True)
    sp0, scales0 = opus_sampling.sampling_inputs(*inputs)
    # two fp32 products of 256 terms of about 1/16 .. apart: 258 steps times the sum of magnitudes, times the points' spread
    assert (scales - scales0).abs().max() < 4 * 258 * STEP * 256 * 0.06
    assert (sp - sp0).abs().max() < 4 * 258 * STEP * 256 * 0.06 * 30
    out = opus_sampling.sampling_4d(sp, feats, scales, torch.from_numpy(occ2img).cuda(), 256, 704, N)
    t = layer_tensors(E=E, S=G * T * P * 64)
    t["sampled"], t["query"] = out.reshape(B, Q, -1), query
    y = layer(od, t, 21)
    grad = n(B, Q, E)
    sampled = t["sampled"]
    got = torch.autograd.grad(y, [sampled, query, *feats], grad)
    assert all(torch.isfinite(g).all() for g in got) and all(g.abs().max() > 0 for g in got)

    d = {k: v.detach().cpu().double() for k, v in t.items()}
    d["sampled"].requires_grad_(True)
    d["query"].requires_grad_(True)
    F = torch.nn.functional
    k = [torch.from_numpy(do.keep(B * Q, c, 0.1, 21, i)).view(B, Q, c) for i, c in enumerate((E, 128, E))]
    q = F.layer_norm(d["query"] + k[0] * F.linear(d["sampled"], d["w0"], d["b0"]), (E,), d["g0"], d["h0"])
    f = k[1] * F.linear(q, d["w1"], d["b1"]).relu()
    want = F.layer_norm(q + k[2] * F.linear(f, d["w2"], d["b2"]), (E,), d["g1"], d["h1"])
    # fp32 end to end: each product's error is at most (terms + 2) steps of sums of magnitudes near sqrt(terms), and the
    # norms pass it on with a factor near 1: 1026 * 2^-23 * sqrt(1024) bounds it, in practice by far
    tol = 1026 * STEP * 32
    assert (y.detach().cpu().double() - want.detach()).abs().max() < tol
    ws, = torch.autograd.grad(want, d["sampled"], grad.cpu().double())
    # a relu whose sign the rounding decides would show: compare where all but a few agree
    off = (got[0].cpu().double() - ws).abs().flatten()
    assert off.kthvalue(int(off.numel() * 0.99)).values < tol


def test_other_streams(od):
    t = layer_tensors()
    want = layer(od, t, 4)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in side:
        with torch.cuda.stream(s):
            outs.append(layer(od, t, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_captured_step_replays_with_new_inputs_and_seeds(od, dtype):
    """Forward and backward in one graph; the seed is a tensor that the graph's user changes between replays."""
    t = layer_tensors(TYPES[dtype])
    leaves = [v.requires_grad_(True) for v in t.values()]
    grad = torch.randn_like(t["query"])
    seed = torch.tensor([5], device="cuda")

    def step():
        y = layer(od, t, seed)
        return [y, *torch.autograd.grad(y, leaves, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        with torch.no_grad():
            seed.fill_(100 + turn)
            t["sampled"].normal_()
        graph.replay()
        got = [o.detach().clone() for o in out]
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b.detach())
    seeds = []
    for turn in range(2):
        with torch.no_grad():
            seed.fill_(turn)
        graph.replay()
        seeds.append(out[0].detach().clone())
    assert not torch.equal(*seeds)


def test_two_captured_graphs_replayed_in_turn(od):
    """Graphs that are captured one after the other own their workspaces (the product's r is cut up here)."""
    rng = np.random.default_rng(6)
    xs = [make(rng, torch.bfloat16, 64, 4096) for _ in range(2)]
    w = make(rng, torch.bfloat16, 64, 4096, std=0.02)
    want = [od.linear(x, w) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(od.linear(x, w))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            assert torch.equal(o, e)


def test_seed_tensor_changed_before_the_backward_is_an_error(od):
    seed = torch.tensor([5], device="cuda")
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    y = od.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_against_differences(od):
    """Directional derivatives of the GPU operators themselves, fp32, central differences: with a step of 2^-6 along a
    unit direction the difference's own error is h^2 / 6 of a third derivative (order 1 here) plus rounding of the loss
    (sum of about 10^3 terms: 2^-24 * 10^3 / h)."""
    t = layer_tensors(Q=20, E=32, S=64, F=40)
    gen = torch.Generator("cuda").manual_seed(8)
    x, w, b = t["sampled"], torch.randn((48, 64), generator=gen, device="cuda") * 0.125, torch.randn(48, generator=gen, device="cuda")
    c = torch.randn((2, 20, 48), generator=gen, device="cuda")
    blk, gate = torch.randn((2, 20, 64), generator=gen, device="cuda"), torch.randn((2, 64), generator=gen, device="cuda")
    c2 = torch.randn((2, 20, 64), generator=gen, device="cuda")
    f1 = lambda x, w, b: (od.linear(x, w, b, activation="gelu", dropout_p=0.2, seed=3).double() * c).sum()         # noqa: E731
    f2 = lambda x, blk, gate: (od.residual_norm(x, blk, post_weight=torch.ones(64, device="cuda"), gate=gate,      # noqa: E731
                                                dropout_p=0.2, seed=3).double() * c2).sum()
    f3 = lambda x: (od.dropout(x, 0.2, 3).double() ** 2 / 2).sum()                                                 # noqa: E731
    h = 2.0 ** -6
    for f, args in ((f1, (x, w, b)), (f2, (x, blk, gate)), (f3, (x,))):
        args = [a.detach().clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(f(*args), args)
        for i, a in enumerate(args):
            v = torch.randn(a.shape, generator=gen, device="cuda")
            v = v / v.norm()
            with torch.no_grad():
                up = f(*[q + h * v if j == i else q for j, q in enumerate(args)])
                down = f(*[q - h * v if j == i else q for j, q in enumerate(args)])
            slope = (grads[i].double() * v).sum()
            assert abs((up - down) / (2 * h) - slope) < 20 * (h * h + 2.0 ** -24 * 1e3 / h) * (1 + abs(slope))


def test_refusals(od):
    x, w = torch.zeros(4, 16, device="cuda"), torch.zeros(8, 16, device="cuda")
    bad = [lambda: od.linear(x, w.half()), lambda: od.linear(x, w[:, :15]), lambda: od.linear(x, w[0]),
           lambda: od.linear(x, w, torch.zeros(7, device="cuda")), lambda: od.linear(x, w, torch.zeros(8)),
           lambda: od.linear(x, w, residual=torch.zeros(4, 7, device="cuda")), lambda: od.linear(x.double(), w.double()),
           lambda: od.linear(x, w, residual=torch.zeros(1, 8, device="cuda")),
           lambda: od.linear(x, w, dropout_p=0.5), lambda: od.linear(x, w, dropout_p=0.5, seed=torch.zeros(1, dtype=torch.int64)),
           lambda: od.linear(torch.zeros((), device="cuda"), w), lambda: od.linear(x, w, activation="tanh"),
           lambda: od.linear(x, w, dropout_p=1.5, seed=1), lambda: od.linear(x, w, dropout_p=0.5, seed=1, offset=-1),
           lambda: od.residual_norm(x, x[:2]), lambda: od.residual_norm(x, x, w), lambda: od.residual_norm(x, x, kind="batch"),
           lambda: od.residual_norm(x, x, post_bias=x[0]), lambda: od.residual_norm(x, x, gate=x[:3]),
           lambda: od.residual_norm(x, x, residual_scale=torch.ones((), device="cuda")), lambda: od.residual_norm(x, x, eps=-1.0),
           lambda: od.residual_norm(x, x, eps=float("nan")), lambda: od.residual_norm(x, x.half()), lambda: od.residual_norm(x[:, :0], x[:, :0]),
           lambda: od.residual_norm(torch.zeros(1, 16385, device="cuda"), torch.zeros(1, 16385, device="cuda")),
           lambda: od.dropout(x, 0.5, None), lambda: od.dropout(x, -0.5, 1), lambda: od.dropout(x, 0.5, 1, residual=x[0]),
           lambda: od.dropout(x.int(), 0.5, 1)]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            raise AssertionError(f"call {i} was taken")


def test_no_second_derivatives(od):
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.randn(16, 16, device="cuda")
    for f in (lambda: od.dropout(x, 0.5, 1), lambda: od.linear(x, w, activation="silu"), lambda: od.residual_norm(x, x)):
        g, = torch.autograd.grad((f() ** 2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_one_dimension_and_no_gradient_modes(od):
    rng = np.random.default_rng(7)
    x, w = make(rng, torch.float32, 40).requires_grad_(True), make(rng, torch.float32, 24, 40)
    y = od.linear(x, w)
    assert y.shape == (24,) and y.requires_grad
    want, bound = linear_bounds(f64(x)[None], f64(w), None, None, None, "none", 1.0, torch.float32)
    check(y[None], want, bound, "one dimension")
    with torch.no_grad():
        assert not od.linear(x, w).requires_grad and not od.dropout(x, 0.5, 1).requires_grad
    with torch.inference_mode():
        assert torch.equal(od.linear(x, w), y.detach())
    n = od.residual_norm(x, x, gate=x)
    assert n.shape == (40,)
    n.sum().backward()
    assert x.grad.shape == (40,)
    assert od.dropout(torch.zeros(3, 0, device="cuda"), 0.5, 1).shape == (3, 0)


def test_backward_twice_and_inputs_changed_in_between(od):
    rng = np.random.default_rng(8)
    x, w = make(rng, torch.float32, 30, 40).requires_grad_(True), make(rng, torch.float32, 24, 40).requires_grad_(True)
    y = od.linear(x, w, activation="gelu", dropout_p=0.2, seed=3)
    a = torch.autograd.grad(y.sum(), [x, w], retain_graph=True)
    b = torch.autograd.grad(y.sum(), [x, w], retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_saved_tensors_that_move_and_checkpointing(od):
    """Saved-tensor hooks hand the backward other tensors (the seed's among them); activation checkpointing runs the
    forward again.  Both give the plain run's gradients, bit for bit."""
    t = layer_tensors()
    leaves = [v.requires_grad_(True) for v in t.values()]
    grad = torch.randn_like(t["query"])

    def grads(run):
        y = run()
        torch.full((64,), -1, device="cuda")                     # (what a freed seed's place may hold next)
        return torch.autograd.grad(y, leaves, grad)

    want = grads(lambda: od.dropout(layer(od, t, 8), 0.3, 8, 9))

    def moved():
        with torch.autograd.graph.save_on_cpu():
            return od.dropout(layer(od, t, torch.tensor([8], device="cuda")), 0.3, torch.tensor([8], device="cuda"), 9)

    def again():
        seed = torch.tensor([8], device="cuda")
        return torch.utils.checkpoint.checkpoint(lambda: od.dropout(layer(od, t, seed), 0.3, seed, 9), use_reentrant=False)

    for run in (moved, again):
        for a, b in zip(grads(run), want):
            assert torch.equal(a, b)


def test_threads_at_once(od):
    """Calls from several host threads, each on a stream of its own."""
    import threading
    t = layer_tensors()
    want = layer(od, t, 4)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = layer(od, t, 4)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(g, want) for g in got)


def test_offsets_beyond_32_bits(od):
    """Matrices of more than 2^32 bytes and 2^31 elements: the last rows are what the same rows give by themselves."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of device memory")
    gen = torch.Generator("cuda").manual_seed(2)
    n = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=torch.bfloat16)       # noqa: E731
    M, K, N, tail = 70000, 64, 40000, 300                                        # 2.8e9 outputs
    x, w, b = n(M, K), n(N, K), n(N)
    y = od.linear(x, w, b, activation="relu")
    part = od.linear(x[-tail:], w, b, activation="relu")
    err = (y[-tail:].float() - part.float()).abs()
    assert (err <= 2 * U[torch.bfloat16] * part.float().abs() + (K + 2) * STEP * 64).all()   # (another plan's order of sums)
    del y, part, err
    dy = n(M, N)
    xr = x.requires_grad_(True)
    dx, = torch.autograd.grad(od.linear(xr, w), xr, dy)
    ref = dy[-tail:].float() @ w.float()
    # fp32 sums of N terms of about 1 on both sides, then one rounding
    assert ((dx[-tail:].float() - ref).abs() <= U[torch.bfloat16] * ref.abs() * 1.01 + 2 * (N + 2) * STEP * N ** 0.5).all()
    del dy, dx, ref
    rows, width = 2 ** 19 + 3, 8200                                              # 4.3e9 elements
    x = torch.empty(rows, width, device="cuda", dtype=torch.bfloat16)
    block = torch.empty_like(x)
    for t in (x, block):
        t.normal_(generator=gen)
    y = od.residual_norm(x, block, dropout_p=0.0)
    assert torch.equal(y[-70:], od.residual_norm(x[-70:], block[-70:]))
    d = od.dropout(x, 0.5, 9)
    k = torch.from_numpy(do.keep(5, width, 0.5, 9, first_row=rows - 5)).cuda()
    assert torch.equal(d[-5:].double(), x[-5:].double() * k)


def test_tangents_are_refused_and_traced_calls_compute(od):
    """A tangent raises instead of being lost, in the backward's own thread too; a traced module runs the kernels."""
    import warnings
    from torch.autograd import forward_ad
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(16, 16, device="cuda")
    for f in (lambda x: od.linear(x, w, activation="gelu"), lambda x: od.residual_norm(x, x, gate=x), lambda x: od.dropout(x, 0.5, 3)):
        want, other = f(x), torch.randn(7, 16, device="cuda")
        with forward_ad.dual_level():
            assert torch.equal(f(x), want)
            with pytest.raises(NotImplementedError):
                f(forward_ad.make_dual(x, x))
            leaf = x.clone().requires_grad_(True)
            with pytest.raises(RuntimeError, match="no tangent goes through"):
                torch.autograd.grad(f(leaf), leaf, forward_ad.make_dual(want, want))
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(f, (x,), check_trace=False)
        held = [torch.full((7, 16), 7.0, device="cuda") for _ in range(20)]
        del held
        assert torch.equal(traced(other), f(other)) and torch.equal(traced(x), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K,N", [(5, 24, 40), (70, 40, 72), (40, 4096, 64), (300, 33, 260)])
def test_linear_gradients_where_x_w_is_beyond_the_type(od, dtype, name, M, K, N):
    """z larger than the type's largest number, which the forward keeps for the backward: slopes are 0 or 1 there, never NaN.
    z = x[m, 0] w[n, 0] is exact in fp32 (the other columns of x are 0), so its own error is the rounding where it is kept
    (eslope as in linear_bounds, up to |z| = 64; beyond, the slopes are 0 or 1 but for 64 exp(-64))."""
    dtype = TYPES[dtype]
    rng = np.random.default_rng(M)
    # fp16: up to 1e6; bf16: 181^2 2^113 = 1.9996 x 2^127, which rounds to inf in bf16 and not in fp32
    big = (1000.0, 1000.0) if dtype == torch.float16 else (181 * 2.0 ** 56, 181 * 2.0 ** 57)
    x, w = torch.zeros(M, K), torch.from_numpy(rng.standard_normal((N, K))).float()
    x[:, 0] = torch.from_numpy(rng.choice([-1.0, 1.0], M) * rng.choice([0.001, 0.5, 1, big[0]], M))
    w[:, 0] = torch.from_numpy(rng.choice([-1.0, 1.0], N) * rng.choice([0.25, 1, big[1]], N))
    x, w = x.to(dtype).cuda().requires_grad_(True), w.to(dtype).cuda().requires_grad_(True)
    b = torch.zeros(N, dtype=dtype, device="cuda", requires_grad=True)
    dy, p = make(rng, dtype, M, N, std=0.01), 0.3
    kept = do.keep(M, N, p, 77, 5)
    with np.errstate(over="ignore"):
        value, z = do.linear(f64(x), f64(w), None, name)
        slope = do.act(z, name)[1]
    far = np.abs(z) > torch.finfo(dtype).max
    assert far.any() and not far.all() and np.abs(z).max() < torch.finfo(torch.float32).max
    slope = np.where(np.abs(z) > 64, (z > 0).astype(float), slope)
    y = od.linear(x, w, b, activation=name, dropout_p=p, seed=77, offset=5)
    low = (z < 0) | (np.abs(z) < 64)                             # where y is small enough for the type too
    value = np.where(low, value * kept, 0.0)
    value = np.where(np.abs(z) > 64, 0.0, value)
    got = np.where(low, f64(y), 0.0)
    assert (np.abs(got - value) <= kept * 2.0 ** -19 * (np.abs(z) * low * (np.abs(z) < 64) + 1) + rounded(value, dtype)).all()
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], dy)
    dz = f64(dy) * kept * slope
    eslope = np.where(np.abs(z) > 64, 0.0, 0.8 * (U[dtype] * np.abs(z) + TINY[dtype]) + 32 * STEP * (1 + np.abs(z))) * (name != "relu")
    edz = np.abs(f64(dy)) * kept * (eslope + 4 * STEP)
    edz = edz + rounded(np.abs(dz) + edz, dtype)
    a = np.abs(dz) + edz
    for n, g, want, e, sums in (("dx", gx, dz @ f64(w), edz @ np.abs(f64(w)), a @ np.abs(f64(w)) * (N + 2)),
                                ("dw", gw, dz.T @ f64(x), edz.T @ np.abs(f64(x)), a.T @ np.abs(f64(x)) * (M + 2)),
                                ("db", gb, dz.sum(0), edz.sum(0), a.sum(0) * (M + 2))):
        e = e + STEP * sums
        check(g, want, e * (1 + U[dtype]) + rounded(want, dtype), f"{dtype} M{M} K{K} N{N} {name} {n}")


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES)
def test_gelu_keeps_its_tail(od, dtype):
    """Relative to the value: z Phi(z) = z erfc(-z / sqrt 2) / 2, far below where 1 + erf is 0 in fp32.  The argument's two
    roundings change erfc by (z^2 + |z|) of it each, erfc itself is good to a few steps: 2^-21 (1 + z^2) of the value; below
    2^-126 of erfc or of exp(-z^2 / 2) what is left may become 0 (times |z| < 16)."""
    if dtype == torch.float32:
        x = torch.linspace(-15, 15, 60001)
    else:
        x = torch.arange(-2 ** 15, 2 ** 15).to(torch.int16).view(dtype)
        x = x[x.abs() <= 15]
    x = x.reshape(-1, 1).cuda().requires_grad_()
    z = f64(x)
    cdf = 0.5 * np.array([math.erfc(-v / math.sqrt(2)) for v in z.ravel()]).reshape(z.shape)
    pdf = np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    y = od.linear(x, torch.ones(1, 1, dtype=dtype, device="cuda"), activation="gelu")
    y.backward(torch.ones_like(y))
    off = 2.0 ** -21 * (1 + z * z)
    check(y, z * cdf, off * np.abs(z * cdf) * (1 + U[dtype]) + rounded(z * cdf, dtype) + 2.0 ** -122, "value")
    slope = cdf + z * pdf
    check(x.grad, slope, off * (cdf + np.abs(z) * pdf) * (1 + U[dtype]) + 2 * rounded(slope, dtype) + 2.0 ** -122, "slope")


# ------------------------------------------------------------------------------------------------
# results over inputs, where include/opus_dense.h allows it
# ------------------------------------------------------------------------------------------------
def c_call(name, *args):
    from opus_amd import _lib
    lib = _lib.load()
    assert getattr(lib, name)(*args, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("M,K,N", [(1, 72, 40), (13, 4099, 57), (256, 128, 256), (1300, 72, 1301), (70, 33, 13), (40, 8192, 61)])
def test_linear_over_its_residual(od, dtype, M, K, N):
    """Few rows, whole and partial tiles, r cut into shares: y in the residual's place, the same bits."""
    from opus_amd import _lib
    rng, kind = np.random.default_rng(M), _lib.DENSE_F32 + list(TYPES).index(dtype)
    dtype = TYPES[dtype]
    x, w, b, r = make(rng, dtype, M, K), make(rng, dtype, N, K, std=K ** -0.5), make(rng, dtype, N), make(rng, dtype, M, N)
    want = od.linear(x, w, b, activation="silu", residual=r, dropout_p=0.2, seed=3, offset=1)
    need = _lib.load().opus_dense_linear_workspace_bytes(kind, M, N, K)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    drop = _lib.DenseDropout(round(0.2 * 65536), 1, 3, None)
    c_call("opus_dense_linear_forward", kind, x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), M, N, K,
           _lib.DENSE_ACTIVATIONS["silu"], drop, r.data_ptr(), None, ws.data_ptr(), need)
    assert torch.equal(r, want)


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("width", [3, 37, 256, 509, 777, 1024, 2047, 4096, 5003, 8192, 10001, 16384])
def test_norm_over_its_inputs(od, dtype, width):
    """y and the stream over x and block, either way round: the same bits, over more rows than the workgroups take at once."""
    import ctypes
    from opus_amd import _lib
    rng, kind = np.random.default_rng(width), list(TYPES).index(dtype)
    dtype = TYPES[dtype]
    rows = 8200 if width == 37 else 2100 if width in (777, 5003) else 9
    one = [make(rng, dtype, 9, width) for _ in range(2)]
    x, h = (t.repeat(-(-rows // 9), 1)[:rows].contiguous() for t in one)
    w, pw, g = make(rng, dtype, width), make(rng, dtype, width), make(rng, dtype, width)
    want = od.residual_norm(x, h, w, post_weight=pw, gate=g, dropout_p=0.2, seed=3, offset=1, return_stream=True)
    drop = _lib.DenseDropout(round(0.2 * 65536), 1, 3, None)
    for y_over, stream_over in ((0, 1), (1, 0), (0, None), (1, None), (None, 0), (None, 1)):
        ins = [x.clone(), h.clone()]
        outs = [torch.empty_like(x) if i is None else ins[i] for i in (y_over, stream_over)]
        s = _lib.DenseNorm(kind, 0, rows, width, 1, 1e-5, 1.0, ins[0].data_ptr(), ins[1].data_ptr(), w.data_ptr(), None,
                           pw.data_ptr(), None, g.data_ptr(), ctypes.addressof(drop))
        c_call("opus_dense_norm_forward", s, outs[0].data_ptr(), outs[1].data_ptr(), None)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]), (y_over, stream_over)


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (70, 13), (33, 256), (9, 70001), (5000, 7)])
def test_dropout_over_its_inputs(od, dtype, rows, cols):
    from opus_amd import _lib
    rng, kind = np.random.default_rng(cols), list(TYPES).index(dtype)
    dtype = TYPES[dtype]
    x, r = make(rng, dtype, rows, cols), make(rng, dtype, rows, cols)
    drop = _lib.DenseDropout(round(0.4 * 65536), 1, 3, None)
    for residual in (None, r):
        want = od.dropout(x, 0.4, 3, offset=1, residual=residual)
        for over in (0, 1) if residual is not None else (0,):
            ins = [x.clone(), None if residual is None else residual.clone()]
            c_call("opus_dense_dropout", kind, ins[0].data_ptr(), None if ins[1] is None else ins[1].data_ptr(), rows, cols, drop,
                   ins[over].data_ptr())
            assert torch.equal(ins[over], want)
    same = x.clone()                                             # x and residual the same buffer, and y too
    want = od.dropout(x, 0.4, 3, offset=1, residual=x)
    c_call("opus_dense_dropout", kind, same.data_ptr(), same.data_ptr(), rows, cols, drop, same.data_ptr())
    assert torch.equal(same, want)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_norm_eps(od, monkeypatch, dtype, kind, post):
    """eps where it weighs as much as the rows' variance does.  (run_norm's bounds take 1 / sigma with 1e-5, which is an upper
    bound for a larger eps.)  Half as much again in the oracle is seen."""
    plain = do.residual_norm

    def run(eps, oracle_eps, **kw):
        monkeypatch.setattr(do, "residual_norm", functools.partial(plain, eps=oracle_eps))
        run_norm(types.SimpleNamespace(residual_norm=functools.partial(od.residual_norm, eps=eps)), 60, TYPES[dtype], 3, 7, 200,
                 kind=kind, post=post, gate="token", **kw)

    run(0.3, 0.3)
    run(2.0, 2.0, p=0.2)
    with pytest.raises(AssertionError, match="off by"):
        run(0.3, 0.45)


@pytest.mark.parametrize("width", [40, 777, 2048, 5003, 16384])
def test_norm_eps_scales_with_the_square(od, width):
    """Rows times 2^k and eps times 4^k give the same bits, in every variant of the kernels, at both norms."""
    rng = np.random.default_rng(width)
    x, h = make(rng, torch.float32, 3, width), make(rng, torch.float32, 3, width)
    w, dy = make(rng, torch.float32, width), make(rng, torch.float32, 3, width)

    def run(k, eps):
        # post's norm has to see the scaled block and hand on what x is scaled by
        a, b, pw = x * 2.0 ** k, h * 2.0 ** k, torch.full((width,), 2.0 ** k, device="cuda")
        leaves = [t.detach().requires_grad_(True) for t in (a, b, w, pw)]
        y = od.residual_norm(leaves[0], leaves[1], leaves[2], post_weight=leaves[3], kind="layer", eps=eps * 4.0 ** k)
        dx, dh, dw, dpw = torch.autograd.grad(y, leaves, dy)
        return y, dx * 2.0 ** k, dh * 2.0 ** k, dw, dpw * 2.0 ** k

    for k in (-9, 7):
        for a, b in zip(run(0, 0.0625), run(k, 0.0625)):
            assert torch.equal(a, b)


def test_gradients_of_sampling_and_decoder_layer_together(od):
    """Every gradient of the step, every element.  From the sampled features on against 64 bits (a smooth activation, so that no
    sign is open); the features' and the query's through the sampling's own backward of that gradient."""
    from opus_amd import opus_sampling
    from helpers import sampling4d_case, TINY_LEVELS
    B, Q, T, G, P, N, E, S, F = 1, 60, 2, 4, 2, 6, 256, 4 * 2 * 2 * 64, 128
    _, _, occ2img = sampling4d_case(5, B, Q, T, G, P, N=N)
    gen = torch.Generator("cuda").manual_seed(19)
    n = lambda *s, std=1.0: torch.randn(s, generator=gen, device="cuda") * std                    # noqa: E731
    feats = [n(B * T * G, N, h, w, 64).requires_grad_(True) for h, w in TINY_LEVELS]
    query = n(B, Q, E).requires_grad_(True)
    points = torch.rand((B, Q, 8, 3), generator=gen, device="cuda")
    ow, ob, sw, sb = n(G * P * 3, E, std=0.06), n(G * P * 3), n(G * P * 4, E, std=0.06), n(G * P * 4)
    sp, scales = opus_sampling.sampling_inputs(points, query, ow, ob, sw, sb, T, G, P, 4, [-40.0, -40.0, -1.0, 40.0, 40.0, 5.4], fused=True)
    out = opus_sampling.sampling_4d(sp, feats, scales, torch.from_numpy(occ2img).cuda(), 256, 704, N)
    sampled = out.reshape(B, Q, -1)
    t = layer_tensors(E=E, S=S, F=F)
    names = ["w0", "b0", "g0", "h0", "w1", "b1", "w2", "b2", "g1", "h1"]
    leaves = [t[k].requires_grad_(True) for k in names]

    def dense(sampled, query, lin, norm, drop, t):
        q = norm(query + drop(lin(sampled, t["w0"], t["b0"]), 0), t["g0"], t["h0"])
        return norm(q + drop(lin(drop(torch.nn.functional.gelu(lin(q, t["w1"], t["b1"])), 1), t["w2"], t["b2"]), 2), t["g1"], t["h1"])

    d = lambda i: dict(dropout_p=0.1, seed=33, offset=i)                                           # noqa: E731
    q = od.residual_norm(query, od.linear(sampled, t["w0"], t["b0"]), t["g0"], t["h0"], **d(0))
    y = od.residual_norm(q, od.linear(od.linear(q, t["w1"], t["b1"], activation="gelu", **d(1)), t["w2"], t["b2"]), t["g1"],
                         t["h1"], **d(2))
    grad = n(B, Q, E)
    got = torch.autograd.grad(y, [sampled, query, *leaves, *feats], grad, retain_graph=True)
    # the same step's parts in 64 bits
    c = {k: v.detach().cpu().double().requires_grad_(True) for k, v in t.items()}
    c["sampled"], c["query"] = (v.detach().cpu().double().requires_grad_(True) for v in (sampled, query))
    keeps = [torch.from_numpy(do.keep(B * Q, w, 0.1, 33, i)).view(B, Q, w) for i, w in enumerate((E, F, E))]
    want = dense(c["sampled"], c["query"], torch.nn.functional.linear, lambda r, g, h: torch.nn.functional.layer_norm(r, (E,), g, h),
                 lambda v, i: keeps[i] * v, c)
    ws, wq, *wl = torch.autograd.grad(want, [c["sampled"], c["query"], *(c[k] for k in names)], grad.cpu().double())
    # A product of r terms is off by (r + 2) steps of the norms it multiplies, which are the root of r times a typical result;
    # at most four such products and norms stand between a gradient and either end.
    tol = 4 * (S + 2) * STEP * S ** 0.5
    for k, a, b in zip(["y", "sampled", *names], [y.detach(), got[0], *got[2:]], [want.detach(), ws, *wl]):
        assert (a.cpu().double() - b).abs().max() <= tol * b.abs().max(), k
    # the sampling's backward is linear in what it is handed (a feature's sum of up to B Q T G P hits in another order, its
    # weights positive), and the query's two ways add up
    handed = got[0].view_as(out)
    through = torch.autograd.grad(out, [query, *feats], handed, retain_graph=True)
    sizes = torch.autograd.grad(out, feats, handed.abs())
    for a, b, size in zip(got[-len(feats):], through[1:], sizes):
        assert ((a - b).abs() <= 2 * B * Q * T * G * P * STEP * size).all() and b.abs().max() > 0
    total = through[0].cpu().double() + wq
    assert (got[1].cpu().double() - total).abs().max() <= tol * wq.abs().max() + 4 * STEP * float(through[0].abs().max())


@pytest.mark.parametrize("dtype", TYPES, ids=list(TYPES))
def test_a_training_step_repeats_bit_for_bit(od, dtype):
    """Results and every gradient, odd sizes, all of the epilogue: the same bits from call to call."""
    rng, dtype = np.random.default_rng(93), TYPES[dtype]
    M, K, N = 1237, 333, 777
    x, w, b, r = (make(rng, dtype, *s).requires_grad_(True) for s in ((M, K), (N, K), (N,), (M, N)))
    dy = make(rng, dtype, M, N)

    def step():
        y = od.linear(x, w, b, activation="gelu", residual=r, dropout_p=0.1, seed=4)
        n, s = od.residual_norm(y, r, b, gate=r, post_weight=b, dropout_p=0.25, seed=4, offset=1, return_stream=True)
        return [y, n, s, *torch.autograd.grad([n, s], [x, w, b, r], [dy, dy])]

    want = step()
    for _ in range(3):
        for p, q in zip(step(), want):
            assert torch.equal(p, q)


@pytest.mark.filterwarnings("ignore")
def test_a_traced_module_trains(od):
    """Results and gradients of a traced module for other shapes and another seed tensor, and its results without gradients."""
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.randn(24, 16, device="cuda"))
            self.g = torch.nn.Parameter(torch.randn(24, device="cuda"))

        def forward(self, x, seed):
            h = od.linear(x, self.w, activation="gelu", dropout_p=0.3, seed=seed)
            return od.residual_norm(h, h, self.g, gate=h, dropout_p=0.2, seed=seed, offset=1)

    m = Block()
    traced = torch.jit.trace(m, (torch.randn(5, 7, 16, device="cuda"), torch.tensor([3], device="cuda")))
    for i, shape in enumerate(((5, 7, 16), (2, 3, 16), (9, 16))):
        x, seed = torch.randn(shape, device="cuda", requires_grad=True), torch.tensor([i], device="cuda")
        want, got = m(x, seed), traced(x, seed)
        dy = torch.randn_like(want)
        assert torch.equal(got, want)
        for a, b in zip(*(torch.autograd.grad(y, [x, m.w, m.g], dy) for y in (got, want))):
            assert torch.equal(a, b)
        with torch.no_grad():
            assert torch.equal(traced(x, seed), want)
