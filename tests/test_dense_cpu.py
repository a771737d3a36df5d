"""The dense operators without a GPU: the library exports what include/opus_dense.h declares, arguments are refused
before anything is launched, the host side refuses what the documentation does not allow, and the oracle's generator
and gradients are right."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from oracle import dense_oracle as do

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(1 << 12)          # an address that is only checked, never read


@pytest.fixture(scope="module")
def lib():
    from opus_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


def test_library_exports_every_declared_symbol(lib):
    from opus_amd import _lib
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "opus_dense.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(opus_dense_\w+)\s*\(", text)))
    assert declared == sorted(_lib.DENSE_SYMBOLS)
    for name in declared:
        assert getattr(lib, name) is not None
    assert lib.opus_dense_strerror(0) == b"ok"
    assert lib.opus_dense_strerror(-99) == b"unknown error code"
    texts = {lib.opus_dense_strerror(-i) for i in range(0, 8)}
    assert len(texts) == 8


def test_linear_arguments(lib):
    from opus_amd import _lib
    fwd, bwd = lib.opus_dense_linear_forward, lib.opus_dense_linear_backward

    def forward(type=0, x=SOME, w=SOME, M=4, N=8, K=16, act=0, drop=None, y=SOME, ws=NULL, nws=0):
        return fwd(type, x, w, NULL, NULL, M, N, K, act, drop, y, NULL, ws, nws, None)

    assert forward(type=3) == -1 and forward(type=-1) == -1
    assert forward(M=-1) == -2 and forward(N=-1) == -2 and forward(K=-1) == -2
    assert forward(x=NULL) == -3 and forward(w=NULL) == -3 and forward(y=NULL) == -3
    assert forward(x=ctypes.c_void_p(4098)) == -3                      # not a multiple of four
    assert forward(M=1 << 31) == -4 and forward(N=1 << 31) == -4 and forward(K=1 << 31) == -4
    assert forward(act=5) == -6 and forward(act=-1) == -6
    assert forward(drop=_lib.DenseDropout(65537, 0, 0, None)) == -6
    assert forward(drop=_lib.DenseDropout(1, 0, 0, 4100)) == -3        # seed address not a multiple of eight
    assert forward(M=0) == 0 and forward(N=0) == 0
    need = lib.opus_dense_linear_workspace_bytes(0, 64, 8, 1 << 16)
    assert need > 0 and forward(M=64, K=1 << 16) == -5
    assert forward(M=64, K=1 << 16, ws=SOME, nws=need - 1) == -5
    assert forward(M=64, K=1 << 16, ws=ctypes.c_void_p(4100), nws=need) == -5

    def backward(dy=SOME, x=SOME, w=SOME, z=SOME, M=4, N=8, K=16, act=0, drop=None, dz=SOME, dx=SOME, dw=SOME, db=SOME,
                 ws=NULL, nws=0):
        return bwd(1, dy, x, w, z, M, N, K, act, drop, dz, dx, dw, db, ws, nws, None)

    assert backward(dx=NULL, dw=NULL, db=NULL, dy=NULL) == 0           # nothing asked for
    assert backward(dy=NULL) == -3 and backward(x=NULL) == -3 and backward(w=NULL) == -3
    assert backward(act=2, z=NULL) == -3 and backward(act=2, dz=NULL) == -3
    assert backward(drop=_lib.DenseDropout(9, 0, 0, None), dz=NULL) == -3
    assert backward() == -5                                            # the column sums' workspace
    assert backward(M=-1) == -2 and backward(M=1 << 31) == -4 and backward(act=7) == -6


def test_norm_and_dropout_arguments(lib):
    from opus_amd import _lib

    def struct(type=0, kind=0, rows=4, width=8, gate_rows=0, x=SOME, block=SOME, gate=None, drop=None):
        return _lib.DenseNorm(type, kind, rows, width, gate_rows, 1e-5, 1.0, x.value, block.value, None, None, None, None,
                              gate, ctypes.addressof(drop) if drop else None)

    def forward(y=SOME, stats=NULL, **kw):
        return lib.opus_dense_norm_forward(struct(**kw), y, NULL, stats, None)

    assert lib.opus_dense_norm_forward(None, SOME, NULL, NULL, None) == -3
    assert forward(type=7) == -1 and forward(kind=2) == -6
    assert forward(rows=-1) == -2 and forward(width=0) == -2
    assert forward(width=16385) == -4 and forward(rows=1 << 61) == -4
    assert forward(x=NULL) == -3 and forward(block=NULL) == -3 and forward(y=ctypes.c_void_p(4098)) == -3
    assert forward(stats=ctypes.c_void_p(4100)) == -3                  # 16-byte aligned
    assert forward(gate=4096, gate_rows=0) == -2 and forward(gate=4096, gate_rows=3) == -2
    assert forward(drop=_lib.DenseDropout(70000, 0, 0, None)) == -6
    assert forward(rows=0, x=NULL, block=NULL) == 0 and forward(y=NULL) == 0

    def backward(stats=SOME, grads=(4096,) + (None,) * 6, ws=SOME, nws=1 << 30, **kw):
        return lib.opus_dense_norm_backward(struct(**kw), SOME, NULL, stats, _lib.DenseNormGrads(*grads), ws, nws, None)

    assert backward(stats=NULL) == -3 and backward(ws=NULL, nws=0) == -5 and backward(nws=16) == -5
    assert backward(grads=(None,) * 4 + (4096, None, None)) == -6      # a post-norm's gradient without a post-norm
    assert backward(grads=(None,) * 6 + (4096,)) == -6                 # a gate's without a gate
    ws = lib.opus_dense_norm_backward_workspace_bytes
    assert ws(0, 0, 8, 0) == 0 and ws(0, 4, 20000, 0) == 0 and ws(0, 4, 8, 0) > 0

    drop = lib.opus_dense_dropout
    assert drop(5, SOME, NULL, 1, 8, None, SOME, None) == -1
    assert drop(0, SOME, NULL, -1, 8, None, SOME, None) == -2 and drop(0, SOME, NULL, 1, -8, None, SOME, None) == -2
    assert drop(0, SOME, NULL, 1, 1 << 31, None, SOME, None) == -4
    assert drop(0, SOME, NULL, 1 << 40, 8, None, SOME, None) == -4     # more threads than a launch counts
    assert drop(0, NULL, NULL, 1, 8, None, SOME, None) == -3 and drop(0, SOME, NULL, 1, 8, None, NULL, None) == -3
    assert drop(0, NULL, NULL, 0, 8, None, NULL, None) == 0 and drop(0, NULL, NULL, 8, 0, None, NULL, None) == 0


def test_norm_gate_without_rows(lib):
    """No rows and a gate of none: nothing to do, and nothing divided by the gate's rows; fewer than none is refused."""
    from opus_amd import _lib

    def struct(rows, gate_rows):
        return _lib.DenseNorm(0, 0, rows, 8, gate_rows, 1e-5, 1.0, SOME.value, SOME.value, None, None, None, None, 4096, None)

    def backward(rows, gate_rows):
        grads = _lib.DenseNormGrads(*(None,) * 6 + (4096,))
        return lib.opus_dense_norm_backward(struct(rows, gate_rows), SOME, NULL, SOME, grads, NULL, 0, None)

    assert lib.opus_dense_norm_forward(struct(0, 0), SOME, NULL, NULL, None) == 0 and backward(0, 0) == 0
    assert lib.opus_dense_norm_forward(struct(0, -1), SOME, NULL, NULL, None) == -2 and backward(0, -1) == -2


def test_host_side_refuses_cpu_tensors_and_other_types():
    from opus_amd import opus_dense as od
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="expected CUDA tensors"):
        od.linear(x, w)
    with pytest.raises(RuntimeError, match="expected CUDA tensors"):
        od.residual_norm(x, x)
    with pytest.raises(RuntimeError, match="expected CUDA tensors"):
        od.dropout(x, 0.5, 1)


def test_gate_rows():
    from opus_amd.opus_dense import _gate_rows
    x = torch.zeros(3, 5, 8)
    for shape, rows in (((8,), 1), ((3, 8), 3), ((3, 1, 8), 3), ((3, 5, 8), 15), ((1, 1, 8), 1)):
        assert _gate_rows(x, torch.zeros(shape)) == rows, shape
    for shape in ((5, 8), (1, 5, 8), (3, 5, 1), (15, 8), (9,), (), (3, 5, 8, 1)):
        with pytest.raises(RuntimeError, match="does not fit"):
            _gate_rows(x, torch.zeros(shape))
    assert _gate_rows(torch.zeros(8), torch.zeros(8)) == 1
    assert _gate_rows(torch.zeros(0, 5, 8), torch.zeros(0, 8)) == 0


def test_dropout_threshold_and_seed_checks():
    from opus_amd.opus_dense import _threshold
    cpu = torch.device("cpu")
    assert _threshold("d", 0.0, None, 0, cpu) == 0
    assert _threshold("d", 0.5, 7, 0, cpu) == 32768
    assert _threshold("d", 0.1, -1, 0, cpu) == 6554
    assert _threshold("d", 1.0, 7, 2 ** 32 - 1, cpu) == 65536
    assert _threshold("d", 2.0 ** -18, None, 0, cpu) == 0
    assert _threshold("d", np.float32(0.5), np.int64(3), np.int32(2), cpu) == 32768
    from opus_amd.opus_dense import _drop_struct
    drop = _drop_struct(32768, np.int64(-3), np.int32(2))
    assert (drop.seed, drop.offset) == (2 ** 64 - 3, 2)
    assert _threshold("d", 0.5, torch.zeros(1, dtype=torch.int64), 0, cpu) == 32768
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            _threshold("d", p, 7, 0, cpu)
    for seed in (None, 1.5, True, torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            _threshold("d", 0.5, seed, 0, cpu)
    for offset in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            _threshold("d", 0.5, 7, offset, cpu)


def test_dropout_offset_is_an_int():
    """1.2 and 1.7 would both have been offset 1: the same mask twice."""
    from opus_amd.opus_dense import _threshold
    for offset in (1.5, 1.0, True, None, torch.zeros((), dtype=torch.int64)):
        with pytest.raises(RuntimeError):
            _threshold("d", 0.5, 7, offset, torch.device("cpu"))


def test_oracle_generator_against_published_vectors():
    """Known answers of philox4x32-10 (Random123's kat_vectors)."""
    ones = 0xFFFFFFFF
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((ones,) * 4, (ones, ones), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
             (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(int(v) for v in do.philox(np.array(ctr, dtype=np.uint64), key)) == want


def test_oracle_keeps_the_right_share():
    for p in (0.1, 0.5, 0.9):
        k = do.keep(512, 333, p, 11, 3)
        n = k.size
        sigma = (p * (1 - p) / n) ** 0.5
        assert abs((k == 0).mean() - p) < 5 * sigma
        assert abs(np.corrcoef(k[:, :-1].ravel(), k[:, 1:].ravel())[0, 1]) < 5 / n ** 0.5
    assert not np.array_equal(do.keep(64, 64, 0.5, 1, 0), do.keep(64, 64, 0.5, 1, 1))
    assert not np.array_equal(do.keep(64, 64, 0.5, 1, 0), do.keep(64, 64, 0.5, 2, 0))
    assert np.array_equal(do.keep(4, 20, 0.5, 1, 0, first_row=60), do.keep(64, 20, 0.5, 1, 0)[60:])


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_oracle_linear_gradients_against_differences(name):
    rng = np.random.default_rng(0)
    x, w, b, r, dy = (rng.standard_normal(s) for s in ((5, 7), (6, 7), (6,), (5, 6), (5, 6)))
    kept = do.keep(5, 6, 0.3, 9)
    y, z = do.linear(x, w, b, name, r, kept)
    dx, dw, db, _ = do.linear_backward(dy, x, w, z, name, kept)
    h = 1e-5
    for arr, grad in ((x, dx), (w, dw), (b, db)):
        for i in np.ndindex(arr.shape):
            old = arr[i]
            arr[i] = old + h
            up = (do.linear(x, w, b, name, r, kept)[0] * dy).sum()
            arr[i] = old - h
            down = (do.linear(x, w, b, name, r, kept)[0] * dy).sum()
            arr[i] = old
            assert abs((up - down) / (2 * h) - grad[i]) < 1e-7


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
def test_oracle_norm_gradients_against_differences(kind, post):
    rng = np.random.default_rng(1)
    a = {n: rng.standard_normal(s) for n, s in (("x", (3, 5)), ("block", (3, 5)), ("weight", (5,)), ("bias", (5,)),
                                                 ("gate", (3, 5)))}
    if post:
        a.update(post_weight=rng.standard_normal(5), post_bias=rng.standard_normal(5))
    dy, ds = rng.standard_normal((3, 5)), rng.standard_normal((3, 5))
    kept = do.keep(3, 5, 0.3, 4)

    def loss():
        o = do.residual_norm(kind=kind, scale=0.7, kept=kept, **a)
        return (o["y"] * dy).sum() + (o["stream"] * ds).sum()

    out = do.residual_norm(kind=kind, scale=0.7, kept=kept, dy=dy, dstream=ds, **a)
    h = 1e-5
    for name, arr in a.items():
        for i in np.ndindex(arr.shape):
            old = arr[i]
            arr[i] = old + h
            up = loss()
            arr[i] = old - h
            down = loss()
            arr[i] = old
            assert abs((up - down) / (2 * h) - out["d" + name][i]) < 1e-7, name


# ------------------------------------------------------------------------------------------------
# tracers and transforms, with C entries of the library's own signatures that work on host memory
# ------------------------------------------------------------------------------------------------
@pytest.fixture
def standin(monkeypatch, lib):
    """opus_dense on CPU tensors: y = x W^T (+ the dropout's offset), y = x + block and r = 2 y, y = 2 x (+ the seed)."""
    from opus_amd import _lib, opus_dense as od

    def array(p, *shape):
        return np.ctypeslib.as_array((ctypes.c_float * int(np.prod(shape))).from_address(p)).reshape(shape)

    def linear(kind, x, w, b, r, M, N, K, act, drop, y, z, ws, need, stream):
        array(y, M, N)[:] = array(x, M, K) @ array(w, N, K).T + (drop.contents.offset if drop else 0)
        return 0

    def norm(s, y, stream_out, stats, stream):
        s = s.contents
        array(y, s.rows, s.width)[:] = array(s.x, s.rows, s.width) + array(s.block, s.rows, s.width)
        if stream_out:
            array(stream_out, s.rows, s.width)[:] = 2 * array(y, s.rows, s.width)
        return 0

    def dropout(kind, x, r, rows, cols, drop, y, stream):
        seed = ctypes.c_longlong.from_address(drop.contents.seed_ptr).value if drop.contents.seed_ptr else drop.contents.seed
        array(y, rows, cols)[:] = 2 * array(x, rows, cols) + seed
        return 0

    class Library:
        pass

    entries = {"opus_dense_linear_forward": linear, "opus_dense_norm_forward": norm, "opus_dense_dropout": dropout}
    for name, (result, arguments) in _lib.DENSE_SYMBOLS.items():
        f = entries.get(name)
        setattr(Library, name, staticmethod(ctypes.CFUNCTYPE(result, *arguments)(f) if f else getattr(lib, name)))
    monkeypatch.setattr(_lib, "load", lambda: Library)
    monkeypatch.setattr(od, "_check", lambda *a: None)
    monkeypatch.setattr(od, "_run", lambda what, fn, device, *args: _lib.check_dense(fn(*args, None), what))
    return od


W = torch.arange(18.0).view(3, 6) - 8
CALLS = {
    "linear": lambda od, x: od.linear(x, W),
    "linear, everything": lambda od, x: od.linear(x, W, torch.ones(3), "gelu", torch.ones(*x.shape[:-1], 3), 0.5, 3, 7),
    "norm": lambda od, x: od.residual_norm(x, x),
    "norm's stream": lambda od, x: od.residual_norm(x, x, gate=x, return_stream=True)[1],
    "dropout": lambda od, x: od.dropout(x, 0.5, 5),
}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("enabled", [False, True])
def test_a_traced_call_runs_its_kernel(standin, name, wants_grad, enabled):
    """The traced module computes, for other values and another number of rows too; it does not hand out memory that was
    only allocated."""
    f = lambda x: CALLS[name](standin, x)                                       # noqa: E731
    with torch.set_grad_enabled(enabled):
        traced = torch.jit.trace(f, (torch.randn(4, 6, requires_grad=wants_grad),), check_trace=False)
        for rows in (4, 9):
            x = torch.randn(rows, 6)
            held = [torch.full((rows, c), 7.0) for c in (3, 6) for _ in range(20)]
            del held                                                            # (what fresh memory may hold)
            assert torch.equal(traced(x).detach(), f(x))


@pytest.mark.filterwarnings("ignore")
def test_a_traced_call_reads_its_seed_tensor_and_checks_its_arguments(standin):
    traced = torch.jit.trace(lambda x, s: standin.dropout(x, 0.5, s), (torch.zeros(2, 3), torch.tensor([4])), check_trace=False)
    assert (traced(torch.zeros(2, 3), torch.tensor([9])) == 9).all()
    traced = torch.jit.trace(lambda x, w: standin.linear(x, w), (torch.zeros(2, 6), W), check_trace=False)
    with pytest.raises(RuntimeError, match="does not fit x"):
        traced(torch.zeros(2, 6), torch.zeros(3, 5))


@pytest.mark.parametrize("name", CALLS)
def test_other_transforms_are_refused(standin, name):
    """An error instead of a result without the kernels' work."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = lambda x: CALLS[name](standin, x), torch.randn(4, 6)                 # noqa: E731
    want = f(x)
    for call in (make_fx(f), make_fx(f, pre_dispatch=True), make_fx(f, tracing_mode="fake"), torch.func.functionalize(f),
                 torch.func.vmap(f), torch.func.grad(lambda v: f(v).sum()), lambda v: torch.func.jvp(f, (v,), (v,))):
        with pytest.raises(RuntimeError):
            call(x)
    assert torch.equal(f(x), want)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
def test_a_traced_backward_is_refused(standin, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 6, requires_grad=True)
    y = CALLS[name](standin, x)
    dy = torch.ones_like(y)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(y, x, g)[0])(dy)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda v: torch.autograd.grad(CALLS[name](standin, v).sum(), v)[0], (x,), check_trace=False)


@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(standin, name):
    """Without a jvp the result would have no tangent, which reads as a derivative of zero."""
    from torch.autograd import forward_ad
    f, x = lambda x: CALLS[name](standin, x), torch.randn(4, 6)                 # noqa: E731
    want = f(x)
    with forward_ad.dual_level():
        assert torch.equal(f(x), want)                                          # no tangent, nothing to lose
        for primal in (x, x.clone().requires_grad_(True)):
            dual = forward_ad.make_dual(primal, torch.ones_like(x))
            for enabled in (True, False):
                with torch.set_grad_enabled(enabled), pytest.raises(NotImplementedError):
                    f(dual)
        leaf = x.clone().requires_grad_(True)
        y = f(leaf)
        with pytest.raises(RuntimeError, match="no tangent goes through"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_a_library_of_the_sampling_alone_loads(lib, monkeypatch, tmp_path):
    """What csrc/abl/build.sh makes has no dense operators; the sampling works from it, a dense call names what is missing."""
    import subprocess
    from opus_amd import _lib, opus_dense as od
    source, out = tmp_path / "sampling.c", tmp_path / "sampling.so"
    source.write_text("const char *opus_msmv_strerror(int code) { return code ? \"error\" : \"ok\"; }\n"
                      + "".join(f"int {n}(void) {{ return 0; }}\n" for n in _lib.SYMBOLS if n != "opus_msmv_strerror"))
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(out), str(source)])
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(out))
    assert _lib.load() is not lib and _lib.strerror(0) == "ok"
    monkeypatch.setattr(od, "_check", lambda *a: None)
    with pytest.raises(AttributeError, match="undefined symbol: opus_dense"):
        od.dropout(torch.zeros(2, 8), 0.5, 1)


def test_ablation_builds_have_every_source_of_the_sampling():
    csrc = os.path.join(ROOT, "opus_amd", "csrc")
    made = re.search(r"^MSMV = (.*)$", open(os.path.join(csrc, "Makefile")).read(), re.M).group(1).split()
    built = re.search(r'^SRCS="(.*)"$', open(os.path.join(csrc, "abl", "build.sh")).read(), re.M).group(1).split()
    assert sorted(built) == sorted(f"{name}.hip" for name in made)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
def test_compiled_functions_break_their_graph_at_a_call(standin, name):
    """torch.compile runs the call as it is, between what it makes of the rest."""
    f = torch.compile(lambda x: CALLS[name](standin, x + 1) * 2, backend="aot_eager")
    for rows in (4, 9):
        for wants_grad in (False, True):
            x = torch.randn(rows, 6, requires_grad=wants_grad)
            assert torch.equal(f(x).detach(), (CALLS[name](standin, x + 1) * 2).detach())
