"""Layer norm and its gradients (gpu_hip_layers.h) against the formulas in 64 bits on the same inputs.

Tolerances, with u the rounding of the sums' type (2^-24; f64 tensors 2^-53) and half the half step of the
output's type. A sum over n values is taken by up to 1024 threads, each adding at most n/1024 + 64 of them, then in
trees of at most 16 + 6 steps: its error is at most k u times the sum of the magnitudes, k = n/1024 + 90. The mean is
off by k u mean|x|, x - mean by that and u |x - mean|, the variance by (k + 2) u relative, 1/sqrt by half of that and
2 u; the products and the last sum add 3 u."""
import ctypes as C
import threading

import numpy as np
import pytest

import eshkol_amd as ea
from layer_util import BF16, F16, F32, F64, FLOOR, HALF, NAMES, Graph, Mat, close, room, run, unit, vec, wide

pytestmark = pytest.mark.gpu

TYPES = [(F64, F64), (F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
# every vector count per thread the kernels have, odd and even ends, rows of one and two elements
COLS = [1, 2, 7, 63, 64, 257, 511, 512, 1000, 1023, 2048, 4096, 4099, 8192, 16390, 33000]


def inputs(rows, cols, dtype, pdtype, seed=0, pad=0, shift=0):
    rng = np.random.default_rng([rows, cols, dtype, pdtype, seed])
    x = Mat((rows, cols), dtype, cols + pad, shift, rng.standard_normal((rows, cols)) * 1.5 + rng.standard_normal((rows, 1)))
    gamma = vec(1.0 + 0.3 * rng.standard_normal(cols), pdtype)
    beta = vec(0.3 * rng.standard_normal(cols), pdtype)
    return rng, x, gamma, beta


def forward(x, gamma, beta, dtype, pdtype, eps=1e-5, y=None, stats=True):
    rows, cols = x.shape
    y = y or Mat((rows, cols), dtype)
    mean, rstd = (Mat((rows,), wide(dtype)), Mat((rows,), wide(dtype))) if stats else (None, None)
    a = ea.HipLayerNormArgs(x=x.ptr, gamma=gamma and gamma.ptr, beta=beta and beta.ptr, y=y.ptr, mean=mean and mean.ptr, rstd=rstd and rstd.ptr,
                            rows=rows, cols=cols, ldx=x.ld, ldy=y.ld, epsilon=eps, dtype=dtype, param_dtype=pdtype)
    assert run(ea.load().hip_layernorm, a) == 0
    return y, mean, rstd


def check_forward(x, gamma, beta, y, mean, rstd, dtype, eps=1e-5):
    X = x.values
    rows, cols = X.shape
    g = gamma.values if gamma else np.ones(cols)
    b = beta.values if beta else np.zeros(cols)
    mu = X.mean(1, keepdims=True)
    d = X - mu
    with np.errstate(divide="ignore", invalid="ignore"):
        r = 1.0 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
        want = d * r * g + b
    u, k = unit(dtype), cols / 1024 + 90
    mag = np.abs(X).mean(1, keepdims=True)
    off_mean = k * u * mag
    # the variance is a mean of squares about a mean that is off_mean off
    rel_r = (k + 4) * u + (off_mean * r) ** 2
    close(mean.get(), mu[:, 0], (off_mean + u * np.abs(mu))[:, 0], "mean")
    close(rstd.get(), r[:, 0], (rel_r * r)[:, 0], "rstd")
    tol = np.abs(g) * r * (off_mean + u * np.abs(d)) + np.abs(g * d * r) * (rel_r + 3 * u) + 2 * u * (np.abs(b) + np.abs(want))
    close(y.get(), want, tol * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + FLOOR[dtype], "y")


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,pdtype", TYPES, ids=lambda t: NAMES[t])
def test_forward(gpu, dtype, pdtype, cols):
    rows = 5 if cols > 5000 else 37
    _, x, gamma, beta = inputs(rows, cols, dtype, pdtype)
    print("case: layernorm forward", NAMES[dtype], rows, cols, flush=True)
    y, mean, rstd = forward(x, gamma, beta, dtype, pdtype)
    check_forward(x, gamma, beta, y, mean, rstd, dtype)
    assert y.surroundings_untouched() and mean.surroundings_untouched() and rstd.surroundings_untouched()


@pytest.mark.parametrize("rows", [1, 2, 5, 1025, 20000])
def test_forward_row_counts(gpu, rows):
    _, x, gamma, beta = inputs(rows, 129, BF16, F32)
    y, mean, rstd = forward(x, gamma, beta, BF16, F32)
    check_forward(x, gamma, beta, y, mean, rstd, BF16)


@pytest.mark.parametrize("dtype", [F64, F32, F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("cols", [64, 333, 4100, 40000])
@pytest.mark.parametrize("pad,shift", [(5, 1), (8, 0), (1, 3)])
def test_pitches_and_starts_off_every_boundary(gpu, dtype, cols, pad, shift):
    rows = 4
    rng, x, _, _ = inputs(rows, cols, dtype, dtype, pad=pad, shift=shift)
    y = Mat((rows, cols), dtype, cols + 2 * pad + 1, shift + 1)
    y, mean, rstd = forward(x, None, None, dtype, dtype, y=y)
    check_forward(x, None, None, y, mean, rstd, dtype)
    assert y.surroundings_untouched()
    dy = Mat((rows, cols), dtype, cols + pad + 2, shift + 2, rng.standard_normal((rows, cols)))
    dx = Mat((rows, cols), dtype, cols + pad, 1)
    got = backward(dy, x, None, mean, rstd, dtype, dtype, dx=dx)
    check_backward(dy, x, None, mean, rstd, None, got, dtype)
    assert dx.surroundings_untouched()


def test_in_place_and_without_statistics(gpu):
    for cols in (100, 4096, 40000):
        _, x, gamma, beta = inputs(3, cols, BF16, BF16)
        y, mean, rstd = forward(x, gamma, beta, BF16, BF16)
        want = y.bits()
        forward(x, gamma, beta, BF16, BF16, y=x, stats=False)
        assert x.bits() == want and x.surroundings_untouched()


def test_constant_rows_and_large_means(gpu):
    # a row of one value: y is beta; a mean of 1000 beside deviations of 1 loses no more than its rounding
    x = Mat((3, 700), F32, values=np.concatenate([np.full((2, 700), 3.25), 1000.0 + np.random.default_rng(3).standard_normal((1, 700))]))
    beta = vec(np.linspace(-1, 1, 700), F32)
    y, mean, rstd = forward(x, None, beta, F32, F32)
    assert np.array_equal(y.get()[:2], np.broadcast_to(beta.values, (2, 700)))
    check_forward(x, None, beta, y, mean, rstd, F32)


@pytest.mark.parametrize("cols", [3, 41, 49, 1000, 3000, 4099, 5001, 16390, 33000, 100003])
@pytest.mark.parametrize("dtype", [F64, F32, F16, BF16], ids=lambda t: NAMES[t])
def test_a_row_of_one_value_has_that_mean(gpu, dtype, cols):
    """The first mean is off by at most k u of the value c, k the steps of its sum (at most cols / 1024 + 90). The deviations from it
    are exact and equal, their mean is k u of them off, so the corrected mean is c but for (k u)^2 c, less than a quarter of c's last
    place, and rounds to c: y is beta. The variance that is left is (k u c)^2 (2 k + 8) u."""
    u, k = unit(dtype), cols / 1024 + 90
    values = [1000.0, 4096.0, 0.1, 1.0, -3.7e4, 1e-3, 65504.0 / 3]
    x = Mat((len(values), cols), dtype, values=np.repeat(np.array(values)[:, None], cols, 1))
    c = x.values[:, 0]
    beta = vec(np.linspace(-2, 2, cols), dtype)
    y, mean, rstd = forward(x, None, beta, dtype, dtype)
    assert (k * u) ** 2 < u / 4
    assert np.array_equal(mean.get(), c)
    assert np.array_equal(y.get(), np.broadcast_to(beta.values, x.shape))
    want = 1e-5 ** -0.5
    close(rstd.get(), np.full(len(c), want), want * ((k * u * c) ** 2 * (2 * k + 8) * u / 2e-5 + 4 * u), "rstd")


@pytest.mark.parametrize("cols", [41, 700, 1000, 3000, 4099, 9000, 16390, 40000])
@pytest.mark.parametrize("dtype", [F64, F32, BF16], ids=lambda t: NAMES[t])
def test_statistics_beside_a_large_mean(gpu, dtype, cols):
    """Deviations of 1 about means of a thousand and more: the mean is rounded once, and beside that off by the sum of the deviations
    from the first mean, k + 3 roundings of their magnitudes; those are off themselves by the rounding of a difference."""
    rng = np.random.default_rng([cols, dtype])
    x = Mat((6, cols), dtype, values=np.array([[1000.0], [-1234.5], [3e4], [77.7], [1.0], [0.0]]) + rng.standard_normal((6, cols)))
    y, mean, rstd = forward(x, None, None, dtype, dtype)
    X = x.values
    mu = X.mean(1)
    u, k = unit(dtype), cols / 1024 + 90
    first = k * u * np.abs(X).mean(1)                    # how far the first mean may be off
    d = np.abs(X - mu[:, None]).mean(1) + first
    # u for the rounding, and 2^-53 of the 64-bit mean this is held to
    close(mean.get(), mu, u * np.abs(mu) + (k + 4) * u * d + 4 * 2.0 ** -53 * np.abs(X).mean(1), "mean")
    check_forward(x, None, None, y, mean, rstd, dtype)


def test_the_mean_of_a_row_with_an_infinity(gpu):
    """The sum's own: an infinity of its sign, NaN beside the other or a NaN; y of such a row is NaN."""
    for cols in (50, 3000, 40000):
        v = np.random.default_rng(cols).standard_normal((5, cols))
        v[0, 3], v[1, cols - 1], v[2, [1, 7]], v[3, 5] = np.inf, -np.inf, [np.inf, -np.inf], np.nan
        x = Mat((5, cols), F32, values=v)
        y, mean, rstd = forward(x, None, None, F32, F32)
        m = mean.get()
        assert m[0] == np.inf and m[1] == -np.inf and np.isnan(m[2:4]).all() and np.isfinite(m[4])
        assert np.isnan(y.get()[:4]).all() and np.isnan(rstd.get()[:4]).all() and np.isfinite(y.get()[4]).all()


def test_infinities_and_nan_stay_in_their_row(gpu):
    for cols in (50, 3000, 40000):
        rng = np.random.default_rng(cols)
        v = rng.standard_normal((6, cols))
        clean = v.copy()
        v[1, 7], v[3, cols - 1], v[4, 0] = np.inf, np.nan, -np.inf
        x, x0 = Mat((6, cols), BF16, values=v), Mat((6, cols), BF16, values=clean)
        y, mean, rstd = forward(x, None, None, BF16, BF16)
        y0, _, _ = forward(x0, None, None, BF16, BF16)
        got, want = y.get(), y0.get()
        assert np.array_equal(got[[0, 2, 5]], want[[0, 2, 5]]) and np.isnan(got[[1, 3, 4]]).all()


def test_no_rows(gpu):
    a = ea.HipLayerNormArgs(rows=0, cols=8, dtype=F32, param_dtype=F32, epsilon=1e-5)
    assert run(gpu.load().hip_layernorm, a) == 0
    gg, gb = Mat((8,), F32), Mat((8,), F32)
    b = ea.HipLayerNormBackwardArgs(rows=0, cols=8, dtype=F32, param_dtype=F32, grad_gamma=gg.ptr, grad_beta=gb.ptr)
    lib = gpu.load()
    assert run(lib.hip_layernorm_backward, b, lib.hip_layernorm_backward_workspace) == 0
    assert not gg.get().any() and not gb.get().any() and gg.surroundings_untouched()


# ---- backward ------------------------------------------------------------------------------------------

def backward(dy, x, gamma, mean, rstd, dtype, pdtype, res=None, dx=True, params=True, stream=None):
    rows, cols = x.shape
    lib = ea.load()
    dx = Mat((rows, cols), dtype) if dx is True else dx
    gg, gb = (Mat((cols,), wide(dtype)), Mat((cols,), wide(dtype))) if params else (None, None)
    a = ea.HipLayerNormBackwardArgs(grad_y=dy.ptr, x=x.ptr, gamma=gamma and gamma.ptr, mean=mean.ptr, rstd=rstd.ptr, grad_residual=res and res.ptr,
                                    grad_x=dx and dx.ptr, grad_gamma=gg and gg.ptr, grad_beta=gb and gb.ptr, rows=rows, cols=cols,
                                    ld_grad_y=dy.ld, ldx=x.ld, ld_grad_residual=res.ld if res else 0, ld_grad_x=dx.ld if dx else 0,
                                    dtype=dtype, param_dtype=pdtype)
    assert run(lib.hip_layernorm_backward, a, lib.hip_layernorm_backward_workspace, stream) == 0
    return dx, gg, gb


def check_backward(dy, x, gamma, mean, rstd, res, got, dtype, before=None):
    """mean and rstd are inputs here: the formula on them, as they were rounded."""
    DY, X = before or (dy.values, x.values)
    rows, cols = X.shape
    g = gamma.values if gamma else np.ones(cols)
    mu, r = mean.get()[:, None], rstd.get()[:, None]
    R = res.values if res else 0.0
    h = (X - mu) * r
    t = DY * g
    a, c = t.mean(1, keepdims=True), (t * h).mean(1, keepdims=True)
    u, k = unit(dtype), cols / 1024 + 90
    dx, gg, gb = got
    if dx:
        want = r * (t - a - h * c) + R
        # h is off by 2 u, t by u; a and c by their sums' errors; three more roundings of what is added
        tol = r * u * (4 * np.abs(t) + (k + 4) * np.abs(t).mean(1, keepdims=True) + np.abs(h) * (k + 8) * np.abs(t * h).mean(1, keepdims=True)) + 2 * u * np.abs(want) + u * np.abs(R)
        close(dx.get(), want, tol * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + FLOOR[dtype], "grad_x")
    if gg:
        # at most rows additions, each off by u of the running sum, and three roundings of a product
        close(gg.get(), (DY * h).sum(0), (rows + 4) * u * np.abs(DY * h).sum(0), "grad_gamma")
        close(gb.get(), DY.sum(0), (rows + 1) * u * np.abs(DY).sum(0), "grad_beta")


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,pdtype", TYPES, ids=lambda t: NAMES[t])
def test_backward(gpu, dtype, pdtype, cols):
    rows = 5 if cols > 5000 else 37
    rng, x, gamma, beta = inputs(rows, cols, dtype, pdtype, seed=1)
    _, mean, rstd = forward(x, gamma, beta, dtype, pdtype)
    dy = Mat((rows, cols), dtype, values=rng.standard_normal((rows, cols)))
    res = Mat((rows, cols), dtype, values=rng.standard_normal((rows, cols))) if cols % 2 else None
    print("case: layernorm backward", NAMES[dtype], rows, cols, flush=True)
    got = backward(dy, x, gamma, mean, rstd, dtype, pdtype, res)
    check_backward(dy, x, gamma, mean, rstd, res, got, dtype)
    assert all(m.surroundings_untouched() for m in got)


@pytest.mark.parametrize("rows", [1, 3, 511, 2049, 30000])
@pytest.mark.parametrize("cols", [33, 520])
def test_backward_row_counts(gpu, rows, cols):
    rng, x, gamma, beta = inputs(rows, cols, F16, F16, seed=2)
    _, mean, rstd = forward(x, gamma, beta, F16, F16)
    dy = Mat((rows, cols), F16, values=rng.standard_normal((rows, cols)))
    got = backward(dy, x, gamma, mean, rstd, F16, F16)
    check_backward(dy, x, gamma, mean, rstd, None, got, F16)


@pytest.mark.parametrize("cols", [40, 3000, 40000])
def test_backward_parts_and_in_place(gpu, cols):
    rows = 6
    rng, x, gamma, beta = inputs(rows, cols, BF16, F32, seed=3)
    _, mean, rstd = forward(x, gamma, beta, BF16, F32)
    vals = rng.standard_normal((rows, cols))
    dy = Mat((rows, cols), BF16, values=vals)
    res = Mat((rows, cols), BF16, values=rng.standard_normal((rows, cols)))
    whole = backward(dy, x, gamma, mean, rstd, BF16, F32, res)
    only_x = backward(dy, x, gamma, mean, rstd, BF16, F32, res, params=False)
    only_p = backward(dy, x, gamma, mean, rstd, BF16, F32, res, dx=None)
    assert only_x[0].bits() == whole[0].bits()
    assert only_p[1].bits() == whole[1].bits() and only_p[2].bits() == whole[2].bits()
    # grad_x over grad_residual, over grad_y, over x
    r2 = Mat((rows, cols), BF16, values=res.values)
    assert backward(dy, x, gamma, mean, rstd, BF16, F32, r2, dx=r2)[0].bits() == whole[0].bits()
    d2 = Mat((rows, cols), BF16, values=vals)
    assert backward(d2, x, gamma, mean, rstd, BF16, F32, res, dx=d2)[0].bits() == whole[0].bits()
    x2 = Mat((rows, cols), BF16, values=x.values)
    assert backward(dy, x2, gamma, mean, rstd, BF16, F32, res, dx=x2)[0].bits() == whole[0].bits()


def test_gradient_against_differences(gpu):
    """The f64 gradients against central differences of the f64 forward pass: with a step e of 1e-5 the quotient
    is off by e^2 times a third derivative (some tens here) and by 2^-53 / e of the loss's size (about 100)."""
    rows, cols, e = 3, 37, 1e-5
    rng, x, gamma, beta = inputs(rows, cols, F64, F64, seed=4)
    dyv = rng.standard_normal((rows, cols))
    dy = Mat((rows, cols), F64, values=dyv)

    def loss(X, G, B):
        y, _, _ = forward(Mat((rows, cols), F64, values=X), vec(G, F64), vec(B, F64), F64, F64)
        return float((y.get() * dyv).sum())

    _, mean, rstd = forward(x, gamma, beta, F64, F64)
    dx, gg, gb = backward(dy, x, gamma, mean, rstd, F64, F64)
    X, G, B = x.values, gamma.values, beta.values
    for i, j in ((0, 0), (1, 17), (2, 36)):
        for base, grad, at in ((X, dx.get(), (i, j)), (G, gg.get(), (j,)), (B, gb.get(), (j,))):
            hi, lo = base.copy(), base.copy()
            hi[at] += e
            lo[at] -= e
            pick = lambda v: [v if base is b else b for b in (X, G, B)]  # noqa: E731
            assert abs((loss(*pick(hi)) - loss(*pick(lo))) / (2 * e) - grad[at]) < 100 * e * e + 100 * 2.0 ** -53 / e * 4


# ---- streams, graphs, threads ---------------------------------------------------------------------------

def test_same_bits_every_time_and_on_another_stream(gpu):
    rng, x, gamma, beta = inputs(700, 1030, BF16, BF16, seed=5)
    _, mean, rstd = forward(x, gamma, beta, BF16, BF16)
    dy = Mat((700, 1030), BF16, values=rng.standard_normal((700, 1030)))
    first = [m.bits() for m in backward(dy, x, gamma, mean, rstd, BF16, BF16)]
    st = C.c_void_p()
    assert ea.hip_runtime().hipStreamCreate(C.byref(st)) == 0
    for stream in (None, st, 0):
        assert [m.bits() for m in backward(dy, x, gamma, mean, rstd, BF16, BF16, stream=stream)] == first
    ea.hip_runtime().hipStreamDestroy(st)


def test_captured_forward_and_backward_replay(gpu):
    lib = gpu.load()
    rows, cols = 130, 700
    rng, x, gamma, beta = inputs(rows, cols, F16, F32, seed=6)
    y, mean, rstd, dx = Mat((rows, cols), F16), Mat((rows,), F32), Mat((rows,), F32), Mat((rows, cols), F16)
    dy = Mat((rows, cols), F16, values=rng.standard_normal((rows, cols)))
    gg, gb = Mat((cols,), F32), Mat((cols,), F32)
    f = ea.HipLayerNormArgs(x=x.ptr, gamma=gamma.ptr, beta=beta.ptr, y=y.ptr, mean=mean.ptr, rstd=rstd.ptr, rows=rows, cols=cols, epsilon=1e-5, dtype=F16, param_dtype=F32)
    b = ea.HipLayerNormBackwardArgs(grad_y=dy.ptr, x=x.ptr, gamma=gamma.ptr, mean=mean.ptr, rstd=rstd.ptr, grad_x=dx.ptr, grad_gamma=gg.ptr, grad_beta=gb.ptr,
                                    rows=rows, cols=cols, dtype=F16, param_dtype=F32)
    need = lib.hip_layernorm_backward_workspace(C.byref(b))
    ws = room(need)
    b.workspace, b.workspace_bytes = ws.ptr, need
    graph = Graph()
    with graph as st:
        assert lib.hip_layernorm(C.byref(f), st) == 0 and lib.hip_layernorm_backward(C.byref(b), st) == 0
    for turn in range(3):
        vals = rng.standard_normal((rows, cols)) * (turn + 1)
        x2 = Mat((rows, cols), F16, values=vals)
        x.host[:] = x2.host
        x.dev.upload(x.host.view(np.uint8))
        graph.replay()
        want = forward(x2, gamma, beta, F16, F32)
        check_forward(x2, gamma, beta, *want, F16)
        back = backward(dy, x2, gamma, want[1], want[2], F16, F32)
        for got, ref in zip((y, mean, rstd, dx, gg, gb), want + back):
            assert got.bits() == ref.bits(), turn
    graph.close()


def test_two_threads_at_once(gpu):
    made = []
    for seed in (7, 8):
        rng, x, gamma, beta = inputs(900, 520, BF16, BF16, seed=seed)
        _, mean, rstd = forward(x, gamma, beta, BF16, BF16)
        dy = Mat((900, 520), BF16, values=rng.standard_normal((900, 520)))
        made.append((dy, x, gamma, mean, rstd))
    want = [[m.bits() for m in backward(*m, BF16, BF16)] for m in made]
    got = [None, None]

    def work(i):
        st = C.c_void_p()
        ea.hip_runtime().hipStreamCreate(C.byref(st))
        got[i] = [[m.bits() for m in backward(*made[i], BF16, BF16, stream=st)] for _ in range(5)]
        ea.hip_runtime().hipStreamDestroy(st)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert got == [[want[0]] * 5, [want[1]] * 5]
