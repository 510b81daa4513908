"""The linear layer with bias, activation and residual in its epilogue, the products by expert, and the gradients of
both (gpu_hip_layers.h), against the formulas in 64 bits on the same inputs.

Tolerances, u = 2^-24. Products of two 16-bit values are exact in fp32; n of them are added in some order, each addition
off by at most 2 u of the running sum (whether the matrix cores round or cut): 2 (n + 8) u times the sum of magnitudes.
The activations are off by u (24 + 2 |z| + 2 z^2) relative (an exponential's argument is off by u of itself; the
argument is z or z^2 / 2), gelu by 3.7e-6 = 62 u more (the fit of the normal integral that its kernel states), and pass
an error of z on by at most 1.13. A rounding to the output's type is off by half a
step. dz enters the products rounded to the 16-bit type (half a step of each value) unless there is no activation."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import eshkol_amd as ea
from conftest import ROOT
from layer_util import BF16, F16, F32, FLOOR, HALF, NAMES, Graph, Mat, act, close, decode, encode, room, run, slope, vec

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = [0, 1, 2, 3, 4]


def act_error(z, code):
    return 0.0 if code in (0, 2) else U * (24 + (62 if code == 3 else 0) + 2 * np.abs(z) + 2 * z * z)


class Layer:
    """A layer's tensors; offsets: the groups of its experts (None: a linear layer)."""

    def __init__(self, M, K, N, dtype, trans=0, code=0, param=None, offsets=None, residual=False, pad=0, shift=0, seed=0, bias=True):
        self.M, self.K, self.N, self.dtype, self.trans, self.code = M, K, N, dtype, trans, code
        self.param = dtype if param is None else param
        self.offsets = None if offsets is None else np.asarray(offsets, dtype=np.int32)
        E = self.E = 1 if offsets is None else len(offsets) - 1
        rng = np.random.default_rng([M, K, N, dtype, trans, code, E, seed])
        mat = lambda shape, s=1.0: Mat(shape, dtype, shape[-1] + pad, shift, rng.standard_normal(shape) * s)  # noqa: E731
        self.x = mat((M, K))
        self.w = mat((E, N, K) if trans else (E, K, N), K ** -0.5)
        self.bias = vec(rng.standard_normal((E, N)) * 0.5, self.param) if bias else None
        self.residual = mat((M, N)) if residual else None
        self.dy = mat((M, N))
        self.pre = mat((M, N), 1.5) if code else None
        self.pad, self.shift = pad, shift
        self.doff = ea.DeviceArray.from_host(self.offsets) if offsets is not None else None

    def groups(self):
        return [(0, self.M)] if self.offsets is None else list(zip(self.offsets[:-1], self.offsets[1:]))

    def W(self):
        """The experts' matrices as [K][N] each."""
        w = self.w.values
        return w.transpose(0, 2, 1) if self.trans else w

    def out(self, shape, dtype=None):
        dtype = self.dtype if dtype is None else dtype
        return Mat(shape, dtype, shape[-1] + (self.pad + 1 if self.pad else 0), self.shift)

    def forward(self, y=None, pre=True, stream=None):
        lib = ea.load()
        y = y or self.out((self.M, self.N))
        z = self.out((self.M, self.N)) if pre else None
        common = dict(x=self.x.ptr, w=self.w.ptr, bias=self.bias and self.bias.ptr, y=y.ptr, pre=z and z.ptr, K=self.K, N=self.N, ldx=self.x.ld, ldw=self.w.ld,
                      ldy=y.ld, ld_pre=z.ld if z else 0, dtype=self.dtype, param_dtype=self.param, act=self.code, trans_w=self.trans)
        if self.offsets is None:
            a = ea.HipLinearArgs(**common, M=self.M, residual=self.residual and self.residual.ptr, ld_residual=self.residual.ld if self.residual else 0)
            rc = run(lib.hip_linear_16, a, lib.hip_linear_16_workspace, stream)
        else:
            a = ea.HipExpertsArgs(**common, rows=self.M, experts=self.E, offsets=self.doff.ptr)
            rc = run(lib.hip_experts_16, a, lib.hip_experts_16_workspace, stream)
        assert rc == 0
        return y, z

    def check_forward(self, y, z, note="", residual=None):
        got_y, got_z = y.get(), z.get() if z else None
        every_x, every_w = self.x.values, self.W()
        every_bias = self.bias.values.reshape(self.E, self.N) if self.bias else np.zeros((self.E, self.N))
        every_r = None if self.residual is None else (self.residual.values if residual is None else residual)
        for e, (a, b) in enumerate(self.groups()):
            X, W, bias = every_x[a:b], every_w[e], every_bias[e]
            want = X @ W + bias
            err = 2 * (self.K + 8) * U * (np.abs(X) @ np.abs(W)) + 2 * U * (np.abs(want) + np.abs(bias))
            if z:
                close(got_z[a:b], want, err * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(want) + FLOOR[self.dtype], note + " pre, expert %d" % e)
            f = act(want, self.code)
            r = 0.0 if every_r is None else every_r[a:b]
            err = 1.13 * err + act_error(want, self.code) * np.abs(f) + 2 * U * (np.abs(f) + np.abs(r))
            close(got_y[a:b], f + r, err * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(f + r) + FLOOR[self.dtype], note + " y, expert %d" % e)
        for m in (y, z):
            assert m is None or self.others_untouched(m), note
        return True

    def others_untouched(self, m):
        """Rows of no expert, and everything around the matrix, are as they were."""
        mine = np.zeros(self.M, bool)
        for a, b in self.groups():
            mine[a:b] = True
        a, b = m.raw().copy(), m.host.copy()
        m.inner(a)[mine] = 0
        m.inner(b)[mine] = 0
        return a.tobytes() == b.tobytes()

    def backward(self, wtype=None, want="xwb", stream=None):
        lib = ea.load()
        wtype = self.dtype if wtype is None else wtype
        gx = self.out((self.M, self.K)) if "x" in want else None
        gw = self.out(self.w.shape, wtype) if "w" in want else None
        gb = Mat((self.E, self.N), F32) if "b" in want else None
        common = dict(grad_y=self.dy.ptr, pre=self.pre and self.pre.ptr, x=self.x.ptr, w=self.w.ptr, grad_x=gx and gx.ptr, grad_w=gw and gw.ptr, grad_bias=gb and gb.ptr,
                      K=self.K, N=self.N, ld_grad_y=self.dy.ld, ld_pre=self.pre.ld if self.pre else 0, ldx=self.x.ld, ldw=self.w.ld, ld_grad_x=gx.ld if gx else 0,
                      ld_grad_w=gw.ld if gw else 0, dtype=self.dtype, grad_w_dtype=wtype, act=self.code, trans_w=self.trans)
        if self.offsets is None:
            a = ea.HipLinearBackwardArgs(**common, M=self.M)
            rc = run(lib.hip_linear_backward_16, a, lib.hip_linear_backward_16_workspace, stream)
        else:
            a = ea.HipExpertsBackwardArgs(**common, rows=self.M, experts=self.E, offsets=self.doff.ptr)
            rc = run(lib.hip_experts_backward_16, a, lib.hip_experts_backward_16_workspace, stream)
        assert rc == 0
        return gx, gw, gb

    def check_backward(self, gx, gw, gb, wtype=None, note=""):
        wtype = self.dtype if wtype is None else wtype
        DY, X = self.dy.values, self.x.values
        if self.code:
            Z = self.pre.values
            s = slope(Z, self.code)
            DZ = DY * s
            raw = np.abs(DY) * (0.0 if self.code == 2 else U * (24 + 2 * np.abs(Z) + 2 * Z * Z) * 1.2) + U * np.abs(DZ)
            cut = raw + HALF[self.dtype] * np.abs(DZ) + FLOOR[self.dtype]
        else:
            DZ, raw, cut = DY, np.zeros_like(DY), np.zeros_like(DY)
        got_x = gx.get() if gx else None
        got_w = gw.get().reshape(self.w.shape) if gw else None
        got_b = gb.get() if gb else None
        every_w = self.W()
        for e, (a, b) in enumerate(self.groups()):
            W, d, x, c = every_w[e], DZ[a:b], X[a:b], cut[a:b]
            if gx:
                want = d @ W.T
                err = c @ np.abs(W.T) + 2 * (self.N + 8) * U * (np.abs(d) @ np.abs(W.T))
                close(got_x[a:b], want, err * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(want) + FLOOR[self.dtype], note + " grad_x, expert %d" % e)
            if gw:
                want = x.T @ d
                err = np.abs(x.T) @ c + 2 * (b - a + 8) * U * (np.abs(x.T) @ np.abs(d))
                g = got_w[e].T if self.trans else got_w[e]
                close(g, want, err * (1 + HALF[wtype]) + HALF[wtype] * np.abs(want) + FLOOR[wtype], note + " grad_w, expert %d" % e)
            if gb:
                close(got_b[e], d.sum(0), raw[a:b].sum(0) + (b - a + 8) * U * np.abs(d).sum(0), note + " grad_bias, expert %d" % e)
        if gx:
            assert self.others_untouched(gx), note
        for m in (gw, gb):
            assert m is None or m.surroundings_untouched(), note


# ---- the linear layer -----------------------------------------------------------------------------------------

# one row; the ends of the kernels for few rows (16, 32, 64); one tile, its neighbours; several; k and n of one, of no
# multiple of eight, of whole blocks; long k beside few tiles (cut and joined)
SIZES = [(1, 1, 1), (1, 64, 128), (1, 4096, 300), (2, 100, 9), (16, 65, 257), (17, 8, 8), (33, 1000, 129), (64, 200, 1000), (65, 1, 1), (65, 64, 128),
         (66, 7, 130), (128, 128, 128), (129, 72, 136), (130, 1001, 127), (300, 264, 520), (70, 5000, 40), (257, 512, 384)]


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_forward(gpu, size, dtype, trans):
    code = (size[0] + size[2] + trans) % 5
    print("case: linear forward", size, NAMES[dtype], trans, code, flush=True)
    t = Layer(*size, dtype, trans, code, residual=size[1] % 2 == 0)
    t.check_forward(*t.forward())


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_backward(gpu, size, dtype, trans):
    code = (size[0] + size[1] + trans) % 5
    wtype = F32 if size[2] % 2 else dtype
    print("case: linear backward", size, NAMES[dtype], trans, code, flush=True)
    t = Layer(*size, dtype, trans, code)
    t.check_backward(*t.backward(wtype), wtype)


# K whole in a workgroup (1 to 4 rows, 16 with W [N][K]); tiles of 32 and of 64 rows, with k in parts
FEW = [(1, 4096, 3000), (4, 1000, 2760), (3, 137, 4099), (2, 2304, 2731), (16, 520, 1400), (5, 4100, 1536), (11, 65, 1501), (20, 128, 3008), (32, 1096, 256),
       (48, 2048, 136), (64, 264, 1416), (40, 72, 8)]


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("size", FEW, ids=str)
def test_few_rows(gpu, size, dtype, trans):
    print("case: few rows", size, NAMES[dtype], trans, flush=True)
    t = Layer(*size, dtype, trans, size[1] % 5, residual=True, seed=9)
    t.check_forward(*t.forward())
    t.check_backward(*t.backward(F32), F32)


# products that take each of the tiles: 256 x 256; 128 x 256, one and two on a CU; 128 x 128, three on a CU and alone
TILES = [(3600, 200, 3592), (2000, 136, 3000), (2816, 96, 3100), (2432, 104, 2400), (1000, 330, 1100)]


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("size", TILES, ids=str)
def test_every_tile_forward(gpu, size, trans):
    print("case: tiles forward", size, trans, flush=True)
    t = Layer(*size, BF16 if trans else F16, trans, 4, residual=True)
    t.check_forward(*t.forward())


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("size", [(2000, 3000, 1999), (1300, 2100, 1500), (2900, 1500, 1504), (1900, 1040, 1000), (900, 600, 1300)], ids=str)
def test_every_tile_backward(gpu, size, trans):
    print("case: tiles backward", size, trans, flush=True)
    t = Layer(*size, F16 if trans else BF16, trans, 0 if trans else 1)
    t.check_backward(*t.backward())


@pytest.mark.parametrize("code", ACTS)
@pytest.mark.parametrize("M", [20, 100])
@pytest.mark.parametrize("param", [BF16, F32])
def test_every_activation(gpu, code, M, param):
    t = Layer(M, 96, 200, BF16, 0, code, param, residual=True, seed=1)
    t.check_forward(*t.forward())
    for wtype in (BF16, F32):
        t.check_backward(*t.backward(wtype), wtype)


@pytest.mark.parametrize("code", ACTS)
def test_activations_far_out(gpu, code):
    """Sums before the activation from -60 to 60, and at 0: x W is the bias's size times zero."""
    N = 1024
    t = Layer(3, 8, N, BF16, 0, code, F32)
    t.x = Mat((3, 8), BF16, values=np.zeros((3, 8)))
    z = np.concatenate([np.linspace(-60, 60, N - 10), [0.0, -0.0, 1e-6, -1e-6, 0.25, -0.25, 0.2499, 1e-20, 88.0, -88.0]])
    t.bias = vec(z[None], F32)
    y, pre = t.forward()
    z = t.bias.values[0]
    f = act(z, code)
    # an exponential below 2^-126 is flushed: one more such step
    tol = (act_error(z, code) + HALF[BF16]) * np.abs(f) * (1 + HALF[BF16]) + 100 * 2.0 ** -126
    close(y.get(), np.broadcast_to(f, (3, N)), tol, "y")
    t = Layer(3, 8, N, BF16, 0, code, F32)
    if code:
        t.pre = Mat((3, N), BF16, values=np.broadcast_to(z, (3, N)))
    _, _, gb = t.backward(want="b")
    t.check_backward(None, None, gb)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("M", [1, 100])
def test_gelu_rounds_to_the_neighbour_the_formula_does(gpu, M, dtype):
    """z Phi(z) of 2^16 sums known exactly (x is 0, so z is the fp32 bias): y is what some value within the evaluation's error of
    the formula rounds to. That error, relative, in u: the rounding of 1 + p a and its reciprocal 3, passed on at most twofold; the
    polynomial's steps 8; the fit 1.5; three products and the hardware's 2^x 6; the last addition 1; the exponent's two roundings
    1.5 z^2. Together at most 24 + 2 z^2."""
    N = 1 << 16
    t = Layer(M, 8, N, dtype, 0, 3, F32, bias=False)
    t.x = Mat((M, 8), dtype, values=np.zeros((M, 8)))
    t.bias = vec(np.random.default_rng(M).uniform(-4, 4, N)[None], F32)
    z = t.bias.values[0]
    y, _ = t.forward(pre=False)
    f = act(z, 3)
    off = (24 + 2 * z * z) * U * np.abs(f)
    least, most = decode(encode(f - off, dtype), dtype), decode(encode(f + off, dtype), dtype)
    got = y.get()
    bad = (got < least) | (got > most)
    assert not bad.any(), "%d of %d values rounded from too far" % (bad.sum(), bad.size)


def test_the_slope_of_a_saturated_tanh_keeps_its_digits(gpu):
    """grad_bias of one row is grad_y act'(pre): relative to 1 / cosh^2 z. The derivative is 4 e r^2, e = exp(-2 |z|),
    r = 1 / (1 + e): e is off by 4 |z| u (two roundings of the exponent) and 2 u, r by 3 u, the products by 2 u and the one
    with grad_y by u: 4 |z| + 11, allowed 4 |z| + 16."""
    for dtype in (F16, BF16):
        z = np.linspace(0, 40, 641)
        z = decode(encode(np.concatenate([z, -z]), dtype), dtype)
        for M in (1, 3):
            t = Layer(M, 8, len(z), dtype, 0, 1, F32)
            dy = np.zeros((M, len(z)))
            dy[M - 1] = 1.5
            t.dy = Mat(dy.shape, dtype, values=dy)
            t.pre = Mat(dy.shape, dtype, values=np.broadcast_to(z, dy.shape))
            got = t.backward(want="b")[2].get()[0]
            want = 1.5 / np.cosh(z) ** 2
            close(got, want, (4 * np.abs(z) + 16) * U * want, "slope of tanh, %s" % NAMES[dtype])


def test_activations_at_the_ends_of_the_range(gpu):
    """Sums of +-infinity, of the type's largest value and NaN: the limits, and NaN."""
    big = 3.3895313892515355e38
    z = np.array([np.inf, -np.inf, big, -big, np.nan, 200.0, -200.0, 14.0, -14.0])
    limits = {0: z, 1: np.array([1, -1, 1, -1, np.nan, 1, -1, 1, -1]), 2: np.array([np.inf, 0, big, 0, np.nan, 200, 0, 14, 0])}
    limits[3] = limits[4] = limits[2]
    flat = {1: np.array([0, 0, 0, 0, np.nan, 0, 0, 0, 0]), 2: np.array([1, 0, 1, 0, np.nan, 1, 0, 1, 0])}
    flat[3] = flat[4] = flat[2]
    for code in ACTS:
        for M in (4, 70):
            t = Layer(M, 8, len(z), BF16, 0, code, F32)
            t.x = Mat((M, 8), BF16, values=np.zeros((M, 8)))
            t.bias = vec(z[None], F32)
            y = t.forward()[0].get()
            # the bf16 nearest to 14 and 200 are exact; tanh(14) and Phi(14) are 1 to 12 digits, z Phi(z) at -14 is 1e-43
            tol = 1e-11 + HALF[BF16] * np.nan_to_num(np.abs(limits[code]), nan=0, posinf=0) * (np.abs(z) > 1e30)
            close(y, np.broadcast_to(limits[code], y.shape), np.broadcast_to(tol + (1.2e-5 if code == 4 else 0), y.shape), "act %d" % code)
        if code:
            t = Layer(1, 8, len(z), BF16, 0, code, F32)
            t.dy = Mat((1, len(z)), BF16, values=np.ones((1, len(z))))
            t.pre = Mat((1, len(z)), BF16, values=z[None])
            got = t.backward(want="b")[2].get()
            close(got, flat[code][None], 1.2e-5, "slope %d" % code)


def test_infinities_and_nan_reach_their_rows_and_columns_alone(gpu):
    for M in (5, 100):
        for trans in (0, 1):
            t = Layer(M, 72, 136, BF16, trans, 0)
            x = t.x.values
            x[3, 71], x[1, 0] = np.inf, np.nan
            t.x = Mat((M, 72), BF16, values=x)
            y, _ = t.forward()
            got = y.get()
            rows = np.isfinite(got).all(1)
            assert not np.isfinite(got[[1, 3]]).any() and rows.sum() == M - 2
            w = t.w.values
            w[0, 5, 70 if trans else 135] = -np.inf
            t = Layer(M, 72, 136, BF16, trans, 0)
            t.w = Mat(w.shape, BF16, values=w)
            got = t.forward()[0].get()
            cols = np.isfinite(got).all(0)
            assert cols.sum() == 135 and not np.isfinite(got[:, 5 if trans else 135]).any()


@pytest.mark.parametrize("M", [1, 40, 140])
@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("pad,shift", [(8, 8), (8, 1), (3, 0), (5, 3)])
def test_pitches_and_starts(gpu, M, trans, pad, shift):
    t = Layer(M, 136, 152, F16, trans, 3, residual=True, pad=pad, shift=shift)
    t.check_forward(*t.forward())
    t.check_backward(*t.backward(F32), F32)


def test_y_over_residual_and_no_pre(gpu):
    for M in (7, 90, 200):
        t = Layer(M, 640, 96, BF16, 0, 4, residual=True)
        want, _ = t.forward()
        r = t.residual.values
        y, _ = t.forward(y=t.residual, pre=False)
        assert y.bits() == want.bits()
        t.check_forward(y, None, residual=r)


def test_parts_of_the_gradients(gpu):
    for M in (9, 150):
        t = Layer(M, 88, 104, BF16, 1, 1)
        whole = [m.bits() for m in t.backward()]
        for i, want in enumerate("xwb"):
            part = t.backward(want=want)
            assert part[i].bits() == whole[i], want
        t = Layer(M, 88, 104, BF16, 0, 0, seed=1)
        t.check_backward(*t.backward(want="xw"))
        t.check_backward(*t.backward(want="b"))


def test_no_rows(gpu):
    lib = gpu.load()
    a = ea.HipLinearArgs(M=0, K=4, N=4, dtype=F16, param_dtype=F16)
    assert run(lib.hip_linear_16, a, lib.hip_linear_16_workspace) == 0
    for trans in (0, 1):
        for wtype in (F32, BF16):
            gw, gb = Mat((20, 36), wtype, 41), Mat((20 if trans else 36,), F32)
            b = ea.HipLinearBackwardArgs(M=0, K=36 if trans else 20, N=20 if trans else 36, dtype=BF16, grad_w_dtype=wtype, act=3, trans_w=trans,
                                         grad_w=gw.ptr, grad_bias=gb.ptr, ld_grad_w=gw.ld)
            assert run(lib.hip_linear_backward_16, b, lib.hip_linear_backward_16_workspace) == 0
            assert not gw.get().any() and not gb.get().any() and gw.surroundings_untouched() and gb.surroundings_untouched()
    gw, gb = Mat((3, 20, 36), BF16), Mat((3, 36), F32)
    e = ea.HipExpertsBackwardArgs(rows=0, experts=3, K=20, N=36, dtype=BF16, grad_w_dtype=BF16, grad_w=gw.ptr, grad_bias=gb.ptr)
    assert run(lib.hip_experts_backward_16, e, lib.hip_experts_backward_16_workspace) == 0
    assert not gw.get().any() and not gb.get().any()


@pytest.mark.parametrize("pad,shift", [(0, 0), (5, 3)])
def test_the_same_call_gives_the_same_bits_where_k_is_cut(gpu, pad, shift):
    """150 x 1024 x 4096: grad_x by itself is cut along K, beside grad_w it is not. Every choice of outputs repeats to the bit and
    is within the tolerances, whichever order it adds in."""
    t = Layer(150, 1024, 4096, BF16, 0, 4, pad=pad, shift=shift)
    first = [m.bits() for m in t.forward()]
    for want in ("xwb", "x", "w", "xb"):
        got = t.backward(F32, want)
        t.check_backward(*got, F32, note=want)
        again = t.backward(F32, want)
        assert [m and m.bits() for m in again] == [m and m.bits() for m in got], want
    assert [m.bits() for m in t.forward()] == first


class Far:
    """A matrix whose rows are so far apart that only its rows are ever on the host."""

    def __init__(self, values, dtype, ld):
        self.shape, self.dtype, self.ld = values.shape, dtype, ld
        self.dev = ea.DeviceArray((((values.shape[0] - 1) * ld + values.shape[1]) * 2,), np.uint8)
        self.ptr = self.dev.ptr
        self.rows = [encode(v, dtype) for v in values]
        for i, r in enumerate(self.rows):
            assert ea.hip_runtime().hipMemcpy(self.ptr + i * ld * 2, r.ctypes.data, r.nbytes, ea.H2D) == 0
        self.values = np.stack([decode(r, dtype) for r in self.rows])

    def get(self):
        out = []
        for i in range(self.shape[0]):
            r = np.empty(self.shape[1], np.uint16 if self.dtype == BF16 else np.float16)
            assert ea.hip_runtime().hipMemcpy(r.ctypes.data, self.ptr + i * self.ld * 2, r.nbytes, ea.D2H) == 0
            out.append(decode(r, self.dtype))
        return np.stack(out)


@pytest.mark.parametrize("M,ld", [(40, 1 << 26), (70, (1 << 22) + 8), (70, 1 << 25)])
def test_rows_far_apart(gpu, M, ld):
    """Element offsets past 32 bits in x, y and the residual, and pitches beyond what the tiled kernel reads itself."""
    t = Layer(M, 72, 40, BF16, 0, 2, residual=True)
    t.x, t.residual = Far(t.x.values, BF16, ld), Far(t.residual.values, BF16, ld)
    y = Far(np.zeros((M, 40)), BF16, ld)
    t.others_untouched = lambda m: True
    t.check_forward(*t.forward(y=y, pre=False))


@pytest.mark.parametrize("M", [30, 200])
def test_experts_far_apart(gpu, M):
    """Three experts' matrices 2^31 elements apart."""
    lib = gpu.load()
    t = Layer(M, 64, 48, F16, 0, 0, offsets=[0, 7, 7, M])
    stride = 1 << 31
    big = ea.DeviceArray(((2 * stride + 64 * 48) * 2,), np.uint8)
    for e in range(3):
        w = encode(t.w.values[e], F16)
        assert ea.hip_runtime().hipMemcpy(big.ptr + e * stride * 2, w.ctypes.data, w.nbytes, ea.H2D) == 0
    y = t.out((M, 48))
    a = ea.HipExpertsArgs(x=t.x.ptr, w=big.ptr, bias=t.bias.ptr, offsets=t.doff.ptr, y=y.ptr, rows=M, experts=3, K=64, N=48, w_stride=stride, dtype=F16, param_dtype=F16)
    assert run(lib.hip_experts_16, a, lib.hip_experts_16_workspace) == 0
    t.check_forward(y, None)


# ---- the products by expert -------------------------------------------------------------------------------------

# (rows, offsets): one expert; empty ones first, last, between; one row each; one with everything; more than 64 experts;
# rows of no expert in front and behind; groups that end on, before and behind a tile's edge; many rows (the tiled kernel)
GROUPS = [(5, [0, 5]), (6, [0, 0, 6, 6]), (3, [0, 1, 2, 3]), (40, [0, 0, 0, 40, 40]), (20, [3, 5, 5, 11]), (7, [0, 0, 0]), (200, list(range(0, 132, 2)) + [200]),
          (300, [0, 128, 256, 300]), (500, [0, 127, 127, 256, 500]), (700, [10, 150, 151, 430, 600]), (1300, [0] * 20 + [600] * 30 + [1299]),
          # a thousand experts, most of them without rows
          (400, [0] * 500 + [3] * 200 + [200] * 200 + [399] * 101),
          # enough tiles for the wide ones; 17 to 64 rows on average, aligned and not
          (5001, list(range(0, 5001, 100)) + [5001]), (1301, list(range(0, 1301, 26)) + [1301]), (1302, list(range(0, 1302, 26)) + [1302])]


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("group", GROUPS, ids=lambda g: "%d rows, %d experts" % (g[0], len(g[1]) - 1))
def test_experts(gpu, group, dtype, trans):
    rows, offsets = group
    K, N = (72, 200) if rows % 2 else (130, 77)
    code = (rows + trans) % 5
    print("case: experts", rows, offsets, NAMES[dtype], trans, code, flush=True)
    t = Layer(rows, K, N, dtype, trans, code, offsets=offsets)
    # rows of no expert hold what would spoil anything it reached
    free = np.ones(rows, bool)
    for a, b in t.groups():
        free[a:b] = False
    for name in ("x", "dy", "pre"):
        m = getattr(t, name)
        if m is not None and free.any():
            v = m.values
            v[free] = np.nan
            setattr(t, name, Mat(v.shape, dtype, values=v))
    t.check_forward(*t.forward())
    wtype = F32 if trans else dtype
    t.check_backward(*t.backward(wtype), wtype)


@pytest.mark.parametrize("rows", [30, 900])
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 1)])
def test_experts_pitches_and_long_k(gpu, rows, pad, shift):
    t = Layer(rows, 1100, 136, BF16, 0, 4, F32, offsets=[0, rows // 3, rows // 2, rows // 2, rows], pad=pad, shift=shift)
    t.check_forward(*t.forward())
    t.check_backward(*t.backward())


def test_an_expert_is_a_linear_layer(gpu):
    """The same rows alone and as one group among others: the same formulas (not the same bits: the kernels differ)."""
    t = Layer(100, 256, 128, BF16, 0, 3, offsets=[0, 0, 100, 100])
    y, _ = t.forward()
    one = Layer(100, 256, 128, BF16, 0, 3)
    one.x, one.w, one.bias = t.x, Mat((1, 256, 128), BF16, values=t.w.values[1:2]), vec(t.bias.values[1:2], BF16)
    z, _ = one.forward()
    close(y.get(), z.get(), 2 * HALF[BF16] * np.abs(z.get()) + 1e-3, "y")          # 2 (256 + 8) u times magnitudes of about 20, twice


# ---- whole numbers ------------------------------------------------------------------------------------------------

# (rows, K, N, offsets): every kernel and cut: K whole in a workgroup, the streaming kernel with parts, tiles of 32 and 64 rows, the
# larger tiles, with K cut and whole, blocks that end inside; experts of few rows, of many, with none
WHOLE = [(1, 4096, 3000, None), (3, 4099, 2800, None), (2, 4096, 520, None), (13, 5000, 264, None), (30, 4104, 264, None), (60, 4096, 136, None), (37, 4101, 130, None),
         (130, 4097, 200, None), (300, 2056, 520, None), (2048, 264, 1536, None), (2300, 200, 2304, None), (4200, 72, 3600, None), (150, 1024, 4096, None),
         (40, 4104, 136, [0, 3, 3, 40]), (45, 4101, 130, [2, 17, 17, 18, 44]), (200, 2056, 264, list(range(0, 200, 50)) + [200]), (1500, 1032, 264, [0, 1, 700, 700, 1499]),
         (6000, 136, 1400, [0] + list(range(100, 6000, 200)) + [6000])]


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("case", WHOLE, ids=lambda c: "%d x %d x %d%s" % (c[:3] + (", %d experts" % (len(c[3]) - 1) if c[3] else "",)))
def test_whole_numbers_are_exact(gpu, case, trans):
    """Operands of -1, 0 and 1 and a whole bias: every product and every partial sum is a whole number below 2^24, exact in fp32 in
    any order, so each output is the rounding of the exact one, and one product lost or taken twice shows. (A sum of K or rows
    products stays below 6000.)"""
    M, K, N, offsets = case
    dtype = BF16 if (M + trans) % 2 else F16
    print("case: whole numbers", case, NAMES[dtype], trans, flush=True)
    t = Layer(M, K, N, dtype, trans, 0, F32, offsets=offsets, seed=4)
    rng = np.random.default_rng([M, K, N, trans])
    ones = lambda shape: Mat(shape, dtype, values=rng.integers(-1, 2, shape))  # noqa: E731
    t.x, t.w, t.dy = ones((M, K)), ones(t.w.shape), ones((M, N))
    t.bias = vec(rng.integers(-3, 4, (t.E, N)), F32)
    X, W, DY, B = (v.astype(np.float32) for v in (t.x.values, t.W(), t.dy.values, t.bias.values.reshape(t.E, N)))
    y = t.forward(pre=False)[0].get()
    gx, gw, gb = t.backward(F32)
    gx, gw, gb = gx.get(), gw.get().reshape(t.w.shape), gb.get()
    rounded = lambda v: decode(encode(v, dtype), dtype)  # noqa: E731
    for e, (a, b) in enumerate(t.groups()):
        # these sums are exact in fp32 as well
        assert np.array_equal(y[a:b], rounded(X[a:b] @ W[e] + B[e])), "y, expert %d" % e
        assert np.array_equal(gx[a:b], rounded(DY[a:b] @ W[e].T)), "grad_x, expert %d" % e
        assert np.array_equal(gw[e].T if trans else gw[e], X[a:b].T @ DY[a:b]), "grad_w, expert %d" % e
        assert np.array_equal(gb[e], DY[a:b].sum(0)), "grad_bias, expert %d" % e


# ---- gradients against differences ---------------------------------------------------------------------------------

def test_gradients_against_differences(gpu):
    """Without an activation the layer is linear, so central differences of any step are exact but for y's rounding:
    half a step of either y per element, over twice the step."""
    for M in (6, 80):
        t = Layer(M, 40, 24, F16, 0, 0)
        gx, gw, gb = [g.get() for g in t.backward(F32)]
        X, W, B, DY = t.x.values, t.w.values, t.bias.values.reshape(1, -1), t.dy.values

        def loss(x, w, b):
            s = Layer(M, 40, 24, F16, 0, 0)
            s.x, s.w, s.bias = Mat(x.shape, F16, values=x), Mat(w.shape, F16, values=w), vec(b, F16)
            y = s.forward()[0].get()
            return (y * DY).sum(), (np.abs(y) * np.abs(DY)).sum() * HALF[F16] + (np.abs(s.x.values) @ np.abs(s.w.values[0])).sum() * 100 * U

        for base, grad, at in ((X, gx, (1, 3)), (X, gx, (M - 1, 39)), (W, gw.reshape(W.shape), (0, 5, 7)), (W, gw.reshape(W.shape), (0, 39, 23)), (B, gb, (0, 11))):
            hi, lo = base.copy(), base.copy()
            hi[at] += 1.0
            lo[at] -= 1.0
            step = decode(encode(hi[at], F16), F16) - decode(encode(lo[at], F16), F16)
            (up, e1), (down, e2) = (loss(*[v if base is q else q for q in (X, W, B)]) for v in (hi, lo))
            assert abs((up - down) / step - grad[at]) <= (e1 + e2) / step + HALF[F16] * abs(grad[at]) + 1e-4


# ---- a feed-forward block, forward and backward -----------------------------------------------------------------------

@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("rows", [12, 300])
def test_a_residual_block_and_its_gradients(gpu, by_expert, rows):
    """out = x + W2 gelu(W1 norm(x) + b1) + b2 and all its gradients as a model runs them, every step checked against the
    formulas on what the step before it gave; the gradient around the block joins in the norm's backward pass."""
    from test_gpu_layernorm import backward as norm_back, check_backward as check_norm_back, check_forward as check_norm, forward as norm
    D, H = 136, 264
    offsets = [0, rows // 4, rows // 4, rows] if by_expert else None
    one = Layer(rows, D, H, BF16, 0, 3, offsets=offsets, seed=2)
    two = Layer(rows, H, D, BF16, 1, 0, offsets=offsets, residual=not by_expert, seed=3)
    rng = np.random.default_rng(rows)
    x = Mat((rows, D), BF16, values=rng.standard_normal((rows, D)))
    gamma, beta = vec(1 + 0.1 * rng.standard_normal(D), F32), vec(0.1 * rng.standard_normal(D), F32)
    h, mean, rstd = norm(x, gamma, beta, BF16, F32)
    check_norm(x, gamma, beta, h, mean, rstd, BF16)

    def given(m):                                         # a tensor of the device as the next step's input
        m.host = m.raw().copy()
        return m

    one.x = given(h)
    a, pre = one.forward()
    one.check_forward(a, pre)
    two.x = given(a)
    if not by_expert:
        two.residual = x
    out, _ = two.forward(pre=False)
    two.check_forward(out, None)
    g2x, g2w, g2b = two.backward()
    two.check_backward(g2x, g2w, g2b)
    one.dy, one.pre = given(g2x), given(pre)
    g1x, g1w, g1b = one.backward()
    one.check_backward(g1x, g1w, g1b)
    dh = given(g1x)
    got = norm_back(dh, x, gamma, mean, rstd, BF16, F32, res=two.dy)
    check_norm_back(dh, x, gamma, mean, rstd, two.dy, got, BF16)


# ---- streams, graphs, threads, torch --------------------------------------------------------------------------------

def test_same_bits_every_time_and_on_other_streams(gpu):
    st = C.c_void_p()
    assert ea.hip_runtime().hipStreamCreate(C.byref(st)) == 0
    for t in (Layer(20, 2000, 300, BF16, 0, 1), Layer(70, 3000, 200, F16, 1, 3), Layer(400, 72, 136, BF16, 0, 4, offsets=[0, 100, 300, 390])):
        first = [m.bits() for m in t.forward() + t.backward()]
        # rows of no expert hold whatever the fresh output held, which is the same pattern every time
        for stream in (None, st, 0):
            assert [m.bits() for m in t.forward(stream=stream) + t.backward(stream=stream)] == first
    ea.hip_runtime().hipStreamDestroy(st)


def test_captured_step_replays(gpu):
    """Forward and backward of a layer and of experts in two graphs, a workspace each, replayed on new inputs."""
    lib = gpu.load()
    made = []
    for t in (Layer(150, 136, 264, BF16, 0, 3), Layer(150, 136, 264, BF16, 0, 3, offsets=[0, 10, 10, 140])):
        y, z = t.out((150, 264)), t.out((150, 264))
        gx, gw, gb = t.out((150, 136)), t.out(t.w.shape), Mat((t.E, 264), F32)
        f = dict(x=t.x.ptr, w=t.w.ptr, bias=t.bias.ptr, y=y.ptr, pre=z.ptr, K=136, N=264, dtype=BF16, param_dtype=BF16, act=3)
        b = dict(grad_y=t.dy.ptr, pre=z.ptr, x=t.x.ptr, w=t.w.ptr, grad_x=gx.ptr, grad_w=gw.ptr, grad_bias=gb.ptr, K=136, N=264, dtype=BF16, grad_w_dtype=BF16, act=3)
        if t.offsets is None:
            calls = [(lib.hip_linear_16, lib.hip_linear_16_workspace, ea.HipLinearArgs(M=150, **f)),
                     (lib.hip_linear_backward_16, lib.hip_linear_backward_16_workspace, ea.HipLinearBackwardArgs(M=150, **b))]
        else:
            more = dict(rows=150, experts=3, offsets=t.doff.ptr)
            calls = [(lib.hip_experts_16, lib.hip_experts_16_workspace, ea.HipExpertsArgs(**f, **more)),
                     (lib.hip_experts_backward_16, lib.hip_experts_backward_16_workspace, ea.HipExpertsBackwardArgs(**b, **more))]
        ws = room(max(size(C.byref(a)) for _, size, a in calls))
        graph = Graph()
        with graph as st:
            for entry, size, a in calls:
                a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
                assert entry(C.byref(a), st) == 0
        made.append((t, graph, ws, (y, z, gx, gw, gb)))
    rng = np.random.default_rng(1)
    for turn in range(3):
        for t, graph, ws, outs in made:
            v = Mat((150, 136), BF16, values=rng.standard_normal((150, 136)))
            t.x.host[:] = v.host
            t.x.dev.upload(t.x.host.view(np.uint8))
        for t, graph, ws, outs in made:
            graph.replay(wait=False)                      # both at once, each on its own stream
        ea.synchronize()
        for t, graph, ws, outs in made:
            t.pre = outs[1]
            t.pre.host = t.pre.raw().copy()
            for got, want in zip(outs, t.forward() + t.backward()):
                assert got.bits() == want.bits(), turn
    for t, graph, ws, outs in made:
        graph.close()


def test_two_threads_at_once(gpu):
    made = [Layer(300, 264, 392, BF16, 0, 3, seed=5), Layer(300, 264, 392, BF16, 0, 3, offsets=[0, 50, 250, 300], seed=6)]
    want = [[m.bits() for m in t.forward() + t.backward()] for t in made]
    got = [None, None]

    def work(i):
        st = C.c_void_p()
        ea.hip_runtime().hipStreamCreate(C.byref(st))
        got[i] = [[m.bits() for m in made[i].forward(stream=st) + made[i].backward(stream=st)] for _ in range(4)]
        ea.hip_runtime().hipStreamDestroy(st)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert got == [[want[0]] * 4, [want[1]] * 4]


TORCH = r"""
import ctypes, sys
import torch
sys.path.insert(0, %r)
import eshkol_amd as ea
lib = ea.load()
torch.manual_seed(0)
M, K, N = 200, 256, 384
x, w, b = (torch.randn(*s, device="cuda").bfloat16() for s in ((M, K), (N, K), (N,)))
w *= K ** -0.5
y = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
a = ea.HipLinearArgs(x=x.data_ptr(), w=w.data_ptr(), bias=b.data_ptr(), y=y.data_ptr(), M=M, K=K, N=N, dtype=3, param_dtype=3, act=ea.ACT_SILU, trans_w=1)
need = lib.hip_linear_16_workspace(ctypes.byref(a))
ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
a.workspace, a.workspace_bytes = ws.data_ptr(), need
def step():
    assert lib.hip_linear_16(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
def want():
    z = x.double() @ w.double().t() + b.double()
    return z * torch.sigmoid(z)
def check():
    torch.cuda.synchronize()
    d = (y.double() - want()).abs()
    assert (d <= 2.0 ** -8 * want().abs() + 1e-3).all(), d.max()
step(); check()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    y.zero_(); step()
check()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
for i in range(3):
    x.copy_(torch.randn(M, K, device="cuda")); y.zero_()
    graph.replay(); check()
print("OK", flush=True)
"""


def test_torch_tensors_streams_and_graphs(gpu):
    """torch's tensors on its streams and in its graphs, in a process that torch's own runtime serves."""
    r = subprocess.run([sys.executable, "-c", TORCH % ROOT], capture_output=True, text=True, timeout=200, env=dict(os.environ))
    assert r.returncode == 0 and "OK" in r.stdout, r.stdout + r.stderr


COLD = r"""
import ctypes, sys
import torch
sys.path.insert(0, %r)
import eshkol_amd as ea
lib = ea.load()
torch.manual_seed(0)
M, K, N = 300, 256, 512
new = lambda *s: torch.randn(*s, device="cuda").bfloat16()
x, w, dy, y, pre, gx, gw, h, dh = new(M, K), new(K, N) * K ** -0.5, new(M, N), new(M, N), new(M, N), new(M, K), new(K, N), new(M, K), new(M, K)
gb, mean, rstd, gg, gbeta = (torch.empty(n, device="cuda") for n in (N, M, M, K, K))
n = ea.HipLayerNormArgs(x=x.data_ptr(), y=h.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), rows=M, cols=K, epsilon=1e-5, dtype=3, param_dtype=3)
f = ea.HipLinearArgs(x=h.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), pre=pre.data_ptr(), M=M, K=K, N=N, dtype=3, param_dtype=3, act=3)
b = ea.HipLinearBackwardArgs(grad_y=dy.data_ptr(), pre=pre.data_ptr(), x=h.data_ptr(), w=w.data_ptr(), grad_x=gx.data_ptr(), grad_w=gw.data_ptr(), grad_bias=gb.data_ptr(),
                             M=M, K=K, N=N, dtype=3, grad_w_dtype=3, act=3)
m = ea.HipLayerNormBackwardArgs(grad_y=gx.data_ptr(), x=x.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(), grad_residual=gx.data_ptr(), grad_x=dh.data_ptr(),
                                grad_gamma=gg.data_ptr(), grad_beta=gbeta.data_ptr(), rows=M, cols=K, dtype=3, param_dtype=3)
calls = [(lib.hip_layernorm, n), (lib.hip_linear_16, f), (lib.hip_linear_backward_16, b), (lib.hip_layernorm_backward, m)]
room = []
for entry, size, a in ((lib.hip_linear_16, lib.hip_linear_16_workspace, f), (lib.hip_linear_backward_16, lib.hip_linear_backward_16_workspace, b),
                       (lib.hip_layernorm_backward, lib.hip_layernorm_backward_workspace, m)):
    need = size(ctypes.byref(a))
    room.append(torch.empty(max(need, 1), dtype=torch.uint8, device="cuda"))
    a.workspace, a.workspace_bytes = room[-1].data_ptr(), need
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for entry, a in calls:
        assert entry(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
outs = [h, mean, rstd, y, pre, gx, gw, gb, dh, gg, gbeta]
for turn in range(3):
    x.copy_(new(M, K))
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in outs]
    for entry, a in calls:
        assert entry(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(g, o) for g, o in zip(got, outs)) and all(g.abs().max() > 0 for g in got)
print("OK", flush=True)
"""


def test_the_first_calls_of_a_process_are_captured(gpu):
    """Nothing has to run before a capture: a block's forward and backward pass go into a graph as a process's first calls,
    and replay to the bits of eager calls."""
    r = subprocess.run([sys.executable, "-c", COLD % ROOT], capture_output=True, text=True, timeout=200, env=dict(os.environ))
    assert r.returncode == 0 and "OK" in r.stdout, r.stdout + r.stderr
