"""Helpers for the tests of the layer operators (gpu_hip_layers.h): element types in numpy, matrices in
device memory with a pitch and an odd start, HIP graphs, and the plain forms in 64 bits."""
import ctypes as C
from math import erfc

import numpy as np

import eshkol_amd as ea

F64, F32, F16, BF16 = 0, 1, 2, 3
NAMES = {F64: "f64", F32: "f32", F16: "f16", BF16: "bf16"}
STORE = {F64: np.float64, F32: np.float32, F16: np.float16, BF16: np.uint16}
# half a step of a rounding to the type, relative to the value
HALF = {F64: 2.0 ** -53, F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# what half a step is where the value is below the type's normal range
FLOOR = {F64: 0.0, F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def unit(dtype):
    """The rounding of the type sums are held in."""
    return 2.0 ** -53 if dtype == F64 else 2.0 ** -24


def wide(dtype):
    return F64 if dtype == F64 else F32


def encode(a, dtype):
    a = np.asarray(a, dtype=np.float64)
    if dtype != BF16:
        with np.errstate(over="ignore"):
            return a.astype(STORE[dtype])
    bits = a.astype(np.float32).view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(a)
    out[nan] = 0x7fc0
    return out


def decode(a, dtype):
    if dtype != BF16:
        return a.astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Mat:
    """A matrix (or a stack of them) in device memory: rows `ld` elements apart, its first element `shift`
    elements behind a 16-byte boundary, a known pattern in every element around it."""

    def __init__(self, shape, dtype, ld=None, shift=0, values=None, tail=16):
        self.shape = tuple(int(n) for n in (shape if hasattr(shape, "__len__") else (shape,)))
        self.dtype, self.shift = dtype, shift
        cols = self.shape[-1]
        self.ld = cols if ld is None else ld
        self.rows = int(np.prod(self.shape[:-1])) if len(self.shape) > 1 else 1
        n = shift + self.rows * self.ld + tail
        rng = np.random.default_rng(n)
        self.host = rng.integers(0, 255, n * np.dtype(STORE[dtype]).itemsize, dtype=np.uint8).view(STORE[dtype]).copy()
        if values is not None:
            self.inner(self.host)[:] = encode(values, dtype).reshape(self.rows, cols)
        self.dev = ea.DeviceArray.from_host(self.host.view(np.uint8))
        self.ptr = self.dev.ptr + shift * self.host.itemsize

    def inner(self, flat):
        return flat[self.shift:self.shift + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.shape[-1]]

    @property
    def values(self):
        """What the device was given, in 64 bits."""
        return decode(self.inner(self.host).copy(), self.dtype).reshape(self.shape)

    def raw(self):
        return self.dev.download().view(STORE[self.dtype])

    def get(self):
        return decode(self.inner(self.raw()).copy(), self.dtype).reshape(self.shape)

    def bits(self):
        return self.inner(self.raw()).copy().tobytes()

    def surroundings_untouched(self):
        a, b = self.raw().copy(), self.host.copy()
        self.inner(a)[:] = 0
        self.inner(b)[:] = 0
        return a.tobytes() == b.tobytes()


def vec(values, dtype):
    values = np.asarray(values, dtype=np.float64)
    return Mat(values.shape, dtype, values=values)


def room(n):
    """A workspace of n bytes, its contents as unhelpful as they come (NaN)."""
    d = ea.DeviceArray((max(int(n), 16),), np.uint8)
    d.upload(np.full(max(int(n), 16), 0xff, np.uint8))
    return d


def run(entry, args, size=None, stream=None):
    """Calls an entry point with the workspace it asks for and waits; returns its status."""
    ws = None
    if size is not None:
        need = size(C.byref(args))
        assert need >= 0, "refused"
        ws = room(need)
        args.workspace, args.workspace_bytes = ws.ptr, need
    rc = entry(C.byref(args), ea.load().eshkol_hip_get_stream() if stream is None else stream)
    ea.synchronize()
    return rc


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise; infinities and NaN in the same places."""
    got, want = np.asarray(got), np.asarray(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), what + ": infinities in other places"
    tol = np.broadcast_to(tol, got.shape)
    off = np.abs(got - want)[fine] - tol[fine]
    if off.size and off.max() > 0:
        k = int(np.argmax(off))
        raise AssertionError("%s: %d of %d values off, worst by %.3g where %.3g is allowed (got %.9g, want %.9g)" % (
            what, int((off > 0).sum()), off.size, off[k] + tol[fine][k], tol[fine][k], got[fine][k], want[fine][k]))


class Graph:
    """Calls captured on a stream of their own and replayed."""

    def __init__(self):
        h = self.h = ea.hip_runtime()
        self.stream, self.graph, self.exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        assert h.hipStreamCreate(C.byref(self.stream)) == 0

    def __enter__(self):
        assert self.h.hipStreamBeginCapture(self.stream, C.c_int(2)) == 0          # relaxed
        return self.stream

    def __exit__(self, kind, value, tb):
        assert self.h.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0
        if kind is None:
            assert self.h.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, C.c_size_t(0)) == 0

    def replay(self, wait=True):
        assert self.h.hipGraphLaunch(self.exe, self.stream) == 0
        if wait:
            assert self.h.hipStreamSynchronize(self.stream) == 0

    def close(self):
        self.h.hipGraphExecDestroy(self.exe)
        self.h.hipGraphDestroy(self.graph)
        self.h.hipStreamDestroy(self.stream)


# ---- activations in 64 bits ---------------------------------------------------------------------------

_erfc = np.vectorize(erfc, otypes=[np.float64])         # 1 + erf would lose every digit of the lower tail


def act(z, code):
    if code == 1:
        return np.tanh(z)
    if code == 2:
        return np.maximum(z, 0.0)
    if code == 3:
        return 0.5 * z * _erfc(-z / np.sqrt(2.0))
    if code == 4:
        return z / (1.0 + np.exp(-z))
    return z


def slope(z, code):
    if code == 1:
        return 1.0 - np.tanh(z) ** 2
    if code == 2:
        return (z > 0).astype(np.float64)
    if code == 3:
        return 0.5 * _erfc(-z / np.sqrt(2.0)) + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)
    if code == 4:
        s = 1.0 / (1.0 + np.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return np.ones_like(z)
