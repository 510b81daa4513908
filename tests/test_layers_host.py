"""The layer operators' checks of their arguments (gpu_hip_layers.h), all on the host: what is refused, what a
workspace has to hold, and that header, binding and library name the same things."""
import ctypes as C
import os
import re

import pytest

import eshkol_amd as ea
from test_abi_host import INC, declared_functions, run_child

ODD = 0x10001           # an address off every boundary; nothing here is ever followed


def test_header_binding_and_library_agree():
    lib = ea.load()
    names = declared_functions("gpu_hip_layers.h")
    assert names
    for name in names:
        assert hasattr(lib, name) and name in ea.SIGNATURES, name


def test_structs_have_the_headers_fields_in_order():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INC, "gpu_hip_layers.h")).read(), flags=re.S)
    sizes = {"uint64_t": C.c_uint64, "int32_t": C.c_int32, "double": C.c_double}
    found = 0
    for body, name in re.findall(r"typedef struct \{(.*?)\} (\w+);", text, flags=re.S):
        fields = []
        for line in body.split(";"):
            line = line.strip()
            if not line:
                continue
            kind, rest = re.match(r"((?:const )?\w+\*?) (.*)", line, flags=re.S).groups()
            for item in rest.split(","):
                pointer = kind.endswith("*") or item.strip().startswith("*")
                fields.append((item.strip().lstrip("*"), C.c_void_p if pointer else sizes[kind]))
        assert [(n, t) for n, t in getattr(ea, name)._fields_] == fields, name
        found += 1
    assert found == len([n for n in dir(ea) if re.match(r"Hip(LayerNorm|Linear|Experts)\w*Args$", n)])


# ---- layer norm -------------------------------------------------------------------------------------------

def norm(**changes):
    a = dict(x=1 << 20, gamma=1 << 12, beta=1 << 12, y=1 << 21, mean=1 << 13, rstd=1 << 14, rows=4, cols=100, ldx=100, ldy=100,
             epsilon=1e-5, dtype=3, param_dtype=3)
    a.update(changes)
    return ea.HipLayerNormArgs(**a)


def norm_back(**changes):
    a = dict(grad_y=1 << 20, x=1 << 21, gamma=1 << 12, mean=1 << 13, rstd=1 << 14, grad_x=1 << 22, grad_gamma=1 << 15, grad_beta=1 << 16,
             rows=4, cols=100, dtype=3, param_dtype=3)
    a.update(changes)
    return ea.HipLayerNormBackwardArgs(**a)


NORM_REFUSED = [dict(x=None), dict(y=None), dict(cols=0), dict(cols=(1 << 24) + 1), dict(rows=(1 << 40) + 1), dict(ldx=99), dict(ldy=99),
                dict(dtype=4), dict(dtype=-1), dict(param_dtype=2), dict(dtype=0, param_dtype=1), dict(dtype=1, param_dtype=3), dict(x=ODD), dict(y=ODD),
                dict(gamma=ODD), dict(beta=ODD), dict(mean=ODD), dict(rstd=0x10002), dict(epsilon=-1e-9), dict(epsilon=float("nan")), dict(epsilon=float("inf")),
                dict(y=1 << 20, ldy=104)]


@pytest.mark.parametrize("change", NORM_REFUSED, ids=str)
def test_layernorm_refuses(change):
    assert ea.load().hip_layernorm(C.byref(norm(**change)), None) == -1


def test_layernorm_without_rows_needs_nothing():
    lib = ea.load()
    assert lib.hip_layernorm(None, None) == -1
    assert lib.hip_layernorm(C.byref(norm(rows=0, x=None, y=None)), None) == 0
    assert lib.hip_layernorm(C.byref(norm(rows=0, cols=0)), None) == -1


BACK_REFUSED = [dict(grad_y=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(grad_x=None, grad_gamma=None, grad_beta=None), dict(cols=0),
                dict(ld_grad_y=99), dict(ldx=99), dict(ld_grad_x=99), dict(grad_residual=1 << 23, ld_grad_residual=50), dict(dtype=7), dict(param_dtype=0),
                dict(grad_y=ODD), dict(x=ODD), dict(grad_x=ODD), dict(grad_gamma=0x10002), dict(grad_beta=0x10002), dict(mean=0x10002), dict(gamma=ODD),
                dict(grad_residual=ODD), dict(grad_x=1 << 20, ld_grad_x=104), dict(grad_x=1 << 21, ld_grad_x=104), dict(grad_beta=1 << 15),
                dict(grad_residual=1 << 23, grad_x=1 << 23, ld_grad_x=200)]


@pytest.mark.parametrize("change", BACK_REFUSED, ids=str)
def test_layernorm_backward_refuses(change):
    lib = ea.load()
    a = norm_back(**change)
    assert lib.hip_layernorm_backward_workspace(C.byref(a)) == -1
    assert lib.hip_layernorm_backward(C.byref(a), None) == -1


def test_layernorm_backward_workspace():
    lib = ea.load()
    size = lambda **c: lib.hip_layernorm_backward_workspace(C.byref(norm_back(**c)))  # noqa: E731
    assert lib.hip_layernorm_backward_workspace(None) == -1
    assert size() > 0 and size(grad_gamma=None) > 0
    assert size(grad_gamma=None, grad_beta=None) == 0            # nothing to add up
    assert size(rows=0) == 0 and size(rows=0, x=None, grad_y=None, mean=None, rstd=None) == 0
    assert 0 < size(rows=1 << 20, cols=4096) <= 1 << 28          # bounded, whatever the row count
    need = size()
    for given in (dict(workspace=None, workspace_bytes=need), dict(workspace=1 << 24, workspace_bytes=need - 1), dict(workspace=(1 << 24) + 8, workspace_bytes=need)):
        assert lib.hip_layernorm_backward(C.byref(norm_back(**given)), None) == -2


def test_a_refusal_says_why():
    body = r"""
import ctypes as C
a = ea.HipLayerNormArgs(rows=4, cols=100, dtype=3, param_dtype=2)
assert lib.hip_layernorm(C.byref(a), None) == -1
"""
    r = run_child(body, {"ESHKOL_GPU_VERBOSE": "1"})
    assert r.returncode == 0 and "[GPU] hip_layernorm: param_dtype 2 beside dtype 3" in r.stderr, r.stderr
    assert run_child(body).stderr.count("hip_layernorm") == 0


# ---- linear layer and experts -------------------------------------------------------------------------------

def linear(**changes):
    a = dict(x=1 << 20, w=1 << 21, bias=1 << 12, residual=1 << 22, y=1 << 23, pre=1 << 24, M=100, K=64, N=96, dtype=3, param_dtype=3, act=3)
    a.update(changes)
    return ea.HipLinearArgs(**a)


def linear_back(**changes):
    a = dict(grad_y=1 << 20, pre=1 << 21, x=1 << 22, w=1 << 23, grad_x=1 << 24, grad_w=1 << 25, grad_bias=1 << 26, M=100, K=64, N=96, dtype=3, grad_w_dtype=3, act=3)
    a.update(changes)
    return ea.HipLinearBackwardArgs(**a)


def experts(**changes):
    a = dict(x=1 << 20, w=1 << 21, bias=1 << 12, offsets=1 << 10, y=1 << 23, pre=1 << 24, rows=100, experts=4, K=64, N=96, dtype=2, param_dtype=1, act=4)
    a.update(changes)
    return ea.HipExpertsArgs(**a)


def experts_back(**changes):
    a = dict(grad_y=1 << 20, pre=1 << 21, x=1 << 22, w=1 << 23, offsets=1 << 10, grad_x=1 << 24, grad_w=1 << 25, grad_bias=1 << 26, rows=100, experts=4, K=64, N=96,
             dtype=2, grad_w_dtype=1, act=4)
    a.update(changes)
    return ea.HipExpertsBackwardArgs(**a)


SIZES_REFUSED = [dict(K=0), dict(N=0), dict(K=(1 << 22) + 1), dict(N=(1 << 22) + 1), dict(dtype=0), dict(dtype=1), dict(dtype=4), dict(act=5), dict(act=-1)]
FORWARD_REFUSED = SIZES_REFUSED + [dict(x=None), dict(w=None), dict(y=None), dict(x=ODD), dict(w=ODD), dict(y=ODD), dict(pre=ODD), dict(ldx=63), dict(ldw=95),
                                   dict(ldw=63, trans_w=1), dict(ldy=95), dict(ld_pre=95), dict(param_dtype=0), dict(y=1 << 20), dict(y=1 << 21), dict(pre=1 << 23),
                                   dict(pre=1 << 20), dict(pre=1 << 21)]
BACKWARD_REFUSED = SIZES_REFUSED + [dict(grad_y=None), dict(pre=None), dict(x=None), dict(w=None), dict(grad_x=None, grad_w=None, grad_bias=None), dict(grad_y=ODD), dict(pre=ODD),
                                    dict(x=ODD), dict(w=ODD), dict(grad_x=ODD), dict(grad_w=ODD), dict(grad_bias=0x10002), dict(ld_grad_y=95), dict(ld_pre=95), dict(ldx=63),
                                    dict(ldw=95), dict(ld_grad_x=63), dict(ld_grad_w=95), dict(grad_w_dtype=0), dict(grad_x=1 << 20), dict(grad_w=1 << 23), dict(grad_bias=1 << 25)]
EXPERTS_REFUSED = [dict(experts=0), dict(experts=4097), dict(offsets=None), dict(offsets=ODD), dict(rows=1 << 31), dict(w_stride=64 * 96 - 1)]
KINDS = {"hip_linear_16": (linear, FORWARD_REFUSED + [dict(M=1 << 31), dict(bias=ODD), dict(param_dtype=2), dict(residual=ODD), dict(ld_residual=95), dict(pre=1 << 22), dict(y=1 << 22, ldy=104)]),
         "hip_linear_backward_16": (linear_back, BACKWARD_REFUSED + [dict(M=1 << 31), dict(grad_w_dtype=2)]),
         "hip_experts_16": (experts, FORWARD_REFUSED + EXPERTS_REFUSED + [dict(bias=0x10002), dict(param_dtype=3)]),
         "hip_experts_backward_16": (experts_back, BACKWARD_REFUSED + EXPERTS_REFUSED + [dict(grad_w_stride=100), dict(grad_w_dtype=3)])}


@pytest.mark.parametrize("name,change", [(n, c) for n, (_, cs) in KINDS.items() for c in cs], ids=str)
def test_refuses(name, change):
    lib = ea.load()
    a = KINDS[name][0](**change)
    assert getattr(lib, name + "_workspace")(C.byref(a)) == -1
    assert getattr(lib, name)(C.byref(a), None) == -1


@pytest.mark.parametrize("name", list(KINDS))
def test_accepts_and_says_what_it_needs(name):
    lib = ea.load()
    make, size, entry = KINDS[name][0], getattr(lib, name + "_workspace"), getattr(lib, name)
    assert size(None) == -1 and entry(None, None) == -1
    need = size(C.byref(make()))
    assert need >= 0
    rows = "M" if "linear" in name else "rows"
    assert size(C.byref(make(**{rows: 0}))) == 0                 # no rows: nothing to hold
    # operands off 16-byte boundaries are copied for the tiled kernel (a few rows are read as they are)
    assert size(C.byref(make(ldx=67, **{rows: 1000}))) > size(C.byref(make(**{rows: 1000})))
    if "backward" in name:
        assert need > 0
    if need:
        for given in (dict(), dict(workspace=1 << 27, workspace_bytes=need - 1), dict(workspace=(1 << 27) + 8, workspace_bytes=need)):
            assert entry(C.byref(make(**given)), None) == -2


def test_forward_without_rows_needs_nothing():
    lib = ea.load()
    assert lib.hip_linear_16(C.byref(linear(M=0, x=None, w=None, y=None)), None) == 0
    assert lib.hip_experts_16(C.byref(experts(rows=0, x=None, w=None, y=None, offsets=None)), None) == 0
    assert lib.hip_linear_16(C.byref(linear(M=0, N=0)), None) == -1


def test_more_workgroups_than_a_launch_holds_are_refused_before_anything_is_queued():
    lib = ea.load()
    big = dict(K=1 << 21, N=1 << 22, act=0, pre=None)
    assert lib.hip_linear_16_workspace(C.byref(linear(M=(1 << 31) - 1, **big))) == -1
    assert lib.hip_linear_16(C.byref(linear(M=(1 << 31) - 1, **big)), None) == -1
    assert lib.hip_linear_backward_16_workspace(C.byref(linear_back(M=(1 << 31) - 1, **big))) == -1
    assert lib.hip_experts_16_workspace(C.byref(experts(rows=(1 << 31) - 1, **big))) == -1
    assert lib.hip_experts_backward_16_workspace(C.byref(experts_back(experts=4096, rows=100, **big))) == -1


def test_optional_arguments():
    lib = ea.load()
    assert lib.hip_linear_16_workspace(C.byref(linear(bias=None, residual=None, pre=None))) >= 0
    assert lib.hip_linear_backward_16_workspace(C.byref(linear_back(act=0, pre=None))) >= 0
    assert lib.hip_linear_backward_16_workspace(C.byref(linear_back(grad_w=None, x=None))) >= 0
    assert lib.hip_linear_backward_16_workspace(C.byref(linear_back(grad_x=None, w=None))) >= 0
    assert lib.hip_experts_backward_16_workspace(C.byref(experts_back(grad_x=None, w=None))) >= 0


def test_the_derivatives_the_gpu_tests_use_are_the_activations_own():
    """Central differences of a step of 1e-5: off by the third derivative (at most 2) times 1e-10 / 6 and by the
    rounding of two values up to 6 over 2e-5."""
    import numpy as np
    from layer_util import act, slope
    z = np.concatenate([np.linspace(-6, 6, 997), [1e-3, -1e-3]])
    for code in (1, 2, 3, 4):
        d = (act(z + 1e-5, code) - act(z - 1e-5, code)) / 2e-5
        far = np.abs(z) > 1e-4 if code == 2 else np.ones_like(z, bool)
        assert np.abs(d - slope(z, code))[far].max() < 1e-10 + 8 * 6 * 2.0 ** -53 / 1e-5, code
