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
