"""What is measured of the layer operators: layer norm, the linear layer with its epilogue, and the
products grouped by expert, each forward and backward, in plain torch and through the library's entry points."""
import ctypes
import math
import random

import torch

own = False

KINDS = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}
ACTS = {"none": 0, "tanh": 1, "relu": 2, "gelu": 3, "silu": 4}
EPSILON = 1e-5


# ---- cases ------------------------------------------------------------------------------------------

def listed():
    return [
        # the norm in front of a layer when one token is served: latency is all of it
        dict(name="norm_one_token", op="norm", way="forward", rows=1, cols=4096, dtype="f16", param="f16", pad=0, residual=False),
        # a training batch's norm, mean and 1/deviation kept for the backward pass
        dict(name="norm_batch", op="norm", way="forward", rows=32768, cols=4096, dtype="bf16", param="bf16", pad=0, residual=False),
        # single precision training, sizes that are multiples of nothing
        dict(name="norm_back_odd", op="norm", way="backward", rows=4095, cols=1023, dtype="f32", param="f32", pad=0, residual=False),
        # a training batch's backward pass in a residual block: the gradient around the block is added on the way
        dict(name="norm_back_batch", op="norm", way="backward", rows=32768, cols=4096, dtype="bf16", param="f32", pad=0, residual=True),
        # a layer when one token is served: the weights are read once
        dict(name="linear_one_token", op="linear", way="forward", rows=1, k=4096, n=4096, dtype="bf16", param="bf16", act="gelu", trans=False, residual=False, pad=0),
        # the second layer of a block for a small serving batch, its input added in the epilogue
        dict(name="linear_32_rows", op="linear", way="forward", rows=32, k=4096, n=4096, dtype="f16", param="f16", act="none", trans=True, residual=True, pad=0),
        # the largest product: training, the sums before the activation kept
        dict(name="linear_large", op="linear", way="forward", rows=8192, k=8192, n=8192, dtype="bf16", param="bf16", act="gelu", trans=False, residual=False, pad=0),
        # the first layer of the 1024-4096-4096-1024 network at batch 4096, backward
        dict(name="linear_back", op="linear", way="backward", rows=4096, k=1024, n=4096, dtype="bf16", param="bf16", act="gelu", trans=False, residual=False, pad=0),
        # backward at odd sizes and pitches, weights held transposed
        dict(name="linear_back_odd", op="linear", way="backward", rows=1023, k=1000, n=2047, dtype="f16", param="f32", act="tanh", trans=True, residual=False, pad=5),
        # serving: a few tokens spread over the experts, whose weights are all of the traffic
        dict(name="experts_few_rows", op="experts", way="forward", rows=128, k=1024, n=4096, experts=64, active=48, most=9, dtype="bf16", param="bf16", act="silu", trans=False),
        # training: ragged groups, some experts without rows
        dict(name="experts_batch", op="experts", way="forward", rows=16384, k=1024, n=4096, experts=64, active=60, most=640, dtype="bf16", param="bf16", act="gelu", trans=False),
        dict(name="experts_back", op="experts", way="backward", rows=8191, k=1024, n=2048, experts=32, active=30, most=640, dtype="bf16", param="f32", act="silu", trans=True),
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm; one in three is odd, the others multiples of 8 where they can be."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    v = max(low, min(high, v))
    if v >= 16 and rng.random() < 0.67:
        return v // 8 * 8
    return v


def draw(rng):
    op, way = rng.choice(("norm", "linear", "experts")), rng.choice(("forward", "backward"))
    if op == "norm":
        dtype = rng.choice(("f64", "f32", "f16", "bf16"))
        cols = _spread(rng, 64, 16384)
        rows = _spread(rng, 1, min(32768, 2 ** 26 // cols))
        return dict(op=op, way=way, rows=rows, cols=cols, dtype=dtype, param=rng.choice((dtype, dtype if dtype == "f64" else "f32")),
                    pad=rng.choice((0, 0, 8, 5)), residual=way == "backward" and rng.random() < 0.5)
    dtype = rng.choice(("f16", "bf16"))
    k, n = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
    common = dict(op=op, way=way, k=k, n=n, dtype=dtype, param=rng.choice((dtype, "f32")), act=rng.choice(sorted(ACTS)), trans=rng.random() < 0.5)
    if op == "linear":
        rows = _spread(rng, 1, max(1, min(16384, 2 ** 37 // (k * n))))
        return dict(common, rows=rows, residual=way == "forward" and rng.random() < 0.5, pad=rng.choice((0, 0, 8, 5)))
    experts = _spread(rng, 2, max(2, min(128, 2 ** 28 // (k * n))))
    rows = _spread(rng, 1, max(1, min(32768, 2 ** 35 // (k * n))))
    active = rng.randint(1, min(experts, rows))
    return dict(common, rows=rows, experts=experts, active=active, most=-(-2 * rows // active))


def work(case):
    size = torch.empty(0, dtype=KINDS[case["dtype"]]).element_size()
    wide = 8 if case["dtype"] == "f64" else 4
    psize = torch.empty(0, dtype=KINDS[case["param"]]).element_size()
    rows, back = case["rows"], case["way"] == "backward"
    if case["op"] == "norm":
        cols = case["cols"]
        if back:
            return {"bytes": rows * cols * size * (4 if case["residual"] else 3) + 2 * rows * wide + cols * (psize + 2 * wide), "flops": 14 * rows * cols}
        return {"bytes": 2 * rows * cols * size + 2 * rows * wide + 2 * cols * psize, "flops": 8 * rows * cols}
    k, n = case["k"], case["n"]
    held = case["experts"] if case["op"] == "experts" else 1
    used = case["active"] if case["op"] == "experts" else 1
    acts = case["act"] != "none"
    if back:
        moved = rows * n * (1 + acts) + 2 * rows * k + used * k * n + held * k * n
        return {"bytes": moved * size + held * n * 4, "flops": 4 * rows * k * n}
    moved = rows * k + used * k * n + rows * n * (1 + acts + (1 if case.get("residual") else 0))
    return {"bytes": moved * size + used * n * psize, "flops": 2 * rows * k * n}


# ---- inputs -----------------------------------------------------------------------------------------

def _counts(case, seed):
    """Rows of each expert: `active` of them have at least one row, none more than `most`."""
    rng = random.Random(seed)
    who = rng.sample(range(case["experts"]), case["active"])
    share = [0.1 + rng.random() ** 2 for _ in who]
    total, left = sum(share), case["rows"] - len(who)
    got = [1 + min(case["most"] - 1, int(left * s / total)) for s in share]
    left = case["rows"] - sum(got)
    while left > 0:
        for i in rng.sample(range(len(who)), len(who)):
            more = min(left, case["most"] - got[i], 1 + left // len(who))
            got[i] += more
            left -= more
    counts = [0] * case["experts"]
    for e, c in zip(who, got):
        counts[e] = c
    return counts


def _offsets(case, seed):
    at = [0]
    for c in _counts(case, seed):
        at.append(at[-1] + c)
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, param = KINDS[case["dtype"]], KINDS[case["param"]]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32
    rows, pad, back = case["rows"], case.get("pad", 0), case["way"] == "backward"

    def normal(*shape, kind=kind, scale=1.0, mean=0.0):
        t = torch.randn(*shape, device="cuda", generator=g, dtype=torch.float64 if kind == torch.float64 else torch.float32)
        return t.mul_(scale).add_(mean).to(kind)

    def matrix(r, c, scale=1.0, mean=0.0):                  # rows of a wider buffer where the case pads them
        return normal(r, c + pad, scale=scale, mean=mean)[:, :c]

    def room(r, c, kind=kind):
        return torch.empty(r, c + pad, device="cuda", dtype=kind)[:, :c]

    s = dict(case=dict(case))
    if case["op"] == "norm":
        cols = case["cols"]
        s["x"] = matrix(rows, cols, 1.5, 0.3)
        s["gamma"] = normal(cols, kind=param, scale=0.2, mean=1.0)
        if back:
            x = s["x"].to(torch.float64)
            s["mean"] = x.mean(1).to(wide)
            s["rstd"] = (x.var(1, unbiased=False) + EPSILON).rsqrt().to(wide)
            del x
            s["grad_y"] = matrix(rows, cols)
            s["grad_residual"] = matrix(rows, cols) if case["residual"] else None
            s["out"] = dict(grad_x=room(rows, cols), grad_gamma=torch.empty(cols, device="cuda", dtype=wide), grad_beta=torch.empty(cols, device="cuda", dtype=wide))
        else:
            s["beta"] = normal(cols, kind=param, scale=0.2)
            s["out"] = dict(y=room(rows, cols), mean=torch.empty(rows, device="cuda", dtype=wide), rstd=torch.empty(rows, device="cuda", dtype=wide))
        return s
    k, n, acts = case["k"], case["n"], case["act"] != "none"
    if case["op"] == "linear":
        s["x"] = matrix(rows, k)
        s["w"] = matrix(n, k, k ** -0.5) if case["trans"] else matrix(k, n, k ** -0.5)
        held = (n,)
    else:
        s["x"] = normal(rows, k)
        s["w"] = normal(case["experts"], *((n, k) if case["trans"] else (k, n)), scale=k ** -0.5)
        held = (case["experts"], n)
        s["offsets"] = torch.tensor(_offsets(case, seed), dtype=torch.int32, device="cuda")
    if back:
        s["grad_y"] = matrix(rows, n)
        s["pre"] = matrix(rows, n) if acts else None
        s["out"] = dict(grad_x=room(rows, k), grad_w=torch.empty(s["w"].shape, device="cuda", dtype=kind), grad_bias=torch.empty(*held, device="cuda", dtype=torch.float32))
    else:
        s["bias"] = normal(*held, kind=param, scale=0.3)
        s["residual"] = matrix(rows, n) if case.get("residual") else None
        s["out"] = dict(y=room(rows, n), **(dict(pre=room(rows, n)) if acts else {}))
    return s


# ---- the library's entry points ---------------------------------------------------------------------

def _at(t):
    return None if t is None else t.data_ptr()


def _pitch(t):
    return 0 if t is None else t.stride(-2)


def _call(s):
    """The entry point and its arguments, with a workspace of the size that it asks for: what a program sets up once for a layer."""
    import eshkol_amd as ea
    c, o = s["case"], s["out"]
    lib, code, param, back = ea.load(), CODES[c["dtype"]], CODES[c["param"]], c["way"] == "backward"
    common = dict(x=_at(s["x"]), ldx=_pitch(s["x"]), dtype=code)
    if c["op"] == "norm":
        common |= dict(gamma=_at(s["gamma"]), rows=c["rows"], cols=c["cols"], param_dtype=param)
        if not back:
            a = ea.HipLayerNormArgs(**common, beta=_at(s["beta"]), y=_at(o["y"]), mean=_at(o["mean"]), rstd=_at(o["rstd"]), ldy=_pitch(o["y"]), epsilon=EPSILON)
            return lib.hip_layernorm, a, None
        a = ea.HipLayerNormBackwardArgs(**common, grad_y=_at(s["grad_y"]), mean=_at(s["mean"]), rstd=_at(s["rstd"]), grad_residual=_at(s["grad_residual"]),
                                        grad_x=_at(o["grad_x"]), grad_gamma=_at(o["grad_gamma"]), grad_beta=_at(o["grad_beta"]), ld_grad_y=_pitch(s["grad_y"]),
                                        ld_grad_residual=_pitch(s["grad_residual"]), ld_grad_x=_pitch(o["grad_x"]))
        entry, size = lib.hip_layernorm_backward, lib.hip_layernorm_backward_workspace
    else:
        common |= dict(w=_at(s["w"]), ldw=_pitch(s["w"]), K=c["k"], N=c["n"], act=ACTS[c["act"]], trans_w=int(c["trans"]))
        grouped = c["op"] == "experts"
        if grouped:
            common |= dict(offsets=_at(s["offsets"]), rows=c["rows"], experts=c["experts"], w_stride=s["w"].stride(0))
        else:
            common |= dict(M=c["rows"])
        if back:
            common |= dict(grad_y=_at(s["grad_y"]), pre=_at(s["pre"]), grad_x=_at(o["grad_x"]), grad_w=_at(o["grad_w"]), grad_bias=_at(o["grad_bias"]),
                           ld_grad_y=_pitch(s["grad_y"]), ld_pre=_pitch(s["pre"]), ld_grad_x=_pitch(o["grad_x"]), ld_grad_w=_pitch(o["grad_w"]), grad_w_dtype=code)
            if grouped:
                a = ea.HipExpertsBackwardArgs(**common, grad_w_stride=o["grad_w"].stride(0))
                entry, size = lib.hip_experts_backward_16, lib.hip_experts_backward_16_workspace
            else:
                a = ea.HipLinearBackwardArgs(**common)
                entry, size = lib.hip_linear_backward_16, lib.hip_linear_backward_16_workspace
        else:
            common |= dict(bias=_at(s["bias"]), y=_at(o["y"]), pre=_at(o.get("pre")), ldy=_pitch(o["y"]), ld_pre=_pitch(o.get("pre")), param_dtype=param)
            if grouped:
                a = ea.HipExpertsArgs(**common)
                entry, size = lib.hip_experts_16, lib.hip_experts_16_workspace
            else:
                a = ea.HipLinearArgs(**common, residual=_at(s["residual"]), ld_residual=_pitch(s["residual"]))
                entry, size = lib.hip_linear_16, lib.hip_linear_16_workspace
    need = size(ctypes.byref(a))
    if need < 0:
        raise RuntimeError("refused: %s" % (c,))
    room = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = room.data_ptr(), need
    return entry, a, room


# ---- plain forms ------------------------------------------------------------------------------------

def _act(z, act):
    if act == "tanh":
        return torch.tanh(z)
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "tanh":
        return 1 - torch.tanh(z) ** 2
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    one = 1 / (1 + torch.exp(-z))
    return one * (1 + z * (1 - one))


def _plain_norm(s):
    c = s["case"]
    wide = torch.float64 if c["dtype"] == "f64" else torch.float32
    kind = s["x"].dtype
    x, gamma = s["x"].to(wide), s["gamma"].to(wide)
    if c["way"] == "forward":
        mean = x.sum(1) / c["cols"]
        d = x - mean[:, None]
        rstd = 1 / torch.sqrt((d * d).sum(1) / c["cols"] + EPSILON)
        return dict(y=(d * rstd[:, None] * gamma + s["beta"].to(wide)).to(kind), mean=mean, rstd=rstd)
    h = (x - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["grad_y"].to(wide)
    t = dy * gamma
    dx = s["rstd"][:, None] * (t - t.sum(1, keepdim=True) / c["cols"] - h * ((t * h).sum(1, keepdim=True) / c["cols"]))
    if s["grad_residual"] is not None:
        dx = dx + s["grad_residual"].to(wide)
    return dict(grad_x=dx.to(kind), grad_gamma=(dy * h).sum(0), grad_beta=dy.sum(0))


def _plain_linear(s):
    c, kind = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    w = w.t() if c["trans"] else w
    if c["way"] == "forward":
        z = x @ w + s["bias"].float()
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return dict(y=y.to(kind), **(dict(pre=z.to(kind)) if c["act"] != "none" else {}))
    dz = s["grad_y"].float()
    if c["act"] != "none":
        dz = dz * _slope(s["pre"].float(), c["act"])
    dw = dz.t() @ x if c["trans"] else x.t() @ dz
    return dict(grad_x=(dz @ w.t()).to(kind), grad_w=dw.to(kind), grad_bias=dz.sum(0))


def _plain_experts(s):
    """Every expert's rows in a block of `most` of them, padded with zeros, and one batched product."""
    c, kind, at = s["case"], s["x"].dtype, s["offsets"].long()
    place = at[:-1, None] + torch.arange(c["most"], device=at.device)
    there = (place < at[1:, None])[:, :, None]
    place = place.clamp(max=c["rows"] - 1)
    row = torch.arange(c["rows"], device=at.device)
    which = torch.searchsorted(at, row, right=True) - 1
    x, w = torch.where(there, s["x"].float()[place], 0.0), s["w"].float()
    w = w.transpose(1, 2).contiguous() if c["trans"] else w
    if c["way"] == "forward":
        z = (torch.bmm(x, w) + s["bias"].float()[:, None, :])[which, row - at[which]]
        return dict(y=_act(z, c["act"]).to(kind), **(dict(pre=z.to(kind)) if c["act"] != "none" else {}))
    dz = s["grad_y"].float()
    if c["act"] != "none":
        dz = dz * _slope(s["pre"].float(), c["act"])
    dz = torch.where(there, dz[place], 0.0)
    dx = torch.bmm(dz, w.transpose(1, 2).contiguous())[which, row - at[which]]
    dw = torch.bmm(dz.transpose(1, 2).contiguous(), x) if c["trans"] else torch.bmm(x.transpose(1, 2).contiguous(), dz)
    return dict(grad_x=dx.to(kind), grad_w=dw.to(kind), grad_bias=dz.sum(1))


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        entry, args, _ = state["call"]
        if entry(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) != 0:
            raise RuntimeError("%s failed: %s" % (entry.__name__, state["case"]))
        return state["out"]
    op = state["case"]["op"]
    return _plain_norm(state) if op == "norm" else _plain_linear(state) if op == "linear" else _plain_experts(state)


# ---- 64 bits ----------------------------------------------------------------------------------------

def _exact_layer(c, x, w, bias, residual, pre, grad_y):
    """One product with its epilogue, or its gradients, from the definition: w is [k][n], all in 64 bits."""
    if grad_y is None:
        z = torch.addmm(bias, x, w)
        y = {"none": lambda: z, "tanh": lambda: 2 * torch.special.expit(2 * z) - 1,
             "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * 0.5 * torch.special.erfc(-z / 2 ** 0.5),
             "silu": lambda: z * torch.special.expit(z)}[c["act"]]()
        return (y if residual is None else y + residual), z
    if c["act"] == "none":
        dz = grad_y
    else:
        leaf = pre.clone().requires_grad_(True)
        value = {"tanh": lambda: torch.tanh(leaf), "relu": lambda: torch.relu(leaf), "gelu": lambda: leaf * 0.5 * torch.special.erfc(-leaf / 2 ** 0.5),
                 "silu": lambda: leaf * torch.special.expit(leaf)}[c["act"]]()
        dz, = torch.autograd.grad(value, leaf, grad_y)
    return torch.mm(dz, w.t()), torch.mm(x.t(), dz), dz.sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: (v.to(torch.float64) if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in s.items() if k != "out"}
    if case["op"] == "norm":
        if case["way"] == "forward":
            var, mean = torch.var_mean(wide["x"], 1, unbiased=False)
            rstd = (var + EPSILON) ** -0.5
            return dict(y=torch.addcmul(wide["beta"], (wide["x"] - mean[:, None]) * rstd[:, None], wide["gamma"].expand_as(wide["x"])), mean=mean, rstd=rstd)
        # the kept mean and 1/deviation are inputs here, so the definition is the gradient's formula on them
        mean, rstd, n = wide["mean"][:, None], wide["rstd"][:, None], case["cols"]
        unit = (wide["x"] - mean) * rstd
        scaled = wide["grad_y"] * wide["gamma"]
        along = torch.einsum("rc,rc->r", scaled, unit)[:, None] / n
        dx = rstd * (scaled - scaled.mean(1, keepdim=True) - unit * along)
        if wide["grad_residual"] is not None:
            dx = dx + wide["grad_residual"]
        return dict(grad_x=dx, grad_gamma=torch.einsum("rc,rc->c", wide["grad_y"], unit), grad_beta=wide["grad_y"].sum(0))
    back, trans, acts = case["way"] == "backward", case["trans"], case["act"] != "none"
    groups = [(0, case["rows"])] if case["op"] == "linear" else list(zip(_offsets(case, seed)[:-1], _offsets(case, seed)[1:]))
    first, second, third = [], [], []
    for e, (a, b) in enumerate(groups):
        w = wide["w"] if case["op"] == "linear" else wide["w"][e]
        part = lambda t: None if t is None else t[a:b]  # noqa: E731
        bias = None if back else wide["bias"] if case["op"] == "linear" else wide["bias"][e]
        got = _exact_layer(case, part(wide["x"]), w.t() if trans else w, bias, part(wide.get("residual")), part(wide.get("pre")), part(wide.get("grad_y")))
        first.append(got[0])
        second.append((got[1].t() if trans else got[1]) if back else got[1])
        third.append(got[2] if back else None)
    if not back:
        return dict(y=torch.cat(first), **(dict(pre=torch.cat(second)) if acts else {}))
    if case["op"] == "linear":
        return dict(grad_x=first[0], grad_w=second[0].contiguous(), grad_bias=third[0])
    return dict(grad_x=torch.cat(first), grad_w=torch.stack(second), grad_bias=torch.stack(third))
