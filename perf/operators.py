"""The transformer-block normalization operators as measured work: what is
called, on which inputs, in plain torch and through this package.

Operators
  rms_fwd, rms_bwd   root-mean-square normalization of rows
  res_fwd, res_bwd   the step between two blocks of a residual stream:
                     h = res_scale*res + branch_scale*gate*post(x), y = pre(h),
                     where post and pre are row norms (either may be absent)
  act8               8-bit activation checkpoint: packed, then read back
  norm_bwd8          backward of a row norm whose input was kept in 8 bits
  res_fwd8           the step's forward that also keeps x and h in 8 bits for the
                     backward; the copies are read back
  res_bwd8           the step's backward from those copies
"""
import importlib.util
import math
import os
import sys

import torch

own = False

GROUP = 32           # columns that share one scale of an 8-bit checkpoint
EPS = 1e-5

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _package():
    """This repository's package (its directory name is not an identifier)."""
    name = "nnabla_ext_cuda_amd"
    if name not in sys.modules:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                            "nnabla-ext-cuda_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def _case(name, op, dtype, rows, cols, norm="rms", post=True, pre=True, res=True, gate="none",
          samples=1, form="int8", res_scale=1.0, branch_scale=1.0):
    """gate: none | channel (one row for all tokens) | sample (one row per
    sample of rows/samples tokens) | full (an element each).  form: of the
    8-bit copies, where there are any."""
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "norm": norm,
            "post": post, "pre": pre, "res": res, "gate": gate, "samples": samples, "form": form,
            "res_scale": res_scale, "branch_scale": branch_scale}


def listed():
    return [
        # Serving: one new token of a sandwich-norm decoder with layer scale; latency is all.
        _case("step_fwd_one_token", "res_fwd", "bf16", 1, 4096, gate="channel"),
        # Serving: a batch of single tokens of a pre-norm decoder (add, then LayerNormalization).
        _case("step_fwd_decode_batch", "res_fwd", "f16", 48, 2560, norm="layer", post=False),
        # Prefill or training: 16K tokens of a sandwich-norm decoder with layer scale.
        _case("step_fwd_16k_tokens", "res_fwd", "bf16", 16384, 4096, gate="channel",
              branch_scale=0.5),
        # Training of a conditioned transformer: 32 samples of 512 tokens, a gate row per sample.
        _case("step_bwd_sample_gate", "res_bwd", "f16", 16384, 1024, norm="layer", gate="sample",
              samples=32),
        # Training of the widest hidden size, the largest tensors here.
        _case("step_bwd_wide", "res_bwd", "bf16", 8192, 8192, gate="channel", res_scale=0.8),
        # Training in float with rows that no vector divides and a gate computed per element.
        _case("step_bwd_odd_full_gate", "res_bwd", "f32", 1531, 1027, norm="layer", gate="full"),
        # Normalized queries and keys: very many rows of one head.
        _case("rms_fwd_heads", "rms_fwd", "f16", 131072, 128),
        # Training of a pre-norm decoder.
        _case("rms_bwd_4k_tokens", "rms_bwd", "bf16", 4096, 8192),
        # A checkpoint of a layer's input: written in the forward, read back in the backward.
        _case("act8_int8_16k_tokens", "act8", "bf16", 16384, 4096, form="int8"),
        # A training forward that keeps 8-bit copies, rows that end inside a group.
        _case("step_fwd8_e4m3_ragged", "res_fwd8", "f16", 5003, 1000, gate="channel", form="e4m3"),
        # LayerNormalization backward from an 8-bit input: 32 sequences of 512.
        _case("norm_bwd8_layer", "norm_bwd8", "f16", 16384, 1024, norm="layer", form="int8"),
        # Training of a sandwich-norm decoder from the 8-bit copies of its forward.
        _case("step_bwd8_e4m3", "res_bwd8", "bf16", 8192, 4096, gate="channel", form="e4m3"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms_fwd", "rms_bwd", "res_fwd", "res_bwd", "act8", "norm_bwd8", "res_fwd8",
                     "res_bwd8"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cols = _log_uniform(rng, 64, 16384)
    if rng.random() < 0.7:      # most models' sizes are round ones
        cols = max(64, cols // 64 * 64)
    cap = (1 << 24) if dtype == "f32" else (1 << 25)
    rows = _log_uniform(rng, 1, min(131072, max(1, cap // cols)))
    post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
    if op == "res_fwd8" and dtype == "f32":
        post, pre = True, False     # a float h next to a step of its 8-bit copy may go either way
    gate = rng.choice(["none", "channel", "sample", "full"])
    samples = 1
    if gate == "sample":
        samples = _log_uniform(rng, 1, min(64, rows))
        rows = rows // samples * samples
    return {"op": op, "dtype": dtype, "rows": rows, "cols": cols,
            "norm": rng.choice(["rms", "layer"]), "post": post, "pre": pre,
            "res": rng.random() < 0.9, "gate": gate, "samples": samples,
            "form": rng.choice(["int8", "e4m3"]), "res_scale": rng.choice([1.0, 0.8, 1.25]),
            "branch_scale": rng.choice([1.0, 0.5])}


def work(case):
    n, e = case["rows"] * case["cols"], 2 if case["dtype"] != "f32" else 4
    packed = n + case["rows"] * -(-case["cols"] // GROUP)
    op, layer = case["op"], case["norm"] == "layer"
    stat = 4 * case["rows"] * (2 if layer else 1)
    par = 4 * case["cols"] * (2 if layer else 1)
    post, pre, gated = case["post"], case["pre"], case["gate"] != "none"
    gate_bytes = {"none": 0, "channel": 4 * case["cols"],
                  "sample": 4 * case["cols"] * case["samples"], "full": n * e}[case["gate"]]
    norms = int(post) + int(pre)
    fwd = n * e * (2 + int(case["res"]) + int(pre)) + gate_bytes + norms * (par + stat)
    fwd_flops = n * (10 * norms + 4)
    reads_x = post or gated
    bwd_tensors = 2 + int(case["res"]) + int(pre)          # dh, dx, dres, dy
    bwd = n * e * bwd_tensors + 2 * gate_bytes + norms * (2 * par + stat)
    bwd_flops = n * (16 * norms + 6)
    if op == "rms_fwd":
        return {"bytes": 2 * n * e + 4 * case["cols"] + 4 * case["rows"], "flops": 5 * n}
    if op == "rms_bwd":
        return {"bytes": 3 * n * e + 8 * case["cols"] + 4 * case["rows"], "flops": 12 * n}
    if op == "res_fwd":
        return {"bytes": fwd, "flops": fwd_flops}
    if op == "res_bwd":
        return {"bytes": bwd + n * e * (int(reads_x) + int(pre)), "flops": bwd_flops}
    if op == "act8":
        return {"bytes": 2 * (n * e + packed), "flops": 4 * n}
    if op == "norm_bwd8":
        return {"bytes": packed + 2 * n * e + 2 * par + stat, "flops": 14 * n}
    copies = int(reads_x) + int(pre)
    if op == "res_fwd8":                                    # copies written, read, written out
        return {"bytes": fwd + copies * (2 * packed + n * e), "flops": fwd_flops + 4 * n * copies}
    return {"bytes": bwd + copies * packed, "flops": bwd_flops}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _inputs(case, seed):
    """Activations as deep networks have them: unit-scale values, one channel in
    a hundred twenty times larger; gradients of unit scale; parameters near one."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, cols = DTYPES[case["dtype"]], case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    channel = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    layer = case["norm"] == "layer"
    st = {"x": (normal(rows, cols) * channel + 0.1).to(dt)}
    for which in ("post", "pre"):
        st["gamma_" + which] = 1 + 0.1 * normal(cols)
        st["beta_" + which] = 0.1 * normal(cols) if layer else None
    if case["op"].startswith("res"):
        st["res"] = (normal(rows, cols) * channel * 2).to(dt) if case["res"] else None
        st["gate"] = {"none": lambda: None,
                      "channel": lambda: 0.5 + 0.2 * normal(1, cols),
                      "sample": lambda: 0.5 * normal(case["samples"], cols),
                      "full": lambda: (0.5 * normal(rows, cols)).to(dt)}[case["gate"]]()
        if not case["post"]:
            st["gamma_post"] = st["beta_post"] = None
        if not case["pre"]:
            st["gamma_pre"] = st["beta_pre"] = None
    # A backward pass starts from what its forward kept.
    if case["op"] in ("rms_bwd", "norm_bwd8"):
        st["dy"] = normal(rows, cols).to(dt)
        mean, var = _stats(st["x"].double(), case["op"] == "norm_bwd8" and layer)
        st["mean"], st["var"] = None if mean is None else mean.float(), var.float()
    if case["op"] in ("res_bwd", "res_bwd8"):
        st["dh"] = normal(rows, cols).to(dt)
        st["dy"] = normal(rows, cols).to(dt) if case["pre"] else None
        h, _, stats = _plain_step(st, case, torch.float64)
        st["h"], st["stats"] = h, tuple(None if t is None else t.float() for t in stats)
    if case["op"] == "norm_bwd8":
        st["x"] = _plain_pack(st["x"], case["form"])
    if case["op"] == "res_bwd8":
        reads_x = case["post"] or st["gate"] is not None
        st["x"] = _plain_pack(st["x"], case["form"]) if reads_x else None
        st["h"] = _plain_pack(st["h"], case["form"]) if case["pre"] else None
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = dict(case)
    return st


# --------------------------------------------------------------------------
# The plain forms: elementary torch operations in float32, rounded at the end
# --------------------------------------------------------------------------
def _stats(x, layer):
    """(mean or None, variance or mean square) of each row."""
    if layer:
        mean = x.mean(1)
        d = x - mean[:, None]
        return mean, (d * d).mean(1)
    return None, (x * x).mean(1)


def _unit(x, stats):
    mean, var = stats
    d = x if mean is None else x - mean[:, None]
    return d * (1.0 / torch.sqrt(var + EPS))[:, None]


def _affine(xh, gamma, beta):
    y = xh * gamma
    return y if beta is None else y + beta


def _gate_rows(gate, rows):
    """The gate as float, a row per token."""
    g = gate.float()
    return g if g.shape[0] in (1, rows) else g.repeat_interleave(rows // g.shape[0], 0)


def _plain_step(st, case, wide=torch.float32):
    """h and y, rounded, and the statistics (mean_post, var_post, mean_pre, var_pre)."""
    dt, layer = st["x"].dtype, case["norm"] == "layer"
    u = st["x"].to(wide)
    post = pre = (None, None)
    if case["post"]:
        post = _stats(u, layer)
        u = _affine(_unit(u, post), st["gamma_post"], st["beta_post"])
    if st["gate"] is not None:
        u = u * _gate_rows(st["gate"], case["rows"])
    h = u * case["branch_scale"]
    if st["res"] is not None:
        h = h + case["res_scale"] * st["res"].to(wide)
    y = None
    if case["pre"]:
        pre = _stats(h, layer)
        y = _affine(_unit(h, pre), st["gamma_pre"], st["beta_pre"]).to(dt)
    return h.to(dt), y, post + pre


def _plain_norm_bwd(x, dy, gamma, stats, layer):
    """dx, dgamma, dbeta (None for rms) in float32."""
    xh = _unit(x, stats)
    g = dy * gamma
    dx = g - xh * (g * xh).mean(1)[:, None]
    if layer:
        dx = dx - g.mean(1)[:, None]
    dx = dx * (1.0 / torch.sqrt(stats[1] + EPS))[:, None]
    return dx, (dy * xh).sum(0), dy.sum(0) if layer else None


def _plain_step_bwd(st, x, h):
    case, stats = st["case"], st["stats"]
    dt, layer, rows = st["dh"].dtype, case["norm"] == "layer", case["rows"]
    dh = st["dh"].float()
    out = dict.fromkeys(("dx", "dres", "dgate", "dgamma_post", "dbeta_post", "dgamma_pre",
                         "dbeta_pre"))
    if case["pre"]:
        d, out["dgamma_pre"], out["dbeta_pre"] = _plain_norm_bwd(
            h, st["dy"].float(), st["gamma_pre"], stats[2:], layer)
        dh = dh + d
    if st["res"] is not None:
        out["dres"] = (case["res_scale"] * dh).to(dt)
    du = case["branch_scale"] * dh
    if st["gate"] is not None:
        u = x
        if case["post"]:
            u = _affine(_unit(u, stats[:2]), st["gamma_post"], st["beta_post"])
        dg = du * u
        groups = st["gate"].shape[0]
        if case["gate"] != "full":
            dg = dg.view(groups, rows // groups, -1).sum(1)
        out["dgate"] = dg.to(st["gate"].dtype)
        du = du * _gate_rows(st["gate"], rows)
    if case["post"]:
        du, out["dgamma_post"], out["dbeta_post"] = _plain_norm_bwd(
            x, du, st["gamma_post"], stats[:2], layer)
    out["dx"] = du.to(dt)
    return [v for v in out.values() if v is not None]


def _power_of_two(k):
    """2^k of integers in [-126, 127], exactly: the exponent field of a float."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _plain_pack(x, form):
    """q [rows, cols] and the scale's exponent code [rows, groups]: x is about
    q * 2^(code - 127), with the least scale, not below 2^-120, at which the
    group's largest magnitude fits (int8: rounds to 127 or less; e4m3: is 448 or
    less).  A group with an infinity or NaN holds q = 0 and the code 255, NaN."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    v = torch.zeros(rows, groups * GROUP, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, groups, GROUP)
    amax = v.abs().amax(2)
    finite = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(finite, amax, torch.ones_like(amax)))   # m * 2^e, m < 1
    if form == "int8":
        k = e - 7 + (m >= 127.5 / 128).int()
        stored = torch.int8
    else:
        k = e - 9 + (m > 448.0 / 512).int()
        stored = torch.float8_e4m3fn
    k = torch.where(amax > 0, k, torch.full_like(k, -120)).clamp_min(-120)
    q = v * _power_of_two(-k)[:, :, None]
    q = torch.where(finite[:, :, None], q, torch.zeros_like(q))
    if form == "int8":
        q = torch.round(q)
    code = torch.where(finite, k + 127, torch.full_like(k, 255)).to(torch.uint8)
    return q.view(rows, -1)[:, :cols].contiguous().to(stored), code


def _plain_unpack(q, code):
    scale = _power_of_two(code.int() - 127)
    scale = torch.where(code == 255, torch.full_like(scale, float("nan")), scale)
    return q.float() * scale.repeat_interleave(GROUP, 1)[:, :q.shape[1]]


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def _run_plain(st):
    case = st["case"]
    op, layer, x = case["op"], case["norm"] == "layer", st["x"]
    if op == "rms_fwd":
        stats = _stats(x.float(), False)
        return [_affine(_unit(x.float(), stats), st["gamma_post"], None).to(x.dtype), stats[1]]
    if op == "act8":
        return [_plain_unpack(*_plain_pack(x, case["form"])).to(x.dtype)]
    if op in ("rms_bwd", "norm_bwd8"):
        wide = _plain_unpack(*x) if op == "norm_bwd8" else x.float()
        dx, dg, db = _plain_norm_bwd(wide, st["dy"].float(), st["gamma_post"],
                                     (st["mean"], st["var"]), layer and op == "norm_bwd8")
        return [t for t in (dx.to(st["dy"].dtype), dg, db) if t is not None]
    if op == "res_bwd":
        return _plain_step_bwd(st, x.float(), st["h"].float())
    if op == "res_bwd8":
        return _plain_step_bwd(st, *(None if t is None else _plain_unpack(*t)
                                     for t in (x, st["h"])))
    h, y, stats = _plain_step(st, case)
    out = [t for t in (h, y) + tuple(stats) if t is not None]
    if op == "res_fwd8":
        kept = ([x] if case["post"] or st["gate"] is not None else []) + ([h] if case["pre"] else [])
        out += [_plain_unpack(*_plain_pack(t, case["form"])).to(t.dtype) for t in kept]
    return out


def _run_own(st):
    case, k = st["case"], _package()
    op, rows = case["op"], case["rows"]
    x, h = (k.Act8(*t) if isinstance(t, tuple) else t for t in (st["x"], st.get("h")))
    if op == "rms_fwd":
        return list(k.rms_forward(x, st["gamma_post"], rows, EPS))
    if op == "act8":
        return [k.act8_unpack(k.act8_pack(x, rows, case["form"]), rows, x.dtype)]
    if op == "norm_bwd8" and case["norm"] == "layer":
        return list(k.ln_backward_act8(x, st["dy"], st["gamma_post"], st["mean"], st["var"], rows,
                                       EPS))
    if op in ("rms_bwd", "norm_bwd8"):
        return list(k.rms_backward(x, st["dy"], st["gamma_post"], st["var"], rows, EPS))
    args = dict(gate=st["gate"], gamma_post=st["gamma_post"], beta_post=st["beta_post"],
                gamma_pre=st["gamma_pre"], beta_pre=st["beta_pre"], norm=case["norm"],
                post=case["post"], pre=case["pre"], res_scale=case["res_scale"],
                branch_scale=case["branch_scale"], eps=EPS)
    if op in ("res_bwd", "res_bwd8"):
        grads = k.resnorm_backward(x, h, st["dh"], st["dy"], st["stats"], rows,
                                   has_res=st["res"] is not None, **args)
        return [g for g in grads if g is not None]
    f = k.resnorm_forward(x, st["res"], rows, checkpoint=case["form"] if op == "res_fwd8" else None,
                          **args)
    out = [t for t in (f.h, f.y) + tuple(f.stats) if t is not None]
    return out + [k.act8_unpack(t, rows, x.dtype) for t in (f.x8, f.h8) if t is not None]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_moments(x, norm):
    """Row mean (zero for rms), second moment about it."""
    mu = x.mean(dim=1, keepdim=True) if norm == "layer" else torch.zeros_like(x[:, :1])
    return mu, ((x - mu) ** 2).mean(dim=1, keepdim=True)


def _exact_norm_vjp(v, grad, gamma, mu, var, norm):
    """Gradients of gamma * (v - mu) / sqrt(var + eps) + beta for given moments."""
    inv = (var + EPS) ** -0.5
    unit = (v - mu) * inv
    w = grad * gamma
    centred = w - w.mean(dim=1, keepdim=True) if norm == "layer" else w
    dv = inv * (centred - unit * (w * unit).mean(dim=1, keepdim=True))
    return dv, (grad * unit).sum(dim=0), grad.sum(dim=0)


def _exact_power(k):
    """2^k in 64 bits, exactly."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _exact_value(copy):
    """What an 8-bit copy (codes, exponent codes) stands for."""
    codes, exponents = copy
    column = torch.arange(codes.shape[1], device=codes.device) // GROUP
    return codes.double() * _exact_power(exponents.long() - 127)[:, column]


def _exact_round_trip(v, form):
    """The values that an 8-bit copy of v holds."""
    out = torch.empty_like(v)
    for c0 in range(0, v.shape[1], GROUP):
        part = v[:, c0:c0 + GROUP]
        mantissa, power = torch.frexp(part.abs().max(dim=1, keepdim=True).values)
        power = torch.where(mantissa > 0, power, torch.full_like(power, -200))
        if form == "int8":      # integers to 127: the least step that rounds no value to 128
            step = _exact_power((power - 7 + (128 * mantissa >= 127.5)).clamp(min=-120))
            out[:, c0:c0 + GROUP] = torch.round(part / step) * step
        else:                   # three mantissa bits, exponents from 2^-6, at most 448
            step = _exact_power((power - 9 + (512 * mantissa > 448)).clamp(min=-120))
            z = part / step
            _, p = torch.frexp(z)
            ulp = _exact_power(torch.where(z == 0, torch.full_like(p, -5), p).clamp(min=-5) - 4)
            out[:, c0:c0 + GROUP] = torch.round(z / ulp) * ulp * step
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    op, norm, rows = case["op"], case["norm"], case["rows"]
    layer = norm == "layer"
    d = {k: v.double() for k, v in st.items() if torch.is_tensor(v)}
    d.update({k: _exact_value(st[k]) for k in ("x", "h") if isinstance(st.get(k), tuple)})
    x = d.get("x")
    if op == "act8":
        return [_exact_round_trip(x, case["form"])]
    if op == "rms_fwd":
        _, var = _exact_moments(x, "rms")
        return [x * (var + EPS) ** -0.5 * d["gamma_post"], var[:, 0]]
    if op in ("rms_bwd", "norm_bwd8"):
        kind = "rms" if op == "rms_bwd" else norm
        mu = d["mean"][:, None] if "mean" in d else torch.zeros_like(x[:, :1])
        dx, dg, db = _exact_norm_vjp(x, d["dy"], d["gamma_post"], mu, d["var"][:, None], kind)
        return [dx, dg, db] if kind == "layer" else [dx, dg]

    gate = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    if "gate" in d:
        gate = d["gate"][torch.arange(rows, device="cuda") * d["gate"].shape[0] // rows]
    if op in ("res_fwd", "res_fwd8"):
        kept = []                   # moments in the order the forward returns them
        u = x
        if case["post"]:
            mu, var = _exact_moments(x, norm)
            kept += ([mu[:, 0]] if layer else []) + [var[:, 0]]
            u = (x - mu) * (var + EPS) ** -0.5 * d["gamma_post"]
            if layer:
                u = u + d["beta_post"]
        h = case["branch_scale"] * gate * u
        if "res" in d:
            h = h + case["res_scale"] * d["res"]
        out = [h]
        if case["pre"]:
            mu, var = _exact_moments(h, norm)
            kept += ([mu[:, 0]] if layer else []) + [var[:, 0]]
            y = (h - mu) * (var + EPS) ** -0.5 * d["gamma_pre"]
            out.append(y + d["beta_pre"] if layer else y)
        out += kept
        if op == "res_fwd8":
            if case["post"] or "gate" in d:
                out.append(_exact_round_trip(x, case["form"]))
            if case["pre"]:
                out.append(_exact_round_trip(h.to(st["x"].dtype).double(), case["form"]))
        return out

    # the step's backward, from what its forward kept
    moments = [None if t is None else t.double()[:, None] for t in st["stats"]]
    zero = torch.zeros(rows, 1, dtype=torch.float64, device="cuda")
    mu1, var1, mu2, var2 = moments
    grad_h, pre_grads = d["dh"], []
    if case["pre"]:
        back, dg, db = _exact_norm_vjp(d["h"], d["dy"], d["gamma_pre"],
                                       zero if mu2 is None else mu2, var2, norm)
        grad_h = grad_h + back
        pre_grads = [dg, db] if layer else [dg]
    u = x
    if case["post"]:
        mu1 = zero if mu1 is None else mu1
        u = (x - mu1) * (var1 + EPS) ** -0.5 * d["gamma_post"]
        if layer:
            u = u + d["beta_post"]
    grad_u = case["branch_scale"] * grad_h * gate
    gate_grad, post_grads, grad_x = [], [], grad_u
    if "gate" in d:
        per_token = case["branch_scale"] * grad_h * u
        groups = d["gate"].shape[0]
        gate_grad = [per_token.reshape(groups, rows // groups, -1).sum(dim=1)]
    if case["post"]:
        grad_x, dg, db = _exact_norm_vjp(x, grad_u, d["gamma_post"], mu1, var1, norm)
        post_grads = [dg, db] if layer else [dg]
    return ([grad_x] + ([case["res_scale"] * grad_h] if "res" in d else []) + gate_grad
            + post_grads + pre_grads)
