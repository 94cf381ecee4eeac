"""Shared by the tests of the transformer-block functions: inputs, the oracle's
answers and tolerances.

Tolerance of an output of type t with reference value v and terms s (the sum of
the magnitudes added up to it, from the oracle):
    |got - v| <= (eps_t / 2) |v| + depth * 2^-24 * s  (+ 2^-25 in float16, half
                                                       of its least step)
the first part is the one rounding to t.  depth counts float32 roundings along
the longest chain of an evaluation: a row sum adds at most 32 values (4 vectors
of 8) in a thread and 10 more levels over 1024 threads, and enters the result
through a root, a product and a sum (rows beyond 16384 columns add cols / 4096
vectors of 8 in a thread); two norms after one another double it: 64 per norm
and a factor of 2 in hand for the products in between: 256, with cols / 256 for
the long rows.  Column sums add a run of rows one after another, then the runs
in 16 lanes: at most rows / 64 + 64 more."""
import numpy as np
import torch

from oracle import step_ref as S

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def depth(rows, cols, column_sum):
    return 256 + cols / 256 + (rows / 64 + 64 if column_sum else 0)


def close(got, value, terms, rows, cols, name, column_sum=False):
    half = torch.finfo(got.dtype).eps / 2
    g = got.detach().double().cpu().numpy().reshape(value.shape)
    bound = half * np.abs(value) + depth(rows, cols, column_sum) * 2.0 ** -24 * terms
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    err = np.abs(g - value)
    bad = ~(err <= bound)
    if bad.any():
        i = np.unravel_index(int(np.argmax(np.where(np.isnan(err), np.inf, err - bound))), err.shape)
        raise AssertionError(f"{name}: {int(bad.sum())}/{bad.size} off; worst at {i}: got {g[i]!r} "
                             f"ref {value[i]!r} bound {np.broadcast_to(bound, err.shape)[i]:.3e}")


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


class Step:
    """One residual step: tensors on the GPU and their float64 values."""

    def __init__(self, rows, cols, dtype="f32", norm="rms", post=True, pre=True, res=True,
                 gate="none", samples=1, rs=1.0, bs=1.0, eps=1e-5, seed=0, affine=True):
        gen = torch.Generator().manual_seed(seed + rows * 7 + cols)
        self.rows, self.cols, self.dt, self.norm = rows, cols, DTYPES[dtype], norm
        self.post, self.pre, self.rs, self.bs, self.eps = post, pre, rs, bs, eps
        layer = norm == "layer"

        def n(*s):
            return torch.randn(*s, generator=gen)

        def act(scale=1.0, shift=0.0):
            return (n(rows, cols) * scale + shift).to(self.dt).cuda()
        self.x = act(2.0, 0.5)
        self.res = act(3.0) if res else None
        self.dh, self.dy = act(), act() if pre else None
        self.gp = (1 + 0.2 * n(cols)).cuda() if post and affine else None
        self.bp = (0.3 * n(cols)).cuda() if post and layer and affine else None
        self.gn = (1 + 0.2 * n(cols)).cuda() if pre and affine else None
        self.bn = (0.3 * n(cols)).cuda() if pre and layer and affine else None
        self.full = gate == "full"
        self.gate = {"none": lambda: None, "channel": lambda: (0.7 * n(1, cols)).cuda(),
                     "sample": lambda: (0.7 * n(samples, cols)).cuda(),
                     "full": lambda: act(0.7)}[gate]()

    def args(self):
        return dict(gate=self.gate, gamma_post=self.gp, beta_post=self.bp, gamma_pre=self.gn,
                    beta_pre=self.bn, norm=self.norm, post=self.post, pre=self.pre,
                    res_scale=self.rs, branch_scale=self.bs, eps=self.eps)

    def oracle_fwd(self):
        return S.step_fwd(f64(self.x), f64(self.res), f64(self.gate), f64(self.gp), f64(self.bp),
                          f64(self.gn), f64(self.bn), self.norm, self.post, self.pre, self.rs, self.bs,
                          self.eps)

    def oracle_bwd(self, x, h, stats, dh="dh"):
        cols = [None if s is None else f64(s)[:, None] for s in stats]
        zero = np.zeros((self.rows, 1))
        cols = [zero if c is None else c for c in cols]
        return S.step_bwd(x, h, f64(self.dh) if dh == "dh" else dh, f64(self.dy), cols, f64(self.gate),
                          self.full, f64(self.gp), f64(self.bp), f64(self.gn), self.norm, self.post,
                          self.pre, self.res is not None, self.rs, self.bs, self.eps)

    def check_fwd(self, f, ref=None):
        ref = self.oracle_fwd() if ref is None else ref
        r, c = self.rows, self.cols
        close(f.h, *ref["h"], r, c, "h")
        if self.pre:
            close(f.y, *ref["y"], r, c, "y")
        layer = self.norm == "layer"
        for i, k in enumerate(("post", "pre")):
            mean, var = f.stats[2 * i], f.stats[2 * i + 1]
            if not getattr(self, k):
                assert mean is None and var is None
                continue
            terms = ref["pre_terms"] if k == "pre" else (f64(self.x) ** 2).mean(1, keepdims=True)
            # the error of a mean of squares about a mean: relative to the
            # squares' own, and to mean^2 for the rounding of the mean
            close(var, ref["var_" + k][:, 0], terms[:, 0], r, c, "var_" + k)
            assert (mean is None) == (not layer)
            if layer:
                close(mean, ref["mean_" + k][:, 0], np.sqrt(terms[:, 0]), r, c, "mean_" + k)

    def check_grads(self, grads, ref):
        for name, got in grads._asdict().items():
            want = ref.get(name)
            if name.startswith("dbeta") and self.norm == "rms":
                want = None
            assert (got is None) == (want is None), name
            if got is not None:
                close(got, *want, self.rows, self.cols, name,
                      column_sum=name.startswith(("dgamma", "dbeta")) or
                      (name == "dgate" and not self.full))
