"""ctypes binding of the nblahip C-ABI (include/nblahip.h) for tests, the
smoke check and the benchmark.

The product is the C/C++ library; this module only hands it device pointers.
torch supplies device memory and the current stream, nothing else: there is
no fallback implementation here, and loading fails loudly when the HIP
library has not been built.
"""
from __future__ import annotations

import collections
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libnblahip.so")
HOST_LIB_PATH = os.path.join(_HERE, "lib", "libnnabla_hip.so")
CSRC = os.path.join(_HERE, "csrc")

F32, F16, BF16 = 0, 1, 2

_c_void_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f = ctypes.c_float
_sz = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/nblahip.h one to one.
SIGNATURES = {
    "nblahip_error_string": (ctypes.c_char_p, [_int]),
    "nblahip_abi_version": (_int, []),
    "nblahip_bn_fwd_infer": (_int, [_c_void_p] * 6 + [_i64] * 3 + [_f, _int, _c_void_p]),
    "nblahip_bn_workspace_bytes": (_sz, [_i64] * 3 + [_int]),
    "nblahip_bn_fwd_train": (_int, [_c_void_p] * 8 + [_i64] * 3 + [_f, _f, _int, _c_void_p, _sz,
                                                              _c_void_p]),
    "nblahip_bn_fwd_train_static_max_workspace": (_sz, []),
    "nblahip_bn_fwd_train_static": (_int, [_c_void_p] * 8 + [_i64] * 3 + [_f, _f, _int, _c_void_p]),
    "nblahip_bn_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 3 + [_f, _int, _int,
                                                                   _c_void_p, _sz, _c_void_p]),
    "nblahip_bn_local_stats": (_int, [_c_void_p] * 3 + [_i64] * 3 + [_int, _c_void_p, _sz, _c_void_p]),
    "nblahip_bn_merge_stats": (_int, [_c_void_p, _int, _i64] + [_c_void_p] * 4 + [_f, _c_void_p]),
    "nblahip_bn_bwd_local_sums": (_int, [_c_void_p] * 7 + [_int, _int] + [_i64] * 3 + [_f, _int,
                                                                          _c_void_p, _sz, _c_void_p]),
    "nblahip_bn_bwd_apply_sums": (_int, [_c_void_p] * 6 + [ctypes.c_double] + [_c_void_p] * 3 +
                                  [_int] + [_i64] * 3 + [_f, _int, _c_void_p, _sz, _c_void_p]),
    "nblahip_fused_bn_fwd_infer": (_int, [_c_void_p] * 7 + [_i64] * 3 + [_f, _int, _c_void_p]),
    "nblahip_fused_bn_fwd_train": (_int, [_c_void_p] * 9 + [_i64] * 3 + [_f, _f, _int, _c_void_p,
                                                                         _sz, _c_void_p]),
    "nblahip_fused_bn_bwd": (_int, [_c_void_p] * 12 + [_int] * 4 + [_i64] * 3 + [_f, _int, _int,
                                                                         _c_void_p, _sz, _c_void_p]),
    "nblahip_ln_fwd": (_int, [_c_void_p] * 6 + [_i64] * 2 + [_f, _int, _c_void_p]),
    "nblahip_ln_bwd_workspace_bytes": (_sz, [_i64] * 2 + [_int]),
    "nblahip_ln_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 2 + [_f, _int, _c_void_p,
                                                                   _sz, _c_void_p]),
    "nblahip_gn_fwd": (_int, [_c_void_p] * 6 + [_i64] * 3 + [_int, _f, _int, _c_void_p]),
    "nblahip_gn_bwd_workspace_bytes": (_sz, [_i64] * 3 + [_int, _int]),
    "nblahip_gn_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 3 + [_int, _f, _int,
                                                                   _c_void_p, _sz, _c_void_p]),
    "nblahip_in_fwd": (_int, [_c_void_p] * 6 + [_i64] * 3 + [_int, _int, _f, _int, _c_void_p]),
    "nblahip_in_bwd_workspace_bytes": (_sz, [_i64] * 3 + [_int]),
    "nblahip_in_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 3 + [_int, _int, _f, _int,
                                                                   _c_void_p, _sz, _c_void_p]),
    "nblahip_gn_cl_workspace_bytes": (_sz, [_i64] * 3 + [_int, _int]),
    "nblahip_gn_cl_fwd": (_int, [_c_void_p] * 6 + [_i64] * 3 + [_int, _f, _int, _c_void_p, _sz,
                                                                _c_void_p]),
    "nblahip_gn_cl_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 3 + [_int, _f, _int,
                                                                      _c_void_p, _sz, _c_void_p]),
    "nblahip_in_cl_workspace_bytes": (_sz, [_i64] * 3 + [_int]),
    "nblahip_in_cl_fwd": (_int, [_c_void_p] * 6 + [_i64] * 3 + [_int, _int, _f, _int, _c_void_p,
                                                                _sz, _c_void_p]),
    "nblahip_in_cl_bwd": (_int, [_c_void_p] * 10 + [_int] * 3 + [_i64] * 3 + [_int, _int, _f, _int,
                                                                      _c_void_p, _sz, _c_void_p]),
    "nblahip_act8_scales_per_row": (_i64, [_i64]),
    "nblahip_act8_pack": (_int, [_c_void_p] * 3 + [_i64] * 2 + [_int, _int, _c_void_p]),
    "nblahip_act8_unpack": (_int, [_c_void_p] * 3 + [_i64] * 2 + [_int, _int, _c_void_p]),
    "nblahip_rms_fwd": (_int, [_c_void_p] * 4 + [_i64] * 2 + [_f, _int, _c_void_p]),
    "nblahip_rms_bwd_workspace_bytes": (_sz, [_i64] * 2 + [_int]),
    "nblahip_rms_bwd": (_int, [_c_void_p] * 2 + [_int] + [_c_void_p] * 5 + [_int] * 2 + [_i64] * 2 +
                        [_f, _int, _c_void_p, _sz, _c_void_p]),
    "nblahip_ln_bwd_act8_workspace_bytes": (_sz, [_i64] * 2 + [_int]),
    "nblahip_ln_bwd_act8": (_int, [_c_void_p] * 2 + [_int] + [_c_void_p] * 7 + [_int] * 3 +
                            [_i64] * 2 + [_f, _int, _c_void_p, _sz, _c_void_p]),
    "nblahip_resnorm_fwd": (_int, [_c_void_p] * 3 + [_int, _i64] + [_c_void_p] * 14 + [_int] +
                            [_i64] * 2 + [_f] * 3 + [_int] * 4 + [_c_void_p]),
    "nblahip_resnorm_bwd_workspace_bytes": (_sz, [_i64] * 2 + [_int, _i64] + [_int] * 4),
    "nblahip_resnorm_bwd": (_int, [_c_void_p] * 4 + [_int] + [_c_void_p] * 3 + [_int, _i64] +
                            [_c_void_p] * 14 + [ctypes.c_uint] + [_i64] * 2 + [_f] * 3 + [_int] * 4 +
                            [_c_void_p, _sz, _c_void_p]),
    "nblahip_device_count": (_int, [ctypes.POINTER(_int)]),
    "nblahip_set_device": (_int, [_int]),
    "nblahip_get_device": (_int, [ctypes.POINTER(_int)]),
    "nblahip_device_synchronize": (_int, []),
    "nblahip_stream_synchronize": (_int, [_c_void_p]),
    "nblahip_device_info": (_int, [_int, ctypes.c_char_p, _sz, ctypes.POINTER(_int),
                                   ctypes.POINTER(_int), ctypes.POINTER(_sz)]),
    "nblahip_malloc": (_int, [ctypes.POINTER(_c_void_p), _sz]),
    "nblahip_free": (_int, [_c_void_p]),
    "nblahip_host_malloc": (_int, [ctypes.POINTER(_c_void_p), _sz]),
    "nblahip_host_free": (_int, [_c_void_p]),
    "nblahip_memcpy_h2d": (_int, [_c_void_p, _c_void_p, _sz, _c_void_p]),
    "nblahip_memcpy_d2h": (_int, [_c_void_p, _c_void_p, _sz, _c_void_p]),
    "nblahip_memcpy_d2d": (_int, [_c_void_p, _c_void_p, _sz, _c_void_p]),
    "nblahip_memcpy_h2d_async": (_int, [_c_void_p, _c_void_p, _sz, _c_void_p]),
    "nblahip_memcpy_d2h_async": (_int, [_c_void_p, _c_void_p, _sz, _c_void_p]),
    "nblahip_stream_create": (_int, [ctypes.POINTER(_c_void_p)]),
    "nblahip_stream_destroy": (_int, [_c_void_p]),
    "nblahip_event_create": (_int, [ctypes.POINTER(_c_void_p)]),
    "nblahip_event_destroy": (_int, [_c_void_p]),
    "nblahip_event_record": (_int, [_c_void_p, _c_void_p]),
    "nblahip_stream_wait_event": (_int, [_c_void_p, _c_void_p]),
    "nblahip_event_synchronize": (_int, [_c_void_p]),
    "nblahip_event_query": (_int, [_c_void_p, ctypes.POINTER(_int)]),
    "nblahip_memset": (_int, [_c_void_p, _int, _sz, _c_void_p]),
    "nblahip_convert": (_int, [_c_void_p, _int, _c_void_p, _int, _i64, _c_void_p]),
    "nblahip_fill": (_int, [_c_void_p, _int, _f, _i64, _c_void_p]),
    "nblahip_fill_bytes": (_int, [_c_void_p, _int, ctypes.c_ulonglong, _i64, _c_void_p]),
    "nblahip_permute": (_int, [_c_void_p, _c_void_p, _int, ctypes.POINTER(_i64),
                               ctypes.POINTER(_int), _int, _int, _c_void_p]),
    "nblahip_profile_enable": (_int, [_int]),
    "nblahip_profile_reset": (_int, []),
    "nblahip_profile_query": (_int, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_double),
                                     ctypes.POINTER(_i64)]),
    "nblahip_profile_kernels": (_int, [ctypes.c_char_p, _sz, ctypes.POINTER(_sz)]),
    "nblahip_tune_set": (_int, [ctypes.c_char_p, _int]),
    "nblahip_tune_get": (_int, [ctypes.c_char_p, _int]),
    "nblahip_tune_reset": (_int, []),
    "nblahip_xchg_set_epoch": (_int, [ctypes.c_uint]),
    "nblahip_stage_params": (_int, [_int, ctypes.POINTER(_c_void_p), _int, ctypes.POINTER(_c_void_p),
                                    _int, ctypes.POINTER(_i64), _c_void_p]),
}

_lib = None


class NblaHipError(RuntimeError):
    def __init__(self, code, text):
        super().__init__(f"nblahip status {code}: {text}")
        self.code = code


def lib():
    """The loaded libnblahip.so.  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C {CSRC} -j8` "
                "(or __graft_entry__.build()); there is no fallback path")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def check(code):
    if code != 0:
        raise NblaHipError(code, lib().nblahip_error_string(code).decode())


def profile_query(kernel_name):
    """(total_ms, launches) of the recorded launches of one kernel."""
    total = ctypes.c_double(0.0)
    count = _i64(0)
    check(lib().nblahip_profile_query(kernel_name.encode(), ctypes.byref(total),
                                      ctypes.byref(count)))
    return total.value, count.value


def profile_kernels():
    """Names of the kernels recorded since the last profile reset, in order of
    first launch."""
    need = _sz(0)
    check(lib().nblahip_profile_kernels(None, 0, ctypes.byref(need)))
    buf = ctypes.create_string_buffer(need.value)
    check(lib().nblahip_profile_kernels(buf, need.value, ctypes.byref(need)))
    return [n for n in buf.value.decode().split("\n") if n]


def tune_set(name, value):
    """Override plan knob NBLAHIP_<name> from the next call on (-1: undo)."""
    check(lib().nblahip_tune_set(name.encode(), int(value)))


def tune_get(name, fallback=-1):
    return lib().nblahip_tune_get(name.encode(), int(fallback))


def tune_reset():
    check(lib().nblahip_tune_reset())


# ---------------------------------------------------------------------------
# torch-tensor conveniences (device memory + current stream only)
# ---------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def _dtype_code(t):
    import torch
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.float16:
        return F16
    raise TypeError(f"unsupported activation dtype {t.dtype}")


def _f32(t, name):
    import torch
    if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
        raise TypeError(f"{name} must be a contiguous float32 tensor")
    return t


def _workspace(nbytes, device):
    import torch
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _bn_sizes(shape, axis):
    size0 = 1
    for s in shape[:axis]:
        size0 *= s
    size2 = 1
    for s in shape[axis + 1:]:
        size2 *= s
    return size0, shape[axis], size2


def bn_forward_global(x, beta, gamma, rmean, rvar, axis=1, eps=1e-5):
    import torch
    assert x.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    y = torch.empty_like(x)
    check(lib().nblahip_bn_fwd_infer(_ptr(x), _ptr(_f32(rmean, "rmean")), _ptr(_f32(rvar, "rvar")),
                                     _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")), _ptr(y),
                                     s0, c, s2, eps, _dtype_code(x), _stream()))
    return y


def bn_forward_batch(x, beta, gamma, rmean, rvar, axis=1, decay_rate=0.9, eps=1e-5, ws=None,
                     y=None):
    """Returns y, batch_mean, batch_var; rmean/rvar are updated in place.
    y: the output tensor (x itself for an in-place call); allocated when None."""
    import torch
    assert x.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    y = torch.empty_like(x) if y is None else y
    mean = torch.empty(c, dtype=torch.float32, device=x.device)
    var = torch.empty(c, dtype=torch.float32, device=x.device)
    need = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(need, x.device)
    check(lib().nblahip_bn_fwd_train(_ptr(x), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")),
                                     _ptr(y), _ptr(mean), _ptr(var), _ptr(_f32(rmean, "rmean")),
                                     _ptr(_f32(rvar, "rvar")), s0, c, s2, decay_rate, eps, dt,
                                     _ptr(ws), ws.numel(), _stream()))
    return y, mean, var


def bn_forward_batch_static(x, beta, gamma, rmean, rvar, axis=1, decay_rate=0.9, eps=1e-5,
                            out=None):
    """bn_forward_batch through the entry point that allocates nothing; out =
    (y, mean, var) preallocated by the caller (allocated here when None)."""
    import torch
    assert x.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    if out is None:
        out = (torch.empty_like(x), torch.empty(c, dtype=torch.float32, device=x.device),
               torch.empty(c, dtype=torch.float32, device=x.device))
    y, mean, var = out
    check(lib().nblahip_bn_fwd_train_static(
        _ptr(x), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")), _ptr(y), _ptr(mean),
        _ptr(var), _ptr(_f32(rmean, "rmean")), _ptr(_f32(rvar, "rvar")), s0, c, s2, decay_rate,
        eps, _dtype_code(x), _stream()))
    return y, mean, var


def bn_backward(x, dy, gamma, mean, var, axis=1, eps=1e-5, batch_stat=True, dmean=None,
                dvar=None, dx=None, dgamma=None, dbeta=None, accum=(False, False, False),
                need=(True, True, True), ws=None):
    """need = (dx, dgamma, dbeta) propagate_down flags; accum likewise.
    Returns dx, dgamma, dbeta (None where not needed)."""
    import torch
    assert x.is_contiguous() and dy.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    if need[0] and dx is None:
        dx = torch.empty_like(x)
    if need[1] and dgamma is None:
        dgamma = torch.empty(c, dtype=torch.float32, device=x.device)
    if need[2] and dbeta is None:
        dbeta = torch.empty(c, dtype=torch.float32, device=x.device)
    nbytes = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(nbytes, x.device)
    check(lib().nblahip_bn_bwd(_ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var),
                               _ptr(dmean), _ptr(dvar), _ptr(dx if need[0] else None),
                               _ptr(dgamma if need[1] else None), _ptr(dbeta if need[2] else None),
                               int(accum[0]), int(accum[1]), int(accum[2]), s0, c, s2, eps,
                               int(batch_stat), dt, _ptr(ws), ws.numel(), _stream()))
    return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)


def bn_local_stats(x, axis=1, ws=None):
    """mean[C], biased var[C] of this shard of the batch."""
    import torch
    assert x.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    mean = torch.empty(c, dtype=torch.float32, device=x.device)
    var = torch.empty(c, dtype=torch.float32, device=x.device)
    need = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(need, x.device)
    check(lib().nblahip_bn_local_stats(_ptr(x), _ptr(mean), _ptr(var), s0, c, s2, dt, _ptr(ws),
                                       ws.numel(), _stream()))
    return mean, var


def bn_merge_stats(stats, channels, rmean=None, rvar=None, decay_rate=0.9):
    """stats: float32 [workers, 2*channels+1] = {mean, var, count} per worker."""
    import torch
    assert stats.is_contiguous() and stats.dtype == torch.float32
    mean = torch.empty(channels, dtype=torch.float32, device=stats.device)
    var = torch.empty(channels, dtype=torch.float32, device=stats.device)
    check(lib().nblahip_bn_merge_stats(_ptr(stats), stats.shape[0], channels, _ptr(mean), _ptr(var),
                                       _ptr(_f32(rmean, "rmean")), _ptr(_f32(rvar, "rvar")),
                                       decay_rate, _stream()))
    return mean, var


def bn_backward_local_sums(x, dy, mean, var, axis=1, eps=1e-5, need_params=True, ws=None):
    """Returns sums[C, 2] = (sum dy*(x-mean), sum dy) of this shard, dgamma, dbeta."""
    import torch
    assert x.is_contiguous() and dy.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    sums = torch.empty(c, 2, dtype=torch.float32, device=x.device)
    dg = torch.empty(c, dtype=torch.float32, device=x.device) if need_params else None
    db = torch.empty(c, dtype=torch.float32, device=x.device) if need_params else None
    need = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(need, x.device)
    check(lib().nblahip_bn_bwd_local_sums(_ptr(x), _ptr(dy), _ptr(mean), _ptr(var), _ptr(sums),
                                          _ptr(dg), _ptr(db), 0, 0, s0, c, s2, eps, dt, _ptr(ws),
                                          ws.numel(), _stream()))
    return sums, dg, db


def bn_backward_apply_sums(x, dy, gamma, mean, var, sums, total_count, axis=1, eps=1e-5,
                           dmean=None, dvar=None, dx=None, accum=False, ws=None):
    import torch
    assert x.is_contiguous() and dy.is_contiguous() and sums.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    if dx is None:
        dx = torch.empty_like(x)
    need = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(need, x.device)
    check(lib().nblahip_bn_bwd_apply_sums(_ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean),
                                          _ptr(var), _ptr(sums), float(total_count), _ptr(dmean),
                                          _ptr(dvar), _ptr(dx), int(accum), s0, c, s2, eps, dt,
                                          _ptr(ws), ws.numel(), _stream()))
    return dx


def fused_bn_forward_global(x, z, beta, gamma, rmean, rvar, axis=1, eps=1e-5):
    """y = max(0, bn_inference(x) + z); z may be None."""
    import torch
    assert x.is_contiguous() and (z is None or z.is_contiguous())
    s0, c, s2 = _bn_sizes(x.shape, axis)
    y = torch.empty_like(x)
    check(lib().nblahip_fused_bn_fwd_infer(
        _ptr(x), _ptr(z), _ptr(_f32(rmean, "rmean")), _ptr(_f32(rvar, "rvar")),
        _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")), _ptr(y), s0, c, s2, eps,
        _dtype_code(x), _stream()))
    return y


def fused_bn_forward_batch(x, z, beta, gamma, rmean, rvar, axis=1, decay_rate=0.9, eps=1e-5,
                           ws=None):
    """y = max(0, bn_training(x) + z); returns y, batch_mean, batch_var."""
    import torch
    assert x.is_contiguous() and (z is None or z.is_contiguous())
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    y = torch.empty_like(x)
    mean = torch.empty(c, dtype=torch.float32, device=x.device)
    var = torch.empty(c, dtype=torch.float32, device=x.device)
    need = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(need, x.device)
    check(lib().nblahip_fused_bn_fwd_train(
        _ptr(x), _ptr(z), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")), _ptr(y),
        _ptr(mean), _ptr(var), _ptr(_f32(rmean, "rmean")), _ptr(_f32(rvar, "rvar")), s0, c, s2,
        decay_rate, eps, dt, _ptr(ws), ws.numel(), _stream()))
    return y, mean, var


def fused_bn_backward(x, y, dy, gamma, mean, var, axis=1, eps=1e-5, batch_stat=True, dmean=None,
                      dvar=None, dx=None, dz=None, dgamma=None, dbeta=None,
                      accum=(False, False, False, False), need=(True, True, True, True), ws=None):
    """need / accum = (dx, dz, dgamma, dbeta).  Returns dx, dz, dgamma, dbeta."""
    import torch
    assert x.is_contiguous() and dy.is_contiguous() and y.is_contiguous()
    s0, c, s2 = _bn_sizes(x.shape, axis)
    dt = _dtype_code(x)
    if need[0] and dx is None:
        dx = torch.empty_like(x)
    if need[1] and dz is None:
        dz = torch.empty_like(x)
    if need[2] and dgamma is None:
        dgamma = torch.empty(c, dtype=torch.float32, device=x.device)
    if need[3] and dbeta is None:
        dbeta = torch.empty(c, dtype=torch.float32, device=x.device)
    nbytes = lib().nblahip_bn_workspace_bytes(s0, c, s2, dt)
    ws = ws if ws is not None else _workspace(nbytes, x.device)
    check(lib().nblahip_fused_bn_bwd(
        _ptr(x), _ptr(y), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var), _ptr(dmean),
        _ptr(dvar), _ptr(dx if need[0] else None), _ptr(dz if need[1] else None),
        _ptr(dgamma if need[2] else None), _ptr(dbeta if need[3] else None), int(accum[0]),
        int(accum[1]), int(accum[2]), int(accum[3]), s0, c, s2, eps, int(batch_stat), dt, _ptr(ws),
        ws.numel(), _stream()))
    return (dx if need[0] else None, dz if need[1] else None, dgamma if need[2] else None,
            dbeta if need[3] else None)


def ln_forward(x, beta, gamma, outer, eps=1e-5):
    import torch
    assert x.is_contiguous()
    reduce = x.numel() // outer if outer else 0
    y = torch.empty_like(x)
    mean = torch.empty(outer, dtype=torch.float32, device=x.device)
    var = torch.empty(outer, dtype=torch.float32, device=x.device)
    check(lib().nblahip_ln_fwd(_ptr(x), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")),
                               _ptr(y), _ptr(mean), _ptr(var), outer, reduce, eps, _dtype_code(x),
                               _stream()))
    return y, mean, var


def ln_backward(x, dy, gamma, mean, var, outer, eps=1e-5, dmean=None, dvar=None, dx=None,
                dgamma=None, dbeta=None, accum=(False, False, False), need=(True, True, True),
                ws=None):
    import torch
    assert x.is_contiguous() and dy.is_contiguous()
    reduce = x.numel() // outer if outer else 0
    dt = _dtype_code(x)
    if need[0] and dx is None:
        dx = torch.empty_like(x)
    if need[1] and dgamma is None:
        dgamma = torch.empty(reduce, dtype=torch.float32, device=x.device)
    if need[2] and dbeta is None:
        dbeta = torch.empty(reduce, dtype=torch.float32, device=x.device)
    nbytes = lib().nblahip_ln_bwd_workspace_bytes(outer, reduce, dt)
    ws = ws if ws is not None else _workspace(nbytes, x.device)
    check(lib().nblahip_ln_bwd(_ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var),
                               _ptr(dmean), _ptr(dvar), _ptr(dx if need[0] else None),
                               _ptr(dgamma if need[1] else None), _ptr(dbeta if need[2] else None),
                               int(accum[0]), int(accum[1]), int(accum[2]), outer, reduce, eps, dt,
                               _ptr(ws), ws.numel(), _stream()))
    return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)


def _ncs(x, channel_last=False):
    """(batch, channels, spatial) of [N, C, *spatial] or, channel-last, [N, *spatial, C]."""
    n = x.shape[0]
    c = x.shape[-1] if channel_last else x.shape[1]
    sp = 1
    for s in (x.shape[1:-1] if channel_last else x.shape[2:]):
        sp *= s
    return n, c, sp


def gn_forward(x, beta, gamma, num_groups, eps=1e-5, channel_last=False, ws=None, y=None):
    import torch
    assert x.is_contiguous()
    n, c, sp = _ncs(x, channel_last)
    y = torch.empty_like(x) if y is None else y
    mean = torch.empty(n * num_groups, dtype=torch.float32, device=x.device)
    var = torch.empty(n * num_groups, dtype=torch.float32, device=x.device)
    if channel_last:
        dt = _dtype_code(x)
        nbytes = lib().nblahip_gn_cl_workspace_bytes(n, sp, c, num_groups, dt)
        ws = ws if ws is not None else _workspace(nbytes, x.device)
        check(lib().nblahip_gn_cl_fwd(_ptr(x), _ptr(_f32(gamma, "gamma")),
                                      _ptr(_f32(beta, "beta")), _ptr(y), _ptr(mean), _ptr(var),
                                      n, sp, c, num_groups, eps, dt, _ptr(ws), ws.numel(),
                                      _stream()))
        return y, mean, var
    check(lib().nblahip_gn_fwd(_ptr(x), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")),
                               _ptr(y), _ptr(mean), _ptr(var), n, c, sp, num_groups, eps,
                               _dtype_code(x), _stream()))
    return y, mean, var


def gn_backward(x, dy, gamma, mean, var, num_groups, eps=1e-5, dmean=None, dvar=None, dx=None,
                dgamma=None, dbeta=None, accum=(False, False, False), need=(True, True, True),
                ws=None, channel_last=False):
    import torch
    assert x.is_contiguous() and dy.is_contiguous()
    n, c, sp = _ncs(x, channel_last)
    dt = _dtype_code(x)
    if need[0] and dx is None:
        dx = torch.empty_like(x)
    if need[1] and dgamma is None:
        dgamma = torch.empty(c, dtype=torch.float32, device=x.device)
    if need[2] and dbeta is None:
        dbeta = torch.empty(c, dtype=torch.float32, device=x.device)
    if channel_last:
        nbytes = lib().nblahip_gn_cl_workspace_bytes(n, sp, c, num_groups, dt)
        ws = ws if ws is not None else _workspace(nbytes, x.device)
        check(lib().nblahip_gn_cl_bwd(
            _ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var), _ptr(dmean),
            _ptr(dvar), _ptr(dx if need[0] else None), _ptr(dgamma if need[1] else None),
            _ptr(dbeta if need[2] else None), int(accum[0]), int(accum[1]), int(accum[2]), n, sp, c,
            num_groups, eps, dt, _ptr(ws), ws.numel(), _stream()))
        return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)
    nbytes = lib().nblahip_gn_bwd_workspace_bytes(n, c, sp, num_groups, dt)
    ws = ws if ws is not None else _workspace(nbytes, x.device)
    check(lib().nblahip_gn_bwd(_ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var),
                               _ptr(dmean), _ptr(dvar), _ptr(dx if need[0] else None),
                               _ptr(dgamma if need[1] else None), _ptr(dbeta if need[2] else None),
                               int(accum[0]), int(accum[1]), int(accum[2]), n, c, sp, num_groups,
                               eps, dt, _ptr(ws), ws.numel(), _stream()))
    return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)


def in_forward(x, beta, gamma, eps=1e-5, bc_gamma=True, bc_beta=True, channel_last=False,
               ws=None, y=None):
    import torch
    assert x.is_contiguous()
    n, c, sp = _ncs(x, channel_last)
    y = torch.empty_like(x) if y is None else y
    mean = torch.empty(n * c, dtype=torch.float32, device=x.device)
    var = torch.empty(n * c, dtype=torch.float32, device=x.device)
    if channel_last:
        dt = _dtype_code(x)
        nbytes = lib().nblahip_in_cl_workspace_bytes(n, sp, c, dt)
        ws = ws if ws is not None else _workspace(nbytes, x.device)
        check(lib().nblahip_in_cl_fwd(_ptr(x), _ptr(_f32(gamma, "gamma")),
                                      _ptr(_f32(beta, "beta")), _ptr(y), _ptr(mean), _ptr(var),
                                      n, sp, c, int(bc_gamma), int(bc_beta), eps, dt, _ptr(ws),
                                      ws.numel(), _stream()))
        return y, mean, var
    check(lib().nblahip_in_fwd(_ptr(x), _ptr(_f32(gamma, "gamma")), _ptr(_f32(beta, "beta")),
                               _ptr(y), _ptr(mean), _ptr(var), n, c, sp, int(bc_gamma),
                               int(bc_beta), eps, _dtype_code(x), _stream()))
    return y, mean, var


def in_backward(x, dy, gamma, mean, var, eps=1e-5, bc_gamma=True, bc_beta=True, dmean=None,
                dvar=None, dx=None, dgamma=None, dbeta=None, accum=(False, False, False),
                need=(True, True, True), ws=None, channel_last=False):
    import torch
    assert x.is_contiguous() and dy.is_contiguous()
    n, c, sp = _ncs(x, channel_last)
    dt = _dtype_code(x)
    if need[0] and dx is None:
        dx = torch.empty_like(x)
    if need[1] and dgamma is None:
        dgamma = torch.empty(c if bc_gamma else n * c, dtype=torch.float32, device=x.device)
    if need[2] and dbeta is None:
        dbeta = torch.empty(c if bc_beta else n * c, dtype=torch.float32, device=x.device)
    if channel_last:
        nbytes = lib().nblahip_in_cl_workspace_bytes(n, sp, c, dt)
        ws = ws if ws is not None else _workspace(nbytes, x.device)
        check(lib().nblahip_in_cl_bwd(
            _ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var), _ptr(dmean),
            _ptr(dvar), _ptr(dx if need[0] else None), _ptr(dgamma if need[1] else None),
            _ptr(dbeta if need[2] else None), int(accum[0]), int(accum[1]), int(accum[2]), n, sp, c,
            int(bc_gamma), int(bc_beta), eps, dt, _ptr(ws), ws.numel(), _stream()))
        return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)
    nbytes = lib().nblahip_in_bwd_workspace_bytes(n, c, sp, dt)
    ws = ws if ws is not None else _workspace(nbytes, x.device)
    check(lib().nblahip_in_bwd(_ptr(x), _ptr(dy), _ptr(_f32(gamma, "gamma")), _ptr(mean), _ptr(var),
                               _ptr(dmean), _ptr(dvar), _ptr(dx if need[0] else None),
                               _ptr(dgamma if need[1] else None), _ptr(dbeta if need[2] else None),
                               int(accum[0]), int(accum[1]), int(accum[2]), n, c, sp,
                               int(bc_gamma), int(bc_beta), eps, dt, _ptr(ws), ws.numel(),
                               _stream()))
    return (dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None)


def permute(x, perm, out=None, accum=False):
    """out (+)= x.permute(perm), contiguous (nblahip_permute)."""
    import torch
    assert x.is_contiguous()
    nd = x.dim()
    shape = (_i64 * nd)(*x.shape)
    pm = (_int * nd)(*perm)
    if out is None:
        out = torch.empty([x.shape[p] for p in perm], dtype=x.dtype, device=x.device)
    check(lib().nblahip_permute(_ptr(x), _ptr(out), nd, shape, pm, int(accum), _dtype_code(x),
                                _stream()))
    return out


# ---------------------------------------------------------------------------
# Transformer blocks: RMSNormalization, the residual step, 8-bit copies.  Rows
# are `outer` runs of x.numel() // outer columns, as for ln_forward; float32,
# float16 or bfloat16.
# ---------------------------------------------------------------------------
NORMS = {"rms": 0, "layer": 1}
ACT8_FORMATS = {"int8": 1, "e4m3": 2}
_ACCUM_BITS = (1, 2, 4, 8, 16, 32, 64)

# 8-bit copy of a tensor: codes (int8 or float8_e4m3fn, the tensor's shape) and
# scales (uint8 exponent codes, [rows, ceil(cols / 32)]).
Act8 = collections.namedtuple("Act8", "codes scales")
# stats = (mean_post, var_post, mean_pre, var_pre), None where there is none; x8
# and h8: 8-bit copies for the backward (checkpoint), of what it will read.
ResNorm = collections.namedtuple("ResNorm", "h y stats x8 h8")
ResNormGrads = collections.namedtuple(
    "ResNormGrads", "dx dres dgate dgamma_post dbeta_post dgamma_pre dbeta_pre")

_token_dtypes = {}


def _token_dtype(t):
    code = _token_dtypes.get(t)
    if code is None:
        import torch
        _token_dtypes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        code = _token_dtypes.get(t)
        if code is None:
            raise TypeError(f"unsupported activation dtype {t}")
    return code


def _act8_format(a):
    import torch
    if a.codes.dtype == torch.int8:
        return ACT8_FORMATS["int8"]
    if a.codes.dtype == torch.float8_e4m3fn:
        return ACT8_FORMATS["e4m3"]
    raise TypeError(f"8-bit codes must be int8 or float8_e4m3fn, not {a.codes.dtype}")


def _one_gpu(first, *rest):
    """Index of the GPU that all tensors (None: none) are on, contiguous."""
    index = first.get_device()
    if index < 0:
        raise TypeError(f"tensors must be on a GPU, not on {first.device}")
    ok = first.is_contiguous()
    for t in rest:
        if t is not None:
            if t.get_device() != index:
                raise ValueError(f"tensors on {first.device} and on {t.device} in one call")
            ok = ok and t.is_contiguous()
    if not ok:
        raise ValueError("tensors must be contiguous")
    return index


def _stream_of(index):
    """GPU `index`'s current stream, and what to hold while launching on it (None
    where it is the current device)."""
    import torch
    if index == torch.cuda.current_device():
        return torch._C._cuda_getCurrentRawStream(index), None
    return torch._C._cuda_getCurrentRawStream(index), torch.cuda.device(index)


def _call(index, fn, *args):
    """fn(*args, stream) on GPU `index`, on that GPU's current stream."""
    stream, device = _stream_of(index)
    if device is None:
        code = fn(*args, stream)
    else:
        with device:
            code = fn(*args, stream)
    if code != 0:
        check(code)


def _rows_cols(t, outer):
    n = t.numel()
    if outer < 0 or (outer == 0 and n) or (outer and n % outer):
        raise ValueError(f"{n} elements are not {outer} rows")
    if outer:
        return outer, n // outer
    return 0, t.shape[-1] if t.dim() else 0


def _like(t, n, dtype, name):
    if t is not None and (t.dtype != dtype or t.numel() != n):
        raise ValueError(f"{name}: {t.numel()} elements of {t.dtype} where {n} of {dtype} are needed")
    return t


def _check_adds(adds, name, given):
    if adds and given is None:
        raise ValueError(f"{name}: accumulation needs the tensor to add to")


def _check_kept(k, name, rows, cols, dtype):
    """A kept tensor (or its 8-bit copy) of rows x cols: (data, scales, format)."""
    import torch
    if k is None:
        return None, None, 0
    if isinstance(k, Act8):
        _like(k.scales, rows * ((cols + 31) // 32), torch.uint8, name + ".scales")
        if k.codes.numel() != rows * cols:
            raise ValueError(f"{name}.codes: {k.codes.numel()} elements, not {rows} x {cols}")
        return k.codes, k.scales, _act8_format(k)
    _like(k, rows * cols, dtype, name)
    return k, None, 0


def _new_act8(x, rows, cols, f):
    import torch
    return Act8(torch.empty(x.shape, dtype=torch.int8 if f == 1 else torch.float8_e4m3fn,
                            device=x.device),
                torch.empty((rows, (cols + 31) // 32), dtype=torch.uint8, device=x.device))


def act8_pack(x, outer, format="int8"):
    """8-bit copy of x: Act8(codes like x, scales [outer, ceil(cols / 32)])."""
    rows, cols = _rows_cols(x, outer)
    f = ACT8_FORMATS[format]
    dt, gpu = _token_dtype(x.dtype), _one_gpu(x)
    a = _new_act8(x, rows, cols, f)
    _call(gpu, lib().nblahip_act8_pack, _ptr(x), _ptr(a.codes), _ptr(a.scales), rows, cols, f, dt)
    return a


def act8_unpack(a, outer, dtype, out=None):
    """The values an 8-bit copy stands for, rounded to dtype."""
    import torch
    rows, cols = _rows_cols(a.codes, outer)
    codes, scales, f = _check_kept(a, "a", rows, cols, dtype)
    dt, gpu = _token_dtype(dtype), _one_gpu(codes, scales, out)
    if out is None:
        out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _like(out, rows * cols, dtype, "out")
    _call(gpu, lib().nblahip_act8_unpack, _ptr(codes), _ptr(scales), _ptr(out), rows, cols, f, dt)
    return out


def rms_forward(x, gamma, outer, eps=1e-5, y=None):
    """RMSNormalization: y, ms (the rows' mean squares).  gamma may be None."""
    import torch
    rows, cols = _rows_cols(x, outer)
    dt = _token_dtype(x.dtype)
    gpu = _one_gpu(x, gamma, y)
    _like(gamma, cols, torch.float32, "gamma")
    y = torch.empty_like(x) if y is None else _like(y, rows * cols, x.dtype, "y")
    ms = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call(gpu, lib().nblahip_rms_fwd, _ptr(x), _ptr(gamma), _ptr(y), _ptr(ms), rows, cols, eps, dt)
    return y, ms


def rms_backward(x, dy, gamma, ms, outer, eps=1e-5, dx=None, dgamma=None, accum=(False, False),
                 need=(True, True), ws=None):
    """dx, dgamma of RMSNormalization; x is the forward's input or its 8-bit copy
    (Act8).  need / accum = (dx, dgamma)."""
    import torch
    rows, cols = _rows_cols(dy, outer)
    dt = _token_dtype(dy.dtype)
    xd, xs, f = _check_kept(x, "x", rows, cols, dy.dtype)
    gpu = _one_gpu(dy, xd, xs, gamma, ms, dx, dgamma, ws)
    _like(gamma, cols, torch.float32, "gamma")
    _like(ms, rows, torch.float32, "ms")
    _check_adds(need[0] and accum[0], "dx", dx)
    _check_adds(need[1] and accum[1], "dgamma", dgamma)
    dx = None if not need[0] else torch.empty_like(dy) if dx is None else _like(
        dx, rows * cols, dy.dtype, "dx")
    dgamma = None if not need[1] else torch.empty(
        cols, dtype=torch.float32, device=dy.device) if dgamma is None else _like(
            dgamma, cols, torch.float32, "dgamma")
    if ws is None:
        ws = _workspace(lib().nblahip_rms_bwd_workspace_bytes(rows, cols, dt), dy.device)
    _call(gpu, lib().nblahip_rms_bwd, _ptr(xd), _ptr(xs), f, _ptr(dy), _ptr(gamma), _ptr(ms), _ptr(dx),
          _ptr(dgamma), int(accum[0]), int(accum[1]), rows, cols, eps, dt, _ptr(ws), ws.nbytes)
    return dx, dgamma


def ln_backward_act8(x8, dy, gamma, mean, var, outer, eps=1e-5, dx=None, dgamma=None, dbeta=None,
                     accum=(False, False, False), need=(True, True, True), ws=None):
    """ln_backward (one-output form) from the 8-bit copy of the forward's input."""
    import torch
    if not isinstance(x8, Act8):
        raise TypeError("x8 must be an Act8 (act8_pack)")
    rows, cols = _rows_cols(dy, outer)
    dt = _token_dtype(dy.dtype)
    xd, xs, f = _check_kept(x8, "x8", rows, cols, dy.dtype)
    gpu = _one_gpu(dy, xd, xs, gamma, mean, var, dx, dgamma, dbeta, ws)
    _like(gamma, cols, torch.float32, "gamma")
    _like(mean, rows, torch.float32, "mean")
    _like(var, rows, torch.float32, "var")
    for i, t, name in ((0, dx, "dx"), (1, dgamma, "dgamma"), (2, dbeta, "dbeta")):
        _check_adds(need[i] and accum[i], name, t)
    dx = None if not need[0] else torch.empty_like(dy) if dx is None else _like(
        dx, rows * cols, dy.dtype, "dx")
    par = [None if not need[i] else torch.empty(cols, dtype=torch.float32, device=dy.device)
           if t is None else _like(t, cols, torch.float32, n)
           for i, t, n in ((1, dgamma, "dgamma"), (2, dbeta, "dbeta"))]
    if ws is None:
        ws = _workspace(lib().nblahip_ln_bwd_act8_workspace_bytes(rows, cols, dt), dy.device)
    _call(gpu, lib().nblahip_ln_bwd_act8, _ptr(xd), _ptr(xs), f, _ptr(dy), _ptr(gamma), _ptr(mean),
          _ptr(var), _ptr(dx), _ptr(par[0]), _ptr(par[1]), int(accum[0]), int(accum[1]), int(accum[2]),
          rows, cols, eps, dt, _ptr(ws), ws.nbytes)
    return dx, par[0], par[1]


def _gate_args(gate, rows, cols, dtype):
    """(kind, gate rows): an element each in the activations' dtype, or float32
    rows [G, cols] ([cols]: one) that each serve rows / G tokens."""
    import torch
    if gate is None:
        return 0, 0
    n = gate.numel()
    if gate.dtype == dtype and n == rows * cols and not (dtype == torch.float32 and rows == 1):
        return 2, 0
    if gate.dtype != torch.float32:
        raise TypeError(f"gate: {tuple(gate.shape)} of {gate.dtype} for {rows} x {cols} of {dtype}; a "
                        "gate of fewer rows is float32")
    g = n // cols if cols else 0
    if g == 0 or n != g * cols or rows % g:
        raise ValueError(f"gate: {n} elements are no rows of {cols} that divide {rows}")
    return 1, g


def _step_params(cols, post, pre, kind, gamma_post, beta_post, gamma_pre, beta_pre):
    import torch
    if not (post or pre):
        raise ValueError("a step has the norm after the block (post), the one before the next (pre) "
                         "or both")
    if not kind and (beta_post is not None or beta_pre is not None):
        raise ValueError("RMS normalization has no beta")
    if not post and (gamma_post is not None or beta_post is not None):
        raise ValueError("gamma_post / beta_post without their norm")
    if not pre and (gamma_pre is not None or beta_pre is not None):
        raise ValueError("gamma_pre / beta_pre without their norm")
    _like(gamma_post, cols, torch.float32, "gamma_post")
    _like(beta_post, cols, torch.float32, "beta_post")
    _like(gamma_pre, cols, torch.float32, "gamma_pre")
    _like(beta_pre, cols, torch.float32, "beta_pre")


def resnorm_forward(x, res, outer, gate=None, gamma_post=None, beta_post=None, gamma_pre=None,
                    beta_pre=None, norm="rms", post=True, pre=True, res_scale=1.0, branch_scale=1.0,
                    eps=1e-5, checkpoint=None, h=None, y=None):
    """The step between two blocks of a residual stream:
        u = norm(x; gamma_post, beta_post) if post else x
        h = res_scale * res + branch_scale * gate * u
        y = norm(h; gamma_pre, beta_pre) if pre else None
    gate: None, float32 [G, cols] (G divides outer) or a tensor like x.
    checkpoint "int8" / "e4m3": also 8-bit copies x8, h8 of what the backward
    reads.  h may be res, y may be x (in place).  Returns ResNorm."""
    import torch
    rows, cols = _rows_cols(x, outer)
    act, dev = x.dtype, x.device
    dt, kind = _token_dtype(act), NORMS[norm]
    gpu = _one_gpu(x, res, gate, gamma_post, beta_post, gamma_pre, beta_pre, h, y)
    _like(res, rows * cols, act, "res")
    _step_params(cols, post, pre, kind, gamma_post, beta_post, gamma_pre, beta_pre)
    gk, gr = _gate_args(gate, rows, cols, act)
    h = torch.empty_like(x) if h is None else _like(h, rows * cols, act, "h")
    if pre:
        y = torch.empty_like(x) if y is None else _like(y, rows * cols, act, "y")
    else:
        y = None

    def stat(on):
        return torch.empty(rows, dtype=torch.float32, device=dev) if on else None
    stats = (stat(post and kind), stat(post), stat(pre and kind), stat(pre))
    x8 = h8 = None
    f = 0
    if checkpoint is not None:
        f = ACT8_FORMATS[checkpoint]
        x8 = _new_act8(x, rows, cols, f) if post or gk else None
        h8 = _new_act8(x, rows, cols, f) if pre else None
    _call(gpu, lib().nblahip_resnorm_fwd, _ptr(x), _ptr(res), _ptr(gate), gk, gr, _ptr(gamma_post),
          _ptr(beta_post), _ptr(gamma_pre), _ptr(beta_pre), _ptr(h), _ptr(y), _ptr(stats[0]),
          _ptr(stats[1]), _ptr(stats[2]), _ptr(stats[3]), _ptr(x8 and x8.codes),
          _ptr(x8 and x8.scales), _ptr(h8 and h8.codes), _ptr(h8 and h8.scales), f, rows, cols,
          res_scale, branch_scale, eps, kind, int(post), int(pre), dt)
    return ResNorm(h, y, stats, x8, h8)


def resnorm_backward(x, h, dh, dy, stats, outer, gate=None, gamma_post=None, beta_post=None,
                     gamma_pre=None, beta_pre=None, norm="rms", post=True, pre=True, res_scale=1.0,
                     branch_scale=1.0, eps=1e-5, has_res=True, need=(True,) * 7, accum=(False,) * 7,
                     out=None, ws=None):
    """Gradients of resnorm_forward.  x, h: its tensors, or their 8-bit copies
    (both); dh: gradient of h from its later readers (None: none), dy: of y.
    need / accum / out follow ResNormGrads' fields; what does not exist (dres
    without a residual, dgate without a gate, parameters of an absent norm, beta
    of RMS) is None."""
    import torch
    lead = dh if dh is not None else dy
    if lead is None:
        raise ValueError("dh or dy is needed")
    rows, cols = _rows_cols(lead, outer)
    act, dt, kind = lead.dtype, _token_dtype(lead.dtype), NORMS[norm]
    layer = kind == 1
    gk, gr = _gate_args(gate, rows, cols, act)
    if not (post or gk):
        x = None
    if not pre:
        h = dy = None
    xd, xs, xf = _check_kept(x, "x", rows, cols, act)
    hd, hs, hf = _check_kept(h, "h", rows, cols, act)
    if x is not None and h is not None and xf != hf:
        raise TypeError("x and h must be kept in the same form")
    given = out if out is not None else (None,) * 7
    gpu = _one_gpu(lead, dh, dy, xd, xs, hd, hs, gate, gamma_post, beta_post, gamma_pre, beta_pre,
                   *stats, *given, ws)
    _step_params(cols, post, pre, kind, gamma_post, beta_post, gamma_pre, beta_pre)
    n = rows * cols
    _like(dh, n, act, "dh")
    _like(dy, n, act, "dy")
    for s, name in zip(stats, ("mean_post", "var_post", "mean_pre", "var_pre")):
        _like(s, rows, torch.float32, name)
    dev, f32 = lead.device, torch.float32

    def tensor(i):
        t = given[i]
        return torch.empty_like(lead) if t is None else _like(t, n, act, ResNormGrads._fields[i])

    def param(i):
        t = given[i]
        return torch.empty(cols, dtype=f32, device=dev) if t is None else _like(
            t, cols, f32, ResNormGrads._fields[i])
    dgate = None
    if gk and need[2]:
        dgate = torch.empty_like(gate) if given[2] is None else _like(
            given[2], gate.numel(), gate.dtype, "dgate")
    grads = (tensor(0) if need[0] else None, tensor(1) if has_res and need[1] else None, dgate,
             param(3) if post and need[3] else None, param(4) if post and layer and need[4] else None,
             param(5) if pre and need[5] else None, param(6) if pre and layer and need[6] else None)
    mask = 0
    if any(accum):
        for i in range(7):
            if accum[i] and grads[i] is not None:
                _check_adds(True, ResNormGrads._fields[i], given[i])
                mask |= _ACCUM_BITS[i]
    if ws is None:
        ws = _workspace(lib().nblahip_resnorm_bwd_workspace_bytes(
            rows, cols, gk, gr, kind, int(post), int(pre), dt), dev)
    p = [None if g is None else g.data_ptr() for g in grads]
    _call(gpu, lib().nblahip_resnorm_bwd, _ptr(xd), _ptr(xs), _ptr(hd), _ptr(hs), xf or hf, _ptr(dh),
          _ptr(dy), _ptr(gate), gk, gr, _ptr(gamma_post), _ptr(beta_post), _ptr(gamma_pre),
          _ptr(stats[0]), _ptr(stats[1]), _ptr(stats[2]), _ptr(stats[3]), p[0], p[1], p[2], p[3], p[4],
          p[5], p[6], mask, rows, cols, res_scale, branch_scale, eps, kind, int(post), int(pre), dt,
          _ptr(ws), ws.nbytes)
    return ResNormGrads(*grads)
