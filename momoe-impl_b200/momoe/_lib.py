"""ctypes binding of libmomoe_b200.so (the C ABI declared in include/momoe_b200.h), and the compiled binding `native` of
the operators around the expert layer (csrc/binding.cpp), whose calls are too short for Python on the way.

There is no fallback: if the library is missing, importing this module raises with the build command, and so does the first
use of the binding if that is missing.
"""
import contextlib
import ctypes as C
import os
import sys

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("MOMOE_B200_LIB", os.path.join(_HERE, "libmomoe_b200.so"))

if not os.path.exists(LIB_PATH):
    raise ImportError(
        "libmomoe_b200.so is not built; run `python momoe-impl_b200/build.py` (needs nvcc, targets sm_100a). "
        "There is no CPU or PyTorch fallback for the MoMoE kernels.")

lib = C.CDLL(LIB_PATH)

_BUILT_FOR = "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])


def require_fitting(binding):
    """A binding of another torch or Python may load and misread its tensors."""
    built_for = getattr(binding, "built_for", "unknown versions")
    if built_for != _BUILT_FOR:
        raise ImportError("_native.so was built for %s, not for %s: run `python momoe-impl_b200/build.py`"
                          % (built_for, _BUILT_FOR))


class _Native:
    """The compiled binding: torch tensors in, the same library underneath.  Loaded when first used, since the layer in 16
    bits does without it."""

    def __getattr__(self, name):
        try:
            from . import _native
        except ImportError as e:
            raise ImportError("_native.so is not built or does not fit %s: run `python momoe-impl_b200/build.py` (needs g++ "
                              "and torch's headers)" % _BUILT_FOR) from e
        require_fitting(_native)
        _native.bind(LIB_PATH)
        self.__dict__.update({k: v for k, v in vars(_native).items() if k not in ("__class__", "__dict__")})
        return getattr(_native, name)

    def launches(self):
        """Kernels queued through it; replaced by its own count once it is loaded."""
        return 0


native = _Native()

c_i32, c_i64, c_vp, c_sz, c_u32 = C.c_int32, C.c_int64, C.c_void_p, C.c_size_t, C.c_uint32


class Plan(C.Structure):
    """Mirror of momoe_plan_t."""
    _fields_ = [("M", c_i32), ("N", c_i32), ("K", c_i32), ("D", c_i32), ("H", c_i32), ("reserved", c_i32),
                ("rows_capacity", c_i64), ("sched", c_vp), ("tile_expert", c_vp), ("pad_off", c_vp),
                ("row_token", c_vp), ("row_weight", c_vp), ("pos_MK", c_vp), ("status", c_vp), ("pair_info", c_vp)]


PlanP = C.POINTER(Plan)

_PROTOS = {
    "momoe_version": (C.c_int, []),
    "momoe_sorted_rows_capacity": (c_i64, [c_i32, c_i32, c_i32]),
    "momoe_tile_capacity": (c_i64, [c_i32, c_i32, c_i32]),
    "momoe_route_topk": (C.c_int, [c_vp, c_vp, c_i32, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                   c_vp]),
    "momoe_topk_from_mask": (C.c_int, [c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp,
                                       c_vp]),
    "momoe_permutation_launches": (C.c_int, [c_i32, c_i32, c_i32]),
    "momoe_permutation_workspace_bytes": (c_sz, [c_i32, c_i32, c_i32]),
    "momoe_build_permutation": (C.c_int, [c_vp, c_vp, c_i32, c_i32, c_i32, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                          c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_sz, c_vp, c_vp]),
    "momoe_build_permutation_static": (C.c_int, [c_vp, c_vp, c_i32, c_i32, c_i32, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp,
                                                 c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_vp]),
    "momoe_gather_rows": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_vp]),
    "momoe_combine_rows": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_vp]),
    "momoe_up_swiglu": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_i32, c_vp]),
    "momoe_up_swiglu_tokens": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_i32, c_vp]),
    "momoe_down_scale": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp]),
    "momoe_up_swiglu_decode": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp]),
    "momoe_down_scale_decode": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp]),
    "momoe_dgrad2_swiglu_bwd": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_dgrad2_swiglu_bwd_tokens": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_dgrad1": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp]),
    "momoe_wgrad": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_i32, c_vp, c_vp]),
    "momoe_wgrad_tokens": (C.c_int, [PlanP, c_vp, c_i32, c_i32, c_vp, c_i32, c_i32, c_vp, c_vp]),
    "momoe_scatter_gs": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_vp]),
    "momoe_router_backward": (C.c_int, [c_vp, c_i64, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_i32, c_i32, c_i32, c_vp,
                                        c_vp]),
    "momoe_router_backward_compact": (C.c_int, [c_vp, c_vp, c_i32, c_vp, c_vp, c_vp, c_vp, c_i32, c_vp, c_vp]),
    "momoe_bias_update": (C.c_int, [c_vp, c_vp, c_i32, c_i32, C.c_float, C.c_float, c_vp]),
    "momoe_rms_norm": (C.c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i32, c_i32, c_i32, c_i32, C.c_float, c_vp, c_vp, c_vp,
                                 c_vp, c_vp, c_vp]),
    "momoe_rms_norm_backward_workspace_bytes": (c_sz, [c_i32, c_i32]),
    "momoe_rms_norm_backward": (C.c_int, [c_vp, c_vp, c_vp, c_i64, c_vp, c_vp, c_i32, c_i32, c_i32, c_i32, c_vp, c_vp,
                                          c_vp, c_sz, c_vp]),
    "momoe_quantize_rows": (C.c_int, [c_vp, c_i64, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp]),
    "momoe_balance_loss_workspace_bytes": (c_sz, [c_i32, c_i32, c_i32]),
    "momoe_balance_loss": (C.c_int, [c_vp, c_i32, c_vp, c_vp, c_i32, c_i32, c_i32, c_i32, c_i32, c_i32, C.c_float,
                                     C.c_float, c_vp, c_vp, c_vp, c_vp, c_sz, c_vp]),
    "momoe_balance_loss_backward": (C.c_int, [c_vp, c_i32, c_vp, c_i32, c_vp, c_i32, c_i32, c_i32, c_i32, C.c_float,
                                              c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_quantize_weights": (C.c_int, [c_vp, c_i32, c_i32, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp]),
    "momoe_fp8_dispatch_workspace_bytes": (c_sz, [c_i32, c_i32, c_i32]),
    "momoe_fp8_dispatch_rows": (C.c_int, [c_vp, c_vp, c_vp, c_vp, c_i32, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp,
                                          c_vp, c_vp, c_i64, c_vp, c_sz, c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_up_swiglu": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_up_swiglu_decode": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_down_scale": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_down_scale_decode": (C.c_int, [PlanP, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "momoe_fp8_combine_rows": (C.c_int, [c_vp, c_vp, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp]),
    "momoe_fp8_experts_workspace_bytes": (c_sz, [c_i32, c_i32, c_i32, c_i32, c_i32]),
    "momoe_fp8_experts_launches": (C.c_int, [c_i32, c_i32, c_i32]),
    "momoe_fp8_experts_forward": (C.c_int, [c_vp, c_vp, c_vp, c_vp, c_i32, c_i32, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp,
                                            c_vp, c_i32, c_vp, c_vp, c_vp, c_sz, c_vp, c_vp]),
    "momoe_ep_set_wait_limit": (c_i64, [c_i64]),
    "momoe_ep_publish_counts": (C.c_int, [c_vp, c_i32, c_vp, c_vp, c_i32, c_i32, c_u32, c_vp, c_vp]),
    "momoe_ep_barrier": (C.c_int, [c_vp, c_i32, c_i32, c_u32, c_vp, c_vp]),
    "momoe_ep_plan": (C.c_int, [c_vp, c_i32, c_i32, c_i32, C.c_double, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                c_vp, c_vp]),
    "momoe_ep_dispatch_rows": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_i32, c_vp, c_vp, c_vp, c_i32, c_i32, c_vp, c_vp,
                                         c_i32, c_vp]),
    "momoe_ep_combine_rows": (C.c_int, [PlanP, c_vp, c_vp, c_i32, c_i32, c_vp, c_i32, c_i32, c_vp]),
    "momoe_ep_plan_split": (C.c_int, [c_vp, c_i32, c_i32, c_i32, C.c_double, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                      c_vp, c_i32, c_vp, c_vp, c_vp, c_vp]),
    "momoe_ep_dispatch_rows_range": (C.c_int, [PlanP, c_vp, c_i32, c_vp, c_i32, c_vp, c_vp, c_vp, c_i32, c_i32, c_vp,
                                               c_vp, c_i32, c_i32, c_i32, c_vp]),
    "momoe_ep_pull_rows": (C.c_int, [PlanP, c_vp, c_vp, c_i32, c_i32, c_vp, c_i32, c_i32, c_i32, c_i32, c_i32, c_vp]),
    "momoe_ep_combine_rows_staged": (C.c_int, [PlanP, c_vp, c_vp, c_i32, c_i32, c_vp, c_i32, c_vp, c_i32, c_i32, c_i32,
                                               c_vp]),
    "momoe_ep_reduce_gs": (C.c_int, [c_vp, c_i32, c_vp, c_vp, c_vp]),
    "momoe_ep_pull_gs_compact": (C.c_int, [PlanP, c_vp, c_vp, c_i32, c_vp, c_i32, c_vp]),
}
for _name, (_res, _args) in _PROTOS.items():
    _f = getattr(lib, _name)
    _f.restype = _res
    _f.argtypes = _args

EXPORTED = tuple(_PROTOS)

_ERRORS = {-1: "bad argument (null pointer, size or alignment)", -2: "unsupported shape (D and H must be multiples "
           "of 8)", -3: "a CUDA call failed", -4: "exceeds a fixed capacity (N <= 1024, K <= 32)"}


def check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed: {_ERRORS.get(rc, 'code %d' % rc)}")


def ptr(t):
    """Device pointer of a tensor (None -> NULL)."""
    if t is None:
        return None
    return C.c_void_p(t.data_ptr())


def stream_ptr():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}     # type codes of the C ABI


def require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("momoe (B200 build) runs on CUDA tensors only; there is no CPU path")


def require_one_device(*tensors):
    """The CUDA device that all given tensors (None is skipped) are on."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.device
        if dev is None:
            dev = d
        if d.type != "cuda":
            require_cuda(t)
        if d != dev:
            raise RuntimeError("all tensors must be on the same device, but got: %s and %s" % (dev, d))
    return dev


_STAY = contextlib.nullcontext()


def on_device(dev):
    """Context in which `dev` is the current device; costs nothing where it already is."""
    return _STAY if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def raw_stream(dev):
    """The current stream of a device as an integer (what a c_void_p argument takes)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def aligned(t, n=16):
    """t itself where it starts on an n-byte boundary, a copy otherwise."""
    return t if t.data_ptr() % n == 0 else t.clone()


def as_rows(t):
    """t [..., D] as a [M, D] tensor whose rows the kernels can read: contiguous columns, a row pitch of a multiple of 8
    elements, a 16-byte aligned start.  A view where the layout allows it, a copy otherwise."""
    r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if r.is_contiguous():
        return aligned(r)
    if r.stride(1) != 1 or r.stride(0) % 8 != 0 or r.stride(0) < 0 or r.data_ptr() % 16 != 0:
        return r.contiguous()
    return r


def pitch(r):
    """Row pitch in elements of a tensor from as_rows."""
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]
