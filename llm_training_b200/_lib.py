"""ctypes binding of the C ABI in include/sqrtblock.h (libsqrtblock.so).

The shared library is built in-tree by ``python -m llm_training_b200.build``.
There is no fallback: if the library is missing or fails to load, ``lib()``
raises, and every op that needs it fails with that error.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import threading

import torch

from .build import BINDING, BINDINGPATH, LIBPATH

SQB_F32 = 0
SQB_BF16 = 1

IMPL_AUTO = 0
IMPL_SIMT = 1
IMPL_TCGEN05 = 2
IMPLS = {"auto": IMPL_AUTO, "simt": IMPL_SIMT, "tcgen05": IMPL_TCGEN05}

SQB_OK = 0
SQB_ERR_TIMEOUT = 7

# Every symbol declared in include/sqrtblock.h, with its ctypes signature.
_c_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
SIGNATURES = {
    "sqb_version": (ctypes.c_int, []),
    "sqb_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "sqb_geometry": (ctypes.c_int, [_c_i64, _c_i64, ctypes.POINTER(_c_i64),
                                    ctypes.POINTER(_c_i64), ctypes.POINTER(_c_i64)]),
    "sqb_workspace_bytes": (ctypes.c_size_t, [_c_i64] * 5),
    "sqb_fwd": (ctypes.c_int, [_vp] * 7 + [_c_i64] * 5 + [ctypes.POINTER(_c_i64), ctypes.c_int,
                                                           ctypes.c_float, ctypes.c_int, _vp,
                                                           ctypes.c_size_t, _vp]),
    "sqb_bwd": (ctypes.c_int, [_vp] * 11 + [_c_i64] * 5 + [ctypes.POINTER(_c_i64), ctypes.c_int,
                                                            ctypes.c_float, ctypes.c_int, _vp,
                                                            ctypes.c_size_t, _vp]),
    "sqb_read_status": (ctypes.c_int, [_vp, _vp, ctypes.POINTER(_c_i64)]),
    "sqb_read_status_noalloc": (ctypes.c_int, [_vp, ctypes.POINTER(_c_i64)]),
    "sqb_attach_status": (ctypes.c_int, [_vp, _vp, ctypes.c_uint32, _vp]),
    "sqb_bwd_noalloc": (ctypes.c_int, [_vp] * 11 + [_c_i64] * 5 + [ctypes.POINTER(_c_i64),
                                                                    ctypes.c_int, ctypes.c_float,
                                                                    ctypes.c_int, _vp]),
    "sqb_refsem_workspace_bytes": (ctypes.c_size_t, [_c_i64] * 4),
    "sqb_refsem_fwd": (ctypes.c_int, [_vp] * 6 + [_c_i64] * 4 + [ctypes.POINTER(_c_i64),
                                                                 ctypes.c_int, ctypes.c_float,
                                                                 _vp, ctypes.c_size_t, _vp]),
    "sqb_refsem_bwd": (ctypes.c_int, [_vp] * 9 + [_c_i64] * 4 + [ctypes.POINTER(_c_i64),
                                                                 ctypes.c_int, ctypes.c_float,
                                                                 _vp, ctypes.c_size_t, _vp]),
}

_lock = threading.Lock()
_lib = None


class SqrtBlockError(RuntimeError):
    """An sqb_* call returned an error code."""

    def __init__(self, fn: str, code: int, msg: str):
        super().__init__(f"{fn} failed with code {code}: {msg}")
        self.code = code


# Training-caller helpers (include/sqb_train.h), bound on the same library.
TRAIN_SIGNATURES = {
    "sqb_xent_fwd": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                    ctypes.c_void_p, _c_i64, _c_i64, _c_i64, ctypes.c_int,
                                    ctypes.c_void_p]),
    "sqb_xent_bwd": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                    ctypes.c_void_p, ctypes.c_void_p, _c_i64, _c_i64, _c_i64,
                                    ctypes.c_int, ctypes.c_void_p]),
    "sqb_layernorm_fwd": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_int] +
                          [ctypes.c_void_p] * 2 + [_c_i64, _c_i64, ctypes.c_float,
                                                   ctypes.c_void_p]),
    "sqb_layernorm_workspace_bytes": (ctypes.c_size_t, [_c_i64, _c_i64]),
    "sqb_layernorm_bwd": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int] + [ctypes.c_void_p] * 8 +
                          [ctypes.c_size_t, _c_i64, _c_i64, ctypes.c_void_p]),
    "sqb_add_layernorm_fwd": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int] +
                              [ctypes.c_void_p] * 4 + [ctypes.c_int] + [ctypes.c_void_p] * 2 +
                              [_c_i64, _c_i64, ctypes.c_float, ctypes.c_void_p]),
    "sqb_add_layernorm_bwd": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int] +
                              [ctypes.c_void_p] * 10 +
                              [ctypes.c_size_t, _c_i64, _c_i64, ctypes.c_void_p]),
    # token log-probabilities and the losses on them
    "sqb_logp_fwd": (ctypes.c_int, [_vp] * 4 + [_c_i64] * 5 + [ctypes.c_int, _vp]),
    "sqb_logp_bwd": (ctypes.c_int, [_vp] * 6 + [_c_i64] * 7 + [ctypes.c_int, _vp]),
    "sqb_preference_workspace_bytes": (ctypes.c_size_t, [_c_i64] * 2),
    "sqb_preference_fwd": (ctypes.c_int, [_vp] * 4 + [_c_i64] + [ctypes.c_double] * 2 +
                           [_vp] * 4 + [_c_i64] * 5 + [ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    "sqb_policy_workspace_bytes": (ctypes.c_size_t, [_c_i64] * 2),
    "sqb_policy_fwd": (ctypes.c_int, [_vp] * 3 + [_c_i64] + [_vp] * 3 + [ctypes.c_int] +
                       [ctypes.c_double] * 3 + [ctypes.c_int] + [_vp] * 6 + [ctypes.c_float] +
                       [_c_i64] * 7 + [ctypes.c_int, _vp, ctypes.c_size_t, _vp]),
    # gradient norm and clipping
    "sqb_grad_norm_workspace_bytes": (ctypes.c_size_t, [_c_i64]),
    "sqb_grad_norm": (ctypes.c_int, [_vp] * 3 + [_c_i64, _vp, ctypes.c_size_t, _vp, _vp]),
    "sqb_grad_clip": (ctypes.c_int, [_vp] * 5 + [_c_i64, ctypes.c_float, _vp, ctypes.c_size_t,
                                                 _vp, _vp]),
    # the residual step between two norms
    "sqb_residual_norm_fwd": (ctypes.c_int, [_vp, ctypes.c_int] * 2 + [_vp] * 5 +
                              [_c_i64, ctypes.c_float, ctypes.c_float, ctypes.c_int] +
                              [_vp] * 2 + [ctypes.c_int, _vp, _c_i64, _c_i64, _vp]),
    "sqb_residual_norm_workspace_bytes": (ctypes.c_size_t, [_c_i64] * 3),
    "sqb_residual_norm_bwd": (ctypes.c_int, [_vp, ctypes.c_int, _vp] + [_vp, ctypes.c_int] * 2 +
                              [_vp] * 5 +
                              [_c_i64, ctypes.c_float, ctypes.c_float, ctypes.c_int] +
                              [_vp] * 9 + [ctypes.c_size_t, _c_i64, _c_i64, _vp]),
}


_binding = None


def binding():
    """The C++ PyTorch binding of the post-training operators, on the library of ``lib()``;
    raises if it is absent."""
    global _binding
    if _binding is None:
        lib()
        with _lock:
            if _binding is None:
                if not os.path.exists(BINDINGPATH):
                    raise RuntimeError(f"PyTorch binding not found at {BINDINGPATH}; build it "
                                       "with `python -m llm_training_b200.build`")
                loader = importlib.machinery.ExtensionFileLoader(BINDING, BINDINGPATH)
                module = importlib.util.module_from_spec(
                    importlib.util.spec_from_loader(BINDING, loader))
                loader.exec_module(module)
                module.attach(library_path())
                _binding = module
    return _binding


_ORDINARY = (torch.Tensor, torch.nn.Parameter, type(None))
# (looked up once: every call of a post-training op asks)
_compiling = torch.compiler.is_compiling
_transformed = torch._C._are_functorch_transforms_active
_dispatch_modes = torch._C._len_torch_dispatch_stack
_jit_traced = torch._C._is_tracing


def eager() -> bool:
    """Whether an op is run where it is called: by no tracer (torch.compile's or torch.jit's),
    dispatch mode or torch.func transform, none of which would see a launch of the binding."""
    if _compiling():
        return False
    if _transformed():
        # the dispatcher takes an op without a forward-mode derivative for a constant
        jvp = torch._C._functorch.TransformType.Jvp
        if any(level.key() == jvp for level in torch._C._functorch.get_interpreter_stack()):
            raise NotImplementedError("the post-training operators have no forward-mode "
                                      "derivative")
        return False
    return _dispatch_modes() == 0 and not _jit_traced()


def plain(*tensors) -> bool:
    """Whether `tensors` (None where one is not given) are ordinary tensors in an eager call.
    The post-training ops then run without the dispatcher, whose custom-op layers cost 100 us
    a call; a traced, fake or otherwise intercepted call goes through the registered custom
    op."""
    return all([type(x) in _ORDINARY for x in tensors]) and eager()


def library_path() -> str:
    return os.environ.get("SQB_LIBRARY", LIBPATH)


def lib() -> ctypes.CDLL:
    """Load (once) and return the shared library; raises if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            path = library_path()
            if not os.path.exists(path):
                raise RuntimeError(
                    f"sqrt-block CUDA library not found at {path}; build it with "
                    "`python -m llm_training_b200.build` (there is no CPU fallback)")
            handle = ctypes.CDLL(path)
            for name, (res, args) in {**SIGNATURES, **TRAIN_SIGNATURES}.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            _lib = handle
    return _lib


def check(fn: str, code: int) -> None:
    if code != SQB_OK:
        raise SqrtBlockError(fn, code, lib().sqb_strerror(code).decode())


def geometry(T: int, block: int | None = None):
    """(b, G, Gc) as the library computes it."""
    b, g, gc = _c_i64(), _c_i64(), _c_i64()
    check("sqb_geometry", lib().sqb_geometry(T, block or 0, ctypes.byref(b), ctypes.byref(g),
                                             ctypes.byref(gc)))
    return b.value, g.value, gc.value


def workspace_bytes(B, T, H, D, block) -> int:
    return int(lib().sqb_workspace_bytes(B, T, H, D, block))


def strides_array(*strides) -> ctypes.Array:
    flat = [int(s) for st in strides for s in st]
    return (_c_i64 * len(flat))(*flat)
