"""Loads the in-tree native libraries.  There is no CPU fallback: if a library is
missing the import of anything that computes fails with a clear error."""
import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
KERNEL_LIB = os.path.join(HERE, "lib", "libseraph_hip.so")
BACKEND_LIB = os.path.join(HERE, "lib", "libseraph_hip_backend.so")

_kernels = None
_backend = None


class SeraphError(RuntimeError):
    pass


def kernels():
    """ctypes handle of libseraph_hip.so (the C-ABI kernel library)."""
    global _kernels
    if _kernels is None:
        if not os.path.exists(KERNEL_LIB):
            raise SeraphError(f"{KERNEL_LIB} is not built; run `python -m seraph_amd.build` (needs hipcc)")
        lib = C.CDLL(KERNEL_LIB, mode=C.RTLD_GLOBAL)
        lib.seraph_hip_last_error.restype = C.c_char_p
        for name in ("seraph_attention_backward_ws_bytes", "seraph_attention_backward_ws_bytes_banded",
                     "seraph_rmsnorm_backward_ws_bytes", "seraph_embedding_backward_ws_bytes",
                     "seraph_gemm_scaled_ws_bytes", "seraph_rmsnorm_backward_static_max_bytes"):
            getattr(lib, name).restype = C.c_size_t
        _bind_objectives(lib)
        lib.seraph_gemm_grouped_kernel_name.restype = C.c_char_p
        lib.seraph_gemm_chain_kernel_name.restype = C.c_char_p
        lib.seraph_gemm_kernel_name.restype = C.c_char_p
        _kernels = lib
    return _kernels


class PolicyOptions(C.Structure):
    _fields_ = [("clip_low", C.c_float), ("clip_high", C.c_float), ("kl_coef", C.c_float), ("entropy_coef", C.c_float)]


class PreferenceOptions(C.Structure):
    _fields_ = [("kind", C.c_int), ("beta", C.c_float), ("label_smoothing", C.c_float), ("margin", C.c_float), ("average", C.c_int)]


class DistillOptions(C.Structure):
    _fields_ = [("temperature", C.c_float), ("soft_coef", C.c_float), ("hard_coef", C.c_float), ("teacher_type", C.c_int)]


def _bind_objectives(lib):
    """Argument types of the objectives over logits: plain Python numbers and addresses then go in as they are."""
    p, i, n, z = C.c_void_p, C.c_int, C.c_int64, C.c_size_t
    for name, args in (("seraph_token_logprobs", [n, n]), ("seraph_policy_grad", [n, n]), ("seraph_preference_grad", [n, n]),
                       ("seraph_distill_grad", [n, n, n])):
        query = getattr(lib, name + "_ws_bytes")
        query.restype, query.argtypes = z, args
    lib.seraph_token_logprobs.argtypes = [p] * 6 + [i, n, n, p, z, p]
    lib.seraph_policy_grad.argtypes = [p] * 11 + [C.POINTER(PolicyOptions), p, i, n, n, n, p, z, p]
    lib.seraph_preference_grad.argtypes = [p] * 7 + [C.POINTER(PreferenceOptions), p, i, n, n, p, z, p]
    lib.seraph_distill_grad.argtypes = [p] * 8 + [C.POINTER(DistillOptions), p, i, n, n, n, n, p, z, p]


def backend():
    """ctypes handle of libseraph_hip_backend.so (vulkan_* compatible host backend + step drivers)."""
    global _backend
    if _backend is None:
        kernels()
        if not os.path.exists(BACKEND_LIB):
            raise SeraphError(f"{BACKEND_LIB} is not built; run `python -m seraph_amd.build`")
        _backend = C.CDLL(BACKEND_LIB, mode=C.RTLD_GLOBAL)
    return _backend


def check(rc, what=""):
    if rc != 0:
        msg = kernels().seraph_hip_last_error()
        raise SeraphError(f"{what} failed ({rc}): {msg.decode() if msg else ''}")
