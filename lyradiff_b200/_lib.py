"""ctypes loader for liblyraq.so, the C-ABI CUDA library.  There is no fallback: if the library is
missing or lacks a symbol the import of the ops fails with a clear error."""

import ctypes
import os
import sysconfig

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("LYRAQ_LIB_PATH", os.path.join(_HERE, "liblyraq.so"))

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_size_t = ctypes.c_size_t
c_float = ctypes.c_float
c_double = ctypes.c_double



class GatedNormArgs(ctypes.Structure):
    """lyraq_gated_norm_t."""
    _fields_ = ([(n, c_void_p) for n in ("y", "x")] + [(n, c_size_t) for n in ("y_batch", "y_row", "x_batch", "x_row")]
                + [(n, c_void_p) for n in ("x_out", "h")] + [(n, c_size_t) for n in ("x_out_batch", "x_out_row", "h_batch", "h_row")]
                + [(n, c_void_p) for n in ("qf8", "f8_scale", "q4", "q4_scales", "q4_tensor_scale")] + [("q4_format", c_int)]
                + [(n, c_void_p) for n in ("gate", "scale", "shift")] + [(n, c_size_t) for n in ("gate_batch", "scale_batch", "shift_batch")]
                + [(n, c_void_p) for n in ("post_weight", "pre_weight")] + [("post", c_int), ("pre", c_int)]
                + [("residual_scale", c_float), ("eps", c_float), ("dtype", c_int)] + [(n, c_size_t) for n in ("batch", "seq_len", "dim")])


class RopeAxesArgs(ctypes.Structure):
    """lyraq_rope_axes_t."""
    _fields_ = ([(n, c_void_p) for n in ("q", "k")] + [(a + n, c_size_t) for a in ("q_", "k_") for n in ("batch", "token", "head")]
                + [(n, c_void_p) for n in ("q_out", "k_out")] + [(a + n, c_size_t) for a in ("q_out_", "k_out_") for n in ("batch", "token", "head")]
                + [(n, c_void_p) for n in ("q_norm", "k_norm", "positions")] + [(n, c_size_t) for n in ("pos_batch", "pos_token", "pos_axis")]
                + [(n, c_void_p) for n in ("turns", "axis")]
                + [(n, c_int) for n in ("pos_dtype", "dtype", "q_heads", "k_heads", "head_dim", "pairs", "interleaved")] + [("eps", c_float)]
                + [(n, c_size_t) for n in ("batch", "seq_len")])


# name -> (restype, argtypes); mirrors include/lyraq.h declaration by declaration
SIGNATURES = {
    "lyraq_version": (ctypes.c_char_p, []),
    "lyraq_status_string": (ctypes.c_char_p, [c_int]),
    "lyraq_last_status": (c_int, [c_void_p, ctypes.POINTER(ctypes.c_uint32)]),
    "lyraq_debug_force_gemm_tile": (c_int, [c_int]),
    "lyraq_debug_set_dependent_launch": (c_int, [c_int]),
    "lyraq_debug_attention_wait_test": (c_int, [c_int, ctypes.c_uint]),
    "lyraq_debug_skinny_wait_test": (c_int, [c_int, ctypes.c_uint]),
    "lyraq_debug_force_w4a4_wide": (c_int, [c_int]),
    "lyraq_debug_force_fp4_tile": (c_int, [c_int]),
    "lyraq_debug_fp4_skinny_wait_test": (c_int, [c_int, ctypes.c_uint]),
    "lyraq_last_cuda_error": (ctypes.c_char_p, []),
    "lyraq_debug_set_row_vectors_per_thread": (c_int, [c_int]),
    "lyraq_debug_set_special_row_kernels": (c_int, [c_int]),
    "lyraq_quant_int8": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int, c_size_t, c_size_t, c_void_p]),
    "lyraq_quant_fp8": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_size_t, c_void_p]),
    "lyraq_fp8_amax_scale": (c_int, [c_void_p, c_void_p, c_int, c_size_t, c_void_p]),
    "lyraq_weight_quant_fp8": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_size_t, c_void_p]),
    "lyraq_quant_int4_g64": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_size_t,
                                     c_size_t, c_void_p]),
    "lyraq_weight_quant_int8": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_size_t, c_size_t, c_void_p]),
    "lyraq_weight_quant_int4_g64": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_size_t, c_size_t, c_void_p]),
    "lyraq_quant_fp4": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_size_t, c_void_p, c_int, c_size_t, c_size_t, c_void_p]),
    "lyraq_fp4_scale_bytes": (c_size_t, [c_size_t, c_size_t, c_int]),
    "lyraq_weight_quant_fp4": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_size_t, c_size_t, c_void_p]),
    "lyraq_adaln_quant": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                  c_void_p, c_size_t, c_size_t, c_size_t, c_double, c_void_p]),
    "lyraq_adaln_quant_fp8x2": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                        c_size_t, c_size_t, c_size_t, c_double, c_void_p]),
    "lyraq_ln_quant_int8": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p,
                                    c_void_p, c_size_t, c_size_t, c_double, c_void_p]),
    "lyraq_geglu_quant_int8": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_size_t, c_size_t,
                                       c_void_p]),
    "lyraq_workspace_bytes": (c_size_t, [c_int, c_int, c_int, c_int]),
    "lyraq_workspace_min_bytes": (c_size_t, [c_int, c_int, c_int, c_int]),
    "lyraq_gemm_int8": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_int,
                                c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_int8_residual": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
                                         c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp8": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_float,
                               c_float, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp8_gate": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int,
                                    c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp8_quant": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                     c_float, c_float, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp8_quant_ld": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p, c_int, c_void_p,
                                        c_void_p, c_float, c_float, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp8_qk_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_int, c_void_p, c_void_p, c_void_p,
                                       c_int, c_int, c_double, c_int, c_int, c_int, c_void_p]),
    "lyraq_rmsnorm_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_double, c_size_t, c_size_t, c_int, c_int,
                                   c_void_p]),
    "lyraq_attention": (c_int, [c_void_p, c_int, c_size_t, c_void_p, c_void_p, c_size_t, c_void_p, c_size_t, c_void_p, c_int,
                                c_size_t, c_size_t, c_int, c_int, c_float, c_void_p]),
    "lyraq_quant_fp8_2d": (c_int, [c_void_p, c_size_t, c_void_p, c_int, c_void_p, c_size_t, c_size_t, c_void_p]),
    "lyraq_load_lora": (c_int, [c_void_p, c_void_p, c_int, c_float, c_size_t, c_void_p]),
    "lyraq_gate_residual": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_size_t, c_size_t, c_size_t, c_void_p]),
    "lyraq_rope_axes": (c_int, [c_void_p, c_void_p]),
    "lyraq_gated_residual_norm": (c_int, [c_void_p, c_void_p]),
    "lyraq_gemm_w4a4": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_void_p,
                                c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_gemm_fp4": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
                               c_float, c_int, c_int, c_int, c_int, c_void_p]),
    "lyraq_linear_fp4_forward": (c_int, [c_void_p, c_void_p, c_int, c_size_t, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p,
                                         c_void_p, c_float, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_linear_fp8_forward": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_float,
                                         c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_linear_int8_forward": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p,
                                          c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_w4a4_forward": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int,
                                   c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_w4a4_lora_forward": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                        c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "lyraq_w4a4_forward_static": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                          c_int, c_int, c_int, c_int, c_void_p]),
    "lyraq_static_scratch_bytes": (c_size_t, []),
}

_lib = None
_host = None


class LyraqError(RuntimeError):
    def __init__(self, status, where):
        self.status = status
        msg = lib().lyraq_status_string(status).decode() if _lib is not None else str(status)
        if status == 3 and _lib is not None:
            msg += " [" + lib().lyraq_last_cuda_error().decode() + "]"
        super().__init__("%s failed: %s (status %d)" % (where, msg, status))


def lib():
    """The loaded library with every declared symbol bound and typed."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                "liblyraq.so not found at %s; build it with `python -m lyradiff_b200.build` "
                "(there is no CPU or PyTorch fallback)" % LIB_PATH)
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)  # AttributeError if the library lacks a declared symbol
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def host():
    """The extension module _host (csrc/host_calls.cpp), bound to the loaded library's functions."""
    global _host
    if _host is None:
        path = os.path.join(_HERE, "_host" + sysconfig.get_config_var("EXT_SUFFIX"))    # this interpreter's: another's would crash it
        if not os.path.exists(path):
            raise ImportError("%s is not built: run `python -m lyradiff_b200.build` (there is no fallback)" % path)
        import torch  # noqa: F401  (its libraries are what the module links to)
        from . import _host as module
        handle = lib()
        names = ("lyraq_gated_residual_norm", "lyraq_rope_axes", "lyraq_linear_fp4_forward", "lyraq_gemm_fp4", "lyraq_quant_fp4",
                 "lyraq_workspace_bytes", "lyraq_fp4_scale_bytes")
        module.bind({n: ctypes.cast(getattr(handle, n), c_void_p).value for n in names}, LyraqError)
        _host = module
    return _host


def check(status, where):
    if status != 0:
        raise LyraqError(status, where)
