"""ctypes binding of include/h2o4gpu_experts.h: expert layers and 4-bit products on device pointers.

Same library as kmeans_hip; the torch-facing functions are h2o4gpu_amd.experts, h2o4gpu_amd.codebook4
and h2o4gpu_amd.microscale4.
"""
import ctypes

from . import kmeans_hip

c_int = ctypes.c_int
c_size_t = ctypes.c_size_t
c_ssize_t = ctypes.c_ssize_t
c_float = ctypes.c_float
c_void_p = ctypes.c_void_p

FLOAT32, BFLOAT16, FLOAT16 = 0, 1, 2
MAX_EXPERTS = 16384
MAX_TOP_K = 64
MAX_GROUP = 1 << 30
MAX_SIDE = 1 << 20

# every symbol include/h2o4gpu_experts.h declares: name -> (restype, argtypes)
PROTOTYPES = {
    "h2o4gpu_experts_route": (c_int, [c_int, c_size_t, c_int, c_int, c_int, c_int, c_float, c_void_p, c_ssize_t,
                                      c_ssize_t, c_void_p, c_void_p, c_void_p]),
    "h2o4gpu_experts_route_backward": (c_int, [c_int, c_size_t, c_int, c_int, c_int, c_int, c_float, c_void_p,
                                               c_ssize_t, c_ssize_t, c_void_p, c_void_p, c_void_p, c_void_p,
                                               c_ssize_t, c_ssize_t, c_void_p]),
    "h2o4gpu_experts_sort_workspace": (c_size_t, [c_size_t, c_int]),
    "h2o4gpu_experts_sort": (c_int, [c_size_t, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t,
                                     c_void_p]),
    "h2o4gpu_experts_dispatch": (c_int, [c_int, c_size_t, c_int, c_size_t, c_void_p, c_size_t, c_void_p, c_void_p,
                                         c_size_t, c_void_p]),
    "h2o4gpu_experts_dispatch_backward": (c_int, [c_int, c_size_t, c_int, c_size_t, c_void_p, c_size_t, c_void_p,
                                                  c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_experts_combine": (c_int, [c_int, c_size_t, c_int, c_size_t, c_void_p, c_size_t, c_void_p, c_void_p,
                                        c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_experts_combine_backward": (c_int, [c_int, c_size_t, c_int, c_size_t, c_void_p, c_size_t, c_void_p,
                                                 c_size_t, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p,
                                                 c_void_p]),
    "h2o4gpu_codebook4_quantize": (c_int, [c_int, c_size_t, c_size_t, c_int, c_float, c_void_p, c_size_t, c_void_p,
                                           c_void_p, c_size_t, c_int, c_void_p, c_void_p]),
    "h2o4gpu_codebook4_codes_bytes": (c_size_t, [c_size_t, c_size_t, c_size_t]),
    "h2o4gpu_codebook4_scales_bytes": (c_size_t, [c_size_t, c_size_t, c_size_t, c_int, c_int]),
    "h2o4gpu_codebook4_layout": (c_int, [c_size_t, c_size_t, c_size_t, c_int, c_void_p, c_size_t, c_int, c_void_p,
                                         c_void_p, c_void_p, c_void_p]),
    "h2o4gpu_codebook4_product": (c_int, [c_int, c_size_t, c_size_t, c_size_t, c_int, c_void_p, c_size_t, c_void_p,
                                          c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_codebook4_experts_product": (c_int, [c_int, c_size_t, c_int, c_int, c_size_t, c_size_t, c_int,
                                                  c_void_p, c_size_t, c_void_p, c_int, c_void_p, c_void_p, c_size_t,
                                                  c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_experts_product": (c_int, [c_int, c_size_t, c_int, c_size_t, c_size_t, c_void_p, c_size_t, c_void_p,
                                        c_size_t, c_size_t, c_void_p, c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_experts_product_drows": (c_int, [c_int, c_size_t, c_int, c_size_t, c_size_t, c_void_p, c_size_t,
                                              c_void_p, c_size_t, c_size_t, c_void_p, c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_experts_product_dweights": (c_int, [c_int, c_size_t, c_int, c_size_t, c_size_t, c_void_p, c_size_t,
                                                 c_void_p, c_size_t, c_void_p, c_void_p, c_void_p, c_size_t,
                                                 c_void_p]),
    "h2o4gpu_experts_align_rows": (c_int, [c_int, c_size_t, c_size_t, c_size_t, c_void_p, c_size_t, c_size_t, c_void_p,
                                           c_void_p]),
    "h2o4gpu_experts_product_dweights_workspace": (c_size_t, [c_int, c_size_t, c_int, c_size_t, c_size_t]),
    "h2o4gpu_microscale4_codes_pitch": (c_size_t, [c_size_t]),
    "h2o4gpu_microscale4_scales_pitch": (c_size_t, [c_size_t]),
    "h2o4gpu_microscale4_quantize": (c_int, [c_int, c_size_t, c_size_t, c_void_p, c_size_t, c_void_p, c_void_p,
                                             c_void_p]),
    "h2o4gpu_microscale4_dequantize": (c_int, [c_int, c_size_t, c_size_t, c_void_p, c_void_p, c_void_p, c_size_t,
                                               c_void_p]),
    "h2o4gpu_microscale4_layout": (c_int, [c_size_t, c_size_t, c_void_p, c_size_t, c_void_p, c_void_p, c_void_p,
                                           c_void_p]),
    "h2o4gpu_microscale4_product": (c_int, [c_int, c_size_t, c_size_t, c_size_t, c_void_p, c_void_p, c_void_p,
                                            c_void_p, c_void_p, c_size_t, c_void_p]),
    "h2o4gpu_microscale4_experts_product": (c_int, [c_int, c_size_t, c_int, c_int, c_size_t, c_size_t, c_void_p,
                                                    c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                                    c_size_t, c_void_p]),
}

_lib = None


def lib():
    """The shared library with these functions' signatures set (loaded once)."""
    global _lib
    if _lib is None:
        handle = kmeans_hip.lib()
        for name, (res, args) in PROTOTYPES.items():
            fn = getattr(handle, name)  # AttributeError if the symbol is not exported
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def check(name, rc):
    if rc != 0:
        raise kmeans_hip.KMeansHipError(name, rc)
