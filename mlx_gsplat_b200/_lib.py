"""ctypes binding of ``libgsplat_b200.so`` (C ABI in ``include/gsplat_b200.h``).

The product has no CPU fallback: every call goes to the CUDA library, and
loading fails loudly when the library is missing or CUDA is unavailable.
"""
from __future__ import annotations

import ctypes
import os
import sys
import warnings
from typing import Optional

import torch

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libgsplat_b200.so")
TENSORS_PATH = os.path.join(PKG, "libgsplat_tensors.so")

GS_OK, GS_ERR_INVALID, GS_ERR_CUDA, GS_ERR_CAPACITY = 0, 1, 2, 3
GS_ADAM_FUSED, GS_ADAM_PURE, GS_ADAM_EXACT = 0, 1, 0x100
GS_LOSS_NONE, GS_LOSS_L1_U8, GS_LOSS_L1_F32, GS_LOSS_MEAN = 0, 1, 2, 3
GS_SH_REFERENCE, GS_SH_FULL = 0, 1
GS_ROWS_ALL, GS_ROWS_SEEN, GS_ROWS_UNSEEN = 0, 1, 2
GS_F32, GS_BF16, GS_F16 = 0, 1, 2
GS_MOMENT_BLOCK = 256

c_float_p = ctypes.POINTER(ctypes.c_float)
c_vp = ctypes.c_void_p
i64 = ctypes.c_int64
i32 = ctypes.c_int32


class GsGaussians(ctypes.Structure):
    _fields_ = [("means", c_vp), ("means_stride", i64),
                ("quats", c_vp), ("quats_stride", i64),
                ("scales", c_vp), ("scales_stride", i64),
                ("opac", c_vp), ("opac_stride", i64),
                ("colors", c_vp), ("colors_stride", i64),
                ("colors_dim", i32), ("colors_by_visible", i32),
                ("table", c_vp), ("sh_mode", i32)]


class GsGaussianGrads(ctypes.Structure):
    _fields_ = [("means", c_vp), ("means_stride", i64),
                ("quats", c_vp), ("quats_stride", i64),
                ("scales", c_vp), ("scales_stride", i64),
                ("opac", c_vp), ("opac_stride", i64),
                ("colors", c_vp), ("colors_stride", i64),
                ("colors_write", i32), ("colors_by_visible", i32), ("accumulate", i32),
                ("reg", ctypes.c_float), ("reg_color_cols", i32), ("reg_geometry", i32), ("count_col", i32)]


class GsCamera(ctypes.Structure):
    _fields_ = [("viewmat", ctypes.c_float * 16),
                ("fx", ctypes.c_float), ("fy", ctypes.c_float), ("cx", ctypes.c_float), ("cy", ctypes.c_float),
                ("width", i32), ("height", i32), ("render_width", i32), ("render_height", i32)]


class GsRasterSettings(ctypes.Structure):
    _fields_ = [("alpha_cutoff", ctypes.c_float), ("transmittance_min", ctypes.c_float), ("alpha_mask", i32)]


class GsAdamWState(ctypes.Structure):
    _fields_ = [("m", c_vp), ("v", c_vp), ("m_exp", c_vp), ("v_exp", c_vp), ("master", c_vp), ("control", c_vp),
                ("bits", i32), ("counted", i32)]


class GsAdamWSettings(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double),
                ("eps", ctypes.c_float), ("grad_scale", ctypes.c_double), ("lr_device", c_vp),
                ("norm_partials", c_vp), ("num_partials", i64), ("max_norm", ctypes.c_double), ("norm_out", c_vp)]


_SIGS = {
    "gs_last_error": (ctypes.c_char_p, []),
    "gs_abi_version": (ctypes.c_int, []),
    "gs_kernel_launches": (ctypes.c_ulonglong, []),
    "gs_launch_fused_adam_step": (ctypes.c_int, [ctypes.c_uint64] * 5 + [ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int,
                                                                        ctypes.c_float, ctypes.c_float, ctypes.c_float,
                                                                        ctypes.c_float, ctypes.c_float, ctypes.c_int,
                                                                        ctypes.c_float, ctypes.c_float, c_vp]),
    "gs_clear_buffer_cache": (ctypes.c_int, []),
    "gs_fused_adam_group": (ctypes.c_int, [c_vp] * 5 + [i64, ctypes.c_int, i64, i64] + [ctypes.c_double] * 3 +
                            [ctypes.c_float] * 2 + [ctypes.c_int] + [ctypes.c_float] * 4 + [ctypes.c_int, c_vp]),
    "gs_fused_adam_slab": (ctypes.c_int, [c_vp] * 5 + [i64, ctypes.c_int, i64, i64, c_float_p, c_float_p, c_float_p,
                                                       ctypes.c_int] + [ctypes.c_double] * 3 + [ctypes.c_float] * 2 +
                           [ctypes.c_int, ctypes.c_float, ctypes.c_int, c_vp, c_float_p, c_float_p,
                            ctypes.c_int, ctypes.c_int, c_float_p, ctypes.c_int, c_vp]),
    "gs_cull_scratch_bytes": (ctypes.c_size_t, [i64]),
    "gs_cull": (ctypes.c_int, [ctypes.POINTER(GsGaussians), i64, ctypes.POINTER(GsCamera), ctypes.c_float,
                               ctypes.c_float, ctypes.c_float, c_vp, c_vp, c_vp, ctypes.c_size_t, c_vp]),
    "gs_cull_noalloc": (ctypes.c_int, [ctypes.POINTER(GsGaussians), i64, ctypes.POINTER(GsCamera), ctypes.c_float,
                                       ctypes.c_float, ctypes.c_float, c_vp, c_vp, c_vp]),
    "gs_radix_sort_scratch_bytes": (ctypes.c_size_t, [i64]),
    "gs_radix_sort_pairs": (ctypes.c_int, [c_vp] * 4 + [i64, ctypes.c_int, ctypes.c_int, c_vp, ctypes.c_size_t, c_vp]),
    "gs_scan_scratch_bytes": (ctypes.c_size_t, [i64]),
    "gs_exclusive_scan_u32": (ctypes.c_int, [c_vp, c_vp, i64, c_vp, ctypes.c_size_t, c_vp]),
    "gs_project_forward": (ctypes.c_int, [ctypes.POINTER(GsGaussians), c_vp, i64, ctypes.POINTER(GsCamera),
                                          ctypes.POINTER(GsRasterSettings), c_vp, c_vp, c_vp, c_vp, c_vp]),
    "gs_bin_scratch_bytes": (ctypes.c_size_t, [i64]),
    "gs_bin_offsets_scratch_bytes": (ctypes.c_size_t, [i64]),
    "gs_bin_offsets": (ctypes.c_int, [c_vp, c_vp, i64, c_vp, c_vp, ctypes.c_size_t, c_vp]),
    "gs_bin_emit": (ctypes.c_int, [c_vp] * 4 + [i64, ctypes.POINTER(GsCamera), ctypes.POINTER(GsRasterSettings),
                                                c_vp, c_vp, i64, c_vp, c_vp, c_vp]),
    "gs_tile_ranges": (ctypes.c_int, [c_vp, i64, ctypes.c_int32, c_vp, c_vp]),
    "gs_tile_order": (ctypes.c_int, [c_vp, ctypes.c_int32, c_vp, c_vp]),
    "gs_render_forward": (ctypes.c_int, [c_vp, c_vp, c_vp, c_vp, i64, ctypes.POINTER(GsCamera),
                                         ctypes.POINTER(GsRasterSettings), c_vp, c_vp, c_vp, c_vp, ctypes.c_int,
                                         c_vp, c_vp, c_vp]),
    "gs_render_pair_count": (ctypes.c_int, [c_vp, c_vp, c_vp, c_vp, i64, ctypes.POINTER(GsCamera),
                                             ctypes.POINTER(GsRasterSettings), c_vp, c_vp]),
    "gs_fp32_peak_probe": (ctypes.c_int, [c_vp, i64, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                          ctypes.POINTER(ctypes.c_double), c_vp]),
    "gs_apply_sorted_mask": (ctypes.c_int, [c_vp, c_vp, c_vp, i64, ctypes.POINTER(GsRasterSettings), c_vp]),
    "gs_render_backward": (ctypes.c_int, [c_vp, c_vp, c_vp, c_vp, i64, ctypes.POINTER(GsCamera),
                                          ctypes.POINTER(GsRasterSettings), c_vp, c_vp, c_vp, ctypes.c_int, c_vp,
                                          c_vp, c_vp, c_vp, c_vp]),
    "gs_project_backward": (ctypes.c_int, [ctypes.POINTER(GsGaussians), c_vp, i64, ctypes.POINTER(GsCamera), c_vp,
                                           ctypes.POINTER(GsGaussianGrads), c_vp, c_vp, c_vp]),
    "gs_export_rows": (ctypes.c_int, [c_vp, i64, c_vp, i64] + [ctypes.c_int] * 6 + [c_vp, i64, c_vp]),
    "gs_l1_dssim_scratch_bytes": (ctypes.c_size_t, [i32, i32]),
    "gs_l1_dssim_loss": (ctypes.c_int, [c_vp, c_vp, ctypes.c_int, i32, i32, ctypes.c_float, ctypes.c_float, c_vp,
                                        c_vp, c_vp, c_vp, ctypes.c_size_t, c_vp]),
    "gs_resize_bilinear": (ctypes.c_int, [c_vp, ctypes.c_int, i32, i32, i32, c_vp, i32, i32, c_vp]),
    "gs_group_barrier": (ctypes.c_int, [c_vp, i32, i32, i32, ctypes.c_uint32, c_vp, i64, c_vp]),
    "gs_rows_sum_multicast": (ctypes.c_int, [c_vp, i64, i64, i64, c_vp, c_vp]),
    "gs_fused_adam_slab_sharded": (ctypes.c_int, [c_vp] * 6 + [i64, ctypes.c_int, i64, i64, c_float_p, c_float_p,
                                                               ctypes.c_int] + [ctypes.c_double] * 3 +
                                   [ctypes.c_float, ctypes.c_float, ctypes.c_int, ctypes.c_float, c_float_p,
                                    ctypes.c_int, ctypes.c_int, c_float_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                    c_vp, c_vp]),
    "gs_compact_flags": (ctypes.c_int, [c_vp, i64, ctypes.c_uint8, ctypes.c_uint8, c_vp, c_vp, c_vp, c_vp,
                                        ctypes.c_size_t, c_vp]),
    "gs_densify_masks": (ctypes.c_int, [ctypes.POINTER(GsGaussians), c_vp, c_vp, i64] + [ctypes.c_float] * 5 +
                         [ctypes.c_int, c_vp, c_vp]),
    "gs_densify_children": (ctypes.c_int, [c_vp, i64, ctypes.c_int] + [c_vp] * 6 + [i64] + [ctypes.c_int] * 4 +
                            [c_vp, c_vp, c_vp]),
    "gs_pool_write_rows": (ctypes.c_int, [c_vp, c_vp, c_vp, i64, c_vp, i64, c_vp, i64, c_float_p, c_vp, c_vp, c_vp]),
    "gs_free_pop_reversed": (ctypes.c_int, [c_vp, i64, i64, c_vp, c_vp]),
    "gs_fill_rows": (ctypes.c_int, [c_vp, i64, i64, c_float_p, c_vp]),
    "gs_fill_column": (ctypes.c_int, [c_vp, i64, i64, ctypes.c_int, ctypes.c_float, c_vp]),
    "gs_mark_slots": (ctypes.c_int, [c_vp, i64, c_vp, i64, ctypes.c_int, c_vp]),
    # many-tensor calls: the first argument is the address of an array of gs_tensor
    "gs_adamw_step": (ctypes.c_int, [c_vp, i64, ctypes.POINTER(GsAdamWState), ctypes.POINTER(GsAdamWSettings), c_vp]),
    "gs_grad_norm_max_partials": (i64, [i64]),
    "gs_grad_norm_partials": (ctypes.c_int, [c_vp, i64, c_vp, i64, ctypes.POINTER(i64), c_vp]),
    "gs_clip_gradients": (ctypes.c_int, [c_vp, i64, c_vp, i64, ctypes.c_double, c_vp, c_vp]),
    "gs_moments8_quantize": (ctypes.c_int, [c_vp, i64, c_vp, c_vp, c_vp, c_vp, i64, c_vp]),
    "gs_moments8_dequantize": (ctypes.c_int, [c_vp, c_vp, c_vp, c_vp, i64, ctypes.c_int, c_vp, c_vp, c_vp]),
    "gs_copy_rows": (ctypes.c_int, [c_vp, i64, c_vp, c_vp, i64, c_vp, i64, ctypes.c_int, c_vp]),
}

_LIB: Optional[ctypes.CDLL] = None


class GsplatError(RuntimeError):
    pass


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the library and declare every signature (no CUDA needed to load)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(path):
        raise GsplatError(f"{path} is missing: build it with `python -m mlx_gsplat_b200.build` "
                          "(there is no CPU fallback)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in _SIGS.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _LIB = lib
    return lib


_TENSORS: Optional[ctypes.PyDLL] = None
_TENSORS_DECIDED = False


def tensors_abi() -> str:
    """What the tensor helper is compiled against: it reads the insides of
    torch's tensors, which change between versions."""
    return f"torch {torch.__version__}, python {sys.version_info.major}.{sys.version_info.minor}"


def load_tensors(path: str) -> ctypes.PyDLL:
    """The helper at ``path``; OSError where it cannot be loaded or was compiled
    against another torch or Python."""
    dll = ctypes.PyDLL(path)
    try:
        dll.gst_abi.restype = ctypes.c_char_p
        abi = dll.gst_abi().decode()
    except AttributeError:
        abi = "an unknown torch"
    if not all(hasattr(dll, name) for name in ("gst_fill", "gst_step", "gst_params_unmoved", "gst_params_as_taken",
                                                "gst_clip")):
        raise OSError(f"{path} is not the tensor helper")
    if abi != tensors_abi():
        raise OSError(f"{path} was compiled against {abi}, not {tensors_abi()}")
    obj, size = ctypes.py_object, ctypes.c_ssize_t
    dll.gst_fill.argtypes = [obj, obj, obj, obj, c_vp, size, ctypes.c_int]
    dll.gst_step.argtypes = [obj, obj, obj, obj, c_vp, size, ctypes.c_int, ctypes.POINTER(size)]
    dll.gst_params_unmoved.argtypes = [obj, c_vp, size]
    dll.gst_params_as_taken.argtypes = [obj, obj, c_vp, size]
    dll.gst_clip.argtypes = [obj, obj, c_vp, size, ctypes.POINTER(ctypes.c_int)]
    return dll


def tensors() -> Optional[ctypes.PyDLL]:
    """The helper that reads tensors' metadata natively (``csrc/tensors.cpp``;
    called with the GIL held), or None where there is none for this torch: the
    callers' own checks in Python then do the same.  Decided at the first call."""
    global _TENSORS, _TENSORS_DECIDED
    if not _TENSORS_DECIDED:
        _TENSORS_DECIDED = True
        if os.path.exists(TENSORS_PATH):
            try:
                _TENSORS = load_tensors(TENSORS_PATH)
            except OSError as e:
                warnings.warn(f"tensors are read in Python, not natively: {e}; rebuild with "
                              "`python -m mlx_gsplat_b200.build`", RuntimeWarning, stacklevel=2)
    return _TENSORS


def exported_names():
    return list(_SIGS.keys())


def lib() -> ctypes.CDLL:
    """The library, for compute calls: also requires a CUDA device."""
    if not torch.cuda.is_available():
        raise GsplatError("libgsplat_b200 needs a CUDA device; there is no CPU fallback")
    return load()


def check(status: int, what: str = "") -> None:
    if status == GS_OK:
        return
    msg = load().gs_last_error().decode(errors="replace")
    if status == GS_ERR_CAPACITY:
        raise MemoryError(f"{what}: {msg}")
    raise GsplatError(f"{what} failed ({status}): {msg}")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device: Optional[torch.device] = None) -> int:
    """The device's current stream (without building a Stream object where
    torch offers its address, which is most of a small call's host time)."""
    if _raw_stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    index = None if device is None else device.index
    return _raw_stream(torch.cuda.current_device() if index is None else index)


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def fptr(arr) -> "ctypes.Array":
    """Host float32 array argument."""
    vals = [float(x) for x in arr]
    return (ctypes.c_float * len(vals))(*vals)
