"""ctypes binding of libmvr.so (the C ABI of include/mvr.h).

The library is the only implementation: if it is missing or cannot be loaded, importing
this module raises -- nothing falls back to torch or to the CPU.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmvr.so")

MVR_F32, MVR_F16, MVR_F64, MVR_BF16 = 0, 1, 2, 3
MVR_ROI_BOX, MVR_ROI_ROTATED = 0, 1
MVR_ERR_ROI_WIDTH = -7
MVR_ERR_UNSUPPORTED = -13
MVR_STATUS_BAD_BATCH_INDEX = 1
MVR_STATUS_TMA_TIMEOUT = 2

_i64, _i32, _f32, _vp = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_void_p
_u64, _f64 = ctypes.c_uint64, ctypes.c_double


class Attention(ctypes.Structure):
    """struct mvr_attention of include/mvr.h."""
    _fields_ = [("dtype", _i32), ("has_index", _i32)] + [(n, _i64) for n in ("R", "T", "Hq", "Hk", "N", "L", "D")] + \
        [("q", _vp), ("k", _vp), ("v", _vp), ("q_strides", _i64 * 3), ("k_strides", _i64 * 3), ("v_strides", _i64 * 3),
         ("index", _vp), ("index_type", _i32), ("lengths_64", _i32), ("index_stride", _i64), ("lengths", _vp), ("mask", _vp),
         ("scale", _f32), ("out", _vp), ("lse", _vp), ("grad_out", _vp), ("g_strides", _i64 * 3), ("grad_q", _vp),
         ("grad_k", _vp), ("grad_v", _vp)]


class Window(ctypes.Structure):
    """struct mvr_window of include/mvr.h."""
    _fields_ = [("before", _i64), ("after", _i64), ("sinks", _i64), ("offset", _i64), ("offsets", _vp), ("offsets_64", _i32), ("rest", _vp),
                ("rounded_weights", _i32)]


class GroupNorm(ctypes.Structure):
    """struct mvr_group_norm of include/mvr.h."""
    _fields_ = [("dtype", _i32), ("parameter_dtype", _i32), ("activation", _i32), ("eps", _f32)] + [(n, _i64) for n in ("N", "S", "C", "groups")] + \
        [(n, _vp) for n in ("x", "weight", "bias", "out", "mean", "rstd", "mean_rest", "grad_out", "grad_x", "grad_weight", "grad_bias")]


class Rotary(ctypes.Structure):
    """struct mvr_rotary of include/mvr.h."""
    _fields_ = [("dtype", _i32), ("interleaved", _i32), ("inverse", _i32), ("axes", _i32), ("N", _i64), ("L", _i64), ("D", _i64), ("heads", _i64 * 2),
                ("sections", _i64 * 4), ("base", _f64), ("x", _vp * 2), ("strides", (_i64 * 3) * 2), ("out", _vp * 2), ("positions", _vp),
                ("position_dtype", _i32), ("position_strides", _i64 * 3)]


_attention, _window, _norm = ctypes.POINTER(Attention), ctypes.POINTER(Window), ctypes.POINTER(GroupNorm)

# name -> argtypes, exactly the prototypes of include/mvr.h
_GENERAL = [_vp, _vp, _vp, _i32, _i32, _i32, _i64, _i64, _i64, _i64, _i64, _i64, _i32,
            _i32, _i32, _i32, _f32, _i32, _i32, _i32, _vp, _vp]
_BOX2D = [_vp, _vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _f32, _i32, _i32, _vp, _vp]
_BOX3D = [_vp, _vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _f32, _i32, _i32, _vp, _vp]
_ROT2D = [_vp, _vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _f32, _i32, _i32, _i32, _vp, _vp]
_ROT3D = [_vp, _vp, _vp, _i32, _i64, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _f32, _i32, _i32, _i32,
          _vp, _vp]

PROTOTYPES = {
    "mvr_roi_resample_fwd": _GENERAL,
    "mvr_roi_resample_bwd": _GENERAL,
    "mvr_roi_resample_bwd_noalloc": _GENERAL,
    "mvr_roi_resample_touched": [_vp, _vp, _i32, _i32, _i32, _i64, _i64, _i64, _i64, _i64, _i64, _i32,
                                 _i32, _i32, _i32, _f32, _i32, _i32, _i32, _vp],
    "mvr_roi_align_2d_forward": _BOX2D,
    "mvr_roi_align_2d_backward": _BOX2D,
    "mvr_roi_align_3d_forward": _BOX3D,
    "mvr_roi_align_3d_backward": _BOX3D,
    "mvr_roi_align_rotated_2d_forward": _ROT2D,
    "mvr_roi_align_rotated_2d_backward": _ROT2D,
    "mvr_roi_align_rotated_3d_forward": _ROT3D,
    "mvr_roi_align_rotated_3d_backward": _ROT3D,
    "mvr_apply_offset_2d": [_vp, _vp, _vp, _i32, _i32, _i64, _i64, _i64, _i64, _i32, _vp],
    "mvr_apply_offset_3d": [_vp, _vp, _vp, _i32, _i32, _i64, _i64, _i64, _i64, _i64, _i32, _vp],
    "mvr_affine_label_2d": [_vp, _i32, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _f32, _i32, _vp, _vp],
    "mvr_affine_label_3d": [_vp, _i32, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _f32,
                            _i32, _vp, _vp],
    "mvr_affine_fields_3d": [_vp, _i32, _vp, _vp, _i64, _vp, _i32, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i32,
                             _i32, _i32, _i32, _f32, _i32, _i32, _vp, _vp],
    "mvr_affine_fields_2d": [_vp, _i32, _vp, _vp, _i64, _vp, _i32, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i32,
                             _f32, _i32, _i32, _vp, _vp],
    "mvr_elastic": [_vp, _i32, _i32, _i32, _i32, _i32, _vp, _i32, _vp, _i64, _vp, _i32, _vp, _i64, _vp, _i64, _i64, _i64,
                    _i64, _vp],
    "mvr_attention_workspace": [_attention, _i32, ctypes.POINTER(_i64)],
    "mvr_attention_forward": [_attention, _vp, _i64, _vp, _vp],
    "mvr_attention_backward": [_attention, _vp, _i64, _vp, _vp],
    "mvr_window_attention_workspace": [_attention, _window, _i32, ctypes.POINTER(_i64)],
    "mvr_window_attention_forward": [_attention, _window, _vp, _i64, _vp, _vp],
    "mvr_window_attention_backward": [_attention, _window, _vp, _i64, _vp, _vp],
    "mvr_group_norm_workspace": [_norm, _i32, ctypes.POINTER(_i64)],
    "mvr_group_norm_forward": [_norm, _vp, _i64, _vp],
    "mvr_group_norm_backward": [_norm, _vp, _i64, _vp],
    "mvr_rotary_positions": [ctypes.POINTER(Rotary), _vp],
    "mvr_dropout": [_vp, _vp, _vp, _i32, _i64, _f64, _u64, _vp, _u64, _vp],
    "mvr_label_log_probs_forward": [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _vp],
    "mvr_label_log_probs_backward": [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64,
                                     _vp],
    "mvr_label_log_probs_forward_rest": [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i32, _vp],
    "mvr_label_log_probs_backward_rest": [_vp, _i32, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64,
                                          _vp],
    "mvr_affine_2d": _ROT2D,
    "mvr_affine_3d": _ROT3D,
}
OTHER_SYMBOLS = ["mvr_strerror", "mvr_version", "mvr_set_float_contraction", "mvr_get_float_contraction",
                 "mvr_selftest_tma_skip_plane", "mvr_cached_memory_bytes", "mvr_release_cached_memory"]


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m medvision_b200.build` "
            "(medvision_b200 has no CPU or torch fallback)")
    lib = ctypes.CDLL(LIB_PATH)
    for name, argtypes in PROTOTYPES.items():
        fn = getattr(lib, name)
        fn.restype = _i32
        fn.argtypes = argtypes
    lib.mvr_strerror.restype = ctypes.c_char_p
    lib.mvr_strerror.argtypes = [_i32]
    lib.mvr_version.restype = _i32
    lib.mvr_set_float_contraction.restype = _i32
    lib.mvr_set_float_contraction.argtypes = [_i32]
    lib.mvr_get_float_contraction.restype = _i32
    lib.mvr_selftest_tma_skip_plane.restype = _i32
    lib.mvr_cached_memory_bytes.restype = ctypes.c_longlong
    lib.mvr_cached_memory_bytes.argtypes = []
    lib.mvr_release_cached_memory.restype = _i32
    lib.mvr_release_cached_memory.argtypes = []
    lib.mvr_selftest_tma_skip_plane.argtypes = [_i32]
    return lib


lib = _load()


def strerror(code):
    return lib.mvr_strerror(code).decode()
