"""ctypes view of the paged operators of libminfer_attn.so (include/minfer_attn.h), beside capi.py."""
import ctypes

import capi

FP8_E4M3 = 256


class KvPages(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("n_pages", ctypes.c_int64), ("page_size", ctypes.c_int64),
                ("stride_page", ctypes.c_int64), ("stride_head", ctypes.c_int64), ("stride_row", ctypes.c_int64),
                ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("pages_per_seq", ctypes.c_int64)]


def lib():
    L = capi.lib()
    i64, vp, sz, i = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
    L.minfer_rope_kv_append_paged.restype = i
    L.minfer_rope_kv_append_paged.argtypes = [i, i, i, vp, vp, vp, vp, vp, ctypes.POINTER(KvPages)] + [i64] * 6 + [ctypes.c_double, vp]
    L.minfer_flash_attn_paged_workspace_bytes.restype = sz
    L.minfer_flash_attn_paged_workspace_bytes.argtypes = [i64] * 7
    L.minfer_flash_attn_paged.restype = i
    L.minfer_flash_attn_paged.argtypes = [i, i, vp, ctypes.POINTER(KvPages), vp, vp, vp] + [i64] * 6 + [ctypes.POINTER(capi.Strides), vp, sz, vp]
    return L
