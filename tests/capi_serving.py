"""ctypes view of the operators of a serving step in libminfer_attn.so (include/minfer_attn.h), beside capi.py and capi_paged.py."""
import ctypes

import capi
import capi_paged


class PageRing(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("state", ctypes.c_void_p), ("state_after", ctypes.c_void_p), ("n_pages", ctypes.c_int64)]


def lib():
    L = capi_paged.lib()
    i64, vp, sz, i, ring = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.POINTER(PageRing)
    L.minfer_paged_tables.restype = i
    L.minfer_paged_tables.argtypes = [i64, vp, vp, vp, ring, vp, i64, i64, vp, vp, vp, i64, vp, i64, vp]
    L.minfer_paged_release_workspace_bytes.restype = sz
    L.minfer_paged_release_workspace_bytes.argtypes = [i64]
    L.minfer_paged_release.restype = i
    L.minfer_paged_release.argtypes = [i64, vp, vp, ring, vp, i64, i64, vp, i64, vp, sz, vp]
    L.minfer_verify_drafts_workspace_bytes.restype = sz
    L.minfer_verify_drafts_workspace_bytes.argtypes = [i64, i64]
    L.minfer_verify_drafts.restype = i
    L.minfer_verify_drafts.argtypes = [i, i] + [vp] * 8 + [i64] * 5 + [vp, sz, vp]
    L.minfer_flash_attn_paged_shared_workspace_bytes.restype = sz
    L.minfer_flash_attn_paged_shared_workspace_bytes.argtypes = [i64] * 8
    L.minfer_flash_attn_paged_shared.restype = i
    L.minfer_flash_attn_paged_shared.argtypes = [i, i, vp, ctypes.POINTER(capi_paged.KvPages)] + [vp] * 5 + [i64] * 7 + [ctypes.POINTER(capi.Strides), vp, sz, vp]
    return L
