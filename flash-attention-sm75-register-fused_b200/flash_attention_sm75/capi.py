"""ctypes binding of the C ABI in include/fa_b200.h.

Loads the in-tree ``lib/libfa_b200.so`` and declares every entry point with
its C signature, so Python callers (tests, bench.py, hosts without the pybind
module) call the same boundary a C or cgo host would.  Torch is used only to
obtain device pointers and the current stream in the tensor helpers.
"""
import ctypes
import os

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG_DIR, "lib", "libfa_b200.so")

c_vp, c_int, c_float, c_bool = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_bool

c_ll = ctypes.c_longlong


class PagedCache(ctypes.Structure):
    """fa_paged_cache of include/fa_b200.h."""
    _fields_ = [("k", c_vp), ("v", c_vp), ("k_scale", c_vp), ("v_scale", c_vp),
                ("page_stride", c_ll), ("head_stride", c_ll), ("row_stride", c_ll),
                ("scale_page_stride", c_ll), ("scale_head_stride", c_ll),
                ("scale_row_stride", c_ll), ("block_table", c_vp), ("table_stride", c_ll),
                ("max_pages", c_int), ("num_pages", c_int), ("kv_heads", c_int),
                ("page_size", c_int), ("head_dim", c_int), ("dtype", c_int)]


SIGNATURES = {
    "fa_kvcache_write": (c_int, [ctypes.POINTER(PagedCache), c_vp, c_vp, c_ll, c_ll, c_ll, c_ll,
                                 c_vp, c_vp, c_int, c_int, c_int, c_vp]),
    "fa_kvcache_read": (c_int, [ctypes.POINTER(PagedCache), c_vp, c_vp, c_vp, c_vp, c_int, c_int,
                                c_int, c_vp]),
    "fa_fwd_paged": (c_int, [ctypes.POINTER(PagedCache), c_vp, c_ll, c_ll, c_vp, c_vp, c_vp, c_vp,
                             c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_vp,
                             ctypes.c_size_t, c_vp]),
    "fa_fwd_paged_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(PagedCache), c_int, c_int,
                                                       c_int, c_int, c_int]),
    "fa_fwd": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_int, c_float,
                       c_int, c_int, c_vp]),
    "fa_fwd_kvcache": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_int,
                               c_int, c_float, c_int, c_int, c_vp, ctypes.c_size_t, c_vp]),
    "fa_fwd_kvcache_workspace_bytes": (ctypes.c_size_t, [c_int, c_int, c_int, c_int, c_int, c_int]),
    "fa_bwd": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int,
                       c_int, c_int, c_float, c_int, c_int, c_vp, ctypes.c_size_t, c_vp]),
    "fa_bwd_workspace_bytes": (ctypes.c_size_t, [c_int, c_int, c_int]),
    "fa_bwd_padded": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                              c_vp, c_vp, c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int,
                              c_vp, ctypes.c_size_t, c_vp]),
    "fa_bwd_varlen": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_int,
                              c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_vp,
                              ctypes.c_size_t, c_vp]),
    "fa_fwd_varlen": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int,
                              c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_vp]),
    "fa_fwd_padded": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_int,
                              c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_vp]),
    "launch_flash_attention_forward": (None, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int,
                                              c_float, c_bool]),
    "launch_flash_attention_forward_scalar": (None, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int,
                                                     c_int, c_float, c_bool]),
    "launch_flash_attention_forward_wmma_qk": (None, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int,
                                                      c_int, c_float, c_bool]),
    "launch_naive_attention": (None, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_float,
                                      c_bool, c_vp]),
    "fa_naive_fwd": (c_int, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_float, c_int,
                             c_vp, c_vp]),
    "fa_naive_fwd_noalloc": (c_int, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_float,
                                     c_int, c_vp]),
    "flatargs_launch": (c_int, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_float, c_vp]),
    "launch_v2": (c_int, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_float, c_int, c_vp]),
    "fa_device_status": (c_int, [c_int]),
    "fa_set_watchdog_ns": (None, [ctypes.c_ulonglong]),
    "fa_set_debug_flags": (None, [c_int]),
    "fa_set_trace_buffer": (None, [c_vp]),
    "fa_error_string": (ctypes.c_char_p, [c_int]),
    "fa_smem_bytes": (c_int, [c_int]),
    "fa_version": (ctypes.c_char_p, []),
}

_lib = None


def load():
    global _lib
    if _lib is None:
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def stream_ptr(torch_stream=None):
    import torch
    s = torch_stream or torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def fa_fwd(q, k, v, o, lse=None, causal=False, scale=None, stream=None):
    """Call fa_fwd on torch CUDA tensors laid out [B, H, N, d]; returns the status."""
    import math
    import torch
    B, Hq, N, d = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    return load().fa_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), B, Hq, Hkv, N, d,
                         float(scale), int(bool(causal)), dtype, stream_ptr(stream))


CAUSAL_NONE, CAUSAL_BOTTOM_RIGHT, CAUSAL_TOP_LEFT = 0, 1, 2


def fa_fwd_kvcache(q, k, v, o, lse=None, causal=CAUSAL_NONE, scale=None, stream=None,
                   workspace=True):
    """Call fa_fwd_kvcache on torch CUDA tensors (Q/O [B, Hq, Nq, d], K/V
    [B, Hkv, Nk, d]); ``workspace=True`` allocates the split workspace the
    library asks for, ``None`` runs unsplit.  Returns the status."""
    import math
    import torch
    B, Hq, Nq, d = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    lib = load()
    ws, nbytes = None, 0
    if workspace is True:
        nbytes = lib.fa_fwd_kvcache_workspace_bytes(B, Hq, Hkv, Nq, Nk, d)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    elif workspace is not None:
        ws, nbytes = workspace, workspace.numel() * workspace.element_size()
    return lib.fa_fwd_kvcache(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), B, Hq, Hkv, Nq, Nk, d,
                              float(scale), int(causal), dtype, ptr(ws), nbytes,
                              stream_ptr(stream))


def fa_bwd(q, k, v, o, do, lse, dq, dk, dv, causal=False, scale=None, stream=None):
    """Call fa_bwd on torch CUDA tensors ([B, H, N, d]; lse [B, Hq, N] fp32);
    allocates the workspace.  Returns the status."""
    import math
    import torch
    B, Hq, N, d = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    lib = load()
    nbytes = lib.fa_bwd_workspace_bytes(B, Hq, N)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    return lib.fa_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(do), ptr(lse), ptr(dq), ptr(dk), ptr(dv),
                      B, Hq, Hkv, N, d, float(scale), int(bool(causal)), dtype, ptr(ws), nbytes,
                      stream_ptr(stream))


def fa_fwd_varlen(q, k, v, o, lse, cu_q, cu_k, max_q, max_k, causal=CAUSAL_NONE, scale=None,
                  stream=None):
    """Call fa_fwd_varlen on packed torch CUDA tensors (Q/O [total_q, Hq, d],
    K/V [total_k, Hkv, d], LSE [Hq, total_q] or None, cu_* int32 [B + 1] on the
    device).  Returns the status."""
    import math
    import torch
    Tq, Hq, d = q.shape
    Tk, Hkv = k.shape[0], k.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    return load().fa_fwd_varlen(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(cu_q), ptr(cu_k),
                                cu_q.numel() - 1, Hq, Hkv, Tq, Tk, int(max_q), int(max_k), d,
                                float(scale), int(causal), dtype, stream_ptr(stream))


def fa_fwd_padded(q, k, v, o, lse, q_start, q_end, k_start, k_end, causal=CAUSAL_NONE,
                  scale=None, stream=None):
    """Call fa_fwd_padded on torch CUDA tensors (Q/O [B, Hq, Nq, d], K/V
    [B, Hkv, Nk, d], LSE [B, Hq, Nq] or None, row ranges int32 [B] on the
    device).  Returns the status."""
    import math
    import torch
    B, Hq, Nq, d = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    return load().fa_fwd_padded(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(q_start),
                                ptr(q_end), ptr(k_start), ptr(k_end), B, Hq, Hkv, Nq, Nk, d,
                                float(scale), int(causal), dtype, stream_ptr(stream))


def fa_bwd_padded(q, k, v, o, do, lse, q_start, q_end, k_start, k_end, dq, dk, dv, causal=False,
                  scale=None, stream=None):
    """Call fa_bwd_padded on torch CUDA tensors ([B, H, N, d]; lse [B, Hq, N]
    fp32; row ranges int32 [B]); allocates the workspace.  Returns the status."""
    import math
    import torch
    B, Hq, N, d = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    lib = load()
    nbytes = lib.fa_bwd_workspace_bytes(B, Hq, N)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    return lib.fa_bwd_padded(ptr(q), ptr(k), ptr(v), ptr(o), ptr(do), ptr(lse), ptr(q_start),
                             ptr(q_end), ptr(k_start), ptr(k_end), ptr(dq), ptr(dk), ptr(dv), B, Hq,
                             Hkv, N, d, float(scale), int(bool(causal)), dtype, ptr(ws), nbytes,
                             stream_ptr(stream))


def fa_bwd_varlen(q, k, v, o, do, lse, cu, max_seqlen, dq, dk, dv, causal=False, scale=None,
                  stream=None):
    """Call fa_bwd_varlen on packed torch CUDA tensors ([total, H, d]; lse
    [Hq, total] fp32; cu int32 [B + 1]); allocates the workspace.  Returns the
    status."""
    import math
    import torch
    T, Hq, d = q.shape
    Hkv = k.shape[1]
    B = cu.numel() - 1
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    dtype = 1 if q.dtype == torch.bfloat16 else 0
    lib = load()
    nbytes = lib.fa_bwd_workspace_bytes(B, Hq, int(max_seqlen))
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    return lib.fa_bwd_varlen(ptr(q), ptr(k), ptr(v), ptr(o), ptr(do), ptr(lse), ptr(cu), ptr(dq),
                             ptr(dk), ptr(dv), B, Hq, Hkv, T, int(max_seqlen), d, float(scale),
                             int(bool(causal)), dtype, ptr(ws), nbytes, stream_ptr(stream))


def paged_cache(k_cache, v_cache, block_table, k_scale=None, v_scale=None):
    """fa_paged_cache of torch tensors: pages [num_pages, Hkv, page, d] (any
    strides), block_table int32 [B, max_pages], scales [num_pages, Hkv, page]."""
    import torch
    kinds = {torch.float16: 0, torch.bfloat16: 1, torch.int8: 2, torch.float8_e4m3fn: 3}
    c = PagedCache()
    c.k, c.v = k_cache.data_ptr(), v_cache.data_ptr()
    c.page_stride, c.head_stride, c.row_stride = k_cache.stride()[:3]
    if k_scale is not None:
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.scale_page_stride, c.scale_head_stride, c.scale_row_stride = k_scale.stride()
    c.block_table, c.table_stride = block_table.data_ptr(), block_table.stride(0)
    c.max_pages = block_table.size(1)
    c.num_pages, c.kv_heads, c.page_size, c.head_dim = k_cache.shape
    c.dtype = kinds[k_cache.dtype]
    return c


def fa_kvcache_write(cache, k, v, cu_seqlens, seqlens_k, stream=None):
    """Call fa_kvcache_write on torch CUDA tensors (k, v [total, Hkv, d]).  Returns the status."""
    import torch
    return load().fa_kvcache_write(ctypes.byref(cache), ptr(k), ptr(v), k.stride(0), k.stride(1),
                                   v.stride(0), v.stride(1), ptr(cu_seqlens), ptr(seqlens_k),
                                   seqlens_k.numel(), k.shape[0],
                                   1 if k.dtype == torch.bfloat16 else 0, stream_ptr(stream))


def fa_kvcache_read(cache, k, v, cu_seqlens, seqlens_k, stream=None):
    """Call fa_kvcache_read into torch CUDA tensors (k, v [total, Hkv, d]).  Returns the status."""
    import torch
    return load().fa_kvcache_read(ctypes.byref(cache), ptr(k), ptr(v), ptr(cu_seqlens),
                                  ptr(seqlens_k), seqlens_k.numel(), k.shape[0],
                                  1 if k.dtype == torch.bfloat16 else 0, stream_ptr(stream))


def fa_fwd_paged(cache, q, o, lse, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k,
                 causal=CAUSAL_NONE, scale=None, stream=None):
    """Call fa_fwd_paged on torch CUDA tensors (q, o [total_q, Hq, d], lse
    [Hq, total_q] or None); allocates the workspace.  Returns the status."""
    import math
    import torch
    T, Hq, d = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    lib = load()
    B = seqlens_k.numel()
    nbytes = lib.fa_fwd_paged_workspace_bytes(ctypes.byref(cache), B, Hq, T, int(max_seqlen_q),
                                              int(max_seqlen_k))
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    return lib.fa_fwd_paged(ctypes.byref(cache), ptr(q), q.stride(0), q.stride(1), ptr(o), ptr(lse),
                            ptr(cu_seqlens_q), ptr(seqlens_k), B, Hq, T, int(max_seqlen_q),
                            int(max_seqlen_k), float(scale), int(causal),
                            1 if q.dtype == torch.bfloat16 else 0, ptr(ws), nbytes,
                            stream_ptr(stream))
