"""Thin ctypes binding of libbitsknn.so (the C ABI declared in include/bitsknn.h).

Used by the parity tests and the benchmark to call the HIP kernels on torch-allocated device
memory.  torch is plumbing here (device buffers, the current stream); every computation goes
through the C ABI.  There is no CPU fallback: a missing library raises ImportError-like
RuntimeError on first use, and every non-zero status raises BitsKnnError with the library's
message.
"""
import ctypes
import os
from typing import NamedTuple

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "libbitsknn.so")

OK, ERR_UNSUPPORTED, ERR_INVALID, ERR_HIP, ERR_INTERNAL = 0, 1, 2, 3, 4
DIST_L2, DIST_PARTIAL_L2, DIST_EXPANDED, DIST_PARTIAL_L2_BF16X3 = 0, 1, 2, 3

# every symbol include/bitsknn.h declares
EXPORTS = (
    "bitsknn_last_error",
    "bitsknn_version",
    "bitsknn_topk_bits_f32",
    "bitsknn_topk_bits_parts_f32",
    "bitsknn_topk_partial_bitonic_f32",
    "bitsknn_label_offsets",
    "bitsknn_fill_f32",
    "bitsknn_stream_read_f32",
    "bitsknn_dist_f32",
    "bitsknn_dist_layout_workspace_bytes",
    "bitsknn_dist_layout_f32",
    "bitsknn_fused_l2_topk_f32",
    "bitsknn_fused_workspace_bytes",
    "bitsknn_fused_image_bytes",
    "bitsknn_fused_l2_topk_f32_ws",
    "bitsknn_fused_l2_topk_f32_ex",
    "bitsknn_fused_l2_topk_f32_tuned",
    "bitsknn_fused_static_scratch_bytes",
    "bitsknn_fused_l2_topk_f32_static",
    "bitsknn_fused_status",
    "bitsknn_cross_attention_workspace_bytes",
    "bitsknn_cross_attention",
    "bitsknn_cross_attention_backward_workspace_bytes",
    "bitsknn_cross_attention_backward",
    "bitsknn_cache_store",
    "bitsknn_cached_attention_workspace_bytes",
    "bitsknn_cached_attention",
)


class FusedTuning(ctypes.Structure):
    """bitsknn_fused_tuning of include/bitsknn.h"""
    _fields_ = [("ranges", ctypes.c_int32), ("first_radius", ctypes.c_int32), ("image", ctypes.c_int32),
                ("workgroup", ctypes.c_int32), ("reserved", ctypes.c_int32 * 4)]


class Rows(ctypes.Structure):
    """bitsknn_rows of include/bitsknn.h"""
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("row_stride", ctypes.c_int64)]


class AttentionShape(ctypes.Structure):
    """bitsknn_attention_shape of include/bitsknn.h"""
    _fields_ = [("type", ctypes.c_int32), ("dim", ctypes.c_int32), ("batch", ctypes.c_int32),
                ("query_heads", ctypes.c_int32), ("state_heads", ctypes.c_int32), ("queries", ctypes.c_int32),
                ("states", ctypes.c_int32), ("scale", ctypes.c_float)]


class Cache(ctypes.Structure):
    """bitsknn_state_cache of include/bitsknn.h"""
    _fields_ = [("key_codes", ctypes.c_void_p), ("value_codes", ctypes.c_void_p), ("key_scales", ctypes.c_void_p),
                ("value_scales", ctypes.c_void_p), ("block_counts", ctypes.c_void_p), ("blocks", ctypes.c_int32),
                ("state_heads", ctypes.c_int32), ("block", ctypes.c_int32), ("dim", ctypes.c_int32)]


class BitsKnnError(RuntimeError):
    def __init__(self, code, message):
        super().__init__(message)
        self.code = code


_lib = None


def lib():
    """Load libbitsknn.so (built in-tree by `make -C bits-knn-jpdc2024_amd lib`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C {os.path.dirname(_HERE)} lib` "
                "(there is no fallback path)")
        # torch bundles its own HIP runtime under the same soname as the system one; it has to be
        # loaded first so that this library binds to the runtime that owns torch's device memory
        # and streams instead of bringing up a second runtime in the process
        import torch  # noqa: F401
        L = ctypes.CDLL(LIB_PATH)
        vp, sz, i32, u32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_uint32
        L.bitsknn_last_error.restype = ctypes.c_char_p
        L.bitsknn_last_error.argtypes = []
        L.bitsknn_version.restype = ctypes.c_char_p
        L.bitsknn_version.argtypes = []
        L.bitsknn_topk_bits_f32.restype = ctypes.c_int
        L.bitsknn_topk_bits_f32.argtypes = [vp, sz, vp, sz, vp, sz, sz, vp, vp, sz, u32, u32, u32,
                                            ctypes.c_int, vp]
        L.bitsknn_topk_bits_parts_f32.restype = ctypes.c_int
        L.bitsknn_topk_bits_parts_f32.argtypes = [vp, sz, sz, u32, vp, vp, vp, vp, vp, sz, u32, u32, u32, vp]
        L.bitsknn_topk_partial_bitonic_f32.restype = ctypes.c_int
        L.bitsknn_topk_partial_bitonic_f32.argtypes = [vp, sz, sz, sz, vp, vp, sz, u32, u32, vp]
        L.bitsknn_label_offsets.restype = ctypes.c_int
        L.bitsknn_label_offsets.argtypes = [vp, sz, sz, sz, vp]
        L.bitsknn_fill_f32.restype = ctypes.c_int
        L.bitsknn_fill_f32.argtypes = [vp, sz, ctypes.c_float, vp]
        L.bitsknn_stream_read_f32.restype = ctypes.c_int
        L.bitsknn_stream_read_f32.argtypes = [vp, sz, sz, sz, vp, vp]
        L.bitsknn_dist_f32.restype = ctypes.c_int
        L.bitsknn_dist_f32.argtypes = [ctypes.c_int, ctypes.c_int, sz, sz, vp, sz, vp, sz, vp, sz, vp]
        L.bitsknn_dist_layout_workspace_bytes.restype = ctypes.c_size_t
        L.bitsknn_dist_layout_workspace_bytes.argtypes = [ctypes.c_int, sz, sz, ctypes.c_int, ctypes.c_int]
        L.bitsknn_dist_layout_f32.restype = ctypes.c_int
        L.bitsknn_dist_layout_f32.argtypes = [ctypes.c_int, ctypes.c_int, sz, sz, vp, ctypes.c_int, sz, vp,
                                              ctypes.c_int, sz, vp, sz, vp, sz, vp]
        L.bitsknn_fused_l2_topk_f32.restype = ctypes.c_int
        L.bitsknn_fused_l2_topk_f32.argtypes = [vp, vp, ctypes.c_int, i32, i32, vp, vp, ctypes.c_int,
                                                ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                                ctypes.c_int, ctypes.c_int, vp]
        L.bitsknn_fused_l2_topk_f32_ex.restype = ctypes.c_int
        L.bitsknn_fused_l2_topk_f32_ex.argtypes = [vp, vp, ctypes.c_int, i32, i32, vp, vp, ctypes.c_int,
                                                   ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                                   ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, sz, vp]
        L.bitsknn_fused_workspace_bytes.restype = ctypes.c_size_t
        L.bitsknn_fused_workspace_bytes.argtypes = [i32, i32, ctypes.c_int]
        L.bitsknn_fused_image_bytes.restype = ctypes.c_size_t
        L.bitsknn_fused_image_bytes.argtypes = [ctypes.c_int, i32]
        L.bitsknn_fused_l2_topk_f32_ws.restype = ctypes.c_int
        L.bitsknn_fused_l2_topk_f32_ws.argtypes = [vp, vp, ctypes.c_int, i32, i32, vp, vp, ctypes.c_int,
                                                   ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                                   ctypes.c_int, ctypes.c_int, vp, sz, vp]
        L.bitsknn_fused_static_scratch_bytes.restype = ctypes.c_size_t
        L.bitsknn_fused_static_scratch_bytes.argtypes = []
        L.bitsknn_fused_l2_topk_f32_static.restype = ctypes.c_int
        L.bitsknn_fused_l2_topk_f32_static.argtypes = L.bitsknn_fused_l2_topk_f32.argtypes
        L.bitsknn_fused_l2_topk_f32_tuned.restype = ctypes.c_int
        L.bitsknn_fused_l2_topk_f32_tuned.argtypes = [vp, vp, ctypes.c_int, i32, i32, vp, vp, ctypes.c_int,
                                                      ctypes.c_int, ctypes.POINTER(FusedTuning), vp, sz, vp]
        L.bitsknn_fused_status.restype = ctypes.c_int
        L.bitsknn_fused_status.argtypes = [vp]
        rows, shape = ctypes.POINTER(Rows), ctypes.POINTER(AttentionShape)
        L.bitsknn_cross_attention_workspace_bytes.restype = ctypes.c_size_t
        L.bitsknn_cross_attention_workspace_bytes.argtypes = [shape]
        L.bitsknn_cross_attention.restype = ctypes.c_int
        L.bitsknn_cross_attention.argtypes = [shape, rows, rows, rows, vp, vp, sz, rows, vp, vp, sz, vp]
        L.bitsknn_cross_attention_backward_workspace_bytes.restype = ctypes.c_size_t
        L.bitsknn_cross_attention_backward_workspace_bytes.argtypes = [shape]
        L.bitsknn_cross_attention_backward.restype = ctypes.c_int
        L.bitsknn_cross_attention_backward.argtypes = [shape] + [rows] * 5 + [vp, vp, vp, sz] + [rows] * 3 + [vp, sz, vp]
        cache = ctypes.POINTER(Cache)
        L.bitsknn_cache_store.restype = ctypes.c_int
        L.bitsknn_cache_store.argtypes = [cache, i32, i32, i32, rows, rows, vp, vp, sz, vp]
        L.bitsknn_cached_attention_workspace_bytes.restype = ctypes.c_size_t
        L.bitsknn_cached_attention_workspace_bytes.argtypes = [shape]
        L.bitsknn_cached_attention.restype = ctypes.c_int
        L.bitsknn_cached_attention.argtypes = [shape, rows, cache, vp, sz, vp, rows, vp, vp, sz, vp]
        _lib = L
    return _lib


def _check(status):
    if status != OK:
        raise BitsKnnError(status, lib().bitsknn_last_error().decode())


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _row_stride(t):
    # torch reports arbitrary strides for dimensions of extent 1
    rows, cols = t.shape
    return max(t.stride(0), cols) if rows > 1 else cols


def version():
    return lib().bitsknn_version().decode()


def topk_bits(dist, k, block_size=256, items_per_thread=16, prefetch=False, in_label=None,
              label_offsets=None, out_dist=None, out_label=None):
    """bits top-k of every row of a 2-D float32 device tensor (last dim contiguous).
    Returns (values, labels), each rows x k."""
    import torch
    assert dist.is_cuda and dist.dtype == torch.float32 and dist.dim() == 2
    assert dist.shape[1] == 1 or dist.stride(1) == 1
    rows, cols = dist.shape
    if out_dist is None:
        out_dist = torch.empty((rows, k), dtype=torch.float32, device=dist.device)
    if out_label is None:
        out_label = torch.empty((rows, k), dtype=torch.int32, device=dist.device)
    label_stride = 0
    if in_label is not None:
        assert in_label.dtype == torch.int32 and in_label.shape == dist.shape and (cols == 1 or in_label.stride(1) == 1)
        label_stride = _row_stride(in_label)
    if label_offsets is not None:
        assert label_offsets.dtype == torch.int32 and label_offsets.numel() == rows
    _check(lib().bitsknn_topk_bits_f32(_ptr(dist), _row_stride(dist),
                                       _ptr(in_label), label_stride, _ptr(label_offsets), rows, cols,
                                       _ptr(out_dist), _ptr(out_label), _row_stride(out_dist), k,
                                       block_size, items_per_thread, 1 if prefetch else 0, _stream()))
    return out_dist, out_label


def topk_bits_parts(dist, k, parts, block_size=256, items_per_thread=16, scratch=None, out_dist=None,
                    out_label=None):
    """bits-sq: bits top-k of every row of a contiguous 2-D float32 device tensor with the rows cut
    into `parts` parts (bitsknn_topk_bits_parts_f32).  scratch: a dict that keeps the device memory
    for the parts' results and the counters between calls.  Returns (values, labels), rows x k."""
    import torch
    assert dist.is_cuda and dist.dtype == torch.float32 and dist.dim() == 2 and dist.is_contiguous()
    rows, cols = dist.shape
    if out_dist is None:
        out_dist = torch.empty((rows, k), dtype=torch.float32, device=dist.device)
    if out_label is None:
        out_label = torch.empty((rows, k), dtype=torch.int32, device=dist.device)
    key = (rows, parts, k, str(dist.device))
    scratch = scratch if scratch is not None else {}
    if key not in scratch:
        scratch[key] = (torch.empty(rows * parts * k, dtype=torch.float32, device=dist.device),
                        torch.empty(rows * parts * k, dtype=torch.int32, device=dist.device),
                        torch.zeros(rows, dtype=torch.int32, device=dist.device))
    part_d, part_l, counters = scratch[key]
    _check(lib().bitsknn_topk_bits_parts_f32(_ptr(dist), rows, cols, parts, _ptr(part_d), _ptr(part_l),
                                             _ptr(counters), _ptr(out_dist), _ptr(out_label),
                                             _row_stride(out_dist), k, block_size, items_per_thread, _stream()))
    return out_dist, out_label


def topk_partial_bitonic(dist, k, block_size=256, out_dist=None, out_label=None):
    """partial-bitonic-regs top-k (no filtering) of every row of a 2-D float32 device tensor."""
    import torch
    assert dist.is_cuda and dist.dtype == torch.float32 and dist.dim() == 2
    assert dist.shape[1] == 1 or dist.stride(1) == 1
    rows, cols = dist.shape
    if out_dist is None:
        out_dist = torch.empty((rows, k), dtype=torch.float32, device=dist.device)
    if out_label is None:
        out_label = torch.empty((rows, k), dtype=torch.int32, device=dist.device)
    _check(lib().bitsknn_topk_partial_bitonic_f32(_ptr(dist), _row_stride(dist), rows, cols,
                                                  _ptr(out_dist), _ptr(out_label),
                                                  _row_stride(out_dist), k, block_size, _stream()))
    return out_dist, out_label


def label_offsets(rows, parts, cols_per_part, device="cuda"):
    import torch
    out = torch.empty(rows * parts, dtype=torch.int32, device=device)
    _check(lib().bitsknn_label_offsets(_ptr(out), rows, parts, cols_per_part, _stream()))
    return out


def fill(t, value):
    _check(lib().bitsknn_fill_f32(_ptr(t), t.numel(), float(value), _stream()))
    return t


def stream_read(matrix, out=None):
    """Row minima by a plain streaming read (calibration of the achievable read rate)."""
    import torch
    rows, cols = matrix.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=matrix.device)
    _check(lib().bitsknn_stream_read_f32(_ptr(matrix), _row_stride(matrix), rows, cols, _ptr(out), _stream()))
    return out


def distances(queries_dm, points_dm, op=DIST_L2, out=None):
    """Distance matrix q x n from dim-major inputs (d x q and d x n float32 device tensors)."""
    import torch
    d, q = queries_dm.shape
    d2, n = points_dm.shape
    assert d == d2 and (q == 1 or queries_dm.stride(1) == 1) and (n == 1 or points_dm.stride(1) == 1)
    if out is None:
        out = torch.empty((q, n), dtype=torch.float32, device=queries_dm.device)
    _check(lib().bitsknn_dist_f32(op, d, q, n, _ptr(queries_dm), _row_stride(queries_dm),
                                  _ptr(points_dm), _row_stride(points_dm), _ptr(out),
                                  _row_stride(out), _stream()))
    return out


LAYOUT_ROW_MAJOR, LAYOUT_COLUMN_MAJOR = 0, 1


def distances_layout(queries, queries_layout, points, points_layout, op=DIST_L2, out=None):
    """Distance matrix q x n from 2-D float32 device tensors in the caller's layout: LAYOUT_ROW_MAJOR
    (count x dim, the vectors one after the other) or LAYOUT_COLUMN_MAJOR (dim x count)."""
    import torch
    q, d = queries.shape if queries_layout == LAYOUT_ROW_MAJOR else queries.shape[::-1]
    n, d2 = points.shape if points_layout == LAYOUT_ROW_MAJOR else points.shape[::-1]
    assert d == d2
    if out is None:
        out = torch.empty((q, n), dtype=torch.float32, device=queries.device)
    need = int(lib().bitsknn_dist_layout_workspace_bytes(d, q, n, queries_layout, points_layout))
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=queries.device)
    _check(lib().bitsknn_dist_layout_f32(op, d, q, n, _ptr(queries), queries_layout, _row_stride(queries),
                                         _ptr(points), points_layout, _row_stride(points), _ptr(out),
                                         _row_stride(out), _ptr(workspace), need, _stream()))
    return out


FUSED_FP32, FUSED_BF16X3, FUSED_EXACT = 0, 1, 2


def fused_l2_topk(queries_dm, points_dm, k, params=(8, 4, 2), block_query_dim=1, dim_mult=1,
                  out_dist=None, out_label=None, workspace=None, arithmetic=None, tuning=None):
    """bits-fused: top-k of ||p||^2 - 2 q.p without materialising the distance matrix.
    workspace: None -> the plain entry point; "auto" -> allocate what
    bitsknn_fused_workspace_bytes asks for; "image" -> that plus room for the stage image
    (fused_workspace_with_image_bytes); "static" -> the entry point that uses the library's own
    scratch memory and allocates nothing; or a uint8 device tensor.
    arithmetic: None -> the plain entry points (FUSED_EXACT); FUSED_FP32 / FUSED_BF16X3 /
    FUSED_EXACT -> bitsknn_fused_l2_topk_f32_ex with that arithmetic.
    tuning: None, or (ranges, first_radius[, image[, workgroup]]) -> bitsknn_fused_l2_topk_f32_tuned."""
    import torch
    d, q = queries_dm.shape
    d2, n = points_dm.shape
    assert d == d2 and queries_dm.is_contiguous() and points_dm.is_contiguous()
    if out_dist is None:
        out_dist = torch.empty((q, k), dtype=torch.float32, device=queries_dm.device)
    if out_label is None:
        out_label = torch.empty((q, k), dtype=torch.int32, device=queries_dm.device)
    if isinstance(workspace, str) and workspace == "auto":
        workspace = torch.empty(max(1, fused_workspace_bytes(q, n, k)), dtype=torch.uint8,
                                device=queries_dm.device)
    if isinstance(workspace, str) and workspace == "image":
        workspace = torch.empty(max(1, fused_workspace_with_image_bytes(d, q, n, k)), dtype=torch.uint8,
                                device=queries_dm.device)
    head = (_ptr(queries_dm), _ptr(points_dm), d, q, n, _ptr(out_dist), _ptr(out_label), k,
            params[0], params[1], params[2], block_query_dim, dim_mult)
    if tuning is not None:
        assert not isinstance(workspace, str)
        knobs = FusedTuning(int(tuning[0]), int(tuning[1]), int(tuning[2]) if len(tuning) > 2 else 0,
                            int(tuning[3]) if len(tuning) > 3 else 0, (ctypes.c_int32 * 4)())
        _check(lib().bitsknn_fused_l2_topk_f32_tuned(*head[:8], FUSED_EXACT if arithmetic is None else int(arithmetic),
                                                     ctypes.byref(knobs), _ptr(workspace),
                                                     workspace.numel() if workspace is not None else 0, _stream()))
    elif isinstance(workspace, str) and workspace == "static":
        assert arithmetic is None
        _check(lib().bitsknn_fused_l2_topk_f32_static(*head, _stream()))
    elif arithmetic is not None:
        _check(lib().bitsknn_fused_l2_topk_f32_ex(*head, int(arithmetic), _ptr(workspace),
                                                  workspace.numel() if workspace is not None else 0,
                                                  _stream()))
    elif workspace is None:
        _check(lib().bitsknn_fused_l2_topk_f32(*head, _stream()))
    else:
        _check(lib().bitsknn_fused_l2_topk_f32_ws(*head, _ptr(workspace), workspace.numel(), _stream()))
    return out_dist, out_label


def fused_workspace_bytes(q, n, k):
    return int(lib().bitsknn_fused_workspace_bytes(q, n, k))


def fused_image_bytes(dim, n):
    return int(lib().bitsknn_fused_image_bytes(dim, n))


def fused_workspace_with_image_bytes(dim, q, n, k):
    """Partial lists, rounded up to a multiple of 256 bytes, then the stage image."""
    return (fused_workspace_bytes(q, n, k) + 255) // 256 * 256 + fused_image_bytes(dim, n)


def fused_static_scratch_bytes():
    return int(lib().bitsknn_fused_static_scratch_bytes())


def fused_status():
    """Synchronises the current stream and raises BitsKnnError(ERR_INTERNAL) if a fused kernel has
    reported a wait that ran out of polls since the last check."""
    _check(lib().bitsknn_fused_status(_stream()))


BF16, FP16, F32 = 0, 1, 2


def _attention_type(dtype):
    import torch
    assert dtype in (torch.bfloat16, torch.float16), dtype
    return BF16 if dtype == torch.bfloat16 else FP16


def _rows(t):
    """batch x heads x rows x dim, the last dimension contiguous"""
    strides = t.stride()
    assert t.shape[3] <= 1 or strides[3] == 1, "the values of a vector must be contiguous"
    return Rows(t.data_ptr(), strides[0], strides[1], strides[2])


def _attention_shape(queries, state_heads, states, scale):
    batch, heads, rows, dim = queries.shape
    assert states < 2 ** 31 and max(queries.shape) < 2 ** 31  # ctypes would cut them silently
    return AttentionShape(_attention_type(queries.dtype), dim, batch, heads, state_heads, rows, states,
                          dim ** -0.5 if scale is None else scale)


def _int32(t, shape, device):
    import torch
    if t is not None:
        assert t.dtype == torch.int32 and tuple(t.shape) == shape and t.device == device and t.is_contiguous()
    return _ptr(t)


def _mask_args(mask, batch, states, device):
    import torch
    if mask is None:
        return None, 0
    assert mask.dtype in (torch.bool, torch.uint8) and tuple(mask.shape) == (batch, states) and mask.device == device
    assert states <= 1 or mask.stride(1) == 1
    return _ptr(mask), mask.stride(0) if batch > 1 else 0


def _outputs(queries, out, lse):
    import torch
    if out is None:
        out = torch.empty_like(queries)
    if lse is None:
        lse = torch.empty(queries.shape[:3], dtype=torch.float32, device=queries.device)
    assert out.shape == queries.shape and out.dtype == queries.dtype and out.device == queries.device
    assert lse.shape == queries.shape[:3] and lse.dtype == torch.float32 and lse.is_contiguous()
    assert lse.device == queries.device
    return out, lse


def _workspace(workspace, need, device):
    """The caller's bytes, or as many as the call wants."""
    import torch
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    if workspace is None:
        return None, 0
    assert workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == device
    return workspace, workspace.numel()


def _call(entry, device, *args):
    """A call of the library on the tensors' own device, on that device's current stream."""
    import torch
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    if torch.cuda.current_device() == device.index:
        _check(entry(*args, stream))
    else:
        with torch.cuda.device(device):
            _check(entry(*args, stream))


def cross_attention(queries, keys, values, counts=None, mask=None, scale=None, out=None, lse=None, workspace=None):
    """Attention of queries (batch x query heads x rows x dim) over keys and values (batch x state heads
    x states x dim), bfloat16 or float16 device tensors with contiguous vectors (bitsknn_cross_attention).
    counts: None or batch int32, the states of each sequence; mask: None or batch x states bool / uint8,
    the states that take part; scale: None -> dim ** -0.5.  workspace: None -> allocated here; or a uint8
    device tensor (cross_attention_workspace_bytes; a smaller one is used as far as it goes).
    torch's autograd does not see the call: gradients are those that cross_attention_backward returns.
    Returns (out, lse): out like queries, lse batch x query heads x rows float32."""
    batch, state_heads, states, dim = keys.shape
    device = queries.device
    assert queries.is_cuda and keys.device == device and values.device == device
    assert keys.shape == values.shape and queries.shape[0] == batch and queries.shape[3] == dim
    assert keys.dtype == queries.dtype and values.dtype == queries.dtype
    out, lse = _outputs(queries, out, lse)
    shape = _attention_shape(queries, state_heads, states, scale)
    need = int(lib().bitsknn_cross_attention_workspace_bytes(shape)) if workspace is None else 0
    workspace, size = _workspace(workspace, need, device)
    _call(lib().bitsknn_cross_attention, device, shape, _rows(queries), _rows(keys), _rows(values),
          _int32(counts, (batch,), device), *_mask_args(mask, batch, states, device), _rows(out), _ptr(lse),
          _ptr(workspace), size)
    return out, lse


def cross_attention_workspace_bytes(queries, keys):
    """What cross_attention wants as a workspace for tensors of these shapes."""
    return int(lib().bitsknn_cross_attention_workspace_bytes(
        _attention_shape(queries, keys.shape[1], keys.shape[2], 1.0)))


def cross_attention_backward(grad_out, queries, keys, values, out, lse, counts=None, mask=None, scale=None,
                             grad_queries=None, grad_keys=None, grad_values=None, workspace=None):
    """Gradients of cross_attention's out with respect to queries, keys and values, given the gradient of
    out and what the forward call read and returned (bitsknn_cross_attention_backward); scale as there.
    workspace: None -> allocated here; or a uint8 device tensor
    (cross_attention_backward_workspace_bytes).  Returns (grad_queries, grad_keys, grad_values)."""
    import torch
    batch, state_heads, states, dim = keys.shape
    device = queries.device
    assert queries.is_cuda and keys.shape == values.shape
    assert queries.shape[0] == batch and queries.shape[3] == dim
    assert grad_out.shape == queries.shape and out.shape == queries.shape
    for t in (grad_out, keys, values, out):
        assert t.dtype == queries.dtype and t.device == device
    assert lse.dtype == torch.float32 and lse.shape == queries.shape[:3] and lse.is_contiguous()
    assert lse.device == device
    grads = []
    for given, like in ((grad_queries, queries), (grad_keys, keys), (grad_values, values)):
        given = torch.empty_like(like) if given is None else given
        assert given.shape == like.shape and given.dtype == like.dtype and given.device == device
        grads.append(given)
    shape = _attention_shape(queries, state_heads, states, scale)
    need = int(lib().bitsknn_cross_attention_backward_workspace_bytes(shape)) if workspace is None else 0
    workspace, size = _workspace(workspace, need, device)
    _call(lib().bitsknn_cross_attention_backward, device, shape, _rows(grad_out), _rows(queries), _rows(keys),
          _rows(values), _rows(out), _ptr(lse), _int32(counts, (batch,), device),
          *_mask_args(mask, batch, states, device), *(_rows(t) for t in grads), _ptr(workspace), size)
    return tuple(grads)


def cross_attention_backward_workspace_bytes(queries, keys):
    """What cross_attention_backward wants as a workspace for tensors of these shapes."""
    return int(lib().bitsknn_cross_attention_backward_workspace_bytes(
        _attention_shape(queries, keys.shape[1], keys.shape[2], 1.0)))


class StateCache(NamedTuple):
    """States in 8 bits, in blocks (bitsknn_state_cache): e4m3 codes (uint8 or float8_e4m3fn, blocks x
    state heads x block x dim), float32 scales (blocks x state heads), int32 states per block."""
    key_codes: object
    value_codes: object
    key_scales: object
    value_scales: object
    block_counts: object


def state_cache(blocks, state_heads, block, dim, device="cuda"):
    """An empty cache."""
    import torch
    codes = [torch.zeros((blocks, state_heads, block, dim), dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.ones((blocks, state_heads), dtype=torch.float32, device=device) for _ in range(2)]
    return StateCache(*codes, *scales, torch.zeros(blocks, dtype=torch.int32, device=device))


def _cache_args(cache, device):
    import torch
    blocks, state_heads, block, dim = cache.key_codes.shape
    for codes in (cache.key_codes, cache.value_codes):
        assert codes.dtype in (torch.uint8, torch.float8_e4m3fn) and codes.is_contiguous()
        assert codes.shape == cache.key_codes.shape and codes.device == device
    for scales in (cache.key_scales, cache.value_scales):
        assert scales.dtype == torch.float32 and scales.is_contiguous() and scales.device == device
        assert tuple(scales.shape) == (blocks, state_heads)
    return Cache(cache.key_codes.data_ptr(), cache.value_codes.data_ptr(), cache.key_scales.data_ptr(),
                 cache.value_scales.data_ptr(), _int32(cache.block_counts, (blocks,), device), blocks, state_heads,
                 block, dim)


def _table_args(table, batch, device):
    import torch
    assert table.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == batch and table.device == device
    assert table.shape[1] <= 1 or table.stride(1) == 1
    return _ptr(table), table.stride(0) if batch > 1 else 0


def cache_store(cache, keys, values, table, counts=None):
    """Writes keys and values (batch x state heads x states x dim; bfloat16, float16 or float32) into the
    blocks of the cache that table (batch x at least ceil(states / block) int32) names
    (bitsknn_cache_store).  A block is written from its first state, with a new scale: to append to one,
    store it again from all its states.  counts: None or batch int32.  Returns the cache."""
    import torch
    batch, state_heads, states, dim = keys.shape
    device = keys.device
    block = cache.key_codes.shape[2]
    assert keys.is_cuda and values.shape == keys.shape and values.device == device and values.dtype == keys.dtype
    assert (state_heads, dim) == (cache.key_codes.shape[1], cache.key_codes.shape[3])
    assert table.shape[1] * block >= states, "the table has too few entries for the states"
    kind = F32 if keys.dtype == torch.float32 else _attention_type(keys.dtype)
    _call(lib().bitsknn_cache_store, device, _cache_args(cache, device), kind, batch, states, _rows(keys),
          _rows(values), _int32(counts, (batch,), device), *_table_args(table, batch, device))
    return cache


def cached_attention(queries, cache, table, counts=None, scale=None, out=None, lse=None, workspace=None):
    """cross_attention over the states of a cache (bitsknn_cached_attention): table (batch x entries int32)
    names each sequence's blocks, an entry outside the cache's blocks none; counts: None, or batch int32,
    the places of each sequence that take part.  Returns (out, lse)."""
    batch, _, _, dim = queries.shape
    device = queries.device
    _, state_heads, block, cache_dim = cache.key_codes.shape
    assert queries.is_cuda and cache_dim == dim
    out, lse = _outputs(queries, out, lse)
    shape = _attention_shape(queries, state_heads, table.shape[1] * block, scale)
    need = int(lib().bitsknn_cached_attention_workspace_bytes(shape)) if workspace is None else 0
    workspace, size = _workspace(workspace, need, device)
    _call(lib().bitsknn_cached_attention, device, shape, _rows(queries), _cache_args(cache, device),
          *_table_args(table, batch, device), _int32(counts, (batch,), device), _rows(out), _ptr(lse), _ptr(workspace),
          size)
    return out, lse


def cached_attention_workspace_bytes(queries, cache, entries):
    """What cached_attention wants as a workspace for tables of this many entries per sequence."""
    _, state_heads, block, _ = cache.key_codes.shape
    return int(lib().bitsknn_cached_attention_workspace_bytes(
        _attention_shape(queries, state_heads, entries * block, 1.0)))
