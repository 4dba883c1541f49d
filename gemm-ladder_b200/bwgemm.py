"""Python view of the Blackwell rung's C ABI (include/bwgemm.h) over gemm-ladder_b200/lib/libbwgemm.so.

The product is the native library; this module only binds it with ctypes for Python callers (tests, bench.py) and
passes torch tensors' device pointers and torch's current CUDA stream.  There is no fallback: if the library is
missing or the device is not an sm_100 GPU, calls raise.

    import bwgemm
    C = bwgemm.gemm(A, B)          # A (M x K), B (K x N) fp16 CUDA tensors, row-major; C (M x N) fp16
"""
import ctypes
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
# BWGEMM_LIB picks another build of the library in lib/ (e.g. libbwgemm_next.so from build.py --next), or a path
LIB_PATH = os.path.join(HERE, "lib", os.environ.get("BWGEMM_LIB") or "libbwgemm.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "bwgemm.h")

BW_OK, BW_ERR_SHAPE, BW_ERR_LAUNCH, BW_ERR_TIMEOUT, BW_ERR_ARG, BW_ERR_DEVICE = 0, 1, 2, 3, 4, 5
BW_ERR_SCRATCH = 6
BW_KERNEL_TILE, BW_KERNEL_SWAP, BW_KERNEL_PAIR = 0, 1, 2
BW_TYPE_F16, BW_TYPE_BF16, BW_TYPE_F32 = 0, 1, 2


class Plan(ctypes.Structure):
    _fields_ = [
        ("kernel", ctypes.c_int),
        ("bn", ctypes.c_int),
        ("stages", ctypes.c_int),
        ("tiles_m", ctypes.c_int),
        ("tiles_n", ctypes.c_int),
        ("tiles", ctypes.c_int),
        ("kblocks", ctypes.c_int),
        ("grid", ctypes.c_int),
        ("dp_tiles", ctypes.c_int),
        ("sk_tiles", ctypes.c_int),
        ("splits", ctypes.c_int),
        ("sk_iters", ctypes.c_longlong),
        ("group_rows", ctypes.c_int),
        ("workspace_bytes", ctypes.c_size_t),
        ("counters", ctypes.c_int),
        ("smem_bytes", ctypes.c_int),
        ("tmem_cols", ctypes.c_int),
        ("ksplit", ctypes.c_int),
        ("wm", ctypes.c_int),
        ("dyn", ctypes.c_int),
    ]

    def as_dict(self):
        return {name: getattr(self, name) for name, _ in self._fields_}


class BwError(RuntimeError):
    def __init__(self, status, msg):
        super().__init__(msg)
        self.status = status


_lib = None


def lib():
    """The loaded library (raises if it was not built: python gemm-ladder_b200/build.py)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with python gemm-ladder_b200/build.py")
        L = ctypes.CDLL(LIB_PATH)
        vp, i = ctypes.c_void_p, ctypes.c_int
        L.bw_gemm_f16.argtypes = [vp, vp, vp, i, i, i, vp]
        L.bw_gemm_f16.restype = i
        L.bw_gemm_f16_variant.argtypes = [vp, vp, vp, i, i, i, vp, i]
        L.bw_gemm_f16_variant.restype = i
        L.bw_gemm_f16_tn.argtypes = [vp, vp, vp, i, i, i, vp]
        L.bw_gemm_f16_tn.restype = i
        L.bw_gemm_f16_f32out.argtypes = [vp, vp, vp, i, i, i, vp]
        L.bw_gemm_f16_f32out.restype = i
        L.bw_gemm_f16_swiglu.argtypes = [vp, vp, vp, i, i, i, vp]
        L.bw_gemm_f16_swiglu.restype = i
        L.bw_gemm_variant_count.argtypes = []
        L.bw_gemm_variant_count.restype = i
        L.bw_gemm_variant_name.argtypes = [i]
        L.bw_gemm_variant_name.restype = ctypes.c_char_p
        L.bw_gemm_dirty.argtypes = []
        L.bw_gemm_dirty.restype = i
        L.bw_gemm_plan.argtypes = [i, i, i, i, i, ctypes.POINTER(Plan)]
        L.bw_gemm_plan.restype = i
        L.bw_gemm_device_plan.argtypes = [i, i, i, i, i, ctypes.POINTER(Plan)]
        L.bw_gemm_device_plan.restype = i
        L.bw_gemm_f16_noalloc.argtypes = [vp, vp, vp, i, i, i, vp]
        L.bw_gemm_f16_noalloc.restype = i
        u = ctypes.POINTER(ctypes.c_uint)
        L.bw_gemm_status.argtypes = [ctypes.POINTER(ctypes.c_int), u, u, u]
        L.bw_gemm_status.restype = i
        L.bw_gemm_clear_status.argtypes = []
        L.bw_gemm_clear_status.restype = i
        L.bw_gemm_set_wait_limit_ns.argtypes = [ctypes.c_ulonglong]
        L.bw_gemm_set_wait_limit_ns.restype = ctypes.c_ulonglong
        L.bw_wait_selftest.argtypes = [ctypes.c_ulonglong, vp]
        L.bw_wait_selftest.restype = i
        L.bw_rs_create.argtypes = [i, i, i, i, ctypes.POINTER(vp)]
        L.bw_rs_create.restype = i
        L.bw_rs_region_bytes.argtypes = [vp]
        L.bw_rs_region_bytes.restype = ctypes.c_size_t
        L.bw_rs_handle.argtypes = [vp, ctypes.c_char_p]
        L.bw_rs_handle.restype = i
        L.bw_rs_connect.argtypes = [vp, ctypes.c_char_p]
        L.bw_rs_connect.restype = i
        L.bw_gemm_f16_rs.argtypes = [vp, vp, vp, vp, i, vp]
        L.bw_gemm_f16_rs.restype = i
        L.bw_rs_destroy.argtypes = [vp]
        L.bw_rs_destroy.restype = i
        ll, sz = ctypes.c_longlong, ctypes.c_size_t
        L.bw_quant_rows_i8.argtypes = [vp, i, ll, vp, vp, i, i, vp]
        L.bw_quant_rows_i8.restype = i
        L.bw_gemm_i8_work_bytes.argtypes = [i, i, i, i, i, i, ctypes.POINTER(sz)]
        L.bw_gemm_i8_work_bytes.restype = i
        L.bw_gemm_i8.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp, sz, vp]
        L.bw_gemm_i8.restype = i
        L.bw_gemm_i8_swiglu.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp, sz, vp]
        L.bw_gemm_i8_swiglu.restype = i
        L.bw_linear_i8.argtypes = [vp, i, ll, vp, vp, vp, i, i, i, i, vp, sz, vp]
        L.bw_linear_i8.restype = i
        L.bw_moe_work_bytes.argtypes = [i, i, i, i, i, ctypes.POINTER(sz)]
        L.bw_moe_work_bytes.restype = i
        L.bw_moe_mlp.argtypes = [vp, ll, vp, vp, vp, vp, i, i, i, i, i, i, i, vp, vp, vp, sz, vp]
        L.bw_moe_mlp.restype = i
        L.bw_status_string.argtypes = [i]
        L.bw_status_string.restype = ctypes.c_char_p
        L.bw_last_error_string.argtypes = []
        L.bw_last_error_string.restype = ctypes.c_char_p
        _lib = L
    return _lib


def declared_symbols():
    """The functions include/bwgemm.h declares."""
    with open(HEADER) as f:
        text = f.read()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[\w\s\*]+?\b(bw_\w+)\s*\(", text, flags=re.M)))


def check(status):
    if status != BW_OK:
        L = lib()
        msg = L.bw_status_string(status).decode()
        if status == BW_ERR_LAUNCH:
            msg += ": " + L.bw_last_error_string().decode()
        raise BwError(status, msg)


def variants():
    L = lib()
    return [L.bw_gemm_variant_name(v).decode() for v in range(L.bw_gemm_variant_count())]


def plan(M, N, K, sms=148, variant=0):
    p = Plan()
    check(lib().bw_gemm_plan(M, N, K, sms, variant, ctypes.byref(p)))
    return p.as_dict()


def device_plan(M, N, K, variant=0, noalloc=False):
    """The plan a call takes on the current device (bw_gemm_device_plan): the rule on the device's own pair count, or
    the no-allocation entry's plan (the rule's, or the fallback that fits its fixed array)."""
    p = Plan()
    check(lib().bw_gemm_device_plan(M, N, K, variant, 1 if noalloc else 0, ctypes.byref(p)))
    return p.as_dict()


def gemm_ptr(a_ptr, b_ptr, c_ptr, M, N, K, stream_handle=0, variant=0):
    """C = A B on raw device pointers (the C ABI as it is); returns the status code."""
    return lib().bw_gemm_f16_variant(a_ptr, b_ptr, c_ptr, M, N, K, stream_handle, variant)


def gemm(A, B, C=None, variant=0, stream=None):
    """C = A B for fp16 CUDA tensors: A (M x K) and B (K x N) row-major (contiguous); C (M x N) is made if not given."""
    import torch

    M, K = A.shape
    K2, N = B.shape
    if K2 != K:
        raise ValueError(f"A is {M} x {K} but B is {K2} x {N}")
    for t in (A, B):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("A and B must be contiguous fp16 CUDA tensors")
    if C is None:
        C = torch.empty((M, N), dtype=torch.float16, device=A.device)
    elif C.shape != (M, N) or C.dtype != torch.float16 or not C.is_contiguous():
        raise ValueError("C must be a contiguous fp16 M x N tensor")
    s = stream if stream is not None else torch.cuda.current_stream(A.device)
    with torch.cuda.device(A.device):
        check(gemm_ptr(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, s.cuda_stream, variant))
    return C


def gemm_tn(A, Bt, C=None, stream=None):
    """C (fp16, M x N) = A Bt^T for fp16 CUDA tensors, Bt being N x K row-major (a linear layer's weight layout)."""
    import torch

    M, K = A.shape
    N, K2 = Bt.shape
    if K2 != K:
        raise ValueError(f"A is {M} x {K} but Bt is {N} x {K2}")
    for t in (A, Bt):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("A and Bt must be contiguous fp16 CUDA tensors")
    if C is None:
        C = torch.empty((M, N), dtype=torch.float16, device=A.device)
    elif C.shape != (M, N) or C.dtype != torch.float16 or not C.is_contiguous():
        raise ValueError("C must be a contiguous fp16 M x N tensor")
    s = stream if stream is not None else torch.cuda.current_stream(A.device)
    with torch.cuda.device(A.device):
        check(lib().bw_gemm_f16_tn(A.data_ptr(), Bt.data_ptr(), C.data_ptr(), M, N, K, s.cuda_stream))
    return C


def gemm_f32out(A, B, C=None, stream=None):
    """C (fp32, M x N) = A B for fp16 CUDA tensors: the partial sums of a row-parallel layer."""
    import torch

    M, K = A.shape
    K2, N = B.shape
    if K2 != K:
        raise ValueError(f"A is {M} x {K} but B is {K2} x {N}")
    for t in (A, B):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("A and B must be contiguous fp16 CUDA tensors")
    if C is None:
        C = torch.empty((M, N), dtype=torch.float32, device=A.device)
    elif C.shape != (M, N) or C.dtype != torch.float32 or not C.is_contiguous():
        raise ValueError("C must be a contiguous fp32 M x N tensor")
    s = stream if stream is not None else torch.cuda.current_stream(A.device)
    with torch.cuda.device(A.device):
        check(lib().bw_gemm_f16_f32out(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, s.cuda_stream))
    return C


def gemm_swiglu(A, B, C=None, stream=None):
    """C (M x N/2, fp16) = silu(A B_gate) * (A B_up), B's 256-column groups being 128 gate then 128 up columns."""
    import torch

    M, K = A.shape
    K2, N = B.shape
    if K2 != K:
        raise ValueError(f"A is {M} x {K} but B is {K2} x {N}")
    for t in (A, B):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("A and B must be contiguous fp16 CUDA tensors")
    if C is None:
        C = torch.empty((M, N // 2), dtype=torch.float16, device=A.device)
    elif C.shape != (M, N // 2) or C.dtype != torch.float16 or not C.is_contiguous():
        raise ValueError("C must be a contiguous fp16 M x N/2 tensor")
    s = stream if stream is not None else torch.cuda.current_stream(A.device)
    with torch.cuda.device(A.device):
        check(lib().bw_gemm_f16_swiglu(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, s.cuda_stream))
    return C


# ---------------------------------------------------------------------------------- 8-bit integer products
# These calls are made once per layer of a decode step, so their host side is kept short: plain comparisons, the raw
# stream handle, torch's allocator only for what the call needs.  `stream` (None: the current one) is the stream a call
# runs on; what it returns belongs to that stream.  Inputs are taken as they are on that stream: a caller whose inputs
# are still being written on another orders the two, as for any call with a stream.
torch = None
_type_codes = {}


def _types():
    """torch's types by the C ABI's codes; the first call imports torch for the functions below (this module itself is
    used without it)."""
    if not _type_codes:
        global torch
        import torch

        _type_codes.update({torch.float16: BW_TYPE_F16, torch.bfloat16: BW_TYPE_BF16, torch.float32: BW_TYPE_F32})
    return _type_codes


def _on(device, stream, call, *tensors):
    """call(stream handle) with `device` current and `stream` (None: the device's current stream) the current stream there,
    so that memory made inside belongs to the stream the call runs on; the caller's tensors are marked as used by a
    stream that is not the current one, so that their memory is not handed out again before it is done with them."""
    if stream is None:
        if torch.cuda.current_device() == device.index:
            return call(torch._C._cuda_getCurrentRawStream(device.index))
        with torch.cuda.device(device):
            return call(torch._C._cuda_getCurrentRawStream(device.index))
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    with torch.cuda.stream(stream):
        out = call(stream.cuda_stream)
        if not torch.cuda.is_current_stream_capturing():
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)
    return out


def _rows16(X, what):
    """X as rows of 16-bit values a kernel reads as they are: (rows, cols, elements from row to row, type code)."""
    code = _types().get(X.dtype)
    if code is None or code == BW_TYPE_F32 or not X.is_cuda or X.dim() != 2:
        raise ValueError(f"{what} must be a 2-D fp16 or bf16 CUDA tensor")
    rows, cols = X.shape
    ld, step = X.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    if rows <= 1:
        ld = cols
    if ld < cols or ld % 8 or X.data_ptr() % 16:
        raise ValueError(f"{what}'s rows must start on 16-byte boundaries and not overlap")
    return rows, cols, ld, code


def _i8_weight(B, b_scale, device):
    if B.dtype != torch.int8 or B.dim() != 2 or B.device != device or not B.is_contiguous():
        raise ValueError("B must be a contiguous int8 N x K tensor on A's device")
    if b_scale.dtype != torch.float32 or b_scale.dim() != 1 or b_scale.shape[0] != B.shape[0] or \
            b_scale.device != device or not b_scale.is_contiguous():
        raise ValueError("b_scale must be a contiguous fp32 tensor of B's N scales on A's device")


def _out(C, like, rows, cols, dtype, what="C"):
    """C, checked, or a new one on `like`'s device (and the current stream)."""
    if C is None:
        return like.new_empty((rows, cols), dtype=dtype)
    if C.dim() != 2 or C.shape[0] != rows or C.shape[1] != cols or C.dtype != dtype or C.device != like.device or \
            not C.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of {rows} x {cols} on the inputs' device")
    return C


_work_sizes = {}  # (entry, device, sizes ...) -> bytes of workspace: the plan's, a constant of the device


def _work(query, like, *sizes):
    """The call's own workspace from torch's allocator (so of the stream, or the CUDA graph, that the call is part of):
    (tensor or None, address, bytes)."""
    key = (query, like.device.index, *sizes)
    n = _work_sizes.get(key)
    if n is None:
        size = ctypes.c_size_t()
        check(getattr(lib(), query)(*sizes, ctypes.byref(size)))
        if len(_work_sizes) >= 4096:
            _work_sizes.clear()
        n = _work_sizes[key] = size.value
    if not n:
        return None, None, 0
    t = like.new_empty((n,), dtype=torch.uint8)
    return t, t.data_ptr(), n


def quantize_rows(X, Q=None, scale=None, stream=None):
    """(Q, scale): the rows of a 2-D fp16 or bf16 CUDA tensor (rows may be strided) as int8 and their fp32 scales,
    scale = max|row| / 127, Q = round-half-even(127 X / max|row|); made if not given.  X's columns: a multiple of 16."""
    rows, cols, ld, code = _rows16(X, "X")
    if scale is not None and (scale.dim() != 1 or scale.shape[0] != rows or scale.dtype != torch.float32 or
                              scale.device != X.device or not scale.is_contiguous()):
        raise ValueError("scale must be a contiguous fp32 tensor of X's rows")

    def call(s):
        q = _out(Q, X, rows, cols, torch.int8, "Q")
        sc = X.new_empty((rows,), dtype=torch.float32) if scale is None else scale
        check(lib().bw_quant_rows_i8(X.data_ptr(), code, ld, q.data_ptr(), sc.data_ptr(), rows, cols, s))
        return q, sc

    return _on(X.device, stream, call, X, Q, scale)


def _gemm_i8(A, a_scale, B, b_scale, C, dtype, stream, swiglu):
    types = _types()
    dtype = torch.float16 if dtype is None else dtype
    code = types.get(dtype)
    if code is None or (swiglu and code == BW_TYPE_F32):
        raise ValueError(f"C cannot be {dtype}")
    if A.dtype != torch.int8 or A.dim() != 2 or not A.is_cuda or not A.is_contiguous():
        raise ValueError("A must be a contiguous int8 M x K CUDA tensor")
    M, K = A.shape
    if a_scale.dtype != torch.float32 or a_scale.dim() != 1 or a_scale.shape[0] != M or a_scale.device != A.device or \
            not a_scale.is_contiguous():
        raise ValueError("a_scale must be a contiguous fp32 tensor of A's M scales on A's device")
    _i8_weight(B, b_scale, A.device)
    N, K2 = B.shape
    if K2 != K:
        raise ValueError(f"A is {M} x {K} but B is {N} x {K2}")

    def call(s):
        out = _out(C, A, M, N // 2 if swiglu else N, dtype)
        _t, work, n = _work("bw_gemm_i8_work_bytes", A, M, N, K, code, swiglu, 0)
        f = lib().bw_gemm_i8_swiglu if swiglu else lib().bw_gemm_i8
        check(f(A.data_ptr(), a_scale.data_ptr(), B.data_ptr(), b_scale.data_ptr(), out.data_ptr(), M, N, K, code, work, n,
                s))
        return out

    return _on(A.device, stream, call, A, a_scale, B, b_scale, C)


def gemm_i8(A, a_scale, B, b_scale, C=None, dtype=None, stream=None):
    """C (M x N) = a_scale[m] b_scale[n] sum_k A[m][k] B[n][k] for int8 CUDA tensors A (M x K) and B (N x K), exact integer
    sums, in `dtype` (fp16 by default, bf16 or fp32)."""
    return _gemm_i8(A, a_scale, B, b_scale, C, dtype, stream, 0)


def gemm_i8_swiglu(A, a_scale, B, b_scale, C=None, dtype=None, stream=None):
    """C (M x N/2, fp16 or bf16) = silu(gate) * up of the scaled products, B's rows in groups of 128 gate then 128 up."""
    return _gemm_i8(A, a_scale, B, b_scale, C, dtype, stream, 1)


def linear_i8(X, B, b_scale, C=None, swiglu=False, stream=None):
    """C = X B^T in X's type (fp16 or bf16): X (M x K, rows may be strided) quantised to int8 by row (quantize_rows), B
    (N x K) int8 with a scale per row; swiglu: silu(gate) * up, M x N/2, B's rows in groups of 128 gate then 128 up."""
    M, K, ld, code = _rows16(X, "X")
    _i8_weight(B, b_scale, X.device)
    N, K2 = B.shape
    if K2 != K:
        raise ValueError(f"X is {M} x {K} but B is {N} x {K2}")
    swiglu = 1 if swiglu else 0

    def call(s):
        out = _out(C, X, M, N // 2 if swiglu else N, X.dtype)
        _t, work, n = _work("bw_gemm_i8_work_bytes", X, M, N, K, code, swiglu, 1)
        check(lib().bw_linear_i8(X.data_ptr(), code, ld, B.data_ptr(), b_scale.data_ptr(), out.data_ptr(), M, N, K, swiglu,
                                 work, n, s))
        return out

    return _on(X.device, stream, call, X, B, b_scale, C)


# ---------------------------------------------------------------------------------- mixture of experts
MOE_MAX_TOKENS = 128


def moe_mlp(X, R, W1, W2, top_k, renormalize=True, Y=None, ids=None, weights=None, stream=None):
    """Y (T x D): the mixture-of-experts MLP of up to 128 tokens, fp16 or bf16 throughout.  X (T x D, rows may be
    strided), R (E x D) the router, W1 (E x 2F x D) the experts' gate rows then up rows, W2 (E x D x F); each token takes
    its top_k experts by logit (equal ones: the lower index) with softmax weights over them (renormalize) or over all
    experts.  ids (T x top_k int32) and weights (T x top_k fp32), where given, receive the routing."""
    T, D, ld, code = _rows16(X, "X")
    for t, what, dim in ((R, "R", 2), (W1, "W1", 3), (W2, "W2", 3)):
        if t.dtype != X.dtype or t.device != X.device or t.dim() != dim or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous {dim}-D tensor of X's type on X's device")
    E, F = R.shape[0], W2.shape[2]
    if R.shape[1] != D or tuple(W1.shape) != (E, 2 * F, D) or tuple(W2.shape) != (E, D, F):
        raise ValueError(f"X {tuple(X.shape)}, R {tuple(R.shape)}, W1 {tuple(W1.shape)} and W2 {tuple(W2.shape)} do not "
                         "make a layer (T x D, E x D, E x 2F x D, E x D x F)")
    for t, what, dtype in ((ids, "ids", torch.int32), (weights, "weights", torch.float32)):
        if t is not None and (tuple(t.shape) != (T, top_k) or t.dtype != dtype or t.device != X.device or
                              not t.is_contiguous()):
            raise ValueError(f"{what} must be a contiguous {dtype} T x top_k tensor on X's device")

    def call(s):
        out = _out(Y, X, T, D, X.dtype, "Y")
        _t, work, n = _work("bw_moe_work_bytes", X, T, E, top_k, D, F)
        check(lib().bw_moe_mlp(X.data_ptr(), ld, R.data_ptr(), W1.data_ptr(), W2.data_ptr(), out.data_ptr(), T, E, top_k, D,
                               F, code, 1 if renormalize else 0, ids.data_ptr() if ids is not None else None,
                               weights.data_ptr() if weights is not None else None, work, n, s))
        return out

    return _on(X.device, stream, call, X, R, W1, W2, Y, ids, weights)


def status():
    """The device status word of the current device (after a synchronisation): (code, site, block, segment)."""
    code = ctypes.c_int()
    site, block, seg = ctypes.c_uint(), ctypes.c_uint(), ctypes.c_uint()
    check(lib().bw_gemm_status(ctypes.byref(code), ctypes.byref(site), ctypes.byref(block), ctypes.byref(seg)))
    return code.value, site.value, block.value, seg.value


def clear_status():
    check(lib().bw_gemm_clear_status())


def dirty():
    return lib().bw_gemm_dirty()


def set_wait_limit_ns(ns):
    return lib().bw_gemm_set_wait_limit_ns(ns)


def wait_selftest(limit_ns=0, stream=None):
    """Runs the bounded-wait check (a wait on a barrier that nothing arrives on) and returns the C status: 3
    (BW_ERR_TIMEOUT) is the expected outcome; the status word then holds the selftest site."""
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return lib().bw_wait_selftest(limit_ns, s.cuda_stream)


RS_HANDLE_BYTES = 64


class ReduceScatterGemm:
    """The fused reduce-scatter of a row-parallel layer on this rank (bw_rs_* of bwgemm.h): for fp16 A_r (M x K) and
    B_r (K x N), C_r = this rank's rows [r M/world, (r+1) M/world) of sum_r A_r B_r in fp16, one kernel per rank that
    pushes the partial tiles of the other ranks' rows into their memory and sums its own rows' partials in rank order.

    Every rank of `group` constructs it with the same M and N (its receive region's CUDA IPC handle is exchanged with
    all_gather_object, then every rank opens the others' and a barrier follows), and calls it with the same shapes in
    the same order.  Capturable in a CUDA graph (every rank then replays the same graphs).  After a BW_ERR_TIMEOUT
    (another rank never came), close it and make a new one."""

    def __init__(self, M, N, group=None):
        import torch.distributed as dist

        L = lib()
        self.M, self.N = M, N
        self.world, self.rank = dist.get_world_size(group), dist.get_rank(group)
        self._ctx = ctypes.c_void_p()
        check(L.bw_rs_create(M, N, self.world, self.rank, ctypes.byref(self._ctx)))
        try:
            h = ctypes.create_string_buffer(RS_HANDLE_BYTES)
            check(L.bw_rs_handle(self._ctx, h))
            handles = [None] * self.world
            dist.all_gather_object(handles, h.raw, group=group)
            check(L.bw_rs_connect(self._ctx, b"".join(handles)))
            dist.barrier(group=group)
        except Exception:
            self.close()
            raise

    def region_bytes(self):
        return lib().bw_rs_region_bytes(self._ctx)

    def __call__(self, A, B, C=None, stream=None):
        import torch

        M, K = A.shape
        K2, N = B.shape
        if (M, N) != (self.M, self.N) or K2 != K:
            raise ValueError(f"A {tuple(A.shape)} and B {tuple(B.shape)} do not make the context's {self.M} x {self.N}")
        for t in (A, B):
            if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
                raise ValueError("A and B must be contiguous fp16 CUDA tensors")
        rows = M // self.world
        if C is None:
            C = torch.empty((rows, N), dtype=torch.float16, device=A.device)
        elif C.shape != (rows, N) or C.dtype != torch.float16 or not C.is_contiguous():
            raise ValueError(f"C must be a contiguous fp16 {rows} x {N} tensor")
        s = stream if stream is not None else torch.cuda.current_stream(A.device)
        with torch.cuda.device(A.device):
            check(lib().bw_gemm_f16_rs(self._ctx, A.data_ptr(), B.data_ptr(), C.data_ptr(), K, s.cuda_stream))
        return C

    def close(self):
        if self._ctx:
            lib().bw_rs_destroy(self._ctx)
            self._ctx = ctypes.c_void_p()
