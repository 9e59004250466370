"""gern_amd: Gern's fused kernels on MI355X (gfx950).

This Python module is a thin ctypes view of the package's C ABI
(include/gern_hip.h, include/gern_pipelines.h) for tests, the smoke check and
the benchmark.  The product is the native code: Gern's C++ front end, the HIP
code generator and Runner (libgern.so), the hiprtc/hipModule runtime behind a C
ABI (libgern_hip.so), the hand-written gernels (gernels/*.h) and the composed
pipelines (libgern_pipelines.so).

There is no CPU fallback: every compute entry point raises if the native
libraries or a GPU are missing.
"""
import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))

COMPILE_ONLY = 1
NO_XCD_REMAP = 2
GEMM_OVERWRITE = 4
GEMM_GENERAL_ONLY = 8
BLUR_PLAIN_STORES = 16
QK_ROW_BLOCKS = 32
XCD_TILE_BLOCKS = 64

_libs = None


class GernError(RuntimeError):
    pass


def _load():
    """Loads the native libraries (built in-tree by gern_amd/build.py)."""
    global _libs
    if _libs is not None:
        return _libs
    # PyTorch ships its own HIP runtime under the same sonames.  Loading it
    # first makes the whole process share ONE runtime; two runtimes in one
    # process each open the device and the second one finds no GPU.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    paths = {n: os.path.join(_HERE, "lib%s.so" % n) for n in ("gern_hip", "gern", "gern_pipelines")}
    for n, p in paths.items():
        if not os.path.exists(p):
            raise GernError("%s is missing: run `python gern_amd/build.py` (or __graft_entry__.build())" % p)
    hip = C.CDLL(paths["gern_hip"], mode=C.RTLD_GLOBAL)
    C.CDLL(paths["gern"], mode=C.RTLD_GLOBAL)
    pipes = C.CDLL(paths["gern_pipelines"], mode=C.RTLD_GLOBAL)

    i64, vp, sz = C.c_int64, C.c_void_p, C.c_size_t
    hip.gern_hip_last_error.restype = sz
    hip.gern_hip_last_error.argtypes = [C.c_char_p, sz]
    pipes.gern_pipelines_last_error.restype = sz
    pipes.gern_pipelines_last_error.argtypes = [C.c_char_p, sz]
    pipes.gern_pipeline_source.restype = C.c_char_p
    pipes.gern_pipeline_source.argtypes = [vp]
    pipes.gern_pipeline_kernel_name.restype = C.c_char_p
    pipes.gern_pipeline_kernel_name.argtypes = [vp]
    pipes.gern_pipeline_destroy.argtypes = [vp]
    pipes.gern_pipeline_faults.argtypes = [vp, C.POINTER(i64)]
    pipes.gern_blur_chain_create.argtypes = [C.c_char_p, i64, i64, i64, C.c_int, C.c_int, C.POINTER(vp)]
    pipes.gern_blur_chain_run.argtypes = [vp, vp, i64, i64, i64, vp, i64, vp]
    pipes.gern_softmax_create.argtypes = [i64, i64, C.c_int, C.POINTER(vp)]
    pipes.gern_softmax_run.argtypes = [vp, vp, vp, i64, i64, vp]
    if hasattr(pipes, "gern_gemm_create"):
        pipes.gern_gemm_create.argtypes = [C.c_int, C.c_int, C.POINTER(vp)]
        pipes.gern_gemm_run.argtypes = [vp, vp, vp, vp, i64, i64, i64, vp]
    if hasattr(pipes, "gern_qk_softmax_create"):
        pipes.gern_qk_softmax_create.argtypes = [i64, i64, C.c_int, C.POINTER(vp)]
        pipes.gern_qk_softmax_run.argtypes = [vp, vp, vp, vp, i64, i64, C.c_float, vp]
        pipes.gern_qk_softmax_run_no_alloc.argtypes = [vp, vp, vp, vp, i64, i64, C.c_float, vp]
    pipes.gern_gemm_schedule_create.argtypes = [C.c_int, C.c_int, C.POINTER(vp)]
    pipes.gern_gemm_schedule_run.argtypes = [vp, vp, vp, vp, vp]
    pipes.gern_page_table_create.argtypes = [i64, C.c_int, C.POINTER(vp)]
    pipes.gern_page_table_run.argtypes = [vp, vp, vp, i64, vp, i64, vp, vp, i64, vp, vp, vp, i64, vp, vp]
    pipes.gern_cache_write_create.argtypes = [i64, i64, C.c_int, C.c_int, C.POINTER(vp)]
    pipes.gern_cache_write_run.argtypes = [vp, vp, i64, vp, i64, vp, i64, i64, vp, vp, vp, vp, i64, vp]
    pipes.gern_cache_attention_create.argtypes = [i64, i64, C.c_int, C.c_int, C.POINTER(vp)]
    pipes.gern_cache_attention_workspace.argtypes = [vp, i64, i64, i64, i64, i64, i64, C.POINTER(i64)]
    pipes.gern_cache_attention_run.argtypes = [vp, vp, i64, vp, vp, vp, vp, i64, vp, i64, vp, vp, i64, i64, i64, i64, vp, i64, C.c_float, i64, i64, vp,
                                               i64, vp]
    pipes.gern_matvec4_create.argtypes = [i64, C.c_int, C.c_int, C.POINTER(vp)]
    pipes.gern_matvec4_run.argtypes = [vp, vp, i64, vp, vp, vp, vp, i64, i64, i64, i64, vp]
    cpp = C.POINTER(C.c_char_p)
    hip.gern_hip_compile.argtypes = [C.c_char_p, cpp, C.c_int, cpp, C.c_int, C.c_char_p, C.POINTER(vp)]
    hip.gern_hip_compile_only.argtypes = [C.c_char_p, cpp, C.c_int, cpp, C.c_int, C.c_char_p, C.POINTER(sz)]
    hip.gern_hip_get_kernel.argtypes = [vp, C.c_char_p, C.POINTER(vp)]
    hip.gern_hip_launch.argtypes = [vp, C.POINTER(C.c_uint32), C.POINTER(C.c_uint32), C.c_uint32, C.POINTER(vp), vp]
    hip.gern_hip_event_create.argtypes = [C.POINTER(vp)]
    hip.gern_hip_event_record.argtypes = [vp, vp]
    hip.gern_hip_event_elapsed_ms.argtypes = [vp, vp, C.POINTER(C.c_float)]
    hip.gern_hip_event_destroy.argtypes = [vp]
    hip.gern_hip_stream_sync.argtypes = [vp]
    _libs = (hip, pipes)
    return _libs


def hip_lib():
    return _load()[0]


def pipelines_lib():
    return _load()[1]


def _pipe_error():
    n = pipelines_lib().gern_pipelines_last_error(None, 0)
    buf = C.create_string_buffer(n + 1)
    pipelines_lib().gern_pipelines_last_error(buf, n + 1)
    return buf.value.decode(errors="replace")


def _hip_error():
    n = hip_lib().gern_hip_last_error(None, 0)
    buf = C.create_string_buffer(n + 1)
    hip_lib().gern_hip_last_error(buf, n + 1)
    return buf.value.decode(errors="replace")


def _check(rc):
    if rc != 0:
        raise GernError(_pipe_error())


class Limits(C.Structure):
    _fields_ = [("wavefront_size", C.c_int32), ("max_threads_per_block", C.c_int32),
                ("max_block_dim", C.c_int32 * 3), ("max_grid_dim", C.c_int32 * 3),
                ("lds_bytes_per_block", C.c_int64), ("compute_units", C.c_int32), ("clock_khz", C.c_int32),
                ("hbm_bytes", C.c_int64), ("arch", C.c_char * 64)]


def device_limits():
    lim = Limits()
    if hip_lib().gern_hip_device_limits(C.byref(lim)) != 0:
        raise GernError(_hip_error())
    return lim


def device_count():
    n = C.c_int(0)
    hip_lib().gern_hip_device_count(C.byref(n))
    return n.value


class Event:
    """A HIP event recorded on the stream the kernels are launched on."""

    def __init__(self):
        self.h = C.c_void_p()
        if hip_lib().gern_hip_event_create(C.byref(self.h)) != 0:
            raise GernError(_hip_error())

    def record(self, stream=None):
        if hip_lib().gern_hip_event_record(self.h, stream) != 0:
            raise GernError(_hip_error())

    def elapsed_ms_until(self, stop):
        ms = C.c_float()
        if hip_lib().gern_hip_event_elapsed_ms(self.h, stop.h, C.byref(ms)) != 0:
            raise GernError(_hip_error())
        return ms.value

    def __del__(self):
        try:
            hip_lib().gern_hip_event_destroy(self.h)
        except Exception:
            pass


def _ptr(t):
    """Device pointer of a torch tensor (or a raw integer address)."""
    return C.c_void_p(t if isinstance(t, int) else t.data_ptr())


class _Pipeline:
    def __init__(self):
        self.h = C.c_void_p()

    @property
    def source(self):
        return pipelines_lib().gern_pipeline_source(self.h).decode()

    @property
    def kernel_name(self):
        return pipelines_lib().gern_pipeline_kernel_name(self.h).decode()

    def faults(self):
        """gern_pipeline_faults: waits for the device; what the kernels could only signal in their results
        (QK tile kernel: wavefronts that gave up waiting, rows whose logits did not fit), read and cleared."""
        n = C.c_int64(-1)
        _check(pipelines_lib().gern_pipeline_faults(self.h, C.byref(n)))
        return n.value

    def __del__(self):
        try:
            if self.h:
                pipelines_lib().gern_pipeline_destroy(self.h)
        except Exception:
            pass


class BlurChain(_Pipeline):
    """Fused separable box blur, e.g. BlurChain("xyx")."""

    def __init__(self, pattern, stride=3, tile_rows=4, tile_cols=None, waves_per_block=1, flags=0):
        super().__init__()
        nx = pattern.count("x")
        if tile_cols is None:
            # the widest tile that writes line-aligned windows (include/gern_pipelines.h)
            tile_cols = (256 - 28 - nx * (stride - 1)) // 32 * 32
        self.pattern, self.stride = pattern, stride
        self.nx, self.ny = nx, pattern.count("y")
        _check(pipelines_lib().gern_blur_chain_create(pattern.encode(), stride, tile_rows, tile_cols,
                                                      waves_per_block, flags, C.byref(self.h)))

    def out_shape(self, rows, cols):
        return rows - self.ny * (self.stride - 1), cols - self.nx * (self.stride - 1)

    def __call__(self, img, out, stream=None):
        """img, out: contiguous fp32 CUDA tensors; out has out_shape(*img.shape)."""
        rows, cols = img.shape
        assert tuple(out.shape) == self.out_shape(rows, cols)
        _check(pipelines_lib().gern_blur_chain_run(self.h, _ptr(img), rows, cols, img.stride(0), _ptr(out),
                                                   out.stride(0), stream))
        return out


class Softmax(_Pipeline):
    """Fused row softmax over matrices with `ncol` columns."""

    def __init__(self, ncol, rows_per_wave=1, flags=0):
        super().__init__()
        self.ncol = ncol
        _check(pipelines_lib().gern_softmax_create(ncol, rows_per_wave, flags, C.byref(self.h)))

    def __call__(self, x, out, stream=None):
        rows, cols = x.shape
        assert cols == self.ncol and tuple(out.shape) == (rows, cols) and x.stride(0) == out.stride(0)
        _check(pipelines_lib().gern_softmax_run(self.h, _ptr(x), _ptr(out), rows, x.stride(0), stream))
        return out


class Gemm(_Pipeline):
    """C += A @ B (or C = A @ B with overwrite=True).  variant "f32" or "bf16"
    (fp32 accumulate); general_only=True keeps shapes that the direct-to-LDS
    matrix-core kernels could take on the kernel for every shape."""

    def __init__(self, variant="f32", overwrite=False, general_only=False, flags=0):
        super().__init__()
        self.variant = variant
        if overwrite:
            flags |= GEMM_OVERWRITE
        if general_only:
            flags |= GEMM_GENERAL_ONLY
        _check(pipelines_lib().gern_gemm_create({"f32": 0, "bf16": 1}[variant], flags, C.byref(self.h)))

    def __call__(self, A, B, Cm, stream=None):
        M, K = A.shape
        N = B.shape[1]
        assert tuple(B.shape) == (K, N) and tuple(Cm.shape) == (M, N)
        assert A.is_contiguous() and B.is_contiguous() and Cm.is_contiguous()
        _check(pipelines_lib().gern_gemm_run(self.h, _ptr(A), _ptr(B), _ptr(Cm), M, N, K, stream))
        return Cm


class GemmSchedule(_Pipeline):
    """C += A @ B on 1024 x 1024 fp32 matrices through a schedule written at the level of Gern's API
    (the reference's gernels/mm/kernel_3.cu, kernel_6.cu or kernel_10.cu)."""

    SIZE = 1024

    def __init__(self, schedule, flags=0):
        super().__init__()
        self.schedule = schedule
        _check(pipelines_lib().gern_gemm_schedule_create(schedule, flags, C.byref(self.h)))

    def __call__(self, A, B, Cm, stream=None):
        n = self.SIZE
        assert tuple(A.shape) == (n, n) and tuple(B.shape) == (n, n) and tuple(Cm.shape) == (n, n)
        assert A.is_contiguous() and B.is_contiguous() and Cm.is_contiguous()
        _check(pipelines_lib().gern_gemm_schedule_run(self.h, _ptr(A), _ptr(B), _ptr(Cm), stream))
        return Cm


class QKSoftmax(_Pipeline):
    """S = softmax_rows(scale * Q @ K^T), Q and K in bf16, S in fp32."""

    def __init__(self, head_dim=128, max_keys=4096, flags=0):
        super().__init__()
        self.head_dim = head_dim
        _check(pipelines_lib().gern_qk_softmax_create(head_dim, max_keys, flags, C.byref(self.h)))

    def __call__(self, Q, K, S, scale, stream=None, no_alloc=False):
        """no_alloc=True: gern_qk_softmax_run_no_alloc (exchange memory from the library's device array)."""
        M, D = Q.shape
        N = K.shape[0]
        assert D == self.head_dim and K.shape[1] == D and tuple(S.shape) == (M, N)
        assert Q.is_contiguous() and K.is_contiguous() and S.is_contiguous()
        run = pipelines_lib().gern_qk_softmax_run_no_alloc if no_alloc else pipelines_lib().gern_qk_softmax_run
        _check(run(self.h, _ptr(Q), _ptr(K), _ptr(S), M, N, float(scale), stream))
        return S


_TYPES = {"bf16": 0, "f16": 1}


def _type(dtype):
    if dtype not in _TYPES:
        raise GernError("dtype must be \"bf16\" or \"f16\", not %r" % (dtype,))
    return _TYPES[dtype]


def _expect(ok, what):
    if not ok:
        raise GernError(what)


class _ServingPipeline(_Pipeline):
    """A pipeline of torch tensors: it checks types, layouts and devices before it hands addresses to the C ABI.  The
    checks are written out for what they cost: a decoding step makes several of these calls of a few microseconds.

    A call runs on `stream`, a HIP stream's address (0: the default stream), by default on torch's current stream, in order
    with the torch operations before and after it, also where torch captures a graph."""

    def __init__(self, dtype=None):
        super().__init__()
        import torch
        self._device = torch.cuda.current_device() if torch.cuda.is_available() else None
        self._int32_type, self._uint8, self._float32 = torch.int32, torch.uint8, torch.float32
        self._code_types = (torch.float8_e4m3fn, torch.uint8)
        self._half = {"bf16": torch.bfloat16, "f16": torch.float16, None: None}[dtype]
        # the address of a device's current stream: torch.cuda.current_stream makes an object around it, for a microsecond
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)

    def _on_gpu(self, *tensors):
        """All on the GPU that the pipeline was created on (a kernel runs where its code was loaded)."""
        device = self._device
        for t in tensors:
            if t.get_device() != device:
                raise GernError("every tensor must be on the pipeline's GPU (%s), not on %s" % (device, t.device))

    def _int32(self, **tensors):
        for name, t in tensors.items():
            if t.dtype is not self._int32_type or not t.is_contiguous():
                raise GernError(name + " must be a contiguous int32 tensor")

    def _rows(self, name, t):
        """16-bit floats of the pipeline's type, contiguous but for the stride of their first dimension, which is returned."""
        if t.dtype is not self._half:
            raise GernError("%s must be %s" % (name, self._half))
        strides, shape = t.stride(), t.shape
        inner = 1
        for i in range(len(shape) - 1, 0, -1):
            if strides[i] != inner and shape[i] != 1:
                raise GernError(name + " must be contiguous in all but its first dimension")
            inner *= shape[i]
        return strides[0] if len(shape) > 0 and shape[0] > 1 else inner

    def _cache(self, k_cache, v_cache, k_scales, v_scales):
        """(pages, heads) of a paged cache."""
        shape = k_cache.shape
        if len(shape) != 4 or shape[2] != self.page_size or shape[3] != self.head_dim or v_cache.shape != shape:
            raise GernError("the cache's codes must be [pages, heads, page_size = %d, head_dim = %d]" % (self.page_size, self.head_dim))
        if k_scales.shape != shape[:2] or v_scales.shape != shape[:2]:
            raise GernError("the cache's scales must be [pages, heads]")
        if (k_cache.dtype not in self._code_types or v_cache.dtype not in self._code_types or not k_cache.is_contiguous() or
                not v_cache.is_contiguous()):
            raise GernError("the cache's codes must be contiguous float8_e4m3fn (or uint8)")
        if (k_scales.dtype is not self._float32 or v_scales.dtype is not self._float32 or not k_scales.is_contiguous() or
                not v_scales.is_contiguous()):
            raise GernError("the cache's scales must be contiguous float32")
        return shape[0], shape[1]


class PageTable(_ServingPipeline):
    """Block tables and slot maps of a batch of requests (gern_page_table_run)."""

    def __init__(self, page_size=16, flags=0):
        super().__init__()
        self.page_size, self._run = page_size, pipelines_lib().gern_page_table_run
        _check(pipelines_lib().gern_page_table_create(page_size, flags, C.byref(self.h)))

    def __call__(self, cached, added, free_pages, free_count, table, lengths, starts, slots, counts, stream=None):
        """cached, added [requests], free_pages [any], free_count [1] in; table [requests, width] (new entries only),
        lengths [requests], starts [requests + 1], slots [tokens], counts [2] (pages left, pages missing) out; int32."""
        self._int32(cached=cached, added=added, free_pages=free_pages, free_count=free_count, table=table, lengths=lengths, starts=starts, slots=slots,
                    counts=counts)
        n = cached.shape[0] if cached.dim() == 1 else -1
        _expect(n >= 0 and added.shape == lengths.shape == (n,) and starts.shape == (n + 1,) and table.dim() == 2 and table.shape[0] == n and
                free_pages.dim() == slots.dim() == 1 and free_count.numel() == 1 and counts.numel() == 2,
                "cached, added and lengths must be [requests], starts [requests + 1], table [requests, width], free_pages and slots one-dimensional, "
                "free_count [1] and counts [2]")
        self._on_gpu(cached, added, free_pages, free_count, table, lengths, starts, slots, counts)
        _check(self._run(self.h, cached.data_ptr(), added.data_ptr(), n, free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(),
                         table.data_ptr(), table.shape[1], lengths.data_ptr(), starts.data_ptr(), slots.data_ptr(), slots.shape[0], counts.data_ptr(),
                         self._current_stream(self._device) if stream is None else stream))
        return table, slots


class CacheWrite(_ServingPipeline):
    """New keys and values into a paged cache in 8 bits (gern_cache_write_run)."""

    def __init__(self, head_dim=128, page_size=16, dtype="bf16", flags=0):
        kind = _type(dtype)
        super().__init__(dtype)
        self.head_dim, self.page_size, self.dtype, self._run = head_dim, page_size, dtype, pipelines_lib().gern_cache_write_run
        _check(pipelines_lib().gern_cache_write_create(head_dim, page_size, kind, flags, C.byref(self.h)))

    def __call__(self, k, v, slots, k_cache, v_cache, k_scales, v_scales, stream=None):
        """k, v [tokens, heads, head_dim] (any stride from token to token); slots [tokens] int32, -1 = not stored; the
        cache [pages, heads, page_size, head_dim] float8_e4m3fn with scales [pages, heads] float32 is updated."""
        pages, heads = self._cache(k_cache, v_cache, k_scales, v_scales)
        self._int32(slots=slots)
        ldk, ldv = self._rows("k", k), self._rows("v", v)
        _expect(slots.dim() == 1 and k.shape == v.shape == (slots.shape[0], heads, self.head_dim), "slots must be [tokens], k and v [tokens, heads, head_dim]")
        self._on_gpu(k, v, slots, k_cache, v_cache, k_scales, v_scales)
        _check(self._run(self.h, k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), slots.shape[0], heads, k_cache.data_ptr(), v_cache.data_ptr(),
                         k_scales.data_ptr(), v_scales.data_ptr(), pages, self._current_stream(self._device) if stream is None else stream))


class CacheAttention(_ServingPipeline):
    """Causal attention of ragged batches of queries over a paged cache in 8 bits (gern_cache_attention_run)."""

    def __init__(self, head_dim=128, page_size=16, dtype="bf16", flags=0):
        kind = _type(dtype)
        super().__init__(dtype)
        self.head_dim, self.page_size, self.dtype, self._run = head_dim, page_size, dtype, pipelines_lib().gern_cache_attention_run
        _check(pipelines_lib().gern_cache_attention_create(head_dim, page_size, kind, flags, C.byref(self.h)))

    def workspace_bytes(self, tokens, requests, q_heads, kv_heads, max_queries, max_length):
        """Bytes of device memory that a call of these sizes needs."""
        n = C.c_int64(-1)
        _check(pipelines_lib().gern_cache_attention_workspace(self.h, tokens, requests, q_heads, kv_heads, max_queries, max_length, C.byref(n)))
        return n.value

    def __call__(self, q, k_cache, v_cache, k_scales, v_scales, table, lengths, starts, out, scale, max_queries=1, max_length=None, workspace=None,
                 stream=None):
        """q, out [tokens, q_heads, head_dim] (any stride from token to token); the cache as CacheWrite fills it; table
        [requests, width], lengths [requests], starts [requests + 1] int32.  max_length: the most keys of a request, by
        default what the table has room for; workspace: a uint8 tensor of workspace_bytes."""
        pages, heads = self._cache(k_cache, v_cache, k_scales, v_scales)
        self._int32(table=table, lengths=lengths, starts=starts)
        ldq, ldo = self._rows("q", q), self._rows("out", out)
        shape, width = q.shape, table.shape
        _expect(len(shape) == 3 and shape[2] == self.head_dim and out.shape == shape, "q and out must be [tokens, q_heads, head_dim]")
        _expect(len(width) == 2 and lengths.shape == (width[0],) and starts.shape == (width[0] + 1,),
                "table must be [requests, width], lengths [requests] and starts [requests + 1]")
        self._on_gpu(q, k_cache, v_cache, k_scales, v_scales, table, lengths, starts, out)
        at, size = None, 0
        if workspace is not None:
            _expect(workspace.is_contiguous(), "the workspace must be contiguous")
            self._on_gpu(workspace)
            at, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        _check(self._run(self.h, q.data_ptr(), ldq, k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages, table.data_ptr(),
                         width[1], lengths.data_ptr(), starts.data_ptr(), width[0], shape[0], shape[1], heads, out.data_ptr(), ldo, scale, max_queries,
                         width[1] * self.page_size if max_length is None else max_length, at, size,
                         self._current_stream(self._device) if stream is None else stream))
        return out


class Matvec4(_ServingPipeline):
    """y = x W^T for up to 64 rows of x and W in 4 bits with scales (and zero points) of groups of columns (gern_matvec4_run)."""

    def __init__(self, group=128, dtype="bf16", flags=0):
        kind = _type(dtype)
        super().__init__(dtype)
        self.group, self.dtype, self._run = group, dtype, pipelines_lib().gern_matvec4_run
        _check(pipelines_lib().gern_matvec4_create(group, kind, flags, C.byref(self.h)))

    def __call__(self, x, codes, scales, y, zeros=None, stream=None):
        """x [rows, K] and y [rows, N] (any stride from row to row); codes [N, K / 2] uint8, the even column in the lower
        half; scales [K / group, N] of x's type; zeros [K / group, N] uint8, by default 8 everywhere."""
        ldx, ldy = self._rows("x", x), self._rows("y", y)
        _expect(x.dim() == y.dim() == 2 and y.shape[0] == x.shape[0], "x must be [rows, K] and y [rows, N]")
        (m, k), n = x.shape, y.shape[1]
        groups = (k // self.group, n)
        _expect(codes.dtype is self._uint8 and codes.shape == (n, k // 2) and codes.is_contiguous(), "codes must be a contiguous uint8 tensor [N, K / 2]")
        _expect(scales.dtype is self._half and scales.shape == groups and scales.is_contiguous(), "scales must be a contiguous tensor [K / group, N] of x's type")
        at = None
        if zeros is not None:
            _expect(zeros.dtype is self._uint8 and zeros.shape == groups and zeros.is_contiguous(), "zeros must be a contiguous uint8 tensor [K / group, N]")
            self._on_gpu(zeros)
            at = zeros.data_ptr()
        self._on_gpu(x, codes, scales, y)
        _check(self._run(self.h, x.data_ptr(), ldx, codes.data_ptr(), scales.data_ptr(), at, y.data_ptr(), ldy, m, n, k,
                         self._current_stream(self._device) if stream is None else stream))
        return y
