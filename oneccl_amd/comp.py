"""ctypes binding of libmi_ccl_comp.so (C ABI: include/mi_ccl_comp.h).

Every function takes device tensors (or raw device pointers) and a HIP stream and enqueues the HIP kernels;
there is no CPU fallback: a missing library raises at load time.
"""
import array
import ctypes as C
import functools
import operator
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("MI_CCL_COMP_LIB") or os.path.join(HERE, "libmi_ccl_comp.so")     # another build, for A/B runs

# ccl::datatype (include/oneapi/ccl/types.hpp:52-69)
INT8, UINT8, INT16, UINT16, INT32, UINT32, INT64, UINT64, FLOAT16, FLOAT32, FLOAT64, BFLOAT16 = range(12)
# ccl::reduction (types.hpp:41-47)
SUM, PROD, MIN, MAX, CUSTOM = range(5)
# ccl::status (src/internal_types.hpp:29-37)
SUCCESS, OUT_OF_RESOURCE, INVALID_ARGUMENTS, RUNTIME_ERROR = range(4)
# ccl_bf16_impl_type (src/comp/bf16/bf16_utils.hpp:26)
BF16_SCALAR, BF16_AVX512F, BF16_AVX512BF = 0, 1, 2
# ccl_fp16_impl_type (src/comp/fp16/fp16_utils.hpp:26-32); 0 = the process-wide default (set_param("fp16_impl"))
FP16_DEFAULT, FP16_F16C, FP16_AVX512F, FP16_AVX512FP16 = 0, 2, 3, 4
LP_PAIRWISE, LP_KEEP_PRECISION, LP_TAIL_QUIRK = 0, 1, 2

DTYPE_SIZE = [1, 1, 2, 2, 4, 4, 8, 8, 2, 4, 8, 2]

EXPORTS = [
    "mi_ccl_datatype_size", "mi_ccl_datatype_name", "mi_ccl_reduction_to_str", "mi_ccl_status_str",
    "mi_ccl_kernel_name", "mi_ccl_comp_reduce", "mi_ccl_bf16_reduce", "mi_ccl_fp16_reduce",
    "mi_ccl_comp_reduce_n", "mi_ccl_comp_reduce_write_n", "mi_ccl_comp_reduce_batch", "mi_ccl_comp_batch_reduce",
    "mi_ccl_comp_copy",
    "mi_ccl_convert_fp32_to_bf16_arrays", "mi_ccl_convert_bf16_to_fp32_arrays",
    "mi_ccl_convert_fp32_to_fp16_arrays", "mi_ccl_convert_fp16_to_fp32_arrays", "mi_ccl_fusion_offsets",
    "mi_ccl_fusion_plan_create", "mi_ccl_fusion_plan_destroy", "mi_ccl_fusion_plan_bytes",
    "mi_ccl_fusion_plan_offset", "mi_ccl_fusion_pack", "mi_ccl_fusion_unpack", "mi_ccl_fusion_reduce",
    "mi_ccl_fusion_reduce_static",
    "mi_ccl_fusion_plan_elements", "mi_ccl_fusion_norm_workspace", "mi_ccl_fusion_norm", "mi_ccl_fusion_adamw",
    "mi_ccl_fusion_state_decode", "mi_ccl_fusion_state_encode",
    "mi_ccl_token_rows", "mi_ccl_token_sort_workspace", "mi_ccl_token_sort", "mi_ccl_token_order_workspace", "mi_ccl_token_dispatch", "mi_ccl_token_combine",
    "mi_ccl_token_combine_backward",
    "mi_ccl_probe_bandwidth", "mi_ccl_last_kernel", "mi_ccl_set_param", "mi_ccl_get_param",
]


STATE_FP32, STATE_8BIT = 0, 1          # formats of the AdamW states
STATE_BLOCK = 256                      # elements that share a scale in the 8-bit format
ADAMW_WORKSPACE = 16                   # bytes, of a step whose number or learning rate is read from the device


class AdamwOptions(C.Structure):
    """mi_ccl_adamw_options"""
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double),
                ("step", C.c_int64), ("seed", C.c_uint64), ("stochastic", C.c_int), ("step_ptr", C.c_void_p), ("lr_ptr", C.c_void_p),
                ("grad_scale", C.c_void_p), ("workspace", C.c_void_p)]


class CclError(RuntimeError):
    def __init__(self, status, what):
        self.status = status
        super().__init__(f"{what}: {status_str(status)} ({status})")


_lib = None


def lib():
    """Load the HIP library; raises if it was not built (no fallback of any kind)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C oneccl_amd/csrc` "
                           "(or __graft_entry__.build()); there is no CPU fallback")
    L = C.CDLL(LIB_PATH)
    vp, sz, i = C.c_void_p, C.c_size_t, C.c_int
    L.mi_ccl_datatype_size.restype = sz
    L.mi_ccl_datatype_size.argtypes = [i]
    for f in ("mi_ccl_datatype_name", "mi_ccl_reduction_to_str", "mi_ccl_status_str"):
        getattr(L, f).restype = C.c_char_p
        getattr(L, f).argtypes = [i]
    L.mi_ccl_kernel_name.argtypes = [C.c_char_p, i, i, C.c_char_p, sz]
    L.mi_ccl_comp_reduce.argtypes = [i, i, vp, sz, vp, i, i, vp]
    L.mi_ccl_bf16_reduce.argtypes = [vp, sz, vp, i, i, vp]
    L.mi_ccl_fp16_reduce.argtypes = [vp, sz, vp, i, i, vp]
    L.mi_ccl_comp_reduce_n.argtypes = [i, i, vp, i, vp, sz, i, i, i, vp]
    L.mi_ccl_comp_reduce_write_n.argtypes = [i, i, vp, i, vp, i, sz, i, i, i, vp]
    L.mi_ccl_comp_reduce_batch.argtypes = [i, i, vp, i, vp, vp, i, i, i, i, vp]
    L.mi_ccl_comp_batch_reduce.argtypes = [vp, vp, sz, sz, vp, i, i, i, i, i, vp]
    L.mi_ccl_comp_copy.argtypes = [vp, vp, sz, i, vp]
    L.mi_ccl_convert_fp32_to_bf16_arrays.argtypes = [vp, vp, sz, i, vp]
    L.mi_ccl_convert_bf16_to_fp32_arrays.argtypes = [vp, vp, sz, vp]
    L.mi_ccl_convert_fp32_to_fp16_arrays.argtypes = [vp, vp, sz, vp]
    L.mi_ccl_convert_fp16_to_fp32_arrays.argtypes = [vp, vp, sz, vp]
    L.mi_ccl_fusion_offsets.argtypes = [vp, sz, sz, sz, vp, vp]
    L.mi_ccl_fusion_plan_create.argtypes = [vp, sz, i, sz, C.POINTER(vp)]
    L.mi_ccl_fusion_plan_destroy.argtypes = [vp]
    L.mi_ccl_fusion_plan_bytes.restype = sz
    L.mi_ccl_fusion_plan_bytes.argtypes = [vp]
    L.mi_ccl_fusion_plan_offset.restype = sz
    L.mi_ccl_fusion_plan_offset.argtypes = [vp, sz]
    L.mi_ccl_fusion_pack.argtypes = [vp, vp, vp, vp]
    L.mi_ccl_fusion_unpack.argtypes = [vp, vp, vp, vp]
    L.mi_ccl_fusion_reduce.argtypes = [vp, i, vp, vp, i, vp, i, i, i, vp]
    L.mi_ccl_fusion_reduce_static.argtypes = [vp, sz, i, sz, i, vp, vp, i, vp, i, i, i, vp]
    L.mi_ccl_fusion_plan_elements.restype = sz
    L.mi_ccl_fusion_plan_elements.argtypes = [vp]
    L.mi_ccl_fusion_norm_workspace.restype = sz
    L.mi_ccl_fusion_norm_workspace.argtypes = [vp]
    L.mi_ccl_fusion_norm.argtypes = [vp, vp, vp, C.c_double, C.c_double, vp, vp, sz, vp]
    L.mi_ccl_fusion_adamw.argtypes = [vp, i, vp, vp, vp, i, vp, vp, vp, vp, C.POINTER(AdamwOptions), vp]
    L.mi_ccl_fusion_state_decode.argtypes = [vp, vp, vp, vp, i, vp, vp, vp]
    L.mi_ccl_fusion_state_encode.argtypes = [vp, i, vp, vp, vp, vp, vp, vp]
    L.mi_ccl_token_rows.argtypes = [sz, i, i, sz, sz, C.POINTER(sz)]
    L.mi_ccl_token_sort_workspace.argtypes = [sz, i, i, C.POINTER(sz)]
    L.mi_ccl_token_sort.argtypes = [i, vp, sz, i, i, sz, sz, vp, vp, vp, vp, sz, vp]
    L.mi_ccl_token_order_workspace.argtypes = [i, sz, i, sz, C.POINTER(sz)]
    L.mi_ccl_token_dispatch.argtypes = [i, vp, sz, sz, i, sz, vp, vp, vp, i, vp, sz, sz, vp, sz, vp]
    L.mi_ccl_token_combine.argtypes = [i, vp, sz, sz, vp, vp, sz, i, sz, vp, sz, vp]
    L.mi_ccl_token_combine_backward.argtypes = [i, vp, sz, vp, sz, sz, vp, vp, vp, vp, i, sz, i, sz, vp, sz, vp, vp, sz, vp]
    L.mi_ccl_probe_bandwidth.argtypes = [i, vp, i, sz, vp]
    L.mi_ccl_last_kernel.restype = C.c_char_p
    L.mi_ccl_last_kernel.argtypes = []
    L.mi_ccl_set_param.argtypes = [C.c_char_p, C.c_long]
    L.mi_ccl_get_param.restype = C.c_long
    L.mi_ccl_get_param.argtypes = [C.c_char_p]
    _lib = L
    return L


def status_str(status):
    return lib().mi_ccl_status_str(int(status)).decode()


def _check(status, what):
    if status != SUCCESS:
        raise CclError(status, what)


def _ptr(x):
    """Device address of a torch tensor, or an int address passed through."""
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        # what torch.cuda.current_stream().cuda_stream is, without building a Stream object (0.3 against 2.6 us)
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


_native = None              # oneccl_amd._tensors, loaded behind torch, whose libraries it needs; False where it was not built


def _device():
    global _native
    import torch
    if _native is None:
        try:
            from . import _tensors as _native
        except ImportError:
            _native = False
    return torch.cuda.current_device()


def _ptr_array(xs):
    return (C.c_void_p * len(xs))(*[_ptr(x) for x in xs])


_TORCH_DTYPE = {INT32: "int32", INT64: "int64", FLOAT16: "float16", FLOAT32: "float32", BFLOAT16: "bfloat16"}
_CCL_DTYPE = {v: k for k, v in _TORCH_DTYPE.items()}
_KINDS = {}                 # torch.dtype -> (ccl dtype or -1)


def _kind(t):
    """The ccl datatype of a tensor's elements, -1 for one that no operator takes (the library refuses it)."""
    k = _KINDS.get(t.dtype)
    if k is None:
        k = _KINDS[t.dtype] = _CCL_DTYPE.get(str(t.dtype).replace("torch.", ""), -1)
    return k


def _refuse(what, t, wanted):
    if t is None:
        raise ValueError(f"{what}: missing")
    raise ValueError(f"{what}: {wanted} is wanted, got {t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}")


def _memory(what, t, dtype, least, here):
    """Address of a contiguous tensor of the current GPU with at least `least` elements."""
    if _native:
        address = _native.memory(t, dtype, least, here)
        if address is not None:
            return address
    if t is None or t.dtype is not dtype or t.numel() < least or t.get_device() != here or not t.is_contiguous():
        _refuse(what, t, f"contiguous {dtype}, {least} elements at least, on cuda:{here}")
    return t.data_ptr()


def _optional(what, t, dtype, least, here):
    return None if t is None else _memory(what, t, dtype, least, here)


def _workspace(workspace, need, here, stream):
    """(address, bytes, what has to live until the call has returned) of a call's scratch memory, allocated when there is none:
    from the pool of the stream that the call runs on, whose order is what makes the memory free for it and, later, for others."""
    import torch
    if workspace is None:
        if not need:
            return None, 0, None
        if stream is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=here)
        else:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
            with torch.cuda.stream(stream):
                workspace = torch.empty(need, dtype=torch.uint8, device=here)
    elif workspace.get_device() != here or not workspace.is_contiguous():
        _refuse("workspace", workspace, f"contiguous memory on cuda:{here}")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace


def _table(what, tensors, dtype, least, here):
    """(what ctypes takes as the address of a table of the tensors' addresses, what holds it): _memory's conditions for a list, least[i]
    elements of the i-th (an array of 64-bit numbers)."""
    import torch
    if _native:
        table = _native.addresses(tensors, dtype, least, here)
        if table is not None:
            return table, table
    T = torch.Tensor
    try:
        devices, kinds = set(map(T.get_device, tensors)), {t.dtype for t in tensors}
        whole, sizes = all(map(T.is_contiguous, tensors)), list(map(T.numel, tensors))
    except (TypeError, AttributeError):
        raise ValueError(f"{what}: a tensor is missing") from None
    if devices != {here}:
        raise ValueError(f"{what}: not on the current device, cuda:{here}")
    if not whole:
        raise ValueError(f"{what}: not contiguous")
    if kinds != {dtype}:
        raise ValueError(f"{what}: {kinds}, {dtype} is wanted")
    if any(map(operator.lt, sizes, least)):
        raise ValueError(f"{what}: a tensor has fewer elements than the plan says")
    table = array.array("Q", list(map(T.data_ptr, tensors)))
    return table.buffer_info()[0], table


def datatype_size(dtype):
    return lib().mi_ccl_datatype_size(dtype)


def datatype_name(dtype):
    return lib().mi_ccl_datatype_name(dtype).decode()


def reduction_to_str(op):
    return lib().mi_ccl_reduction_to_str(op).decode()


def kernel_name(kernel, dtype, op):
    buf = C.create_string_buffer(128)
    _check(lib().mi_ccl_kernel_name(kernel.encode(), dtype, op, buf, 128), "mi_ccl_kernel_name")
    return buf.value.decode()


def comp_reduce(dtype, op, inp, count, inout, bf16_impl=BF16_AVX512BF, fp16_impl=FP16_DEFAULT, stream=None):
    """inout[i] = inout[i] OP inp[i] (ccl_comp_reduce)."""
    _check(lib().mi_ccl_comp_reduce(dtype, op, _ptr(inp), count, _ptr(inout), bf16_impl, fp16_impl, _stream(stream)),
           "mi_ccl_comp_reduce")


def bf16_reduce(inp, count, inout, op, bf16_impl=BF16_AVX512BF, stream=None):
    _check(lib().mi_ccl_bf16_reduce(_ptr(inp), count, _ptr(inout), op, bf16_impl, _stream(stream)),
           "mi_ccl_bf16_reduce")


def fp16_reduce(inp, count, inout, op, fp16_impl=FP16_DEFAULT, stream=None):
    _check(lib().mi_ccl_fp16_reduce(_ptr(inp), count, _ptr(inout), op, fp16_impl, _stream(stream)),
           "mi_ccl_fp16_reduce")


def comp_reduce_n(dtype, op, srcs, dst, count, lp_mode=LP_PAIRWISE, bf16_impl=BF16_AVX512BF, fp16_impl=FP16_DEFAULT,
                  stream=None):
    """dst = srcs[0] OP srcs[1] OP ... in argument order, one pass."""
    arr = _ptr_array(srcs)
    _check(lib().mi_ccl_comp_reduce_n(dtype, op, arr, len(srcs), _ptr(dst), count, lp_mode, bf16_impl, fp16_impl,
                                      _stream(stream)), "mi_ccl_comp_reduce_n")


def comp_reduce_write_n(dtype, op, srcs, dsts, count, lp_mode=LP_PAIRWISE, bf16_impl=BF16_AVX512BF,
                        fp16_impl=FP16_DEFAULT, stream=None):
    """Every dsts[k] = srcs[0] OP srcs[1] OP ... in argument order, one pass; one source and LP_PAIRWISE is a
    copy of one buffer to len(dsts) buffers."""
    s, d = _ptr_array(srcs), _ptr_array(dsts)
    _check(lib().mi_ccl_comp_reduce_write_n(dtype, op, s, len(srcs), d, len(dsts), count, lp_mode, bf16_impl,
                                            fp16_impl, _stream(stream)), "mi_ccl_comp_reduce_write_n")


def comp_reduce_batch(dtype, op, jobs, lp_mode=LP_PAIRWISE, bf16_impl=BF16_AVX512BF, fp16_impl=FP16_DEFAULT, stream=None):
    """Many independent reduces in one launch.  jobs: list of (srcs, dst, count), every job with the same number of
    inputs; dst = srcs[0] OP srcs[1] OP ... over count elements."""
    if not jobs:
        return
    n = len(jobs[0][0])
    assert all(len(j[0]) == n for j in jobs), "every job takes the same number of inputs"
    srcs = _ptr_array([s for j in jobs for s in j[0]])
    dsts = _ptr_array([j[1] for j in jobs])
    counts = (C.c_size_t * len(jobs))(*[int(j[2]) for j in jobs])
    _check(lib().mi_ccl_comp_reduce_batch(dtype, op, srcs, n, dsts, counts, len(jobs), lp_mode, bf16_impl, fp16_impl,
                                          _stream(stream)), "mi_ccl_comp_reduce_batch")


class BatchJobs:
    """The pointer and count tables of a batch, built once: calling it costs one foreign call instead of one
    data_ptr() per buffer (which a timing loop would otherwise measure)."""

    def __init__(self, jobs):
        self.n = len(jobs[0][0])
        assert all(len(j[0]) == self.n for j in jobs), "every job takes the same number of inputs"
        self.keep = jobs                      # the tensors stay alive with the tables
        self.srcs = _ptr_array([s for j in jobs for s in j[0]])
        self.dsts = _ptr_array([j[1] for j in jobs])
        self.counts = (C.c_size_t * len(jobs))(*[int(j[2]) for j in jobs])
        self.n_jobs = len(jobs)

    def reduce(self, dtype, op, lp_mode=LP_PAIRWISE, bf16_impl=BF16_AVX512BF, fp16_impl=FP16_DEFAULT, stream=None):
        _check(lib().mi_ccl_comp_reduce_batch(dtype, op, self.srcs, self.n, self.dsts, self.counts, self.n_jobs, lp_mode,
                                              bf16_impl, fp16_impl, _stream(stream)), "mi_ccl_comp_reduce_batch")


def comp_batch_reduce(in_buf, offsets, count, inout, dtype, op, keep_precision, bf16_impl=BF16_AVX512BF,
                      fp16_impl=FP16_DEFAULT, stream=None):
    offs = (C.c_size_t * len(offsets))(*[int(o) for o in offsets])
    _check(lib().mi_ccl_comp_batch_reduce(_ptr(in_buf), offs, len(offsets), count, _ptr(inout), dtype, op,
                                          int(keep_precision), bf16_impl, fp16_impl, _stream(stream)),
           "mi_ccl_comp_batch_reduce")


def comp_copy(inp, out, nbytes, use_nontemporal=False, stream=None):
    _check(lib().mi_ccl_comp_copy(_ptr(inp), _ptr(out), nbytes, int(use_nontemporal), _stream(stream)),
           "mi_ccl_comp_copy")


def convert_fp32_to_bf16_arrays(fp32_buf, bf16_buf, count, bf16_impl=BF16_AVX512BF, stream=None):
    _check(lib().mi_ccl_convert_fp32_to_bf16_arrays(_ptr(fp32_buf), _ptr(bf16_buf), count, bf16_impl,
                                                    _stream(stream)), "mi_ccl_convert_fp32_to_bf16_arrays")


def convert_fp32_to_fp16_arrays(fp32_buf, fp16_buf, count, stream=None):
    _check(lib().mi_ccl_convert_fp32_to_fp16_arrays(_ptr(fp32_buf), _ptr(fp16_buf), count, _stream(stream)),
           "mi_ccl_convert_fp32_to_fp16_arrays")


def convert_fp16_to_fp32_arrays(fp16_buf, fp32_buf, count, stream=None):
    _check(lib().mi_ccl_convert_fp16_to_fp32_arrays(_ptr(fp16_buf), _ptr(fp32_buf), count, _stream(stream)),
           "mi_ccl_convert_fp16_to_fp32_arrays")


def convert_bf16_to_fp32_arrays(bf16_buf, fp32_buf, count, stream=None):
    _check(lib().mi_ccl_convert_bf16_to_fp32_arrays(_ptr(bf16_buf), _ptr(fp32_buf), count, _stream(stream)),
           "mi_ccl_convert_bf16_to_fp32_arrays")


def fusion_offsets(counts, dtype_size, align):
    k = len(counts)
    cnt = (C.c_size_t * k)(*[int(c) for c in counts])
    offs = (C.c_size_t * k)()
    total = C.c_size_t(0)
    _check(lib().mi_ccl_fusion_offsets(cnt, k, dtype_size, align, offs, C.byref(total)), "mi_ccl_fusion_offsets")
    return list(offs), total.value


class FusionPlan:
    """Layout of one fused group (counts, dtype, alignment) and its device-side work table."""

    def __init__(self, counts, dtype, align=256):
        k = len(counts)
        cnt = (C.c_size_t * k)(*[int(c) for c in counts])
        h = C.c_void_p()
        _check(lib().mi_ccl_fusion_plan_create(cnt, k, dtype, align, C.byref(h)), "mi_ccl_fusion_plan_create")
        self._h = h
        self.k = k
        self.dtype = dtype
        self.counts = [int(c) for c in counts]
        self._least = array.array("q", self.counts)
        import torch
        self._torch_dtype = getattr(torch, _TORCH_DTYPE.get(dtype, "float32"))
        self.norm_workspace = lib().mi_ccl_fusion_norm_workspace(h)       # bytes
        self._here = _device()              # the GPU that holds the plan's table
        self.elements = lib().mi_ccl_fusion_plan_elements(h)      # of a state or fp32 copy of the weights in the plan's layout

    @property
    def nbytes(self):
        return lib().mi_ccl_fusion_plan_bytes(self._h)

    def offset(self, i):
        return lib().mi_ccl_fusion_plan_offset(self._h, i)

    def pack(self, tensors, fusion_buf, stream=None):
        assert len(tensors) == self.k
        _check(lib().mi_ccl_fusion_pack(self._h, _ptr_array(tensors), _ptr(fusion_buf), _stream(stream)),
               "mi_ccl_fusion_pack")

    def unpack(self, fusion_buf, tensors, stream=None):
        assert len(tensors) == self.k
        _check(lib().mi_ccl_fusion_unpack(self._h, _ptr(fusion_buf), _ptr_array(tensors), _stream(stream)),
               "mi_ccl_fusion_unpack")

    def reduce(self, op, own_tensors, peers, out_tensors, lp_mode=LP_PAIRWISE, bf16_impl=BF16_AVX512BF,
               fp16_impl=FP16_DEFAULT, stream=None):
        assert len(own_tensors) == self.k and len(out_tensors) == self.k
        _check(lib().mi_ccl_fusion_reduce(self._h, op, _ptr_array(own_tensors), _ptr_array(peers), len(peers),
                                          _ptr_array(out_tensors), lp_mode, bf16_impl, fp16_impl, _stream(stream)),
               "mi_ccl_fusion_reduce")

    # ---- the optimizer step behind the reduce: gradients are the plan's tensors (a list) or its fusion buffer (one tensor) ----

    def _device(self):
        here = _device()
        if here != self._here:
            raise ValueError(f"the plan was made on cuda:{self._here}, the current device is cuda:{here}")
        return here

    def _gradients(self, grads, here):
        """(address of a table of addresses, address of a fusion buffer, what has to live until the call has returned)."""
        kind = self._torch_dtype
        if isinstance(grads, (list, tuple)):
            if len(grads) != self.k:
                raise ValueError("the gradients are not the plan's tensors")
            address, table = _table("gradients", grads, kind, self._least, here)
            return address, None, table
        return None, _memory("gradients", grads, kind, self.elements, here), None

    def norm(self, grads, result, multiplier=1.0, max_norm=0.0, workspace=None, stream=None):
        """result[0] = the norm of all gradients times `multiplier`, result[1] = the factor of a clipped step's gradients (two
        floats on the device).  workspace: norm_workspace bytes of device memory; allocated for the call when None."""
        import torch
        here = self._device()
        res = _memory("result", result, torch.float32, 2, here)
        lst, buf, _held = self._gradients(grads, here)
        ws, size, _keep = _workspace(workspace, self.norm_workspace, here, stream)
        _check(lib().mi_ccl_fusion_norm(self._h, lst, buf, multiplier, max_norm, res, ws, size, _stream(stream)), "mi_ccl_fusion_norm")

    def adamw(self, params, grads, exp_avg, exp_avg_sq, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1, scales=None,
              master=None, grad_scale=None, seed=None, step_ptr=None, lr_ptr=None, workspace=None, stream=None):
        """One AdamW step over the plan's tensors, in place.  States: float32 (32 bits) or uint8 (8 bits, with `scales`) in the
        plan's layout.  seed: not None rounds 8-bit states stochastically.  step_ptr (int64), lr_ptr and grad_scale (float32):
        one-element device tensors read by the kernel.  workspace: with step_ptr or lr_ptr, ADAMW_WORKSPACE bytes; allocated for
        the call when None."""
        import torch
        here = self._device()
        if len(params) != self.k or params[0] is None:
            raise ValueError("the parameters are not the plan's tensors")
        weights, _held_too = _table("params", params, params[0].dtype, self._least, here)
        eight = exp_avg.dtype is torch.uint8
        kind = torch.uint8 if eight else torch.float32
        m, v = _memory("exp_avg", exp_avg, kind, self.elements, here), _memory("exp_avg_sq", exp_avg_sq, kind, self.elements, here)
        sc = _memory("scales", scales, torch.uint8, 2 * ((self.elements + STATE_BLOCK - 1) // STATE_BLOCK), here) if eight else None
        ws, size, _keep = _workspace(workspace, ADAMW_WORKSPACE if step_ptr is not None or lr_ptr is not None else 0, here, stream)
        if workspace is not None and size < ADAMW_WORKSPACE:
            raise ValueError(f"workspace: {size} bytes, {ADAMW_WORKSPACE} are needed")
        o = AdamwOptions(lr, beta1, beta2, eps, weight_decay, int(step), 0 if seed is None else int(seed), int(seed is not None),
                         _optional("step_ptr", step_ptr, torch.int64, 1, here), _optional("lr_ptr", lr_ptr, torch.float32, 1, here),
                         _optional("grad_scale", grad_scale, torch.float32, 1, here), ws)
        lst, buf, _held = self._gradients(grads, here)
        _check(lib().mi_ccl_fusion_adamw(self._h, _kind(params[0]), weights, lst, buf, STATE_8BIT if eight else STATE_FP32,
                                         m, v, sc, _optional("master", master, torch.float32, self.elements, here), C.byref(o),
                                         _stream(stream)), "mi_ccl_fusion_adamw")

    def _state_memory(self, exp_avg, exp_avg_sq, scales, values_avg, values_sq):
        import torch
        here = self._device()
        return (_memory("exp_avg", exp_avg, torch.uint8, self.elements, here), _memory("exp_avg_sq", exp_avg_sq, torch.uint8, self.elements, here),
                _memory("scales", scales, torch.uint8, 2 * ((self.elements + STATE_BLOCK - 1) // STATE_BLOCK), here),
                _memory("values", values_avg, values_avg.dtype, self.elements, here), _memory("values", values_sq, values_avg.dtype, self.elements, here))

    def state_decode(self, exp_avg, exp_avg_sq, scales, values_avg, values_sq, stream=None):
        """The values of 8-bit states, float32 or bfloat16."""
        m, v, sc, vm, vv = self._state_memory(exp_avg, exp_avg_sq, scales, values_avg, values_sq)
        _check(lib().mi_ccl_fusion_state_decode(self._h, m, v, sc, _kind(values_avg), vm, vv, _stream(stream)), "mi_ccl_fusion_state_decode")

    def state_encode(self, values_avg, values_sq, exp_avg, exp_avg_sq, scales, stream=None):
        """Values (float32 or bfloat16) to 8-bit states, rounded to nearest."""
        m, v, sc, vm, vv = self._state_memory(exp_avg, exp_avg_sq, scales, values_avg, values_sq)
        _check(lib().mi_ccl_fusion_state_encode(self._h, _kind(values_avg), vm, vv, m, v, sc, _stream(stream)), "mi_ccl_fusion_state_encode")

    def close(self):
        if self._h:
            lib().mi_ccl_fusion_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


FUSION_STATIC_MAX_TENSORS, FUSION_STATIC_MAX_ITEMS = 1024, 131072


def fusion_reduce_static(counts, dtype, align, op, own_tensors, peers, out_tensors, lp_mode=LP_PAIRWISE,
                         bf16_impl=BF16_AVX512BF, fp16_impl=FP16_DEFAULT, stream=None):
    """FusionPlan.reduce without a plan and without any allocation (mi_ccl_fusion_reduce_static)."""
    k = len(counts)
    cnt = (C.c_size_t * k)(*[int(c) for c in counts])
    _check(lib().mi_ccl_fusion_reduce_static(cnt, k, dtype, align, op, _ptr_array(own_tensors), _ptr_array(peers),
                                             len(peers), _ptr_array(out_tensors), lp_mode, bf16_impl, fp16_impl,
                                             _stream(stream)), "mi_ccl_fusion_reduce_static")


# ---- tokens sorted by expert, and back --------------------------------------------------------------------------------

def _rows(what, t, hidden, dtype, here):
    """(rows, elements from row to row, address) of a matrix whose rows are contiguous and do not overlap."""
    if _native:
        found = _native.rows(t, hidden, dtype, here)
        if found is not None:
            return found
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[1] != hidden or t.dtype is not dtype or t.get_device() != here or (hidden > 1 and stride[1] != 1) or \
            (shape[0] > 1 and stride[0] < hidden):
        _refuse(what, t, f"rows of {hidden} {dtype} on cuda:{here}")
    # one row, or none, has no distance to the next
    return shape[0], stride[0] if shape[0] > 1 else hidden, t.data_ptr()


def token_rows(n_tokens, top_k, n_experts, align=1, capacity=0):
    """Most rows that the sorted buffer can take."""
    r = C.c_size_t()
    _check(lib().mi_ccl_token_rows(n_tokens, top_k, n_experts, align, capacity, C.byref(r)), "mi_ccl_token_rows")
    return r.value


# both are arithmetic on the sizes, looked up by them: a step asks for the same ones again and again, at 1.2 us each
@functools.lru_cache(maxsize=1024)
def token_sort_workspace(n_tokens, top_k, n_experts):
    r = C.c_size_t()
    _check(lib().mi_ccl_token_sort_workspace(n_tokens, top_k, n_experts, C.byref(r)), "mi_ccl_token_sort_workspace")
    return r.value


def token_sort(expert_ids, n_experts, positions, counts, offsets, align=1, capacity=0, workspace=None, stream=None):
    """Row of every entry of expert_ids [tokens, top_k] (int32 or int64) in the buffer sorted by expert, into positions (int32,
    the same shape; -1: none); rows of each expert into counts, first rows and the end into offsets [n_experts + 1] (int32).
    workspace: token_sort_workspace bytes; allocated for the call when None."""
    import torch
    here = _device()
    shape = expert_ids.shape
    if len(shape) != 2 or positions.shape != shape:
        raise ValueError("expert_ids and positions are [tokens, top_k]")
    n, k = shape
    ids = _memory("expert_ids", expert_ids, expert_ids.dtype, 0, here)
    pos = _memory("positions", positions, torch.int32, 0, here)
    cnt, off = _memory("counts", counts, torch.int32, n_experts, here), _memory("offsets", offsets, torch.int32, n_experts + 1, here)
    ws, size, _keep = _workspace(workspace, token_sort_workspace(n, k, n_experts), here, stream)
    _check(lib().mi_ccl_token_sort(_kind(expert_ids), ids, n, k, n_experts, align, capacity, pos, cnt, off, ws, size, _stream(stream)),
           "mi_ccl_token_sort")


@functools.lru_cache(maxsize=1024)
def token_order_workspace(dtype, n_tokens, top_k, hidden):
    """Bytes of scratch memory that a large token_dispatch or token_combine_backward goes faster with."""
    r = C.c_size_t()
    _check(lib().mi_ccl_token_order_workspace(dtype, n_tokens, top_k, hidden, C.byref(r)), "mi_ccl_token_order_workspace")
    return r.value


def _weights(what, t, positions, here):
    """Address of fp32 numbers, one per entry; None for None."""
    import torch
    if t is not None and t.shape != positions.shape:
        _refuse(what, t, f"{tuple(positions.shape)}, the shape of positions,")
    return _optional(what, t, torch.float32, 0, here)


def _positions(positions, tokens, here):
    import torch
    shape = positions.shape
    if len(shape) != 2 or shape[0] != tokens:
        _refuse("positions", positions, f"[{tokens}, top_k]")
    return shape[1], _memory("positions", positions, torch.int32, 0, here)


def token_dispatch(x, positions, counts, offsets, out, workspace=None, stream=None):
    """out[positions[t, j]] = x[t]; padding rows become zero, rows behind the last expert's stay as they are.  workspace:
    token_order_workspace bytes; allocated for the call when None."""
    import torch
    here = _device()
    hidden, experts = x.shape[-1], counts.numel()
    n, ldx, px = _rows("x", x, hidden, x.dtype, here)
    rows, ldo, po = _rows("out", out, hidden, x.dtype, here)
    k, pos = _positions(positions, n, here)
    kind = _kind(x)
    ws, size, _keep = _workspace(workspace, token_order_workspace(kind, n, k, hidden), here, stream)
    _check(lib().mi_ccl_token_dispatch(kind, px, ldx, n, k, hidden, pos, _memory("counts", counts, torch.int32, experts, here),
                                       _memory("offsets", offsets, torch.int32, experts + 1, here), experts, po, ldo, rows, ws, size,
                                       _stream(stream)), "mi_ccl_token_dispatch")


def token_combine(y, positions, weights, out, stream=None):
    """out[t] = sum over j of weights[t, j] * y[positions[t, j]]; weights (float32, the shape of positions) may be None for ones."""
    import torch
    here = _device()
    hidden = y.shape[-1]
    rows, ldy, py = _rows("y", y, hidden, y.dtype, here)
    n, ldo, po = _rows("out", out, hidden, y.dtype, here)
    k, pos = _positions(positions, n, here)
    _check(lib().mi_ccl_token_combine(_kind(y), py, ldy, rows, pos, _weights("weights", weights, positions, here), n, k, hidden, po, ldo,
                                      _stream(stream)), "mi_ccl_token_combine")


def token_combine_backward(grad_out, y, positions, weights, counts, offsets, grad_y, grad_weights=None, workspace=None, stream=None):
    """The gradient of token_combine: grad_y[positions[t, j]] = weights[t, j] * grad_out[t], with padding rows zero, and unless
    None grad_weights[t, j] = <grad_out[t], y[positions[t, j]]>.  y may be None without grad_weights.  workspace:
    token_order_workspace bytes; allocated for the call when None."""
    import torch
    here = _device()
    hidden, kind, experts = grad_out.shape[-1], grad_out.dtype, counts.numel()
    n, ldg, pg = _rows("grad_out", grad_out, hidden, kind, here)
    rows, ldd, pd = _rows("grad_y", grad_y, hidden, kind, here)
    ldy, py = hidden, None
    if y is not None:
        y_rows, ldy, py = _rows("y", y, hidden, kind, here)
        if y_rows != rows:
            raise ValueError(f"y has {y_rows} rows, grad_y {rows}")
    elif grad_weights is not None:
        raise ValueError("grad_weights needs y")
    k, pos = _positions(positions, n, here)
    dtype = _kind(grad_out)
    ws, size, _keep = _workspace(workspace, token_order_workspace(dtype, n, k, hidden), here, stream)
    _check(lib().mi_ccl_token_combine_backward(dtype, pg, ldg, py, ldy, rows, pos,
                                               _weights("weights", weights, positions, here),
                                               _memory("counts", counts, torch.int32, experts, here),
                                               _memory("offsets", offsets, torch.int32, experts + 1, here), experts, n, k, hidden, pd, ldd,
                                               _weights("grad_weights", grad_weights, positions, here), ws, size, _stream(stream)),
           "mi_ccl_token_combine_backward")


def token_dispatch_backward(grad_rows, positions, grad_x, stream=None):
    """The gradient of token_dispatch: grad_x[t] = sum over j of grad_rows[positions[t, j]]."""
    token_combine(grad_rows, positions, None, grad_x, stream)


PROBE_READ, PROBE_WRITE_ONE, PROBE_WRITE_FOUR = 0, 1, 2


def probe_bandwidth(kind, bufs, nbytes, stream=None):
    """Read-only (kind PROBE_READ, all of bufs) or write-only (PROBE_WRITE_ONE / PROBE_WRITE_FOUR, bufs[0]) stream."""
    _check(lib().mi_ccl_probe_bandwidth(kind, _ptr_array(bufs), len(bufs), nbytes, _stream(stream)),
           "mi_ccl_probe_bandwidth")


def last_kernel():
    """Kernel template the calling thread's most recent call launched."""
    return lib().mi_ccl_last_kernel().decode()


def set_param(name, value):
    _check(lib().mi_ccl_set_param(name.encode(), int(value)), f"mi_ccl_set_param({name})")
    token_order_workspace.cache_clear()         # "variant" is in it


def get_param(name):
    return lib().mi_ccl_get_param(name.encode())
