"""ctypes binding of libmi_ccl_comp.so (C ABI: include/mi_ccl_comp.h).

Every function takes device tensors (or raw device pointers) and a HIP stream and enqueues the HIP kernels;
there is no CPU fallback: a missing library raises at load time.
"""
import ctypes as C
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
    "mi_ccl_token_rows", "mi_ccl_token_sort_workspace", "mi_ccl_token_sort", "mi_ccl_token_dispatch", "mi_ccl_token_combine",
    "mi_ccl_token_combine_backward",
    "mi_ccl_probe_bandwidth", "mi_ccl_last_kernel", "mi_ccl_set_param", "mi_ccl_get_param",
]


STATE_FP32, STATE_8BIT = 0, 1          # formats of the AdamW states
STATE_BLOCK = 256                      # elements that share a scale in the 8-bit format


class AdamwOptions(C.Structure):
    """mi_ccl_adamw_options"""
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double),
                ("step", C.c_int64), ("seed", C.c_uint64), ("stochastic", C.c_int), ("step_ptr", C.c_void_p), ("lr_ptr", C.c_void_p),
                ("grad_scale", C.c_void_p)]


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
    L.mi_ccl_token_dispatch.argtypes = [i, vp, sz, sz, i, sz, vp, vp, vp, i, vp, sz, sz, vp]
    L.mi_ccl_token_combine.argtypes = [i, vp, sz, sz, vp, vp, sz, i, sz, vp, sz, vp]
    L.mi_ccl_token_combine_backward.argtypes = [i, vp, sz, vp, sz, sz, vp, vp, vp, vp, i, sz, i, sz, vp, sz, vp, vp]
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
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _ptr_array(xs):
    return (C.c_void_p * len(xs))(*[_ptr(x) for x in xs])


_TORCH_DTYPE = {INT32: "int32", INT64: "int64", FLOAT16: "float16", FLOAT32: "float32", BFLOAT16: "bfloat16"}
_CCL_DTYPE = {v: k for k, v in _TORCH_DTYPE.items()}


def _dtype_name(t):
    name = str(t.dtype).replace("torch.", "")
    if name not in _CCL_DTYPE and name != "uint8":
        raise ValueError(f"tensors of {name} are not taken")
    return name


def _ptr_or_none(x):
    return None if x is None else _ptr(x)


def _check_tensors(what, tensors, dtype=None, least=0):
    """Raises unless every tensor is contiguous memory of the current GPU, of the dtype and with at least `least` elements."""
    import torch
    here = torch.cuda.current_device()
    for t in tensors:
        if t is None:
            raise ValueError(f"{what}: missing")
        if not t.is_cuda or t.device.index != here:
            raise ValueError(f"{what}: on {t.device}, the current device is cuda:{here}")
        if not t.is_contiguous():
            raise ValueError(f"{what}: not contiguous")
        if dtype is not None and str(t.dtype) != "torch." + dtype:
            raise ValueError(f"{what}: {t.dtype}, {dtype} is wanted")
        if t.numel() < least:
            raise ValueError(f"{what}: {t.numel()} elements, {least} are needed")


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

    @property
    def elements(self):
        """Elements of a state or fp32 copy of the weights in the plan's layout."""
        return lib().mi_ccl_fusion_plan_elements(self._h)

    def _gradients(self, grads):
        if isinstance(grads, (list, tuple)):
            if len(grads) != self.k or any(t.numel() < c for t, c in zip(grads, self.counts)):
                raise ValueError("the gradients are not the plan's tensors")
            _check_tensors("gradients", grads, _TORCH_DTYPE[self.dtype])
            return _ptr_array(grads), None
        _check_tensors("gradients", [grads], _TORCH_DTYPE[self.dtype], self.elements)
        return None, _ptr(grads)

    def norm(self, grads, result, multiplier=1.0, max_norm=0.0, workspace=None, stream=None):
        """result[0] = the norm of all gradients times `multiplier`, result[1] = the factor of a clipped step's gradients (two
        floats on the device).  workspace: norm_workspace bytes of device memory; allocated for the call when None."""
        import torch
        _check_tensors("result", [result], "float32", 2)
        if workspace is None:
            workspace = torch.empty(self.norm_workspace, dtype=torch.uint8, device=result.device)
        _check_tensors("workspace", [workspace])
        lst, buf = self._gradients(grads)
        _check(lib().mi_ccl_fusion_norm(self._h, lst, buf, multiplier, max_norm, _ptr(result), _ptr(workspace),
                                        workspace.numel() * workspace.element_size(), _stream(stream)), "mi_ccl_fusion_norm")

    @property
    def norm_workspace(self):
        return lib().mi_ccl_fusion_norm_workspace(self._h)

    def adamw(self, params, grads, exp_avg, exp_avg_sq, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1, scales=None,
              master=None, grad_scale=None, seed=None, step_ptr=None, lr_ptr=None, stream=None):
        """One AdamW step over the plan's tensors, in place.  States: float32 (32 bits) or uint8 (8 bits, with `scales`) in the
        plan's layout.  seed: not None rounds 8-bit states stochastically.  step_ptr (int64), lr_ptr and grad_scale (float32):
        one-element device tensors read by the kernel."""
        if len(params) != self.k or any(t.numel() < c for t, c in zip(params, self.counts)):
            raise ValueError("the parameters are not the plan's tensors")
        kind = _dtype_name(params[0])
        _check_tensors("params", params, kind)
        eight = _dtype_name(exp_avg) == "uint8"
        _check_tensors("states", [exp_avg, exp_avg_sq], "uint8" if eight else "float32", self.elements)
        if eight:
            _check_tensors("scales", [scales], "uint8", 2 * ((self.elements + STATE_BLOCK - 1) // STATE_BLOCK))
        if master is not None:
            _check_tensors("master", [master], "float32", self.elements)
        for name, t, dt in (("grad_scale", grad_scale, "float32"), ("step_ptr", step_ptr, "int64"), ("lr_ptr", lr_ptr, "float32")):
            if t is not None:
                _check_tensors(name, [t], dt, 1)
        lst, buf = self._gradients(grads)
        o = AdamwOptions(lr, beta1, beta2, eps, weight_decay, int(step), 0 if seed is None else int(seed), int(seed is not None),
                         _ptr_or_none(step_ptr), _ptr_or_none(lr_ptr), _ptr_or_none(grad_scale))
        _check(lib().mi_ccl_fusion_adamw(self._h, _CCL_DTYPE[kind], _ptr_array(params), lst, buf, STATE_8BIT if eight else STATE_FP32,
                                         _ptr(exp_avg), _ptr(exp_avg_sq), _ptr_or_none(scales), _ptr_or_none(master), C.byref(o),
                                         _stream(stream)), "mi_ccl_fusion_adamw")

    def _state_tensors(self, exp_avg, exp_avg_sq, scales, values_avg, values_sq):
        _check_tensors("states", [exp_avg, exp_avg_sq], "uint8", self.elements)
        _check_tensors("scales", [scales], "uint8", 2 * ((self.elements + STATE_BLOCK - 1) // STATE_BLOCK))
        _check_tensors("values", [values_avg, values_sq], _dtype_name(values_avg), self.elements)

    def state_decode(self, exp_avg, exp_avg_sq, scales, values_avg, values_sq, stream=None):
        """The values of 8-bit states, float32 or bfloat16."""
        self._state_tensors(exp_avg, exp_avg_sq, scales, values_avg, values_sq)
        _check(lib().mi_ccl_fusion_state_decode(self._h, _ptr(exp_avg), _ptr(exp_avg_sq), _ptr(scales), _CCL_DTYPE[_dtype_name(values_avg)],
                                                _ptr(values_avg), _ptr(values_sq), _stream(stream)), "mi_ccl_fusion_state_decode")

    def state_encode(self, values_avg, values_sq, exp_avg, exp_avg_sq, scales, stream=None):
        """Values (float32 or bfloat16) to 8-bit states, rounded to nearest."""
        self._state_tensors(exp_avg, exp_avg_sq, scales, values_avg, values_sq)
        _check(lib().mi_ccl_fusion_state_encode(self._h, _CCL_DTYPE[_dtype_name(values_avg)], _ptr(values_avg), _ptr(values_sq), _ptr(exp_avg),
                                                _ptr(exp_avg_sq), _ptr(scales), _stream(stream)), "mi_ccl_fusion_state_encode")

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

def _check_rows(what, t, hidden=None, dtype=None):
    """(dtype, elements between rows) of a matrix of rows, whose rows are contiguous."""
    import torch
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (hidden is not None and t.shape[1] != hidden):
        raise ValueError(f"{what}: rows of {'contiguous' if hidden is None else hidden} elements are wanted, got {tuple(t.shape)}, strides {t.stride()}")
    if not t.is_cuda or t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what}: on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    name = _dtype_name(t)
    if dtype is not None and name != dtype:
        raise ValueError(f"{what}: {name}, {dtype} is wanted")
    # one row, or none, has no distance to the next
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if t.shape[0] > 1 and ld < t.shape[1]:
        raise ValueError(f"{what}: rows overlap (strides {t.stride()})")
    return name, ld


def token_rows(n_tokens, top_k, n_experts, align=1, capacity=0):
    """Most rows that the sorted buffer can take."""
    r = C.c_size_t()
    _check(lib().mi_ccl_token_rows(n_tokens, top_k, n_experts, align, capacity, C.byref(r)), "mi_ccl_token_rows")
    return r.value


def token_sort_workspace(n_tokens, top_k, n_experts):
    r = C.c_size_t()
    _check(lib().mi_ccl_token_sort_workspace(n_tokens, top_k, n_experts, C.byref(r)), "mi_ccl_token_sort_workspace")
    return r.value


def token_sort(expert_ids, n_experts, positions, counts, offsets, align=1, capacity=0, workspace=None, stream=None):
    """Row of every entry of expert_ids [tokens, top_k] (int32 or int64) in the buffer sorted by expert, into positions (int32,
    the same shape; -1: none); rows of each expert into counts, first rows and the end into offsets [n_experts + 1] (int32).
    workspace: token_sort_workspace bytes; allocated for the call when None."""
    import torch
    if expert_ids.dim() != 2 or tuple(positions.shape) != tuple(expert_ids.shape):
        raise ValueError("expert_ids and positions are [tokens, top_k]")
    n, k = expert_ids.shape
    _check_tensors("expert_ids", [expert_ids])
    _check_tensors("positions", [positions], "int32")
    _check_tensors("counts", [counts], "int32", n_experts)
    _check_tensors("offsets", [offsets], "int32", n_experts + 1)
    if workspace is None:
        need = token_sort_workspace(n, k, n_experts)
        workspace = torch.empty(need, dtype=torch.uint8, device=expert_ids.device) if need else None
    size = 0
    if workspace is not None:
        _check_tensors("workspace", [workspace])
        size = workspace.numel() * workspace.element_size()
    _check(lib().mi_ccl_token_sort(_CCL_DTYPE.get(_dtype_name(expert_ids), -1), _ptr(expert_ids), n, k, n_experts, align, capacity,
                                   _ptr(positions), _ptr(counts), _ptr(offsets), _ptr_or_none(workspace), size, _stream(stream)),
           "mi_ccl_token_sort")


def _check_segments(positions, counts, offsets, tokens):
    _check_tensors("positions", [positions], "int32")
    if positions.dim() != 2 or positions.shape[0] != tokens:
        raise ValueError(f"positions: [{tokens}, top_k] is wanted, got {tuple(positions.shape)}")
    if counts is not None:
        _check_tensors("counts", [counts], "int32")
        _check_tensors("offsets", [offsets], "int32", counts.numel() + 1)


def token_dispatch(x, positions, counts, offsets, out, stream=None):
    """out[positions[t, j]] = x[t]; padding rows become zero, rows behind the last expert's stay as they are."""
    kind, ldx = _check_rows("x", x)
    _, ldo = _check_rows("out", out, x.shape[1], kind)
    _check_segments(positions, counts, offsets, x.shape[0])
    _check(lib().mi_ccl_token_dispatch(_CCL_DTYPE.get(kind, -1), _ptr(x), ldx, x.shape[0], positions.shape[1], x.shape[1], _ptr(positions),
                                       _ptr(counts), _ptr(offsets), counts.numel(), _ptr(out), ldo, out.shape[0], _stream(stream)),
           "mi_ccl_token_dispatch")


def token_combine(y, positions, weights, out, stream=None):
    """out[t] = sum over j of weights[t, j] * y[positions[t, j]]; weights (float32, the shape of positions) may be None for ones."""
    kind, ldy = _check_rows("y", y)
    _, ldo = _check_rows("out", out, y.shape[1], kind)
    _check_segments(positions, None, None, out.shape[0])
    if weights is not None:
        _check_tensors("weights", [weights], "float32", positions.numel())
    _check(lib().mi_ccl_token_combine(_CCL_DTYPE.get(kind, -1), _ptr(y), ldy, y.shape[0], _ptr(positions), _ptr_or_none(weights),
                                      out.shape[0], positions.shape[1], y.shape[1], _ptr(out), ldo, _stream(stream)), "mi_ccl_token_combine")


def token_combine_backward(grad_out, y, positions, weights, counts, offsets, grad_y, grad_weights=None, stream=None):
    """The gradient of token_combine: grad_y[positions[t, j]] = weights[t, j] * grad_out[t], with padding rows zero, and unless
    None grad_weights[t, j] = <grad_out[t], y[positions[t, j]]>.  y may be None without grad_weights."""
    kind, ldg = _check_rows("grad_out", grad_out)
    hidden = grad_out.shape[1]
    _, ldd = _check_rows("grad_y", grad_y, hidden, kind)
    ldy = hidden
    if y is not None:
        _, ldy = _check_rows("y", y, hidden, kind)
        if y.shape[0] != grad_y.shape[0]:
            raise ValueError(f"y has {y.shape[0]} rows, grad_y {grad_y.shape[0]}")
    elif grad_weights is not None:
        raise ValueError("grad_weights needs y")
    _check_segments(positions, counts, offsets, grad_out.shape[0])
    for name, t in (("weights", weights), ("grad_weights", grad_weights)):
        if t is not None:
            _check_tensors(name, [t], "float32", positions.numel())
    _check(lib().mi_ccl_token_combine_backward(_CCL_DTYPE.get(kind, -1), _ptr(grad_out), ldg, _ptr_or_none(y), ldy, grad_y.shape[0],
                                               _ptr(positions), _ptr_or_none(weights), _ptr(counts), _ptr(offsets), counts.numel(),
                                               grad_out.shape[0], positions.shape[1], hidden, _ptr(grad_y), ldd,
                                               _ptr_or_none(grad_weights), _stream(stream)), "mi_ccl_token_combine_backward")


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


def get_param(name):
    return lib().mi_ccl_get_param(name.encode())
