"""ctypes binding of libtwg_hip.so (the C ABI declared in include/twg.h).

This is the stub a host language binds the kernel library with; the torch
extension (torch_webgpu._C) links the same symbols directly.  It is independent
of torch_webgpu._C so the kernels can be driven, tested and timed without the
dispatcher in the way.  There is no CPU fallback: if the library is missing or a
call fails, an exception is raised.
"""
import collections
import ctypes
import os
import struct

# torch bundles its own HIP runtime under the same SONAME as /opt/rocm's; it has to
# be the first one loaded into the process or two runtimes end up side by side.
import torch
from torch.autograd.graph import increment_version

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "torch_webgpu", "libtwg_hip.so")
MAX_DIMS = 8
OUT, A, B = 0, 1, 2

UNARY_COPY, UNARY_RELU, UNARY_GELU_ERF, UNARY_GELU_TANH, UNARY_SILU, UNARY_ABS = 0, 1, 2, 3, 4, 5
# enum twg_dtype, keyed by torch dtype
DTYPES = {torch.bool: 0, torch.uint8: 1, torch.int32: 2, torch.int64: 3, torch.float16: 4,
          torch.bfloat16: 5, torch.float32: 6, torch.float64: 7, torch.int8: 8, torch.int16: 9}

E_INVALID_ARG, E_UNSUPPORTED, E_SCRATCH_SMALL = -1, -2, -3
E_TOO_LARGE = -5
E_BUSY, E_WAIT_ABANDONED = -6, -7
MS_STATIC_MAX_NUMEL = 1 << 30


class TwgError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"libtwg_hip: {msg} (code {code})")
        self.code = code


class Iter(ctypes.Structure):
    """twg_iter_t: dimension 0 fastest, strides in elements."""
    _fields_ = [
        ("ndim", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("numel", ctypes.c_int64),
        ("shape", ctypes.c_int64 * MAX_DIMS),
        ("stride", (ctypes.c_int64 * MAX_DIMS) * 3),
    ]


class MemStats(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in
                ("bytes_in_use", "bytes_cached", "n_device_mallocs", "n_cache_hits", "n_allocs",
                 "bytes_pending")]


ROPE_MAX_HEAD_DIM, ROPE_MAX_AXES = 512, 8
LOGPROBS_MAX_TOP_K = 64
STREAM_NULL = 1  # TWG_STREAM_NULL: the process's null stream, for the calls on tensors below


class RopePart(ctypes.Structure):
    """twg_rope_part_t: the heads of one tensor, queries or keys."""
    _fields_ = [("heads", ctypes.c_int64)] + [
        (n, ctypes.c_void_p) for n in ("x", "dy", "out", "weight", "dweight")] + [
        (n, ctypes.c_int64 * 3) for n in ("x_stride", "dy_stride", "out_stride")]


class NormRope(ctypes.Structure):
    """twg_norm_rope_t"""
    _fields_ = [(n, ctypes.c_int32) for n in ("dtype", "weight_dtype", "position_dtype", "norm", "adjacent", "n_axes",
                                              "head_dim", "rot_dim")] + [
        ("eps", ctypes.c_float), ("reserved", ctypes.c_int32), ("batch", ctypes.c_int64), ("tokens", ctypes.c_int64),
        ("positions", ctypes.c_void_p), ("pos_stride", ctypes.c_int64 * 3), ("inv_freq", ctypes.c_void_p),
        ("pair_axis", ctypes.c_uint8 * (ROPE_MAX_HEAD_DIM // 2)), ("part", RopePart * 2)]


class TokenLogprobsArgs(ctypes.Structure):
    """twg_token_logprobs_t"""
    _fields_ = [("dtype", ctypes.c_int32), ("target_dtype", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("vocab", ctypes.c_int64), ("row_stride", ctypes.c_int64), ("logits", ctypes.c_void_p),
                ("targets", ctypes.c_void_p), ("ignore_index", ctypes.c_int64), ("scale", ctypes.c_float),
                ("top_k", ctypes.c_int32)] + [
        (n, ctypes.c_void_p) for n in ("logprob", "entropy", "row_max", "row_sum", "top_logprobs", "top_ids", "g_logprob",
                                       "g_entropy", "grad")] + [("grad_stride", ctypes.c_int64)]


# Every symbol include/twg.h declares; tests check that the library exports them all.
SYMBOLS = [
    "twg_init", "twg_is_initialized", "twg_error_string", "twg_device_info",
    "twg_default_stream", "twg_stream_sync", "twg_device_sync",
    "twg_event_create", "twg_event_destroy", "twg_event_record", "twg_event_sync",
    "twg_event_elapsed_ms",
    "twg_malloc", "twg_free", "twg_record_stream", "twg_empty_cache", "twg_mem_stats",
    "twg_memcpy_h2d", "twg_memcpy_d2h", "twg_memcpy_d2d", "twg_fill_bytes",
    "twg_add_f32", "twg_add_scalar_f32", "twg_mul_f32", "twg_mul_scalar_f32",
    "twg_add_relu_f32", "twg_unary_f32", "twg_copy_strided", "twg_cast",
    "twg_eq_f32", "twg_ne_scalar_f32", "twg_and_u8",
    "twg_masked_select_scratch_bytes", "twg_masked_select_f32", "twg_masked_select_count",
    "twg_masked_select_f32_static", "twg_masked_select_f32_wait_probe",
    "twg_eq", "twg_ne_scalar", "twg_and", "twg_abs",
    "twg_norm_rope", "twg_norm_rope_backward", "twg_norm_rope_backward_scratch_bytes",
    "twg_token_logprobs", "twg_token_logprobs_scratch_bytes", "twg_token_logprobs_backward",
    "twg_dropout",
]

_lib = None


def load():
    """dlopen the library and declare prototypes.  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python torch-webgpu_amd/build.py hip` "
            "(there is no fallback path)")
    L = ctypes.CDLL(LIB_PATH)
    vp, i64, i32, f32, sz = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float,
                             ctypes.c_size_t)
    ip = ctypes.POINTER(Iter)
    L.twg_init.argtypes = []
    L.twg_is_initialized.argtypes = []
    L.twg_error_string.argtypes = [ctypes.c_int]
    L.twg_error_string.restype = ctypes.c_char_p
    L.twg_device_info.argtypes = [ctypes.c_char_p, sz, ctypes.POINTER(i32), ctypes.POINTER(i64)]
    L.twg_default_stream.argtypes = []
    L.twg_default_stream.restype = vp
    L.twg_stream_sync.argtypes = [vp]
    L.twg_device_sync.argtypes = []
    L.twg_event_create.argtypes = [ctypes.POINTER(vp)]
    L.twg_event_destroy.argtypes = [vp]
    L.twg_event_record.argtypes = [vp, vp]
    L.twg_event_sync.argtypes = [vp]
    L.twg_event_elapsed_ms.argtypes = [ctypes.POINTER(f32), vp, vp]
    L.twg_malloc.argtypes = [ctypes.POINTER(vp), sz]
    L.twg_free.argtypes = [vp]
    L.twg_record_stream.argtypes = [vp, vp]
    L.twg_empty_cache.argtypes = []
    L.twg_mem_stats.argtypes = [ctypes.POINTER(MemStats)]
    L.twg_memcpy_h2d.argtypes = [vp, vp, sz, vp]
    L.twg_memcpy_d2h.argtypes = [vp, vp, sz, vp]
    L.twg_memcpy_d2d.argtypes = [vp, vp, sz, vp]
    L.twg_fill_bytes.argtypes = [vp, ctypes.c_int, sz, vp]
    L.twg_add_f32.argtypes = [vp, vp, vp, f32, ip, vp]
    L.twg_add_scalar_f32.argtypes = [vp, vp, f32, f32, ip, vp]
    L.twg_mul_f32.argtypes = [vp, vp, vp, ip, vp]
    L.twg_mul_scalar_f32.argtypes = [vp, vp, f32, ip, vp]
    L.twg_add_relu_f32.argtypes = [vp, vp, vp, ip, vp]
    L.twg_unary_f32.argtypes = [ctypes.c_int, vp, vp, ip, vp]
    L.twg_copy_strided.argtypes = [vp, vp, i32, ip, vp]
    L.twg_cast.argtypes = [vp, i32, vp, i32, ip, vp]
    L.twg_eq_f32.argtypes = [vp, vp, vp, ip, vp]
    L.twg_ne_scalar_f32.argtypes = [vp, vp, f32, ip, vp]
    L.twg_and_u8.argtypes = [vp, vp, vp, ip, vp]
    L.twg_masked_select_scratch_bytes.argtypes = [i64]
    L.twg_masked_select_scratch_bytes.restype = sz
    L.twg_masked_select_f32.argtypes = [vp, vp, vp, vp, ip, vp, sz, vp]
    L.twg_masked_select_f32_static.argtypes = [vp, vp, vp, vp, ip, vp]
    L.twg_masked_select_f32_wait_probe.argtypes = [vp, vp, vp, vp, ip, vp, sz, ctypes.c_uint32,
                                                   ctypes.c_uint32, vp]
    L.twg_masked_select_count.argtypes = [vp, ctypes.POINTER(ctypes.c_int64), vp, i32, vp, ip, vp, sz, vp]
    L.twg_eq.argtypes = [vp, vp, vp, i32, ip, vp]
    L.twg_ne_scalar.argtypes = [vp, vp, i32, ctypes.c_double, i64, ip, vp]
    L.twg_and.argtypes = [vp, vp, vp, i32, ip, vp]
    L.twg_abs.argtypes = [vp, vp, i32, ip, vp]
    # (argument structures: a byref, or the packed bytes that the functions on tensors build)
    rp, lp, u64 = vp, vp, ctypes.c_uint64
    L.twg_norm_rope.argtypes = [rp, vp]
    L.twg_norm_rope_backward.argtypes = [rp, vp, sz, vp]
    L.twg_norm_rope_backward_scratch_bytes.argtypes = [rp]
    L.twg_norm_rope_backward_scratch_bytes.restype = sz
    L.twg_token_logprobs.argtypes = [lp, vp, sz, vp]
    L.twg_token_logprobs_scratch_bytes.argtypes = [lp]
    L.twg_token_logprobs_scratch_bytes.restype = sz
    L.twg_token_logprobs_backward.argtypes = [lp, vp]
    L.twg_dropout.argtypes = [vp, vp, vp, i32, ctypes.c_double, u64, u64, vp, ip, vp]
    _lib = L
    return L


def check(code):
    if code != 0:
        raise TwgError(code, load().twg_error_string(code).decode())


def init():
    check(load().twg_init())


def device_info():
    name = ctypes.create_string_buffer(256)
    cus, mem = ctypes.c_int32(), ctypes.c_int64()
    check(load().twg_device_info(name, 256, ctypes.byref(cus), ctypes.byref(mem)))
    return name.value.decode(), cus.value, mem.value


def sync():
    check(load().twg_stream_sync(None))


def mem_stats():
    st = MemStats()
    check(load().twg_mem_stats(ctypes.byref(st)))
    return {n: getattr(st, n) for n, _ in MemStats._fields_}


# ---------------------------------------------------------------- geometry

def make_iter(shape, strides_out, strides_a, strides_b=None):
    """Build a twg_iter_t from LOGICAL (row-major, last dimension fastest) shape and
    element strides: dimensions are reversed so that dimension 0 is the fastest."""
    n = len(shape)
    if n > MAX_DIMS:
        raise ValueError("more than 8 dimensions")
    it = Iter()
    it.ndim = n
    numel = 1
    for d in range(n):
        ld = n - 1 - d
        it.shape[d] = shape[ld]
        numel *= shape[ld]
        it.stride[OUT][d] = strides_out[ld] if strides_out is not None else 0
        it.stride[A][d] = strides_a[ld]
        it.stride[B][d] = strides_b[ld] if strides_b is not None else 0
    it.numel = numel
    return it


def dense_iter(numel):
    it = Iter()
    it.ndim = 1
    it.numel = numel
    it.shape[0] = numel
    for o in range(3):
        it.stride[o][0] = 1
    return it


# ------------------------------------------------------------ device memory

_DTYPE_SIZE = {torch.float32: 4, torch.bool: 1, torch.uint8: 1, torch.int64: 8, torch.int32: 4}


class DeviceBuffer:
    """A block from the library's caching allocator (twg_malloc / twg_free)."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        p = ctypes.c_void_p()
        check(load().twg_malloc(ctypes.byref(p), self.nbytes))
        self.ptr = p.value or 0

    def free(self):
        if self.ptr:
            check(load().twg_free(self.ptr))
            self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def at(self, byte_offset):
        return ctypes.c_void_p(self.ptr + byte_offset)

    def upload(self, t, byte_offset=0):
        """Copy the raw storage bytes of a contiguous CPU tensor to the device."""
        assert t.device.type == "cpu" and t.is_contiguous()
        nbytes = t.numel() * t.element_size()
        assert byte_offset + nbytes <= self.nbytes
        check(load().twg_memcpy_h2d(self.ptr + byte_offset, t.data_ptr(), nbytes, None))

    def download(self, shape, dtype, byte_offset=0):
        t = torch.empty(shape, dtype=dtype)
        nbytes = t.numel() * t.element_size()
        assert byte_offset + nbytes <= self.nbytes
        check(load().twg_memcpy_d2h(t.data_ptr(), self.ptr + byte_offset, nbytes, None))
        return t


def to_device(t):
    """Upload a contiguous CPU tensor; returns a DeviceBuffer holding its bytes."""
    t = t.contiguous()
    buf = DeviceBuffer(max(t.numel() * t.element_size(), 1))
    if t.numel():
        buf.upload(t)
    return buf


def upload_storage(t):
    """Upload the whole storage behind a (possibly strided) CPU tensor; returns the
    buffer and the byte offset of the tensor's first element."""
    st = t.untyped_storage()
    flat = torch.empty(0, dtype=torch.uint8).set_(st)
    buf = DeviceBuffer(max(st.nbytes(), 1))
    if st.nbytes():
        buf.upload(flat)
    return buf, t.storage_offset() * t.element_size()


# ------------------------------------------------------------------ events

class Event:
    def __init__(self):
        e = ctypes.c_void_p()
        check(load().twg_event_create(ctypes.byref(e)))
        self.ev = e

    def record(self):
        check(load().twg_event_record(self.ev, None))

    def sync(self):
        check(load().twg_event_sync(self.ev))

    def elapsed_ms(self, stop):
        ms = ctypes.c_float()
        check(load().twg_event_elapsed_ms(ctypes.byref(ms), self.ev, stop.ev))
        return ms.value

    def __del__(self):
        try:
            load().twg_event_destroy(self.ev)
        except Exception:
            pass


# ------------------------------------------------- steps of a transformer layer, on tensors
#
# The same entry points called on torch tensors whose memory the GPU addresses: tensors of the
# "webgpu" device (the work goes to the library's stream) or of PyTorch-ROCm's device 0 (it goes
# to torch's current stream, so it is ordered with torch's own products there and can be
# captured with them).  Results and scratch are allocated with torch on the same device.
# Arguments are checked here; what the library refuses raises TwgError.  Nothing is recorded for autograd:
# an input that requires grad is refused while gradients are recorded, so that none is lost in silence
# (call under torch.no_grad(), or in a torch.autograd.Function whose backward calls the _backward form);
# a tensor that is written to has its version counted, as after torch's own in-place operators.

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_POSITIONS = (torch.int32, torch.int64, torch.float32)

# twg_norm_rope_t, twg_rope_part_t and twg_token_logprobs_t, packed in one go: setting the fields of
# a ctypes structure one by one costs more than the rest of a call
_ROPE_HEAD = struct.Struct("@8if i 2q P 3q P %ds" % (ROPE_MAX_HEAD_DIM // 2))
_ROPE_PART = struct.Struct("@q 5P 9q")
_NO_PART = bytes(_ROPE_PART.size)
_LOGPROBS = struct.Struct("@2i 3q 2P q f i 9P q")


def _stream_for(t):
    """The stream argument for work on t."""
    if t.is_cuda:
        if t.get_device() != 0:
            raise ValueError("the library is bound to device 0")
        return torch._C._cuda_getCurrentRawStream(0) or STREAM_NULL  # torch.cuda.current_stream() takes 2 us
    if t.device.type != "webgpu":
        raise ValueError(f"expected a tensor in GPU memory, got {t.device}")
    return None


def _same_device(first, *others):
    if first.is_cuda:  # (cheaper than comparing devices)
        for t in others:
            if t is not None and not (t.is_cuda and t.get_device() == 0):
                raise ValueError("all tensors must be on one device")
        return
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")


def _refuse_unrecorded():
    raise ValueError("no gradient is recorded here for a tensor that requires grad: call under torch.no_grad(), "
                     "or in a torch.autograd.Function with the _backward form")


def _written(t):
    if t is not None and not t.is_inference():
        increment_version(t)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _norm_rope_head(q, k, positions, inv_freq, q_weight, k_weight, eps, pair_axis, adjacent):
    """The checked arguments that the forward and the backward call share, packed."""
    dtype = q.dtype
    if q.dim() != 4 or dtype not in _FLOATS:
        raise ValueError("q must be [batch, tokens, heads, head_dim] of float16, bfloat16 or float32")
    B, T, _, D = q.shape
    if k is not None:
        ks = k.shape
        if len(ks) != 4 or ks[0] != B or ks[1] != T or ks[3] != D or k.dtype != dtype:
            raise ValueError("k must have q's dtype and shape up to the number of heads")
    _same_device(q, k, positions, inv_freq, q_weight, k_weight)
    pairs = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if pairs < 0 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float32 vector, one entry per rotated pair")
    if 2 * pairs > D or D > ROPE_MAX_HEAD_DIM:
        raise ValueError("more pairs than the head has, or a head beyond 512 elements")
    ps, st, pt = positions.shape, positions.stride(), positions.dtype
    nd = len(ps)
    if not 1 <= nd <= 3 or pt not in _POSITIONS or ps[-1] != T or (nd > 1 and ps[-2] != B):
        raise ValueError("positions must be [tokens], [batch, tokens] or [axes, batch, tokens] of int32, int64 or float32")
    axes = ps[0] if nd == 3 else 1
    if not 1 <= axes <= ROPE_MAX_AXES:
        raise ValueError("1 to 8 position axes")
    if pair_axis is None:
        if axes != 1 and pairs:
            raise ValueError("several position axes need pair_axis")
    elif len(pair_axis) != pairs:
        raise ValueError("pair_axis must name an axis for each rotated pair")
    if eps is not None and not 0.0 <= eps <= 3.4e38:
        raise ValueError("eps must be finite and not negative")
    weight_dtype = dtype
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if eps is None:
            raise ValueError("weights without a norm (eps is None)")
        if w.shape != (D,) or not w.is_contiguous() or (w.dtype != dtype and w.dtype != torch.float32):
            raise ValueError("a norm weight must be a contiguous vector [head_dim] of q's dtype or float32")
        weight_dtype = w.dtype
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("norm weights of two dtypes")
    return _ROPE_HEAD.pack(DTYPES[dtype], DTYPES[weight_dtype], DTYPES[pt], eps is not None, bool(adjacent), axes, D, 2 * pairs,
                           0.0 if eps is None else eps, 0, B, T, positions.data_ptr(), st[0] if nd == 3 else 0,
                           st[-2] if nd > 1 else 0, st[-1], inv_freq.data_ptr(), b"" if pair_axis is None else bytes(pair_axis))


def _dense_heads(x):
    """x, or a copy of it, with unit stride along the last dimension."""
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, pair_axis=None, adjacent=False,
              q_out=None, k_out=None):
    """RMS norm of every head of q and k and rotation by position: (q_out, k_out).

    q, k: [batch, tokens, heads, head_dim], any strides (views of a packed projection, heads
    first); k may be None.  eps=None leaves the norm out.  positions: [tokens], [batch, tokens]
    or [axes, batch, tokens]; inv_freq: one frequency per rotated pair (2 * len(inv_freq) elements of
    a head are rotated, the rest passes through); pair_axis: for each pair the position axis it
    follows (bytes or a list).  adjacent: pairs are neighbours (2i, 2i + 1) instead of halves.
    q_out / k_out: where the results go (unit stride along head_dim); q and k themselves for a
    call in place, and no other memory that the call reads or writes."""
    stream = _stream_for(q)
    if torch.is_grad_enabled() and (  # (written out: a loop over the tensors takes longer)
            q.requires_grad or inv_freq.requires_grad or positions.requires_grad or (k is not None and k.requires_grad)
            or (q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad)
            or (q_out is not None and q_out.requires_grad) or (k_out is not None and k_out.requires_grad)):
        _refuse_unrecorded()
    args = _norm_rope_head(q, k, positions, inv_freq, q_weight, k_weight, eps, pair_axis, adjacent)
    outs, keep = [], []
    for x, w, out in ((q, q_weight, q_out), (k, k_weight, k_out)):
        if x is None:
            if out is not None:
                raise ValueError("an output without its input")
            args += _NO_PART
            outs.append(None)
            continue
        shape, strides = x.shape, x.stride()
        H, D = shape[2:]
        if strides[3] != 1 and D != 1:
            x = x.contiguous()
            strides = x.stride()
        if out is None:
            out = x.new_empty(shape)
            to = (shape[1] * H * D, H * D, D)
        else:
            _same_device(x, out)
            to = out.stride()
            if out.shape != shape or out.dtype != x.dtype or (to[3] != 1 and D != 1):
                raise ValueError("an output must have its input's shape and dtype and unit stride along head_dim")
        args += _ROPE_PART.pack(H, x.data_ptr(), 0, out.data_ptr(), _ptr(w), 0, *strides[:3], 0, 0, 0, *to[:3])
        keep.append(x)
        outs.append(out)
    check(load().twg_norm_rope(args, stream))
    _written(q_out)
    _written(k_out)
    return tuple(outs)


def norm_rope_backward(dq, dk, q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, pair_axis=None,
                       adjacent=False):
    """Gradients of norm_rope for the incoming gradients dq and dk of its results:
    (grad q, grad k, grad q_weight, grad k_weight), None for what the call does not have."""
    stream = _stream_for(q)
    if torch.is_grad_enabled() and ((dq is not None and dq.requires_grad) or (dk is not None and dk.requires_grad)):
        _refuse_unrecorded()
    args = _norm_rope_head(q, k, positions, inv_freq, q_weight, k_weight, eps, pair_axis, adjacent)
    grads, keep = [None] * 4, []
    for i, (x, dy, w) in enumerate(((q, dq, q_weight), (k, dk, k_weight))):
        if x is None:
            if dy is not None:
                raise ValueError("a gradient without its input")
            args += _NO_PART
            continue
        _same_device(x, dy)
        if dy is None or dy.shape != x.shape or dy.dtype != x.dtype:
            raise ValueError("an incoming gradient must have its input's shape and dtype")
        x, dy = _dense_heads(x), _dense_heads(dy)
        keep.append((x, dy))
        g = grads[i] = x.new_empty(x.shape)
        gw = 0
        if w is not None:
            grads[2 + i] = w.new_empty(w.shape)
            gw = grads[2 + i].data_ptr()
        args += _ROPE_PART.pack(x.shape[2], x.data_ptr(), dy.data_ptr(), g.data_ptr(), _ptr(w), gw, *x.stride()[:3],
                                *dy.stride()[:3], *g.stride()[:3])
    L = load()
    need = L.twg_norm_rope_backward_scratch_bytes(args)
    scratch = q.new_empty(need // 4, dtype=torch.float32) if need else None
    check(L.twg_norm_rope_backward(args, _ptr(scratch), need, stream))
    return tuple(grads)


TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprob entropy row_max row_sum top_logprobs top_ids")


def _rows(logits):
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


def _check_rows(logits, targets, scale):
    if not 0.0 < scale <= 3.4e38:
        raise ValueError("scale must be positive and finite")
    if logits.dim() != 2 or logits.dtype not in _FLOATS:
        raise ValueError("logits must be [rows, vocab] of float16, bfloat16 or float32")
    if targets.shape != logits.shape[:1] or targets.dtype not in (torch.int32, torch.int64) or not targets.is_contiguous():
        raise ValueError("targets must be a contiguous int32 or int64 vector, one per row")
    _same_device(logits, targets)


def token_logprobs(logits, targets, top_k=0, scale=1.0, ignore_index=-100):
    """TokenLogprobs of logits [rows, vocab] and one given token per row: its log probability
    (0 where the token is ignore_index), the row's entropy, the maximum and sum that the backward
    call takes, and the top_k alternatives (ties: the lowest id first), all float32 but the
    int64 ids.  scale multiplies the logits (one over the temperature); -inf logits are masked."""
    stream = _stream_for(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        _refuse_unrecorded()
    _check_rows(logits, targets, scale)
    logits = _rows(logits)
    rows, vocab = logits.shape
    if not 0 <= top_k <= min(LOGPROBS_MAX_TOP_K, vocab):
        raise ValueError("top_k must be in 0..min(64, vocab)")
    stats = logits.new_empty((4, rows), dtype=torch.float32)
    top = logits.new_empty((rows, top_k), dtype=torch.float32)
    ids = logits.new_empty((rows, top_k), dtype=torch.int64)
    base, row = stats.data_ptr(), 4 * rows
    args = _LOGPROBS.pack(DTYPES[logits.dtype], DTYPES[targets.dtype], rows, vocab, logits.stride(0), logits.data_ptr(),
                          targets.data_ptr(), ignore_index, scale, top_k, base, base + row, base + 2 * row, base + 3 * row,
                          top.data_ptr(), ids.data_ptr(), 0, 0, 0, 0)
    L = load()
    need = L.twg_token_logprobs_scratch_bytes(args)
    scratch = logits.new_empty(need // 8, dtype=torch.int64) if need else None
    check(L.twg_token_logprobs(args, _ptr(scratch), need, stream))
    return TokenLogprobs(*stats.unbind(), top, ids)


def token_logprobs_backward(g_logprob, g_entropy, logits, targets, row_max, row_sum, entropy=None, scale=1.0,
                            ignore_index=-100, out=None):
    """Gradient of the logits for the incoming gradients of logprob and entropy (either may be
    None).  row_max, row_sum and entropy come from token_logprobs with the same scale.  out may
    be logits itself, and overlaps nothing else."""
    stream = _stream_for(logits)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (g_logprob, g_entropy, out)):
        _refuse_unrecorded()
    _check_rows(logits, targets, scale)
    src = _rows(logits)
    given = out
    for v in (g_logprob, g_entropy, row_max, row_sum, entropy):
        if v is not None and (v.shape != targets.shape or v.dtype != torch.float32 or not v.is_contiguous()):
            raise ValueError("gradients and statistics must be contiguous float32 vectors, one entry per row")
    _same_device(logits, g_logprob, g_entropy, row_max, row_sum, entropy, out)
    if out is None:
        out = src.new_empty(src.shape)
    elif out.shape != src.shape or out.dtype != src.dtype or (out.stride(1) != 1 and out.shape[1] != 1):
        raise ValueError("out must have the logits' shape and dtype and unit stride along vocab")
    args = _LOGPROBS.pack(DTYPES[src.dtype], DTYPES[targets.dtype], *src.shape, src.stride(0), src.data_ptr(),
                          targets.data_ptr(), ignore_index, scale, 0, 0, _ptr(entropy), _ptr(row_max), _ptr(row_sum), 0, 0,
                          _ptr(g_logprob), _ptr(g_entropy), out.data_ptr(), out.stride(0))
    check(load().twg_token_logprobs_backward(args, stream))
    _written(given)
    return out


def dropout(x, p, seed, offset=0, residual=None, out=None, d_offset=None):
    """residual + dropout(x), or dropout(x): elements are kept by Philox4x32-10 of (seed, offset,
    element index), so the gradient of x is dropout(grad, p, seed, offset) and no mask exists.  Each call of a
    training step takes an offset of its own.  p is rounded to a multiple of 2^-16 (below
    2^-17 nothing is dropped, above 1 - 2^-17 everything).  out may be x or residual itself, and overlaps
    nothing else.  d_offset: an int64 tensor of one element, added to offset when the kernel runs (captured graphs)."""
    stream = _stream_for(x)
    if x.dtype not in _FLOATS:
        raise ValueError("x must be float16, bfloat16 or float32")
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)
                                    or (out is not None and out.requires_grad)):
        _refuse_unrecorded()
    _same_device(x, residual, out, d_offset)
    given = out
    if out is None:
        out = x.new_empty(x.shape)
    for t in (residual, out):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError("x, residual and out must agree in shape and dtype")
    if d_offset is not None and (d_offset.dtype != torch.int64 or d_offset.numel() != 1):
        raise ValueError("d_offset must be one int64")
    if x.is_contiguous() and out.is_contiguous() and (residual is None or residual.is_contiguous()):
        it = dense_iter(x.numel())
    else:
        it = make_iter(x.shape, out.stride(), x.stride(), None if residual is None else residual.stride())
    check(load().twg_dropout(out.data_ptr(), x.data_ptr(), _ptr(residual), DTYPES[x.dtype], p, seed & (2 ** 64 - 1),
                             offset & (2 ** 64 - 1), _ptr(d_offset), ctypes.byref(it), stream))
    _written(given)
    return out
