"""Python binding of the MI355X routed-MoE expert FFN C ABI (include/moe_ffn.h).

This is the host-side operator surface used by the tests and bench.py.  It
mirrors the reference's expert operator (src/gpu_expert.hpp:7-17, the Experts /
Layer::ffn path of src/session.hip:976-1078, 1446-1541): token activations,
top-k expert ids and route weights go in, the routing-weighted FFN output in
token order comes out.  Every call goes through libmoe_ffn.so; there is no
CPU or PyTorch fallback -- a missing library raises.

PyTorch is only used to own device memory and streams.
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmoe_ffn.so")
ROOT = os.path.dirname(HERE)
HEADER = os.path.join(ROOT, "include", "moe_ffn.h")

Q8_BLOCK = 36
Q4_BLOCK = 18
Q4_1_BLOCK = 20
DOWN_Q4_0, DOWN_Q4_1 = 0, 1     # MOE_DOWN_Q4_0 / MOE_DOWN_Q4_1
PATH_AUTO, PATH_STREAM, PATH_MFMA = 0, 1, 2
TYPE_Q4_0, TYPE_Q4_1 = 2, 3     # MOE_TYPE_Q4_0 / MOE_TYPE_Q4_1 (the reference's TensorType ids)
F32, BF16, F16 = 0, 1, 2        # MOE_F32 / MOE_BF16 / MOE_F16
GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_ELEMENT = 0, 1, 2, 3   # MOE_GATE_*
SUMS_AUTO, SUMS_F32 = 0, 1      # MOE_SUMS_*
E4M3_GROUP = 128                # elements per scale of an e4m3 row
STAGE_PREPARE, STAGE_GATE_UP, STAGE_DOWN, STAGE_FOLD = 0, 1, 2, 3


class MoeError(RuntimeError):
    def __init__(self, what, status):
        super().__init__(f"{what} failed with status {status}")
        self.status = status


class Config(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int), ("intermediate", ctypes.c_int), ("experts", ctypes.c_int),
                ("top_k", ctypes.c_int), ("has_shared", ctypes.c_int), ("max_tokens", ctypes.c_int),
                ("down_type", ctypes.c_int)]


class Fp8LayerConfig(ctypes.Structure):
    """moe_fp8_layer_config."""
    _fields_ = [("hidden", ctypes.c_int), ("intermediate", ctypes.c_int), ("experts", ctypes.c_int),
                ("top_k", ctypes.c_int), ("has_shared", ctypes.c_int), ("max_tokens", ctypes.c_int)]


class Fp8Matrix(ctypes.Structure):
    """moe_fp8_matrix."""
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


class I8LayerConfig(ctypes.Structure):
    """moe_i8_layer_config."""
    _fields_ = [("hidden", ctypes.c_int), ("intermediate", ctypes.c_int), ("experts", ctypes.c_int),
                ("top_k", ctypes.c_int), ("has_shared", ctypes.c_int), ("max_tokens", ctypes.c_int)]


class I8Matrix(ctypes.Structure):
    """moe_i8_matrix."""
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


class BlockNormArgs(ctypes.Structure):
    """moe_block_norm_args."""
    _fields_ = ([(n, ctypes.c_int) for n in ("hidden", "tokens", "type", "residual_type")] +
                [(n, ctypes.c_float) for n in ("eps", "weight_offset", "residual_scale", "block_scale")] +
                [("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64), ("block", ctypes.c_void_p),
                 ("block_stride", ctypes.c_int64), ("post_weight", ctypes.c_void_p), ("gate", ctypes.c_void_p),
                 ("gate_stride", ctypes.c_int64), ("gate_form", ctypes.c_int), ("gate_sigmoid", ctypes.c_int),
                 ("residual_out", ctypes.c_void_p), ("residual_out_stride", ctypes.c_int64),
                 ("pre_weight", ctypes.c_void_p), ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64),
                 ("q8", ctypes.c_void_p), ("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                 ("error", ctypes.c_void_p)])


class ExpertTiming(ctypes.Structure):
    """moe_expert_timing (ExpertTiming, src/gpu_expert.hpp:6)."""
    _fields_ = [("upload_ms", ctypes.c_double), ("resident_ms", ctypes.c_double),
                ("completed_wall_ms", ctypes.c_double)]


_lib = None
_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_int64


def library():
    """Load libmoe_ffn.so (built in-tree by __graft_entry__.build())."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"HIP extension missing: {LIB_PATH}; run __graft_entry__.build()")
        lib = ctypes.CDLL(LIB_PATH)
        lib.moe_ffn_create.argtypes = [ctypes.POINTER(Config), _P, _P, _I, ctypes.POINTER(_P)]
        lib.moe_ffn_create_from_device.argtypes = [ctypes.POINTER(Config), _P, _P, _I, ctypes.POINTER(_P)]
        lib.moe_ffn_create_tensors.argtypes = [ctypes.POINTER(Config), _P, _P, _P, _P, _P, _P, _I,
                                               ctypes.POINTER(_P)]
        lib.moe_ffn_create_synthetic.argtypes = [ctypes.POINTER(Config), ctypes.c_uint64, _I, ctypes.POINTER(_P)]
        lib.moe_ffn_destroy.argtypes = [_P]
        lib.moe_ffn_memory_bytes.argtypes = [ctypes.POINTER(Config), ctypes.POINTER(ctypes.c_size_t),
                                             ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_ffn_export_expert.argtypes = [_P, _I, _P]
        lib.moe_ffn_forward.argtypes = [_P, _P, _P, _P, _I, _P, _P, _P, _P]
        lib.moe_ffn_forward_q8.argtypes = [_P, _P, _P, _P, _I, _P, _P, _P, _P]
        lib.moe_quantize_q8_1.argtypes = [_P, _P, _I, _I, _P, _P]
        lib.moe_ffn_group_routes.argtypes = [_P, _P, _P, _I, _P, _P, _P, _P, _P, _P]
        lib.moe_ffn_expert_gate_up.argtypes = [_P, _I, _P, _I, _P, _P, _P, _P, _I, _P, _P]
        lib.moe_ffn_expert_down.argtypes = [_P, _I, _P, _I, _P, _P, _I, _P, _P]
        lib.moe_ffn_expert_run.argtypes = [_P, _I, _P, _I, _P, _I, _I, ctypes.POINTER(_I), ctypes.POINTER(ExpertTiming),
                                           _P]
        lib.moe_combine.argtypes = [_P, _P, _P, _P, _I, _I, _I, _P, _P, _P]
        lib.moe_ffn_debug_last.argtypes = [_P, _P, _P, _P, _P, _P]
        lib.moe_ffn_replay_stage.argtypes = [_P, _I, _P]
        lib.moe_ffn_profile.argtypes = [_P, _I]
        lib.moe_ffn_profile_read.argtypes = [_P, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(_I)]
        lib.moe_expf_device.argtypes = [_P, _P, _I, _P]
        lib.moe_expf_host.argtypes = [_P, _P, ctypes.c_size_t]
        lib.moe_read_probe.argtypes = [_P, ctypes.c_size_t, _P, _P]
        lib.moe_router_select.argtypes = [_P, _I, _I, _I, _P, _P, _P, _P, _P]
        lib.moe_ffn_last_stats.argtypes = [_P, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int32),
                                           ctypes.POINTER(ctypes.c_int32)]
        lib.moe_linear_create.argtypes = [_I, _I, _I, _I, _P, _I, _I, ctypes.POINTER(_P)]
        lib.moe_linear_destroy.argtypes = [_P]
        lib.moe_linear_bytes.argtypes = [_P, ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_linear_forward_q8.argtypes = [_P, _P, _I, _P, _P]
        lib.moe_linear_apply.argtypes = [_P, _P, _I, _P, _P, _P]
        lib.moe_linear_apply_noalloc.argtypes = [_P, _P, _I, _P, _P, _P]
        lib.moe_quantize_e4m3.argtypes = [_P, _I, _L, _I, _I, _P, _P, _P, _P]
        lib.moe_fp8_linear_create.argtypes = [_I, _I, _I, _P, _P, _I, _I, ctypes.POINTER(_P)]
        lib.moe_fp8_linear_destroy.argtypes = [_P]
        lib.moe_fp8_linear_bytes.argtypes = [_P, ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_fp8_linear_set_sums.argtypes = [_P, _I]
        lib.moe_fp8_linear_forward.argtypes = [_P, _P, _P, _I, _P, _I, _L, _P]
        lib.moe_fp8_linear_apply.argtypes = [_P, _P, _I, _L, _I, _P, _I, _L, _P, _P]
        lib.moe_fp8_layer_memory_bytes.argtypes = [ctypes.POINTER(Fp8LayerConfig), ctypes.POINTER(ctypes.c_size_t),
                                                   ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_fp8_layer_create.argtypes = [ctypes.POINTER(Fp8LayerConfig), ctypes.POINTER(Fp8Matrix),
                                             ctypes.POINTER(Fp8Matrix), _I, _I, ctypes.POINTER(_P)]
        lib.moe_fp8_layer_destroy.argtypes = [_P]
        lib.moe_fp8_layer_forward.argtypes = [_P, _P, _I, _P, _P, _I, _P, _P, _P, _P]
        lib.moe_block_norm.argtypes = [ctypes.POINTER(BlockNormArgs), _P]
        lib.moe_quantize_i8.argtypes = [_P, _I, _L, _I, _I, _P, _P, _P, _P]
        lib.moe_i8_linear_create.argtypes = [_I, _I, _I, _P, _P, _I, _I, ctypes.POINTER(_P)]
        lib.moe_i8_linear_destroy.argtypes = [_P]
        lib.moe_i8_linear_bytes.argtypes = [_P, ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_i8_linear_forward.argtypes = [_P, _P, _P, _I, _P, _I, _L, _P]
        lib.moe_i8_linear_apply.argtypes = [_P, _P, _I, _L, _I, _P, _I, _L, _P, _P]
        lib.moe_i8_bank_create.argtypes = [_I, _I, _I, _P, _P, _I, _I, ctypes.POINTER(_P)]
        lib.moe_i8_bank_destroy.argtypes = [_P]
        lib.moe_i8_bank_bytes.argtypes = [_P, ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_i8_bank_forward.argtypes = [_P, _P, _P, _I, _P, _P, _I, _P, _I, _L, _P, _P]
        lib.moe_i8_layer_memory_bytes.argtypes = [ctypes.POINTER(I8LayerConfig), ctypes.POINTER(ctypes.c_size_t),
                                                  ctypes.POINTER(ctypes.c_size_t)]
        lib.moe_i8_layer_create.argtypes = [ctypes.POINTER(I8LayerConfig), ctypes.POINTER(I8Matrix),
                                            ctypes.POINTER(I8Matrix), _I, _I, ctypes.POINTER(_P)]
        lib.moe_i8_layer_destroy.argtypes = [_P]
        lib.moe_i8_layer_forward.argtypes = [_P, _P, _I, _P, _P, _I, _P, _P, _P, _P]
        _lib = lib
    return _lib


def header_symbols():
    """Function names declared in include/moe_ffn.h."""
    import re
    text = open(HEADER).read()
    return sorted(set(re.findall(r"^int\s+(moe_\w+)\s*\(", text, flags=re.M)))


def _check(status, what):
    if status != 0:
        raise MoeError(what, status)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _need(t, name, dtype, shape, device=None):
    """Check a tensor handed to the C ABI: dtype, exact shape, contiguity and
    device.  The ABI takes raw pointers and sizes, so a tensor with fewer rows,
    another element type or a strided view would be read past its end on the
    GPU; the reference's RouteGroups::prepare likewise rejects a size
    mismatch before touching anything (src/routes.cpp:63-68)."""
    import torch
    if t is None:
        raise ValueError(f"{name} is required")
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on {device if device is not None else 'a GPU'}, got {t.device}")
    return t


def _routes_check(ids, weights, n, k, device):
    import torch
    _need(ids, "ids", torch.int32, (n, k), device)
    _need(weights, "weights", torch.float32, (n, k), device)


def _stream(stream):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _making(stream):
    """Context in which a call makes the tensors it was not given: on the stream
    that it launches on, so that an error word's zeros come before the kernels'
    flags and no other stream's pending work still uses the memory."""
    import contextlib
    import torch
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _on_device(device):
    """Context in which `device` is current, for the calls without a handle."""
    import torch
    return torch.cuda.device(device)


def _stream_on(stream, device):
    """The stream handle of a call on tensors of `device`: its current stream
    when none is given."""
    import torch
    s = stream if stream is not None else torch.cuda.current_stream(device)
    return ctypes.c_void_p(s.cuda_stream)


def _elem_type(t, name):
    import torch
    types = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype not in types:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return types[t.dtype]


def _need_rows(t, name, shape, device=None, dtypes=None):
    """Check a matrix whose rows may be further apart than they are long (a
    slice of a wider one): element type, exact shape, unit stride within a row
    and rows that do not run into each other.  Returns (type id, row stride)."""
    type_ = _elem_type(t, name)
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {dtypes}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have consecutive elements within a row")
    stride = t.stride(0) if t.shape[0] > 1 else max(t.shape[1], t.stride(0))
    if stride < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (stride {stride} < {t.shape[1]})")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on {device if device is not None else 'a GPU'}, got {t.device}")
    return type_, stride


def expert_bytes(hidden, intermediate, down_type=DOWN_Q4_0):
    """Canonical bytes of one expert: gate and up Q4_0, down Q4_0 or Q4_1."""
    return hidden // 32 * intermediate * (2 * Q4_BLOCK + (Q4_1_BLOCK if down_type == DOWN_Q4_1 else Q4_BLOCK))


class MoeLayer:
    """One MoE layer resident on the GPU (weights + workspace for max_tokens)."""

    def __init__(self, hidden, intermediate, experts, top_k, has_shared, max_tokens, experts_q4=None,
                 shared_q4=None, synthetic_seed=None, device=0, tensors=None, shared_tensors=None,
                 down_type=DOWN_Q4_0):
        self.cfg = Config(hidden, intermediate, experts, top_k, 1 if has_shared else 0, max_tokens, down_type)
        self.down_type = down_type
        self.H, self.I, self.E, self.k = hidden, intermediate, experts, top_k
        self.has_shared = bool(has_shared)
        self.max_tokens = max_tokens
        self.device = device
        handle = ctypes.c_void_p()
        lib = library()
        if tensors is not None:   # (gate_exps, up_exps, down_exps) host arrays, reference tensor layout
            ts = [np.ascontiguousarray(t, dtype=np.uint8) for t in tensors]
            nb = hidden // 32 * intermediate
            mb = [nb * Q4_BLOCK, nb * Q4_BLOCK, nb * (Q4_1_BLOCK if down_type == DOWN_Q4_1 else Q4_BLOCK)]
            assert all(t.size == experts * m for t, m in zip(ts, mb))
            ss = [None, None, None]
            if has_shared:
                ss = [np.ascontiguousarray(t, dtype=np.uint8) for t in shared_tensors]
                assert all(t.size == m for t, m in zip(ss, mb))
            ptr = lambda a: None if a is None else ctypes.c_void_p(a.ctypes.data)
            st = lib.moe_ffn_create_tensors(ctypes.byref(self.cfg), *[ptr(t) for t in ts], *[ptr(t) for t in ss],
                                            device, ctypes.byref(handle))
        elif synthetic_seed is not None:
            st = lib.moe_ffn_create_synthetic(ctypes.byref(self.cfg), ctypes.c_uint64(synthetic_seed), device,
                                              ctypes.byref(handle))
        elif isinstance(experts_q4, np.ndarray):
            experts_q4 = np.ascontiguousarray(experts_q4, dtype=np.uint8)
            assert experts_q4.size == experts * expert_bytes(hidden, intermediate, down_type)
            sh = None
            if has_shared:
                sh = np.ascontiguousarray(shared_q4, dtype=np.uint8)
                assert sh.size == expert_bytes(hidden, intermediate, down_type)
            st = lib.moe_ffn_create(ctypes.byref(self.cfg), ctypes.c_void_p(experts_q4.ctypes.data),
                                    None if sh is None else ctypes.c_void_p(sh.ctypes.data), device,
                                    ctypes.byref(handle))
        else:   # torch device tensors
            st = lib.moe_ffn_create_from_device(ctypes.byref(self.cfg), _ptr(experts_q4), _ptr(shared_q4), device,
                                                ctypes.byref(handle))
        _check(st, "moe_ffn_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_ffn_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------ queries --
    def export_expert(self, expert):
        out = np.zeros(expert_bytes(self.H, self.I, self.down_type), np.uint8)
        _check(library().moe_ffn_export_expert(self.handle, expert, ctypes.c_void_p(out.ctypes.data)),
               "moe_ffn_export_expert")
        return out

    def last_stats(self):
        a, b, c = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
        _check(library().moe_ffn_last_stats(self.handle, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c)),
               "moe_ffn_last_stats")
        return dict(stream_items=a.value, mfma_items=b.value, active_experts=c.value)

    # ------------------------------------------------------------ forward --
    def _io_check(self, n, dev, ids, weights, shared_gate, y, error, stream=None):
        import torch
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"tokens {n} outside 1..{self.max_tokens}")
        _routes_check(ids, weights, n, self.k, dev)
        if shared_gate is not None:
            _need(shared_gate, "shared_gate", torch.float32, (n,), dev)
        with _making(stream):
            if y is None:
                y = torch.empty((n, self.H), dtype=torch.float32, device=dev)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=dev)
        _need(y, "y", torch.float32, (n, self.H), dev)
        _need(error, "error", torch.int32, (1,), dev)
        return y, error

    def forward(self, x, ids, weights, shared_gate=None, y=None, error=None, stream=None):
        import torch
        n = x.shape[0]
        _need(x, "x", torch.float32, (n, self.H), x.device)
        y, error = self._io_check(n, x.device, ids, weights, shared_gate, y, error, stream)
        _check(library().moe_ffn_forward(self.handle, _ptr(x), _ptr(ids), _ptr(weights), n, _ptr(shared_gate),
                                         _ptr(y), _ptr(error), _stream(stream)), "moe_ffn_forward")
        return y, error

    def bind_forward(self, x, ids, weights, y, error, shared_gate=None, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues that forward with no per-call checks (the
        pointers and the stream handle are resolved here).  For loops that
        time the library rather than the Python checks; the tensors must stay
        alive and keep their shapes while the callable is used."""
        import torch
        n = x.shape[0]
        _need(x, "x", torch.float32, (n, self.H), x.device)
        self._io_check(n, x.device, ids, weights, shared_gate, y, error)
        fn, handle = library().moe_ffn_forward, self.handle
        args = (_ptr(x), _ptr(ids), _ptr(weights), n, _ptr(shared_gate), _ptr(y), _ptr(error), _stream(stream))

        def call():
            st = fn(handle, *args)
            if st != 0:
                raise MoeError("moe_ffn_forward", st)
        return call

    def forward_q8(self, x_q8, ids, weights, shared_gate=None, y=None, error=None, stream=None):
        """forward() from canonical Q8_1 rows x_q8 (uint8 [tokens][H/32*36])."""
        import torch
        n = ids.shape[0]
        _need(x_q8, "x_q8", torch.uint8, (n, self.H // 32 * Q8_BLOCK), ids.device)
        y, error = self._io_check(n, ids.device, ids, weights, shared_gate, y, error, stream)
        _check(library().moe_ffn_forward_q8(self.handle, _ptr(x_q8), _ptr(ids), _ptr(weights), n, _ptr(shared_gate),
                                            _ptr(y), _ptr(error), _stream(stream)), "moe_ffn_forward_q8")
        return y, error

    def replay_stage(self, stage, stream=None):
        _check(library().moe_ffn_replay_stage(self.handle, stage, _stream(stream)), "moe_ffn_replay_stage")

    def profile(self, forwards):
        """Record stage timing events for the next `forwards` forward() calls."""
        _check(library().moe_ffn_profile(self.handle, forwards), "moe_ffn_profile")

    def profile_read(self):
        """(seconds per stage summed over the recorded forwards, count)."""
        ms = (ctypes.c_double * (STAGE_FOLD + 1))()
        n = ctypes.c_int()
        _check(library().moe_ffn_profile_read(self.handle, ms, ctypes.byref(n)), "moe_ffn_profile_read")
        return [v / 1e3 for v in ms], n.value

    def debug_last(self, tokens, stream=None):
        import torch
        P = tokens * self.k + (tokens if self.has_shared else 0)
        dev = f"cuda:{self.device}"
        with _making(stream):
            xq = torch.empty((tokens, self.H // 32 * Q8_BLOCK), dtype=torch.uint8, device=dev)
            mq = torch.empty((P, self.I // 32 * Q8_BLOCK), dtype=torch.uint8, device=dev)
            rt = torch.empty(tokens * self.k, dtype=torch.int32, device=dev)
            rr = torch.empty(tokens * self.k, dtype=torch.int32, device=dev)
        _check(library().moe_ffn_debug_last(self.handle, _ptr(xq), _ptr(mq), _ptr(rt), _ptr(rr), _stream(stream)),
               "moe_ffn_debug_last")
        return dict(x_q8=xq, middle_q8=mq, route_token=rt, route_rank=rr)

    def group_routes(self, ids, weights, stream=None):
        import torch
        n = ids.shape[0]
        dev = ids.device
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"tokens {n} outside 1..{self.max_tokens}")
        _routes_check(ids, weights, n, self.k, dev)
        with _making(stream):
            counts = torch.empty(self.E, dtype=torch.int32, device=dev)
            offsets = torch.empty(self.E + 1, dtype=torch.int32, device=dev)
            rt = torch.empty(n * self.k, dtype=torch.int32, device=dev)
            rr = torch.empty(n * self.k, dtype=torch.int32, device=dev)
            error = torch.zeros(1, dtype=torch.int32, device=dev)
        _check(library().moe_ffn_group_routes(self.handle, _ptr(ids), _ptr(weights), n, _ptr(counts), _ptr(offsets),
                                              _ptr(rt), _ptr(rr), _ptr(error), _stream(stream)),
               "moe_ffn_group_routes")
        return dict(counts=counts, offsets=offsets, token=rt, rank=rr, error=error)

    def expert_gate_up(self, expert, x_q8, columns, path=PATH_AUTO, dots=False, stream=None):
        import torch
        dev = x_q8.device
        gd = ud = None
        with _making(stream):
            middle = torch.empty((columns, self.I), dtype=torch.float32, device=dev)
            mq = torch.empty((columns, self.I // 32 * Q8_BLOCK), dtype=torch.uint8, device=dev)
            if dots:
                gd = torch.full((columns, self.I, self.H // 32), -2**31, dtype=torch.int32, device=dev)
                ud = torch.full((columns, self.I, self.H // 32), -2**31, dtype=torch.int32, device=dev)
            error = torch.zeros(1, dtype=torch.int32, device=dev)
        _check(library().moe_ffn_expert_gate_up(self.handle, expert, _ptr(x_q8), columns, _ptr(middle), _ptr(mq),
                                                _ptr(gd), _ptr(ud), path, _ptr(error), _stream(stream)),
               "moe_ffn_expert_gate_up")
        return dict(middle=middle, middle_q8=mq, gate_dots=gd, up_dots=ud, error=error)

    def expert_down(self, expert, middle_q8, columns, path=PATH_AUTO, dots=False, stream=None):
        import torch
        dev = middle_q8.device
        dd = None
        with _making(stream):
            y = torch.empty((columns, self.H), dtype=torch.float32, device=dev)
            if dots:
                dd = torch.full((columns, self.H, self.I // 32), -2**31, dtype=torch.int32, device=dev)
            error = torch.zeros(1, dtype=torch.int32, device=dev)
        _check(library().moe_ffn_expert_down(self.handle, expert, _ptr(middle_q8), columns, _ptr(y), _ptr(dd), path,
                                             _ptr(error), _stream(stream)), "moe_ffn_expert_down")
        return dict(y=y, down_dots=dd, error=error)

    def expert_run(self, expert, x, repeats, path=PATH_AUTO, stream=None):
        """GpuExpert::run (src/hip/expert.hip:228-241): host float32 x
        [columns][H] through one resident expert's whole forward, `repeats`
        timed forwards.  Returns (y, timing dict, error word); y and timing are
        None when the warm-up forward raised the error word."""
        x = np.ascontiguousarray(x, dtype=np.float32)
        if x.ndim != 2 or x.shape[1] != self.H:
            raise ValueError(f"x: expected [columns][{self.H}] float32, got {x.shape}")
        columns = x.shape[0]
        y = np.empty_like(x)
        flags = _I(0)
        t = ExpertTiming()
        _check(library().moe_ffn_expert_run(self.handle, expert, ctypes.c_void_p(x.ctypes.data), columns,
                                            ctypes.c_void_p(y.ctypes.data), repeats, path, ctypes.byref(flags),
                                            ctypes.byref(t), _stream(stream)), "moe_ffn_expert_run")
        if flags.value:
            return None, None, flags.value
        return y, dict(upload_ms=t.upload_ms, resident_ms=t.resident_ms,
                       completed_wall_ms=t.completed_wall_ms), 0


def expf_host(x):
    """The kernels' expf (moe_expf.h) run on the CPU: float32 array in, out."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(library().moe_expf_host(ctypes.c_void_p(x.ctypes.data), ctypes.c_void_p(y.ctypes.data), x.size),
           "moe_expf_host")
    return y


def expf_device(x, stream=None):
    """The kernels' expf on the GPU: float32 device tensor in, out."""
    import torch
    with _making(stream):
        y = torch.empty_like(x)
    _check(library().moe_expf_device(_ptr(x), _ptr(y), x.numel(), _stream(stream)), "moe_expf_device")
    return y


def router_select(logits, top_k=10, probabilities=False, error=None, stream=None, ids=None, weights=None):
    """Device router: fp32 logits [tokens][experts] -> (ids int32 [tokens][top_k],
    weights fp32 [tokens][top_k], probabilities or None, error).  `ids` /
    `weights` may be given to write into existing tensors."""
    import torch
    n, e = logits.shape
    dev = logits.device
    _need(logits, "logits", torch.float32, (n, e), dev)
    with _making(stream):
        if ids is None:
            ids = torch.empty((n, top_k), dtype=torch.int32, device=dev)
        w = weights if weights is not None else torch.empty((n, top_k), dtype=torch.float32, device=dev)
        p = torch.empty((n, e), dtype=torch.float32, device=dev) if probabilities else None
        if error is None:
            error = torch.zeros(1, dtype=torch.int32, device=dev)
    _routes_check(ids, w, n, top_k, dev)
    _need(error, "error", torch.int32, (1,), dev)
    _check(library().moe_router_select(_ptr(logits), n, e, top_k, _ptr(p), _ptr(ids), _ptr(w), _ptr(error),
                                       _stream(stream)), "moe_router_select")
    return ids, w, p, error


def read_probe(buffer, sink, nbytes=None, stream=None):
    """Enqueue a plain streaming read of `nbytes` (default: all) of a device tensor."""
    n = buffer.numel() * buffer.element_size() if nbytes is None else nbytes
    _check(library().moe_read_probe(_ptr(buffer), n, _ptr(sink), _stream(stream)), "moe_read_probe")


def quantize_q8_1(x, error=None, stream=None):
    """fp32 [cols, width] (device) -> uint8 [cols, width/32*36] canonical Q8_1."""
    import torch
    cols, width = x.shape
    _need(x, "x", torch.float32, (cols, width), x.device)
    with _making(stream):
        out = torch.empty((cols, width // 32 * Q8_BLOCK), dtype=torch.uint8, device=x.device)
        if error is None:
            error = torch.zeros(1, dtype=torch.int32, device=x.device)
    _need(error, "error", torch.int32, (1,), x.device)
    _check(library().moe_quantize_q8_1(_ptr(x), _ptr(out), width, cols, _ptr(error), _stream(stream)),
           "moe_quantize_q8_1")
    return out, error


def combine(contributions, weights, shared=None, shared_gate=None, stream=None):
    import torch
    n, k, h = contributions.shape
    dev = contributions.device
    _need(contributions, "contributions", torch.float32, (n, k, h), dev)
    _need(weights, "weights", torch.float32, (n, k), dev)
    if shared is not None:
        _need(shared, "shared", torch.float32, (n, h), dev)
    if shared_gate is not None:
        _need(shared_gate, "shared_gate", torch.float32, (n,), dev)
    with _making(stream):
        y = torch.empty((n, h), dtype=torch.float32, device=contributions.device)
        error = torch.zeros(1, dtype=torch.int32, device=contributions.device)
    _check(library().moe_combine(_ptr(contributions), _ptr(weights), _ptr(shared), _ptr(shared_gate), n, k, h,
                                 _ptr(y), _ptr(error), _stream(stream)), "moe_combine")
    return y, error


def memory_bytes(hidden, intermediate, experts, top_k, has_shared, max_tokens):
    cfg = Config(hidden, intermediate, experts, top_k, 1 if has_shared else 0, max_tokens)
    w, s = ctypes.c_size_t(), ctypes.c_size_t()
    _check(library().moe_ffn_memory_bytes(ctypes.byref(cfg), ctypes.byref(w), ctypes.byref(s)), "memory_bytes")
    return w.value, s.value


class MoeLinear:
    """One resident Q4_0 / Q4_1 matrix [output][input/32] (moe_linear_create):
    forward_q8 takes canonical Q8_1 columns, apply takes fp32 columns."""

    def __init__(self, type_, input, output, weights, max_columns=0, device=0):
        import torch
        self.type, self.K, self.M, self.max_columns = type_, input, output, max_columns
        self.device = device
        handle = ctypes.c_void_p()
        if isinstance(weights, np.ndarray):
            w = np.ascontiguousarray(weights, dtype=np.uint8)
            st = library().moe_linear_create(type_, input, output, max_columns, ctypes.c_void_p(w.ctypes.data), 0,
                                             device, ctypes.byref(handle))
        else:
            assert isinstance(weights, torch.Tensor) and weights.is_cuda
            st = library().moe_linear_create(type_, input, output, max_columns, _ptr(weights), 1, device,
                                             ctypes.byref(handle))
        _check(st, "moe_linear_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight_bytes(self):
        n = ctypes.c_size_t()
        _check(library().moe_linear_bytes(self.handle, ctypes.byref(n)), "moe_linear_bytes")
        return n.value

    def forward_q8(self, x_q8, columns, y=None, stream=None):
        import torch
        if x_q8.dtype != torch.uint8 or not x_q8.is_contiguous() or x_q8.numel() < columns * (self.K // 32) * Q8_BLOCK:
            raise ValueError("x_q8 must be contiguous uint8 holding columns x input/32 Q8_1 blocks")
        if y is None:
            with _making(stream):
                y = torch.empty((columns, self.M), dtype=torch.float32, device=x_q8.device)
        _need(y, "y", torch.float32, (columns, self.M), x_q8.device)
        _check(library().moe_linear_forward_q8(self.handle, _ptr(x_q8), columns, _ptr(y), _stream(stream)),
               "moe_linear_forward_q8")
        return y

    def apply(self, x, y=None, error=None, stream=None):
        import torch
        n = x.shape[0]
        _need(x, "x", torch.float32, (n, self.K), x.device)
        with _making(stream):
            if y is None:
                y = torch.empty((n, self.M), dtype=torch.float32, device=x.device)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x.device)
        _need(y, "y", torch.float32, (n, self.M), x.device)
        _need(error, "error", torch.int32, (1,), x.device)
        _check(library().moe_linear_apply(self.handle, _ptr(x), n, _ptr(y), _ptr(error), _stream(stream)),
               "moe_linear_apply")
        return y, error

    def apply_noalloc(self, x, y, error, stream=None):
        """apply() through moe_linear_apply_noalloc: the activation staging is
        the library's static per-device array (4 MiB), not the handle's
        workspace; y and error must be given (nothing is allocated)."""
        import torch
        n = x.shape[0]
        dev = torch.device("cuda", self.device)   # the static array is set up for the handle's GPU
        _need(x, "x", torch.float32, (n, self.K), dev)
        _need(y, "y", torch.float32, (n, self.M), dev)
        _need(error, "error", torch.int32, (1,), dev)
        _check(library().moe_linear_apply_noalloc(self.handle, _ptr(x), n, _ptr(y), _ptr(error), _stream(stream)),
               "moe_linear_apply_noalloc")
        return y, error


def _e4m3(t, name, shape, device=None):
    """Check e4m3 codes: torch.float8_e4m3fn or uint8, contiguous."""
    import torch
    if isinstance(t, torch.Tensor) and t.dtype == torch.uint8:
        return _need(t, name, torch.uint8, shape, device)
    return _need(t, name, torch.float8_e4m3fn, shape, device)


def _blocks(n):
    return (n + E4M3_GROUP - 1) // E4M3_GROUP


def _e4m3_matrices(codes, scales, shape, name, device):
    """(code pointer, scale pointer, on device, kept alive) of e4m3 matrices of
    `shape` [..][rows][cols], torch tensors on `device` or numpy arrays."""
    import torch
    shape = tuple(shape)
    blocks = (*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1]))
    if isinstance(codes, np.ndarray):
        c, s = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
        if c.dtype != np.uint8 or s.dtype != np.float32:
            raise TypeError(f"{name}: numpy codes are uint8 and scales float32, got {c.dtype} and {s.dtype}")
        if c.shape != shape or s.shape != blocks:
            raise ValueError(f"{name}: expected codes {shape} and scales {blocks}, got {c.shape} and {s.shape}")
        return ctypes.c_void_p(c.ctypes.data), ctypes.c_void_p(s.ctypes.data), 0, (c, s)
    dev = torch.device("cuda", device)
    _e4m3(codes, f"{name} codes", shape, dev)
    _need(scales, f"{name} scales", torch.float32, blocks, dev)
    return _ptr(codes), _ptr(scales), 1, (codes, scales)


def quantize_e4m3(x, codes=None, scales=None, error=None, stream=None):
    """Rows x [n][width] (float32, bfloat16 or float16; rows may be strided)
    -> (codes float8_e4m3fn [n][width], scales float32 [n][ceil(width/128)],
    error)."""
    import torch
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a two-dimensional torch tensor")
    n, width = x.shape
    type_, stride = _need_rows(x, "x", (n, width))
    with _making(stream):
        if codes is None:
            codes = torch.empty((n, width), dtype=torch.float8_e4m3fn, device=x.device)
        if scales is None:
            scales = torch.empty((n, _blocks(width)), dtype=torch.float32, device=x.device)
        if error is None:
            error = torch.zeros(1, dtype=torch.int32, device=x.device)
    _e4m3(codes, "codes", (n, width), x.device)
    _need(scales, "scales", torch.float32, (n, _blocks(width)), x.device)
    _need(error, "error", torch.int32, (1,), x.device)
    with _on_device(x.device):
        _check(library().moe_quantize_e4m3(_ptr(x), type_, stride, width, n, _ptr(codes), _ptr(scales), _ptr(error),
                                           _stream_on(stream, x.device)), "moe_quantize_e4m3")
    return codes, scales, error


class MoeFp8Linear:
    """One resident e4m3 matrix [output][input] with a scale per block of 128 x
    128 (moe_fp8_linear_create): codes float8_e4m3fn (or uint8) and scales
    float32 [ceil(output/128)][ceil(input/128)], both torch tensors on a GPU
    or both numpy arrays.  forward takes e4m3 rows, apply rows of float32,
    bfloat16 or float16.  sums: SUMS_F32 for fp32 sums within every block, also
    of wide batches with 16-bit results, which otherwise (SUMS_AUTO) come from
    the faster e4m3 instruction (moe_fp8_linear_forward says what it drops)."""

    def __init__(self, input, output, codes, scales, max_columns=0, device=0, sums=SUMS_AUTO):
        self.K, self.M, self.max_columns, self.device = input, output, max_columns, device
        c, s, on_device, _keep = _e4m3_matrices(codes, scales, (output, input), "weights", device)
        handle = ctypes.c_void_p()
        _check(library().moe_fp8_linear_create(input, output, max_columns, c, s, on_device, device,
                                               ctypes.byref(handle)), "moe_fp8_linear_create")
        self.handle = handle
        self.set_sums(sums)

    def close(self):
        if getattr(self, "handle", None):
            library().moe_fp8_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_sums(self, sums):
        """SUMS_AUTO or SUMS_F32 for the calls made from here on."""
        _check(library().moe_fp8_linear_set_sums(self.handle, sums), "moe_fp8_linear_set_sums")

    def weight_bytes(self):
        n = ctypes.c_size_t()
        _check(library().moe_fp8_linear_bytes(self.handle, ctypes.byref(n)), "moe_fp8_linear_bytes")
        return n.value

    def bind_forward(self, x_codes, x_scales, y, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues it with no per-call checks; the tensors must
        stay alive and keep their shapes while the callable is used.  It keeps
        the matrix alive, and raises after close()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x_codes.shape[0]
        _e4m3(x_codes, "x_codes", (n, self.K), dev)
        _need(x_scales, "x_scales", torch.float32, (n, _blocks(self.K)), dev)
        type_, stride = _need_rows(y, "y", (n, self.M), dev)
        fn = library().moe_fp8_linear_forward
        args = (_ptr(x_codes), _ptr(x_scales), n, _ptr(y), type_, stride, _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_fp8_linear_forward", st)
        return call

    def forward(self, x_codes, x_scales, y=None, dtype=None, stream=None):
        """y [n][output] (given, or a new tensor of `dtype`, float32 unless
        said) from e4m3 rows."""
        import torch
        if y is None:
            with _making(stream):
                y = torch.empty((x_codes.shape[0], self.M), dtype=dtype or torch.float32, device=x_codes.device)
        self.bind_forward(x_codes, x_scales, y, stream)()
        return y

    def bind_apply(self, x, y, error, stream=None):
        """bind_forward's counterpart for apply()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x.shape[0]
        x_type, x_stride = _need_rows(x, "x", (n, self.K), dev)
        y_type, y_stride = _need_rows(y, "y", (n, self.M), dev)
        _need(error, "error", torch.int32, (1,), dev)
        fn = library().moe_fp8_linear_apply
        args = (_ptr(x), x_type, x_stride, n, _ptr(y), y_type, y_stride, _ptr(error), _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_fp8_linear_apply", st)
        return call

    def apply(self, x, y=None, error=None, dtype=None, stream=None):
        """(y, error) from rows x [n][input]; y in x's type unless given."""
        import torch
        with _making(stream):
            if y is None:
                y = torch.empty((x.shape[0], self.M), dtype=dtype or x.dtype, device=x.device)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x.device)
        self.bind_apply(x, y, error, stream)()
        return y, error


class MoeFp8Layer:
    """One MoE layer of e4m3 matrices for batches of up to 64 tokens
    (moe_fp8_layer_create).  gate and up are (codes [E][I][H], scales
    [E][ceil(I/128)][ceil(H/128)]), down is (codes [E][H][I], scales
    [E][ceil(H/128)][ceil(I/128)]) and shared, for a layer with a shared
    expert, its (gate, up, down) of the same without E; all torch tensors on
    the layer's GPU (float8_e4m3fn or uint8 codes) or all numpy arrays."""

    def __init__(self, hidden, intermediate, experts, top_k, has_shared, max_tokens, gate, up, down, shared=None, device=0):
        self.cfg = Fp8LayerConfig(hidden, intermediate, experts, top_k, 1 if has_shared else 0, max_tokens)
        self.H, self.I, self.E, self.k = hidden, intermediate, experts, top_k
        self.has_shared, self.max_tokens, self.device = bool(has_shared), max_tokens, device
        if self.has_shared != (shared is not None) or (self.has_shared and len(shared) != 3):
            raise ValueError("shared: three matrices where the layer has a shared expert, None where not")
        gate_up, down_shape = (intermediate, hidden), (hidden, intermediate)
        parts = [_e4m3_matrices(*m, (experts, *shape), name, device)
                 for m, shape, name in ((gate, gate_up, "gate"), (up, gate_up, "up"), (down, down_shape, "down"))]
        if self.has_shared:
            parts += [_e4m3_matrices(*m, shape, f"shared {name}", device)
                      for m, shape, name in zip(shared, (gate_up, gate_up, down_shape), ("gate", "up", "down"))]
        if len({p[2] for p in parts}) != 1:
            raise ValueError("the matrices must be all torch tensors or all numpy arrays")
        banks = [(Fp8Matrix * 3)(*[Fp8Matrix(p[0], p[1]) for p in parts[i:i + 3]]) for i in range(0, len(parts), 3)]
        handle = ctypes.c_void_p()
        _check(library().moe_fp8_layer_create(ctypes.byref(self.cfg), banks[0], banks[1] if self.has_shared else None,
                                              parts[0][2], device, ctypes.byref(handle)), "moe_fp8_layer_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_fp8_layer_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bind_forward(self, x, ids, weights, y, error, shared_gate=None, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues it with no per-call checks (as
        MoeLayer.bind_forward); it keeps the layer alive, and raises after
        close()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x.shape[0]
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"tokens {n} outside 1..{self.max_tokens}")
        type_ = _elem_type(x, "x")
        _need(x, "x", x.dtype, (n, self.H), dev)
        _routes_check(ids, weights, n, self.k, dev)
        if shared_gate is not None:
            _need(shared_gate, "shared_gate", torch.float32, (n,), dev)
        _need(y, "y", x.dtype, (n, self.H), dev)
        _need(error, "error", torch.int32, (1,), dev)
        fn = library().moe_fp8_layer_forward
        args = (_ptr(x), type_, _ptr(ids), _ptr(weights), n, _ptr(shared_gate), _ptr(y), _ptr(error),
                _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_fp8_layer_forward", st)
        return call

    def forward(self, x, ids, weights, shared_gate=None, y=None, error=None, stream=None):
        """(y, error) for x [n][H] of float32, bfloat16 or float16; y has x's
        type."""
        import torch
        with _making(stream):
            if y is None:
                y = torch.empty_like(x)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x.device)
        self.bind_forward(x, ids, weights, y, error, shared_gate, stream)()
        return y, error


def bind_quantize_i8(x, codes, scales, error, stream=None):
    """Validate the tensors of a quantize_i8() once and return a no-argument
    callable that enqueues it with no per-call checks; the tensors must stay
    alive and keep their shapes while the callable is used."""
    import torch
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a two-dimensional torch tensor")
    n, width = x.shape
    dev = x.device
    type_, stride = _need_rows(x, "x", (n, width))
    _need(codes, "codes", torch.int8, (n, width), dev)
    _need(scales, "scales", torch.float32, (n,), dev)
    _need(error, "error", torch.int32, (1,), dev)
    fn = library().moe_quantize_i8
    args = (_ptr(x), type_, stride, width, n, _ptr(codes), _ptr(scales), _ptr(error), _stream_on(stream, dev))
    current, switch = torch.cuda.current_device, dev.index

    def call():
        if current() != switch:
            with _on_device(dev):
                st = fn(*args)
        else:
            st = fn(*args)
        if st != 0:
            raise MoeError("moe_quantize_i8", st)
    return call


def quantize_i8(x, codes=None, scales=None, error=None, stream=None):
    """Rows x [n][width] (float32, bfloat16 or float16; rows may be strided)
    -> (codes int8 [n][width], scales float32 [n], error)."""
    import torch
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a two-dimensional torch tensor")
    with _making(stream):
        if codes is None:
            codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        if scales is None:
            scales = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
        if error is None:
            error = torch.zeros(1, dtype=torch.int32, device=x.device)
    bind_quantize_i8(x, codes, scales, error, stream)()
    return codes, scales, error


def _i8_matrices(codes, scales, shape, name, device):
    """(code pointer, scale pointer, on device, kept alive) of int8 matrices of
    `shape` [..][rows][cols] with scales [..][rows], torch tensors on `device`
    or numpy arrays."""
    import torch
    shape = tuple(shape)
    if isinstance(codes, np.ndarray):
        c, s = np.ascontiguousarray(codes), np.ascontiguousarray(scales)
        if c.dtype != np.int8 or s.dtype != np.float32:
            raise TypeError(f"{name}: numpy codes are int8 and scales float32, got {c.dtype} and {s.dtype}")
        if c.shape != shape or s.shape != shape[:-1]:
            raise ValueError(f"{name}: expected codes {shape} and scales {shape[:-1]}, got {c.shape} and {s.shape}")
        return ctypes.c_void_p(c.ctypes.data), ctypes.c_void_p(s.ctypes.data), 0, (c, s)
    dev = torch.device("cuda", device)
    _need(codes, f"{name} codes", torch.int8, shape, dev)
    _need(scales, f"{name} scales", torch.float32, shape[:-1], dev)
    return _ptr(codes), _ptr(scales), 1, (codes, scales)


class MoeI8Linear:
    """One resident int8 matrix [output][input] with a scale per output channel
    (moe_i8_linear_create): codes int8 and scales float32 [output], both torch
    tensors on a GPU or both numpy arrays.  forward takes int8 rows with a scale
    each, apply rows of float32, bfloat16 or float16.  The sums are exact."""

    def __init__(self, input, output, codes, scales, max_columns=0, device=0):
        self.K, self.M, self.max_columns, self.device = input, output, max_columns, device
        c, s, on_device, _keep = _i8_matrices(codes, scales, (output, input), "weights", device)
        handle = ctypes.c_void_p()
        _check(library().moe_i8_linear_create(input, output, max_columns, c, s, on_device, device,
                                              ctypes.byref(handle)), "moe_i8_linear_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_i8_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight_bytes(self):
        n = ctypes.c_size_t()
        _check(library().moe_i8_linear_bytes(self.handle, ctypes.byref(n)), "moe_i8_linear_bytes")
        return n.value

    def bind_forward(self, x_codes, x_scales, y, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues it with no per-call checks; the tensors must
        stay alive and keep their shapes while the callable is used.  It keeps
        the matrix alive, and raises after close()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x_codes.shape[0]
        _need(x_codes, "x_codes", torch.int8, (n, self.K), dev)
        _need(x_scales, "x_scales", torch.float32, (n,), dev)
        type_, stride = _need_rows(y, "y", (n, self.M), dev)
        fn = library().moe_i8_linear_forward
        args = (_ptr(x_codes), _ptr(x_scales), n, _ptr(y), type_, stride, _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_i8_linear_forward", st)
        return call

    def forward(self, x_codes, x_scales, y=None, dtype=None, stream=None):
        """y [n][output] (given, or a new tensor of `dtype`, float32 unless
        said) from int8 rows."""
        import torch
        if y is None:
            with _making(stream):
                y = torch.empty((x_codes.shape[0], self.M), dtype=dtype or torch.float32, device=x_codes.device)
        self.bind_forward(x_codes, x_scales, y, stream)()
        return y

    def bind_apply(self, x, y, error, stream=None):
        """bind_forward's counterpart for apply()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x.shape[0]
        x_type, x_stride = _need_rows(x, "x", (n, self.K), dev)
        y_type, y_stride = _need_rows(y, "y", (n, self.M), dev)
        _need(error, "error", torch.int32, (1,), dev)
        fn = library().moe_i8_linear_apply
        args = (_ptr(x), x_type, x_stride, n, _ptr(y), y_type, y_stride, _ptr(error), _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_i8_linear_apply", st)
        return call

    def apply(self, x, y=None, error=None, dtype=None, stream=None):
        """(y, error) from rows x [n][input]; y in x's type unless given."""
        import torch
        with _making(stream):
            if y is None:
                y = torch.empty((x.shape[0], self.M), dtype=dtype or x.dtype, device=x.device)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x.device)
        self.bind_apply(x, y, error, stream)()
        return y, error


class MoeI8Bank:
    """Resident int8 matrices of a number of experts (moe_i8_bank_create): codes
    int8 [experts][output][input] and scales float32 [experts][output], both
    torch tensors on a GPU or both numpy arrays.  forward multiplies rows that
    are grouped by expert, in groups of any sizes that only the device knows."""

    def __init__(self, experts, input, output, codes, scales, device=0):
        self.E, self.K, self.M, self.device = experts, input, output, device
        c, s, on_device, _keep = _i8_matrices(codes, scales, (experts, output, input), "weights", device)
        handle = ctypes.c_void_p()
        _check(library().moe_i8_bank_create(experts, input, output, c, s, on_device, device, ctypes.byref(handle)),
               "moe_i8_bank_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_i8_bank_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight_bytes(self):
        n = ctypes.c_size_t()
        _check(library().moe_i8_bank_bytes(self.handle, ctypes.byref(n)), "moe_i8_bank_bytes")
        return n.value

    def bind_forward(self, x_codes, x_scales, offsets, y, error, index=None, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues it with no per-call checks; the tensors must
        stay alive and keep their shapes while the callable is used.  It keeps
        the bank alive, and raises after close()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x_codes.shape[0]
        _need(x_codes, "x_codes", torch.int8, (n, self.K), dev)
        _need(x_scales, "x_scales", torch.float32, (n,), dev)
        _need(offsets, "offsets", torch.int32, (self.E + 1,), dev)
        if not isinstance(y, torch.Tensor) or y.dim() != 2:
            raise ValueError("y must be a two-dimensional torch tensor")
        rows = y.shape[0]
        if index is not None:
            _need(index, "index", torch.int32, (rows,), dev)
        elif rows > n:
            raise ValueError(f"y has {rows} rows, x_codes {n}; without an index they are the same rows")
        type_, stride = _need_rows(y, "y", (rows, self.M), dev)
        _need(error, "error", torch.int32, (1,), dev)
        fn = library().moe_i8_bank_forward
        args = (_ptr(x_codes), _ptr(x_scales), n, _ptr(index), _ptr(offsets), rows, _ptr(y), type_, stride, _ptr(error),
                _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_i8_bank_forward", st)
        return call

    def forward(self, x_codes, x_scales, offsets, y=None, error=None, index=None, dtype=None, stream=None):
        """(y, error): rows offsets[e] .. offsets[e + 1] - 1 of y (given, or new
        zeros of `dtype`, float32 unless said) are x_codes' rows, or its rows
        index[i], times expert e's matrix.  Rows of no group stay as they are."""
        import torch
        with _making(stream):
            if y is None:
                rows = (index if index is not None else x_codes).shape[0]
                y = torch.zeros((rows, self.M), dtype=dtype or torch.float32, device=x_codes.device)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x_codes.device)
        self.bind_forward(x_codes, x_scales, offsets, y, error, index, stream)()
        return y, error


class MoeI8Layer:
    """One MoE layer of int8 matrices, for one token as for whole prompts
    (moe_i8_layer_create).  gate and up are (codes [E][I][H], scales [E][I]),
    down is (codes [E][H][I], scales [E][H]) and shared, for a layer with a
    shared expert, its (gate, up, down) of the same without E; all torch tensors
    on the layer's GPU or all numpy arrays."""

    def __init__(self, hidden, intermediate, experts, top_k, has_shared, max_tokens, gate, up, down, shared=None, device=0):
        self.cfg = I8LayerConfig(hidden, intermediate, experts, top_k, 1 if has_shared else 0, max_tokens)
        self.H, self.I, self.E, self.k = hidden, intermediate, experts, top_k
        self.has_shared, self.max_tokens, self.device = bool(has_shared), max_tokens, device
        if self.has_shared != (shared is not None) or (self.has_shared and len(shared) != 3):
            raise ValueError("shared: three matrices where the layer has a shared expert, None where not")
        gate_up, down_shape = (intermediate, hidden), (hidden, intermediate)
        parts = [_i8_matrices(*m, (experts, *shape), name, device)
                 for m, shape, name in ((gate, gate_up, "gate"), (up, gate_up, "up"), (down, down_shape, "down"))]
        if self.has_shared:
            parts += [_i8_matrices(*m, shape, f"shared {name}", device)
                      for m, shape, name in zip(shared, (gate_up, gate_up, down_shape), ("gate", "up", "down"))]
        if len({p[2] for p in parts}) != 1:
            raise ValueError("the matrices must be all torch tensors or all numpy arrays")
        banks = [(I8Matrix * 3)(*[I8Matrix(p[0], p[1]) for p in parts[i:i + 3]]) for i in range(0, len(parts), 3)]
        handle = ctypes.c_void_p()
        _check(library().moe_i8_layer_create(ctypes.byref(self.cfg), banks[0], banks[1] if self.has_shared else None,
                                             parts[0][2], device, ctypes.byref(handle)), "moe_i8_layer_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            library().moe_i8_layer_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bind_forward(self, x, ids, weights, y, error, shared_gate=None, stream=None):
        """Validate the tensors of a forward() once and return a no-argument
        callable that enqueues it with no per-call checks (as
        MoeLayer.bind_forward); it keeps the layer alive, and raises after
        close()."""
        import torch
        dev = torch.device("cuda", self.device)
        n = x.shape[0]
        if not 1 <= n <= self.max_tokens:
            raise ValueError(f"tokens {n} outside 1..{self.max_tokens}")
        type_ = _elem_type(x, "x")
        _need(x, "x", x.dtype, (n, self.H), dev)
        _routes_check(ids, weights, n, self.k, dev)
        if shared_gate is not None:
            _need(shared_gate, "shared_gate", torch.float32, (n,), dev)
        _need(y, "y", x.dtype, (n, self.H), dev)
        _need(error, "error", torch.int32, (1,), dev)
        fn = library().moe_i8_layer_forward
        args = (_ptr(x), type_, _ptr(ids), _ptr(weights), n, _ptr(shared_gate), _ptr(y), _ptr(error),
                _stream_on(stream, dev))

        def call():
            st = fn(self.handle, *args)
            if st != 0:
                raise MoeError("moe_i8_layer_forward", st)
        return call

    def forward(self, x, ids, weights, shared_gate=None, y=None, error=None, stream=None):
        """(y, error) for x [n][H] of float32, bfloat16 or float16; y has x's
        type."""
        import torch
        with _making(stream):
            if y is None:
                y = torch.empty_like(x)
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=x.device)
        self.bind_forward(x, ids, weights, y, error, shared_gate, stream)()
        return y, error


class BlockNorm:
    """The norm after a block and the norm before the next one, with the gate,
    the scales and the residual sum between them (moe_block_norm):

        b = rms(block) * (weight_offset + post_weight)   (post_weight None: block)
        h = residual_scale * residual + block_scale * gate(b)
        n = rms(h) * (weight_offset + pre_weight)

    Weights are float32 [hidden] tensors on a GPU.  pre_weight None: only h.
    gate(b) multiplies by the gate given to a call, or by its sigmoid with
    gate_sigmoid."""

    def __init__(self, hidden, pre_weight=None, post_weight=None, eps=1e-6, weight_offset=0.0, residual_scale=1.0,
                 block_scale=1.0, gate_sigmoid=False):
        import torch
        if pre_weight is None and post_weight is None:
            raise ValueError("pre_weight or post_weight is required")
        self.hidden, self.pre_weight, self.post_weight = hidden, pre_weight, post_weight
        self.device = (pre_weight if pre_weight is not None else post_weight).device
        for name, w in (("pre_weight", pre_weight), ("post_weight", post_weight)):
            if w is not None:
                _need(w, name, torch.float32, (hidden,), self.device)
        if not eps > 0:
            raise ValueError("eps must be positive")
        self.eps, self.weight_offset, self.gate_sigmoid = eps, weight_offset, gate_sigmoid
        self.residual_scale, self.block_scale = residual_scale, block_scale

    def bind(self, residual, block=None, gate=None, residual_out=None, out=None, q8=None, codes=None, scales=None,
             error=None, stream=None):
        """Validate the tensors of a call once and return a no-argument
        callable that enqueues it; the tensors must stay alive and keep their
        shapes while the callable is used.

        residual, residual_out [n][hidden] of the block's type or float32;
        block, out [n][hidden] float32, bfloat16 or float16; gate float32 [n, 1]
        (one value a row), float32 [hidden] (one a channel) or [n][hidden] of
        the block's type; q8 uint8 [n][hidden/32*36]; codes float8_e4m3fn
        [n][hidden] with scales float32 [n][ceil(hidden/128)].  Rows of the
        [n][hidden] tensors other than codes may be strided.  Without a block
        the norm of the residual alone is taken."""
        import torch
        h = self.hidden
        if not isinstance(residual, torch.Tensor) or residual.dim() != 2:
            raise ValueError("residual must be a two-dimensional torch tensor")
        n, dev = residual.shape[0], self.device
        a = BlockNormArgs(hidden=h, tokens=n, eps=self.eps, weight_offset=self.weight_offset,
                          residual_scale=self.residual_scale, block_scale=self.block_scale,
                          gate_sigmoid=1 if self.gate_sigmoid else 0)
        a.residual_type, a.residual_stride = _need_rows(residual, "residual", (n, h), dev)
        a.residual = residual.data_ptr()
        like = block if block is not None else out if out is not None else residual
        a.type = _elem_type(like, "block")
        if residual.dtype not in (torch.float32, like.dtype):
            raise TypeError(f"residual must be float32 or {like.dtype}, got {residual.dtype}")
        if block is not None:
            _, a.block_stride = _need_rows(block, "block", (n, h), dev)
            a.block = block.data_ptr()
            if self.post_weight is not None:
                a.post_weight = self.post_weight.data_ptr()
        if gate is not None:
            if block is None:
                raise ValueError("a gate needs a block")
            if not isinstance(gate, torch.Tensor):
                raise TypeError("gate must be a torch tensor")
            if tuple(gate.shape) == (n, 1) and (h > 1 or gate.dtype != like.dtype):
                a.gate_form = GATE_TOKEN
                _need(gate, "gate", torch.float32, (n, 1), dev)
            elif gate.dim() == 1:
                a.gate_form = GATE_CHANNEL
                _need(gate, "gate", torch.float32, (h,), dev)
            else:
                a.gate_form = GATE_ELEMENT
                _, a.gate_stride = _need_rows(gate, "gate", (n, h), dev, dtypes=(like.dtype,))
            a.gate = gate.data_ptr()
        if residual_out is not None:
            _, a.residual_out_stride = _need_rows(residual_out, "residual_out", (n, h), dev, dtypes=(residual.dtype,))
            a.residual_out = residual_out.data_ptr()
        if (codes is None) != (scales is None):
            raise ValueError("codes and scales come together")
        if self.pre_weight is None:
            if out is not None or q8 is not None or codes is not None:
                raise ValueError("out, q8 and codes need a pre_weight")
            if residual_out is None:
                raise ValueError("residual_out is required without a pre_weight")
        elif out is not None or q8 is not None or codes is not None:
            a.pre_weight = self.pre_weight.data_ptr()
        elif residual_out is None:
            raise ValueError("one of residual_out, out, q8 and codes is required")
        if out is not None:
            _, a.out_stride = _need_rows(out, "out", (n, h), dev, dtypes=(like.dtype,))
            a.out = out.data_ptr()
        if q8 is not None:
            if h % 32:
                raise ValueError("q8 needs a multiple of 32 channels")
            a.q8 = _need(q8, "q8", torch.uint8, (n, h // 32 * Q8_BLOCK), dev).data_ptr()
        if codes is not None:
            a.codes = _e4m3(codes, "codes", (n, h), dev).data_ptr()
            a.scales = _need(scales, "scales", torch.float32, (n, _blocks(h)), dev).data_ptr()
        if q8 is not None or codes is not None:
            a.error = _need(error, "error", torch.int32, (1,), dev).data_ptr()
        a.weights = self.pre_weight, self.post_weight   # alive while the callable is
        fn, arg, s = library().moe_block_norm, ctypes.byref(a), _stream_on(stream, dev)
        current, switch = torch.cuda.current_device, dev.index

        def call():
            if current() != switch:
                with _on_device(dev):
                    st = fn(arg, s)
            else:
                st = fn(arg, s)
            if st != 0:
                raise MoeError("moe_block_norm", st)
        return call

    def __call__(self, residual, block=None, gate=None, outputs=("residual", "out"), error=None, stream=None):
        """One call into new tensors: `outputs` names which of residual, out,
        q8 and e4m3 are wanted.  Returns a dict of them (e4m3 as codes and
        scales) and the error word."""
        import torch
        unknown = set(outputs) - {"residual", "out", "q8", "e4m3"}
        if unknown:
            raise ValueError(f"unknown outputs {sorted(unknown)}")
        n, h, dev = residual.shape[0], self.hidden, residual.device
        made = {}
        with _making(stream):
            if error is None:
                error = torch.zeros(1, dtype=torch.int32, device=dev)
            if "residual" in outputs:
                made["residual_out"] = torch.empty((n, h), dtype=residual.dtype, device=dev)
            if "out" in outputs and self.pre_weight is not None:
                made["out"] = torch.empty((n, h), dtype=(block if block is not None else residual).dtype, device=dev)
            if "q8" in outputs:
                made["q8"] = torch.empty((n, h // 32 * Q8_BLOCK), dtype=torch.uint8, device=dev)
            if "e4m3" in outputs:
                made["codes"] = torch.empty((n, h), dtype=torch.float8_e4m3fn, device=dev)
                made["scales"] = torch.empty((n, _blocks(h)), dtype=torch.float32, device=dev)
        self.bind(residual, block=block, gate=gate, error=error, stream=stream, **made)()
        if "residual_out" in made:
            made["residual"] = made.pop("residual_out")
        return dict(made, error=error)


class MoeStack:
    """A stack of resident MoE layers run back to back on one stream, eagerly
    or replayed from one captured HIP graph (torch.cuda.CUDAGraph over the
    library's launches).

    Layers, projections and routers may be Q4 (MoeLayer, MoeLinear), e4m3
    (MoeFp8Layer, MoeFp8Linear) or int8 (MoeI8Layer, MoeI8Linear) handles.

    Without `norms`, layer l takes its own input batch x[l] (fp32 [N_l][H],
    device; e4m3 and int8 layers also bfloat16 or float16).  With `projections` (H -> H
    per layer) the layer input is h = projection.apply(x); with `routers` (H ->
    E per layer) the routes are chosen on the device from router.apply(h) by
    router_select; otherwise fixed device ids / weights are given to bind().
    Fewer batches than layers run the first layers.

    With `norms` (len(layers) + 1 BlockNorms) the layers run on one residual
    stream, xs = [x]: norms[0] makes the first layer's input from x, norms[l]
    adds layer l - 1's output to the stream and makes layer l's input, and the
    last one closes the stack (with a pre_weight: the final norm as well).  An
    e4m3 projection takes its input as the e4m3 rows that the norm writes, and
    a Q4 layer without a projection as its Q8_1 rows.

    Every buffer is allocated by bind(), so run() allocates nothing and can be
    captured."""

    def __init__(self, layers, projections=None, routers=None, norms=None):
        self.layers = list(layers)
        self.projections = projections
        self.routers = routers
        self.norms = norms
        if norms is not None:
            if len(norms) != len(self.layers) + 1:
                raise ValueError("norms: one before the first layer and one after each")
            if not self.layers:
                raise ValueError("a stack with norms needs a layer")
            if any(n.pre_weight is None for n in norms[:-1]):
                raise ValueError("norms before a layer need a pre_weight")
            if any(n.hidden != L.H for n in norms for L in self.layers):
                raise ValueError("norms and layers need one hidden size")
        self.graph = None

    def bind(self, xs, ids=None, weights=None, dtype=None):
        """Allocate every buffer for the input batches xs, on the current stream
        (a run on another one has to wait for it).  dtype (with norms): type of
        the layers' inputs and outputs, that of x unless said; x, the residual
        stream, is of that type or float32.  The Q4 handles take float32 rows
        alone."""
        import torch
        if self.norms is not None:
            if len(xs) != 1:
                raise ValueError("a stack with norms takes one input batch")
            if dtype is not None and xs[0].dtype not in (torch.float32, dtype):
                raise TypeError(f"the residual stream must be float32 or {dtype}, got {xs[0].dtype}")
        batches = xs if self.norms is None else list(xs) * len(self.layers)
        kinds = [x.dtype if dtype is None or self.norms is None else dtype for _, x in zip(self.layers, batches)]
        for l, (x, kind) in enumerate(zip(batches, kinds)):
            L, linears = self.layers[l], [handles[l] for handles in (self.projections, self.routers) if handles]
            if kind != torch.float32 and any(isinstance(m, (MoeLayer, MoeLinear)) for m in [L] + linears):
                raise TypeError(f"layer {l}: Q4 layers, projections and routers take float32 rows, got {kind}")
            if x.dim() != 2 or x.shape[1] != L.H:
                raise ValueError(f"layer {l}: expected rows of {L.H}, got {tuple(x.shape)}")
            if self.norms is not None and self.projections and isinstance(self.projections[l], MoeFp8Linear):
                linears = linears[1:]   # takes the norm's rows as they are
            most = min([L.max_tokens] + [m.max_columns for m in linears])
            if not 1 <= x.shape[0] <= most:
                raise ValueError(f"layer {l}: tokens {x.shape[0]} outside 1..{most}")
        dev = xs[0].device
        self.error = torch.zeros(1, dtype=torch.int32, device=dev)
        self.steps = []
        for l, (L, x, kind) in enumerate(zip(self.layers, batches, kinds)):
            n = x.shape[0]
            st = {"y": torch.empty((n, L.H), dtype=kind, device=dev)}
            if self.norms is None:
                st["x"] = x
            elif self.projections and isinstance(self.projections[l], MoeFp8Linear):
                st["codes"] = torch.empty((n, L.H), dtype=torch.float8_e4m3fn, device=dev)
                st["scales"] = torch.empty((n, _blocks(L.H)), dtype=torch.float32, device=dev)
                st["norm"] = {"codes": st["codes"], "scales": st["scales"]}
            else:
                st["x"] = torch.empty((n, L.H), dtype=kind, device=dev)
                st["norm"] = {"out": st["x"]}
                if not self.projections and isinstance(L, MoeLayer):
                    st["q8"] = torch.empty((n, L.H // 32 * Q8_BLOCK), dtype=torch.uint8, device=dev)
                    st["norm"]["q8"] = st["q8"]
            st["h"] = torch.empty((n, L.H), dtype=kind, device=dev) if self.projections else st["x"]
            if self.routers:
                st["logits"] = torch.empty((n, L.E), dtype=torch.float32, device=dev)
                st["ids"] = torch.empty((n, L.k), dtype=torch.int32, device=dev)
                st["w"] = torch.empty((n, L.k), dtype=torch.float32, device=dev)
            else:
                st["ids"], st["w"] = ids[l], weights[l]
            self.steps.append(st)
        if self.norms is not None:
            self.x = xs[0]
            self.residual = torch.empty_like(self.x)
            self.last = {"residual_out": self.residual}
            if self.norms[-1].pre_weight is not None:
                self.last["out"] = torch.empty_like(self.steps[-1]["y"])
        self.graph = None

    def run(self, stream=None):
        for l, (L, st) in enumerate(zip(self.layers, self.steps)):
            if self.norms is not None:
                self._norm(l, st["norm"], stream)
            if self.projections:
                if "codes" in st:
                    self.projections[l].forward(st["codes"], st["scales"], y=st["h"], stream=stream)
                else:
                    self.projections[l].apply(st["x"], y=st["h"], error=self.error, stream=stream)
            if self.routers:
                self.routers[l].apply(st["h"], y=st["logits"], error=self.error, stream=stream)
                router_select(st["logits"], top_k=L.k, error=self.error, stream=stream, ids=st["ids"],
                              weights=st["w"])
            if "q8" in st:
                L.forward_q8(st["q8"], st["ids"], st["w"], y=st["y"], error=self.error, stream=stream)
            else:
                L.forward(st["h"], st["ids"], st["w"], y=st["y"], error=self.error, stream=stream)
        if self.norms is not None:
            self._norm(len(self.layers), self.last, stream)

    def _norm(self, l, outputs, stream):
        """norms[l]: the stream starts as x and is self.residual from the first
        layer's output on."""
        if l > 0:
            outputs = dict(outputs, block=self.steps[l - 1]["y"], residual_out=self.residual)
        self.norms[l].bind(self.x if l <= 1 else self.residual, error=self.error, stream=stream, **outputs)()

    def capture(self):
        """Record one run() into a HIP graph (after one eager run as warm-up)."""
        import torch
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.run()
        return self.graph

    def replay(self):
        self.graph.replay()

    def outputs(self):
        """Each layer's output; with norms the residual stream at the end and,
        where the last norm has a pre_weight, the final norm."""
        if self.norms is not None:
            return [self.residual] + ([self.last["out"]] if "out" in self.last else [])
        return [st["y"] for st in self.steps]
