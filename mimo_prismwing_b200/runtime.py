"""Python mirror of the reference's routed-MoE runtime over the C ABI.

The class and method names follow the reference's Rust runtime
(`WideMetalMoeRuntime`, src/wide_metal_moe.rs:165-1316) so that tests read
like the reference's own: `compile`, `compile_with_fused_gate_up`,
`execute_fp8_linear`, `execute`, `execute_fused_gate_up`.  Every call goes
through include/pw_cuda.h into mimo_prismwing_b200/lib/libpw_cuda.so; there is
no CPU fallback, and loading fails loudly when the library is missing.

Tensors: weights and scales are torch CUDA tensors (uint8 e4m3 bytes, float32
scale grids); activations may be CUDA tensors (device I/O) or CPU tensors /
numpy arrays (host I/O: the call copies in and out, as the reference's
commit + wait_until_completed does).
"""
from __future__ import annotations

import ctypes
import os
import struct
import warnings
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib

PW_OK = 0
LAYOUT_PLAIN = 0
LAYOUT_FULL_QKV = 1
LAYOUT_SWA_QKV = 2
OUTPUT_F32 = 0x100
MEM_DEVICE = 0
MEM_HOST = 1
MEM_ASYNC = 2
EP_NCCL_TRANSPORT = 1
RUNTIME_FUSED_GATE_UP = 1
ROUTER_F32 = 0
ROUTER_BF16 = 1
NORM_F32 = 0
NORM_BF16 = 1
NORM_F16 = 2
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PW_DTYPE_*, and PW_NORM_* of the same order
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}  # PW_ACT_*
CUDA_STREAM_LEGACY = 1  # cudaStreamLegacy, the handle of the stream that torch calls 0

ERRORS = {
    -1: "argument", -2: "shape", -3: "nonfinite", -4: "device_flags", -5: "cuda", -6: "nccl",
    -7: "timeout", -8: "schedule", -9: "unsupported",
}


class PrismwingError(RuntimeError):
    """A non-zero status from the C ABI (the reference's Err(String))."""

    def __init__(self, status: int, message: str):
        super().__init__(f"[{ERRORS.get(status, status)}] {message}")
        self.status = status
        self.kind = ERRORS.get(status, str(status))


class Fp8Tensor(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("rows", ctypes.c_uint32),
                ("cols", ctypes.c_uint32), ("scale_rows", ctypes.c_uint32), ("scale_cols", ctypes.c_uint32)]


class ExpertWeights(ctypes.Structure):
    _fields_ = [("gate", Fp8Tensor), ("up", Fp8Tensor), ("down", Fp8Tensor)]


class ExpertBinding(ctypes.Structure):
    _fields_ = [("expert", ctypes.c_uint32), ("count", ctypes.c_uint32), ("positions", ctypes.c_void_p),
                ("route_weights", ctypes.c_void_p), ("weights", ExpertWeights)]


class Router(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("experts", ctypes.c_uint32),
                ("hidden", ctypes.c_uint32), ("top_k", ctypes.c_uint32), ("weight_dtype", ctypes.c_uint32)]


class Norm(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("hidden", ctypes.c_uint32), ("weight_dtype", ctypes.c_uint32),
                ("epsilon", ctypes.c_float)]


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_uint64), ("dtype", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32)]


class Dense(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("stride", ctypes.c_uint64), ("rows", ctypes.c_uint32),
                ("cols", ctypes.c_uint32), ("dtype", ctypes.c_uint32), ("reserved", ctypes.c_uint32)]


class Epilogue(ctypes.Structure):
    _fields_ = [("bias", ctypes.c_void_p), ("bias_dtype", ctypes.c_uint32), ("activation", ctypes.c_uint32),
                ("residual", Rows)]


class Stats(ctypes.Structure):
    _fields_ = [("wall_ms", ctypes.c_double), ("device_ms", ctypes.c_float), ("error_flags", ctypes.c_uint32),
                ("unique_experts", ctypes.c_uint32), ("expert_rows", ctypes.c_uint32),
                ("boundary_tie_rows", ctypes.c_uint32), ("weight_bytes", ctypes.c_uint64)]

    def as_dict(self) -> dict:
        return {k: getattr(self, k) for k, _ in self._fields_}


class Profile(ctypes.Structure):
    _fields_ = [("quantize_ms", ctypes.c_float), ("router_ms", ctypes.c_float), ("schedule_ms", ctypes.c_float),
                ("gate_up_ms", ctypes.c_float), ("down_ms", ctypes.c_float), ("combine_ms", ctypes.c_float),
                ("projection_ms", ctypes.c_float), ("launches", ctypes.c_uint32)]

    def as_dict(self) -> dict:
        return {k: getattr(self, k) for k, _ in self._fields_}


# ------------------------------------------------------------------ bindings
@dataclass
class WideProjectionBinding:
    """One e4m3 matrix + f32 scale grid on the GPU (src/wide_metal_moe.rs:80)."""
    weight: torch.Tensor  # uint8 [rows, cols], CUDA
    scale: torch.Tensor   # float32 [scale_rows, scale_cols], CUDA

    @property
    def rows(self) -> int:
        return int(self.weight.shape[0])

    @property
    def columns(self) -> int:
        return int(self.weight.shape[1])

    def c(self) -> Fp8Tensor:
        w, s = self.weight, self.scale
        if not (w.is_cuda and s.is_cuda and w.dtype == torch.uint8 and s.dtype == torch.float32):
            raise PrismwingError(-1, "projection weight must be CUDA uint8 and scale CUDA float32")
        if not (w.is_contiguous() and s.is_contiguous()):
            raise PrismwingError(-1, "projection tensors must be contiguous")
        return Fp8Tensor(w.data_ptr(), s.data_ptr(), w.shape[0], w.shape[1], s.shape[0], s.shape[1])


@dataclass
class WideExpertBinding:
    """An expert's placements and projections (src/wide_metal_moe.rs:88)."""
    expert: int
    positions: Sequence[int]
    route_weights: Sequence[float]
    gate: WideProjectionBinding
    up: WideProjectionBinding
    down: WideProjectionBinding

    def weights_c(self) -> ExpertWeights:
        return ExpertWeights(self.gate.c(), self.up.c(), self.down.c())


@dataclass
class Execution:
    """WideLinearExecution / WideMoeExecution (src/wide_metal_moe.rs:97-111)."""
    output: torch.Tensor
    wall_ms: float
    device_ms: float
    unique_experts: int = 0
    expert_rows: int = 0
    boundary_tie_rows: int = 0
    weight_bytes: int = 0
    selected: Optional[torch.Tensor] = None
    weights: Optional[torch.Tensor] = None


@dataclass
class NormExecution:
    """What add_rms_norm was asked for (None: not asked for)."""
    sum: Optional[torch.Tensor]
    y: Optional[torch.Tensor]
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def _as_f32(x) -> torch.Tensor:
    if isinstance(x, np.ndarray):
        x = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
    if x.dtype != torch.float32:
        x = x.float()
    return x.contiguous()


class WideMoeRuntime:
    """B200 counterpart of the reference's WideMetalMoeRuntime."""

    def __init__(self, device: int = 0, fused_gate_up: bool = True):
        self._L = _lib.load()
        rt = ctypes.c_void_p()
        st = self._L.pw_runtime_create(device, RUNTIME_FUSED_GATE_UP if fused_gate_up else 0, ctypes.byref(rt))
        if st != PW_OK:
            raise PrismwingError(st, f"pw_runtime_create failed on device {device}")
        self._rt = rt
        self.device = device
        self.fused_gate_up = fused_gate_up
        self._banks = []
        self._bank_refs = []
        self._init_args()
        try:
            calls = _lib.binding().Calls
        except (RuntimeError, ImportError) as e:  # not built for this torch and Python: the calls below run without it
            warnings.warn(f"short calls take longer on the host: {e}", RuntimeWarning, stacklevel=2)
        else:
            entry = [ctypes.cast(f, ctypes.c_void_p).value for f in
                     (self._L.pw_add_rms_norm, self._L.pw_linear, self._L.pw_fp8_linear_codes)]
            self._calls = calls(rt.value, device, *entry)

    # reference constructors (src/wide_metal_moe.rs:165-171)
    @classmethod
    def compile(cls, device: int = 0) -> "WideMoeRuntime":
        return cls(device, fused_gate_up=False)

    @classmethod
    def compile_with_fused_gate_up(cls, device: int = 0) -> "WideMoeRuntime":
        return cls(device, fused_gate_up=True)

    def close(self) -> None:
        self._calls = None
        for b in self._banks:
            self._L.pw_bank_destroy(b)
        self._banks = []
        self._bank_refs = []
        if getattr(self, "_rt", None):
            self._L.pw_runtime_destroy(self._rt)
            self._rt = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------ plumbing
    def _check(self, status: int) -> None:
        if status != PW_OK:
            raise PrismwingError(status, self._L.pw_last_error(self._rt).decode())

    def last_error(self) -> str:
        return self._L.pw_last_error(self._rt).decode()

    def set_stream(self, stream: Optional[torch.cuda.Stream]) -> None:
        """Run later calls on `stream`; None: on the runtime's own stream.  torch's default stream
        (handle 0, which the C ABI takes for "the runtime's own") goes by its explicit handle."""
        handle = (stream.cuda_stream or CUDA_STREAM_LEGACY) if stream is not None else 0
        self._check(self._L.pw_set_stream(self._rt, ctypes.c_void_p(handle)))

    def synchronize(self) -> None:
        self._check(self._L.pw_synchronize(self._rt))

    def set_profiling(self, enable: bool) -> None:
        """Per-kernel CUDA-event timing of subsequent synchronous calls."""
        self._check(self._L.pw_set_profiling(self._rt, 1 if enable else 0))

    def last_profile(self) -> dict:
        p = Profile()
        self._check(self._L.pw_last_profile(self._rt, ctypes.byref(p)))
        return p.as_dict()

    def error_flags(self) -> int:
        f = ctypes.c_uint32()
        self._check(self._L.pw_read_error_flags(self._rt, ctypes.byref(f)))
        return f.value

    def _io(self, x, out_shape, out_dtype=torch.float32):
        x = _as_f32(x)
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        dev = x.device if x.is_cuda else torch.device("cpu")
        out = torch.empty(out_shape, dtype=out_dtype, device=dev)
        return x, out, mem

    # -------------------------------------------------------- primitives
    def quantize(self, x):
        """dynamic_fp8_activations (src/text_endpoint.rs:3008) -> (codes u8, scales f32)."""
        x = _as_f32(x)
        rows, cols = x.shape
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        codes = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
        scales = torch.empty((rows, cols // 128 if cols % 128 == 0 else 1), dtype=torch.float32, device=x.device)
        self._check(self._L.pw_quantize_fp8(self._rt, ctypes.c_void_p(x.data_ptr()), rows, cols,
                                            ctypes.c_void_p(codes.data_ptr()), ctypes.c_void_p(scales.data_ptr()),
                                            mem))
        return codes, scales

    def validate(self, binding: WideProjectionBinding) -> None:
        """validate_fp8_views_internal (src/lib.rs:1217); raises on a bad byte or scale."""
        t = binding.c()
        bad = ctypes.c_uint64()
        self._check(self._L.pw_validate_fp8(self._rt, ctypes.byref(t), ctypes.byref(bad)))

    def _io_async(self, x, out_shape, asynchronous, out):
        """(x, out, mem, stats pointer) for a call that may be enqueued without
        waiting (PW_MEM_ASYNC: device I/O, no stats; CUDA-graph capturable once
        the same call has run before)."""
        if asynchronous:
            if not x.is_cuda:
                raise PrismwingError(-1, "asynchronous calls need device I/O")
            if out is None:
                out = torch.empty(out_shape, dtype=torch.float32, device=x.device)
            return x, out, MEM_DEVICE | MEM_ASYNC, None
        x, o, mem = self._io(x, out_shape)
        return x, (out if out is not None and x.is_cuda else o), mem, Stats()

    def fp8_gemv(self, x, binding: WideProjectionBinding, asynchronous: bool = False,
                 out: Optional[torch.Tensor] = None) -> Execution:
        """Readable projection (src/lib.rs:1272 mapped_fp8_gemv): x f32 [w, cols] -> f32 [w, rows]."""
        x = _as_f32(x)
        if x.dim() == 1:
            x = x.unsqueeze(0)
        x, out, mem, st = self._io_async(x, (x.shape[0], binding.rows), asynchronous, out)
        t = binding.c()
        self._check(self._L.pw_fp8_gemv(self._rt, ctypes.byref(t), ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                        ctypes.c_void_p(out.data_ptr()), mem, ctypes.byref(st) if st else None))
        return Execution(out, st.wall_ms if st else 0.0, st.device_ms if st else 0.0,
                         weight_bytes=st.weight_bytes if st else 0)

    def execute_fp8_linear(self, x, binding: WideProjectionBinding, full_qkv_layout: bool = False,
                           layout: Optional[int] = None, f32_output: bool = False, asynchronous: bool = False,
                           out: Optional[torch.Tensor] = None) -> Execution:
        """src/wide_metal_moe.rs:241: quantize, block-scaled projection, bf16 round.

        Like the reference, a [14848, 4096] projection selects the SWA-QKV row map
        and full_qkv_layout=True the full-QKV map.  f32_output skips the final
        bf16 round (PW_OUTPUT_F32)."""
        x = _as_f32(x)
        if layout is None:
            if full_qkv_layout:
                layout = LAYOUT_FULL_QKV
            elif binding.rows == 14848 and binding.columns == 4096:
                layout = LAYOUT_SWA_QKV
            else:
                layout = LAYOUT_PLAIN
        if f32_output:
            layout |= OUTPUT_F32
        x, out, mem, st = self._io_async(x, (x.shape[0], binding.rows), asynchronous, out)
        t = binding.c()
        self._check(self._L.pw_fp8_linear(self._rt, ctypes.byref(t), layout, ctypes.c_void_p(x.data_ptr()),
                                          x.shape[0], ctypes.c_void_p(out.data_ptr()), mem,
                                          ctypes.byref(st) if st else None))
        return Execution(out, st.wall_ms if st else 0.0, st.device_ms if st else 0.0,
                         weight_bytes=st.weight_bytes if st else 0)

    def expert_forward(self, x, gate: WideProjectionBinding, up: WideProjectionBinding,
                       down: WideProjectionBinding, asynchronous: bool = False,
                       out: Optional[torch.Tensor] = None) -> Execution:
        """One routed expert at weight 1 (src/text_endpoint.rs:5311-5346)."""
        x = _as_f32(x)
        x, out, mem, st = self._io_async(x, (x.shape[0], down.rows), asynchronous, out)
        w = ExpertWeights(gate.c(), up.c(), down.c())
        self._check(self._L.pw_expert_forward(self._rt, ctypes.byref(w), ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                              ctypes.c_void_p(out.data_ptr()), mem,
                                              ctypes.byref(st) if st else None))
        return Execution(out, st.wall_ms if st else 0.0, st.device_ms if st else 0.0,
                         weight_bytes=st.weight_bytes if st else 0)

    def dense_mlp(self, x, gate: WideProjectionBinding, up: WideProjectionBinding,
                  down: WideProjectionBinding) -> Execution:
        """dense_mlp (src/text_endpoint.rs:4266): layer 0's dense FP8 MLP
        (gate/up [16384, 4096], down [4096, 16384] for MiMo-V2.5)."""
        x = _as_f32(x)
        x, out, mem = self._io(x, (x.shape[0], down.rows))
        w = ExpertWeights(gate.c(), up.c(), down.c())
        st = Stats()
        self._check(self._L.pw_dense_mlp(self._rt, ctypes.byref(w), ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                         ctypes.c_void_p(out.data_ptr()), mem, ctypes.byref(st)))
        return Execution(out, st.wall_ms, st.device_ms, weight_bytes=st.weight_bytes)

    def route(self, x, router_weight: torch.Tensor, bias: torch.Tensor):
        """route_mlp + pytorch_noaux_routes (src/text_endpoint.rs:4342-4470).

        router_weight: CUDA [E, H], float32 (the checkpoint's F32 gate.weight) or
        bf16 (or int16 bits); bias CUDA f32 [E].
        Returns (selected int64 [T, 8], weights f32 [T, 8], stats dict)."""
        x = _as_f32(x)
        r = self._router(router_weight, bias)
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        sel = torch.empty((x.shape[0], 8), dtype=torch.int32, device=x.device)
        wts = torch.empty((x.shape[0], 8), dtype=torch.float32, device=x.device)
        st = Stats()
        self._check(self._L.pw_route(self._rt, ctypes.byref(r), ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                     ctypes.c_void_p(sel.data_ptr()), ctypes.c_void_p(wts.data_ptr()), mem,
                                     ctypes.byref(st)))
        return sel.long() & 0xFFFFFFFF, wts, st.as_dict()

    @staticmethod
    def _router(w: torch.Tensor, bias: torch.Tensor) -> Router:
        """pw_router for a CUDA float32 (PW_ROUTER_F32) or bf16/int16 (PW_ROUTER_BF16) weight."""
        if w.dtype == torch.float32:
            dtype = ROUTER_F32
        elif w.dtype in (torch.bfloat16, torch.int16):
            dtype = ROUTER_BF16
        else:
            raise PrismwingError(-1, f"router weight must be float32 or bf16, not {w.dtype}")
        if not (w.is_cuda and bias.is_cuda and bias.dtype == torch.float32):
            raise PrismwingError(-1, "router weight and bias must be CUDA tensors, bias float32")
        if not (w.is_contiguous() and bias.is_contiguous()):
            raise PrismwingError(-1, "router tensors must be contiguous")
        return Router(w.data_ptr(), bias.data_ptr(), w.shape[0], w.shape[1], 8, dtype)

    @staticmethod
    def _norm(weight: torch.Tensor, epsilon: float) -> Norm:
        """pw_norm for a CUDA float32 (PW_NORM_F32) or bf16/int16 (PW_NORM_BF16) weight."""
        if weight.dtype == torch.float32:
            dtype = NORM_F32
        elif weight.dtype in (torch.bfloat16, torch.int16):
            dtype = NORM_BF16
        else:
            raise PrismwingError(-1, f"norm weight must be float32 or bf16, not {weight.dtype}")
        if not (weight.is_cuda and weight.is_contiguous() and weight.dim() == 1):
            raise PrismwingError(-1, "norm weight must be a contiguous 1-D CUDA tensor")
        return Norm(weight.data_ptr(), weight.shape[0], dtype, float(epsilon))

    def rms_norm(self, x, weight: torch.Tensor, epsilon: float = 1e-5):
        """rms_norm (src/text_endpoint.rs:2939): (y f32 [rows, H], inverse f32 [rows])."""
        x = _as_f32(x)
        n = self._norm(weight, epsilon)
        x, out, mem = self._io(x, tuple(x.shape))
        inv = torch.empty((x.shape[0],), dtype=torch.float32, device=out.device)
        self._check(self._L.pw_rms_norm(self._rt, ctypes.byref(n), ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                        ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(inv.data_ptr()), mem, None))
        return out, inv

    # ------------------------------------- residual, norm, linear layers
    # These calls take a few microseconds on the device for a single token, so
    # their host side is kept short.  An asynchronous call on device tensors goes
    # through the compiled binding where there is one (one token's linear layer 4.5 us on
    # the host, 9.5 without; the norm with all its outputs 7.5 and 14.5); what that does
    # not take (None) comes here: one check per tensor, and the descriptors (the
    # structures above) packed at once into a block that the runtime keeps (like the
    # runtime's other state, it serves one call at a time).
    _calls = None
    _NORM_ARGS = struct.Struct("=QIIf4x" + "QQII" * 4)       # Norm, then Rows of x, residual, sum, y
    _LINEAR_ARGS = struct.Struct("=QQIIII" + "QQII" + "QIIQQII" + "QQII")  # Dense, Rows of x, Epilogue, Rows of y
    _CODES_ARGS = struct.Struct("=QIIQQII" + "QQII")         # Epilogue, Rows of y

    def _init_args(self) -> None:
        self._args = ctypes.create_string_buffer(256)
        self._args_at = ctypes.addressof(self._args)

    def _rows(self, t: torch.Tensor, name: str, where: int):
        """(data, stride, dtype) of a 2-D tensor whose rows are contiguous, on device `where` (-1: the host)."""
        shape, code = t.shape, DTYPES.get(t.dtype)
        if len(shape) == 2 and code is not None and t.get_device() == where:
            rows, cols = shape
            stride, step = t.stride()
            if rows <= 1:  # one row may have any stride in torch
                stride = 0
            if (step == 1 or cols <= 1) and (stride >= cols or not stride and rows <= 1):
                return t.data_ptr(), stride, code
        if code is None:
            raise PrismwingError(-1, f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
        if t.get_device() != where:
            raise PrismwingError(-1, f"{name} is on {t.device}, not with x on the runtime's device or the host")
        raise PrismwingError(-1, f"{name} must be 2-D with contiguous rows that do not overlap")

    def _vector(self, t: torch.Tensor, name: str, n: int) -> int:
        if t.dtype not in DTYPES or t.shape != (n,) or t.get_device() != self.device or not t.is_contiguous():
            raise PrismwingError(-1, f"{name} must be a contiguous [{n}] float tensor on the runtime's device")
        return t.data_ptr()

    def _where(self, x: torch.Tensor) -> int:
        """The device index of a call's rows: the runtime's device, or -1 for the host."""
        where = x.get_device()
        if where != self.device and where != -1:
            raise PrismwingError(-1, f"x is on {x.device}, not on the runtime's device or the host")
        return where

    @staticmethod
    def _input(x) -> torch.Tensor:
        if isinstance(x, np.ndarray):
            x = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
        return x

    @staticmethod
    def _mem(where: int, asynchronous: bool):
        if asynchronous:
            if where < 0:
                raise PrismwingError(-1, "asynchronous calls need device I/O")
            return MEM_DEVICE | MEM_ASYNC, None
        return MEM_DEVICE if where >= 0 else MEM_HOST, Stats()

    def add_rms_norm(self, x, weight: torch.Tensor, epsilon: float = 1e-5, residual=None, want_y: bool = True,
                     want_codes: bool = False, out_dtype: Optional[torch.dtype] = None, in_place: bool = False,
                     asynchronous: bool = False) -> NormExecution:
        """s = x + residual in x's dtype; y = s / sqrt(mean(s^2) + epsilon) * weight, rounded once to out_dtype
        (x's, or float32); with want_codes y's e4m3 codes (uint8 [rows, hidden]) and their scales per 128 columns
        (float32 [rows, ceil(hidden / 128)]), taken from y before its rounding.  x, residual [rows, hidden],
        float32, bfloat16 or float16; weight a CUDA [hidden] of any of them.  in_place writes s over residual."""
        if asynchronous and self._calls is not None:
            ran = self._calls.add_rms_norm(x, weight, epsilon, residual, want_y, want_codes, out_dtype, in_place)
            if ran is not None:
                if ran.__class__ is int:
                    self._check(ran)
                return NormExecution(*ran)
        x = self._input(x)
        where = self._where(x)
        x_at, x_stride, dt = self._rows(x, "x", where)
        T, H = x.shape
        dtype, dev = x.dtype, x.device
        if weight.dtype not in DTYPES:
            raise PrismwingError(-1, f"norm weight must be float32, bfloat16 or float16, not {weight.dtype}")
        w_at = self._vector(weight, "norm weight", H)
        mem, st = self._mem(where, asynchronous)
        empty, at = torch.empty_strided, self._args_at
        r_at = r_stride = s_at = s_stride = y_at = y_dt = 0
        rp = sp = yp = cp = gp = total = y = codes = scales = None
        if residual is not None:
            residual = self._input(residual)
            r_at, r_stride, r_dt = self._rows(residual, "residual", where)
            if residual.shape != x.shape:
                raise PrismwingError(-2, "residual must have x's shape")
            if r_dt != dt:
                raise PrismwingError(-1, "residual must have x's dtype")
            if in_place:
                total, s_at, s_stride = residual, r_at, r_stride
            else:
                total = empty((T, H), (H, 1), dtype=dtype, device=dev)
                s_at, s_stride = total.data_ptr(), H
            rp, sp = at + 48, at + 72
        if want_y:
            if out_dtype is None:
                out_dtype = dtype
            elif out_dtype not in DTYPES:
                raise PrismwingError(-1, f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
            y = empty((T, H), (H, 1), dtype=out_dtype, device=dev)
            y_at, y_dt, yp = y.data_ptr(), DTYPES[out_dtype], at + 96
        if want_codes:
            G = (H + 127) // 128
            codes = empty((T, H), (H, 1), dtype=torch.uint8, device=dev)
            scales = empty((T, G), (G, 1), dtype=torch.float32, device=dev)
            cp, gp = codes.data_ptr(), scales.data_ptr()
        self._NORM_ARGS.pack_into(self._args, 0, w_at, H, DTYPES[weight.dtype], epsilon, x_at, x_stride, dt, 0,
                                  r_at, r_stride, dt, 0, s_at, s_stride, dt, 0, y_at, H, y_dt, 0)
        status = self._L.pw_add_rms_norm(self._rt, at, at + 24, rp, T, sp, yp, cp, gp, mem,
                                         ctypes.byref(st) if st else None)
        if status:
            self._check(status)
        return NormExecution(total, y, codes, scales)

    def _epilogue(self, where: int, dev, width: int, cols: int, bias, activation: str, residual, out_dtype, out):
        """The fields of a linear layer's pw_epilogue and of its output's pw_rows, and the output."""
        act = ACTIVATIONS.get(activation)
        if act is None:
            raise PrismwingError(-1, f"unknown activation {activation!r}")
        b_at = b_dt = r_at = r_stride = r_dt = 0
        if bias is not None:
            b_at, b_dt = self._vector(bias, "bias", cols), DTYPES[bias.dtype]
        if residual is not None:
            if residual.shape != (width, cols):
                raise PrismwingError(-2, f"residual must be [{width}, {cols}]")
            r_at, r_stride, r_dt = self._rows(residual, "residual", where)
        if out is not None:
            if out.shape != (width, cols):
                raise PrismwingError(-2, f"out must be [{width}, {cols}]")
            y_at, y_stride, y_dt = self._rows(out, "out", where)
        else:
            y_dt = DTYPES.get(out_dtype)
            if y_dt is None:
                raise PrismwingError(-1, f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
            out = torch.empty_strided((width, cols), (cols, 1), dtype=out_dtype, device=dev)
            y_at, y_stride = out.data_ptr(), cols
        return (b_at, b_dt, act, r_at, r_stride, r_dt, 0, y_at, y_stride, y_dt, 0), out

    def linear(self, x, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               asynchronous: bool = False, out: Optional[torch.Tensor] = None) -> Execution:
        """activation(x W^T + bias) + residual for a CUDA bfloat16 or float16 weight [rows, cols] whose rows start at
        16-byte boundaries (execute_bf16_linear, kernels/block_fp8_gemv.metal:358): sums in 32 bits, rounded once to
        out_dtype (x's).  x [width, cols] of the weight's dtype, or float32, which is rounded to it first; bias a
        CUDA [rows], residual [width, rows], of any float dtype; `out` may be `residual`.  activation: "none",
        "relu", "gelu", "gelu_tanh" or "silu"."""
        if asynchronous and self._calls is not None:
            ran = self._calls.linear(x, weight, bias, ACTIVATIONS.get(activation), residual, out_dtype, out)
            if ran is not None:
                if ran.__class__ is int:
                    self._check(ran)
                return Execution(ran, 0.0, 0.0)
        x = self._input(x)
        where = self._where(x)
        x_at, x_stride, x_dt = self._rows(x, "x", where)
        w_at, w_stride, w_dt = self._rows(weight, "weight", self.device)
        rows, cols = weight.shape
        width, columns = x.shape
        if columns != cols:
            raise PrismwingError(-2, f"x has {columns} columns, the weight {cols}")
        mem, st = self._mem(where, asynchronous)
        fields, out = self._epilogue(where, x.device, width, rows, bias, activation, residual, out_dtype or x.dtype, out)
        at = self._args_at
        self._LINEAR_ARGS.pack_into(self._args, 0, w_at, w_stride, rows, cols, w_dt, 0, x_at, x_stride, x_dt, 0, *fields)
        status = self._L.pw_linear(self._rt, at, at + 32, width, at + 56, at + 96, mem, ctypes.byref(st) if st else None)
        if status:
            self._check(status)
        if st is None:
            return Execution(out, 0.0, 0.0)
        return Execution(out, st.wall_ms, st.device_ms, weight_bytes=st.weight_bytes)

    def fp8_linear_codes(self, codes: torch.Tensor, scales: torch.Tensor, binding: WideProjectionBinding,
                         layout: int = LAYOUT_PLAIN, bias: Optional[torch.Tensor] = None, activation: str = "none",
                         residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
                         asynchronous: bool = False, out: Optional[torch.Tensor] = None) -> Execution:
        """execute_fp8_linear on activations that are already quantized (quantize, add_rms_norm), with linear's
        epilogue: codes uint8 [width, cols], scales float32 [width, cols / 128], both contiguous."""
        if asynchronous and self._calls is not None:
            ran = self._calls.fp8_linear_codes(codes, scales, binding.weight, binding.scale, layout, bias,
                                               ACTIVATIONS.get(activation), residual, out_dtype, out)
            if ran is not None:
                if ran.__class__ is int:
                    self._check(ran)
                return Execution(ran, 0.0, 0.0)
        if codes.dtype != torch.uint8 or scales.dtype != torch.float32 or codes.dim() != 2 or scales.dim() != 2:
            raise PrismwingError(-1, "codes must be uint8 and scales float32, both 2-D")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise PrismwingError(-1, "codes and scales must be contiguous")
        where = self._where(codes)
        if scales.get_device() != where:
            raise PrismwingError(-1, "codes and scales must both be on the runtime's device or the host")
        width, cols = codes.shape
        t = binding.c()
        if binding.weight.get_device() != self.device or binding.scale.get_device() != self.device:
            raise PrismwingError(-1, "the projection is not on the runtime's device")
        if cols != t.cols or scales.shape != (width, cols // 128):
            raise PrismwingError(-2, f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not fit a "
                                     f"[{t.rows}, {t.cols}] projection")
        mem, st = self._mem(where, asynchronous)
        fields, out = self._epilogue(where, codes.device, width, t.rows, bias, activation, residual, out_dtype, out)
        at = self._args_at
        self._CODES_ARGS.pack_into(self._args, 0, *fields)
        status = self._L.pw_fp8_linear_codes(self._rt, ctypes.byref(t), layout, codes.data_ptr(), scales.data_ptr(), width,
                                             at, at + 40, mem, ctypes.byref(st) if st else None)
        if status:
            self._check(status)
        if st is None:
            return Execution(out, 0.0, 0.0)
        return Execution(out, st.wall_ms, st.device_ms, weight_bytes=st.weight_bytes)

    # ------------------------------------------------------------ layers
    def execute(self, x, experts: Sequence[WideExpertBinding]) -> Execution:
        """src/wide_metal_moe.rs:836 execute: host-built schedule, whole layer on device."""
        return self._execute(x, experts)

    def execute_fused_gate_up(self, x, experts: Sequence[WideExpertBinding]) -> Execution:
        """src/wide_metal_moe.rs:844 execute_fused_gate_up (this runtime must be fused)."""
        if not self.fused_gate_up:
            raise PrismwingError(-1, "fused gate/up pipelines were not requested")
        return self._execute(x, experts)

    def _execute(self, x, experts: Sequence[WideExpertBinding]) -> Execution:
        x = _as_f32(x)
        rows = x.shape[0]
        x, out, mem = self._io(x, (rows, x.shape[1]))
        arr = (ExpertBinding * len(experts))()
        keep = []
        for i, e in enumerate(experts):
            pos = np.ascontiguousarray(np.asarray(e.positions, dtype=np.uint32))
            wts = np.ascontiguousarray(np.asarray(e.route_weights, dtype=np.float32))
            keep += [pos, wts]
            arr[i] = ExpertBinding(e.expert, len(pos), pos.ctypes.data, wts.ctypes.data, e.weights_c())
        st = Stats()
        self._check(self._L.pw_moe_execute(self._rt, ctypes.c_void_p(x.data_ptr()), rows, arr, len(experts),
                                           ctypes.c_void_p(out.data_ptr()), mem, ctypes.byref(st)))
        return Execution(out, st.wall_ms, st.device_ms, st.unique_experts, st.expert_rows, weight_bytes=st.weight_bytes)

    def create_bank(self, experts: Sequence[tuple]) -> ctypes.c_void_p:
        """Register experts [(gate, up, down) WideProjectionBinding triples]; validates every byte."""
        arr = (ExpertWeights * len(experts))()
        for i, (g, u, d) in enumerate(experts):
            arr[i] = ExpertWeights(g.c(), u.c(), d.c())
        bank = ctypes.c_void_p()
        self._check(self._L.pw_bank_create(self._rt, arr, len(experts), ctypes.byref(bank)))
        self._banks.append(bank)
        # the library keeps raw device pointers: hold the tensors as long as the bank
        self._bank_refs.append(list(experts))
        return bank

    # ------------------------------------------------- expert parallelism
    @staticmethod
    def ep_unique_id() -> bytes:
        """A fresh NCCL communicator id (128 bytes) for pw_ep_init; create it on
        one rank and send it to the others."""
        L = _lib.load()
        buf = ctypes.create_string_buffer(128)
        rc = L.pw_ep_unique_id(buf, 128)
        if rc != 0:
            raise PrismwingError(rc, "pw_ep_unique_id failed (is libnccl.so.2 loadable?)")
        return buf.raw

    def ep_init(self, rank: int, world: int, uid: bytes, timeout_ms: int = 60000, max_tokens: int = 2048,
                hidden: int = 0, local_experts: int = 0, nccl_transport: bool = False) -> None:
        """Join the expert-parallel group (collective).  max_tokens bounds the
        tokens per rank and layer (same on every rank); with hidden and
        local_experts the peer-memory windows are mapped here; nccl_transport
        moves the rows with NCCL send/recv instead of peer-memory stores."""
        buf = ctypes.create_string_buffer(bytes(uid), len(uid))
        self._check(self._L.pw_ep_init(self._rt, rank, world, buf, len(uid), timeout_ms, max_tokens, hidden,
                                       local_experts, EP_NCCL_TRANSPORT if nccl_transport else 0))

    def ep_moe_layer(self, x, router_weight: torch.Tensor, bias: torch.Tensor, bank,
                     want_routes: bool = False, stats: bool = True, asynchronous: bool = False,
                     out: Optional[torch.Tensor] = None) -> Execution:
        """Collective routed layer over this rank's tokens; `bank` holds this
        rank's experts (rank g: experts [g n, (g + 1) n))."""
        x = _as_f32(x)
        T, H = x.shape
        r = self._router(router_weight, bias)
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        if asynchronous:
            if not x.is_cuda:
                raise PrismwingError(-1, "asynchronous calls need device I/O")
            mem |= MEM_ASYNC
            stats = False
        if out is None:
            out = torch.empty((T, H), dtype=torch.float32, device=x.device)
        sel = torch.empty((T, 8), dtype=torch.int32, device=x.device) if want_routes else None
        wts = torch.empty((T, 8), dtype=torch.float32, device=x.device) if want_routes else None
        st = Stats()
        self._check(self._L.pw_ep_moe_layer(
            self._rt, ctypes.byref(r), bank, ctypes.c_void_p(x.data_ptr() if T else 0), T,
            ctypes.c_void_p(out.data_ptr() if T else 0),
            ctypes.c_void_p(sel.data_ptr() if sel is not None and T else 0),
            ctypes.c_void_p(wts.data_ptr() if wts is not None and T else 0), mem,
            ctypes.byref(st) if stats else None))
        return Execution(out, st.wall_ms, st.device_ms, st.unique_experts, st.expert_rows, st.boundary_tie_rows,
                         st.weight_bytes, sel, wts)

    def moe_layer(self, x, router_weight: torch.Tensor, bias: torch.Tensor, bank,
                  want_routes: bool = False, stats: bool = True, asynchronous: bool = False,
                  out: Optional[torch.Tensor] = None) -> Execution:
        """routed_mlp_metal_wide_configured (src/text_endpoint.rs:4750) fully on the device."""
        x = _as_f32(x)
        T, H = x.shape
        r = self._router(router_weight, bias)
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        if asynchronous:
            if not x.is_cuda:
                raise PrismwingError(-1, "asynchronous calls need device I/O")
            mem |= MEM_ASYNC
            stats = False
        if out is None:
            out = torch.empty((T, H), dtype=torch.float32, device=x.device)
        sel = torch.empty((T, 8), dtype=torch.int32, device=x.device) if want_routes else None
        wts = torch.empty((T, 8), dtype=torch.float32, device=x.device) if want_routes else None
        st = Stats()
        self._check(self._L.pw_moe_layer(
            self._rt, ctypes.byref(r), bank, ctypes.c_void_p(x.data_ptr()), T, ctypes.c_void_p(out.data_ptr()),
            ctypes.c_void_p(sel.data_ptr() if sel is not None else 0),
            ctypes.c_void_p(wts.data_ptr() if wts is not None else 0), mem,
            ctypes.byref(st) if stats else None))
        return Execution(out, st.wall_ms, st.device_ms, st.unique_experts, st.expert_rows, st.boundary_tie_rows,
                         st.weight_bytes, sel, wts)

    def moe_block(self, residual, norm_weight: torch.Tensor, epsilon: float, router_weight: torch.Tensor,
                  bias: torch.Tensor, bank, want_routes: bool = False, stats: bool = True,
                  asynchronous: bool = False, out: Optional[torch.Tensor] = None, expert_parallel: bool = False
                  ) -> Execution:
        """The MoE half of a decoder layer (src/text_endpoint.rs:5507-5580):
        out = bf16(residual + routed_layer(rms_norm(residual))).  With
        expert_parallel the call is pw_ep_moe_block (collective)."""
        x = _as_f32(residual)
        T, H = x.shape
        n = self._norm(norm_weight, epsilon)
        r = self._router(router_weight, bias)
        mem = MEM_DEVICE if x.is_cuda else MEM_HOST
        if asynchronous:
            if not x.is_cuda:
                raise PrismwingError(-1, "asynchronous calls need device I/O")
            mem |= MEM_ASYNC
            stats = False
        if out is None:
            out = torch.empty((T, H), dtype=torch.float32, device=x.device)
        sel = torch.empty((T, 8), dtype=torch.int32, device=x.device) if want_routes else None
        wts = torch.empty((T, 8), dtype=torch.float32, device=x.device) if want_routes else None
        st = Stats()
        fn = self._L.pw_ep_moe_block if expert_parallel else self._L.pw_moe_block
        self._check(fn(self._rt, ctypes.byref(n), ctypes.byref(r), bank, ctypes.c_void_p(x.data_ptr() if T else 0), T,
                       ctypes.c_void_p(out.data_ptr() if T else 0),
                       ctypes.c_void_p(sel.data_ptr() if sel is not None and T else 0),
                       ctypes.c_void_p(wts.data_ptr() if wts is not None and T else 0), mem,
                       ctypes.byref(st) if stats else None))
        return Execution(out, st.wall_ms, st.device_ms, st.unique_experts, st.expert_rows, st.boundary_tie_rows,
                         st.weight_bytes, sel, wts)
