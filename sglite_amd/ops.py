"""Torch custom ops over the C ABI (namespace ``torch.ops.sglite_awq``).

PyTorch supplies device memory and the current HIP stream; all arithmetic runs
in the HIP kernels of libsglite_awq.so.  Every C-ABI entry point that launches
work is registered with ``torch.library.custom_op`` and a fake (meta)
implementation, so the ops are visible to ``torch.ops``, FakeTensor shape
propagation and ``torch.compile``; this replaces the reference's dispatch
through its torch ops ``sgl_kernel.gptq_marlin_gemm`` and
``sgl_kernel.awq_marlin_repack``
(python/sglite/srt/model_executor/layers/quantization/marlin_utils.py:388-410,
awq_marlin.py:300-305).

Every op launches on ``torch.cuda.current_stream()`` of its tensors' device,
never synchronises and allocates only through torch's caching allocator, so
it can be captured in a ``torch.cuda.graph``.  The plain-Python functions
below (``gemm``, ``repack`` ...) are the wrappers the linear methods call;
they validate arguments and call the registered ops.
"""

from __future__ import annotations

import contextlib
import ctypes
import threading
from typing import Dict, Iterator, List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch._subclasses.fake_tensor import is_fake

from . import _lib

NAMESPACE = "sglite_awq"
_DTYPE_CODE = {torch.float16: _lib.AWQ_DTYPE_FP16, torch.bfloat16: _lib.AWQ_DTYPE_BF16}
SUPPORTED_GROUP_SIZES = (-1, 32, 64, 128)


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise ValueError(f"AWQ W4A16 supports float16 and bfloat16 activations/scales, got {dtype}") from None


def _stream(device: torch.device) -> int:
    if device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return torch._C._cuda_getCurrentRawStream(device.index)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("AWQ HIP kernels need device tensors")


def _aligned(t: torch.Tensor, a: int = 16) -> torch.Tensor:
    """Contiguous and ``a``-byte aligned (a fresh allocation is 256-byte aligned)."""
    if t.is_contiguous() and t.data_ptr() % a == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


@contextlib.contextmanager
def _on_device(device: torch.device) -> Iterator[None]:
    """Make ``device`` current for the C ABI's planning (it fills that device's CUs)."""
    if device.index is None or torch.cuda.current_device() == device.index:
        yield
    else:
        with torch.cuda.device(device):
            yield


# Tensors without handlers of their own (a Parameter has none), compared exactly: subclasses may bring some.
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _undispatched(*tensors: Optional[torch.Tensor]) -> bool:
    """True where the dispatcher would only hand these tensors on to the device implementation: plain tensors
    and Parameters outside every mode, trace, transform, profiler and gradient.  A call may then run that
    implementation itself, without the dispatcher's Python layers (a loaded 4096 x 2560 layer called eagerly at
    M = 1, a call among others: 18.5 us through them, 11.8 without)."""
    if torch.compiler.is_compiling():  # first: a tracing compiler takes it as a constant and looks no further
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or t.is_neg() or torch._is_functional_tensor(t)
                              or (grad and t.requires_grad)):
            return False
    return (torch._C._len_torch_dispatch_stack() == 0 and torch._C._len_torch_function_stack() == 0
            and torch._C._functorch.peek_interpreter_stack() is None and torch._C._get_tracing_state() is None
            and torch.autograd.forward_ad._current_level < 0 and not torch._C._autograd._profiler_enabled())


def resolve_group_size(group_size: int, K: int) -> int:
    return K if group_size == -1 else group_size


class Repacked(NamedTuple):
    """Repacked tensors of one linear in the CDNA4 tile layout."""
    w: torch.Tensor  # int32 [NT * KT * 256]
    s: torch.Tensor  # scale dtype [NT, NG, 16]
    z: torch.Tensor  # int64 [NT, NG]  (16 zero nibbles per word)


def repacked_sizes(K: int, N: int, group_size: int) -> Tuple[int, int, int]:
    lib = _lib.load()
    G = resolve_group_size(group_size, K)
    wb = _lib.check(lib.awq_repacked_weight_bytes(K, N), "awq_repacked_weight_bytes")
    sb = _lib.check(lib.awq_repacked_scale_bytes(K, N, G), "awq_repacked_scale_bytes")
    zb = _lib.check(lib.awq_repacked_zero_bytes(K, N, G), "awq_repacked_zero_bytes")
    return wb, sb, zb


def _check_awq_shapes(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> Tuple[int, int, int]:
    if qweight.dtype != torch.int32 or qzeros.dtype != torch.int32:
        raise ValueError("qweight and qzeros must be int32")
    if qweight.dim() != 2 or qzeros.dim() != 2 or scales.dim() != 2:
        raise ValueError("qweight, qzeros and scales must be 2-D")
    K, N8 = qweight.shape
    N = N8 * 8
    ng = qzeros.shape[0]
    if ng == 0 or K % ng:
        raise ValueError(f"qzeros rows ({ng}) must divide K ({K})")
    G = K // ng
    if qzeros.shape[1] != N8 or tuple(scales.shape) != (ng, N):
        raise ValueError(f"inconsistent AWQ shapes: qweight {tuple(qweight.shape)}, qzeros {tuple(qzeros.shape)}, "
                         f"scales {tuple(scales.shape)}")
    return K, N, G


# ---------------------------------------------------------------------------
# Registered ops: repack / unrepack / dequantisation probes.
# ---------------------------------------------------------------------------

@torch.library.custom_op(f"{NAMESPACE}::awq_repack_cdna4", mutates_args=(), device_types="cuda")
def _repack_op(qweight: torch.Tensor, qzeros: torch.Tensor,
               scales: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    K, N, G = _check_awq_shapes(qweight, qzeros, scales)
    code = dtype_code(scales.dtype)
    wb, sb, zb = repacked_sizes(K, N, G)
    dev = qweight.device
    NT, NG = (N + 15) // 16, K // G
    w = torch.empty(wb // 4, dtype=torch.int32, device=dev)
    s = torch.empty((NT, NG, 16), dtype=scales.dtype, device=dev)
    z = torch.empty((NT, NG), dtype=torch.int64, device=dev)
    assert s.numel() * 2 == sb and z.numel() * 8 == zb
    qweight, qzeros, scales = qweight.contiguous(), qzeros.contiguous(), scales.contiguous()
    with _on_device(dev):
        _lib.check(_lib.load().awq_repack_cdna4(qweight.data_ptr(), qzeros.data_ptr(), scales.data_ptr(), code, K, N,
                                                G, w.data_ptr(), s.data_ptr(), z.data_ptr(), _stream(dev)),
                   "awq_repack_cdna4")
    return w, s, z


@_repack_op.register_fake
def _(qweight, qzeros, scales):
    K, N8 = qweight.shape
    N, NG = N8 * 8, qzeros.shape[0]
    NT, KT = (N + 15) // 16, (K + 127) // 128
    return (qweight.new_empty(NT * KT * 256), scales.new_empty((NT, NG, 16)),
            qweight.new_empty((NT, NG), dtype=torch.int64))


@torch.library.custom_op(f"{NAMESPACE}::awq_unrepack_cdna4", mutates_args=(), device_types="cuda")
def _unrepack_op(w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, K: int, N: int,
                 G: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dev = w.device
    qweight = torch.empty((K, N // 8), dtype=torch.int32, device=dev)
    qzeros = torch.empty((K // G, N // 8), dtype=torch.int32, device=dev)
    scales = torch.empty((K // G, N), dtype=s.dtype, device=dev)
    with _on_device(dev):
        _lib.check(_lib.load().awq_unrepack_cdna4(w.data_ptr(), s.data_ptr(), z.data_ptr(), dtype_code(s.dtype), K, N,
                                                  G, qweight.data_ptr(), qzeros.data_ptr(), scales.data_ptr(),
                                                  _stream(dev)), "awq_unrepack_cdna4")
    return qweight, qzeros, scales


@_unrepack_op.register_fake
def _(w, s, z, K, N, G):
    return (w.new_empty((K, N // 8)), w.new_empty((K // G, N // 8)), s.new_empty((K // G, N)))


@torch.library.custom_op(f"{NAMESPACE}::awq_dequant", mutates_args=(), device_types="cuda")
def _dequant_op(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    K, N, G = _check_awq_shapes(qweight, qzeros, scales)
    out = torch.empty((K, N), dtype=scales.dtype, device=qweight.device)
    with _on_device(qweight.device):
        _lib.check(_lib.load().awq_dequant(qweight.contiguous().data_ptr(), qzeros.contiguous().data_ptr(),
                                           scales.contiguous().data_ptr(), dtype_code(scales.dtype), K, N, G,
                                           out.data_ptr(), _stream(qweight.device)), "awq_dequant")
    return out


@_dequant_op.register_fake
def _(qweight, qzeros, scales):
    return scales.new_empty((qweight.shape[0], qweight.shape[1] * 8))


@torch.library.custom_op(f"{NAMESPACE}::awq_dequant_repacked", mutates_args=(), device_types="cuda")
def _dequant_repacked_op(w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, K: int, N: int, G: int) -> torch.Tensor:
    out = torch.empty((K, N), dtype=s.dtype, device=w.device)
    with _on_device(w.device):
        _lib.check(_lib.load().awq_dequant_repacked(w.data_ptr(), s.data_ptr(), z.data_ptr(), dtype_code(s.dtype), K,
                                                    N, G, out.data_ptr(), _stream(w.device)), "awq_dequant_repacked")
    return out


@_dequant_repacked_op.register_fake
def _(w, s, z, K, N, G):
    return s.new_empty((K, N))


def repack(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> Repacked:
    """AWQ checkpoint tensors -> CDNA4 tile layout (device side, no host copy)."""
    _require_cuda(qweight, qzeros, scales)
    _check_awq_shapes(qweight, qzeros, scales)
    dtype_code(scales.dtype)
    return Repacked(*torch.ops.sglite_awq.awq_repack_cdna4(qweight, qzeros, scales))


def unrepack(r: Repacked, K: int, N: int, group_size: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """CDNA4 tile layout -> AWQ (qweight, qzeros, scales)."""
    _require_cuda(r.w, r.s, r.z)
    return tuple(torch.ops.sglite_awq.awq_unrepack_cdna4(r.w, r.s, r.z, K, N, resolve_group_size(group_size, K)))


def dequant(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """W[K, N] = rnd((q - z) * s) from AWQ tensors (bit-exact probe)."""
    _require_cuda(qweight, qzeros, scales)
    _check_awq_shapes(qweight, qzeros, scales)
    return torch.ops.sglite_awq.awq_dequant(qweight, qzeros, scales)


def dequant_repacked(r: Repacked, K: int, N: int, group_size: int) -> torch.Tensor:
    """W[K, N] from the repacked tensors, via Dq<>::word (the prefill and MoE kernels' dequant routine)."""
    _require_cuda(r.w, r.s, r.z)
    return torch.ops.sglite_awq.awq_dequant_repacked(r.w, r.s, r.z, K, N, resolve_group_size(group_size, K))


# ---------------------------------------------------------------------------
# Planning queries and overrides.
# ---------------------------------------------------------------------------

def workspace_bytes(M: int, N: int, K: int, group_size: int) -> int:
    G = resolve_group_size(group_size, K)
    return _lib.check(_lib.load().awq_workspace_bytes(M, N, K, G), "awq_workspace_bytes")


def workspace_bytes_act(M: int, N: int, K: int, group_size: int) -> int:
    """Split-K workspace of ``gemm(..., activation=...)`` (its plan pairs gate and up tiles)."""
    G = resolve_group_size(group_size, K)
    return _lib.check(_lib.load().awq_workspace_bytes_act(M, N, K, G), "awq_workspace_bytes_act")


KERNEL_NAMES = {0: "skinny_kernel", 1: "tiled_kernel", 2: "gemv_kernel", 3: "kslice_kernel"}


def gemm_kernel(M: int, N: int, K: int, group_size: int, activation: Optional[str] = None) -> str:
    """Name of the kernel kind ``gemm`` plans for this shape (with ``activation``:
    the fused gate/up GEMM's); ``launch_info`` names the function that runs."""
    G = resolve_group_size(group_size, K)
    lib = _lib.load()
    if activation is None:
        return KERNEL_NAMES[_lib.check(lib.awq_gemm_kernel_kind(M, N, K, G), "awq_gemm_kernel_kind")]
    return KERNEL_NAMES[_lib.check(lib.awq_gemm_kernel_kind_act(M, N, K, G), "awq_gemm_kernel_kind_act")]


class PlanInfo(NamedTuple):
    kernel: str           # kernel kind (KERNEL_NAMES): which family and planner branch
    variant: int
    k_slices: int
    workgroups: int
    threads: int
    workspace_bytes: int
    function: str = ""    # the __global__ function the GEMM launch runs
    fixup: bool = False   # split K summed inside the GEMM kernel (no second launch, given counters)
    ring: int = 0         # shape code of ring_kernel where the launch takes it in place of ``function`` (17-64 rows)
    ring_slices: int = 0  # ... and its k-slices


def kernel_function(kind: str, variant: int) -> str:
    """Name of the HIP kernel a plan's GEMM launch runs: the tiled kind runs
    ``tiled_kernel`` for row-block codes below 1000 (16x16x32 MFMAs) and
    ``mfma32_kernel`` for the others (32x32x16 MFMAs)."""
    if kind == "tiled_kernel" and variant >= 1000:
        return "mfma32_kernel"
    return kind


def plan_info(M: int, N: int, K: int, group_size: int, activation: Optional[str] = None) -> PlanInfo:
    """The plan of ``gemm`` for this shape on the current device: what it launches, except where ``ring`` names
    the form of ring_kernel that runs in its place (``launch_info``)."""
    G = resolve_group_size(group_size, K)
    info = (ctypes.c_int64 * 6)()
    act = 0 if activation is None else _GATED_ACT[activation]
    lib = _lib.load()
    _lib.check(lib.awq_gemm_plan_info(M, N, K, G, act, info), "awq_gemm_plan_info")
    fixup = _lib.check(lib.awq_gemm_plan_fixup(M, N, K, G, act), "awq_gemm_plan_fixup") == 1
    slices = ctypes.c_int()
    ring = _lib.check(lib.awq_gemm_plan_ring(M, N, K, G, act, ctypes.byref(slices)), "awq_gemm_plan_ring")
    kind = KERNEL_NAMES[int(info[0])]
    return PlanInfo(kind, *[int(v) for v in info[1:]], function=kernel_function(kind, int(info[1])), fixup=fixup,
                    ring=ring, ring_slices=slices.value)


def launch_info(M: int, N: int, K: int, group_size: int, activation: Optional[str] = None) -> PlanInfo:
    """``plan_info`` with the function, shape code, k-slices, workgroups and threads that ``gemm`` launches."""
    plan = plan_info(M, N, K, group_size, activation)
    if not plan.ring:
        return plan
    info = (ctypes.c_int64 * 6)()
    act = 0 if activation is None else _GATED_ACT[activation]
    _lib.check(_lib.load().awq_gemm_launch_info(M, N, K, resolve_group_size(group_size, K), act, info),
               "awq_gemm_launch_info")
    return plan._replace(variant=int(info[1]), k_slices=int(info[2]), workgroups=int(info[3]), threads=int(info[4]),
                         function="ring_kernel")


PLAN_KNOBS = {"gemv_max_m": _lib.AWQ_PLAN_GEMV_MAX_M, "gemv_variant": _lib.AWQ_PLAN_GEMV_VARIANT,
              "gemv_ks": _lib.AWQ_PLAN_GEMV_KS, "skinny_variant": _lib.AWQ_PLAN_SKINNY_VARIANT,
              "skinny_ks": _lib.AWQ_PLAN_SKINNY_KS, "tiled_min_m": _lib.AWQ_PLAN_TILED_MIN_M,
              "tiled_bm": _lib.AWQ_PLAN_TILED_BM, "tiled_ks": _lib.AWQ_PLAN_TILED_KS,
              "kslice_variant": _lib.AWQ_PLAN_KSLICE_VARIANT, "tiled_fixup": _lib.AWQ_PLAN_TILED_FIXUP,
              "fixup_polls": _lib.AWQ_PLAN_FIXUP_POLLS, "ring": _lib.AWQ_PLAN_RING,
              "ring_ks": _lib.AWQ_PLAN_RING_KS}


def set_plan_override(knob: str, value: int) -> None:
    """Force a planner choice for every later GEMM of the process (tests and sweeps)."""
    _lib.check(_lib.load().awq_set_plan_override(PLAN_KNOBS[knob], int(value)), "awq_set_plan_override")


def clear_plan_overrides() -> None:
    _lib.load().awq_clear_plan_overrides()


@contextlib.contextmanager
def plan_overrides(**knobs: int) -> Iterator[None]:
    """``with plan_overrides(gemv_max_m=0, skinny_variant=10104): ...`` -- all overrides are cleared on exit."""
    try:
        for k, v in knobs.items():
            set_plan_override(k, v)
        yield
    finally:
        clear_plan_overrides()


def device_cu_count() -> int:
    return int(_lib.load().awq_device_cu_count())


def make_counters(N: int, device: torch.device) -> torch.Tensor:
    """Split-K counters (awq_counter_bytes): zeroed once here; every GEMM call leaves them valid for the
    next, whatever its shape (torch allocations are 512-byte aligned, as the 128 the library needs)."""
    nbytes = _lib.check(_lib.load().awq_counter_bytes(N), "awq_counter_bytes")
    return torch.zeros(nbytes // 4, dtype=torch.int32, device=device)


def counters_settled(counters: torch.Tensor) -> bool:
    """True when no GEMM is in flight on ``counters``: the decode kernels' per-column-tile counters are
    zero and every split tile of the tiled kernels has as many arrivals as its base (each launch that
    split a tile advanced both by its k-slice count)."""
    nt = _lib.AWQ_COUNTER_TILE_BYTES // 4
    tiles = counters[:nt].view(-1, 32)
    return bool(torch.equal(tiles[:, 0], tiles[:, 1])) and int(counters[nt:].abs().sum()) == 0


# ---------------------------------------------------------------------------
# Workspace of split-K sums and of the adapters' A x: one growing buffer per
# (device, stream) of a thread for eager calls (the reference sizes its Marlin
# workspace once at load, awq_marlin.py:298).  A call may launch two kernels,
# and another thread's launch on the same stream may come between them (the C
# call runs without the interpreter's lock): with a buffer of its own it leaves
# the first one's sums alone.  A call being captured into a graph takes a fresh
# buffer from the graph's pool instead, so that replays never share eager memory.
# ---------------------------------------------------------------------------

class _Workspaces(threading.local):
    def __init__(self) -> None:
        self.buffers: Dict[Tuple[int, int], torch.Tensor] = {}


_WS = _Workspaces()


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    if nbytes <= 0:
        return None
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream(device))
    buf = _WS.buffers.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WS.buffers[key] = buf
    return buf


_GATED_ACT = {"silu": _lib.AWQ_ACT_SILU, "gelu": _lib.AWQ_ACT_GELU}


def _gemm_launch(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, bias: Optional[torch.Tensor],
                 counters: Optional[torch.Tensor], out: torch.Tensor, K: int, N: int, G: int, act: int) -> None:
    M = x.shape[0]
    if M == 0:
        return
    dev = x.device
    if dev.index is not None and torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):  # the C ABI's planning fills the current device's CUs
            return _gemm_launch(x, w, s, z, bias, counters, out, K, N, G, act)
    lib = _lib.load()
    if act == 0:
        wsb = _lib.check(lib.awq_workspace_bytes(M, N, K, G), "awq_workspace_bytes")
    else:
        wsb = _lib.check(lib.awq_workspace_bytes_act(M, N, K, G), "awq_workspace_bytes_act")
    ws = _workspace(wsb, dev)
    cb = 0 if counters is None else counters.numel() * 4
    if act == 0:
        _lib.check(lib.awq_w4a16_gemm(x.data_ptr(), w.data_ptr(), s.data_ptr(), z.data_ptr(), _ptr(bias),
                                      out.data_ptr(), M, N, K, G, dtype_code(x.dtype), _ptr(ws), wsb,
                                      _ptr(counters), cb, _stream(dev)), "awq_w4a16_gemm")
    else:
        _lib.check(lib.awq_w4a16_gemm_act(x.data_ptr(), w.data_ptr(), s.data_ptr(), z.data_ptr(), _ptr(bias),
                                          out.data_ptr(), M, N, K, G, dtype_code(x.dtype), act, _ptr(ws), wsb,
                                          _ptr(counters), cb, _stream(dev)), "awq_w4a16_gemm_act")


@torch.library.custom_op(f"{NAMESPACE}::awq_w4a16_gemm", mutates_args=("counters",), device_types="cuda")
def _gemm_op(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, bias: Optional[torch.Tensor],
             counters: Optional[torch.Tensor], K: int, N: int, G: int) -> torch.Tensor:
    out = torch.empty((x.shape[0], N), dtype=x.dtype, device=x.device)
    _gemm_launch(x, w, s, z, bias, counters, out, K, N, G, 0)
    return out


@_gemm_op.register_fake
def _(x, w, s, z, bias, counters, K, N, G):
    return x.new_empty((x.shape[0], N))


@torch.library.custom_op(f"{NAMESPACE}::awq_w4a16_gemm_out", mutates_args=("counters", "out"), device_types="cuda")
def _gemm_out_op(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, bias: Optional[torch.Tensor],
                 counters: Optional[torch.Tensor], out: torch.Tensor, K: int, N: int, G: int) -> None:
    _gemm_launch(x, w, s, z, bias, counters, out, K, N, G, 0)


@_gemm_out_op.register_fake
def _(x, w, s, z, bias, counters, out, K, N, G):
    return None


@torch.library.custom_op(f"{NAMESPACE}::awq_w4a16_gemm_act", mutates_args=("counters",), device_types="cuda")
def _gemm_act_op(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, bias: Optional[torch.Tensor],
                 counters: Optional[torch.Tensor], K: int, N: int, G: int, activation: str) -> torch.Tensor:
    out = torch.empty((x.shape[0], N // 2), dtype=x.dtype, device=x.device)
    _gemm_launch(x, w, s, z, bias, counters, out, K, N, G, _GATED_ACT[activation])
    return out


@_gemm_act_op.register_fake
def _(x, w, s, z, bias, counters, K, N, G, activation):
    return x.new_empty((x.shape[0], N // 2))


@torch.library.custom_op(f"{NAMESPACE}::awq_w4a16_gemm_act_out", mutates_args=("counters", "out"),
                         device_types="cuda")
def _gemm_act_out_op(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, bias: Optional[torch.Tensor],
                     counters: Optional[torch.Tensor], out: torch.Tensor, K: int, N: int, G: int,
                     activation: str) -> None:
    _gemm_launch(x, w, s, z, bias, counters, out, K, N, G, _GATED_ACT[activation])


@_gemm_act_out_op.register_fake
def _(x, w, s, z, bias, counters, out, K, N, G, activation):
    return None


def _check_out(out: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, device: torch.device,
               what: str = "out") -> None:
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(out.shape)}")
    if out.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {out.dtype}")
    if out.device != device:
        raise ValueError(f"{what} must be on {device}, got {out.device}")
    if not out.is_contiguous() or out.data_ptr() % 8:
        raise ValueError(f"{what} must be contiguous and 8-byte aligned")


def _overlap(s: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the address ranges that two tensors' elements span meet (the tensors of a trace have none)."""
    if torch.compiler.is_compiling() or s.numel() == 0 or t.numel() == 0:
        return False

    def end(v: torch.Tensor) -> int:
        return v.data_ptr() + (sum((n - 1) * st for n, st in zip(v.shape, v.stride())) + 1) * v.element_size()
    return s.data_ptr() < end(t) and t.data_ptr() < end(s) and not (is_fake(s) or is_fake(t))


def _check_counters(counters: torch.Tensor, N: int, device: torch.device) -> None:
    if counters.dtype != torch.int32:
        raise ValueError(f"counters must be int32, got {counters.dtype}")
    if counters.device != device:
        raise ValueError(f"counters must be on {device}, got {counters.device}")
    if not counters.is_contiguous():
        raise ValueError("counters must be contiguous")
    need = (_lib.AWQ_COUNTER_TILE_BYTES + (N + 15) // 16 * 4) // 4  # awq_counter_bytes
    if counters.numel() < need:
        raise ValueError(f"counters must hold at least {need} int32 (awq_counter_bytes({N}) bytes), "
                         f"got {counters.numel()}")
    if counters.data_ptr() % 128:
        raise ValueError("counters must be 128-byte aligned")


def gemm(x: torch.Tensor, r: Repacked, K: int, N: int, group_size: int, bias: Optional[torch.Tensor] = None,
         counters: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
         activation: Optional[str] = None) -> torch.Tensor:
    """out[M, N] = rnd(x[M, K] @ W) (+ bias), fp32 accumulation, on x's current stream.

    With ``activation`` ("silu" or "gelu") the two column halves of W are a
    merged gate/up projection and the output is ``act(gate) * up``, [M, N / 2],
    each half rounded (bias added) as the plain GEMM stores it, then the
    product in fp32, rounded once.  ``counters`` (from ``make_counters``, zero
    between calls) is needed whenever the plan splits K across workgroups."""
    _require_cuda(x, r.w, r.s, r.z)
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x must be [M, {K}], got {tuple(x.shape)}")
    if x.dtype != r.s.dtype:
        raise ValueError(f"activation dtype {x.dtype} does not match the scale dtype {r.s.dtype}")
    if activation is not None and activation not in _GATED_ACT:
        raise ValueError(f"unsupported activation {activation!r}")
    if r.w.device != x.device or r.s.device != x.device or r.z.device != x.device:
        raise ValueError("x and the repacked weights must be on one device")
    G = resolve_group_size(group_size, K)
    M = x.shape[0]
    dev = x.device
    x = _aligned(x)
    if bias is not None:
        _require_cuda(bias)
        if bias.numel() != N:
            raise ValueError(f"bias must have {N} elements, got {bias.numel()}")
        bias = _aligned(bias.to(x.dtype).reshape(-1), 8)
    if counters is not None:
        _check_counters(counters, N, dev)
    elif M > 0:
        wsb = workspace_bytes(M, N, K, G) if activation is None else workspace_bytes_act(M, N, K, G)
        if wsb > 0 and plan_info(M, N, K, G, activation).kernel != "tiled_kernel":
            raise ValueError("this shape splits K across workgroups: pass the layer's counters (make_counters)")
    ncols = N if activation is None else N // 2
    if out is not None:
        _check_out(out, (M, ncols), x.dtype, dev)
    if out is None and _undispatched(x, r.w, r.s, r.z, bias, counters):
        out = torch.empty((M, ncols), dtype=x.dtype, device=dev)
        _gemm_launch(x, r.w, r.s, r.z, bias, counters, out, K, N, G, 0 if activation is None else _GATED_ACT[activation])
        return out
    if activation is None:
        if out is None:
            return torch.ops.sglite_awq.awq_w4a16_gemm(x, r.w, r.s, r.z, bias, counters, K, N, G)
        torch.ops.sglite_awq.awq_w4a16_gemm_out(x, r.w, r.s, r.z, bias, counters, out, K, N, G)
        return out
    if out is None:
        return torch.ops.sglite_awq.awq_w4a16_gemm_act(x, r.w, r.s, r.z, bias, counters, K, N, G, activation)
    torch.ops.sglite_awq.awq_w4a16_gemm_act_out(x, r.w, r.s, r.z, bias, counters, out, K, N, G, activation)
    return out


def gemm_noalloc(x: torch.Tensor, r: Repacked, K: int, N: int, group_size: int, out: torch.Tensor,
                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gemm`` through awq_w4a16_gemm_noalloc: the split-K workspace and counters are the library's
    static per-device scratch, so the call allocates nothing (x, out and bias must already be
    contiguous and aligned).  Calls overlapping on one device race on that scratch."""
    _require_cuda(x, r.w, out, bias)
    M = x.shape[0]
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x must be [M, {K}], got {tuple(x.shape)}")
    if x.dtype != r.s.dtype:
        raise ValueError(f"activation dtype {x.dtype} does not match the scale dtype {r.s.dtype}")
    _check_out(out, (M, N), x.dtype, x.device)
    if not x.is_contiguous() or (bias is not None and (not bias.is_contiguous() or bias.numel() != N
                                                       or bias.dtype != x.dtype)):
        raise ValueError("x (and bias: N elements of x's dtype) must be contiguous")
    with _on_device(x.device):
        _noalloc_ready(x.device)
        _lib.check(_lib.load().awq_w4a16_gemm_noalloc(x.data_ptr(), r.w.data_ptr(), r.s.data_ptr(), r.z.data_ptr(),
                                                      _ptr(bias), out.data_ptr(), M, N, K,
                                                      resolve_group_size(group_size, K), dtype_code(x.dtype),
                                                      _stream(x.device)), "awq_w4a16_gemm_noalloc")
    return out


_NOALLOC_READY: set = set()


def _noalloc_ready(device: torch.device) -> None:
    """Resolve the device's static scratch ahead of the first call (awq_noalloc_init), unless that
    call is being captured: then the library's first call puts the counter clearing in the graph."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx in _NOALLOC_READY or torch.cuda.is_current_stream_capturing():
        return
    _lib.check(_lib.load().awq_noalloc_init(_stream(device)), "awq_noalloc_init")
    _NOALLOC_READY.add(idx)


# ---------------------------------------------------------------------------
# Gated MLP block in one launch (awq_gated_mlp): gate_up -> act(gate) * up ->
# down for decode batches, GatedMLP.forward (blocks.py:51-57) as one kernel.
# ---------------------------------------------------------------------------


class MlpPlan(NamedTuple):
    workgroups: int
    k_slices: int         # k-slices of the down projection
    tiles_per_group: int  # down column tiles per column group
    groups: int           # down column groups
    gate_tiles: int       # gate tiles per workgroup
    k_tiles: int          # down k-tiles per slice
    lds_bytes: int
    ws_bytes: int


def gated_mlp_plan(M: int, H: int, I: int, group_size: int, dtype: torch.dtype = torch.float16) -> Optional[MlpPlan]:
    """The one-launch plan for this block on the current device, or None when the shape is outside
    the built forms (then the block runs as its two GEMMs)."""
    info = (ctypes.c_int64 * 8)()
    r = _lib.check(_lib.load().awq_gated_mlp_plan(M, H, I, resolve_group_size(group_size, H), dtype_code(dtype),
                                                  info), "awq_gated_mlp_plan")
    return MlpPlan(*[int(v) for v in info]) if r == 1 else None


def make_mlp_counters(device: torch.device) -> torch.Tensor:
    """Counters of the one-launch gated MLP (AWQ_MLP_COUNTER_BYTES, zeroed once here; every call
    leaves them valid for the next).  Calls that share them must be ordered on one stream."""
    return torch.zeros(_lib.AWQ_MLP_COUNTER_BYTES // 4, dtype=torch.int32, device=device)


def mlp_counters_settled(counters: torch.Tensor) -> bool:
    """True when no one-launch gated MLP is in flight on ``counters``: every 128-byte slot has as many
    arrivals as its base (each launch advanced both by its arrivals)."""
    slots = counters.view(-1, 32)
    return bool(torch.equal(slots[:, 0], slots[:, 1]))


def mlp_take_errors(counters: torch.Tensor) -> int:
    """Synchronize the current stream and return (and clear) the number of workgroups that gave up
    waiting for their k-slice of the intermediate since the last check."""
    _require_cuda(counters)
    with _on_device(counters.device):
        return _lib.check(_lib.load().awq_gated_mlp_take_errors(counters.data_ptr(), counters.numel() * 4,
                                                                _stream(counters.device)), "awq_gated_mlp_take_errors")


def mlp_check(counters: torch.Tensor) -> None:
    """Raise AWQKernelError when a one-launch gated MLP on ``counters`` gave up waiting (its output
    was wrong) since the last check; the counters stay valid for further calls."""
    n = mlp_take_errors(counters)
    if n:
        raise _lib.AWQKernelError(f"awq_gated_mlp: {n} workgroup(s) gave up waiting for the intermediate; "
                                  "the outputs of those calls are invalid")


def _mlp_launch(x: torch.Tensor, gw: torch.Tensor, gs: torch.Tensor, gz: torch.Tensor, dw: torch.Tensor,
                ds: torch.Tensor, dz: torch.Tensor, counters: torch.Tensor, out: torch.Tensor, H: int, I: int,
                G: int, activation: str, polls: int) -> None:
    M = x.shape[0]
    if M == 0:
        return
    dev = x.device
    lib = _lib.load()
    with _on_device(dev):
        wsb = _lib.check(lib.awq_gated_mlp_workspace_bytes(M, H, I, G, dtype_code(x.dtype)),
                         "awq_gated_mlp_workspace_bytes")
        ws = _workspace(wsb, dev)
        _lib.check(lib.awq_gated_mlp(x.data_ptr(), gw.data_ptr(), gs.data_ptr(), gz.data_ptr(), dw.data_ptr(),
                                     ds.data_ptr(), dz.data_ptr(), out.data_ptr(), M, H, I, G, dtype_code(x.dtype),
                                     _GATED_ACT[activation], polls, _ptr(ws), wsb, counters.data_ptr(),
                                     counters.numel() * 4, _stream(dev)), "awq_gated_mlp")


@torch.library.custom_op(f"{NAMESPACE}::awq_gated_mlp_out", mutates_args=("counters", "out"), device_types="cuda")
def _mlp_out_op(x: torch.Tensor, gw: torch.Tensor, gs: torch.Tensor, gz: torch.Tensor, dw: torch.Tensor,
                ds: torch.Tensor, dz: torch.Tensor, counters: torch.Tensor, out: torch.Tensor, H: int, I: int, G: int,
                activation: str, polls: int) -> None:
    _mlp_launch(x, gw, gs, gz, dw, ds, dz, counters, out, H, I, G, activation, polls)


@_mlp_out_op.register_fake
def _(x, gw, gs, gz, dw, ds, dz, counters, out, H, I, G, activation, polls):
    return None


def gated_mlp(x: torch.Tensor, gate_up: Repacked, down: Repacked, H: int, I: int, group_size: int,
              counters: torch.Tensor, activation: str = "silu", out: Optional[torch.Tensor] = None,
              polls: Optional[int] = None) -> torch.Tensor:
    """out[M, H] = down(act(gate) * up) of a gated MLP block in one launch (awq_gated_mlp).

    ``gate_up`` is the merged projection repacked as K = H, N = 2I (gate columns first), ``down`` the
    down projection as K = I, N = H; group size 128, no bias.  The gate and up values are rounded and
    combined exactly as ``gemm(..., activation=...)`` stores them, and the down projection's k-slice
    sums are added in a fixed order.  ``counters`` from ``make_mlp_counters``.  ``polls`` bounds each
    workgroup's wait for its k-slice of the intermediate (None: the library default); a workgroup
    that gives up makes the call's output invalid and is reported by ``mlp_check``.  Raises RuntimeError when
    ``gated_mlp_plan`` has no plan for the shape."""
    _require_cuda(x, gate_up.w, down.w, counters)
    if x.dim() != 2 or x.shape[1] != H:
        raise ValueError(f"x must be [M, {H}], got {tuple(x.shape)}")
    if x.dtype != gate_up.s.dtype or x.dtype != down.s.dtype:
        raise ValueError(f"activation dtype {x.dtype} does not match the scale dtypes")
    if activation not in _GATED_ACT:
        raise ValueError(f"unsupported activation {activation!r}")
    dev = x.device
    for t in (gate_up.w, gate_up.s, gate_up.z, down.w, down.s, down.z):
        if t.device != dev:
            raise ValueError("x and the repacked weights must be on one device")
    if counters.dtype != torch.int32 or counters.device != dev or not counters.is_contiguous() \
            or counters.numel() * 4 < _lib.AWQ_MLP_COUNTER_BYTES or counters.data_ptr() % 128:
        raise ValueError("counters must be make_mlp_counters(device)")
    G = resolve_group_size(group_size, H)
    M = x.shape[0]
    x = _aligned(x)
    if out is None:
        out = torch.empty((M, H), dtype=x.dtype, device=dev)
    else:
        _check_out(out, (M, H), x.dtype, dev)
    torch.ops.sglite_awq.awq_gated_mlp_out(x, gate_up.w, gate_up.s, gate_up.z, down.w, down.s, down.z, counters,
                                           out, H, I, G, activation, -1 if polls is None else int(polls))
    return out


def stream_probe(src: torch.Tensor, nbytes: int, grid: int, block: int, sink: torch.Tensor) -> None:
    """Stream ``nbytes`` of ``src`` with ``grid`` workgroups of ``block`` threads (awq_stream_probe)."""
    _require_cuda(src, sink)
    if nbytes > src.numel() * src.element_size():
        raise ValueError("nbytes exceeds the source buffer")
    with _on_device(src.device):
        _lib.check(_lib.load().awq_stream_probe(src.data_ptr(), nbytes, grid, block, sink.data_ptr(),
                                                sink.numel() * sink.element_size(), _stream(src.device)),
                   "awq_stream_probe")


def mfma_probe(iters: int, grid: int, block: int, sink: torch.Tensor) -> None:
    """``grid`` x ``block`` threads of back-to-back 32x32x16 fp16 MFMAs (awq_mfma_probe)."""
    _require_cuda(sink)
    with _on_device(sink.device):
        _lib.check(_lib.load().awq_mfma_probe(iters, grid, block, sink.data_ptr(), sink.numel() * sink.element_size(),
                                              _stream(sink.device)), "awq_mfma_probe")


# ---------------------------------------------------------------------------
# Grouped MoE (experts stacked on dim 0).
# ---------------------------------------------------------------------------

class RepackedExperts(NamedTuple):
    """Expert-stacked repacked tensors, one row per expert (rows padded to
    256 bytes); ``expert(e)`` views expert e's linear as a ``Repacked``."""
    w: torch.Tensor  # int32 [E, w_stride / 4]
    s: torch.Tensor  # scale dtype [E, s_stride / 2]
    z: torch.Tensor  # int64 [E, z_stride / 8]
    K: int
    N: int
    G: int

    def expert(self, e: int) -> Repacked:
        NT, NG = (self.N + 15) // 16, self.K // self.G
        return Repacked(self.w[e, :NT * ((self.K + 127) // 128) * 256], self.s[e, :NT * NG * 16].view(NT, NG, 16),
                        self.z[e, :NT * NG].view(NT, NG))


def expert_strides(K: int, N: int, group_size: int) -> Tuple[int, int, int]:
    """Byte strides between consecutive experts' weights, scales and zero words."""
    G = resolve_group_size(group_size, K)
    w, s, z = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().awq_moe_expert_strides(K, N, G, ctypes.byref(w), ctypes.byref(s), ctypes.byref(z)),
               "awq_moe_expert_strides")
    return w.value, s.value, z.value


@torch.library.custom_op(f"{NAMESPACE}::awq_repack_experts", mutates_args=(), device_types="cuda")
def _repack_experts_op(qweight: torch.Tensor, qzeros: torch.Tensor,
                       scales: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    E = qweight.shape[0]
    K, N, G = _check_awq_shapes(qweight[0], qzeros[0], scales[0])
    code = dtype_code(scales.dtype)
    ws, ss, zs = expert_strides(K, N, G)
    dev = qweight.device
    w = torch.empty((E, ws // 4), dtype=torch.int32, device=dev)
    s = torch.zeros((E, ss // 2), dtype=scales.dtype, device=dev)
    z = torch.zeros((E, zs // 8), dtype=torch.int64, device=dev)
    qweight, qzeros, scales = qweight.contiguous(), qzeros.contiguous(), scales.contiguous()
    lib = _lib.load()
    with _on_device(dev):
        st = _stream(dev)
        for e in range(E):
            _lib.check(lib.awq_repack_cdna4(qweight[e].data_ptr(), qzeros[e].data_ptr(), scales[e].data_ptr(), code, K,
                                            N, G, w[e].data_ptr(), s[e].data_ptr(), z[e].data_ptr(), st),
                       "awq_repack_cdna4")
    return w, s, z


@_repack_experts_op.register_fake
def _(qweight, qzeros, scales):
    E, K, N8 = qweight.shape
    N, NG = N8 * 8, qzeros.shape[1]
    NT, KT = (N + 15) // 16, (K + 127) // 128

    def up(b):
        return (b + 255) // 256 * 256
    return (qweight.new_empty((E, up(NT * KT * 1024) // 4)), scales.new_empty((E, up(NT * NG * 32) // 2)),
            qweight.new_empty((E, up(NT * NG * 8) // 8), dtype=torch.int64))


def repack_experts(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> RepackedExperts:
    """AWQ expert stacks ``[E, K, N/8]`` / ``[E, K/G, N/8]`` / ``[E, K/G, N]`` -> stacked tile layout.

    Each expert is repacked into its own row of the stacks (the layout
    ``awq_moe_w4a16_gemm`` expects)."""
    _require_cuda(qweight, qzeros, scales)
    if qweight.dim() != 3 or qzeros.dim() != 3 or scales.dim() != 3:
        raise ValueError("expert stacks must be 3-D [E, ...]")
    E = qweight.shape[0]
    if qzeros.shape[0] != E or scales.shape[0] != E:
        raise ValueError("qweight, qzeros and scales must stack the same number of experts")
    K, N, G = _check_awq_shapes(qweight[0], qzeros[0], scales[0])
    dtype_code(scales.dtype)
    w, s, z = torch.ops.sglite_awq.awq_repack_experts(qweight, qzeros, scales)
    return RepackedExperts(w, s, z, K, N, G)


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_topk_softmax", mutates_args=(), device_types="cuda")
def _topk_op(gating_output: torch.Tensor, topk: int, renormalize: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    logits = _aligned(gating_output.float(), 4)
    T, E = logits.shape
    w = torch.empty((T, topk), dtype=torch.float32, device=logits.device)
    ids = torch.empty((T, topk), dtype=torch.int32, device=logits.device)
    with _on_device(logits.device):
        _lib.check(_lib.load().awq_moe_topk_softmax(logits.data_ptr(), w.data_ptr(), ids.data_ptr(), T, E, topk,
                                                    1 if renormalize else 0, _stream(logits.device)),
                   "awq_moe_topk_softmax")
    return w, ids


@_topk_op.register_fake
def _(gating_output, topk, renormalize):
    T = gating_output.shape[0]
    return (gating_output.new_empty((T, topk), dtype=torch.float32),
            gating_output.new_empty((T, topk), dtype=torch.int32))


def moe_topk_softmax(gating_output: torch.Tensor, topk: int, renormalize: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """softmax(fp32 logits) -> top-k -> optional ``w / (sum(w) + 1e-8)``; (weights fp32, ids int32)."""
    _require_cuda(gating_output)
    if gating_output.dim() != 2:
        raise ValueError("gating_output must be [T, E]")
    return tuple(torch.ops.sglite_awq.awq_moe_topk_softmax(gating_output, topk, bool(renormalize)))


class MoeAlignment(NamedTuple):
    sorted_ids: torch.Tensor          # int32 [sorted capacity]
    expert_ids: torch.Tensor          # int32 [block capacity]
    num_tokens_post_pad: torch.Tensor  # int32 [1]
    expert_offsets: torch.Tensor      # int32 [E + 1]


def _align_caps(n: int, num_experts: int, block_size: int) -> Tuple[int, int]:
    lib = _lib.load()
    cap = _lib.check(lib.awq_moe_sorted_capacity(n, num_experts, block_size), "awq_moe_sorted_capacity")
    bcap = _lib.check(lib.awq_moe_block_capacity(n, num_experts, block_size), "awq_moe_block_capacity")
    return cap, bcap


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_align_block_size", mutates_args=(), device_types="cuda")
def _align_op(topk_ids: torch.Tensor, block_size: int,
              num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    ids = topk_ids.contiguous().reshape(-1)
    n = ids.numel()
    cap, bcap = _align_caps(n, num_experts, block_size)
    dev = ids.device
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    expert_ids = torch.empty(bcap, dtype=torch.int32, device=dev)
    npp = torch.empty(1, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    with _on_device(dev):
        _lib.check(_lib.load().awq_moe_align_block_size(ids.data_ptr() if n else None, n, num_experts, block_size,
                                                        sorted_ids.data_ptr(), expert_ids.data_ptr(), npp.data_ptr(),
                                                        offsets.data_ptr(), _stream(dev)), "awq_moe_align_block_size")
    return sorted_ids, expert_ids, npp, offsets


@_align_op.register_fake
def _(topk_ids, block_size, num_experts):
    cap, bcap = _align_caps(topk_ids.numel(), num_experts, block_size)
    return (topk_ids.new_empty(cap), topk_ids.new_empty(bcap), topk_ids.new_empty(1),
            topk_ids.new_empty(num_experts + 1))


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int) -> MoeAlignment:
    """Stable sort of the routed rows by expert, buckets padded to ``block_size`` (sentinel ``topk_ids.numel()``)."""
    _require_cuda(topk_ids)
    if topk_ids.dtype != torch.int32:
        raise ValueError("topk_ids must be int32")
    return MoeAlignment(*torch.ops.sglite_awq.awq_moe_align_block_size(topk_ids, block_size, num_experts))


_LOGITS_CODE = {torch.float16: _lib.AWQ_DTYPE_FP16, torch.bfloat16: _lib.AWQ_DTYPE_BF16,
                torch.float32: _lib.AWQ_DTYPE_FP32}


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_route", mutates_args=(), device_types="cuda")
def _route_op(gating_output: torch.Tensor, topk: int, renormalize: bool, block_size: int) -> Tuple[
        torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    if gating_output.dtype not in _LOGITS_CODE:
        gating_output = gating_output.float()
    logits = _aligned(gating_output, 4)
    T, E = logits.shape
    dev = logits.device
    w = torch.empty((T, topk), dtype=torch.float32, device=dev)
    ids = torch.empty((T, topk), dtype=torch.int32, device=dev)
    cap, bcap = _align_caps(T * topk, E, block_size)
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    expert_ids = torch.empty(bcap, dtype=torch.int32, device=dev)
    npp = torch.empty(1, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    with _on_device(dev):
        _lib.check(_lib.load().awq_moe_route(logits.data_ptr(), _LOGITS_CODE[logits.dtype], T, E, topk,
                                             1 if renormalize else 0, block_size, w.data_ptr(), ids.data_ptr(),
                                             sorted_ids.data_ptr(), expert_ids.data_ptr(), npp.data_ptr(),
                                             offsets.data_ptr(), _stream(dev)), "awq_moe_route")
    return w, ids, sorted_ids, expert_ids, npp, offsets


@_route_op.register_fake
def _(gating_output, topk, renormalize, block_size):
    T, E = gating_output.shape
    cap, bcap = _align_caps(T * topk, E, block_size)
    i32 = [gating_output.new_empty(n, dtype=torch.int32) for n in (cap, bcap, 1, E + 1)]
    return (gating_output.new_empty((T, topk), dtype=torch.float32),
            gating_output.new_empty((T, topk), dtype=torch.int32), *i32)


def moe_route(gating_output: torch.Tensor, topk: int, renormalize: bool,
              block_size: int) -> Tuple[torch.Tensor, torch.Tensor, MoeAlignment]:
    """:func:`moe_topk_softmax` and :func:`moe_align_block_size` of the same tokens (at least one), the logits
    read in their own dtype."""
    _require_cuda(gating_output)
    if gating_output.dim() != 2 or gating_output.shape[0] == 0:
        raise ValueError("gating_output must be [T, E] with T >= 1")
    w, ids, *align = torch.ops.sglite_awq.awq_moe_route(gating_output, topk, bool(renormalize), block_size)
    return w, ids, MoeAlignment(*align)


_ACT_CODE = {None: _lib.AWQ_MOE_ACT_NONE, "silu": _lib.AWQ_MOE_ACT_SILU, "gelu": _lib.AWQ_MOE_ACT_GELU}
_ACT_NAME = {"none": None, "silu": "silu", "gelu": "gelu"}


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_w4a16_gemm", mutates_args=("out",), device_types="cuda")
def _moe_gemm_op(a: torch.Tensor, w: torch.Tensor, s: torch.Tensor, z: torch.Tensor, sorted_ids: torch.Tensor,
                 expert_offsets: torch.Tensor, topk_weights: Optional[torch.Tensor], out: torch.Tensor, K: int, N: int,
                 G: int, num_routed: int, top_k: int, activation: str, mul_routed_weight: bool) -> None:
    E = w.shape[0]
    with _on_device(a.device):
        _lib.check(_lib.load().awq_moe_w4a16_gemm(
            a.data_ptr(), a.shape[0], w.data_ptr(), s.data_ptr(), z.data_ptr(), E, N, K, G, dtype_code(a.dtype),
            sorted_ids.data_ptr(), sorted_ids.numel(), expert_offsets.data_ptr(), _ptr(topk_weights), num_routed,
            top_k, _ACT_CODE[_ACT_NAME[activation]], 1 if mul_routed_weight else 0, out.data_ptr(),
            _stream(a.device)), "awq_moe_w4a16_gemm")


@_moe_gemm_op.register_fake
def _(a, w, s, z, sorted_ids, expert_offsets, topk_weights, out, K, N, G, num_routed, top_k, activation,
      mul_routed_weight):
    return None


def moe_gemm(a: torch.Tensor, experts: RepackedExperts, K: int, N: int, group_size: int, align: MoeAlignment,
             topk_weights: Optional[torch.Tensor], num_routed: int, top_k: int, activation: Optional[str] = None,
             mul_routed_weight: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped W4A16 GEMM over the expert buckets.

    Routed row r reads ``a[r // top_k]``; the output has ``num_routed`` rows of
    ``N`` columns, or ``N / 2`` with a gate/up ``activation`` ("silu"/"gelu")."""
    _require_cuda(a, experts.w)
    if a.dim() != 2 or a.shape[1] != K:
        raise ValueError(f"a must be [rows, {K}], got {tuple(a.shape)}")
    if a.dtype != experts.s.dtype:
        raise ValueError(f"activation dtype {a.dtype} does not match the scale dtype {experts.s.dtype}")
    if activation not in _ACT_CODE:
        raise ValueError(f"unsupported activation {activation!r}")
    if mul_routed_weight and topk_weights is None:
        raise ValueError("mul_routed_weight needs topk_weights")
    G = resolve_group_size(group_size, K)
    ncols = N // 2 if activation is not None else N
    a = _aligned(a)
    if out is None:
        out = torch.empty((num_routed, ncols), dtype=a.dtype, device=a.device)
    else:
        _check_out(out, (num_routed, ncols), a.dtype, a.device)
    if topk_weights is not None:
        topk_weights = _aligned(topk_weights.float().reshape(-1), 4)
        if topk_weights.numel() < num_routed:
            raise ValueError(f"topk_weights must hold {num_routed} routed weights, got {topk_weights.numel()}")
    torch.ops.sglite_awq.awq_moe_w4a16_gemm(a, experts.w, experts.s, experts.z, align.sorted_ids, align.expert_offsets,
                                            topk_weights, out, K, N, G, num_routed, top_k,
                                            "none" if activation is None else activation, bool(mul_routed_weight))
    return out


def _moe_dense_launch(a: torch.Tensor, w: torch.Tensor, sorted_ids: torch.Tensor, expert_offsets: torch.Tensor,
                      topk_weights: Optional[torch.Tensor], out: torch.Tensor, num_routed: int, top_k: int, act: int,
                      mul_routed_weight: bool) -> None:
    dev = a.device
    if dev.index is not None and torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return _moe_dense_launch(a, w, sorted_ids, expert_offsets, topk_weights, out, num_routed, top_k, act,
                                     mul_routed_weight)
    E, N, K = w.shape
    _lib.check(_lib.load().awq_moe_dense_gemm(
        a.data_ptr(), a.shape[0], w.data_ptr(), E, N, K, dtype_code(a.dtype), sorted_ids.data_ptr(),
        sorted_ids.numel(), expert_offsets.data_ptr(), _ptr(topk_weights), num_routed, top_k, act,
        1 if mul_routed_weight else 0, out.data_ptr(), _stream(dev)), "awq_moe_dense_gemm")


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_dense_gemm", mutates_args=("out",), device_types="cuda")
def _moe_dense_op(a: torch.Tensor, w: torch.Tensor, sorted_ids: torch.Tensor, expert_offsets: torch.Tensor,
                  topk_weights: Optional[torch.Tensor], out: torch.Tensor, num_routed: int, top_k: int,
                  activation: str, mul_routed_weight: bool) -> None:
    _moe_dense_launch(a, w, sorted_ids, expert_offsets, topk_weights, out, num_routed, top_k,
                      _ACT_CODE[_ACT_NAME[activation]], mul_routed_weight)


@_moe_dense_op.register_fake
def _(a, w, sorted_ids, expert_offsets, topk_weights, out, num_routed, top_k, activation, mul_routed_weight):
    return None


def moe_dense_gemm(a: torch.Tensor, w: torch.Tensor, align: MoeAlignment, topk_weights: Optional[torch.Tensor],
                   num_routed: int, top_k: int, activation: Optional[str] = None, mul_routed_weight: bool = False,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped product over the expert buckets with dense weights ``w`` [E, N, K].

    Routed row r reads ``a[r // top_k]``; the output has ``num_routed`` rows of ``N`` columns, or ``N / 2`` of
    ``act(gate) * up`` with an ``activation`` ("silu"/"gelu", gate rows of ``w`` first).  fp32 sums, rounded once.
    Rows that ``align`` does not hold (ids outside the experts) are not written."""
    if w.dim() != 3:
        raise ValueError(f"w must be [E, N, K], got {tuple(w.shape)}")
    E, N, K = w.shape
    if a.dim() != 2 or a.shape[1] != K:
        raise ValueError(f"a must be [rows, {K}], got {tuple(a.shape)}")
    dtype_code(a.dtype)
    if a.dtype != w.dtype:
        raise ValueError(f"activation dtype {a.dtype} does not match the weight dtype {w.dtype}")
    if not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError("w must be contiguous and 16-byte aligned")
    if activation not in _ACT_CODE:
        raise ValueError(f"unsupported activation {activation!r}")
    if mul_routed_weight and topk_weights is None:
        raise ValueError("mul_routed_weight needs topk_weights")
    if num_routed < 0 or top_k < 1:
        raise ValueError(f"num_routed must be at least 0 and top_k at least 1, got {num_routed} and {top_k}")
    if align.expert_offsets.numel() != E + 1:
        raise ValueError(f"the rows were aligned for {align.expert_offsets.numel() - 1} experts, w holds {E}")
    if align.sorted_ids.dtype != torch.int32 or align.expert_offsets.dtype != torch.int32 \
            or not align.sorted_ids.is_contiguous() or not align.expert_offsets.is_contiguous():
        raise ValueError("the alignment must be moe_align_block_size's: contiguous int32")
    ncols = N // 2 if activation is not None else N
    if topk_weights is not None and topk_weights.numel() < num_routed:
        raise ValueError(f"topk_weights must hold {num_routed} routed weights, got {topk_weights.numel()}")
    _require_cuda(a, w, topk_weights, align.sorted_ids, align.expert_offsets)
    for t in (w, topk_weights, align.sorted_ids, align.expert_offsets):
        if t is not None and t.device != a.device:
            raise ValueError("a, w, the weights and the alignment must be on one device")
    a = _aligned(a)
    if out is None:
        out = torch.empty((num_routed, ncols), dtype=a.dtype, device=a.device)
    else:
        _check_out(out, (num_routed, ncols), a.dtype, a.device)
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        if _overlap(out, a) or _overlap(out, w):
            raise ValueError("out must not share memory with a or w")
    if topk_weights is not None:
        topk_weights = _aligned(topk_weights.float().reshape(-1), 4)
    if _undispatched(a, w, topk_weights, out, align.sorted_ids, align.expert_offsets):
        _moe_dense_launch(a, w, align.sorted_ids, align.expert_offsets, topk_weights, out, num_routed, top_k,
                          _ACT_CODE[activation], mul_routed_weight)
        return out
    torch.ops.sglite_awq.awq_moe_dense_gemm(a, w, align.sorted_ids, align.expert_offsets, topk_weights, out,
                                            num_routed, top_k, "none" if activation is None else activation,
                                            bool(mul_routed_weight))
    return out


@torch.library.custom_op(f"{NAMESPACE}::awq_moe_sum_reduce", mutates_args=("out",), device_types="cuda")
def _moe_sum_op(inp: torch.Tensor, out: torch.Tensor) -> None:
    T, k, H = inp.shape
    with _on_device(inp.device):
        _lib.check(_lib.load().awq_moe_sum_reduce(inp.data_ptr(), out.data_ptr(), T, k, H, dtype_code(inp.dtype),
                                                  _stream(inp.device)), "awq_moe_sum_reduce")


@_moe_sum_op.register_fake
def _(inp, out):
    return None


def moe_sum_reduce(inp: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """out[t] = rnd(sum_j inp[t, j]) with an fp32 sum (inp [T, k, H], out [T, H])."""
    _require_cuda(inp, out)
    if inp.dim() != 3 or out.dim() != 2 or out.shape[0] != inp.shape[0] or out.shape[1] != inp.shape[2]:
        raise ValueError(f"shapes do not match: in {tuple(inp.shape)}, out {tuple(out.shape)}")
    if inp.dtype != out.dtype:
        raise ValueError("in and out must share a dtype")
    if not (inp.is_contiguous() and out.is_contiguous()):
        raise ValueError("in and out must be contiguous")
    torch.ops.sglite_awq.awq_moe_sum_reduce(inp, out)
    return out


# ---------------------------------------------------------------------------
# Low-rank adapters of many requests beside a projection (awq_lora_add).
# ---------------------------------------------------------------------------

LORA_MAX_ADAPTERS = _lib.AWQ_LORA_MAX_ADAPTERS
LORA_MAX_RANK = _lib.AWQ_LORA_MAX_RANK


class LoraStack(NamedTuple):
    """The adapters of one projection, stacked over ``num_adapters`` slots.

    ``a[e, p * max_rank + j]`` is row j of adapter e's A for column part p and ``b[e, n]`` row n of its B, so
    a slot's values at and past its rank do not count.  Both must be finite."""
    a: torch.Tensor        # [num_adapters, parts * max_rank, K]
    b: torch.Tensor        # [num_adapters, N, max_rank]
    scaling: torch.Tensor  # float32 [num_adapters]
    ranks: torch.Tensor    # int32 [num_adapters]
    parts: Tuple[int, ...]  # columns of each part, summing to N


class LoraBatch(NamedTuple):
    """A step's rows and their adapters (``lora_route``); the tables are None for the few rows of a small step."""
    adapter_ids: torch.Tensor               # int32 [rows], as given
    sorted_ids: Optional[torch.Tensor]      # int32, rows by adapter; the row count in padding
    block_adapters: Optional[torch.Tensor]  # int32, adapter of each 16-row block (num_adapters: none, -1: past the end)
    num_adapters: int

    @property
    def rows(self) -> int:
        return self.adapter_ids.numel()


def _lora_unsorted(rows: int) -> bool:
    """Whether every row is taken by itself and nothing is sorted: a row then reads its adapter alone, and two rows
    of one adapter both read it.  32 projections of four decode layers (us, sorted against not): 8 rows over 4
    adapters of rank 16 149 / 141, over 64 of rank 64 217 / 198; 16 rows over 4 of rank 16 149 / 152, over 32 162 /
    154, over 64 of rank 64 258 / 264; 24 rows over 16 of rank 32 183 / 186; 32 rows 190 / 199, over 4 of rank 16
    156 / 178."""
    return rows <= 16


def make_lora_stack(num_adapters: int, max_rank: int, K: int, parts: Sequence[int], dtype: torch.dtype,
                    device: torch.device) -> LoraStack:
    """An empty stack (every slot of rank 0, which adds nothing).  Sizes that ``lora_add`` cannot take are refused."""
    dtype_code(dtype)
    N, P = sum(parts), len(parts)
    if not 1 <= num_adapters <= LORA_MAX_ADAPTERS:
        raise ValueError(f"num_adapters must be in [1, {LORA_MAX_ADAPTERS}], got {num_adapters}")
    if not 1 <= P <= _lib.AWQ_LORA_MAX_PARTS or any(n <= 0 or n % 8 for n in parts):
        raise ValueError(f"the projection must have 1 to {_lib.AWQ_LORA_MAX_PARTS} parts, their columns positive "
                         f"multiples of 8, got {tuple(parts)}")
    if K <= 0 or K % 8:
        raise ValueError(f"the projection's input size must be a positive multiple of 8, got {K}")
    if not 8 <= max_rank <= LORA_MAX_RANK or max_rank % 8:
        raise ValueError(f"max_rank must be a multiple of 8 in [8, {LORA_MAX_RANK}], got {max_rank}")
    if max(P * K, N) * max_rank * 2 >= 1 << 31 or K >= 1 << 24:
        raise ValueError(f"one adapter's A and B must each span below 2 GiB, got rank {max_rank}, {P} parts, K {K}, "
                         f"N {N}")
    return LoraStack(torch.zeros((num_adapters, len(parts) * max_rank, K), dtype=dtype, device=device),
                     torch.zeros((num_adapters, N, max_rank), dtype=dtype, device=device),
                     torch.zeros(num_adapters, dtype=torch.float32, device=device),
                     torch.zeros(num_adapters, dtype=torch.int32, device=device), tuple(int(n) for n in parts))


def _lora_route_launch(adapter_ids: torch.Tensor, num_adapters: int) -> Tuple[torch.Tensor, torch.Tensor]:
    dev = adapter_ids.device
    if dev.index is not None and torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return _lora_route_launch(adapter_ids, num_adapters)
    M = adapter_ids.numel()
    cap = M + (num_adapters + 1) * 15  # awq_moe_sorted_capacity(M, num_adapters + 1, 16)
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    # Block adapters, then what the projections do not read: offsets and the padded row count.
    bcap = (cap + 15) // 16
    blocks = torch.empty(bcap + num_adapters + 3, dtype=torch.int32, device=dev)
    p = blocks.data_ptr()
    _lib.check(_lib.load().awq_lora_route(adapter_ids.data_ptr() if M else None, M, num_adapters,
                                          sorted_ids.data_ptr(), p, p + 4 * (bcap + num_adapters + 2), p + 4 * bcap,
                                          _stream(dev)), "awq_lora_route")
    return sorted_ids, blocks


@torch.library.custom_op(f"{NAMESPACE}::awq_lora_route", mutates_args=(), device_types="cuda")
def _lora_route_op(adapter_ids: torch.Tensor, num_adapters: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return _lora_route_launch(adapter_ids, num_adapters)


@_lora_route_op.register_fake
def _(adapter_ids, num_adapters):
    cap = adapter_ids.numel() + (num_adapters + 1) * 15
    return adapter_ids.new_empty(cap), adapter_ids.new_empty((cap + 15) // 16 + num_adapters + 3)


def lora_route(adapter_ids: torch.Tensor, num_adapters: int) -> LoraBatch:
    """A step's rows by adapter; one call serves every projection of the step.

    ``adapter_ids`` [M] int32 names each row's slot; an id outside ``[0, num_adapters)``, as -1, names none.  The
    batch refers to them: they stay as they are until its last use.  For few rows nothing is launched, beyond that
    one kernel sorts them."""
    if adapter_ids.dim() != 1 or adapter_ids.dtype != torch.int32:
        raise ValueError(f"adapter_ids must be int32 [M], got {adapter_ids.dtype} {tuple(adapter_ids.shape)}")
    if not 1 <= num_adapters <= _lib.AWQ_LORA_MAX_ADAPTERS:
        raise ValueError(f"num_adapters must be in [1, {_lib.AWQ_LORA_MAX_ADAPTERS}], got {num_adapters}")
    _require_cuda(adapter_ids)
    ids = _aligned(adapter_ids, 4)
    if _lora_unsorted(ids.numel()):
        return LoraBatch(ids, None, None, num_adapters)
    if _undispatched(ids):
        tables = _lora_route_launch(ids, num_adapters)
    else:
        tables = torch.ops.sglite_awq.awq_lora_route(ids, num_adapters)
    return LoraBatch(ids, *tables, num_adapters)


def _lora_launch(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor,
                 ranks: torch.Tensor, adapter_ids: torch.Tensor, sorted_ids: Optional[torch.Tensor],
                 block_adapters: Optional[torch.Tensor], out: torch.Tensor, parts: Sequence[int], act: int) -> None:
    M, K = x.shape
    if M == 0:
        return
    dev = x.device
    if dev.index is not None and torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):  # the C ABI's planning fills the current device's CUs
            return _lora_launch(y, x, a, b, scaling, ranks, adapter_ids, sorted_ids, block_adapters, out, parts, act)
    L, N, R = b.shape
    lib = _lib.load()
    wsb = _lib.check(lib.awq_lora_workspace_bytes(M, N, K, L, R, len(parts), 0 if sorted_ids is None else 1),
                     "awq_lora_workspace_bytes")
    ws = _workspace(wsb, dev)
    cols = (ctypes.c_int64 * len(parts))(*parts)
    _lib.check(lib.awq_lora_add(y.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(), scaling.data_ptr(),
                                ranks.data_ptr(), out.data_ptr(), M, N, K, L, R, len(parts), cols,
                                dtype_code(x.dtype), act, adapter_ids.data_ptr(), _ptr(sorted_ids),
                                _ptr(block_adapters), ws.data_ptr(), wsb, _stream(dev)), "awq_lora_add")


@torch.library.custom_op(f"{NAMESPACE}::awq_lora_add", mutates_args=(), device_types="cuda")
def _lora_add_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor,
                 ranks: torch.Tensor, adapter_ids: torch.Tensor, sorted_ids: Optional[torch.Tensor],
                 block_adapters: Optional[torch.Tensor], parts: List[int], activation: str) -> torch.Tensor:
    act = _ACT_CODE[_ACT_NAME[activation]]
    out = torch.empty((y.shape[0], y.shape[1] // 2 if act else y.shape[1]), dtype=y.dtype, device=y.device)
    _lora_launch(y, x, a, b, scaling, ranks, adapter_ids, sorted_ids, block_adapters, out, parts, act)
    return out


@_lora_add_op.register_fake
def _(y, x, a, b, scaling, ranks, adapter_ids, sorted_ids, block_adapters, parts, activation):
    return y.new_empty((y.shape[0], y.shape[1] if activation == "none" else y.shape[1] // 2))


@torch.library.custom_op(f"{NAMESPACE}::awq_lora_add_", mutates_args=("y",), device_types="cuda")
def _lora_add_inplace_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor,
                         ranks: torch.Tensor, adapter_ids: torch.Tensor, sorted_ids: Optional[torch.Tensor],
                         block_adapters: Optional[torch.Tensor], parts: List[int]) -> None:
    _lora_launch(y, x, a, b, scaling, ranks, adapter_ids, sorted_ids, block_adapters, y, parts, 0)


@_lora_add_inplace_op.register_fake
def _(y, x, a, b, scaling, ranks, adapter_ids, sorted_ids, block_adapters, parts):
    return None


def _check_lora(y: torch.Tensor, x: torch.Tensor, stack: LoraStack, batch: LoraBatch,
                activation: Optional[str]) -> None:
    a, b = stack.a, stack.b
    if a.dim() != 3 or b.dim() != 3:
        raise ValueError("a must be [adapters, parts * max_rank, K] and b [adapters, N, max_rank]")
    L, N, R = b.shape
    P, K = len(stack.parts), a.shape[2]
    if tuple(a.shape) != (L, P * R, K):
        raise ValueError(f"a must be {(L, P * R, K)} beside b {tuple(b.shape)} with {P} parts, got {tuple(a.shape)}")
    if sum(stack.parts) != N:
        raise ValueError(f"the parts {stack.parts} do not sum to the {N} columns of b")
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x must be [M, {K}], got {tuple(x.shape)}")
    M = x.shape[0]
    if tuple(y.shape) != (M, N):
        raise ValueError(f"y must be {(M, N)}, got {tuple(y.shape)}")
    dtype_code(x.dtype)
    if not (x.dtype == y.dtype == a.dtype == b.dtype):
        raise ValueError(f"y, x, a and b must share a dtype, got {y.dtype}, {x.dtype}, {a.dtype}, {b.dtype}")
    if stack.scaling.dtype != torch.float32 or tuple(stack.scaling.shape) != (L,):
        raise ValueError(f"scaling must be float32 [{L}]")
    if stack.ranks.dtype != torch.int32 or tuple(stack.ranks.shape) != (L,):
        raise ValueError(f"ranks must be int32 [{L}]")
    for t in (a, b, stack.scaling, stack.ranks):
        if not t.is_contiguous() or t.data_ptr() % (16 if t.dtype == x.dtype else 4):
            raise ValueError("the stack's tensors must be contiguous (a and b 16-byte aligned)")
    dev = x.device
    for t in (y, a, b, stack.scaling, stack.ranks, batch.adapter_ids, batch.sorted_ids, batch.block_adapters):
        if t is not None and t.device != dev:
            raise ValueError("y, x, the stack and the batch must be on one device")
    if batch.rows != M or batch.num_adapters != L:
        raise ValueError(f"the batch was routed for {batch.rows} rows and {batch.num_adapters} adapters, "
                         f"not {M} and {L}")
    for t, n in ((batch.adapter_ids, M), (batch.sorted_ids, M + 15 * (L + 1)),
                 (batch.block_adapters, (M + 15 * (L + 1) + 15) // 16)):
        if t is not None and (t.dtype != torch.int32 or t.numel() < n or not t.is_contiguous()):
            raise ValueError("the batch must be lora_route's: contiguous int32 ids and tables")
    if (batch.sorted_ids is None) != (batch.block_adapters is None):
        raise ValueError("the batch must have both tables or neither")
    if activation is not None:
        if activation not in _GATED_ACT:
            raise ValueError(f"unsupported activation {activation!r}")
        if P != 2 or stack.parts[0] != stack.parts[1]:
            raise ValueError(f"an activation needs two equal parts, gate and up, got {stack.parts}")
    _require_cuda(y, x, a, b, stack.scaling, stack.ranks, batch.adapter_ids)


def lora_add(y: torch.Tensor, x: torch.Tensor, stack: LoraStack, batch: LoraBatch, activation: Optional[str] = None,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y + scaling * B (A x)`` of every row's adapter, summed in fp32 and rounded once, on x's current stream (for
    fp16, ``A x`` keeps 23 of the 24 bits of its fp32 sum, for bf16 all).

    ``y`` [M, N] is the projection's output for ``x`` [M, K]; rows that name no adapter keep it.  ``out`` may be
    ``y`` itself: then only rows with an adapter are written.  With ``activation`` ("silu" or "gelu") the two
    parts are gate and up and the result is ``act(gate) * up``, [M, N / 2], for every row (``out`` is not taken)."""
    _check_lora(y, x, stack, batch, activation)
    if out is not None:
        if activation is not None:
            raise ValueError("out is not taken with an activation")
        _check_out(out, tuple(y.shape), y.dtype, y.device)
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        if _overlap(out, x) or (_overlap(out, y) and (out.data_ptr() != y.data_ptr() or not y.is_contiguous())):
            raise ValueError("out must not share memory with x, nor with y unless it is y")
    x = _aligned(x)
    a, b, scaling, ranks = stack.a, stack.b, stack.scaling, stack.ranks
    tables = (batch.adapter_ids, batch.sorted_ids, batch.block_adapters)
    if out is not None:
        if out.data_ptr() != y.data_ptr():
            out.copy_(y)
        if _undispatched(out, x, a, b, scaling, ranks, *tables):
            _lora_launch(out, x, a, b, scaling, ranks, *tables, out, stack.parts, 0)
        else:
            torch.ops.sglite_awq.awq_lora_add_(out, x, a, b, scaling, ranks, *tables, list(stack.parts))
        return out
    y = _aligned(y)
    if _undispatched(y, x, a, b, scaling, ranks, *tables):
        act = _ACT_CODE[activation]
        out = torch.empty((y.shape[0], y.shape[1] // 2 if act else y.shape[1]), dtype=y.dtype, device=y.device)
        _lora_launch(y, x, a, b, scaling, ranks, *tables, out, stack.parts, act)
        return out
    return torch.ops.sglite_awq.awq_lora_add(y, x, a, b, scaling, ranks, *tables, list(stack.parts),
                                             "none" if activation is None else activation)


REGISTERED_OPS: List[str] = [
    "awq_repack_cdna4", "awq_unrepack_cdna4", "awq_dequant", "awq_dequant_repacked", "awq_w4a16_gemm",
    "awq_w4a16_gemm_out", "awq_w4a16_gemm_act", "awq_w4a16_gemm_act_out", "awq_repack_experts",
    "awq_moe_topk_softmax", "awq_moe_align_block_size", "awq_moe_route", "awq_moe_w4a16_gemm", "awq_moe_sum_reduce",
    "awq_moe_dense_gemm", "awq_lora_route", "awq_lora_add", "awq_lora_add_",
]
