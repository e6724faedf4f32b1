"""ctypes binding of ``libmoe_bench_b200.so`` (declared in ``include/moe_bench_b200.h``).

There is no fallback: if the library is missing or a call fails, an exception is
raised.  Tensors are passed as raw device pointers and the current torch stream
is used, so calls are ordered with surrounding torch work.
"""

from __future__ import annotations

import ctypes
import os
from typing import Optional

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libmoe_bench_b200.so")

ABI_VERSION = 5
PRECISION_BF16 = 0
PRECISION_FP8 = 1
PRECISION_FP16 = 2
PRECISION_FP32 = 3
PAD_ROWS_BF16 = 16
PAD_ROWS_FP8 = 128

c_i32, c_i64, c_vp = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p

# name -> (restype, argtypes); must list every symbol the header declares.
SIGNATURES = {
    "mb200_abi_version": (c_i32, []),
    "mb200_last_error": (ctypes.c_char_p, []),
    "mb200_route_topk": (c_i32, [c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp]),
    "mb200_row_capacity": (c_i64, [c_i64, c_i32, c_i32, c_i32]),
    "mb200_align_scratch_bytes": (c_i64, [c_i64, c_i32, c_i32]),
    "mb200_align": (c_i32, [c_vp, c_i64, c_i32, c_vp, c_i32, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_vp, c_vp]),
    "mb200_align_noalloc": (c_i32, [c_vp, c_i64, c_i32, c_vp, c_i32, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_vp]),
    "mb200_group_quant_fp8": (c_i32, [c_vp, c_i64, c_i32, c_vp, c_vp, c_vp]),
    "mb200_grouped_gemm_bf16": (
        c_i32,
        [c_i32, c_vp, c_i64, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i32, c_vp],
    ),
    "mb200_grouped_gemm_bf16_gated": (
        c_i32,
        [c_vp, c_i64, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_i32, c_vp, c_vp, c_i32, c_vp],
    ),
    "mb200_workspace_bytes": (c_i64, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32]),
    "mb200_forward_layout": (c_i32, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i64, c_vp]),
    "mb200_moe_forward_bf16": (
        c_i32,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_i32, c_i32, c_i32, c_vp, c_i64, c_i32, c_vp],
    ),
    "mb200_moe_forward_fp16": (
        c_i32,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_i32, c_i32, c_i32, c_vp, c_i64, c_i32, c_vp],
    ),
    "mb200_grouped_gemm_fp8": (
        c_i32,
        [c_i32, c_vp, c_vp, c_i64, c_vp, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
         c_i32, c_vp],
    ),
    "mb200_grouped_gemm_fp8_cols": (
        c_i32,
        [c_i32, c_vp, c_vp, c_i64, c_vp, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
         c_i32, c_vp],
    ),
    "mb200_moe_forward_fp8": (
        c_i32,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_i32, c_i32, c_i32, c_vp, c_i64,
         c_i32, c_vp],
    ),
    "mb200_dist_symmetric_bytes": (c_i64, [c_i32, c_i64, c_i32, c_i32, c_i32]),
    "mb200_dist_workspace_bytes": (c_i64, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i32]),
    "mb200_dist_forward": (
        c_i32,
        [c_i32, c_i32, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i32, c_i32, c_i32, c_i32,
         c_i32, c_i32, c_i32, c_vp, c_i64, ctypes.c_uint32, c_vp, c_i64, c_i32, c_vp],
    ),
    "mb200_peer_barrier": (c_i32, [c_vp, c_i32, c_i32, ctypes.c_uint32, c_vp, c_vp]),
    "mb200_ipc_alloc": (c_i32, [c_i64, c_vp, c_vp]),
    "mb200_ipc_open": (c_i32, [c_vp, c_vp]),
    "mb200_ipc_close": (c_i32, [c_vp]),
    "mb200_ipc_free": (c_i32, [c_vp]),
    "mb200_set_stage_events": (c_i32, [c_vp, c_i32]),
    "mb200_set_fp8_scale_format": (c_i32, [c_i32]),
    "mb200_set_comm_only": (c_i32, [c_i32]),
    "mb200_read_status": (c_i32, [c_vp, c_vp, c_vp]),
    "mb200_linear": (
        c_i32,
        [c_i32, c_vp, c_i64, c_i64, c_vp, c_i64, c_i32, c_i32, c_vp, c_i32, c_i32, c_vp, c_i64, c_vp, c_i32, c_vp,
         c_i32, c_vp],
    ),
    "mb200_linear_backward_workspace_bytes": (c_i64, [c_i64, c_i32, c_i32, c_i32]),
    "mb200_linear_backward": (
        c_i32,
        [c_i32, c_vp, c_i32, c_i64, c_vp, c_vp, c_i64, c_i64, c_vp, c_i64, c_i32, c_i32, c_vp, c_vp, c_i32, c_vp,
         c_vp, c_i64, c_i32, c_vp],
    ),
    "mb200_grouped_linear": (
        c_i32,
        [c_i32, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_vp, c_i32, c_i32, c_i32, c_vp, c_i32, c_vp],
    ),
    "mb200_grouped_linear_backward_workspace_bytes": (c_i64, [c_i64, c_i32]),
    "mb200_grouped_linear_backward": (
        c_i32,
        [c_i32, c_vp, c_i64, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_vp, c_i32, c_i32, c_i32, c_vp, c_vp, c_i32,
         c_vp, c_i64, c_i32, c_vp],
    ),
    "mb200_linear_status": (c_i32, [c_vp, c_i32, c_vp]),
    "mb200_layer_norm": (
        c_i32,
        [c_i32, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_i32, ctypes.c_float, c_vp, c_vp, c_vp, c_i32, c_vp],
    ),
    "mb200_layer_norm_backward_workspace_bytes": (c_i64, [c_i64, c_i64, c_i32]),
    "mb200_layer_norm_backward": (
        c_i32,
        [c_i32, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp, c_i32, c_vp, c_vp, c_vp, c_vp, c_i64,
         c_i32, c_vp],
    ),
}


class MB200Error(RuntimeError):
    """A library call returned a non-zero status."""


_lib: Optional[ctypes.CDLL] = None


def load_library(path: str) -> ctypes.CDLL:
    """Open a build of the library, set the prototypes and check its ABI version."""
    if not os.path.exists(path):
        raise MB200Error(
            f"{path} is missing: build it with `python -m moe_bench_b200.build` "
            "(there is no non-CUDA fallback)"
        )
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    if lib.mb200_abi_version() != ABI_VERSION:
        raise MB200Error(
            f"{path} has ABI version {lib.mb200_abi_version()}, this package needs {ABI_VERSION}: "
            "rebuild with `python -m moe_bench_b200.build --force`"
        )
    return lib


def load() -> ctypes.CDLL:
    """Load the shared library (once) and set the prototypes."""
    global _lib
    if _lib is None:
        _lib = load_library(LIB_PATH)
    return _lib


def use_library(lib: ctypes.CDLL) -> None:
    """Route every later call of this module to ``lib`` (a result of ``load_library``);
    lets one process compare two builds."""
    global _lib
    _lib = lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise MB200Error(f"{what} failed (status {rc}): {load().mb200_last_error().decode()}")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda or not t.is_contiguous() or t.dtype != dtype:
        raise MB200Error(f"{name}: need a contiguous CUDA tensor of {dtype}, got {t.dtype} on {t.device}")


def check_problem_tensors(problem, dtype) -> None:
    """The layer entry points take raw pointers: refuse tensors of another dtype, device or
    layout here instead of computing on garbage (called from ``setup()``, not in the timed path)."""
    _need(problem.hidden_states, dtype, "hidden_states")
    _need(problem.topk_ids, torch.int32, "topk_ids")
    _need(problem.topk_weights, torch.float32, "topk_weights")
    for name in ("w1", "w2"):
        w = getattr(problem, name)
        if not w.is_cuda or not w.is_contiguous():
            raise MB200Error(f"{name}: need a contiguous CUDA tensor")
    if problem.w1.dtype != problem.w2.dtype:
        raise MB200Error(f"w1 is {problem.w1.dtype} but w2 is {problem.w2.dtype}")
    if problem.expert_map is not None:
        _need(problem.expert_map, torch.int32, "expert_map")
        if problem.topk_ids.numel() and int(problem.topk_ids.max()) >= problem.expert_map.numel():
            raise MB200Error("topk_ids holds an expert id beyond the end of expert_map")
    if problem.topk_ids.numel() and int(problem.topk_ids.min()) < 0:
        raise MB200Error("topk_ids holds a negative expert id")


def row_capacity(tokens: int, topk: int, local_experts: int, pad_rows: int = PAD_ROWS_BF16) -> int:
    return int(load().mb200_row_capacity(tokens, topk, local_experts, pad_rows))


def workspace_bytes(precision: int, tokens: int, hidden: int, intermediate: int, local_experts: int, topk: int) -> int:
    n = int(load().mb200_workspace_bytes(precision, tokens, hidden, intermediate, local_experts, topk))
    if n < 0:
        raise MB200Error(f"workspace_bytes: {load().mb200_last_error().decode()}")
    return n


LAYOUT_FIELDS = ("pad_rows", "row_capacity", "counts", "mtile_prefix", "sorted_ids", "inverse", "rows", "row_scales",
                 "act", "y")


def forward_layout(precision: int, tokens: int, hidden: int, intermediate: int, local_experts: int, topk: int,
                   expected_rows: int) -> dict:
    """Padding, row capacity and the byte offsets of the forward's tables inside its workspace."""
    out = (ctypes.c_int64 * 10)()
    _check(load().mb200_forward_layout(precision, tokens, hidden, intermediate, local_experts, topk, expected_rows,
                                       out), "forward_layout")
    return dict(zip(LAYOUT_FIELDS, [int(v) for v in out]))


def route_topk(logits: torch.Tensor, topk: int):
    """softmax -> top-k -> renormalise on the GPU; returns (ids int32, weights fp32)."""
    _need(logits, torch.float32, "logits")
    t, e = logits.shape
    ids = torch.empty(t, topk, dtype=torch.int32, device=logits.device)
    w = torch.empty(t, topk, dtype=torch.float32, device=logits.device)
    _check(load().mb200_route_topk(_ptr(logits), t, e, topk, _ptr(ids), _ptr(w), _stream(logits.device)), "route_topk")
    return ids, w


def align(topk_ids: torch.Tensor, expert_map: Optional[torch.Tensor], local_experts: int,
          pad_rows: int = PAD_ROWS_BF16):
    """Sort-and-pad to ``pad_rows``; returns (counts[E], mtile_prefix[E+1], sorted_ids[cap], inverse[T*k])."""
    _need(topk_ids, torch.int32, "topk_ids")
    if expert_map is not None:
        _need(expert_map, torch.int32, "expert_map")
    t, k = topk_ids.shape
    dev = topk_ids.device
    cap = row_capacity(t, k, local_experts, pad_rows)
    counts = torch.empty(local_experts, dtype=torch.int32, device=dev)
    prefix = torch.empty(local_experts + 1, dtype=torch.int32, device=dev)
    sorted_ids = torch.full((max(cap, 1),), -2, dtype=torch.int32, device=dev)[:cap]
    inverse = torch.empty(max(t * k, 1), dtype=torch.int32, device=dev)
    scratch = torch.empty(load().mb200_align_scratch_bytes(t, k, local_experts), dtype=torch.uint8, device=dev)
    _check(
        load().mb200_align(
            _ptr(topk_ids), t, k, _ptr(expert_map), local_experts, _ptr(counts), _ptr(prefix),
            _ptr(sorted_ids), _ptr(inverse), cap, pad_rows, _ptr(scratch), _stream(dev),
        ),
        "align",
    )
    return counts, prefix, sorted_ids, inverse[: t * k]


def align_noalloc(topk_ids: torch.Tensor, expert_map: Optional[torch.Tensor], local_experts: int, outputs=None,
                  pad_rows: int = PAD_ROWS_BF16):
    """Sort-and-pad through the entry point that needs no scratch buffer.

    For hosts that may not allocate device memory while running (a server
    whose pool owns all of HBM, a latency-bound decode loop): the library's
    built-in 256 KiB array replaces the scratch tensor.  Pass ``outputs`` =
    ``(counts, mtile_prefix, sorted_ids, inverse)`` preallocated to make the
    whole call allocation-free; without it the four output tensors are created
    here for convenience.  Limits: 256 local experts, 2**20 assignments; calls
    on one device must not overlap.
    """
    _need(topk_ids, torch.int32, "topk_ids")
    if expert_map is not None:
        _need(expert_map, torch.int32, "expert_map")
    t, k = topk_ids.shape
    dev = topk_ids.device
    if outputs is None:
        cap = row_capacity(t, k, local_experts, pad_rows)
        outputs = (
            torch.empty(local_experts, dtype=torch.int32, device=dev),
            torch.empty(local_experts + 1, dtype=torch.int32, device=dev),
            torch.full((cap,), -2, dtype=torch.int32, device=dev),
            torch.empty(max(t * k, 1), dtype=torch.int32, device=dev),
        )
    counts, prefix, sorted_ids, inverse = outputs
    _check(
        load().mb200_align_noalloc(
            _ptr(topk_ids), t, k, _ptr(expert_map), local_experts, _ptr(counts), _ptr(prefix),
            _ptr(sorted_ids), _ptr(inverse), sorted_ids.shape[0], pad_rows, _stream(dev),
        ),
        "align_noalloc",
    )
    return counts, prefix, sorted_ids, inverse[: t * k]


def group_quant_fp8(x: torch.Tensor):
    """Per-row, per-128 e4m3 quantisation; returns (q e4m3 [m,K], scales fp32 [m,K/128])."""
    _need(x, torch.bfloat16, "x")
    m, k = x.shape
    q = torch.empty(m, k, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(m, k // 128, dtype=torch.float32, device=x.device)
    _check(load().mb200_group_quant_fp8(_ptr(x), m, k, _ptr(q), _ptr(s), _stream(x.device)), "group_quant_fp8")
    return q, s


def grouped_gemm_bf16(mode, a, w, hidden, intermediate, counts, prefix, sorted_ids, row_scale, out, status):
    """One grouped GEMM stage (mode 0 gate/up + SiLU-mul, mode 1 down + weight)."""
    dev = a.device
    _check(
        load().mb200_grouped_gemm_bf16(
            mode, _ptr(a), a.shape[0], _ptr(w), w.shape[0], hidden, intermediate, _ptr(counts),
            _ptr(prefix), _ptr(sorted_ids), _ptr(row_scale), _ptr(out), _ptr(status), dev.index or 0, _stream(dev),
        ),
        "grouped_gemm_bf16",
    )


def grouped_gemm_bf16_gated(a, w, hidden, intermediate, counts, prefix, sorted_ids, granule_done, granule_target,
                            out, status):
    """The gate/up stage for rows delivered by someone else: a token block is loaded once
    ``granule_done`` of each of its 16-row granules has reached ``granule_target``."""
    dev = a.device
    _need(granule_done, torch.int32, "granule_done")
    _need(status, torch.int32, "status")
    if status.numel() < 2:
        raise MB200Error("status: need the two-word head of a status block")
    _check(
        load().mb200_grouped_gemm_bf16_gated(
            _ptr(a), a.shape[0], _ptr(w), w.shape[0], hidden, intermediate, _ptr(counts), _ptr(prefix),
            _ptr(sorted_ids), _ptr(granule_done), granule_target, _ptr(out), _ptr(status), dev.index or 0,
            _stream(dev),
        ),
        "grouped_gemm_bf16_gated",
    )


def moe_forward_bf16(x, w1, w2, topk_ids, topk_weights, expert_map, out, workspace):
    """Enqueue the 16-bit layer forward on the current stream: bf16 tensors, or
    fp16 when ``x`` is ``torch.float16`` (weights and output must match)."""
    t, hidden = x.shape
    e_local, two_n, _ = w1.shape
    dev = x.device
    if not (x.dtype == w1.dtype == w2.dtype == out.dtype) or x.dtype not in (torch.bfloat16, torch.float16):
        raise MB200Error(f"moe_forward: tensors must all be bf16 or all fp16, got {x.dtype}/{w1.dtype}/{w2.dtype}/{out.dtype}")
    fn = load().mb200_moe_forward_fp16 if x.dtype == torch.float16 else load().mb200_moe_forward_bf16
    _check(
        fn(
            _ptr(x), _ptr(w1), _ptr(w2), _ptr(topk_ids), _ptr(topk_weights), _ptr(expert_map), _ptr(out),
            t, hidden, two_n // 2, e_local, topk_ids.shape[1], _ptr(workspace), workspace.numel(),
            dev.index or 0, _stream(dev),
        ),
        "moe_forward_bf16",
    )


def grouped_gemm_fp8(mode, a, a_scale_t, w, w_scale, hidden, intermediate, counts, prefix, sorted_ids,
                     row_scale, out, out_scale_t, status, cols: bool = False):
    """One fp8 grouped GEMM stage (mode 0 gate/up + SiLU-mul + re-quantise, mode 1 down + weight).
    ``cols``: schedule padded to 16 rows, tokens-on-columns kernel; else 128-row token tiles."""
    dev = a.device
    fn = load().mb200_grouped_gemm_fp8_cols if cols else load().mb200_grouped_gemm_fp8
    _check(
        fn(
            mode, _ptr(a), _ptr(a_scale_t), a.shape[0], _ptr(w), _ptr(w_scale), w.shape[0], hidden, intermediate,
            _ptr(counts), _ptr(prefix), _ptr(sorted_ids), _ptr(row_scale), _ptr(out), _ptr(out_scale_t),
            _ptr(status), dev.index or 0, _stream(dev),
        ),
        "grouped_gemm_fp8",
    )


def moe_forward_fp8(x, w1, w2, w1_scale, w2_scale, topk_ids, topk_weights, expert_map, out, workspace):
    """Enqueue the fp8 block-quantised layer forward on the current stream."""
    t, hidden = x.shape
    e_local, two_n, _ = w1.shape
    dev = x.device
    _check(
        load().mb200_moe_forward_fp8(
            _ptr(x), _ptr(w1), _ptr(w2), _ptr(w1_scale), _ptr(w2_scale), _ptr(topk_ids), _ptr(topk_weights),
            _ptr(expert_map), _ptr(out), t, hidden, two_n // 2, e_local, topk_ids.shape[1], _ptr(workspace),
            workspace.numel(), dev.index or 0, _stream(dev),
        ),
        "moe_forward_fp8",
    )


DIST_SEQ_STRIDE = 4


def dist_symmetric_bytes(precision: int, tokens: int, hidden: int, topk: int, world: int) -> int:
    n = int(load().mb200_dist_symmetric_bytes(precision, tokens, hidden, topk, world))
    if n < 0:
        raise MB200Error("dist_symmetric_bytes: bad shape")
    return n


def dist_workspace_bytes(precision, tokens, hidden, intermediate, local_experts, topk, world) -> int:
    n = int(load().mb200_dist_workspace_bytes(precision, tokens, hidden, intermediate, local_experts, topk, world))
    if n < 0:
        raise MB200Error(f"dist_workspace_bytes: {load().mb200_last_error().decode()}")
    return n


def peer_pointer_array(ptrs):
    """ctypes ``void*[world]`` from a list of integer device addresses."""
    return (ctypes.c_void_p * len(ptrs))(*ptrs)


def peer_barrier(ptr_array, rank: int, world: int, seq: int, status: Optional[torch.Tensor], device) -> None:
    if status is not None:
        _need(status, torch.int32, "status")
        if status.numel() < 4:
            raise MB200Error("status: need the four-word head of a status block")
    _check(load().mb200_peer_barrier(ptr_array, rank, world, seq, _ptr(status), _stream(device)), "peer_barrier")


def dist_forward(precision, expert_parallel, x, w1, w2, w1_scale, w2_scale, topk_ids, topk_weights, expert_map,
                 out, global_experts, rank, world, ptr_array, symmetric_bytes, seq_base, workspace):
    """Enqueue one distributed layer forward (EP or TP) on the current stream."""
    t, hidden = x.shape
    e_local, two_n, _ = w1.shape
    dev = x.device
    _check(
        load().mb200_dist_forward(
            precision, 1 if expert_parallel else 0, _ptr(x), _ptr(w1), _ptr(w2), _ptr(w1_scale), _ptr(w2_scale),
            _ptr(topk_ids), _ptr(topk_weights), _ptr(expert_map), _ptr(out), t, hidden, two_n // 2, e_local,
            global_experts, topk_ids.shape[1], rank, world, ptr_array, symmetric_bytes, seq_base & 0xFFFFFFFF,
            _ptr(workspace), workspace.numel(), dev.index or 0, _stream(dev),
        ),
        "dist_forward",
    )


def read_status(workspace: torch.Tensor) -> int:
    """Synchronise and return the workspace status word (0 = ok)."""
    val = ctypes.c_int32(0)
    _check(load().mb200_read_status(_ptr(workspace), ctypes.byref(val), _stream(workspace.device)), "read_status")
    return int(val.value)


STAGE_NAMES = ("align", "gather_rows", "gate_up_gemm", "down_gemm", "combine")


def set_stage_events(events) -> None:
    """Have forward calls from this thread record ``events`` (six
    ``torch.cuda.Event(enable_timing=True)``, already recorded once so their
    handles exist) around the five stages; ``None`` switches it off."""
    if not events:
        _check(load().mb200_set_stage_events(None, 0), "set_stage_events")
        return
    arr = (ctypes.c_void_p * len(events))(*[ev.cuda_event for ev in events])
    _check(load().mb200_set_stage_events(arr, len(events)), "set_stage_events")


FP8_SCALE_FORMATS = {"fp32": 0, "ue8m0": 1}


def set_fp8_scale_format(fmt: str) -> None:
    """Format of the fp8 activation scales computed by later calls from this thread:
    ``"fp32"`` (amax/448) or ``"ue8m0"`` (rounded up to a power of two)."""
    if fmt not in FP8_SCALE_FORMATS:
        raise MB200Error(f"fp8 scale format {fmt!r}: expected one of {sorted(FP8_SCALE_FORMATS)}")
    _check(load().mb200_set_fp8_scale_format(FP8_SCALE_FORMATS[fmt]), "set_fp8_scale_format")


def reference_fp8_scale_format() -> str:
    """What the reference's activation quantiser does on this box.  The reference calls
    vLLM's ``per_token_group_quant_fp8`` without saying which scale format it wants
    (reference.py:143-145), and vLLM then follows ``is_deep_gemm_e8m0_used()``: power-of-two
    scales on GPUs where its DeepGEMM path is enabled (Hopper, Blackwell), fp32 elsewhere.
    Without vLLM there is no reference to match and the plain fp32 format applies."""
    if not torch.cuda.is_available():
        return "fp32"
    try:
        from vllm.utils.deep_gemm import is_deep_gemm_e8m0_used

        return "ue8m0" if is_deep_gemm_e8m0_used() else "fp32"
    except Exception:  # noqa: BLE001
        return "fp32"


def use_reference_fp8_scale_format() -> str:
    """Select, for this thread's direct calls, the scale format the reference uses on this
    box; returns it ("fp32" or "ue8m0") so that a checker can compute in the same format."""
    fmt = reference_fp8_scale_format()
    set_fp8_scale_format(fmt)
    return fmt


def set_comm_only(enabled: bool) -> None:
    """Forward calls from this thread move data only (GEMM kernels run with zero K steps)."""
    _check(load().mb200_set_comm_only(1 if enabled else 0), "set_comm_only")


def read_kernel_clocks(workspace: torch.Tensor) -> dict:
    """SM clock (MHz) the two GEMM kernels of the last forward ran at, from the
    cycle/nanosecond pairs the kernels leave in the workspace head.  Synchronises."""
    torch.cuda.synchronize(workspace.device)
    vals = workspace[32:64].view(torch.int64).cpu().tolist()
    out = {}
    for name, (cyc, ns) in (("gate_up_gemm", vals[0:2]), ("down_gemm", vals[2:4])):
        out[name] = None if ns <= 0 else round(cyc / ns * 1e3, 1)
    return out


# ---- products and norms around the expert FFN ----
# The tensors of these calls may be on any device: the call runs there, on that device's current stream.
# They stand outside autograd: a result carries no graph, whether or not an operand requires gradients.  A program that trains
# makes the backward calls itself, or from a torch.autograd.Function of its own.

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_H16 = {torch.bfloat16: PRECISION_BF16, torch.float16: PRECISION_FP16}
_NORM_TYPES = {**_H16, torch.float32: PRECISION_FP32}


def _h16(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise MB200Error(f"{name}: need a CUDA tensor, got one on {t.device}; there is no CPU path")
    precision = _H16.get(t.dtype)
    if precision is None:
        raise MB200Error(f"{name}: need bf16 or fp16, got {t.dtype}")
    return precision


# A call through Python costs about as much as the smallest kernels take, so the common case (whole, contiguous tensors
# on the current device) is told apart by a few attributes, and what is wrong is worked out only where something is.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch.cuda.current_device


def _pitch(t: torch.Tensor, like: torch.Tensor, shape, name: str, dtypes=None) -> int:
    """Elements from row to row of a matrix whose columns lie side by side; refuses every other layout."""
    if t.shape == shape and t.is_contiguous() and t.get_device() == like.get_device() and t.dtype in (dtypes or (like.dtype,)):
        # the stride of a single row says nothing, and contiguous rows are as far apart as they are long
        return shape[-1] if shape[-2] > 1 else (shape[-1] + 7) // 8 * 8
    dtypes = (like.dtype,) if dtypes is None else dtypes
    if t.dtype not in dtypes or t.device != like.device:
        raise MB200Error(f"{name}: need {' or '.join(map(str, dtypes))} on {like.device}, got {t.dtype} on {t.device}")
    if tuple(t.shape) != tuple(shape):
        raise MB200Error(f"{name}: need shape {tuple(shape)}, got {tuple(t.shape)}")
    rows, cols = shape[-2:]
    if cols != 1 and t.stride(-1) != 1:
        raise MB200Error(f"{name}: the elements of a row must lie side by side, got strides {t.stride()}")
    if rows <= 1:
        return (cols + 7) // 8 * 8
    if t.stride(-2) < cols:
        raise MB200Error(f"{name}: rows overlap (strides {t.stride()})")
    return t.stride(-2)


def _vector(t: Optional[torch.Tensor], like: torch.Tensor, n: int, name: str, dtypes) -> None:
    if t is None:
        return
    if t.dtype not in dtypes or t.get_device() != like.get_device() or t.shape != (n,) or not t.is_contiguous():
        raise MB200Error(f"{name}: need a contiguous vector of {n} elements of {' or '.join(map(str, dtypes))} on "
                         f"{like.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _output(t: torch.Tensor, like: torch.Tensor, shape, dtype, name: str) -> torch.Tensor:
    if t.dtype != dtype or t.get_device() != like.get_device() or t.shape != shape or not t.is_contiguous():
        raise MB200Error(f"{name}: need a contiguous tensor of {dtype} {tuple(shape)} on {like.device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t


def _dense_like(t: torch.Tensor, dtype) -> torch.Tensor:
    """A new dense tensor of t's shape; of a dense t it costs two thirds of what naming the shape does."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _scratch(nbytes: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    if nbytes < 0:
        raise MB200Error(load().mb200_last_error().decode())
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _elsewhere(device: int) -> bool:
    """Whether that device (negative: the CPU) is another GPU than the current one: the call is then made again with it current."""
    return device >= 0 and device != _current_device()


def linear(x, w, bias=None, activation: str = "none", residual=None, out=None, out_dtype=None, want_slope: bool = False):
    """``act(x @ w.T + bias) + residual`` for ``x [rows, k]``, ``w [n, k]`` of bf16 or fp16, summed in fp32 and rounded
    once.  ``bias [n]`` may be fp32; ``activation``: one of ``ACTIVATIONS``; ``out_dtype``: x's type or ``torch.float32``.
    Rows may be further apart than they are long (a multiple of 8 elements); ``k`` is a multiple of 8, ``n`` is free.
    ``out`` may be the residual itself.  With ``want_slope`` also returns ``act'(x @ w.T + bias)`` in x's type, which
    ``linear_backward`` takes."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return linear(x, w, bias, activation, residual, out, out_dtype, want_slope)
    precision = _h16(x, "x")
    if x.dim() != 2 or w.dim() != 2:
        raise MB200Error(f"linear: need matrices, got x {tuple(x.shape)} and w {tuple(w.shape)}")
    rows, k = x.shape
    n = w.shape[0]
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise MB200Error(f"activation {activation!r}: expected one of {sorted(ACTIVATIONS)}")
    xp = k if rows > 1 and x.is_contiguous() else _pitch(x, x, (rows, k), "x")
    wp = _pitch(w, x, (n, k), "w")
    _vector(bias, x, n, "bias", (x.dtype, torch.float32))
    rp = _pitch(residual, x, (rows, n), "residual") if residual is not None else 0
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise MB200Error(f"linear: output of {out_dtype} for operands of {x.dtype}")
    y = x.new_empty((rows, n), dtype=out_dtype) if out is None else _output(out, x, (rows, n), out_dtype, "out")
    slope = x.new_empty((rows, n)) if want_slope else None
    rc = load().mb200_linear(
        precision, x.data_ptr(), xp, rows, w.data_ptr(), wp, n, k, _ptr(bias), bias is not None and bias.dtype == torch.float32,
        act, _ptr(residual), rp, y.data_ptr(), out_dtype == torch.float32, _ptr(slope), dev,
        _raw_stream(dev),
    )
    _check(rc, "linear")
    return (y, slope) if want_slope else y


def _dw_type(w: torch.Tensor, dw_dtype):
    dw_dtype = w.dtype if dw_dtype is None else dw_dtype
    if dw_dtype not in (w.dtype, torch.float32):
        raise MB200Error(f"weight gradient of {dw_dtype} for weights of {w.dtype}")
    return dw_dtype


def linear_backward(dy, x, w, slope=None, dw_dtype=None, want_dx: bool = True, want_dw: bool = True, want_db: bool = True):
    """Gradients ``(dx, dw, db)`` of ``linear`` (None where not wanted; the residual's gradient is ``dy``).  ``slope``: what
    ``linear(..., want_slope=True)`` returned, None for no activation.  ``dy`` may be fp32 for bf16 operands.  ``dy * slope``
    is rounded to x's type once, for the products; ``db`` is its fp32 sum before that; ``dw`` has w's type, or fp32."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return linear_backward(dy, x, w, slope, dw_dtype, want_dx, want_dw, want_db)
    precision = _h16(x, "x")
    if x.dim() != 2 or w.dim() != 2:
        raise MB200Error(f"linear_backward: need matrices, got x {tuple(x.shape)} and w {tuple(w.shape)}")
    rows, k = x.shape
    n = w.shape[0]
    xp, wp = _pitch(x, x, (rows, k), "x"), _pitch(w, x, (n, k), "w")
    types = (x.dtype, torch.float32) if x.dtype == torch.bfloat16 else (x.dtype,)
    dp = _pitch(dy, x, (rows, n), "dy", types)
    if slope is not None:
        _output(slope, x, (rows, n), x.dtype, "slope")
    dw_dtype = _dw_type(w, dw_dtype)
    dx = _dense_like(x, x.dtype) if want_dx else None
    dw = _dense_like(w, dw_dtype) if want_dw else None
    db = x.new_empty(n, dtype=torch.float32) if want_db else None
    lib = load()
    copied = slope is not None or dp % 8 or dy.dtype == torch.float32 or dy.data_ptr() % 16
    ws = _scratch(lib.mb200_linear_backward_workspace_bytes(rows, n, 1 if copied else 0, dev), x)
    rc = lib.mb200_linear_backward(
        precision, dy.data_ptr(), dy.dtype == torch.float32, dp, _ptr(slope), x.data_ptr(), xp, rows, w.data_ptr(), wp, n, k,
        _ptr(dx), _ptr(dw), dw_dtype == torch.float32, _ptr(db), _ptr(ws), 0 if ws is None else ws.numel(), dev, _raw_stream(dev),
    )
    _check(rc, "linear_backward")
    return dx, dw, db


def _expert_weight(w: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor):
    """(experts, n, k, elements from row to row, from expert to expert)"""
    if x.dim() != 2 or w.dim() != 3:
        raise MB200Error(f"need x [rows, k] and w [experts, n, k], got {tuple(x.shape)} and {tuple(w.shape)}")
    e, n, k = w.shape
    wp = _pitch(w, x, (e, n, x.shape[1]), "w")
    ep = w.stride(0) if e > 1 else (n * wp + 7) // 8 * 8
    if ep < n * wp - (wp - k) and e > 1:
        raise MB200Error(f"w: experts overlap (strides {w.stride()})")
    _vector(offsets, x, e + 1, "offsets", (torch.int32,))
    return e, n, k, wp, ep


def grouped_linear(x, w, offsets, out=None):
    """``x[r] @ w[e].T`` for the rows of segment e = ``offsets[e] .. offsets[e + 1] - 1``, of any length: x [rows, k] and
    w [experts, n, k] of bf16 or fp16, offsets [experts + 1] int32 on x's device (``align(..., pad_rows=1)`` returns them as
    ``mtile_prefix``).  Rows outside the segments are left as they are in ``out``, undefined in a tensor made here."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return grouped_linear(x, w, offsets, out)
    precision = _h16(x, "x")
    e, n, k, wp, ep = _expert_weight(w, x, offsets)
    rows = x.shape[0]
    xp = _pitch(x, x, (rows, k), "x")
    y = x.new_empty((rows, n)) if out is None else _output(out, x, (rows, n), x.dtype, "out")
    rc = load().mb200_grouped_linear(precision, x.data_ptr(), xp, rows, w.data_ptr(), wp, ep, offsets.data_ptr(), e, n, k,
                                     y.data_ptr(), dev, _raw_stream(dev))
    _check(rc, "grouped_linear")
    return y


def grouped_linear_backward(dy, x, w, offsets, dw_dtype=None, dx_out=None, want_dx: bool = True, want_dw: bool = True):
    """Gradients ``(dx, dw)`` of ``grouped_linear`` (None where not wanted).  Rows outside the segments have no part in
    ``dw`` and are left as they are in ``dx_out``; an expert without rows gets a zero gradient.  ``dw`` has w's type, or fp32."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return grouped_linear_backward(dy, x, w, offsets, dw_dtype, dx_out, want_dx, want_dw)
    precision = _h16(x, "x")
    e, n, k, wp, ep = _expert_weight(w, x, offsets)
    rows = x.shape[0]
    xp, dp = _pitch(x, x, (rows, k), "x"), _pitch(dy, x, (rows, n), "dy")
    dw_dtype = _dw_type(w, dw_dtype)
    dx = None
    if want_dx:
        dx = _dense_like(x, x.dtype) if dx_out is None else _output(dx_out, x, (rows, k), x.dtype, "dx_out")
    dw = _dense_like(w, dw_dtype) if want_dw else None
    lib = load()
    copied = dp % 8 or dy.data_ptr() % 16
    ws = _scratch(lib.mb200_grouped_linear_backward_workspace_bytes(rows, n), x) if copied else None
    rc = lib.mb200_grouped_linear_backward(
        precision, dy.data_ptr(), dp, x.data_ptr(), xp, rows, w.data_ptr(), wp, ep, offsets.data_ptr(), e, n, k, _ptr(dx), _ptr(dw),
        dw_dtype == torch.float32, _ptr(ws), 0 if ws is None else ws.numel(), dev, _raw_stream(dev),
    )
    _check(rc, "grouped_linear_backward")
    return dx, dw


def linear_status(device=None, clear: bool = False) -> int:
    """Synchronise the device's current stream and return the status word of the products above (0 = every in-kernel wait
    completed); ``clear`` sets it back to 0."""
    val = ctypes.c_int32(0)
    with torch.cuda.device(device):
        _check(load().mb200_linear_status(ctypes.byref(val), 1 if clear else 0, _stream(device)), "linear_status")
    return int(val.value)


def _norm_operands(x, weight, bias, name: str):
    if not x.is_cuda:
        raise MB200Error(f"{name}: need CUDA tensors, got one on {x.device}; there is no CPU path")
    precision = _NORM_TYPES.get(x.dtype)
    if precision is None:
        raise MB200Error(f"{name}: need bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] == 0:
        raise MB200Error(f"{name}: need x [rows, hidden], got {tuple(x.shape)}")
    rows, h = x.shape
    _vector(weight, x, h, "weight", (x.dtype, torch.float32))
    _vector(bias, x, h, "bias", (x.dtype, torch.float32))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise MB200Error(f"{name}: weight and bias of one type, got {weight.dtype} and {bias.dtype}")
    params = weight if weight is not None else bias
    return precision, rows, h, params is not None and params.dtype == torch.float32


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None):
    """Layer norm of the rows of ``x [rows, hidden]`` (bf16, fp16 or fp32; rows may be any distance apart): returns
    ``(y, mean, rstd)``, the last two in fp32 for ``layer_norm_backward``.  weight and bias have x's type or fp32.
    ``out`` may be a contiguous x itself."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return layer_norm(x, weight, bias, eps, out)
    precision, rows, h, fp32 = _norm_operands(x, weight, bias, "layer_norm")
    xp = _pitch(x, x, (rows, h), "x")
    y = _dense_like(x, x.dtype) if out is None else _output(out, x, (rows, h), x.dtype, "out")
    mean, rstd = x.new_empty(rows, dtype=torch.float32), x.new_empty(rows, dtype=torch.float32)
    rc = load().mb200_layer_norm(precision, x.data_ptr(), xp, rows, h, _ptr(weight), _ptr(bias), fp32, eps, y.data_ptr(),
                                 mean.data_ptr(), rstd.data_ptr(), dev, _raw_stream(dev))
    _check(rc, "layer_norm")
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, want_dx: bool = True, want_dweight: bool = True, want_dbias: bool = True):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm`` (None where not wanted); the last two are fp32 sums over the rows,
    in a fixed order."""
    dev = x.get_device()
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return layer_norm_backward(dy, x, mean, rstd, weight, want_dx, want_dweight, want_dbias)
    precision, rows, h, fp32 = _norm_operands(x, weight, None, "layer_norm_backward")
    xp, dp = _pitch(x, x, (rows, h), "x"), _pitch(dy, x, (rows, h), "dy")
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        _vector(t, x, rows, what, (torch.float32,))
    dx = _dense_like(x, x.dtype) if want_dx else None
    dweight = x.new_empty(h, dtype=torch.float32) if want_dweight else None
    dbias = x.new_empty(h, dtype=torch.float32) if want_dbias else None
    lib = load()
    ws = None
    if want_dweight or want_dbias:
        ws = _scratch(lib.mb200_layer_norm_backward_workspace_bytes(rows, h, dev), x)
    rc = lib.mb200_layer_norm_backward(
        precision, dy.data_ptr(), dp, x.data_ptr(), xp, rows, h, mean.data_ptr(), rstd.data_ptr(), _ptr(weight), fp32, _ptr(dx),
        _ptr(dweight), _ptr(dbias), _ptr(ws), 0 if ws is None else ws.numel(), dev, _raw_stream(dev),
    )
    _check(rc, "layer_norm_backward")
    return dx, dweight, dbias
