"""Torch-facing B200 operators with the reference kernel-registry signatures.

Every function here validates its arguments the way the reference entry point
does (``TypeError`` for rank/dtype, ``ValueError`` for shape/device), allocates
its outputs through the torch caching allocator, and launches the CUDA kernels
of ``libkimi_b200.so`` on ``torch.cuda.current_stream()``.  There is no CPU or
library fallback: CPU tensors raise ``ValueError`` and a missing library
raises ``RuntimeError``.  No call synchronizes the host, so the operators can
be captured in a CUDA graph after one warm-up call per shape (which loads the
kernels).  Scratch with counters is kept between calls; a graph has its own.

Reference entry points mirrored here:
  w4a16_dense       engine/kernels/w4a16_dense_gemv.py:312-336 (validation :171-197)
  w4a16_grouped     engine/kernels/w4a16_gemv.py:610-635 (validation :449-488)
  w4a16_swiglu      engine/kernels/w4a16_gemv.py:772-790, engine/kernels/__init__.py:182-197
  fused_w2_combine  engine/kernels/moe_combine.py:264-324 (validation :157-206)
  fused_qkv_w4a16   engine/kernels/w4a16_fused_qkv.py:342-389
  kda_decode_step   engine/kernels/kda_step.py:273-293 (validation :137-170)
  moe_router        engine/klinear/router.py:47-85
  quantise          engine/quant/w4a16.py:68-105 (group size as a parameter)

Operators of a speculative serving step that the reference has no kernel for
(its MLA attention is torch einsum and softmax over projected keys and values,
engine/klinear/attention.py:586-598): paged_plan, paged_append,
prompt_attention, tree_attention, verify_drafts.
"""

from __future__ import annotations

import threading
from ctypes import byref, c_float, c_int64, c_size_t, c_uint64, c_void_p
from functools import partial
from typing import Callable, NamedTuple

import torch

from . import _lib

REFERENCE_GROUP_SIZE = 32


# ---------------------------------------------------------------------------
# helpers
# ---------------------------------------------------------------------------


def _stream(device: torch.device) -> c_void_p:
    return c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _on(device: torch.device) -> Callable[..., None]:
    """The C call for tensors of a device, which need not be the current one (kernels are
    launched on the current one)."""
    index = device.index
    return _lib.call if index is None or index == _current_device() else partial(_call_on, device)


def _call_on(device: torch.device, function: str, *args: object) -> None:
    with torch.cuda.device(device):
        _lib.call(function, *args)


_current_device = torch._C._cuda_getDevice


def _p(tensor: torch.Tensor | None) -> c_void_p:
    return c_void_p(0 if tensor is None else tensor.data_ptr())


def _require_cuda(tensor: torch.Tensor, what: str) -> None:
    if tensor.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA")


def group_size_of(reduction: int, scale_columns: int) -> int:
    """Group size implied by a reduction width and the scale tensor's width."""
    if scale_columns <= 0 or reduction % scale_columns:
        raise ValueError(
            f"scales with {scale_columns} columns cannot cover a reduction width of {reduction}"
        )
    group = reduction // scale_columns
    if group < 32 or group % 32 or (group & (group - 1)):
        raise ValueError(f"group size {group} must be 32 times a power of two")
    return group


def _rows_16b(t: torch.Tensor) -> torch.Tensor:
    """Return ``t`` (2-D) with unit inner stride, 16-byte aligned rows."""
    if (
        t.stride(-1) != 1
        or t.stride(0) % 8
        or t.data_ptr() % 16
        or t.stride(0) < t.shape[-1]
    ):
        t = t.contiguous()
    return t


def _dense_contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.contiguous()


_WORKSPACES: dict[tuple, torch.Tensor] = {}
_lib.on_wait_error.append(_WORKSPACES.clear)
_CAPTURED: dict[tuple, tuple[int, torch.Tensor]] = {}


def _capturing() -> bool:
    """Whether the current stream records a CUDA graph."""
    return torch._C._cuda_isCurrentStreamCapturing()


def _capture_id(stream: int) -> int:
    """Which capture the stream is in (another one for each)."""
    out = c_uint64(0)
    _lib.call("kb_stream_capture_id", stream, byref(out))
    return out.value


def _kept_scratch(key: tuple, device: torch.device, stream: int, nbytes: int,
                  counters: int) -> torch.Tensor:
    """Scratch whose first ``counters`` bytes are zero, and are left zero by each call.

    Kept per key (which names the stream) for calls that follow each other there.  A
    graph has scratch of its own, made and zeroed by its first call in the graph's
    memory: graphs are replayed in any order and on any stream, beside each other and
    beside calls outside of them.
    """
    if not _capturing():
        ws = _WORKSPACES.get(key)
        if ws is None:
            ws = _WORKSPACES[key] = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        return ws
    capture = _capture_id(stream)
    held = _CAPTURED.get(key)
    if held is None or held[0] != capture:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:counters].zero_()
        held = _CAPTURED[key] = (capture, ws)
    return held[1]


def _workspace(kind: str, device: torch.device, nbytes: int, shape: tuple) -> torch.Tensor:
    """Zero-filled scratch kept per (kind, device, stream, problem shape).

    The router and down+combine kernels keep arrival counters in their scratch
    and leave them at zero after every call.  The counters' position depends on
    the problem shape, so a buffer is reused only for the same shape: a buffer
    shared between shapes could place one shape's counters on another shape's
    leftover data.
    """
    stream = torch.cuda.current_stream(device).cuda_stream
    index = device.index if device.index is not None else torch.cuda.current_device()
    nbytes = max(int(nbytes), 256)
    return _kept_scratch((kind, index, stream, shape), device, stream, nbytes, nbytes)


# ---------------------------------------------------------------------------
# dense
# ---------------------------------------------------------------------------


def _validate_dense(
    activations: torch.Tensor, packed_weights: torch.Tensor, scales: torch.Tensor
) -> tuple[int, int, int, int]:
    if activations.ndim != 2 or activations.dtype != torch.bfloat16:
        raise TypeError("activations must be a BF16 [tokens, reduction] matrix")
    if packed_weights.ndim != 2 or packed_weights.dtype != torch.uint8:
        raise TypeError("packed weights must be a uint8 [output, reduction / 2] matrix")
    if scales.ndim != 2 or scales.dtype != torch.bfloat16:
        raise TypeError("scales must be a BF16 [output, reduction / group] matrix")
    _require_cuda(activations, "W4A16 dense GEMV")
    if not (activations.device == packed_weights.device == scales.device):
        raise ValueError("activations, packed weights, and scales must share a device")
    m, reduction = activations.shape
    output_size, packed_reduction = packed_weights.shape
    if output_size == 0 or reduction == 0:
        raise ValueError("W4A16 dense GEMV requires nonzero dimensions")
    if reduction % 32:
        raise ValueError("the reduction dimension must be divisible by group size 32")
    if packed_reduction * 2 != reduction:
        raise ValueError("packed weights have the wrong reduction width")
    if scales.shape[0] != output_size:
        raise ValueError("W4A16 scales have the wrong shape")
    group = group_size_of(reduction, scales.shape[1])
    return m, output_size, reduction, group


# Tensor-core (tcgen05) limits: K a multiple of 128, N of 8, at most 81 scale
# groups per row (the per-CTA scale buffers).
TC_MAX_GROUPS_PER_ROW = 81


def tc_supported(m: int, n: int, k: int, group: int) -> bool:
    return k % 128 == 0 and n % 8 == 0 and k // group <= TC_MAX_GROUPS_PER_ROW and m > 0


def prefer_tc(m: int, n: int, k: int, group: int) -> bool:
    """Whether the tensor-core path beats the projection engine for this shape.

    Measured on B200 (dense sweep over the decode shapes): the engine decodes
    each weight once per 16-token group, the tensor-core path once per 64
    tokens, so the tensor cores win from 64 tokens on every shape, from 32 on
    matrices of 16M+ weights and from 16 on the 9216-wide reduction.
    """
    if not tc_supported(m, n, k, group):
        return False
    if m >= 64:
        return True
    if m >= 32 and n * k >= 16 * 2**20:
        return True
    return m >= 16 and k >= 8192


def w4a16_dense(
    activations: torch.Tensor, packed_weights: torch.Tensor, scales: torch.Tensor
) -> torch.Tensor:
    """y[M,N] = activations[M,K] . dequant(W[N,K])^T, bf16 out (registry op w4a16_dense).

    Small token counts run on the projection engine, many tokens on the
    tcgen05 tensor-core path (``prefer_tc``); both keep the result contract.
    """
    m, n, k, group = _validate_dense(activations, packed_weights, scales)
    if prefer_tc(m, n, k, group):
        return w4a16_dense_tc(activations, packed_weights, scales)
    return w4a16_dense_engine(activations, packed_weights, scales)


def w4a16_dense_engine(
    activations: torch.Tensor, packed_weights: torch.Tensor, scales: torch.Tensor
) -> torch.Tensor:
    """w4a16_dense on the projection engine (kb_w4a16_dense), whatever the token count."""
    m, n, k, group = _validate_dense(activations, packed_weights, scales)
    out = torch.empty((m, n), dtype=torch.bfloat16, device=activations.device)
    if m == 0:
        return out
    x = _rows_16b(activations)
    packed = _dense_contig(packed_weights)
    sc = _dense_contig(scales)
    _on(x.device)(
        "kb_w4a16_dense",
        _p(x), c_int64(x.stride(0)), c_int64(m), c_int64(k), _p(packed), _p(sc), c_int64(n),
        c_int64(group), _p(out), c_int64(out.stride(0)), _stream(x.device),
    )
    return out


def multi_prefers_tc(problems: list[tuple[torch.Tensor, torch.Tensor, torch.Tensor]]) -> bool:
    """Whether ``w4a16_dense_multi`` runs these problems on the tensor-core path."""
    return bool(problems) and all(prefer_tc(*_validate_dense(*pr)) for pr in problems)


def w4a16_dense_multi(
    problems: list[tuple[torch.Tensor, torch.Tensor, torch.Tensor]],
) -> list[torch.Tensor]:
    """Several independent dense projections in one launch (one tensor-core
    launch each when ``prefer_tc`` picks that path for every problem)."""
    if len(problems) > _lib.MAX_DENSE_PROBLEMS:
        raise ValueError(f"at most {_lib.MAX_DENSE_PROBLEMS} problems per launch")
    if multi_prefers_tc(problems):
        return [w4a16_dense_tc(*pr) for pr in problems]
    arr = (_lib.DenseProblem * max(1, len(problems)))()
    outs: list[torch.Tensor] = []
    keep: list[torch.Tensor] = []
    device = None
    for i, (activations, packed_weights, scales) in enumerate(problems):
        m, n, k, group = _validate_dense(activations, packed_weights, scales)
        if device is None:
            device = activations.device
        elif activations.device != device:
            raise ValueError("all problems must share one device")
        out = torch.empty((m, n), dtype=torch.bfloat16, device=activations.device)
        outs.append(out)
        x = _rows_16b(activations) if m else activations
        packed = _dense_contig(packed_weights)
        sc = _dense_contig(scales)
        keep.extend((x, packed, sc))
        arr[i].x = x.data_ptr() if m else 0
        arr[i].x_stride = x.stride(0) if m else k
        arr[i].M = m
        arr[i].K = k
        arr[i].packed = packed.data_ptr()
        arr[i].scales = sc.data_ptr()
        arr[i].N = n
        arr[i].group = group
        arr[i].y = out.data_ptr()
        arr[i].y_stride = out.stride(0)
    if device is not None:
        _on(device)("kb_w4a16_dense_multi", arr, len(problems), _stream(device))
    return outs


def fused_qkv_w4a16(
    activations: torch.Tensor,
    q_packed: torch.Tensor,
    q_scales: torch.Tensor,
    k_packed: torch.Tensor,
    k_scales: torch.Tensor,
    v_packed: torch.Tensor,
    v_scales: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Q, K and V projections of one activation in one launch."""
    q, k, v = w4a16_dense_multi(
        [(activations, q_packed, q_scales), (activations, k_packed, k_scales),
         (activations, v_packed, v_scales)]
    )
    return q, k, v


def w4a16_dense_tc(
    activations: torch.Tensor, packed_weights: torch.Tensor, scales: torch.Tensor,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """w4a16_dense on the tcgen05 tensor-core path (many tokens); same result contract."""
    m, n, k, group = _validate_dense(activations, packed_weights, scales)
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=activations.device)
    if m == 0:
        return out
    x = _rows_16b(activations)
    packed = _dense_contig(packed_weights)
    sc = _dense_contig(scales)
    need = int(_lib.lib().kb_w4a16_dense_tc_workspace_size(m, k, n))
    ws = _workspace("dense_tc", x.device, need, (m, k, n)) if need else None
    _on(x.device)(
        "kb_w4a16_dense_tc",
        _p(x), c_int64(x.stride(0)), c_int64(m), c_int64(k), _p(packed), _p(sc), c_int64(n),
        c_int64(group), _p(out), c_int64(out.stride(0)), _p(ws),
        c_size_t(0 if ws is None else ws.numel()), _stream(x.device),
    )
    return out


# ---------------------------------------------------------------------------
# grouped
# ---------------------------------------------------------------------------


def _validate_grouped(
    activations: torch.Tensor,
    expert_indices: torch.Tensor,
    packed_weights: torch.Tensor,
    scales: torch.Tensor,
) -> tuple[int, int, int, int, int, int]:
    if activations.ndim != 2 or activations.dtype != torch.bfloat16:
        raise TypeError("activations must be a BF16 [tokens, reduction] matrix")
    if expert_indices.ndim != 2 or expert_indices.dtype != torch.long:
        raise TypeError("expert_indices must be an int64 [tokens, routes] matrix")
    if packed_weights.ndim != 3 or scales.ndim != 3:
        raise ValueError("grouped packed weights and scales must be rank three")
    if packed_weights.dtype != torch.uint8:
        raise TypeError("packed grouped weights must use torch.uint8 storage")
    if scales.dtype != torch.bfloat16:
        raise TypeError("grouped W4A16 scales must use torch.bfloat16 storage")
    _require_cuda(activations, "grouped W4A16 decode")
    if not (
        activations.device == expert_indices.device == packed_weights.device == scales.device
    ):
        raise ValueError("grouped W4A16 inputs must share one device")
    tokens, reduction = activations.shape
    route_tokens, routes = expert_indices.shape
    experts, output_size, packed_reduction = packed_weights.shape
    if route_tokens != tokens:
        raise ValueError("expert routing must have one row per token")
    if routes == 0 or experts == 0 or output_size == 0 or reduction == 0:
        raise ValueError("grouped W4A16 decode requires nonzero dimensions")
    if reduction % 32:
        raise ValueError("grouped W4A16 reduction width must be divisible by 32")
    if packed_reduction * 2 != reduction:
        raise ValueError("packed grouped weights have the wrong reduction width")
    if scales.shape[:2] != (experts, output_size):
        raise ValueError("grouped W4A16 scales have the wrong shape")
    group = group_size_of(reduction, scales.shape[2])
    if tokens * routes > _lib.MAX_ASSIGNMENTS:
        raise ValueError(
            f"tokens * routes = {tokens * routes} exceeds {_lib.MAX_ASSIGNMENTS} per call"
        )
    return tokens, routes, output_size, reduction, experts, group


def w4a16_grouped(
    activations: torch.Tensor,
    expert_indices: torch.Tensor,
    packed_weights: torch.Tensor,
    scales: torch.Tensor,
) -> torch.Tensor:
    """y[t,r] = x[t] . dequant(W[idx[t,r]])^T, bf16 [T,R,N] (registry op w4a16_grouped)."""
    t, r, n, k, e, group = _validate_grouped(activations, expert_indices, packed_weights, scales)
    out = torch.empty((t, r, n), dtype=torch.bfloat16, device=activations.device)
    if t == 0:
        return out
    x = _rows_16b(activations)
    idx = _dense_contig(expert_indices)
    packed = _dense_contig(packed_weights)
    sc = _dense_contig(scales)
    _on(x.device)(
        "kb_w4a16_grouped",
        _p(x), c_int64(x.stride(0)), c_int64(t), c_int64(k), _p(idx), c_int64(r), _p(packed),
        _p(sc), c_int64(e), c_int64(n), c_int64(group), _p(out), _stream(x.device),
    )
    return out


def w4a16_grouped_tc(
    activations: torch.Tensor,
    expert_indices: torch.Tensor,
    packed_weights: torch.Tensor,
    scales: torch.Tensor,
) -> torch.Tensor:
    """w4a16_grouped on the tcgen05 tensor-core path; same result contract."""
    t, r, n, k, e, group = _validate_grouped(activations, expert_indices, packed_weights, scales)
    out = torch.empty((t, r, n), dtype=torch.bfloat16, device=activations.device)
    if t == 0:
        return out
    x = _rows_16b(activations)
    idx = _dense_contig(expert_indices)
    packed = _dense_contig(packed_weights)
    sc = _dense_contig(scales)
    _on(x.device)(
        "kb_w4a16_grouped_tc",
        _p(x), c_int64(x.stride(0)), c_int64(t), c_int64(k), _p(idx), c_int64(r), _p(packed),
        _p(sc), c_int64(e), c_int64(n), c_int64(group), _p(out), _stream(x.device),
    )
    return out


def w4a16_swiglu_tc(
    activations: torch.Tensor,
    expert_indices: torch.Tensor,
    w1_packed: torch.Tensor,
    w1_scales: torch.Tensor,
    w3_packed: torch.Tensor,
    w3_scales: torch.Tensor,
) -> torch.Tensor:
    """w4a16_swiglu on the tcgen05 tensor-core path; same rounding contract."""
    dims = _validate_grouped(activations, expert_indices, w1_packed, w1_scales)
    if _validate_grouped(activations, expert_indices, w3_packed, w3_scales) != dims:
        raise ValueError("grouped W1 and W3 dimensions must match")
    if w3_packed.shape != w1_packed.shape or w3_scales.shape != w1_scales.shape:
        raise ValueError("grouped W1 and W3 shapes must match")
    t, r, n, k, e, group = dims
    out = torch.empty((t, r, n), dtype=torch.bfloat16, device=activations.device)
    if t == 0:
        return out
    x = _rows_16b(activations)
    idx = _dense_contig(expert_indices)
    p1, s1 = _dense_contig(w1_packed), _dense_contig(w1_scales)
    p3, s3 = _dense_contig(w3_packed), _dense_contig(w3_scales)
    _on(x.device)(
        "kb_w4a16_swiglu_tc",
        _p(x), c_int64(x.stride(0)), c_int64(t), c_int64(k), _p(idx), c_int64(r), _p(p1),
        _p(s1), _p(p3), _p(s3), c_int64(e), c_int64(n), c_int64(group), _p(out),
        _stream(x.device),
    )
    return out


def w4a16_swiglu(
    activations: torch.Tensor,
    expert_indices: torch.Tensor,
    w1_packed: torch.Tensor,
    w1_scales: torch.Tensor,
    w3_packed: torch.Tensor,
    w3_scales: torch.Tensor,
) -> torch.Tensor:
    """silu(x.W1[e]) * (x.W3[e]) with the bf16 rounding contract (registry op w4a16_swiglu)."""
    dims = _validate_grouped(activations, expert_indices, w1_packed, w1_scales)
    dims3 = _validate_grouped(activations, expert_indices, w3_packed, w3_scales)
    if dims3 != dims:
        raise ValueError("grouped W1 and W3 dimensions must match")
    if w3_packed.shape != w1_packed.shape:
        raise ValueError("grouped W1 and W3 packed shapes must match")
    if w3_scales.shape != w1_scales.shape:
        raise ValueError("grouped W1 and W3 scale shapes must match")
    t, r, n, k, e, group = dims
    out = torch.empty((t, r, n), dtype=torch.bfloat16, device=activations.device)
    if t == 0:
        return out
    x = _rows_16b(activations)
    idx = _dense_contig(expert_indices)
    p1, s1 = _dense_contig(w1_packed), _dense_contig(w1_scales)
    p3, s3 = _dense_contig(w3_packed), _dense_contig(w3_scales)
    _on(x.device)(
        "kb_w4a16_swiglu",
        _p(x), c_int64(x.stride(0)), c_int64(t), c_int64(k), _p(idx), c_int64(r), _p(p1),
        _p(s1), _p(p3), _p(s3), c_int64(e), c_int64(n), c_int64(group), _p(out),
        _stream(x.device),
    )
    return out


def _validate_combine(
    activated: torch.Tensor,
    expert_indices: torch.Tensor,
    combine_weights: torch.Tensor,
    w2_packed: torch.Tensor,
    w2_scales: torch.Tensor,
    weight_routes: int | None = None,
) -> tuple[int, int, int, int, int, int]:
    if activated.ndim != 3 or activated.dtype != torch.bfloat16:
        raise TypeError("activated must be a BF16 [tokens, routes, reduction] tensor")
    if expert_indices.ndim != 2 or expert_indices.dtype != torch.long:
        raise TypeError("expert_indices must be an int64 [tokens, routes] matrix")
    if combine_weights.ndim != 2 or combine_weights.dtype != torch.float32:
        raise TypeError("combine_weights must be a float32 [tokens, routes] matrix")
    if w2_packed.ndim != 3 or w2_scales.ndim != 3:
        raise ValueError("grouped W2 packed weights and scales must be rank three")
    if w2_packed.dtype != torch.uint8:
        raise TypeError("grouped W2 packed weights must use torch.uint8 storage")
    if w2_scales.dtype != torch.bfloat16:
        raise TypeError("grouped W2 scales must use torch.bfloat16 storage")
    _require_cuda(activated, "fused W2 combine")
    if not (
        activated.device
        == expert_indices.device
        == combine_weights.device
        == w2_packed.device
        == w2_scales.device
    ):
        raise ValueError("fused W2 combine inputs must share one device")
    tokens, routes, reduction = activated.shape
    experts, output_size, packed_reduction = w2_packed.shape
    if expert_indices.shape != (tokens, routes):
        raise ValueError("expert_indices must match the activated token-route shape")
    expected_w = routes if weight_routes is None else weight_routes
    if combine_weights.shape != (tokens, expected_w):
        raise ValueError("combine_weights must match the activated token-route shape")
    if routes == 0 or experts == 0 or output_size == 0 or reduction == 0:
        raise ValueError("fused W2 combine requires nonzero route and weight dimensions")
    if reduction % 32:
        raise ValueError("the grouped W2 reduction width must be divisible by 32")
    if packed_reduction * 2 != reduction:
        raise ValueError("grouped W2 packed weights have the wrong reduction width")
    if w2_scales.shape[:2] != (experts, output_size):
        raise ValueError("grouped W2 scales have the wrong shape")
    group = group_size_of(reduction, w2_scales.shape[2])
    if tokens * routes > _lib.MAX_ASSIGNMENTS:
        raise ValueError(
            f"tokens * routes = {tokens * routes} exceeds {_lib.MAX_ASSIGNMENTS} per call"
        )
    return tokens, routes, output_size, reduction, experts, group


def _down_combine(
    activated: torch.Tensor,
    expert_indices: torch.Tensor,
    combine_weights: torch.Tensor,
    w2_packed: torch.Tensor,
    w2_scales: torch.Tensor,
    dims: tuple[int, int, int, int, int, int],
) -> torch.Tensor:
    t, r, n, k, e, group = dims
    out = torch.empty((t, n), dtype=torch.bfloat16, device=activated.device)
    if t == 0:
        return out
    act = _dense_contig(activated)
    idx = _dense_contig(expert_indices)
    cw = combine_weights if combine_weights.stride(-1) == 1 else combine_weights.contiguous()
    p2, s2 = _dense_contig(w2_packed), _dense_contig(w2_scales)
    lib = _lib.lib()
    need = int(lib.kb_w4a16_w2_combine_workspace_size(t, r, n))
    ws = _workspace("w2_combine", act.device, need, (t, r, n))
    _on(act.device)(
        "kb_w4a16_w2_combine",
        _p(act), c_int64(t), c_int64(r), c_int64(k), _p(idx), _p(cw), c_int64(cw.stride(0)),
        _p(p2), _p(s2), c_int64(e), c_int64(n), c_int64(group), _p(out), _p(ws),
        c_size_t(ws.numel()), _stream(act.device),
    )
    return out


def fused_w2_combine(
    activated: torch.Tensor,
    expert_indices: torch.Tensor,
    combine_weights: torch.Tensor,
    w2_packed: torch.Tensor,
    w2_scales: torch.Tensor,
) -> torch.Tensor:
    """Down projection of every route plus the weighted combine, bf16 [T,N].

    The last route is the shared expert, added with weight exactly 1; its
    entry in ``combine_weights`` is ignored (moe_combine.py:209-261).
    """
    dims = _validate_combine(activated, expert_indices, combine_weights, w2_packed, w2_scales)
    return _down_combine(activated, expert_indices, combine_weights, w2_packed, w2_scales, dims)


def moe_down_combine(
    activated: torch.Tensor,
    stable_indices: torch.Tensor,
    expert_weights: torch.Tensor,
    w2_packed: torch.Tensor,
    w2_scales: torch.Tensor,
) -> torch.Tensor:
    """``fused_w2_combine`` taking the router's [T, R-1] weights directly.

    This is the form the MoE layer uses (engine/klinear/moe.py:317-334): the
    routed weights have one column per routed expert, the shared route last.
    """
    dims = _validate_combine(
        activated, stable_indices, expert_weights, w2_packed, w2_scales,
        weight_routes=activated.shape[1] - 1 if activated.ndim == 3 else None,
    )
    return _down_combine(activated, stable_indices, expert_weights, w2_packed, w2_scales, dims)


def moe_combine_routes(routes: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """bf16(sum_r float(routes[:, r]) * weights[:, r]) + routes[:, -1], bf16 [T, N].

    ``routes`` bf16 [T, R, N] holds the per-route expert outputs with the
    shared expert last; ``weights`` fp32 [T, >= R-1] the routing weights.  The
    combine half of fused_w2_combine, for outputs computed elsewhere (expert
    parallelism).
    """
    if routes.dtype != torch.bfloat16 or routes.ndim != 3:
        raise TypeError("routes must be BF16 [T, R, N]")
    if weights.dtype != torch.float32 or weights.ndim != 2:
        raise TypeError("weights must be FP32 [T, R-1]")
    t, r, n = routes.shape
    if weights.shape[0] != t or (r > 1 and weights.shape[1] < r - 1):
        raise ValueError("weights must have T rows and at least R-1 columns")
    if n % 8:
        raise ValueError("width must be a multiple of 8")
    _require_cuda(routes, "B200 combine")
    if weights.device != routes.device:
        raise ValueError("weights must be on the same CUDA device as routes")
    out = torch.empty((t, n), dtype=torch.bfloat16, device=routes.device)
    if t == 0:
        return out
    y = routes.contiguous()
    w = weights if weights.stride(1) == 1 else weights.contiguous()
    _on(y.device)("kb_moe_combine_routes", _p(y), c_int64(t), c_int64(r), c_int64(n), _p(w),
              c_int64(w.stride(0)), _p(out), _stream(y.device))
    return out


# ---------------------------------------------------------------------------
# expert-parallel data plane
# ---------------------------------------------------------------------------


def ep_dispatch(hidden: torch.Tensor, routed: torch.Tensor, per_rank: int, world: int,
                capacity: int, shared_id: int = -1) -> tuple[torch.Tensor, torch.Tensor]:
    """Pack each routed (token, route) pair's hidden row for its expert's rank.

    hidden bf16 [T, H]; routed int64 [T, k] global expert ids.  Returns
    (payload bf16 [world*capacity, H+8]: per slot the row, then the
    owner-local expert id as an int64 in the next four bf16 -- -1 for an
    unused slot; slots int32 [T*k]: the payload slot of each pair).
    capacity must be at least T*k.  With ``shared_id`` >= 0 the payload has T
    more rows after the slots: row world*capacity + t is hidden[t] with id
    ``shared_id`` (the rank's own rows for its shared expert, not exchanged).
    """
    if hidden.dtype != torch.bfloat16 or hidden.ndim != 2:
        raise TypeError("hidden must be BF16 [T, H]")
    if routed.dtype != torch.long or routed.ndim != 2 or routed.shape[0] != hidden.shape[0]:
        raise TypeError("routed must be int64 [T, k]")
    _require_cuda(hidden, "expert-parallel dispatch")
    if routed.device != hidden.device:
        raise ValueError("routed must be on the device of hidden")
    t, h = hidden.shape
    k = routed.shape[1]
    if capacity < t * k:
        raise ValueError("capacity must be at least tokens * top_k")
    extra = t if shared_id >= 0 else 0
    payload = torch.empty((world * capacity + extra, h + 8), dtype=torch.bfloat16,
                          device=hidden.device)
    slots = torch.empty((t * k,), dtype=torch.int32, device=hidden.device)
    if t == 0:
        payload_ids(payload[:world * capacity]).fill_(-1)
        return payload, slots
    x = _rows_16b(hidden)
    r = routed if routed.stride(1) == 1 else routed.contiguous()
    _on(x.device)("kb_ep_dispatch", _p(x), c_int64(x.stride(0)), c_int64(t), c_int64(h), _p(r),
              c_int64(r.stride(0)), c_int64(k), c_int64(per_rank), c_int64(world),
              c_int64(capacity), c_int64(shared_id), _p(payload), _p(slots), _stream(x.device))
    return payload, slots


def payload_ids(payload: torch.Tensor) -> torch.Tensor:
    """The int64 expert-id column of a dispatch payload, [n, 1] (a view)."""
    h = payload.shape[1] - 8
    return payload[:, h:h + 4].view(torch.long)


def ep_combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor,
               shared: torch.Tensor) -> torch.Tensor:
    """bf16(sum_r float(y[slots[t,r]]) * weights[t,r]) + shared[t], bf16 [T, H]."""
    if y.dtype != torch.bfloat16 or shared.dtype != torch.bfloat16:
        raise TypeError("y and shared must be BF16")
    if weights.dtype != torch.float32 or slots.dtype != torch.int32:
        raise TypeError("weights must be FP32 and slots int32")
    _require_cuda(y, "expert-parallel combine")
    if not (slots.device == weights.device == shared.device == y.device):
        raise ValueError("combine inputs must share one device")
    t, h = shared.shape
    k = weights.shape[1]
    if slots.numel() != t * k or y.shape[1] != h:
        raise ValueError("slots must have T*k entries and y rows the width of shared")
    out = torch.empty((t, h), dtype=torch.bfloat16, device=y.device)
    if t == 0:
        return out
    yc = y.contiguous()
    sc = slots.contiguous()
    s = _rows_16b(shared)
    w = weights if weights.stride(1) == 1 else weights.contiguous()
    _on(yc.device)("kb_ep_combine", _p(yc), _p(sc), c_int64(t), c_int64(k), c_int64(h), _p(w),
              c_int64(w.stride(0)), _p(s), c_int64(s.stride(0)), _p(out), c_int64(out.stride(0)),
              _stream(yc.device))
    return out


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------


def moe_router(
    hidden_states: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    top_k: int,
    *,
    renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
    append_expert: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Sigmoid top-k routing of KLinearRouter.forward (router.py:47-85).

    Returns (indices int64 [T, top_k], weights fp32 [T, top_k]), ordered by
    (biased score desc, expert index asc).  With ``append_expert`` the indices
    are [T, top_k + 1] with that expert id as the last route, the
    shape-stable layout of engine/klinear/moe.py:23-36.
    """
    if hidden_states.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("router hidden states and weight must be BF16")
    if weight.ndim != 2:
        raise ValueError("router weight must have shape [experts, hidden]")
    _require_cuda(hidden_states, "B200 router")
    flat = hidden_states.reshape(-1, hidden_states.shape[-1])
    tokens, hidden = flat.shape
    experts = weight.shape[0]
    if weight.shape[1] != hidden:
        raise ValueError("router weight width does not match the hidden size")
    if not 0 < top_k <= experts:
        raise ValueError("top_k must be in the expert range")
    extra = 0 if append_expert is None else 1
    idx = torch.empty((tokens, top_k + extra), dtype=torch.long, device=flat.device)
    wts = torch.empty((tokens, top_k), dtype=torch.float32, device=flat.device)
    if tokens == 0:
        return idx, wts
    x = _rows_16b(flat)
    w = _dense_contig(weight)
    b = None
    if bias is not None:
        b = bias.detach()
        if b.dtype != torch.float32 or b.device != flat.device or not b.is_contiguous():
            b = b.to(device=flat.device, dtype=torch.float32).contiguous()
    lib = _lib.lib()
    need = int(lib.kb_router_workspace_size(tokens, experts))
    ws = _workspace("router", flat.device, need, (tokens, experts))
    _on(flat.device)(
        "kb_router_topk",
        _p(x), c_int64(x.stride(0)), c_int64(tokens), c_int64(hidden), _p(w), _p(b),
        c_int64(experts), c_int64(top_k), 1 if renormalize else 0,
        c_float(float(routed_scaling_factor)), _p(idx),
        c_int64(-1 if append_expert is None else int(append_expert)), _p(wts), _p(ws),
        c_size_t(ws.numel()), _stream(flat.device),
    )
    return idx, wts


# ---------------------------------------------------------------------------
# KDA
# ---------------------------------------------------------------------------


def kda_decode_step(
    state: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    decay: torch.Tensor,
    beta: torch.Tensor,
    *,
    scale: float,
    out_bf16: torch.Tensor | None = None,
) -> torch.Tensor:
    """One KDA recurrent step; mutates ``state`` in place, returns fp32 [B,H,Dv]."""
    if state.ndim != 4:
        raise ValueError("state must have shape [batch, heads, d_k, d_v]")
    if any(t.dtype != torch.float32 for t in (state, q, k, v, decay, beta)):
        raise TypeError("KDA decode inputs must all use torch.float32")
    if not all(t.device == state.device for t in (q, k, v, decay, beta)):
        raise ValueError("KDA decode inputs must share one device")
    batch, heads, d_k, d_v = state.shape
    if batch == 0 or heads == 0 or d_k == 0 or d_v == 0:
        raise ValueError("KDA decode dimensions must be nonzero")
    if q.shape != (batch, heads, d_k):
        raise ValueError("q must have shape [batch, heads, d_k]")
    if k.shape != (batch, heads, d_k):
        raise ValueError("k must have shape [batch, heads, d_k]")
    if v.shape != (batch, heads, d_v):
        raise ValueError("v must have shape [batch, heads, d_v]")
    if decay.shape != (batch, heads, d_k):
        raise ValueError("decay must have shape [batch, heads, d_k]")
    if beta.shape != (batch, heads):
        raise ValueError("beta must have shape [batch, heads]")
    if state.device.type != "cuda":
        raise ValueError("fused KDA decode requires CUDA inputs")
    out = torch.empty((batch, heads, d_v), dtype=torch.float32, device=state.device)
    if out_bf16 is not None:
        if out_bf16.dtype != torch.bfloat16 or out_bf16.numel() != out.numel() or not (
            out_bf16.is_contiguous()
        ):
            raise ValueError("out_bf16 must be a contiguous BF16 tensor with B*H*Dv elements")
    work = state
    if state.stride(3) != 1 or state.stride(2) < d_v:
        work = state.contiguous()
    qc, kc, vc = q.contiguous(), k.contiguous(), v.contiguous()
    dc, bc = decay.contiguous(), beta.contiguous()
    _on(state.device)(
        "kb_kda_decode_step",
        _p(work), c_int64(work.stride(0)), c_int64(work.stride(1)), c_int64(work.stride(2)),
        _p(qc), _p(kc), _p(vc), _p(dc), _p(bc), c_int64(batch), c_int64(heads), c_int64(d_k),
        c_int64(d_v), c_float(float(scale)), _p(out), _p(out_bf16), _stream(state.device),
    )
    if work is not state:
        state.copy_(work)
    return out


# ---------------------------------------------------------------------------
# codec
# ---------------------------------------------------------------------------


def kda_prepare(q_in: torch.Tensor, k_in: torch.Tensor, v_in: torch.Tensor,
                q_state: torch.Tensor, k_state: torch.Tensor, v_state: torch.Tensor,
                q_weight: torch.Tensor, k_weight: torch.Tensor, v_weight: torch.Tensor,
                raw_decay: torch.Tensor, dt_bias: torch.Tensor, a_log: torch.Tensor,
                raw_beta: torch.Tensor, *, num_heads: int, head_dim: int, eps: float = 1e-6):
    """KDA decode preparation (attention.py:192-230) in one launch: the three
    width-4 short convolutions (states [B, C, 4] updated in place), then the
    gates.  Returns fp32 (q, k, v, decay) [B, H, D] and beta [B, H]: the
    inputs of ``kda_decode_step``.  Projections, states, weights, raw_decay and
    raw_beta are bf16; dt_bias and a_log fp32 (a_log [H] or [1, 1, H, 1])."""
    batch = q_in.shape[0]
    x, weights, rd, rb, a, dt = _kda_prep_args(
        q_in, k_in, v_in, q_state, k_state, v_state, q_weight, k_weight, v_weight, raw_decay,
        dt_bias, a_log, raw_beta, num_heads, head_dim)
    outs = [torch.empty((batch, num_heads, head_dim), dtype=torch.float32, device=q_in.device)
            for _ in range(4)]
    beta = torch.empty((batch, num_heads), dtype=torch.float32, device=q_in.device)
    if batch == 0:
        return (*outs, beta)
    _on(q_in.device)("kb_kda_prepare", _p(x[0]), _p(x[1]), _p(x[2]), c_int64(x[0].stride(0)),
              _p(q_state), _p(k_state), _p(v_state), _p(weights[0]), _p(weights[1]),
              _p(weights[2]), _p(rd), c_int64(rd.stride(0)), _p(dt), _p(a), _p(rb),
              c_int64(rb.stride(0)), c_int64(batch), c_int64(num_heads), c_int64(head_dim),
              c_float(eps), _p(outs[0]), _p(outs[1]), _p(outs[2]), _p(outs[3]), _p(beta),
              _stream(q_in.device))
    return (*outs, beta)


def _kda_prep_args(q_in, k_in, v_in, q_state, k_state, v_state, q_weight, k_weight, v_weight,
                   raw_decay, dt_bias, a_log, raw_beta, num_heads, head_dim):
    """Validated, flattened preparation inputs: (q/k/v rows [B, C] sharing one
    row stride, weights [C, 4], raw_decay [B, C], raw_beta [B, H], a_log [H],
    dt_bias [C])."""
    batch = q_in.shape[0]
    c = num_heads * head_dim
    bf = (q_in, k_in, v_in, q_state, k_state, v_state, q_weight, k_weight, v_weight, raw_decay,
          raw_beta)
    if any(t.dtype != torch.bfloat16 for t in bf):
        raise TypeError("KDA prepare projections, states, weights and gate inputs must be BF16")
    if dt_bias.dtype != torch.float32 or a_log.dtype != torch.float32:
        raise TypeError("dt_bias and A_log must be FP32")
    _require_cuda(q_in, "KDA prepare")
    if any(t.device != q_in.device for t in bf + (dt_bias, a_log)):
        raise ValueError("KDA prepare tensors must share one device")
    x = [t.reshape(batch, c) for t in (q_in, k_in, v_in)]
    if any(t.stride(1) != 1 or t.stride(0) != x[0].stride(0) for t in x):
        x = [t.contiguous() for t in x]
    states = (q_state, k_state, v_state)
    if any(tuple(st.shape) != (batch, c, 4) or not st.is_contiguous() for st in states):
        raise ValueError("each short convolution state must be a contiguous [batch, channels, 4]")
    weights = [w.reshape(c, 4).contiguous() for w in (q_weight, k_weight, v_weight)]
    rd = raw_decay.reshape(batch, c).contiguous()
    rb = raw_beta.reshape(batch, num_heads).contiguous()
    a = a_log.reshape(num_heads).contiguous()
    dt = dt_bias.reshape(c).contiguous()
    return x, weights, rd, rb, a, dt


def kda_prepare_step_supported(state: torch.Tensor, head_dim: int) -> bool:
    """Whether ``kda_prepare_step`` takes this state: head_dim 128, fp32 CUDA
    state [B, H, 128, 128] with contiguous 16-byte aligned rows."""
    return (head_dim == 128 and state.is_cuda and state.dtype == torch.float32
            and state.ndim == 4 and state.shape[2] == 128 and state.shape[3] == 128
            and state.stride(3) == 1 and state.stride(2) == 128 and state.stride(1) % 4 == 0
            and state.stride(0) % 4 == 0 and state.data_ptr() % 16 == 0)


def kda_prepare_step(state: torch.Tensor, q_in: torch.Tensor, k_in: torch.Tensor,
                     v_in: torch.Tensor, q_state: torch.Tensor, k_state: torch.Tensor,
                     v_state: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                     v_weight: torch.Tensor, raw_decay: torch.Tensor, dt_bias: torch.Tensor,
                     a_log: torch.Tensor, raw_beta: torch.Tensor, *, num_heads: int,
                     head_dim: int, scale: float, eps: float = 1e-6,
                     out_bf16: torch.Tensor | None = None) -> torch.Tensor:
    """``kda_prepare`` then ``kda_decode_step`` in one launch (same results):
    the convolution states and the KDA state are updated in place; returns
    the fp32 output [B, H, D] (and fills ``out_bf16`` if given)."""
    if not kda_prepare_step_supported(state, head_dim):
        raise ValueError("kda_prepare_step needs head_dim 128 and a state with contiguous rows")
    batch = q_in.shape[0]
    if tuple(state.shape[:2]) != (batch, num_heads):
        raise ValueError("state must have shape [batch, heads, 128, 128]")
    x, weights, rd, rb, a, dt = _kda_prep_args(
        q_in, k_in, v_in, q_state, k_state, v_state, q_weight, k_weight, v_weight, raw_decay,
        dt_bias, a_log, raw_beta, num_heads, head_dim)
    if state.device != q_in.device:
        raise ValueError("the KDA state must be on the device of the inputs")
    out = torch.empty((batch, num_heads, head_dim), dtype=torch.float32, device=q_in.device)
    if out_bf16 is not None and (out_bf16.dtype != torch.bfloat16 or
                                 out_bf16.numel() != out.numel() or
                                 not out_bf16.is_contiguous()):
        raise ValueError("out_bf16 must be a contiguous BF16 tensor with B*H*D elements")
    if batch == 0:
        return out
    _on(q_in.device)("kb_kda_prepare_step", _p(x[0]), _p(x[1]), _p(x[2]),
            c_int64(x[0].stride(0)),
              _p(q_state), _p(k_state), _p(v_state), _p(weights[0]), _p(weights[1]),
              _p(weights[2]), _p(rd), c_int64(rd.stride(0)), _p(dt), _p(a), _p(rb),
              c_int64(rb.stride(0)), c_float(eps), _p(state), c_int64(state.stride(0)),
              c_int64(state.stride(1)), c_int64(state.stride(2)), c_int64(batch),
              c_int64(num_heads), c_int64(head_dim), c_float(float(scale)), _p(out),
              _p(out_bf16), _stream(q_in.device))
    return out


def quantise(weight: torch.Tensor, group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """On-device quantise of a bf16 [N,K] matrix -> (packed uint8 [N,K/2], bf16 scales).

    Same arithmetic as engine/quant/w4a16.py:68-105 with the group size as a
    parameter.  Raises ValueError for non-finite weights (this check reads a
    flag back, so it synchronizes the stream).
    """
    if weight.ndim != 2:
        raise ValueError("weight must have shape [out_features, in_features]")
    if weight.dtype != torch.bfloat16:
        raise TypeError("weight must have dtype torch.bfloat16")
    _require_cuda(weight, "on-device quantise")
    n, k = weight.shape
    if k % group_size:
        raise ValueError(f"the reduction axis must be divisible by group size {group_size}")
    w = _rows_16b(weight)
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((n, k // group_size), dtype=torch.bfloat16, device=weight.device)
    flag = torch.zeros((1,), dtype=torch.int32, device=weight.device)
    _on(weight.device)(
        "kb_w4a16_quantise",
        _p(w), c_int64(w.stride(0)), c_int64(n), c_int64(k), c_int64(group_size), _p(packed),
        _p(scales), _p(flag), _stream(weight.device),
    )
    if int(flag.item()):
        raise ValueError("weight must contain only finite values")
    return packed, scales


# ---------------------------------------------------------------------------
# speculative serving over a paged cache
# ---------------------------------------------------------------------------

_ELEMENT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HALF = (torch.bfloat16, torch.float16)
_STRIDES = c_int64 * 3
MAX_TREE_TOKENS = 64


class PagedPlan(NamedTuple):
    """What ``paged_plan`` returns (all on the device)."""

    cu_tokens: torch.Tensor         # int32 [B + 1], running sums of the new lengths
    slots: torch.Tensor             # int64 [num_tokens], -1 where a token has no slot
    positions: torch.Tensor         # int32 [num_tokens]
    tree_mask: torch.Tensor | None  # int64 [num_tokens], with parents
    free_head: torch.Tensor         # int32 [1], the next call's free_head
    missing: torch.Tensor           # int32 [1], pages needed and not given


class Verification(NamedTuple):
    """What ``verify_drafts`` returns (all on the device)."""

    tokens: torch.Tensor    # int64 [B, max_tokens]: accepted tokens, the next token, then -1
    path: torch.Tensor      # int32 [B, max_tokens]: 0 and the accepted tree indices, then -1
    accepted: torch.Tensor  # int32 [B]


def _vector(t: torch.Tensor, dtype: torch.dtype, what: str, device: torch.device,
            length: int | None = None) -> torch.Tensor:
    """A 1-D contiguous tensor of a type, length and device."""
    if (t.dtype == dtype and t.dim() == 1 and t.device == device and t.is_contiguous()
            and (length is None or t.numel() == length)):
        return t
    if t.dtype != dtype or t.dim() != 1:
        raise TypeError(f"{what} must be a one-dimensional {dtype} tensor")
    if length is not None and t.numel() != length:
        raise ValueError(f"{what} must have {length} entries")
    if t.device != device:
        raise ValueError(f"{what} must be on the device of the other tensors")
    return t if t.is_contiguous() else t.contiguous()


def _raw_stream(device: torch.device) -> int:
    """The current stream's handle, without a torch.cuda.Stream object around it (a
    microsecond or two that these calls, short beside their launch, would notice)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


# Bytes at the start of tree_attention's workspace that have to be zero (kimi_b200.h).
_TREE_COUNTERS = 4096


class _ThreadScratch(threading.local):
    def __init__(self) -> None:
        self.held: dict[tuple, torch.Tensor] = {}


_THREAD_SCRATCH = _ThreadScratch()


def _verify_scratch(device: torch.device, stream: int, requests: int, rows: int) -> torch.Tensor:
    """Scratch of verify_drafts, with anything in it.

    Its calls are two launches, and another thread's may come between them on the
    stream, so each thread keeps its own, for sizes up to the next power of two; calls
    of one thread follow each other on a stream.  A call in a graph gets its own from
    the graph's memory, since graphs may be replayed on other streams.
    """
    most = (requests - 1).bit_length(), max(rows - 1, 0).bit_length()
    key = (device.index, stream, *most)
    ws = None if _capturing() else _THREAD_SCRATCH.held.get(key)
    if ws is None:
        nbytes = _lib.lib().kb_verify_drafts_workspace_size(1 << most[0], 1 << most[1])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        if not _capturing():
            _THREAD_SCRATCH.held[key] = ws
    return ws


def paged_plan(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    free_head: torch.Tensor,
    page_size: int,
    num_tokens: int,
    *,
    parents: torch.Tensor | None = None,
    reserved_lens: torch.Tensor | None = None,
) -> PagedPlan:
    """Pages, slots and positions for every request's new tokens.

    Request b has ``context_lens[b]`` cached tokens and gets ``new_lens[b]``
    more.  The pages it lacks are taken from ``free_pages`` (from
    ``free_head`` on, in request order) and written to its row of
    ``block_table`` in place.  ``num_tokens`` is the length of the per-token
    outputs: the sum of ``new_lens``, or more (the rest gets slot -1).  With
    ``parents`` (int32 [num_tokens], the tree parent's index in the request,
    -1 for the root) positions count the depth and ``tree_mask`` holds each
    token's ancestors for ``tree_attention``.  ``reserved_lens`` (int32, at
    least the context) says how many tokens a request's pages already reach,
    where refused drafted tokens left it pages beyond its context.
    """
    device = context_lens.device
    if block_table.dtype != torch.int32 or block_table.ndim != 2:
        raise TypeError("block_table must be an int32 [requests, pages] matrix")
    _require_cuda(context_lens, "paged plan")
    requests, width = block_table.shape
    ctx = _vector(context_lens, torch.int32, "context_lens", device, requests)
    new = _vector(new_lens, torch.int32, "new_lens", device, requests)
    free = _vector(free_pages, torch.int32, "free_pages", device)
    head = _vector(free_head, torch.int32, "free_head", device, 1)
    held = None
    if reserved_lens is not None:
        held = _vector(reserved_lens, torch.int32, "reserved_lens", device, requests)
    if block_table.device != device:
        raise ValueError("block_table must be on the device of the other tensors")
    if requests == 0 or width == 0:
        raise ValueError("paged plan requires at least one request and one table column")
    if block_table.stride(1) != 1 or (requests > 1 and block_table.stride(0) < width):
        raise ValueError("block_table is updated in place and needs rows of unit stride")
    if page_size <= 0 or num_tokens < 0:
        raise ValueError("page_size must be positive and num_tokens not negative")
    # The outputs are parts of two buffers: six allocations would take longer
    # than the kernel.
    ints = torch.empty(requests + num_tokens + 3, dtype=torch.int32, device=device)
    head_out, missing, cu, positions = ints.split_with_sizes((1, 1, requests + 1, num_tokens))
    par = mask = None
    if parents is None:
        slots = torch.empty(num_tokens, dtype=torch.long, device=device)
    else:
        par = _vector(parents, torch.int32, "parents", device, num_tokens)
        slots, mask = torch.empty(2, num_tokens, dtype=torch.long, device=device).unbind()
    _on(device)(
        "kb_paged_plan",
        ctx.data_ptr(), None if held is None else held.data_ptr(),
        new.data_ptr(), requests, block_table.data_ptr(),
        max(block_table.stride(0), width), width, free.data_ptr(), free.shape[0],
        head.data_ptr(), page_size, num_tokens, None if par is None else par.data_ptr(),
        cu.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        None if mask is None else mask.data_ptr(), head_out.data_ptr(), missing.data_ptr(),
        _raw_stream(device),
    )
    return PagedPlan(cu, slots, positions, mask, head_out, missing)


def paged_reserve(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    reserved_lens: torch.Tensor,
    page_size: int,
) -> None:
    """What each request's pages reach after a ``paged_plan`` of the same arguments.

    ``reserved_lens`` (int32 [requests], the plan's) is updated in place: at least
    what it was and the context, and ``context_lens + new_lens`` as far as the plan
    gave pages, so that the next plan asks again for those that were missing.
    """
    device = context_lens.device
    if block_table.dtype != torch.int32 or block_table.ndim != 2:
        raise TypeError("block_table must be an int32 [requests, pages] matrix")
    _require_cuda(context_lens, "paged reserve")
    requests, width = block_table.shape
    ctx = _vector(context_lens, torch.int32, "context_lens", device, requests)
    new = _vector(new_lens, torch.int32, "new_lens", device, requests)
    held = _vector(reserved_lens, torch.int32, "reserved_lens", device, requests)
    if block_table.device != device:
        raise ValueError("block_table must be on the device of the other tensors")
    if requests == 0 or width == 0 or page_size <= 0:
        raise ValueError("paged reserve requires a request, a table column and a page size")
    if held is not reserved_lens:
        raise ValueError("reserved_lens is updated in place and needs unit stride")
    if block_table.stride(1) != 1 or (requests > 1 and block_table.stride(0) < width):
        raise ValueError("block_table needs rows of unit stride")
    _on(device)(
        "kb_paged_reserve",
        ctx.data_ptr(), new.data_ptr(), requests, block_table.data_ptr(),
        max(block_table.stride(0), width), width, page_size, held.data_ptr(),
        _raw_stream(device),
    )


def _rows_of_heads(t: torch.Tensor, what: str, expanded: bool = False) -> torch.Tensor:
    """[tokens, heads, width] with unit inner stride, 16-byte aligned rows and, unless
    ``expanded`` ones will do, positive strides (tensor copies take no other)."""
    if t.ndim != 3:
        raise ValueError(f"{what} must have shape [tokens, heads, width]")
    s = t.stride()
    if (s[2] != 1 or (s[0] | s[1]) & 7 or not (s[0] and s[1] or expanded)
            or t.data_ptr() & 15):
        t = t.contiguous()
    return t


def _cache_strides(t: torch.Tensor, what: str) -> object:
    """The page, row and head strides of a cache that kernels use in place."""
    if t.ndim != 4:
        raise ValueError(f"{what} must have shape [pages, page_size, heads, width]")
    s = t.stride()
    if (s[3] != 1 or (s[0] | s[1] | s[2]) & 7 or t.data_ptr() & 15) and t.numel():
        raise ValueError(f"{what} needs unit stride along the width, other strides multiples "
                         "of 8 and a 16-byte aligned start")
    if not (s[0] and s[1] and s[2]) and any(n > 1 and not x for n, x in zip(t.shape, s)):
        raise ValueError(f"{what} needs positive strides: rows of its own for every page, "
                         "place and head")
    return _STRIDES(s[0], s[1], s[2])


def _check_widths(dk: int, dv: int) -> None:
    if not (0 < dk <= 192 and dk % 8 == 0 and 0 < dv <= 128 and dv % 8 == 0):
        raise ValueError("head widths must be multiples of 8, keys up to 192 and values up to 128")


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
) -> None:
    """Store each token's keys and values in its slot of the paged caches.

    ``k`` [tokens, heads, Dk] and ``v`` [tokens, heads, Dv] go to
    ``k_cache`` / ``v_cache`` [pages, page_size, heads, width] (any strides),
    at page ``slot // page_size``, row ``slot % page_size``; a negative slot
    is skipped.  No two tokens may name one slot.
    """
    dtype = k.dtype
    if dtype not in _HALF:
        raise TypeError("keys and values must be BF16 or FP16")
    if not (dtype == v.dtype == k_cache.dtype == v_cache.dtype):
        raise TypeError("keys, values and caches must share one type")
    _require_cuda(k, "paged append")
    device = k.device
    if not (v.device == k_cache.device == v_cache.device == device):
        raise ValueError("paged append inputs must share one device")
    ks, vs = _cache_strides(k_cache, "k_cache"), _cache_strides(v_cache, "v_cache")
    kr, vr = _rows_of_heads(k, "k", expanded=True), _rows_of_heads(v, "v", expanded=True)
    n, heads, dk = k.shape
    v_tokens, v_heads, dv = v.shape
    if v_tokens != n or v_heads != heads:
        raise ValueError("k and v must have the same tokens and heads")
    pages, page_size, k_cache_heads, k_cache_width = k_cache.shape
    v_pages, v_page_size, v_cache_heads, v_cache_width = v_cache.shape
    if not (k_cache_heads == v_cache_heads == heads
            and k_cache_width == dk and v_cache_width == dv):
        raise ValueError("the caches' heads and widths must match k and v")
    if pages != v_pages or page_size != v_page_size:
        raise ValueError("the caches must have the same pages")
    _check_widths(dk, dv)
    sl = _vector(slots, torch.long, "slots", device, n)
    if n == 0 or heads == 0:
        return
    _on(device)(
        "kb_paged_append",
        kr.data_ptr(), kr.stride(0), kr.stride(1), vr.data_ptr(),
        vr.stride(0), vr.stride(1), n, heads, dk, dv, k_cache.data_ptr(), ks,
        v_cache.data_ptr(), vs, pages, page_size, sl.data_ptr(),
        _raw_stream(device),
    )


def _attention_heads(q: torch.Tensor, heads: int, dk: int, dv: int) -> None:
    if q.shape[1] == 0 or heads == 0 or q.shape[1] % heads:
        raise ValueError("query heads must be a multiple of key/value heads")
    if q.shape[2] != dk:
        raise ValueError("queries and keys must have one width")
    _check_widths(dk, dv)


def _scale_of(scale: float | None, dk: int) -> float:
    if scale is None:
        return dk ** -0.5
    if not scale > 0:
        raise ValueError("the scale must be positive")
    return float(scale)


def _no_requests(q: torch.Tensor, dv: int, return_lse: bool):
    """What rows outside every request get, where there is no request."""
    total, hq, _ = q.shape
    out = q.new_zeros(total, hq, dv)
    if not return_lse:
        return out
    return out, torch.full((total, hq), float("-inf"), device=q.device)


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_seqlen: int,
    *,
    cu_seqlens_k: torch.Tensor | None = None,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention over packed prompts, grouped heads.

    ``q`` [tokens, Hq, Dk], ``k`` [keys, Hkv, Dk], ``v`` [keys, Hkv, Dv], bf16
    or f16; request b has the queries ``cu_seqlens[b]:cu_seqlens[b+1]`` (int32)
    and the keys of ``cu_seqlens_k`` (default: the same).  Query i sees keys up
    to ``i + keys - queries``.  No request has more than ``max_seqlen``
    queries.  Returns [tokens, Hq, Dv] and, with ``return_lse``, the fp32
    log-sum-exp [tokens, Hq]; a query without keys gives 0 and -infinity.
    """
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("queries, keys and values must be BF16 or FP16")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("queries, keys and values must share one type")
    _require_cuda(q, "prompt attention")
    device = q.device
    if not (k.device == v.device == device):
        raise ValueError("prompt attention inputs must share one device")
    qr, kr, vr = _rows_of_heads(q, "q"), _rows_of_heads(k, "k"), _rows_of_heads(v, "v")
    total, hq, dk = q.shape
    keys, hkv, dv = v.shape
    if k.shape != (keys, hkv, dk):
        raise ValueError("k must have the tokens and heads of v and the width of q")
    _attention_heads(q, hkv, dk, dv)
    if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must have one entry more than there are requests")
    requests = cu_seqlens.shape[0] - 1
    cq = _vector(cu_seqlens, torch.int32, "cu_seqlens", device)
    if cu_seqlens_k is None:
        if keys != total:
            raise ValueError("cu_seqlens_k is needed where keys and queries differ in number")
        ck = cq
    else:
        ck = _vector(cu_seqlens_k, torch.int32, "cu_seqlens_k", device, requests + 1)
    if max_seqlen < 0 or (total and not max_seqlen):
        raise ValueError("max_seqlen must not be negative, nor 0 with tokens")
    scale = _scale_of(scale, dk)
    if requests == 0:
        return _no_requests(q, dv, return_lse)
    out = torch.empty(total, hq, dv, dtype=q.dtype, device=device)
    lse = torch.empty(total, hq, dtype=torch.float32, device=device) if return_lse else None
    _on(device)(
        "kb_prompt_attention",
        qr.data_ptr(), qr.stride(0), qr.stride(1), kr.data_ptr(),
        kr.stride(0), kr.stride(1), vr.data_ptr(), vr.stride(0), vr.stride(1),
        _ELEMENT[q.dtype], cq.data_ptr(), ck.data_ptr(), requests, total, keys, max_seqlen, hq,
        hkv, dk, dv, scale, out.data_ptr(),
        None if lse is None else lse.data_ptr(), _raw_stream(device),
    )
    return out if lse is None else (out, lse)


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_tokens: torch.Tensor,
    max_tokens: int,
    *,
    tree_mask: torch.Tensor | None = None,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of this step's tokens (one each, or drafted trees) over the paged cache.

    Request b's tokens are ``q[cu_tokens[b]:cu_tokens[b+1]]`` (at most
    ``max_tokens``); their keys and values already are in the caches
    [pages, page_size, Hkv, width], after its ``context_lens[b]`` cached ones,
    in the pages of ``block_table[b]``.  A token sees the context and, of its
    step, the tokens whose bits its ``tree_mask`` word (int64, at most 64
    tokens) has; without masks itself and those before it.  Outputs as
    ``prompt_attention``.
    """
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("queries and caches must be BF16 or FP16")
    if not (q.dtype == k_cache.dtype == v_cache.dtype):
        raise TypeError("queries and caches must share one type")
    if block_table.dtype != torch.int32 or block_table.ndim != 2:
        raise TypeError("block_table must be an int32 [requests, pages] matrix")
    _require_cuda(q, "tree attention")
    device = q.device
    if not (k_cache.device == v_cache.device == block_table.device == device):
        raise ValueError("tree attention inputs must share one device")
    ks, vs = _cache_strides(k_cache, "k_cache"), _cache_strides(v_cache, "v_cache")
    qr = _rows_of_heads(q, "q")
    total, hq, dk = q.shape
    pages, page_size, hkv, dv = v_cache.shape
    if k_cache.shape != (pages, page_size, hkv, dk):
        raise ValueError("k_cache must have the pages and heads of v_cache and the width of q")
    _attention_heads(q, hkv, dk, dv)
    if page_size < 8 or page_size > 4096 or page_size & (page_size - 1):
        raise ValueError("the page size must be a power of two from 8 to 4096")
    requests, width = block_table.shape
    table = block_table
    if width and (table.stride(1) != 1 or (requests > 1 and table.stride(0) < width)):
        table = table.contiguous()
    ctx = _vector(context_lens, torch.int32, "context_lens", device, requests)
    cu = _vector(cu_tokens, torch.int32, "cu_tokens", device, requests + 1)
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    if total and (max_tokens == 0 or pages == 0):
        raise ValueError("tokens need max_tokens of at least 1 and a cache with pages")
    mask = None
    if tree_mask is not None:
        if max_tokens > MAX_TREE_TOKENS:
            raise ValueError(f"a masked tree has at most {MAX_TREE_TOKENS} tokens")
        mask = _vector(tree_mask, torch.long, "tree_mask", device, total)
    scale = _scale_of(scale, dk)
    if requests == 0:
        return _no_requests(q, dv, return_lse)
    out = torch.empty(total, hq, dv, dtype=q.dtype, device=device)
    lse = torch.empty(total, hq, dtype=torch.float32, device=device) if return_lse else None
    if total == 0:
        return out if lse is None else (out, lse)
    stream = _raw_stream(device)
    # Calls of one size share one layout.
    nbytes = _lib.lib().kb_tree_attention_workspace_size(hq // hkv, max_tokens)
    ws = _kept_scratch(("tree_attention", device.index, stream, nbytes), device, stream, nbytes,
                       _TREE_COUNTERS)
    _on(device)(
        "kb_tree_attention",
        qr.data_ptr(), qr.stride(0), qr.stride(1), k_cache.data_ptr(), ks,
        v_cache.data_ptr(), vs, _ELEMENT[q.dtype], pages, page_size, table.data_ptr(),
        max(table.stride(0), width), width, ctx.data_ptr(), cu.data_ptr(),
        None if mask is None else mask.data_ptr(), requests, total, max_tokens, hq, hkv, dk, dv,
        scale, out.data_ptr(),
        None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), stream,
    )
    return out if lse is None else (out, lse)


def verify_drafts(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    cu_tokens: torch.Tensor,
    max_tokens: int,
    accept_u: torch.Tensor,
    noise: torch.Tensor,
    temperature: torch.Tensor,
    *,
    parents: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
) -> Verification:
    """Accept drafted tokens against the target's logits, and draw the next token.

    ``logits`` [rows, V] (bf16, f16 or f32): row ``cu_tokens[b] + t`` is the
    prediction after token t of request b, whose token 0 is the root;
    ``tokens`` int64 [rows].  ``parents`` int32 [rows] gives a tree (default:
    chains).  ``accept_u`` fp32 [rows] in [0, 1) decides each drafted token,
    ``noise`` fp32 [B, V] (exponential, positive) the token after the last
    accepted one, ``temperature`` fp32 [B] (0: greedy).  ``draft_probs`` fp32
    [rows, V] are the distributions the tokens of chains were drawn from;
    without them drafted tokens count as given.  The outputs follow the
    target's distribution exactly (speculative sampling).
    """
    if logits.ndim != 2 or logits.dtype not in _ELEMENT:
        raise TypeError("logits must be a BF16, FP16 or FP32 [rows, vocabulary] matrix")
    _require_cuda(logits, "draft verification")
    device = logits.device
    rows, vocab = logits.shape
    requests = temperature.shape[0] if temperature.ndim == 1 else -1
    temps = _vector(temperature, torch.float32, "temperature", device)
    cu = _vector(cu_tokens, torch.int32, "cu_tokens", device, requests + 1)
    tok = _vector(tokens, torch.long, "tokens", device, rows)
    coin = _vector(accept_u, torch.float32, "accept_u", device, rows)
    if vocab == 0:
        raise ValueError("draft verification requires a vocabulary")
    if not 0 < max_tokens <= MAX_TREE_TOKENS:
        raise ValueError(f"max_tokens must be from 1 to {MAX_TREE_TOKENS}")
    if noise.dtype != torch.float32 or noise.ndim != 2:
        raise TypeError("noise must be an FP32 [requests, vocabulary] matrix")
    if noise.shape != (requests, vocab) or noise.device != device:
        raise ValueError("noise must have a row for each request, on the logits' device")
    par, probs, probs_stride = None, None, vocab
    if parents is not None:
        par = _vector(parents, torch.int32, "parents", device, rows)
    if draft_probs is not None:
        if parents is not None:
            raise ValueError("draft_probs go with chains of drafted tokens, not with parents")
        if draft_probs.dtype != torch.float32 or draft_probs.ndim != 2:
            raise TypeError("draft_probs must be an FP32 [rows, vocabulary] matrix")
        if draft_probs.shape != (rows, vocab) or draft_probs.device != device:
            raise ValueError("draft_probs must have the shape and device of the logits")
        probs, probs_stride = _unit_rows(draft_probs, vocab)
    out = torch.empty(requests, max_tokens, dtype=torch.long, device=device)
    path = torch.empty(requests, max_tokens, dtype=torch.int32, device=device)
    accepted = torch.empty(requests, dtype=torch.int32, device=device)
    if requests == 0:
        return Verification(out, path, accepted)
    (x, x_stride), (e, e_stride) = _unit_rows(logits, vocab), _unit_rows(noise, vocab)
    stream = _raw_stream(device)
    ws = _verify_scratch(device, stream, requests, rows)
    _on(device)(
        "kb_verify_drafts",
        x.data_ptr(), x_stride, rows, vocab,
        _ELEMENT[x.dtype], tok.data_ptr(), None if par is None else par.data_ptr(),
        cu.data_ptr(), requests, max_tokens, coin.data_ptr(), e.data_ptr(),
        e_stride, temps.data_ptr(), None if probs is None else probs.data_ptr(),
        probs_stride, out.data_ptr(),
        path.data_ptr(), accepted.data_ptr(), ws.data_ptr(), ws.numel(), stream,
    )
    return Verification(out, path, accepted)


def _unit_rows(t: torch.Tensor, width: int) -> tuple[torch.Tensor, int]:
    """A matrix whose rows have unit stride and do not overlap, and their stride."""
    row, column = t.stride()
    if column != 1 or (row < width and t.shape[0] > 1):
        t, row = t.contiguous(), width
    return t, max(row, width)
