"""Operators of the detection head: the dense layers between ``RoIPooling`` and ``Decoder`` and what trains with them.

The reference's head is ``Flatten -> Dense(4096, relu) -> Dropout -> Dense(4096, relu) -> Dropout -> Dense(L), Dense(4 L)``
(``models/faster_rcnn.py:320-326``).  Here: the dense product in 8-bit floating point with a scale per block of 128 and the
quantiser of its operands (serving), group normalisation of channels-last tensors with an activation, and dropout whose mask
is never stored (training, with gradients).  Every call enqueues on the current stream of its tensors' device, allocates its
outputs and scratch from torch's allocator (so a captured graph owns them) and never synchronises.
"""

from __future__ import annotations

from typing import Any, List, Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib

BLOCK = 128

_E4M3 = torch.float8_e4m3fn
_E4M3_ONLY = (_E4M3,)
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_SCALE_TYPES = {torch.float32: 0, torch.float8_e8m0fnu: 1}
_ACTIVATIONS = {None: 0, "linear": 0, "relu": 1, "swish": 2}


def _operand(x: Any, name: str, types: Any = _TYPES, device: Optional[torch.device] = None) -> torch.Tensor:
    """``x`` as a device tensor (DLPack objects are imported zero-copy) of one of ``types``; its strides stay."""
    if type(x) is torch.Tensor and x.is_cuda and x.dtype in types and (device is None or x.device == device):
        return x
    if not isinstance(x, torch.Tensor):
        x = torch.from_dlpack(x) if hasattr(x, "__dlpack__") else torch.as_tensor(x)
    if x.dtype not in types:
        raise ValueError(f"{name} must be one of {[str(t) for t in types]}, got {x.dtype}")
    if device is None:
        device = x.device if x.is_cuda else _lib.require_gpu()
    return x if x.device == device else x.to(device)


def _activation(activation: Optional[str], known: Tuple[Optional[str], ...]) -> int:
    if activation not in known:
        raise ValueError(f"activation must be one of {known}, got {activation!r}")
    return _ACTIVATIONS[activation]


def _no_tangent(what: str, *tensors: Any) -> None:
    """Refuse what the kernels would pass by: forward-mode derivatives, and a trace, which records the allocations only."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative")
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{what} cannot be traced: a trace does not see the kernels")


def _no_gradient(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no gradient: detach its inputs or call it under torch.no_grad()")


def _leaves_of(*tensors: Any) -> List[Any]:
    """Refuse a capture that the backward pass would end the process in.

    autograd runs a leaf's accumulation node on the stream on which the node was made, and the node lives as long as any
    graph of the leaf.  If an eager graph still holds it, a captured backward pass makes the capture wait for that other
    stream, which the runtime does not survive.  The node keeps a note of the stream on which it was first met here; one that
    others hold and that bears no note may be an eager graph's, and is refused in a capture too.

    Returns the nodes: the caller keeps them until its own graph does, or the note would be gone with them.
    """
    nodes = []
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.requires_grad and t.is_leaf and t.is_cuda:
            stream = _lib.stream_ptr(t.device)
            capturing = torch.cuda.is_current_stream_capturing()
            node = torch.autograd.graph.get_gradient_edge(t).node
            if capturing and "frcnn_stream" not in node.metadata:
                node.metadata["frcnn_held"] = True
                del node  # without another holder the node is gone now, and the next one is new
                node = torch.autograd.graph.get_gradient_edge(t).node
                if node.metadata.pop("frcnn_held", False):
                    node.metadata["frcnn_stream"] = None
            if node.metadata.setdefault("frcnn_stream", stream) != stream and capturing:
                raise RuntimeError("an autograd graph of the same leaf, made before this capture or by another operator, is alive, so the "
                                   "captured backward pass might wait for its stream: delete what that graph returned, or capture "
                                   "with leaves of its own")
            nodes.append(node)
    return nodes


def _run(device: torch.device, function: Any, *args: Any) -> None:
    """One call through the C ABI, on ``device`` and its current stream."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = function(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _rows_of_16(t: torch.Tensor) -> torch.Tensor:
    """``t`` (rows, K) one byte an element with its rows at multiples of 16 bytes: as it is, or a padded copy."""
    rows, inner = t.shape
    stride, step = t.stride()
    if (step == 1 or inner <= 1) and (rows <= 1 or stride >= inner and stride % 16 == 0) and t.data_ptr() % 16 == 0:
        return t
    wide = torch.empty((rows, -(-inner // 16) * 16), dtype=t.dtype, device=t.device)[:, :inner]
    wide.view(torch.uint8).copy_(t.view(torch.uint8))
    return wide


def quantize_blocks(x: torch.Tensor, block_rows: int = 1,
                    scale_dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows to ``torch.float8_e4m3fn`` with one scale per block of ``block_rows`` x 128 elements.

    ``scale = max(amax * (1 / 448), 2^-126)`` in fp32 over the block's finite values (1 where they are all zero); with ``scale_dtype``
    ``torch.float8_e8m0fnu`` the smallest power of two that is not below ``amax / 448``.  ``q = x / scale`` to nearest even.
    NaN and infinities become NaN and leave the scale to their finite neighbours.

    Args:
        x: ``(..., K)`` fp32, fp16 or bf16; leading axes are flattened to rows.
        block_rows: 1 (activations) or 128 (weights, ``x`` of two axes).

    Returns:
        ``q (..., K)``, whose rows start at multiples of 16 bytes, and ``scales (ceil(rows / block_rows), ceil(K / 128))``,
        stored with the row index innermost: what ``scaled_matmul`` takes without a copy.
    """
    _no_tangent("quantize_blocks", x)
    x = _operand(x, "x")
    _no_gradient("quantize_blocks", x)
    if x.dim() < 1 or (block_rows == BLOCK and x.dim() != 2):
        raise ValueError(f"x must be (..., K) (for block_rows=128: (rows, K)), got {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    if scale_dtype not in _SCALE_TYPES:
        raise ValueError(f"scale_dtype must be one of {[str(t) for t in _SCALE_TYPES]}, got {scale_dtype}")
    device, lead, inner = x.device, x.shape[:-1], x.shape[-1]
    flat = x if x.dim() == 2 else x.reshape(lead.numel(), inner)
    rows = flat.shape[0]
    stride, step = flat.stride()
    if inner > 1 and step != 1 or rows > 1 and stride < inner:
        flat = flat.contiguous()
        stride = inner
    across, up = -(-inner // BLOCK), -(-rows // block_rows)
    # rows of a block or more start at whole lines of memory: the product reads them a line at a time
    wide = -(-inner // BLOCK) * BLOCK if inner >= BLOCK else -(-inner // 16) * 16
    q = flat.new_empty((rows, wide), dtype=_E4M3)
    scales = torch.empty_strided((up, across), (1, up), dtype=scale_dtype, device=device)
    _run(device, _lib.lib().frcnn_quantize_blocks, flat.data_ptr(), _TYPES[x.dtype], max(stride, inner), rows, inner, block_rows,
         q.data_ptr(), wide, scales.data_ptr(), _SCALE_TYPES[scale_dtype], 1, up)
    q = q[:, :inner] if wide != inner else q
    return (q if len(lead) == 1 else q.unflatten(0, lead) if lead else q[0]), scales


def scaled_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor,
                  bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act(dequantised(a) @ dequantised(b).T + bias)`` for block-scaled e4m3 operands: a dense layer when serving.

    Args:
        a: ``(..., K)`` ``torch.float8_e4m3fn`` activations; leading axes are flattened to ``M`` rows.
        a_scales: ``(M, ceil(K / 128))`` fp32 or ``float8_e8m0fnu``: one scale per 1 x 128 block.
        b: ``(N, K)`` ``torch.float8_e4m3fn`` weights (a Keras kernel transposed).
        b_scales: ``(ceil(N / 128), ceil(K / 128))`` of ``a_scales``' type: one scale per 128 x 128 block.
        bias: ``(N,)`` fp32, or ``None``.
        activation: ``None`` / ``"linear"`` or ``"relu"``.
        out_dtype: fp32, fp16 or bf16.

    Returns:
        ``(..., N)`` of ``out_dtype``.  Rows of ``a`` or ``b`` that do not start at multiples of 16 bytes are copied first;
        ``quantize_blocks`` returns rows that do.  No gradient is defined.

    Sums are held in fp32, and with ``out_dtype`` fp32 or up to 16 rows no product loses a bit.  A 16-bit result of more rows
    may come from the e4m3 matrix instructions, which cut the products of 8 neighbouring columns (``k // 8``) below ``2^-13`` of
    the largest of the eight: 1e-5 of the result for operands of random signs, more where large products of an eight cancel.
    """
    _no_tangent("scaled_matmul", a_scales, b_scales, bias)
    a = _operand(a, "a", _E4M3_ONLY)
    device = a.device
    b = _operand(b, "b", _E4M3_ONLY, device)
    a_scales = _operand(a_scales, "a_scales", _SCALE_TYPES, device)
    b_scales = _operand(b_scales, "b_scales", _SCALE_TYPES, device)
    if bias is not None:
        bias = _parameter(bias, device)
    _no_gradient("scaled_matmul", a, b, a_scales, b_scales, bias)
    act = _activation(activation, (None, "linear", "relu"))
    if out_dtype not in _TYPES:
        raise ValueError(f"out_dtype must be one of {[str(t) for t in _TYPES]}, got {out_dtype}")
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"a must be (..., K) and b (N, K), got {tuple(a.shape)} and {tuple(b.shape)}")
    lead, (units, inner) = a.shape[:-1], b.shape
    if len(lead) != 1:
        a = a.reshape(lead.numel(), inner)
    rows, across, up = a.shape[0], -(-inner // BLOCK), -(-units // BLOCK)
    if a_scales.shape != (rows, across):
        raise ValueError(f"a_scales must be ({rows}, {across}), got {tuple(a_scales.shape)}")
    if b_scales.shape != (up, across):
        raise ValueError(f"b_scales must be ({up}, {across}), got {tuple(b_scales.shape)}")
    if a_scales.dtype != b_scales.dtype:
        raise ValueError(f"a_scales and b_scales must be of one type, got {a_scales.dtype} and {b_scales.dtype}")
    if bias is not None and bias.shape != (units,):
        raise ValueError(f"bias must be ({units},), got {tuple(bias.shape)}")
    a, b = _rows_of_16(a), _rows_of_16(b)
    out = a.new_empty((rows, units), dtype=out_dtype)
    lib = _lib.lib()
    pad = -(-inner // 16) * 16
    nbytes = lib.frcnn_scaled_matmul_workspace_bytes(rows, units, inner)
    ws = _workspace(nbytes, device) if nbytes else None
    _run(device, lib.frcnn_scaled_matmul, a.data_ptr(), a.stride(0) if rows > 1 else pad, a_scales.data_ptr(), *a_scales.stride(),
         b.data_ptr(), b.stride(0) if units > 1 else pad, b_scales.data_ptr(), *b_scales.stride(), _SCALE_TYPES[a_scales.dtype],
         None if bias is None else bias.data_ptr(), act, rows, units, inner, out.data_ptr(), _TYPES[out_dtype], units,
         None if ws is None else ws.data_ptr(), nbytes)
    return out if len(lead) == 1 else out.view(*lead, units)


def _norm_shape(x: torch.Tensor, groups: int) -> Tuple[int, int, int]:
    if x.dim() < 2:
        raise ValueError(f"x must be (batch, ..., channels), got {tuple(x.shape)}")
    batch, channels, positions = x.shape[0], x.shape[-1], x.shape[1:-1].numel()
    if groups < 1 or channels < 1 or channels % groups or groups != int(groups):
        raise ValueError(f"{channels} channels are not a multiple of {groups} groups")
    if positions < 1:
        raise ValueError(f"x needs at least one position per image, got {tuple(x.shape)}")
    return batch, positions, channels


def _parameter(p: Any, device: torch.device) -> torch.Tensor:
    if p.__class__ is torch.Tensor and p.dtype is torch.float32 and p.device == device and p.is_contiguous():
        return p
    return _lib.device_tensor(p, torch.float32, device)


def _parameters(gamma: Any, beta: Any, channels: int, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
    gamma, beta = _parameter(gamma, device), _parameter(beta, device)
    if gamma.shape != (channels,) or beta.shape != (channels,):
        raise ValueError(f"gamma and beta must be ({channels},), got {tuple(gamma.shape)} and {tuple(beta.shape)}")
    return gamma, beta


def _norm_forward(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, shape: Tuple[int, int, int], groups: int, epsilon: float,
                  act: int, want_stats: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    batch, positions, channels = shape
    device = x.device
    y = torch.empty_like(x)
    stats = torch.empty((batch, groups, 2), dtype=torch.float32, device=device) if want_stats else None
    lib = _lib.lib()
    nbytes = lib.frcnn_group_norm_workspace_bytes(_TYPES[x.dtype], batch, positions, channels, groups)
    ws = _workspace(nbytes, device) if nbytes else None
    _run(device, lib.frcnn_group_norm, x.data_ptr(), _TYPES[x.dtype], batch, positions, channels, groups, gamma.data_ptr(),
         beta.data_ptr(), epsilon, act, y.data_ptr(), _lib.ptr(stats), _lib.ptr(ws), nbytes)
    return y, stats


def _norm_backward(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, stats: torch.Tensor,
                   shape: Tuple[int, int, int], act: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    (batch, positions, channels), groups = shape, stats.shape[1]
    device = x.device
    if dy.data_ptr() % 16 and x.data_ptr() % 16 == 0:
        # what x allows may not hang on where dy lies: element loads take no groups of more than 512 channels, and their time is
        # 687 us for (6000, 49, 512) bf16 where the copy and 16-byte loads take 378, 46 and 53 for (16, 1024, 576) fp32
        dy = dy.clone()
    dx = torch.empty_like(x)
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
    lib = _lib.lib()
    nbytes = lib.frcnn_group_norm_grad_workspace_bytes(_TYPES[x.dtype], batch, positions, channels, groups)
    ws = _workspace(nbytes, device) if nbytes else None
    _run(device, lib.frcnn_group_norm_grad, dy.data_ptr(), x.data_ptr(), _TYPES[x.dtype], batch, positions, channels, groups,
         gamma.data_ptr(), beta.data_ptr(), stats.data_ptr(), act, dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), _lib.ptr(ws), nbytes)
    return dx, dgamma, dbeta


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, shape, groups, epsilon, act):  # type: ignore[override]
        y, stats = _norm_forward(x, gamma, beta, shape, groups, epsilon, act, True)
        ctx.save_for_backward(x, gamma, beta, stats)
        ctx.act, ctx.shape = act, shape
        ctx.mark_non_differentiable(stats)
        return y, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):  # type: ignore[override]
        x, gamma, beta, stats = ctx.saved_tensors
        dx, dgamma, dbeta = _norm_backward(dy.contiguous(), x, gamma, beta, stats, ctx.shape, ctx.act)
        return dx, dgamma, dbeta, None, None, None, None


def group_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, groups: int, epsilon: float = 1e-3,
               activation: Optional[str] = None, return_stats: bool = False) -> Any:
    """Group normalisation of a channels-last tensor, with an activation.

    Mean and variance per image and group of neighbouring channels, over all positions:
    ``y = act((x - mean) / sqrt(var + epsilon) * gamma + beta)``.

    Args:
        x: ``(batch, ..., channels)`` fp32, fp16 or bf16 (a feature map ``(B, H, W, C)``, or pooled features with batch and
            proposals in one axis ``(B * R, 7, 7, C)``); made contiguous if it is not.
        gamma, beta: ``(channels,)``, used in fp32.
        groups: divides the channels; of up to 512 channels each, or up to 512 times 16 bytes of them where a group is a whole
            number of 16 bytes and the tensor is 16-byte aligned (others raise ``UnsupportedSizeError``).
        activation: ``None`` / ``"linear"``, ``"relu"`` or ``"swish"`` (``z / (1 + exp(-z))``).
        return_stats: also return ``stats (batch, groups, 2)`` fp32: mean and ``1 / sqrt(var + epsilon)``.

    Returns:
        ``y`` of ``x``'s shape and type, or ``(y, stats)``.  Differentiable by ``x``, ``gamma`` and ``beta`` (once).
    """
    _no_tangent("group_norm", x, gamma, beta)
    held = _leaves_of(x, gamma, beta) if torch.is_grad_enabled() else None  # before anything here makes a node of them
    x = _operand(x, "x").contiguous()
    act = _activation(activation, (None, "linear", "relu", "swish"))
    shape = _norm_shape(x, groups)
    gamma, beta = _parameters(gamma, beta, shape[2], x.device)
    epsilon = float(epsilon)
    if not epsilon >= 0.0:
        raise ValueError(f"epsilon must not be negative, got {epsilon}")
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad):
        y, stats = _GroupNorm.apply(x, gamma, beta, shape, int(groups), epsilon, act)
    else:
        y, stats = _norm_forward(x, gamma, beta, shape, int(groups), epsilon, act, return_stats)
    del held  # the graph holds them
    return (y, stats) if return_stats else y


def group_norm_gradients(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, stats: torch.Tensor,
                         activation: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``group_norm`` for a training step that keeps its own tape: ``(dx, dgamma, dbeta)`` from ``dy``, the
    call's arguments and the ``stats`` that it returned.  ``dx`` has ``x``'s type, ``dgamma`` and ``dbeta`` are fp32.
    """
    _no_tangent("group_norm_gradients", dy, x, gamma, beta, stats)
    x = _operand(x, "x").contiguous()
    device = x.device
    dy = _operand(dy, "dy", (x.dtype,), device).contiguous()
    if dy.shape != x.shape:
        raise ValueError(f"dy must be {tuple(x.shape)}, got {tuple(dy.shape)}")
    stats = _parameter(stats, device)
    if stats.dim() != 3 or stats.shape[0] != x.shape[0] or stats.shape[2] != 2:
        raise ValueError(f"stats must be ({x.shape[0]}, groups, 2), got {tuple(stats.shape)}")
    if stats.data_ptr() % 8:
        stats = stats.clone()
    act = _activation(activation, (None, "linear", "relu", "swish"))
    shape = _norm_shape(x, stats.shape[1])
    gamma, beta = _parameters(gamma, beta, shape[2], device)
    _no_gradient("group_norm_gradients", dy, x, gamma, beta, stats)
    return _norm_backward(dy, x, gamma, beta, stats, shape, act)


def _dropout(x: torch.Tensor, rate: float, seed: int, offset: int, state: Optional[torch.Tensor]) -> torch.Tensor:
    y = torch.empty_like(x)
    _run(x.device, _lib.lib().frcnn_dropout, x.data_ptr(), y.data_ptr(), _TYPES[x.dtype], x.numel(), rate, seed, offset, _lib.ptr(state))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rate, seed, offset, state):  # type: ignore[override]
        ctx.rate, ctx.seed, ctx.offset = rate, seed, offset
        # the caller may advance its state before the backward pass runs
        ctx.state = None if state is None else state.clone()
        return _dropout(x, rate, seed, offset, ctx.state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):  # type: ignore[override]
        return _dropout(dy.contiguous(), ctx.rate, ctx.seed, ctx.offset, ctx.state), None, None, None, None


def dropout(x: torch.Tensor, rate: float, seed: Any, offset: int = 0) -> torch.Tensor:
    """Dropout from a counter-based generator: the mask is a function of ``(seed, offset)`` and the element's place in
    row-major order, and is stored nowhere.

    Element ``i`` keeps its value, times ``1 / (1 - rate)``, iff word ``i % 4`` of block ``i // 4`` of Philox4x32 with 7
    rounds (key ``seed``, counter ``(block, offset)``) is at least ``round(rate * 2**32)``; the others become 0, whatever
    they were.  The gradient by ``x`` is ``dropout(dy, rate, seed, offset)``: autograd calls it, and so may a training step
    that keeps its own tape.

    Args:
        x: any shape, fp32, fp16 or bf16; made contiguous if it is not (the mask goes by the logical order).
        rate: share of elements dropped, in ``[0, 1)``.
        seed: 64-bit integer, or an int64 device tensor ``(2,)`` holding ``(seed, offset)``, read when the kernel runs: a
            captured graph that advances it draws a new mask at each replay.
        offset: 64-bit integer, a stream of its own under the same seed (one per call and layer).
    """
    _no_tangent("dropout", x)
    held = _leaves_of(x) if torch.is_grad_enabled() else None  # before anything here makes a node of it
    x = _operand(x, "x").contiguous()
    rate = float(rate)
    if not 0.0 <= rate < 1.0:
        raise ValueError(f"rate must be in [0, 1), got {rate}")
    state = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or tuple(seed.shape) != (2,) or seed.device != x.device:
            raise ValueError(f"a seed tensor must be int64 (2,) on {x.device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        if offset:
            raise ValueError("offset comes with an integer seed; a seed tensor holds its own")
        state, seed = seed.contiguous(), 0
    seed, offset = int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF
    if torch.is_grad_enabled() and x.requires_grad:
        y = _Dropout.apply(x, rate, seed, offset, state)
    else:
        y = _dropout(x, rate, seed, offset, state)
    del held  # the graph holds it
    return y
