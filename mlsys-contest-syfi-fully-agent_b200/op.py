"""Host-side mirror of the reference operator interface.

``run`` takes the eleven arguments of the reference solution's entry point in
the same order and with the same meaning (moe/solution/cuda/moe.cu:2650-2662;
definition full-agent-pipeline/references/moe.py:29-40), destination passing:
the last argument is the pre-allocated bf16 output.  It validates shapes and
dtypes the way the definition asserts them (references/moe.py:66-87) and calls
the C ABI (include/moe_b200.h) on torch's current CUDA stream.  torch is only
used for device memory and streams.
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional

import torch

from . import loader

H, I, E_LOCAL, E_GLOBAL, BLOCK = 7168, 2048, 32, 256, 128


class Workspace:
    """Caller-owned scratch memory, grown on demand (the counterpart of the
    reference's process-global ``Workspace``, moe.cu:2511-2589, but per object
    and released with it)."""

    def __init__(self, device=None):
        self.device = torch.device(device if device is not None else "cuda")
        self._buf: Optional[torch.Tensor] = None
        self._base = 0
        self.nbytes = 0

    def reserve(self, T: int):
        need = _ws_bytes.get(T)
        if need is None:
            need = _ws_bytes[T] = loader.workspace_bytes(T)
        if self._buf is None or need > self.nbytes:
            self._buf = torch.empty(need + 1024, dtype=torch.uint8, device=self.device)
            self._base = (-self._buf.data_ptr()) % 1024
            self.nbytes = need
        return self

    @property
    def ptr(self) -> int:
        return self._buf.data_ptr() + self._base

    def view(self, offset: int, nbytes: int) -> torch.Tensor:
        return self._buf[self._base + offset:self._base + offset + nbytes]


_default_ws: Dict[int, Workspace] = {}
_ws_bytes: Dict[int, int] = {}       # workspace size per token count (a library call otherwise)


def _default_workspace(device: torch.device) -> Workspace:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _default_ws:
        _default_ws[idx] = Workspace(torch.device("cuda", idx))
    return _default_ws[idx]


def _check(cond: bool, msg: str):
    if not cond:
        raise ValueError(msg)


_validated: Dict[tuple, bool] = {}     # signatures of argument sets that passed _validate
_VALIDATED_MAX = 64


def _stream_of(dev: torch.device) -> int:
    """Handle of torch's current stream on ``dev``."""
    try:
        return torch._C._cuda_getCurrentRawStream(dev.index if dev.index is not None else torch.cuda.current_device())
    except AttributeError:      # a torch build without the raw getter
        return torch.cuda.current_stream(dev).cuda_stream


class _on_device:
    """``torch.cuda.device(dev)`` only when ``dev`` is not already current (the context manager costs
    more host time than the launch it wraps)."""

    def __init__(self, dev: torch.device):
        self.ctx = None
        if dev.index is not None and dev.index != torch.cuda.current_device():
            self.ctx = torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


def _validate(routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights, gemm1_weights_scale,
              gemm2_weights, gemm2_weights_scale, output, device_inputs: bool):
    """Checks the nine tensors the way the definition asserts them; returns (T, their addresses)."""
    T = routing_logits.shape[0]
    # A serving loop calls with the same buffers again and again (or rotates over a few sets): an argument set
    # whose addresses, dtypes and shapes equal a validated one is not inspected a second time (the checks cost
    # more host time than a decode step's launch).
    args = (routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights, gemm1_weights_scale,
            gemm2_weights, gemm2_weights_scale, output)
    ptrs = tuple([t.data_ptr() for t in args])
    sig = (device_inputs, ptrs, tuple([(t.dtype, t.shape) for t in args]))
    if sig in _validated:
        return T, ptrs
    _check(routing_logits.dtype == torch.float32 and tuple(routing_logits.shape) == (T, E_GLOBAL),
           "routing_logits must be float32 [T, 256]")
    _check(routing_bias.dtype == torch.bfloat16 and routing_bias.numel() == E_GLOBAL, "routing_bias must be bfloat16 [256]")
    _check(hidden_states.dtype == torch.float8_e4m3fn and tuple(hidden_states.shape) == (T, H),
           "hidden_states must be float8_e4m3fn [T, 7168]")
    _check(hidden_states_scale.dtype == torch.float32 and tuple(hidden_states_scale.shape) == (H // BLOCK, T),
           "hidden_states_scale must be float32 [56, T]")
    _check(gemm1_weights.dtype == torch.float8_e4m3fn and tuple(gemm1_weights.shape) == (E_LOCAL, 2 * I, H),
           "gemm1_weights must be float8_e4m3fn [32, 4096, 7168]")
    _check(gemm1_weights_scale.dtype == torch.float32 and
           tuple(gemm1_weights_scale.shape) == (E_LOCAL, 2 * I // BLOCK, H // BLOCK),
           "gemm1_weights_scale must be float32 [32, 32, 56]")
    _check(gemm2_weights.dtype == torch.float8_e4m3fn and tuple(gemm2_weights.shape) == (E_LOCAL, H, I),
           "gemm2_weights must be float8_e4m3fn [32, 7168, 2048]")
    _check(gemm2_weights_scale.dtype == torch.float32 and
           tuple(gemm2_weights_scale.shape) == (E_LOCAL, H // BLOCK, I // BLOCK),
           "gemm2_weights_scale must be float32 [32, 56, 16]")
    _check(output.dtype == torch.bfloat16 and tuple(output.shape) == (T, H), "output must be bfloat16 [T, 7168]")
    tensors = dict(routing_logits=routing_logits, routing_bias=routing_bias, hidden_states=hidden_states,
                   hidden_states_scale=hidden_states_scale, gemm1_weights=gemm1_weights,
                   gemm1_weights_scale=gemm1_weights_scale, gemm2_weights=gemm2_weights,
                   gemm2_weights_scale=gemm2_weights_scale, output=output)
    for name, t in tensors.items():
        # size-1 dimensions make torch report odd strides for [56, 1]; numel-sized storage is what matters
        _check(t.is_contiguous(), f"{name} must be contiguous")
        on_device = name.startswith("gemm") or device_inputs
        _check(t.is_cuda == on_device, f"{name} must live on the {'GPU' if on_device else 'host'}")
    if len(_validated) >= _VALIDATED_MAX:
        _validated.clear()
    _validated[sig] = True
    return T, ptrs


def run(routing_logits: torch.Tensor, routing_bias: torch.Tensor, hidden_states: torch.Tensor,
        hidden_states_scale: torch.Tensor, gemm1_weights: torch.Tensor, gemm1_weights_scale: torch.Tensor,
        gemm2_weights: torch.Tensor, gemm2_weights_scale: torch.Tensor, local_expert_offset: int,
        routed_scaling_factor: float, output: Optional[torch.Tensor] = None,
        workspace: Optional[Workspace] = None) -> torch.Tensor:
    """The MoE shard, asynchronous on the current CUDA stream.  ``output`` (bf16
    [T, 7168]) is fully overwritten and returned; it is allocated when omitted."""
    if output is None:
        output = torch.empty((routing_logits.shape[0], H), dtype=torch.bfloat16, device=hidden_states.device)
    T, ptrs = _validate(routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights,
                        gemm1_weights_scale, gemm2_weights, gemm2_weights_scale, output, device_inputs=True)
    if T == 0:
        return output
    dev = hidden_states.device
    ws = (workspace or _default_workspace(dev)).reserve(T)
    with _on_device(dev):
        rc = loader.lib.moe_fp8_block_scale_run(*ptrs[:8], T, int(local_expert_offset), float(routed_scaling_factor),
                                                ptrs[8], ws.ptr, ws.nbytes, _stream_of(dev))
    if rc:
        loader.check(rc)
    return output


def run_rows(routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights, gemm1_weights_scale,
             gemm2_weights, gemm2_weights_scale, local_expert_offset: int, routed_scaling_factor: float,
             output_rows: torch.Tensor, workspace: Optional[Workspace] = None) -> None:
    """The operator with a per-token destination: ``output_rows`` is an int64 CUDA tensor of T device
    addresses (16-byte aligned, 7168 bf16 each; peer-mapped memory allowed) that row t is written to."""
    T = routing_logits.shape[0]
    dummy = torch.empty((T, H), dtype=torch.bfloat16, device="meta")
    _check(output_rows.dtype == torch.int64 and output_rows.numel() == T and output_rows.is_cuda and
           output_rows.is_contiguous(), "output_rows must be a contiguous CUDA int64 tensor of T addresses")
    del dummy
    if T == 0:
        return
    dev = hidden_states.device
    ws = (workspace or _default_workspace(dev)).reserve(T)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = loader.lib.moe_fp8_block_scale_run_rows(
            routing_logits.data_ptr(), routing_bias.data_ptr(), hidden_states.data_ptr(),
            hidden_states_scale.data_ptr(), gemm1_weights.data_ptr(), gemm1_weights_scale.data_ptr(),
            gemm2_weights.data_ptr(), gemm2_weights_scale.data_ptr(), int(T), int(local_expert_offset),
            float(routed_scaling_factor), output_rows.data_ptr(), ws.ptr, ws.nbytes, stream)
    loader.check(rc)


def run_host(routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights, gemm1_weights_scale,
             gemm2_weights, gemm2_weights_scale, local_expert_offset: int, routed_scaling_factor: float,
             output: torch.Tensor, workspace: Optional[Workspace] = None) -> torch.Tensor:
    """Same operator for token-side tensors in (pinned) host memory: copies them
    in, runs, copies ``output`` (a host tensor) back and waits."""
    T, ptrs = _validate(routing_logits, routing_bias, hidden_states, hidden_states_scale, gemm1_weights,
                        gemm1_weights_scale, gemm2_weights, gemm2_weights_scale, output, device_inputs=False)
    if T == 0:
        return output
    dev = gemm1_weights.device
    ws = (workspace or _default_workspace(dev)).reserve(T)
    with _on_device(dev):
        rc = loader.lib.moe_fp8_block_scale_run_host(*ptrs[:8], T, int(local_expert_offset),
                                                     float(routed_scaling_factor), ptrs[8], ws.ptr, ws.nbytes,
                                                     _stream_of(dev))
    if rc:
        loader.check(rc)
    return output


def route(routing_logits: torch.Tensor, routing_bias: torch.Tensor, local_expert_offset: int,
          routed_scaling_factor: float):
    """Routing alone: (topk_idx i32 [T,8], topk_w f32 [T,8], local_mask i32 [T]) on the current stream."""
    T = routing_logits.shape[0]
    dev = routing_logits.device
    idx = torch.empty((T, 8), dtype=torch.int32, device=dev)
    w = torch.empty((T, 8), dtype=torch.float32, device=dev)
    mask = torch.empty((T,), dtype=torch.int32, device=dev)
    if T:
        with torch.cuda.device(dev):
            loader.check(loader.lib.moe_fp8_block_scale_route(
                routing_logits.data_ptr(), routing_bias.data_ptr(), int(T), int(local_expert_offset),
                float(routed_scaling_factor), idx.data_ptr(), w.data_ptr(), mask.data_ptr(),
                torch.cuda.current_stream(dev).cuda_stream))
    return idx, w, mask


def quantize_activations(hidden_bf16: torch.Tensor):
    """bf16 [T, 7168] -> (e4m3 [T, 7168], fp32 scales [56, T]) in the operator's input layout."""
    _check(hidden_bf16.dtype == torch.bfloat16 and hidden_bf16.dim() == 2 and hidden_bf16.shape[1] == H and
           hidden_bf16.is_contiguous() and hidden_bf16.is_cuda, "hidden must be a contiguous CUDA bfloat16 [T, 7168]")
    T = hidden_bf16.shape[0]
    dev = hidden_bf16.device
    q = torch.empty((T, H), dtype=torch.float8_e4m3fn, device=dev)
    s = torch.empty((H // BLOCK, T), dtype=torch.float32, device=dev)
    if T:
        with torch.cuda.device(dev):
            loader.check(loader.lib.moe_fp8_block_scale_quantize_activations(
                hidden_bf16.data_ptr(), int(T), q.data_ptr(), s.data_ptr(), torch.cuda.current_stream(dev).cuda_stream))
    return q, s


# ---------------------------------------------------------------------------- operators around the shard
#
# What a decoder layer does directly before the router and the experts and directly after them.  Like ``run`` they work
# on torch's current stream of the tensors' device and can be captured in a CUDA graph; they record nothing for
# autograd: every gradient is a call of its own.  Scratch memory comes from torch's allocator for the call.

_TYPE_CODE = {torch.float32: loader.F32, torch.bfloat16: loader.BF16, torch.float16: loader.F16}
_SCORING = {"sigmoid": loader.SCORE_SIGMOID, "softmax": loader.SCORE_SOFTMAX}
NORM_MAX_WIDTH, BALANCE_MAX_EXPERTS, MATVEC_MAX_PAIRS, MATVEC_MAX_EXPERTS = 16384, 1024, 256, 1024
_scratch_bytes: Dict[tuple, int] = {}          # library's workspace size per kind and sizes


def _scratch(kind, fn, a: int, b: int, like: torch.Tensor) -> torch.Tensor:
    need = _scratch_bytes.get((kind, a, b))
    if need is None:
        if len(_scratch_bytes) >= 4096:
            _scratch_bytes.clear()
        need = _scratch_bytes[kind, a, b] = int(fn(a, b))
    return like.new_empty(need, dtype=torch.uint8)


def _launch(fn, dev: torch.device, *args):
    """Calls an entry point of the library with ``dev`` current and its stream as the last argument.  (A decode step's
    kernel takes a few microseconds: the calls below spend as little host time as they can, so checks are written
    without helpers that would format a message that is not needed.)"""
    try:
        current = torch._C._cuda_getDevice()
    except AttributeError:      # a torch build without the raw getter
        current = torch.cuda.current_device()
    if dev.index == current:
        rc = fn(*args, _stream_of(dev))
    else:
        with torch.cuda.device(dev.index):
            rc = fn(*args, _stream_of(dev))
    if rc:
        loader.check(rc)


def _rows(name: str, t: torch.Tensor, shape, dtype: torch.dtype, dev: torch.device):
    """Checks an activation argument [T, H] whose rows may lie apart; returns (address, row stride)."""
    if t.dtype is not dtype or t.shape != shape or t.device != dev:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on {dev}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: the elements of a row must be adjacent")
    return t.data_ptr(), (stride[0] if shape[0] > 1 else 0)


def _aligned(t: Optional[torch.Tensor]) -> bool:
    """Rows (or the one row) of an argument can be read 16 bytes at a time."""
    return t is None or (t.data_ptr() % 16 == 0 and
                         (t.dim() == 1 or t.shape[0] <= 1 or t.stride(0) * t.element_size() % 16 == 0))


def _new_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (``empty_like`` costs less, but keeps the layout of some views)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _on_gpu(t: torch.Tensor):
    if not t.is_cuda:
        raise ValueError("the tensors must be on a GPU: there is no CPU path")


def _param(name: str, t: torch.Tensor, H: int, dtype: torch.dtype, dev: torch.device):
    """Checks a parameter [H] in the activations' type or float32; returns (address, is float32)."""
    f32 = t.dtype is torch.float32
    if not (f32 or t.dtype is dtype) or t.dim() != 1 or t.shape[0] != H or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} or float32 [{H}] on {dev}")
    return t.data_ptr(), f32


def _norm_inputs(x, pre_weight, y, post_weight, gate, residual_scale):
    """Checks what both directions of the block norm take; returns the leading arguments of the C call."""
    dtype, shape, dev = x.dtype, x.shape, x.device
    code = _TYPE_CODE.get(dtype)
    if code is None or len(shape) != 2:
        raise ValueError("x must be float32, bfloat16 or float16 [T, H]")
    T, H = shape
    if not 1 <= H <= NORM_MAX_WIDTH or T > 2 ** 30:
        raise ValueError(f"x must have at most 2^30 rows and 1 to {NORM_MAX_WIDTH} columns")
    xp, xs = _rows("x", x, shape, dtype, dev)
    pre, f32 = _param("pre_weight", pre_weight, H, dtype, dev)
    params = 1 if f32 else 0
    yp = post = gp = None
    ys = gs = kind = 0
    if y is not None:
        yp, ys = _rows("y", y, shape, dtype, dev)
        if post_weight is not None:
            post, f32 = _param("post_weight", post_weight, H, dtype, dev)
            if f32:
                params |= 2
        if gate is not None:
            if gate.dim() == 1:
                gp, f32 = _param("gate", gate, H, dtype, dev)
                kind = 1
            else:
                f32 = gate.dtype is torch.float32
                kind = 2 if gate.dim() == 2 and gate.shape[1] == 1 else 3
                gp, gs = _rows("gate", gate, (T, 1) if kind == 2 else shape, torch.float32 if f32 else dtype, dev)
            if f32:
                params |= 4
    elif post_weight is not None or gate is not None:
        raise ValueError("post_weight and gate belong to y")
    return T, H, (xp, xs, yp, ys, gp, gs, kind, pre, post, T, H, code, params, float(residual_scale))


def block_norm(x: torch.Tensor, pre_weight: torch.Tensor, y: Optional[torch.Tensor] = None,
               post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
               residual_scale: float = 1.0, eps: float = 1e-6, quantize: bool = False):
    """Joins a block's output ``y`` to the residual stream ``x`` and norms the stream for the next block::

        n = y * rsqrt(mean(y^2) + eps) * post_weight      (n = y without post_weight)
        s = residual_scale * x + gate * n                 (s = x without y, whatever the scale)
        h = s * rsqrt(mean(s^2) + eps) * pre_weight

    x, y: float32 / bfloat16 / float16 [T, H], rows may lie apart; weights [H] and ``gate`` -- [H] per channel, [T, 1]
    per token or [T, H] -- in the same type or float32.  Returns (s, h, rstd): s is ``x`` itself without y, rstd float32
    [T, 2] is what ``block_norm_backward`` takes.  With ``quantize`` h is the pair (e4m3 [T, H], float32 scales
    [H / 128, T]) that ``run`` takes as hidden_states and hidden_states_scale, rounded from the unrounded h; H must then
    be a multiple of 128 and all rows 16-byte aligned.  Arithmetic is float32, what is stored is rounded once."""
    T, H, args = _norm_inputs(x, pre_weight, y, post_weight, gate, residual_scale)
    if not eps >= 2.0 ** -149:
        raise ValueError("eps must be a positive float32")
    if quantize:
        if H % BLOCK != 0:
            raise ValueError(f"quantize needs a multiple of {BLOCK} columns")
        if not (_aligned(x) and _aligned(y) and _aligned(pre_weight) and _aligned(post_weight) and
                (args[6] == 2 or _aligned(gate))):
            raise ValueError("quantize needs rows that are 16-byte aligned")
    _on_gpu(x)
    s = x if y is None else _new_like(x)
    rstd = x.new_empty((T, 2), dtype=torch.float32)
    scale = None
    if quantize:
        h = x.new_empty((T, H), dtype=torch.float8_e4m3fn)
        scale = x.new_empty((H // BLOCK, T), dtype=torch.float32)
    else:
        h = _new_like(x)
    if T:
        _launch(loader.lib.moe_fp8_block_scale_block_norm, x.device, *args, eps, None if y is None else s.data_ptr(),
                h.data_ptr(), scale.data_ptr() if quantize else None, rstd.data_ptr())
    return s, ((h, scale) if quantize else h), rstd


def block_norm_backward(x: torch.Tensor, pre_weight: torch.Tensor, rstd: torch.Tensor, grad_h: torch.Tensor,
                        grad_stream: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None,
                        post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        residual_scale: float = 1.0) -> Dict[str, Optional[torch.Tensor]]:
    """Gradients of ``block_norm`` with the same x, y, weights, gate and scale and the ``rstd`` it returned.  grad_h [T, H]
    belongs to h (straight through the quantisation), grad_stream [T, H] to s (None: zero).  Returns a dict with the
    gradients of ``x``, ``y``, ``gate``, ``pre_weight`` and ``post_weight`` in their shapes and types, None where there
    is no such argument.  Sums over tokens are float32 in a fixed order."""
    T, H, args = _norm_inputs(x, pre_weight, y, post_weight, gate, residual_scale)
    dev, dtype, shape = x.device, x.dtype, x.shape
    if rstd.dtype is not torch.float32 or rstd.shape != (T, 2) or not rstd.is_contiguous() or rstd.device != dev or \
            rstd.data_ptr() % 8 != 0:
        raise ValueError("rstd must be the float32 [T, 2] that block_norm returned")
    gh, gh_stride = _rows("grad_h", grad_h, shape, dtype, dev)
    gs, gs_stride = (None, 0) if grad_stream is None else _rows("grad_stream", grad_stream, shape, dtype, dev)
    _on_gpu(x)
    out = {"x": _new_like(x), "pre_weight": torch.empty_like(pre_weight),
           "y": None if y is None else _new_like(x),
           "post_weight": None if post_weight is None else torch.empty_like(post_weight),
           "gate": None if gate is None else _new_like(gate)}
    if T == 0:                                     # the sums over no token
        for k in ("pre_weight", "post_weight", "gate"):
            if out[k] is not None:
                out[k].zero_()
        return out
    ws = _scratch("norm", loader.lib.moe_fp8_block_scale_block_norm_backward_workspace_bytes, T, H, x)
    _launch(loader.lib.moe_fp8_block_scale_block_norm_backward, dev, *args, rstd.data_ptr(), gh, gh_stride, gs, gs_stride,
            *[None if out[k] is None else out[k].data_ptr() for k in ("x", "y", "gate", "pre_weight", "post_weight")],
            ws.data_ptr(), ws.shape[0])
    return out


def _balance_inputs(logits, top_k, cu_seqlens, token_mask, scoring):
    """Checks what both directions of the balance loss take; returns (type code, T, E, S, arguments after K)."""
    shape, dev = logits.shape, logits.device
    code = _TYPE_CODE.get(logits.dtype)
    if code is None or len(shape) != 2:
        raise ValueError("logits must be float32, bfloat16 or float16 [T, E]")
    T, E = shape
    if not 1 <= E <= BALANCE_MAX_EXPERTS or T > 2 ** 30:
        raise ValueError(f"logits must have at most 2^30 rows and 1 to {BALANCE_MAX_EXPERTS} columns")
    if E > 1 and logits.stride(1) != 1:
        raise ValueError("logits: the elements of a row must be adjacent")
    if not 1 <= top_k <= E:
        raise ValueError("every token selects 1 to E experts")
    if scoring not in _SCORING:
        raise ValueError("scoring must be 'sigmoid' or 'softmax'")
    S, cu, mask = 1, None, None
    if cu_seqlens is not None:
        if cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or \
                not cu_seqlens.is_contiguous() or cu_seqlens.device != dev:
            raise ValueError(f"cu_seqlens must be a contiguous int32 [sequences + 1] on {dev}")
        S, cu = cu_seqlens.shape[0] - 1, cu_seqlens.data_ptr()
    if token_mask is not None:
        if token_mask.dtype is not torch.bool or token_mask.shape != (T,) or not token_mask.is_contiguous() or \
                token_mask.device != dev:
            raise ValueError(f"token_mask must be a contiguous bool [{T}] on {dev}")
        mask = token_mask.data_ptr() or None
    return code, T, E, S, (cu, S, mask, _SCORING[scoring])


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, alpha: float, cu_seqlens: Optional[torch.Tensor] = None,
                 token_mask: Optional[torch.Tensor] = None, scoring: str = "sigmoid"):
    """Balance loss of a routing, per sequence, with the per-expert counts::

        p = s / sum(s),  s = sigmoid(logits) or exp(logits)        ("sigmoid": the routing of ``route``)
        loss[q] = alpha * sum_i f_i P_i,  f_i = E / (K n) counts[q, i],  P_i = mean of p[:, i] over the n tokens

    logits float32 / bfloat16 / float16 [T, E]; topk_idx int32 [T, K], what ``route`` returns (indices outside [0, E)
    count nowhere).  cu_seqlens int32 [S + 1] has the ascending borders of packed sequences (tokens outside every
    sequence are left out; None: one sequence); tokens with a False in token_mask [T] are left out too, whatever their
    rows hold.  Returns (loss float32 [S], counts int32 [S, E], tokens int32 [S]); a sequence without a token has loss 0."""
    if topk_idx.dtype is not torch.int32 or topk_idx.dim() != 2 or not topk_idx.is_contiguous() or \
            topk_idx.device != logits.device:
        raise ValueError("topk_idx must be a contiguous int32 [T, K] on the logits' device")
    rows, K = topk_idx.shape
    code, T, E, S, rest = _balance_inputs(logits, K, cu_seqlens, token_mask, scoring)
    if rows != T:
        raise ValueError("topk_idx must have a row for every token")
    _on_gpu(logits)
    loss = logits.new_empty(S, dtype=torch.float32)
    counts = topk_idx.new_empty((S, E))
    tokens = topk_idx.new_empty(S)
    if S:
        ws = _scratch("balance", loader.lib.moe_fp8_block_scale_balance_loss_workspace_bytes, T, E, logits)
        _launch(loader.lib.moe_fp8_block_scale_balance_loss, logits.device, logits.data_ptr(), logits.stride(0), code,
                topk_idx.data_ptr(), T, E, K, *rest, float(alpha), loss.data_ptr(), counts.data_ptr(), tokens.data_ptr(),
                ws.data_ptr(), ws.shape[0])
    return loss, counts, tokens


def balance_loss_backward(grad_loss: torch.Tensor, logits: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor,
                          top_k: int, alpha: float, cu_seqlens: Optional[torch.Tensor] = None,
                          token_mask: Optional[torch.Tensor] = None, scoring: str = "sigmoid") -> torch.Tensor:
    """Gradient of ``balance_loss`` for the logits, in their type, given the gradient of its losses (float32 [S]) and the
    counts and tokens it returned; the counts are constants.  Rows of tokens that were left out are zero."""
    code, T, E, S, rest = _balance_inputs(logits, top_k, cu_seqlens, token_mask, scoring)
    dev = logits.device
    if grad_loss.dtype is not torch.float32 or grad_loss.shape != (S,) or not grad_loss.is_contiguous() or grad_loss.device != dev:
        raise ValueError(f"grad_loss must be a contiguous float32 [{S}] on {dev}")
    if counts.dtype is not torch.int32 or counts.shape != (S, E) or not counts.is_contiguous() or counts.device != dev:
        raise ValueError(f"counts must be a contiguous int32 [{S}, {E}] on {dev}")
    if tokens.dtype is not torch.int32 or tokens.shape != (S,) or not tokens.is_contiguous() or tokens.device != dev:
        raise ValueError(f"tokens must be a contiguous int32 [{S}] on {dev}")
    _on_gpu(logits)
    grad = logits.new_empty((T, E))
    if T:
        _launch(loader.lib.moe_fp8_block_scale_balance_loss_backward, dev, grad_loss.data_ptr(), logits.data_ptr(),
                logits.stride(0), code, counts.data_ptr(), tokens.data_ptr(), T, E, top_k, *rest, float(alpha), grad.data_ptr())
    return grad


def matvec_w4(x: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None,
              experts: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Products of a decode-sized batch with 4-bit weights and group scales::

        out[r, n] = sum_k x[r, k] * (q[n, k] - zero[n, k // G]) * scale[n, k // G]

    x bfloat16 / float16 [R, K]; qweight uint8 [N, K / 2], two values a byte, the even k in the
    low half; scale [N, K / G] in x's type or float32, G = 32, 64 or 128; zero uint8 [N, K / G], 0 to 15 (None: 8).  With
    ``experts`` the weights have a leading dimension E and every (row, choice) has its own matrix: experts int32 [R] gives
    out [R, N], [R, k] gives [R, k, N] (the experts that ``route`` selected, less the shard's first); an expert outside
    [0, E) gives zeros.  At most 256 (row, choice) pairs and 1024 experts.  out has x's type, or float32 with
    ``out_dtype``; sums are float32.  For a float32 result q - zero is formed exactly; for a 16-bit one a group's sum is
    sum q x - zero sum x, whose float32 errors go with sum |q x|, and bfloat16 wants |x| < 2^63 (an infinite x gives NaN)."""
    dtype, dev, shape = x.dtype, x.device, x.shape
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or len(shape) != 2:
        raise ValueError("x must be bfloat16 or float16 [R, K]")
    R, K = shape
    lead = 0 if experts is None else 1
    wshape = qweight.shape
    if qweight.dtype is not torch.uint8 or len(wshape) != 2 + lead or not qweight.is_contiguous() or \
            qweight.device != dev or K < 1 or wshape[-1] * 2 != K or qweight.numel() == 0:
        raise ValueError(f"qweight must be a contiguous uint8 [{'E, ' if lead else ''}N, {K} / 2] on {dev}")
    E, N = (wshape[0] if lead else 1), wshape[-2]
    if N > 2 ** 22 or K > 2 ** 20 or E > MATVEC_MAX_EXPERTS:
        raise ValueError(f"at most 2^22 rows, 2^20 columns and {MATVEC_MAX_EXPERTS} experts")
    sshape, stype = scale.shape, scale.dtype
    groups = sshape[-1] if len(sshape) else 0
    G = K // groups if groups else 0
    if G not in (32, 64, 128) or G * groups != K or (stype is not dtype and stype is not torch.float32) or \
            sshape[:-1] != wshape[:-1] or not scale.is_contiguous() or scale.device != dev:
        raise ValueError(f"scale must be a contiguous {dtype} or float32 [{'E, ' if lead else ''}N, K / G] on {dev}, "
                         "G = 32, 64 or 128")
    if zero is not None and (zero.dtype is not torch.uint8 or zero.shape != sshape or not zero.is_contiguous() or
                             zero.device != dev):
        raise ValueError("zero must be a contiguous uint8 tensor of scale's shape")
    stride, xp, qp = x.stride(), x.data_ptr(), qweight.data_ptr()
    if (K > 1 and stride[1] != 1) or (R > 1 and stride[0] % 8 != 0) or xp % 16 != 0 or qp % 16 != 0:
        raise ValueError("the rows of x and qweight must be 16-byte aligned and x's elements adjacent")
    per_row, oshape, ids = 1, (R, N), None
    if lead:
        eshape = experts.shape
        if experts.dtype is not torch.int32 or len(eshape) not in (1, 2) or eshape[0] != R or \
                not experts.is_contiguous() or experts.device != dev:
            raise ValueError(f"experts must be a contiguous int32 [{R}] or [{R}, k] on {dev}")
        per_row = eshape[1] if len(eshape) == 2 else 1
        oshape, ids = (*eshape, N), experts.data_ptr()
    pairs = R * per_row
    if pairs > MATVEC_MAX_PAIRS:
        raise ValueError(f"at most {MATVEC_MAX_PAIRS} (row, expert) pairs")
    if out_dtype is not None and out_dtype is not dtype and out_dtype is not torch.float32:
        raise ValueError("out_dtype must be x's type or float32")
    _on_gpu(x)
    out = x.new_empty(oshape, dtype=out_dtype)
    if pairs:
        _launch(loader.lib.moe_fp8_block_scale_matvec_w4, dev, xp, stride[0] if R > 1 else 0, _TYPE_CODE[dtype], qp,
                scale.data_ptr(), stype is torch.float32, None if zero is None else zero.data_ptr(), ids, pairs, per_row, E, N,
                K, G, out.data_ptr(), out_dtype is torch.float32)
    return out


def kernel_status(workspace: Optional[Workspace] = None, device=None) -> int:
    """Waits for the current stream and returns the kernels' error bits (0 = none)."""
    dev = torch.device(device if device is not None else "cuda")
    ws = workspace or _default_workspace(dev)
    st = ctypes.c_int(0)
    with torch.cuda.device(ws.device):
        rc = loader.lib.moe_fp8_block_scale_status(ws.ptr, torch.cuda.current_stream().cuda_stream, ctypes.byref(st))
    if rc not in (loader.OK, loader.EKERNEL):
        loader.check(rc)
    return st.value


def read_schedule(T: int, workspace: Optional[Workspace] = None, device=None) -> "loader.Sched":
    """Waits for the device and returns a host copy of the schedule block the last call with ``T``
    tokens left in the workspace: error bits, rows, active experts, tile widths and split-K factors
    the device chose, per-expert counts and offsets (``include/moe_b200.h``: ``moe_b200_sched``)."""
    dev = torch.device(device if device is not None else "cuda")
    ws = workspace or _default_workspace(dev)
    torch.cuda.synchronize(ws.device)
    L = loader.layout(T)
    raw = ws.view(L.sched, ctypes.sizeof(loader.Sched)).cpu().numpy().tobytes()
    return loader.Sched.from_buffer_copy(raw)
