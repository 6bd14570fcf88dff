"""The whole expert layer, router included, for a few tokens in one kernel.

:func:`b300_moe_forward` takes expert ids and routing weights, which a caller first has to make
from the hidden states (a product with the router's weight, then
:func:`b200moe.topk_routing`), and runs four to five kernels.  With one to eight tokens the time
between those launches is comparable with the layer itself; ``b300_moe_layer`` starts from the
hidden states and the router's weight and runs a single kernel.  No counterpart in the
reference.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .forward import _check_out, _native_args, _resolve_native_backend
from .fp8 import Fp8ExpertWeights
from .validation import MAX_EXPERTS, SUPPORTED_TOP_K, RoutedMoEShape, _positive_int, _tensor
from .workspace import B300MoEWorkspace

MAX_LAYER_TOKENS = 8
MAX_LAYER_HIDDEN = 8192
MAX_LAYER_INTER = 65536


def _validate(hidden_states, router_weight, gate_up, down, scales, num_experts: int, top_k: int,
              kind: torch.dtype, step: int) -> RoutedMoEShape:
    """Argument checks of both entry points; ``gate_up`` / ``down`` are BF16 weights, or E4M3
    codes with their two row scales."""

    _tensor("hidden_states", hidden_states)
    _tensor("router_weight", router_weight)
    _tensor("gate_up_weight", gate_up)
    _tensor("down_weight", down)
    num_experts = _positive_int("num_experts", num_experts)
    top_k = _positive_int("top_k", top_k)
    if top_k not in SUPPORTED_TOP_K:
        raise ValueError(f"top_k must be one of {SUPPORTED_TOP_K}, got {top_k}")
    if top_k > num_experts:
        raise ValueError("top_k must not exceed num_experts")
    if num_experts > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts are supported")
    if hidden_states.ndim != 2 or hidden_states.shape[0] < 1:
        raise ValueError("hidden_states must have shape [num_tokens, hidden_size]")
    tokens, hidden = hidden_states.shape
    if tokens > MAX_LAYER_TOKENS:
        raise ValueError(f"the one-kernel layer takes at most {MAX_LAYER_TOKENS} tokens, got "
                         f"{tokens}; use topk_routing and b300_moe_forward")
    if router_weight.shape != (num_experts, hidden):
        raise ValueError("router_weight must have shape [num_experts, hidden_size]")
    if gate_up.ndim != 3 or gate_up.shape[0] != num_experts or gate_up.shape[2] != hidden or \
            gate_up.shape[1] < 2 or gate_up.shape[1] % 2:
        raise ValueError("gate_up_weight must have shape [E, 2I, H]")
    inter = gate_up.shape[1] // 2
    if down.shape != (num_experts, hidden, inter):
        raise ValueError("down_weight must have shape [E, H, I] compatible with gate_up_weight")
    if scales is not None and (scales[0].shape != (num_experts, 2 * inter)
                               or scales[1].shape != (num_experts, hidden)):
        raise ValueError("scales must have shapes [E, 2I] and [E, H]")
    if hidden_states.dtype != torch.bfloat16:
        raise TypeError("hidden_states must have dtype torch.bfloat16")
    if router_weight.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("router_weight must have dtype torch.bfloat16 or torch.float32")
    if gate_up.dtype != kind or down.dtype != kind:
        raise TypeError(f"gate_up_weight and down_weight must have dtype {kind}")
    if scales is not None and (scales[0].dtype is not torch.float32
                               or scales[1].dtype is not torch.float32):
        raise TypeError("scales must have dtype torch.float32")
    device = hidden_states.device
    if router_weight.device != device or gate_up.device != device or down.device != device or \
            (scales is not None and (scales[0].device != device or scales[1].device != device)):
        raise ValueError("all inputs must be on the same device")
    if not (hidden_states.is_contiguous() and router_weight.is_contiguous()
            and gate_up.is_contiguous() and down.is_contiguous()
            and (scales is None or scales[0].is_contiguous() and scales[1].is_contiguous())):
        raise ValueError("all inputs must be contiguous")
    if hidden_states.requires_grad or router_weight.requires_grad or gate_up.requires_grad or \
            down.requires_grad or \
            (scales is not None and (scales[0].requires_grad or scales[1].requires_grad)):
        raise ValueError("the one-kernel layer does not support autograd")
    if hidden % step or inter % step:
        raise ValueError(f"hidden_size and intermediate_size must be divisible by {step}")
    if hidden > MAX_LAYER_HIDDEN or inter > MAX_LAYER_INTER:
        raise ValueError(f"the one-kernel layer takes hidden_size up to {MAX_LAYER_HIDDEN} and "
                         f"intermediate_size up to {MAX_LAYER_INTER}")
    return RoutedMoEShape(tokens, num_experts, top_k, hidden, inter)


class _Binding:
    """What a workspace keeps for this entry point from one :meth:`reserve` to the next: the
    argument struct with the dimensions and scratch filled in, and the stream of the last use."""

    __slots__ = ("key", "allocations", "tokens", "stream", "stream_ptr", "args", "ref")


def _bind(workspace: B300MoEWorkspace, key, hidden_states, gate_up, down,
          shape: RoutedMoEShape) -> _Binding:
    """Reserves the workspace for this call, by its own rules, and binds an argument struct."""

    device = hidden_states.device
    workspace.reserve(
        num_tokens=shape.num_tokens, num_experts=shape.num_experts, top_k=shape.top_k,
        hidden_size=shape.hidden_size, intermediate_size=shape.intermediate_size,
        device=device, dtype=torch.bfloat16, backend="b200_bf16", quant_mode="bf16")
    b = _Binding()
    b.key, b.allocations, b.tokens = key, workspace.allocation_count, workspace._tokens
    b.stream = torch.cuda.current_stream(device)
    b.stream_ptr = int(b.stream.cuda_stream)
    # a copy: the struct that the workspace caches is bound to the last call's weights.  The
    # routing tensors of the struct are not read by this entry point.
    b.args = _lib.B200MoeArgs.from_buffer_copy(
        _native_args(hidden_states, hidden_states, hidden_states, gate_up, down, shape, workspace,
                     None, 0))
    b.ref = ctypes.byref(b.args)
    workspace._layer_binding = b
    return b


def _run(hidden_states, router_weight, gate_up, down, scales, shape: RoutedMoEShape,
         workspace: B300MoEWorkspace | None, return_routing: bool, check_status: bool,
         out: torch.Tensor | None):
    if workspace is not None and not isinstance(workspace, B300MoEWorkspace):
        raise TypeError("workspace must be a B300MoEWorkspace or None")
    device = hidden_states.device
    active = workspace if workspace is not None else B300MoEWorkspace(device=device)
    key = (device, shape.num_experts, shape.top_k, shape.hidden_size, shape.intermediate_size)
    tokens = shape.num_tokens
    with active._lock:
        b = active._layer_binding
        # the same layout and stream as the last time, and no capture: nothing to reserve
        repeated = (b is not None and b.key == key and b.allocations == active._allocations
                    and tokens <= b.tokens and active._last_stream == b.stream_ptr
                    and torch._C._cuda_getCurrentRawStream(device.index) == b.stream_ptr
                    and not torch._C._cuda_isCurrentStreamCapturing())
        if repeated:
            active._reuses += 1
            active._last_reused = True
            active._last_shape = (tokens, shape.num_experts, shape.top_k, shape.hidden_size,
                                  shape.intermediate_size)
        else:
            _resolve_native_backend("b200_bf16" if scales is None else "b200_fp8", hidden_states,
                                    router_weight, gate_up, down, shape)
            b = _bind(active, key, hidden_states, gate_up, down, shape)
        output = out if out is not None else torch.empty_like(hidden_states)
        ids = weights = None
        if return_routing:
            ids = torch.empty(tokens, shape.top_k, dtype=torch.int64, device=device)
            weights = torch.empty(tokens, shape.top_k, device=device)
        args = b.args
        args.hidden_states = hidden_states.data_ptr()
        args.gate_up_weight, args.down_weight = gate_up.data_ptr(), down.data_ptr()
        args.num_tokens = tokens
        args.output = output.data_ptr()
        if scales is None:
            args.flags = 0
        else:
            args.flags = _lib.FLAG_FP8_WEIGHTS
            args.gate_up_scale, args.down_scale = scales[0].data_ptr(), scales[1].data_ptr()
        call = (b.ref, router_weight.data_ptr(), router_weight.dtype is torch.float32,
                None if ids is None else ids.data_ptr(),
                None if weights is None else weights.data_ptr(),
                torch._C._cuda_getCurrentRawStream(device.index))
        fn = _lib.load().b200moe_layer
        if torch._C._cuda_getDevice() == device.index:
            code = fn(*call)
        else:
            with torch.cuda.device(device):
                code = fn(*call)
        if code:
            _lib.check(code, "b200moe_layer")
        if repeated:
            active._event.record(b.stream)
        else:
            active._record_use()
        if check_status:
            active.raise_for_status()
    return (output, ids, weights) if return_routing else output


def _check_options(hidden_states, out, return_routing, check_status) -> None:
    if not isinstance(return_routing, bool):
        raise TypeError("return_routing must be a bool")
    if not isinstance(check_status, bool):
        raise TypeError("check_status must be a bool")
    if out is not None and isinstance(hidden_states, torch.Tensor):
        _check_out(out, hidden_states)
        if out.device != hidden_states.device:
            raise ValueError("out must be on the inputs' device")


def b300_moe_layer(
    hidden_states: torch.Tensor,
    router_weight: torch.Tensor,
    gate_up_weight: torch.Tensor,
    down_weight: torch.Tensor,
    *,
    num_experts: int,
    top_k: int,
    workspace: B300MoEWorkspace | None = None,
    return_routing: bool = False,
    check_status: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Router, top-k, experts and weighted sum of at most eight tokens, in one kernel.

    ``hidden_states`` [T,H] BF16 with T <= 8 and H <= 8192, ``router_weight`` [E,H] BF16 or FP32,
    ``gate_up_weight`` [E,2I,H] (gate rows first) and ``down_weight`` [E,H,I] BF16; H and I
    multiples of 8; all contiguous on one CUDA device of compute capability 10.0.

    Every token goes to the ``top_k`` experts with the largest logits
    ``hidden_states @ router_weight.T`` (lower id first among equal ones) with the softmax over
    those logits as weights, as :func:`topk_routing` on FP32 logits chooses them; the weights
    are used unrounded.  ``return_routing=True`` also returns ``(ids [T,K] int64,
    weights [T,K] float32)``.  ``workspace``, ``check_status`` and ``out`` as in
    :func:`b300_moe_forward`, except that ``out`` has to be on the device; it may be the hidden
    states themselves, which every block has read before the first row is stored.  A workspace
    serves one call at a time: eager calls on several streams it orders itself, replays of
    captured calls (and eager calls beside them) are ordered by the caller.

    Against the router's product, :func:`topk_routing` and :func:`b300_moe_forward` in one graph
    this is 1.03 to 1.8 times as fast for one token and about the same for eight (H = 2048 with 128
    experts of 768: 25 against 45 us, and 98 against 98 us); outside a graph it also takes one
    call's host time instead of three.  Pass a workspace that is kept: a call without one
    allocates the buffers of the whole forward each time.
    """

    _check_options(hidden_states, out, return_routing, check_status)
    shape = _validate(hidden_states, router_weight, gate_up_weight, down_weight, None,
                      num_experts, top_k, torch.bfloat16, 8)
    return _run(hidden_states, router_weight, gate_up_weight, down_weight, None, shape, workspace,
                return_routing, check_status, out)


def b300_moe_layer_fp8(
    hidden_states: torch.Tensor,
    router_weight: torch.Tensor,
    weights: Fp8ExpertWeights,
    *,
    num_experts: int,
    top_k: int,
    workspace: B300MoEWorkspace | None = None,
    return_routing: bool = False,
    check_status: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`b300_moe_layer` with the E4M3 expert weights of
    :func:`quantize_expert_weights_fp8`; H and I multiples of 16.

    Activations between the two products keep 11 significant bits (twelve in
    :func:`b300_moe_forward_fp8`), scaled by the largest of their row; elements of a token's row
    below 2^-27 of its largest lose some of their eight.  One token is 1.1 to 1.5
    times as fast as through the router's product, :func:`topk_routing` and
    :func:`b300_moe_forward_fp8` in one graph; from three tokens on with large experts those three
    are faster (H = I = 2880, 32 experts, three tokens: 103 against 107 us; H = 4096, I = 14336,
    8 experts, eight tokens: 230 against 246 us)."""

    _check_options(hidden_states, out, return_routing, check_status)
    if not isinstance(weights, Fp8ExpertWeights):
        raise TypeError("weights must be an Fp8ExpertWeights")
    scales = (weights.gate_up_scale, weights.down_scale)
    shape = _validate(hidden_states, router_weight, weights.gate_up_q, weights.down_q, scales,
                      num_experts, top_k, torch.uint8, 16)
    return _run(hidden_states, router_weight, weights.gate_up_q, weights.down_q, scales, shape,
                workspace, return_routing, check_status, out)
