"""A whole expert layer for a few decoding tokens, in two kernels.

``fused_experts`` is built for any number of tokens: it sorts the routes, places rows, multiplies and
combines in five to seven launches.  With one or a few tokens these launches and the half-empty tiles are
a large part of the time.  The forms here take 1 to 32 tokens and leave out everything but
the weights: routing is a bit mask per expert that every block of the kernel builds for itself, the
first kernel does gate, up and activation, the second the down projection and the sum over a token's
experts, and it fills its weight rings while the first one finishes.  (8-bit rows and activations whose codes a
block cannot keep beside its rings, as a rule above eight tokens, are quantised by a kernel of their own in front
of either.  4-bit rows that do not fit in shared memory together, 32 tokens above about 5000 hidden columns, go
in two parts or more, which read the experts that they share again.)

Which layer to call.  Every eight tokens cost a pass of small matrix instructions over widened weights, where
the tensor-core tiles of ``fused_experts`` take up to 128 rows at once, so the forms here are for one to four
tokens.  Kernels alone, us, here / there, routes at random:

    tokens                           1          2          4          8         16         32
    Mixtral, bf16                114/154    194/219    324/358    411/412    511/445    780/448
    Mixtral, fp8 block            72/128    112/157    181/184    255/225    376/235    630/241
    Qwen3-30B, bf16               27/40      41/46      68/69     100/98     165/140    280/179
    Qwen3-30B, int8 channel       28/39      40/44      65/60      94/79     141/105    215/131
    Qwen3-235B, fp8 block         55/55      68/80     113/116    181/172    340/262    539/341
    DeepSeek-V3, fp8 block        74/84     132/140    241/239    473/410    941/703   1735/1124
    DeepSeek-V3, fp8 channel      78/91     136/147    238/248    442/433    823/722   1518/1139
    DeepSeek-V3, int8 block       89/85     151/140    277/237    528/405   1088/706   2048/1109
    DeepSeek-V3, int8 channel     90/91     153/147    275/250    499/435    937/728   1745/1137
    8 experts of 1024 x 512, bf16  9/26      11/26      13/26      17/26      26/26      26/27

Called one by one from Python, a caller that waits for its host gains about 10 us more here.  4-bit experts
against ``fused_experts_fp4``, 128 experts of 2048 x 768, eight a token: nvfp4 51/63 us at 4 tokens, 67/76 at 8,
116/93 at 16, 202/110 at 32; mxfp4 28/37 at one, 58/54 at 4, 165/82 at 16; that layer costs at least 130 us
on the host, this one 33.

Same recipes as ``fused_experts`` (16-bit, fp8 and int8 w8a8 block-scaled and per-channel) and
``fused_experts_fp4`` (w4a4), with fewer roundings: GEMM 1 and the routes' results stay in fp32, quantised
experts quantise the fp32 activation, 16-bit experts round it to the weights' type.  The w8a8 scales are
amax times the rounded 1/448 or 1/127, where ``fused_experts`` divides: they may differ in the last bit,
and with them the codes of values that lie on the border of two.  Sums of int8 products are fp32 here and can
round from 2^24 on; ``fused_experts`` keeps them in 32-bit integers.
"""
from __future__ import annotations

import functools
from typing import List, Optional

import torch

from .. import _cabi
from ..fp4 import FORMATS, check_global_scale, format_of
from . import ops
from .activation import normalize_moe_activation, resolve_kernel

MAX_TOKENS = 32
_FLOAT_OUT = (torch.float16, torch.bfloat16, torch.float32)
_16BIT = (torch.bfloat16, torch.float16)


@functools.lru_cache(maxsize=64)
def gated_activation(activation, gemm1_alpha, gemm1_limit, situ_beta, situ_linear_beta):
    """(kernel activation, alpha, limit) of a gated activation on [gate | up] rows."""
    activation, is_gated = normalize_moe_activation("silu" if activation is None else activation)
    if not is_gated or activation == "swigluoai":
        raise NotImplementedError("gated activations on [gate | up] rows only")
    return resolve_kernel(activation, True, gemm1_alpha, gemm1_limit, situ_beta, situ_linear_beta)


def _kind(w1, w1_scale, use_fp8_w8a8, use_int8_w8a8, use_fp4_w4a4, per_channel_quant, block_shape) -> int:
    if use_fp8_w8a8 + use_int8_w8a8 + use_fp4_w4a4 > 1:
        raise ValueError("the quantisation flags exclude each other")
    if use_fp4_w4a4:
        if per_channel_quant:
            raise ValueError("w4a4 experts have block scales, per_channel_quant does not apply")
        fmt = format_of(w1_scale)
        if block_shape is not None and list(block_shape) != [1, FORMATS[fmt][1]]:
            raise ValueError(f"{fmt} block_shape must be [1, {FORMATS[fmt][1]}]")
        return _cabi.DECODE_NVFP4 if fmt == "nvfp4" else _cabi.DECODE_MXFP4
    if use_fp8_w8a8 or use_int8_w8a8:
        if not per_channel_quant:
            if block_shape is None:
                raise NotImplementedError("per-tensor quantised experts are not built in boltops_b200")
            if list(block_shape) != [128, 128]:
                raise NotImplementedError("only block_shape [128, 128] is built in boltops_b200")
            return _cabi.DECODE_FP8_BLOCK if use_fp8_w8a8 else _cabi.DECODE_INT8_BLOCK
        return _cabi.DECODE_FP8_CHANNEL if use_fp8_w8a8 else _cabi.DECODE_INT8_CHANNEL
    if w1.dtype == torch.bfloat16:
        return _cabi.DECODE_BF16
    if w1.dtype == torch.float16:
        return _cabi.DECODE_F16
    raise NotImplementedError(f"unquantised experts in {w1.dtype} are not built in boltops_b200")


def check_weights(kind_name, w1, w2, w1_scale, w2_scale, hidden, w_dtype, scale_dtype, pack, scale1, scale2,
                  dev):
    """Shapes, types and devices of the weights and their scales; returns (experts, inter, model_dim)."""
    if w1.dim() != 3 or w2.dim() != 3:
        raise ValueError("w1 and w2 are [experts, rows, columns]")
    e, n1, k1 = w1.shape
    model_dim, inter = w2.shape[1], n1 // 2
    if n1 % 2 or k1 * pack != hidden:
        raise ValueError(f"w1 {tuple(w1.shape)} does not fit {hidden} hidden columns ({kind_name})")
    if w2.shape[0] != e or w2.shape[2] * pack != inter:
        raise ValueError(f"w2 {tuple(w2.shape)} does not fit w1 {tuple(w1.shape)} ({kind_name})")
    if w1.dtype != w_dtype or w2.dtype != w_dtype:
        raise TypeError(f"{kind_name} weights are {w_dtype}")
    for name, t in (("w1", w1), ("w2", w2), ("w1_scale", w1_scale), ("w2_scale", w2_scale)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, hidden_states on {dev}")
    if scale_dtype is not None:
        for name, s, shape in (("w1_scale", w1_scale, scale1(e, n1, hidden)),
                               ("w2_scale", w2_scale, scale2(e, model_dim, inter))):
            if s is None:
                raise ValueError(f"{name} is required ({kind_name})")
            # (dimensions of one value apart: per-channel scales come as [E, N] or [E, N, 1])
            if _long_dims(s.shape) != _long_dims(shape):
                raise ValueError(f"{name} {tuple(s.shape)}: expected {shape} ({kind_name})")
            if scale_dtype != torch.float32 and s.dtype != scale_dtype:
                raise TypeError(f"{name} must be {scale_dtype} ({kind_name})")
    return e, inter, model_dim


def _long_dims(shape):
    return [n for n in shape if n != 1]


def _decode(hidden_states, w1, w2, topk_weights, topk_ids, gating, topk, renormalize, is_softmax, *,
            use_fp8_w8a8, use_int8_w8a8, use_fp4_w4a4, per_channel_quant, block_shape, w1_scale, w2_scale,
            w1_global_scale, w2_global_scale, a1_global_scale, a2_global_scale, activation, gemm1_alpha,
            gemm1_limit, activation_situ_beta, activation_situ_linear_beta, global_num_experts, expert_map,
            routed_scaling_factor, output_dtype, out):
    if not hidden_states.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if hidden_states.dim() != 2 or hidden_states.dtype not in _16BIT:
        raise ValueError("hidden_states must be [tokens, hidden] in bf16 or fp16")
    m, hidden = hidden_states.shape
    if m > MAX_TOKENS:
        raise NotImplementedError(f"{m} tokens: this form takes at most {MAX_TOKENS}, fused_experts any number")
    if (use_fp4_w4a4 or use_fp8_w8a8 or use_int8_w8a8) and (w1_scale is None or w2_scale is None):
        raise ValueError("quantised experts need w1_scale and w2_scale")
    kind = _kind(w1, w1_scale, use_fp8_w8a8, use_int8_w8a8, use_fp4_w4a4, per_channel_quant, block_shape)
    dev = hidden_states.device
    fp4 = kind in (_cabi.DECODE_NVFP4, _cabi.DECODE_MXFP4)
    if fp4:
        fmt = format_of(w1_scale)
        block = FORMATS[fmt][1]
        e, inter, model_dim = check_weights(
            fmt, w1, w2, w1_scale, w2_scale, hidden, torch.uint8, FORMATS[fmt][2], 2,
            *[lambda e, n, k: (e, n, k // block)] * 2, dev)
    else:
        fmt = None
        if any(t is not None for t in (w1_global_scale, w2_global_scale, a1_global_scale, a2_global_scale)):
            raise ValueError("scales of whole tensors belong to use_fp4_w4a4")
        if use_fp8_w8a8 or use_int8_w8a8:
            w_dtype = torch.float8_e4m3fn if use_fp8_w8a8 else torch.int8
            shape = (lambda e, n, k: (e, n)) if per_channel_quant else \
                (lambda e, n, k: (e, n // 128, k // 128))
            if not per_channel_quant and (hidden % 128 or w1.shape[1] % 256 or w2.shape[1] % 128):
                raise NotImplementedError("block-scaled experts need sizes in multiples of 128")
            for name, s in (("w1_scale", w1_scale), ("w2_scale", w2_scale)):
                if s.dtype not in _FLOAT_OUT:
                    raise ValueError(f"{name} must be a decoded floating-point multiplier")
            e, inter, model_dim = check_weights("w8a8", w1, w2, w1_scale, w2_scale, hidden, w_dtype,
                                                torch.float32, 1, shape, shape, dev)
            w1_scale, w2_scale = w1_scale.float(), w2_scale.float()
        else:
            if w1_scale is not None or w2_scale is not None:
                raise ValueError("unquantised experts take no scales")
            e, inter, model_dim = check_weights("16-bit", w1, w2, None, None, hidden, hidden_states.dtype,
                                                None, 1, None, None, dev)
    step = {_cabi.DECODE_NVFP4: 64, _cabi.DECODE_MXFP4: 128}.get(kind, 128 if not per_channel_quant else 16) \
        if (fp4 or use_fp8_w8a8 or use_int8_w8a8) else 8
    if hidden % step or inter % step:
        raise NotImplementedError(f"hidden size {hidden} and intermediate size {inter} must be multiples "
                                  f"of {step} here")
    if e == 0 or e > 1024:
        raise NotImplementedError("1 to 1024 local experts")
    if expert_map is not None:
        if expert_map.dim() != 1 or expert_map.device != dev:
            raise ValueError(f"expert_map must be one row of entries on {dev}")
        if global_num_experts == -1:
            global_num_experts = expert_map.numel()
        if expert_map.numel() < global_num_experts:
            raise ValueError("expert_map has fewer entries than there are experts")
        expert_map = expert_map.to(torch.int32).contiguous()
    elif global_num_experts == -1:
        global_num_experts = e
    act, alpha, limit = gated_activation(activation, gemm1_alpha, gemm1_limit, activation_situ_beta,
                                         activation_situ_linear_beta)
    out_dtype = hidden_states.dtype if output_dtype is None else output_dtype
    if out_dtype not in _FLOAT_OUT:
        raise ValueError("output_dtype must be bf16, fp16 or fp32")
    if out is None:
        out = torch.empty((m, model_dim), dtype=out_dtype, device=dev)
    elif tuple(out.shape) != (m, model_dim) or out.dtype != out_dtype or out.device != dev \
            or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {out_dtype} [{m}, {model_dim}] on {dev}")

    keep = []
    if gating is not None:
        if gating.dim() != 2 or tuple(gating.shape) != (m, global_num_experts) or gating.device != dev:
            raise ValueError(f"gating_output must be [{m}, {global_num_experts}] on {dev}")
        if gating.dtype not in _FLOAT_OUT:
            raise ValueError("gating_output must be bf16, fp16 or fp32")
        if global_num_experts > 1024:
            raise NotImplementedError("the router takes at most 1024 experts")
        if not 1 <= topk <= min(32, global_num_experts):
            raise ValueError(f"topk {topk} out of range")
        gating = gating.contiguous()
        routing = (None, None, gating.data_ptr(), _cabi.dtype_code(gating.dtype), int(renormalize),
                   int(is_softmax))
    else:
        if topk_ids.dim() != 2 or topk_weights.shape != topk_ids.shape or topk_ids.shape[0] != m:
            raise ValueError("topk_weights and topk_ids must both be [tokens, topk]")
        for name, t in (("topk_weights", topk_weights), ("topk_ids", topk_ids)):
            if t.device != dev:
                raise ValueError(f"{name} is on {t.device}, hidden_states on {dev}")
        topk = topk_ids.shape[1]
        if not 1 <= topk <= 32:
            raise ValueError(f"topk {topk} out of range")
        ids = topk_ids.to(torch.int32).contiguous()
        wts = topk_weights.to(torch.float32).contiguous()
        routing = (wts.data_ptr(), ids.data_ptr(), None, 0, 0, 0)
    if m == 0:
        return out

    x = ops.aligned(hidden_states)
    w1, w2 = ops.aligned(w1), ops.aligned(w2)
    s1 = s2 = None
    if w1_scale is not None:
        w1_scale, w2_scale = ops.aligned(w1_scale), ops.aligned(w2_scale)
        s1, s2 = w1_scale.data_ptr(), w2_scale.data_ptr()
    whole = (None, None, None, None)
    if fp4:
        keep = [check_global_scale(name, t, fmt, n, dev) for name, t, n in (
            ("w1_global_scale", w1_global_scale, e), ("w2_global_scale", w2_global_scale, e),
            ("a1_global_scale", a1_global_scale, 1), ("a2_global_scale", a2_global_scale, 1))]
        whole = tuple(_cabi.ptr(t) for t in keep)
    lib = _cabi.load()
    args = _cabi.DecodeArgs(
        kind, _cabi.dtype_code(x.dtype), _cabi.dtype_code(out_dtype), m, topk, hidden, inter, model_dim, e,
        global_num_experts, x.data_ptr(), w1.data_ptr(), w2.data_ptr(), s1, s2, *whole, *routing,
        _cabi.ptr(expert_map), act, alpha, limit,
        1.0 if routed_scaling_factor is None else float(routed_scaling_factor), out.data_ptr(), None, 0,
        ops.device_status(dev).data_ptr(), ops.gemm_sm_count(dev))
    need = lib.bolt_moe_decode_workspace_bytes(args)
    if need == 0:
        _cabi.check(1)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    with _cabi.on_device(dev):
        status = lib.bolt_moe_decode(args, _cabi.stream_of(x))
        kernels = lib.bolt_moe_decode_kernel_count(args)
    if status == _cabi.BOLT_ERR_UNSUPPORTED:
        raise NotImplementedError(lib.bolt_last_error().decode(errors="replace"))
    _cabi.check(status)
    ops._count(kernels)
    return out


def fused_experts_decode(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    *,
    activation: Optional[str] = None,
    use_fp8_w8a8: bool = False,
    use_int8_w8a8: bool = False,
    use_fp4_w4a4: bool = False,
    per_channel_quant: bool = False,
    block_shape: Optional[List[int]] = None,
    w1_scale: Optional[torch.Tensor] = None,
    w2_scale: Optional[torch.Tensor] = None,
    w1_global_scale: Optional[torch.Tensor] = None,
    w2_global_scale: Optional[torch.Tensor] = None,
    a1_global_scale: Optional[torch.Tensor] = None,
    a2_global_scale: Optional[torch.Tensor] = None,
    global_num_experts: int = -1,
    expert_map: Optional[torch.Tensor] = None,
    routed_scaling_factor: Optional[float] = 1.0,
    gemm1_alpha: Optional[float] = None,
    gemm1_limit: Optional[float] = None,
    activation_situ_beta: Optional[float] = None,
    activation_situ_linear_beta: Optional[float] = None,
    output_dtype: Optional[torch.dtype] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``fused_experts`` for 1 to 32 tokens; meant for one to four, above which ``fused_experts`` is the faster
    layer for most weights (the module's docstring has the times).

    Arguments as there, without biases, ``is_gated`` (always), ``inplace`` (pass ``out=hidden_states``),
    ``apply_router_weight_on_input`` and ``no_combine``.
    ``use_fp4_w4a4``: weights and scales as ``fused_experts_fp4`` takes them.  Routes whose id (read as int32)
    is out of range or not local under ``expert_map`` add nothing; a token with none gives zeros; an expert
    that a token names twice counts with the sum of its weights.  ``out``: a contiguous buffer for
    the result.  Raises ``NotImplementedError`` above 32 tokens, for sizes that are not multiples of 8
    (16-bit), 16 (per-channel), 64 (nvfp4) or 128 (block-scaled, mxfp4)."""
    return _decode(hidden_states, w1, w2, topk_weights, topk_ids, None, 0, False, True,
                   use_fp8_w8a8=use_fp8_w8a8, use_int8_w8a8=use_int8_w8a8, use_fp4_w4a4=use_fp4_w4a4,
                   per_channel_quant=per_channel_quant, block_shape=block_shape, w1_scale=w1_scale,
                   w2_scale=w2_scale, w1_global_scale=w1_global_scale, w2_global_scale=w2_global_scale,
                   a1_global_scale=a1_global_scale, a2_global_scale=a2_global_scale,
                   activation=activation, gemm1_alpha=gemm1_alpha, gemm1_limit=gemm1_limit,
                   activation_situ_beta=activation_situ_beta,
                   activation_situ_linear_beta=activation_situ_linear_beta,
                   global_num_experts=global_num_experts, expert_map=expert_map,
                   routed_scaling_factor=routed_scaling_factor, output_dtype=output_dtype, out=out)


def fused_moe_decode(
    hidden_states: torch.Tensor,
    gating_output: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    topk: int,
    renormalize: bool,
    is_softmax: bool = True,
    *,
    activation: Optional[str] = None,
    use_fp8_w8a8: bool = False,
    use_int8_w8a8: bool = False,
    use_fp4_w4a4: bool = False,
    per_channel_quant: bool = False,
    block_shape: Optional[List[int]] = None,
    w1_scale: Optional[torch.Tensor] = None,
    w2_scale: Optional[torch.Tensor] = None,
    w1_global_scale: Optional[torch.Tensor] = None,
    w2_global_scale: Optional[torch.Tensor] = None,
    a1_global_scale: Optional[torch.Tensor] = None,
    a2_global_scale: Optional[torch.Tensor] = None,
    global_num_experts: int = -1,
    expert_map: Optional[torch.Tensor] = None,
    routed_scaling_factor: Optional[float] = 1.0,
    gemm1_alpha: Optional[float] = None,
    gemm1_limit: Optional[float] = None,
    activation_situ_beta: Optional[float] = None,
    activation_situ_linear_beta: Optional[float] = None,
    output_dtype: Optional[torch.dtype] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``fused_experts_decode`` from the router's logits [tokens, experts]: the top-k choice of
    ``routing.fused_topk`` (the same one, to the last bit) is made inside the layer's kernels."""
    return _decode(hidden_states, w1, w2, None, None, gating_output, topk, renormalize, is_softmax,
                   use_fp8_w8a8=use_fp8_w8a8, use_int8_w8a8=use_int8_w8a8, use_fp4_w4a4=use_fp4_w4a4,
                   per_channel_quant=per_channel_quant, block_shape=block_shape, w1_scale=w1_scale,
                   w2_scale=w2_scale, w1_global_scale=w1_global_scale, w2_global_scale=w2_global_scale,
                   a1_global_scale=a1_global_scale, a2_global_scale=a2_global_scale,
                   activation=activation, gemm1_alpha=gemm1_alpha, gemm1_limit=gemm1_limit,
                   activation_situ_beta=activation_situ_beta,
                   activation_situ_linear_beta=activation_situ_linear_beta,
                   global_num_experts=global_num_experts, expert_map=expert_map,
                   routed_scaling_factor=routed_scaling_factor, output_dtype=output_dtype, out=out)


__all__ = ["fused_experts_decode", "fused_moe_decode"]
