"""Experts with microscaled 4-bit weights AND activations (w4a4).

    out[m] = s * sum_k w[m, k] * W2[e] . Q2(act(W1[e] . Q1(x[m]))),   e = topk_ids[m, k]

Q1 and Q2 are ``fp4.fp4_quant`` in the weights' format (nvfp4 or mxfp4); between them everything is fp32.
Behind GEMM 2 every route's weighted row is rounded to the output type, as in ``fused_experts``, and the sum over
a token's routes is fp32 again.  Against 64 bits the layer is off by 0.0024 of the result's norm in bf16, of which
0.0017 is the result's own rounding; with fp32 rows (``output_dtype=torch.float32`` has them) the rest would
go, and these rows' bytes double: 720 us instead of 566 for 1500 tokens of 64 experts of 7168 x 2048, 327
instead of 301 for 1024 of 128 of 4096 x 1536, 291 instead of 287 for 333.
Seven launches (eight where the sort of many routes takes two): quantise the rows, sort, copy the rows' codes into
sorted order, lay out the scales for the tensor cores, GEMM 1 (quantises the activation in its epilogue), GEMM 2
(router weight in its epilogue), sum over a token's routes.  Products run on the tensor
cores' 4-bit block-scaled kind, four times the rate of 16-bit ones, and read half the bytes of w4a8.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi
from ..fp4 import FORMATS, check_global_scale, format_of, fp4_quant
from . import ops
from .decode import check_weights, gated_activation

_FLOAT_OUT = (torch.float16, torch.bfloat16, torch.float32)


def fused_experts_fp4(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    w1_scale: torch.Tensor,
    w2_scale: torch.Tensor,
    *,
    w1_global_scale: Optional[torch.Tensor] = None,
    w2_global_scale: Optional[torch.Tensor] = None,
    a1_global_scale: Optional[torch.Tensor] = None,
    a2_global_scale: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    global_num_experts: int = -1,
    expert_map: Optional[torch.Tensor] = None,
    routed_scaling_factor: Optional[float] = 1.0,
    gemm1_alpha: Optional[float] = None,
    gemm1_limit: Optional[float] = None,
    activation_situ_beta: Optional[float] = None,
    activation_situ_linear_beta: Optional[float] = None,
    output_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """Fused experts in w4a4 with caller-provided top-k routing; returns [tokens, model_dim].

    hidden_states [tokens, hidden] bf16 or fp16; w1 [E, 2*inter, hidden/2] (gate rows, then up rows) and
    w2 [E, model_dim, inter/2] packed codes with scales [E, rows, columns/block] (float8_e4m3fn: nvfp4,
    uint8: mxfp4).  nvfp4 only, each optional: ``w*_global_scale`` [E] on the weights, ``a*_global_scale``
    [1] on the activations in front of GEMM 1 and 2.  Routes whose id (read as int32) is out of range or not
    local under ``expert_map`` (one entry per expert, of any integer type) add nothing.  hidden and inter are multiples of 64 (nvfp4) or 128 (mxfp4), model_dim of
    16 bytes' worth of results."""
    if not hidden_states.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if hidden_states.dim() != 2 or hidden_states.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("hidden_states must be [tokens, hidden] in bf16 or fp16")
    m, hidden = hidden_states.shape
    dev = hidden_states.device
    if w1_scale is None or w2_scale is None:
        raise ValueError("w4a4 experts need w1_scale and w2_scale")
    fmt = format_of(w1_scale)
    code, block, scale_dtype = FORMATS[fmt]
    shape = lambda e, n, k: (e, n, k // block)  # noqa: E731
    e, inter, model_dim = check_weights(fmt, w1, w2, w1_scale, w2_scale, hidden, torch.uint8, scale_dtype, 2,
                                        shape, shape, dev)
    if hidden % (4 * block) or inter % (4 * block):
        raise NotImplementedError(f"hidden size {hidden} and intermediate size {inter} must be multiples of "
                                  f"{4 * block} ({fmt})")
    if topk_ids.dim() != 2 or topk_weights.shape != topk_ids.shape or topk_ids.shape[0] != m:
        raise ValueError("topk_weights and topk_ids must both be [tokens, topk]")
    for name, t in (("topk_weights", topk_weights), ("topk_ids", topk_ids), ("expert_map", expert_map)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, hidden_states on {dev}")
    if expert_map is not None and expert_map.dim() != 1:
        raise ValueError("expert_map must be one row of entries")
    act, alpha, limit = gated_activation(activation, gemm1_alpha, gemm1_limit, activation_situ_beta,
                                         activation_situ_linear_beta)
    out_dtype = hidden_states.dtype if output_dtype is None else output_dtype
    if out_dtype not in _FLOAT_OUT:
        raise ValueError("output_dtype must be bf16, fp16 or fp32")
    if (model_dim * out_dtype.itemsize) % 16:
        raise NotImplementedError(f"output size {model_dim} x {out_dtype.itemsize} B is not a multiple of "
                                  f"16 bytes: not built in boltops_b200")
    g1, g2, a1, a2 = (check_global_scale(name, t, fmt, n, dev) for name, t, n in (
        ("w1_global_scale", w1_global_scale, e), ("w2_global_scale", w2_global_scale, e),
        ("a1_global_scale", a1_global_scale, 1), ("a2_global_scale", a2_global_scale, 1)))
    if global_num_experts == -1:
        global_num_experts = expert_map.numel() if expert_map is not None else e
    if expert_map is None and global_num_experts != e:
        raise ValueError(f"{global_num_experts} experts, weights of {e}: an expert_map has to say which are local")
    if expert_map is not None and expert_map.numel() != global_num_experts:
        raise ValueError("expert_map must have one entry per expert")
    topk = topk_ids.shape[1]
    out = torch.empty((m, model_dim), dtype=out_dtype, device=dev)
    if m == 0 or topk == 0:
        return out.zero_()
    scale = 1.0 if routed_scaling_factor is None else float(routed_scaling_factor)
    w1, w2, w1_scale, w2_scale = (ops.aligned(t) for t in (w1, w2, w1_scale, w2_scale))
    mask = None
    if expert_map is not None:
        local = (expert_map >= 0) & (expert_map < e)
        expert_map, mask = torch.where(local, expert_map, -1), local.to(torch.int32)
    ids_all, wts_all = topk_ids.to(torch.int32), topk_weights.to(torch.float32)
    lib = _cabi.load()
    from .layer import _chunk_size
    chunk = _chunk_size()
    for begin in range(0, m, chunk):
        end = min(begin + chunk, m)
        rows = end - begin
        codes, scales = fp4_quant(hidden_states[begin:end], fmt, a1)
        route_pos = torch.empty((rows, topk), dtype=torch.int32, device=dev)
        sorted_ids, sorted_w, expert_ids, num_valid, _, _ = ops.moe_sorting_ck(
            ids_all[begin:end], wts_all[begin:end], global_num_experts, None, None, ops.SORT_UNIT, mask,
            alloc_moe_buf=False, route_pos=route_pos)
        if expert_map is not None:
            expert_ids = ops.relabel_tiles(expert_ids, expert_map)
        cap = sorted_ids.shape[0]
        codes, _ = ops.gather_rows(codes, sorted_ids, num_valid, cap)
        act_codes = torch.empty((cap, inter // 2), dtype=torch.uint8, device=dev)
        # the scales of all four operands in the tensor core's tiles; those of the activation come
        # out of GEMM 1 like that
        sizes = (cap * hidden // block, e * ops.ceil_to(inter, 64) * 2 * hidden // block,
                 e * ops.ceil_to(model_dim, 128) * inter // block, cap * inter // block)
        tiles = torch.empty(sum(sizes), dtype=torch.uint8, device=dev)
        at = [tiles.data_ptr() + sum(sizes[:i]) for i in range(4)]
        lay = _cabi.Fp4TileArgs()
        lay.jobs, lay.num_tokens, lay.capacity = 3, rows, cap
        lay.sorted_ids, lay.expert_ids = sorted_ids.data_ptr(), expert_ids.data_ptr()
        lay.num_valid_ids = num_valid.data_ptr()
        lay.job[0] = (scales.data_ptr(), at[0], rows, hidden // block, 1, 0, 1)
        lay.job[1] = (w1_scale.data_ptr(), at[1], 2 * inter, hidden // block, e, inter, 0)
        lay.job[2] = (w2_scale.data_ptr(), at[2], model_dim, inter // block, e, 0, 0)
        # (16-bit: a rounding per route, and half the bytes of this array; figures at the top)
        rows_out = torch.empty((cap, model_dim), dtype=out_dtype, device=dev)
        args = _cabi.Fp4GemmArgs()
        args.format, args.num_experts, args.capacity, args.num_tokens = code, e, cap, rows
        args.sorted_ids, args.sorted_expert_ids = sorted_ids.data_ptr(), expert_ids.data_ptr()
        args.num_valid_ids = num_valid.data_ptr()
        args.status = ops.device_status(dev).data_ptr()
        args.sm_count = ops.gemm_sm_count(dev)
        stream = _cabi.stream_of(hidden_states)
        with _cabi.on_device(dev):
            _cabi.check(lib.bolt_fp4_tile_scales(lay, stream))
            args.epilogue = _cabi.EPI_SILU_MUL_QUANT
            args.rows, args.n, args.k = cap, 2 * inter, hidden
            args.a, args.a_tiles, args.b, args.b_tiles = codes.data_ptr(), at[0], w1.data_ptr(), at[1]
            args.a_global, args.b_global, args.c_global = _cabi.ptr(a1), _cabi.ptr(g1), _cabi.ptr(a2)
            args.c, args.c_scale = act_codes.data_ptr(), at[3]
            args.activation, args.act_alpha, args.act_limit = act, alpha, limit
            _cabi.check(lib.bolt_fp4_gemm(args, stream))
            args.epilogue = _cabi.EPI_STORE
            args.rows, args.n, args.k = cap, model_dim, inter
            args.a, args.a_tiles, args.b, args.b_tiles = act_codes.data_ptr(), at[3], w2.data_ptr(), at[2]
            args.a_global, args.b_global, args.c_global = _cabi.ptr(a2), _cabi.ptr(g2), None
            args.c, args.c_dtype, args.c_ld = rows_out.data_ptr(), _cabi.dtype_code(out_dtype), model_dim
            args.sorted_weights = sorted_w.data_ptr()
            _cabi.check(lib.bolt_fp4_gemm(args, stream))
        ops._count(3)
        ops.gather_sum(rows_out, route_pos, out[begin:end], scale)
    return out


__all__ = ["fused_experts_fp4"]
