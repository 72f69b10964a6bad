"""Dense block-scaled GEMMs.

``gemm_a8w8_blockscale`` and its other names: 8-bit operands, on the grouped-GEMM kernel (one "expert").

Same call surface as the reference's ``gemm_a8w8_blockscale``
(boltops/gemm/gemm_a8w8_blockscale.py:10-70 in the reference project) and
``w8a8_triton_block_scaled_mm`` for the recipe the fused-MoE path uses: e4m3 or int8
operands, A scales per row and 128 K elements, B scales per 128x128 block.  It is the
op a DeepSeek-style layer calls next to ``fused_experts`` (shared experts, dense layers).

``gemm_a4w4``: microscaled 4-bit operands (``boltops_b200.fp4``).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _cabi
from .fp4 import FORMATS, format_of
from .fused_moe import ops


def gemm_a8w8_blockscale(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor,
                         w_scale: torch.Tensor, dtype: Optional[torch.dtype] = torch.bfloat16,
                         out: Optional[torch.Tensor] = None, config=None, backend=None):
    """``y[m, n] = sum_kb (x[m, kb] . w[n, kb]) * x_scale[m, kb] * w_scale[n//128, kb]``.

    x [M, K] and w [N, K] e4m3 or int8 (same dtype), x_scale [M, K/128], w_scale
    [N/128, K/128] floating point; K and N multiples of 128.  w and w_scale lie on x's device;
    x_scale and ``out`` may lie elsewhere and are copied.  ``config`` / ``backend`` are accepted
    for signature compatibility and ignored (one kernel, one schedule)."""
    if dtype is None:
        dtype = torch.bfloat16
    if not x.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if x.dtype != w.dtype or x.dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError("x and w must both be float8_e4m3fn or int8")
    m, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k or k % 128 or n % 128:
        raise NotImplementedError("K and N must be multiples of 128 (1x128 / 128x128 scale recipe)")
    if tuple(x_scale.shape) != (m, k // 128) or tuple(w_scale.shape) != (n // 128, k // 128):
        raise ValueError("scale shapes do not match the 1x128 / 128x128 recipe")
    kind = _cabi.GEMM_FP8_BLOCK if x.dtype == torch.float8_e4m3fn else _cabi.GEMM_INT8_BLOCK
    dev = x.device
    # the kernels take addresses: none of another device may reach them
    for name, t in (("w", w), ("w_scale", w_scale)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, x on {dev}")
    if out is not None:
        assert out.shape == (m, n) and out.dtype == dtype and out.is_contiguous()
    elsewhere = out is not None and out.device != dev     # the result is copied there
    c = out if out is not None and not elsewhere else torch.empty((m, n), dtype=dtype, device=dev)
    if m == 0:
        return out if elsewhere else c
    # Two launches: the scales to group-major order (with the one "expert"'s tile labels), the GEMM.
    # Rows that only pad the last row tile exist nowhere: the tensor map reads them as zeros and
    # nothing is stored for them.
    x, w = x.contiguous(), w.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()       # the tensor map needs a 16-byte aligned base
    x_scale = x_scale.to(device=dev, dtype=torch.float32).contiguous()
    w_scale = w_scale.float().contiguous()
    cap = ops.ceil_to(m, 128)
    groups, tiles = k // 128, cap // 128
    ws = torch.empty(groups * cap + tiles + 1, dtype=torch.float32, device=dev)
    scale_t = ws.data_ptr()
    tile_ids = scale_t + 4 * groups * cap
    num_rows = tile_ids + 4 * tiles
    args = _cabi.GemmArgs()
    args.kind, args.epilogue = kind, _cabi.EPI_STORE
    args.capacity, args.n, args.k, args.num_experts = cap, n, k, 1
    args.a, args.b, args.c = x.data_ptr(), w.data_ptr(), c.data_ptr()
    args.dense_rows = m
    args.a_scale, args.a_scale_ld, args.b_scale = scale_t, cap, w_scale.data_ptr()
    args.c_dtype = args.mid_dtype = _cabi.dtype_code(dtype)
    args.c_ld, args.topk = n, 1
    args.sorted_expert_ids, args.num_valid_ids = tile_ids, num_rows
    args.status = ops.device_status(dev).data_ptr()
    args.sm_count = ops.gemm_sm_count(dev)
    lib = _cabi.load()
    stream = _cabi.stream_of(x)
    with _cabi.on_device(dev):
        _cabi.check(lib.bolt_dense_prep(x_scale.data_ptr(), m, groups, scale_t, cap, tile_ids,
                                        num_rows, stream))
        _cabi.check(lib.bolt_grouped_gemm(args, stream))
    ops._count(2)
    if elsewhere:
        return out.copy_(c)
    return c


def w8a8_block_scaled_mm(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor,
                         block_size: Sequence[int], output_dtype: torch.dtype = torch.float16):
    """vLLM/SGLang-style name of the same operation (B is [N, K], ``block_size`` [128, 128])."""
    if list(block_size) != [128, 128]:
        raise NotImplementedError("only block_size [128, 128] is built in boltops_b200")
    return gemm_a8w8_blockscale(A, B, As, Bs, dtype=output_dtype)


w8a8_triton_block_scaled_mm = w8a8_block_scaled_mm
w8a8_block_int8_matmul = w8a8_block_scaled_mm


# Which form a product of up to 32 rows takes.  The few-row form reads the weights once and computes on small
# matrix instructions, a column tile per eight rows, so its time grows with weights times row tiles; the tiled
# form has a launch more and whole 128-row tiles, whatever the rows.  Up to a product of weights and row tiles the
# former is ahead.  Kernels alone, us, few / tiled:
#   nvfp4   rows     1          8          16         24         32
#   4096 x 7168   8.2/22.8   8.5/22.8  10.5/22.8  14.2/22.8  16.0/22.9
#   7168 x 7168  13.4/23.3  13.9/23.5  17.6/23.5  25.9/23.6  29.7/23.6
#   8192 x 8192  14.8/25.7  15.5/25.7  19.7/25.9  28.7/25.9  33.2/25.9
#  16384 x 8192  24.2/34.0  26.6/32.4  35.4/33.0  54.1/33.2  62.1/29.1
#  28672 x 8192  38.9/43.6  43.1/41.7  58.7/41.2  91.0/39.7 105.6/39.7
#   mxfp4
#   4096 x 4096   7.4/15.6   7.8/15.6   9.8/15.7  13.2/15.8  15.0/15.8
#   4096 x 7168  10.8/20.8  11.1/20.9  14.1/21.0  19.8/21.0  22.5/21.0
#   7168 x 7168  17.8/21.3  19.0/21.3  25.1/21.5  36.5/21.4  41.6/21.5
#   8192 x 8192  19.8/23.5  21.6/23.4  28.7/23.5  39.6/23.7  44.9/23.7
#  16384 x 8192  35.9/31.3  40.6/29.7  54.6/29.9  76.3/29.1  87.7/24.6
# (a short reduction is best for the tiled form: mxfp4 7168 x 2048, 24 rows 14.2/11.9, where the few-row one
# still saves a caller that waits for its host a launch)
_FEW_ROWS = 32
_FEW_WORK = {"nvfp4": 128 << 20, "mxfp4": 64 << 20}


def _takes_few_rows(fmt: str, m: int, n: int, k: int) -> bool:
    return m <= _FEW_ROWS and n * k * ((m + 7) // 8) <= _FEW_WORK[fmt]


def gemm_a4w4(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
              alpha: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = torch.bfloat16,
              out: Optional[torch.Tensor] = None):
    """``y[m, n] = alpha * sum_k x[m, k] w[n, k]`` of 4-bit codes with block scales (``fp4.fp4_quant``).

    x [M, K/2] and w [N, K/2] packed codes, x_scale [M, K/block] and w_scale [N, K/block] of one format
    (float8_e4m3fn: nvfp4, blocks of 16, K a multiple of 64; uint8: mxfp4, blocks of 32, K a multiple
    of 128); M and N any.  ``alpha``: one fp32 value on the device, the product of both tensors' global
    scales.  Sums are fp32, rounded once to ``dtype`` (bf16, fp16 or fp32).  All tensors lie on x's
    device; ``out`` [M, N] has a dense last dimension."""
    if dtype is None:
        dtype = torch.bfloat16
    if not x.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"gemm_a4w4 gives bf16, fp16 or fp32, not {dtype}")
    if x.dtype != torch.uint8 or w.dtype != torch.uint8:
        raise TypeError("x and w must be packed 4-bit codes (uint8)")
    fmt = format_of(x_scale)
    if format_of(w_scale) != fmt:
        raise TypeError("x and w are of different 4-bit formats")
    code, block, _ = FORMATS[fmt]
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} must be [M, K/2] and [N, K/2]")
    m, n, k = x.shape[0], w.shape[0], 2 * x.shape[1]
    if tuple(x_scale.shape) != (m, k // block) or tuple(w_scale.shape) != (n, k // block):
        raise ValueError(f"scale shapes do not match blocks of {block} values")
    if k == 0 or k % (4 * block):
        raise NotImplementedError(f"K {k} must be a multiple of {4 * block} ({fmt})")
    dev = x.device
    if w.device != dev or x_scale.device != dev or w_scale.device != dev or \
            (alpha is not None and alpha.device != dev) or (out is not None and out.device != dev):
        for name, t in (("w", w), ("x_scale", x_scale), ("w_scale", w_scale), ("alpha", alpha), ("out", out)):
            if t is not None and t.device != dev:
                raise ValueError(f"{name} is on {t.device}, x on {dev}")
    if alpha is not None and (alpha.numel() != 1 or alpha.dtype != torch.float32):
        raise ValueError("alpha must be one float32 value")
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
    elif tuple(out.shape) != (m, n) or out.dtype != dtype or (n > 1 and out.stride(1) != 1) or \
            (m > 1 and out.stride(0) < n):
        raise ValueError(f"out must be [{m}, {n}] in {dtype} with a dense last dimension")
    if m == 0 or n == 0:
        return out
    x, w = ops.aligned(x), ops.aligned(w)
    x_scale, w_scale = ops.aligned(x_scale), ops.aligned(w_scale)
    lib = _cabi.load()
    stream = _cabi.stream_of(x)
    out_ld = out.stride(0) if m > 1 else n
    if _takes_few_rows(fmt, m, n, k):
        few = _cabi.Fp4FewArgs(code, m, n, k, x.data_ptr(), x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(),
                               _cabi.ptr(alpha), out.data_ptr(), _cabi.dtype_code(dtype), out_ld,
                               ops.device_status(dev).data_ptr(), ops.gemm_sm_count(dev))
        _cabi.call(dev, lib.bolt_fp4_gemm_few, few, stream)
        ops._count()
        return out
    args = _cabi.Fp4GemmArgs()
    args.format, args.epilogue = code, _cabi.EPI_STORE
    args.rows, args.n, args.k, args.num_experts = m, n, k, 1
    # the scales in the tensor core's tiles: whole 128-row blocks of both operands
    row_bytes = k // block
    blocks_m = (m + 127) // 128
    tiles = torch.empty((blocks_m + (n + 127) // 128) * 128 * row_bytes, dtype=torch.uint8, device=dev)
    lay = _cabi.Fp4TileArgs()
    lay.jobs = 2
    lay.job[0] = (x_scale.data_ptr(), tiles.data_ptr(), m, row_bytes, 1, 0, 0)
    lay.job[1] = (w_scale.data_ptr(), tiles.data_ptr() + blocks_m * 128 * row_bytes, n, row_bytes, 1, 0, 0)
    args.a, args.b = x.data_ptr(), w.data_ptr()
    args.a_tiles, args.b_tiles = lay.job[0].dst, lay.job[1].dst
    args.alpha = _cabi.ptr(alpha)
    args.c, args.c_dtype, args.c_ld = out.data_ptr(), _cabi.dtype_code(dtype), out_ld
    args.status = ops.device_status(dev).data_ptr()
    args.sm_count = ops.gemm_sm_count(dev)
    _cabi.call(dev, lib.bolt_fp4_tile_scales, lay, stream)
    _cabi.call(dev, lib.bolt_fp4_gemm, args, stream)
    ops._count(2)
    return out
