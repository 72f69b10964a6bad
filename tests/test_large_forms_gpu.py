"""The 4-bit products and the few-token layer in the forms that large operands select.

The forms are chosen by sizes: the few-token layer takes blocks of sixteen warps above 256 KB of
weights a block (1 to 8 tokens), the tiled 4-bit product takes 256 columns a tile where they cost no wave and
gives a block several tiles.  The definition in 64 bits runs on the GPU here."""
import contextlib

import pytest
import torch

import fp4_reference as R
from boltops_b200.fused_moe import fused_experts_decode, fused_experts_fp4, ops
from boltops_b200.gemm import gemm_a4w4
from test_decode_gpu import FLAGS

pytestmark = pytest.mark.gpu
FORMATS = ["nvfp4", "mxfp4"]


@pytest.fixture(autouse=True)
def on_gpu(monkeypatch):
    monkeypatch.setattr(R, "E2M1", R.E2M1.cuda())
    with torch.device("cuda"):
        yield
    ops.set_gemm_sm_reserve(0)


@contextlib.contextmanager
def blocks(count):
    """Products and the few-token layer on `count` SMs (None: all)."""
    total = torch.cuda.get_device_properties(0).multi_processor_count
    ops.set_gemm_sm_reserve(0 if count is None else total - count)
    try:
        yield
    finally:
        ops.set_gemm_sm_reserve(0)


def compare(got, want, bound):
    ops.check_device_status(got.device)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4].tolist(), off.max().item(),
                           (off / bound.clamp_min(1e-300)).max().item())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- the dense product -------------------------------------------------------------------------
# rows, columns, blocks of K, SMs.  On 148 SMs: 256 columns a tile, one tile a block; 256 columns, several tiles a
# block and a last group of row tiles that is not full; 128 columns, several tiles a block.  On few SMs: a
# dozen tiles a block and more, both widths.
DENSE = [(2200, 1401, 3, None), (2437, 3000, 2, None), (3300, 4600, 1, None), (1270, 3801, 2, None),
         (700, 900, 9, 3), (333, 131, 5, 1), (4500, 260, 2, 7)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,kblocks,sms", DENSE)
def test_dense_product(fmt, m, n, kblocks, sms):
    k = kblocks * 4 * R.BLOCK[fmt]
    dtype = (torch.bfloat16, torch.float32, torch.float16)[(m + n) % 3]
    x, xs, xv = R.fp4_quant(fmt, torch.randn(m, k, generator=gen(1)))
    w, ws, wv = R.fp4_quant(fmt, torch.randn(n, k, generator=gen(2)) * 0.05)
    if fmt == "nvfp4":
        xs, ws = xs.view(R.FP8), ws.view(R.FP8)
    with blocks(sms):
        got = gemm_a4w4(x, w, xs, ws, dtype=dtype)
        assert torch.equal(got, gemm_a4w4(x, w, xs, ws, dtype=dtype))
    want = xv @ wv.t()
    # k fp32 products and additions, and the few with scales
    bound = (xv.abs() @ wv.abs().t()) * (k + 8) * 2.0 ** -23
    compare(got, want, bound + (want.abs() + bound) * R.half_step(dtype) + torch.finfo(dtype).tiny)


# ---- layers ----------------------------------------------------------------------------------------
def experts(kind, e, h, i, hout, seed):
    return R.make_weights(kind, e, 2 * i, h, gen(seed)), R.make_weights(kind, e, hout, i, gen(seed + 1))


def scales_of(kind, w1, w2, a1, a2):
    kw = {} if w1[1] is None else dict(w1_scale=w1[1], w2_scale=w2[1])
    if kind in R.BLOCK:
        kw.update(w1_global_scale=w1[2], w2_global_scale=w2[2], a1_global_scale=a1, a2_global_scale=a2)
    return kw


def layer(call, kind, weights_of, m, k, *, experts_of_ids=None, seed=0, round_routes=False, sms=None, **more):
    w1, w2 = weights_of
    e, h = w1[3].shape[0], w1[3].shape[2]
    g = gen(seed)
    x = torch.randn(m, h, generator=g).to(torch.float16 if kind == "f16" else torch.bfloat16)
    count = experts_of_ids or e
    ids = torch.stack([torch.randperm(count, generator=g)[:k] if k > 1 else torch.tensor([t % count])
                       for t in range(m)])
    weights = torch.rand(m, k, generator=g) + 0.1
    a1 = torch.tensor([4.0 / 2688]) if kind == "nvfp4" else None
    a2 = torch.tensor([0.05]) if kind == "nvfp4" else None
    with blocks(sms):
        got = call(x, w1[0], w2[0], weights, ids.to(torch.int32), **scales_of(kind, w1, w2, a1, a2), **more)
    want, bound = R.layer(kind, x, w1[3], w2[3], ids, weights, got.dtype, a1=a1, a2=a2,
                          emap=more.get("expert_map"), round_routes=got.dtype if round_routes else None)
    compare(got, want, bound)
    return got


# hidden and intermediate size, output size: 8 experts are more than 256 KB of weights for each of 148 blocks
LARGE = {"bf16": (2056, 520, 2008), "f16": (2056, 520, 2008), "fp8_block": (2176, 1152, 2048),
         "int8_block": (2176, 1152, 2048), "fp8_channel": (2064, 1040, 2024), "int8_channel": (2064, 1040, 2024),
         "nvfp4": (4160, 1088, 4104), "mxfp4": (4224, 1152, 4104)}
_BYTES = {"bf16": 2, "f16": 2, "nvfp4": 0.5, "mxfp4": 0.5}


def _is_large(kind, e, h, i, hout):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return e * (2 * i * h + hout * i) * _BYTES.get(kind, 1) / sms > 256 << 10


@pytest.mark.parametrize("kind", R.KINDS)
def test_few_tokens_of_large_experts(kind):
    h, i, hout = LARGE[kind]
    assert _is_large(kind, 8, h, i, hout)
    both = experts(kind, 8, h, i, hout, 3)
    # one token; routes of a warp's size; more; two and four tiles of tokens
    for m, k in ((1, 8), (8, 1), (5, 3), (8, 4), (7, 6), (16, 3), (30, 2)):
        layer(fused_experts_decode, kind, both, m, k, seed=m, **FLAGS[kind])


@pytest.mark.parametrize("kind", ["fp8_block", "int8_block", "fp8_channel", "int8_channel"])
@pytest.mark.parametrize("h,i", [(16384, 256), (1024, 2176)])
def test_few_tokens_whose_codes_no_block_keeps(kind, h, i):
    """Rows (the first) or activations (the second) whose 8-bit codes a kernel in front makes, beside the other
    codes that every block keeps."""
    assert _is_large(kind, 8, h, i, 1024)
    both = experts(kind, 8, h, i, 1024, 5)
    layer(fused_experts_decode, kind, both, 8, 8, seed=1, **FLAGS[kind])
    layer(fused_experts_decode, kind, both, 1, 8, seed=2, **FLAGS[kind])


@pytest.mark.parametrize("kind", R.KINDS)
@pytest.mark.parametrize("sms", [1, 5])
def test_few_tokens_on_few_sms(kind, sms):
    """Every block many units and boxes."""
    step = 128 if kind.endswith("block") or kind == "mxfp4" else 64
    both = experts(kind, 6, 6 * step, 3 * step, 384, 7)
    for m, k in ((1, 2), (8, 3), (9, 1), (32, 4)):
        layer(fused_experts_decode, kind, both, m, k, seed=m, sms=sms, **FLAGS[kind])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sms", [None, 5])
def test_expert_layer_with_more_tiles_than_blocks(fmt, sms):
    """Padded tiles, experts that are not local and experts without a token."""
    both = experts(fmt, 48, 256, 640, 1032, 9)
    emap = torch.full((64,), -1, dtype=torch.int32)
    emap[torch.randperm(64, generator=gen(4))[:48]] = torch.randperm(48, generator=gen(5)).to(torch.int32)
    layer(fused_experts_fp4, fmt, both, 300, 4, seed=1, experts_of_ids=64, round_routes=True, sms=sms,
          expert_map=emap)
    layer(fused_experts_fp4, fmt, both, 260, 2, seed=2, experts_of_ids=11, round_routes=True, sms=sms,
          output_dtype=torch.float32)
