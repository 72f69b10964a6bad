"""Microscaled 4-bit quantisation against its definition in 64 bits: codes and scales bit for bit."""
import pytest
import torch

import fp4_reference as R
from boltops_b200.fp4 import fp4_dequant, fp4_quant

pytestmark = pytest.mark.gpu


def check(x, fmt, g=None):
    codes, scales = fp4_quant(x.cuda(), fmt, None if g is None else g.cuda())
    want_codes, want_scales, want_values = R.fp4_quant(fmt, x, g)
    assert torch.equal(scales.cpu().view(torch.uint8), want_scales)
    # the sign of a zero code says nothing
    def plain(c):
        low, high = c & 15, c >> 4
        return torch.stack((torch.where(low == 8, 0, low), torch.where(high == 8, 0, high)))
    assert torch.equal(plain(codes.cpu()), plain(want_codes))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        back = fp4_dequant(codes, scales, None if g is None else g.cuda(), dtype=dtype).cpu().double()
        # code * scale is exact in fp32; the product with g and the output's type round once each
        off = (want_values.abs() * (R.half_step(dtype) * 1.001 + 2.0 ** -23)
               + torch.finfo(dtype).tiny * 2.0 * R.half_step(dtype))
        inside = want_values.abs() <= torch.finfo(dtype).max
        ok = ((back - want_values).abs() <= off) | (torch.isnan(back) & torch.isnan(want_values)) | ~inside
        assert ok.all(), (dtype, (~ok).nonzero()[:4])


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,blocks", [(1, 1), (3, 5), (7, 224), (129, 33), (1000, 3)])
def test_codes_and_scales(fmt, dtype, rows, blocks):
    gen = torch.Generator().manual_seed(rows * 31 + blocks)
    x = (torch.randn(rows, blocks * R.BLOCK[fmt], generator=gen) * 3).to(dtype)
    check(x, fmt)
    if fmt == "nvfp4":
        check(x, fmt, torch.tensor([0.00173]))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_every_16_bit_value_and_the_borders(fmt):
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        x = bits.view(dtype)
        x = x[torch.isfinite(x)]
        x = x[: x.numel() // 32 * 32]
        check(x.reshape(-1, 32), fmt)
        gen = torch.Generator().manual_seed(1)
        check(x[torch.randperm(x.numel(), generator=gen)].reshape(-1, 64), fmt)
    # borders of two codes under every scale: k / 4 of 6 * scale is exact in the input's type
    k = torch.arange(-24, 25, dtype=torch.float32)
    rows = torch.stack([torch.cat((k, torch.zeros(15))) * 0.25 * s for s in (1.0, 1.125, 0.875, 448.0, 2.0 ** -6)])
    rows[:, 49::16] = rows.abs().amax(-1, keepdim=True)
    check(rows.to(torch.bfloat16), fmt)
    check(rows, fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_zeros_extremes_nan_and_infinity(fmt):
    x = torch.zeros(6, 64)
    x[1, 3], x[1, 40] = 3e38, -1e-38
    x[2, 5] = float("nan")
    x[3, 63] = float("-inf")
    x[4, :32] = 1e-30
    x[5] = -0.0
    check(x, fmt)
    codes, scales = fp4_quant(x.cuda(), fmt)
    back = fp4_dequant(codes, scales, dtype=torch.float32).cpu()
    assert torch.isnan(back[2, :16]).all() and torch.isnan(back[3, 48:]).all() and not back[0].any()
    assert torch.isfinite(back[2, 32:]).all() and torch.isfinite(back[3, :32]).all()


def test_strides_offsets_streams_and_graphs():
    gen = torch.Generator().manual_seed(3)
    base = torch.randn(9, 200, generator=gen, dtype=torch.float32).cuda()
    view = base[1::2, 3:131]            # rows apart, off the 16-byte grid
    for fmt in ("nvfp4", "mxfp4"):
        want = fp4_quant(view.clone(), fmt)
        got = fp4_quant(view, fmt)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].view(torch.uint8), want[1].view(torch.uint8))
        flat = torch.randn(161, device="cuda").to(torch.bfloat16)
        odd = flat[1:161]               # contiguous, off the grid
        assert torch.equal(fp4_quant(odd, fmt)[0], fp4_quant(odd.clone(), fmt)[0])
        three = torch.randn(2, 3, 64, device="cuda")
        codes, scales = fp4_quant(three, fmt)
        assert codes.shape == (2, 3, 32) and scales.shape == (2, 3, 64 // R.BLOCK[fmt])
        assert fp4_dequant(codes, scales).shape == three.shape
        empty = fp4_quant(torch.empty(0, 64, device="cuda"), fmt)
        assert empty[0].shape == (0, 32) and fp4_dequant(*empty).shape == (0, 64)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = fp4_quant(three, fmt)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], codes)
        x = torch.zeros(5, 64, device="cuda")
        fp4_quant(x, fmt)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c, s = fp4_quant(x, fmt)
            back = fp4_dequant(c, s)
        for seed in (1, 2):
            x.copy_(torch.randn(5, 64, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            assert torch.equal(back, fp4_dequant(*fp4_quant(x, fmt)))


def test_more_than_two_to_the_31_values():
    rows, cols = (1 << 31) // 4096 + 3, 4096
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(cols, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    codes, scales = fp4_quant(x, "nvfp4")
    want = R.fp4_quant("nvfp4", x[-1:].cpu())
    assert torch.equal(codes[-1:].cpu() & 0x77, want[0] & 0x77)
    assert torch.equal(scales[-1:].cpu().view(torch.uint8), want[1])
    assert not codes[:-1].any()
    back = fp4_dequant(codes, scales)
    assert torch.equal(back[-1].cpu().double(), want[2][0].to(torch.bfloat16).double())
