"""4-bit products against their definition in 64 bits: the dense one and the expert layer."""
import pytest
import torch

import fp4_reference as R
from boltops_b200.fp4 import fp4_quant
from boltops_b200.fused_moe import fused_experts_decode, fused_experts_fp4, ops
from boltops_b200.gemm import gemm_a4w4
from test_decode_gpu import arguments, compare, experts, routing, rows

pytestmark = pytest.mark.gpu
FORMATS = ["nvfp4", "mxfp4"]


def operand(fmt, n, k, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    codes, scales, values = R.fp4_quant(fmt, torch.randn(n, k, generator=gen) * spread)
    return codes, scales.view(R.FP8) if fmt == "nvfp4" else scales, values


def dense(fmt, m, n, k, dtype=torch.bfloat16, alpha=None, out=None):
    x, xs, xv = operand(fmt, m, k, m + 1)
    w, ws, wv = operand(fmt, n, k, n + 2, 0.05)
    a = None if alpha is None else torch.tensor([alpha]).cuda()
    got = gemm_a4w4(x.cuda(), w.cuda(), xs.cuda(), ws.cuda(), alpha=a, dtype=dtype, out=out)
    ops.check_device_status(got.device)
    f = 1.0 if alpha is None else float(torch.tensor(alpha))
    want = xv @ wv.t() * f
    bound = (xv.abs() @ wv.abs().t()) * abs(f) * (k + 8) * 2.0 ** -23
    compare(got, want, bound + (want.abs() + bound) * R.half_step(dtype) + torch.finfo(dtype).tiny)
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,blocks", [(1, 1, 1), (1, 128, 2), (3, 7, 3), (8, 257, 5), (31, 129, 9), (32, 64, 28),
                                        (33, 300, 4), (127, 256, 3), (128, 512, 1), (129, 1000, 7), (300, 131, 16),
                                        (1000, 520, 2)])
def test_dense_sizes(fmt, m, n, blocks):
    dense(fmt, m, n, blocks * 4 * R.BLOCK[fmt])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [5, 200])
def test_dense_types_alpha_and_output_views(fmt, dtype, m):
    dense(fmt, m, 192, 512, dtype, alpha=0.0371)
    wide = torch.full((m, 300), 7.0, dtype=dtype, device="cuda")
    got = dense(fmt, m, 192, 512, dtype, out=wide[:, 5:197])
    assert got.data_ptr() == wide[:, 5:].data_ptr()
    assert (wide[:, :5] == 7).all() and (wide[:, 197:] == 7).all()
    dense(fmt, m, 192, 512, dtype, out=torch.full((m, 200), 7.0, dtype=dtype, device="cuda")[:, :192])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [4, 150])
def test_dense_scales_of_every_size(fmt, m):
    """Scales over the format's whole range, in every place of a block row."""
    gen = torch.Generator().manual_seed(9)
    k, n = 1024, 96
    count = k // R.BLOCK[fmt]
    low, high = (1, 0x7E) if fmt == "nvfp4" else (127 - 30, 127 + 30)
    xs = torch.randint(low, high + 1, (m, count), generator=gen).to(torch.uint8)
    ws = torch.randint(low, high + 1, (n, count), generator=gen).to(torch.uint8)
    x = torch.randint(0, 256, (m, k // 2), generator=gen).to(torch.uint8)
    w = torch.randint(0, 256, (n, k // 2), generator=gen).to(torch.uint8)
    xv, wv = R.fp4_values(fmt, x, xs), R.fp4_values(fmt, w, ws)
    see = (lambda s: s.view(R.FP8).cuda()) if fmt == "nvfp4" else (lambda s: s.cuda())
    got = gemm_a4w4(x.cuda(), w.cuda(), see(xs), see(ws), dtype=torch.float32)
    bound = (xv.abs() @ wv.abs().t()) * (k + 8) * 2.0 ** -23
    compare(got, xv @ wv.t(), bound * 1.01)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [6, 140])
def test_dense_nan_scale_stays_in_its_row(fmt, m):
    x = torch.randn(m, 256, generator=torch.Generator().manual_seed(1))
    x[2, 7] = float("nan")
    w, ws, _ = operand(fmt, 40, 256, 3)
    codes, scales = fp4_quant(x.cuda(), fmt)
    got = gemm_a4w4(codes, w.cuda(), scales, ws.cuda())
    assert torch.isnan(got[2]).all() and torch.isfinite(torch.cat((got[:2], got[3:]))).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [7, 260])
def test_dense_calls_repeat_overlap_and_replay(fmt, m):
    x, xs, _ = operand(fmt, m, 2048, 1)
    w, ws, _ = operand(fmt, 768, 2048, 2)
    x, xs, w, ws = x.cuda(), xs.cuda(), w.cuda(), ws.cuda()
    want = gemm_a4w4(x, w, xs, ws)
    # operands off the 16-byte grid and apart from each other are copied
    odd = torch.empty(x.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(x.shape).copy_(x)
    assert torch.equal(gemm_a4w4(odd, w, xs, ws), want)
    wide = torch.zeros(768, 1500, dtype=torch.uint8, device="cuda")
    wide[:, 30:30 + 1024] = w
    assert torch.equal(gemm_a4w4(x, wide[:, 30:30 + 1024], xs, ws), want)
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams * 3:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(gemm_a4w4(x, w, xs, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm_a4w4(x, w, xs, ws)
    graph.replay()
    assert torch.equal(y, want)


# ---- experts -----------------------------------------------------------------------------
def layer(fmt, e, h, i, m, k, *, hout=None, scaled=True, ids=None, weights=None, x=None, **more):
    w1, w2 = experts(fmt, e, h, i, hout)
    x = rows(fmt, m, h, m) if x is None else x
    if ids is None:
        weights, ids = routing(m, e, k, m + 1)
    a1 = torch.tensor([4.0 / 2688]) if fmt == "nvfp4" and scaled else None
    a2 = torch.tensor([0.011]) if fmt == "nvfp4" and scaled else None
    d1, d2, kw = arguments(fmt, w1, w2, a1, a2)
    kw.pop("use_fp4_w4a4")
    act = more.pop("act", None)
    got = fused_experts_fp4(x.cuda(), d1, d2, weights.cuda(), ids.cuda(), **kw, **more)
    ops.check_device_status(got.device)
    want, bound = R.layer(fmt, x, w1[3], w2[3], ids, weights, got.dtype, a1=a1, a2=a2, act=act,
                          scale=more.get("routed_scaling_factor", 1.0), round_routes=got.dtype,
                          emap=more["expert_map"].cpu() if "expert_map" in more else None)
    compare(got, want, bound)
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 17, 64, 130, 300])
def test_layer_token_counts(fmt, m):
    layer(fmt, 6, 256, 128, m, 2)


@pytest.mark.parametrize("fmt", FORMATS)
def test_layer_sizes(fmt):
    step = 4 * R.BLOCK[fmt]
    layer(fmt, 3, step, step, 20, 2)
    layer(fmt, 2, 11 * step, 3 * step, 9, 1)
    layer(fmt, 5, 1408, 640, 33, 3)
    layer(fmt, 4, 256, 128, 50, 2, hout=72)


@pytest.mark.parametrize("fmt", FORMATS)
def test_layer_routing_maps_types_activations_and_chunks(fmt, monkeypatch):
    weights, ids = routing(40, 8, 3, 11)
    emap = torch.tensor([-1, 2, -1, 0, 1, -1, 3, -1], dtype=torch.int32)
    layer(fmt, 4, 256, 128, 40, 3, ids=ids, weights=weights, expert_map=emap.cuda())
    # (an entry past the local experts is as good as none)
    wild = torch.tensor([9, 2, -1, 0, 1, -7, 3, 4], dtype=torch.int32)
    same = layer(fmt, 4, 256, 128, 40, 3, ids=ids, weights=weights, expert_map=emap.cuda())
    assert torch.equal(layer(fmt, 4, 256, 128, 40, 3, ids=ids, weights=weights, expert_map=wild.cuda()), same)
    one = torch.full((200, 1), 2, dtype=torch.int32)
    layer(fmt, 4, 256, 128, 200, 1, ids=one, weights=torch.rand(200, 1))
    ids = torch.tensor([[1, 1, 3], [-1, 99, 2], [-1, -1, -5]], dtype=torch.int32)
    got = layer(fmt, 4, 256, 128, 3, 3, ids=ids, weights=torch.rand(3, 3))
    assert not got[2].any()
    for dtype in (torch.float32, torch.float16):
        layer(fmt, 6, 256, 128, 20, 2, x=rows(fmt, 20, 256, 1, torch.float16), output_dtype=dtype,
              routed_scaling_factor=2.5)
    layer(fmt, 6, 256, 128, 20, 2, scaled=False,
          act=lambda g, u: 0.5 * g * (1 + torch.erf(g / 2 ** 0.5)) * u, activation="gelu")
    monkeypatch.setenv("BOLTOPS_FUSED_MOE_CHUNK_SIZE", "37")
    layer(fmt, 6, 256, 128, 100, 2)


@pytest.mark.parametrize("fmt", FORMATS)
def test_layer_and_its_few_token_form_together(fmt):
    """A prompt through the one, its next token through the other, captured together."""
    w1, w2 = experts(fmt, 6, 512, 256)
    d1, d2, kw = arguments(fmt, w1, w2)
    few = dict(kw)
    kw.pop("use_fp4_w4a4")
    weights, ids = (t.cuda() for t in routing(40, 6, 2, 5))
    x = rows(fmt, 40, 512, 6).cuda()
    both = fused_experts_fp4(x, d1, d2, weights, ids, **kw)
    step = fused_experts_decode(both[-3:], d1, d2, weights[:3], ids[:3], **few)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = fused_experts_fp4(x, d1, d2, weights, ids, **kw)
        b = fused_experts_decode(a[-3:], d1, d2, weights[:3], ids[:3], **few)
    graph.replay()
    assert torch.equal(a, both) and torch.equal(b, step)
    # the same rows either way: apart by the roundings of the routes and of the sums' order
    same = fused_experts_decode(x[:20], d1, d2, weights[:20], ids[:20], **few)
    wanted, bound = R.layer(fmt, x[:20].cpu(), w1[3], w2[3], ids[:20].cpu(), weights[:20].cpu(), same.dtype,
                            round_routes=same.dtype)
    compare(same, wanted, bound)
    compare(both[:20], wanted, bound)
