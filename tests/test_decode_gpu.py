"""The few-token layer against the layer in 64 bits, element by element within a propagated bound."""
import functools

import pytest
import torch

import fp4_reference as R
from boltops_b200.fused_moe import fused_experts_decode, fused_moe_decode, ops
from boltops_b200.fused_moe.routing import fused_topk

pytestmark = pytest.mark.gpu

FLAGS = {"bf16": {}, "f16": {}, "fp8_block": dict(use_fp8_w8a8=True, block_shape=[128, 128]),
         "int8_block": dict(use_int8_w8a8=True, block_shape=[128, 128]),
         "fp8_channel": dict(use_fp8_w8a8=True, per_channel_quant=True),
         "int8_channel": dict(use_int8_w8a8=True, per_channel_quant=True),
         "nvfp4": dict(use_fp4_w4a4=True), "mxfp4": dict(use_fp4_w4a4=True)}
SIZES = {"bf16": (8, 16), "f16": (8, 16), "fp8_block": (128, 128), "int8_block": (128, 128),
         "fp8_channel": (16, 16), "int8_channel": (16, 16), "nvfp4": (64, 64), "mxfp4": (128, 128)}


@functools.lru_cache(maxsize=4)
def experts(kind, e, h, i, hout=None):
    gen = torch.Generator().manual_seed(e * 1000 + h + i)
    w1 = R.make_weights(kind, e, 2 * i, h, gen)
    w2 = R.make_weights(kind, e, hout or h, i, gen)
    return w1, w2


def arguments(kind, w1, w2, a1=None, a2=None, dev="cuda"):
    kw = dict(FLAGS[kind])
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    if w1[1] is not None:
        kw.update(w1_scale=to(w1[1]), w2_scale=to(w2[1]))
    if kind in R.BLOCK:
        kw.update(w1_global_scale=to(w1[2]), w2_global_scale=to(w2[2]), a1_global_scale=to(a1),
                  a2_global_scale=to(a2))
    return to(w1[0]), to(w2[0]), kw


def rows(kind, m, h, seed, dtype=None):
    gen = torch.Generator().manual_seed(seed)
    dtype = dtype or (torch.float16 if kind == "f16" else torch.bfloat16)
    return torch.randn(m, h, generator=gen).to(dtype)


def routing(m, e, k, seed):
    gen = torch.Generator().manual_seed(seed)
    scores = torch.rand(m, e, generator=gen)
    w, ids = scores.topk(min(k, e), -1)
    return w / w.sum(-1, keepdim=True), ids.to(torch.int32)


def compare(got, want, bound):
    off = (got.cpu().double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4], off.max().item(),
                           (off / bound.clamp_min(1e-300)).max().item())


def run(kind, e, h, i, m, k, *, seed=0, hout=None, scaled=True, x=None, ids=None, weights=None, **more):
    w1, w2 = experts(kind, e, h, i, hout)
    x = rows(kind, m, h, seed) if x is None else x
    if ids is None:
        weights, ids = routing(m, e, k, seed + 1)
    a1 = torch.tensor([4.0 / 2688]) if kind == "nvfp4" and scaled else None
    a2 = torch.tensor([0.011]) if kind == "nvfp4" and scaled else None
    d1, d2, kw = arguments(kind, w1, w2, a1, a2)
    act = more.pop("act", None)
    got = fused_experts_decode(x.cuda(), d1, d2, weights.cuda(), ids.cuda(), **kw, **more)
    ops.check_device_status(got.device)
    want, bound = R.layer(kind, x, w1[3], w2[3], ids, weights, got.dtype, a1=a1, a2=a2, act=act,
                          scale=more.get("routed_scaling_factor", 1.0),
                          emap=more["expert_map"].cpu() if "expert_map" in more else None)
    compare(got, want, bound)
    return got


@pytest.mark.parametrize("kind", R.KINDS)
@pytest.mark.parametrize("m", [1, 2, 5, 8, 9, 17, 32])
def test_token_counts(kind, m):
    run(kind, 6, 256, 128, m, 2, seed=m)


@pytest.mark.parametrize("kind", R.KINDS)
def test_sizes(kind):
    step, istep = SIZES[kind]
    # one step; sizes whose last 128-byte box is partly outside; several units and boxes a warp
    run(kind, 3, step, istep, 3, 2, hout=None)
    run(kind, 2, 11 * step, 3 * istep, 4, 1)
    run(kind, 5, 1408, 640, 7, 3)
    run(kind, 2, 4096, 128, 3, 2)


@pytest.mark.parametrize("kind", ["bf16", "int8_channel", "nvfp4"])
def test_output_size_apart_from_the_hidden_size(kind):
    for hout in (8, 24, 328):
        run(kind, 4, 256, 128, 6, 2, hout=hout)


@pytest.mark.parametrize("kind", R.KINDS)
def test_all_tokens_on_one_expert_and_every_expert_touched(kind):
    m = 32
    ids = torch.full((m, 1), 2, dtype=torch.int32)
    run(kind, 4, 256, 128, m, 1, ids=ids, weights=torch.rand(m, 1, generator=torch.Generator().manual_seed(1)))
    ids = torch.arange(m, dtype=torch.int32).view(m, 1) % 40
    run(kind, 40, 128, 128, m, 1, ids=ids, weights=torch.ones(m, 1))


@pytest.mark.parametrize("kind", ["bf16", "fp8_block", "mxfp4"])
def test_repeated_skipped_and_unrouted(kind):
    weights = torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7], [1.0, 2.0, 3.0], [0.3, 0.3, 0.4]])
    ids = torch.tensor([[1, 1, 3], [-1, 99, 2], [-1, -1, -5], [3, 0, 3]], dtype=torch.int32)
    got = run(kind, 4, 256, 128, 4, 3, ids=ids, weights=weights)
    assert not got[2].any()
    none = run(kind, 4, 256, 128, 4, 3, ids=torch.full((4, 3), -1, dtype=torch.int32), weights=weights)
    assert not none.any()


@pytest.mark.parametrize("kind", ["f16", "int8_channel", "nvfp4"])
def test_expert_map(kind):
    emap = torch.tensor([-1, 2, -1, 0, 1, -1, 3, -1], dtype=torch.int32)
    weights, ids = routing(6, 8, 3, 11)
    run(kind, 4, 256, 128, 6, 3, ids=ids, weights=weights, expert_map=emap.cuda(), global_num_experts=8)
    run(kind, 4, 256, 128, 6, 3, ids=ids, weights=weights, expert_map=emap.cuda())


@pytest.mark.parametrize("kind", R.KINDS)
def test_row_and_output_types_scale_and_int64_ids(kind):
    other = torch.float16 if kind not in ("bf16", "f16") else None
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        weights, ids = routing(3, 6, 2, 5)
        run(kind, 6, 256, 128, 3, 2, x=rows(kind, 3, 256, 4, other), ids=ids.long(), weights=weights.double(),
            output_dtype=out_dtype, routed_scaling_factor=2.5)


def _gelu(g, u):
    return 0.5 * g * (1 + torch.erf(g / 2 ** 0.5)) * u


def _gelu_tanh(g, u):
    return 0.5 * g * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u


def _clamped(g, u):
    g, u = g.clamp(max=0.5), u.clamp(-0.5, 0.5)
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("kind", ["bf16", "fp8_channel", "nvfp4"])
def test_activations(kind):
    run(kind, 4, 256, 128, 5, 2, activation="gelu", act=_gelu)
    run(kind, 4, 256, 128, 5, 2, activation="gelu_tanh", act=_gelu_tanh)
    run(kind, 4, 256, 128, 5, 2, activation="silu", gemm1_limit=0.5, act=_clamped)


@pytest.mark.parametrize("kind", R.KINDS)
def test_other_tokens_infinities_and_nans_stay_with_them(kind):
    """A token's values, and an expert's weights, reach only the tokens that use them."""
    w1, w2 = experts(kind, 4, 256, 128)
    x = rows(kind, 5, 256, 3)
    ids = torch.tensor([[0, 1], [2, 1], [0, 3], [2, 0], [3, 1]], dtype=torch.int32)
    weights = torch.full((5, 2), 0.5)
    d1, d2, kw = arguments(kind, w1, w2)
    want = fused_experts_decode(x.cuda(), d1, d2, weights.cuda(), ids.cuda(), **kw)
    sick = x.clone()
    sick[2, 17] = float("nan")
    sick[3, 200] = float("inf")
    got = fused_experts_decode(sick.cuda(), d1, d2, weights.cuda(), ids.cuda(), **kw)
    assert torch.equal(got[[0, 1, 4]], want[[0, 1, 4]])
    if kind in ("bf16", "f16", "fp8_channel", "fp8_block") or kind in R.BLOCK:
        assert torch.isnan(got[2]).all()
    if kind in ("bf16", "f16"):
        bad = d2.clone()
        bad[3, 5, 7] = float("inf")
        got = fused_experts_decode(x.cuda(), d1, bad, weights.cuda(), ids.cuda(), **kw)
        assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]]) and not torch.isfinite(got[[2, 4], 5]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e,topk,softmax,renorm", [(6, 2, True, True), (40, 8, True, False), (200, 6, False, True),
                                                   (300, 1, True, True), (1024, 32, True, True)])
def test_router_inside_equals_the_router_before(dtype, e, topk, softmax, renorm):
    w1, w2 = experts("bf16", 8, 64, 16)
    emap = torch.full((e,), -1, dtype=torch.int32)
    emap[:: max(1, e // 8)][:8] = torch.arange(min(8, len(emap[:: max(1, e // 8)])), dtype=torch.int32)
    for m in (1, 7, 32):
        x = rows("bf16", m, 64, m).cuda()
        logits = torch.randn(m, e, generator=torch.Generator().manual_seed(m)).to(dtype).cuda()
        weights, ids = fused_topk(x, logits, topk, renorm, is_softmax=softmax)
        common = dict(expert_map=emap.cuda())
        got = fused_moe_decode(x, logits, w1[0].cuda(), w2[0].cuda(), topk, renorm, softmax, **common)
        assert torch.equal(got, fused_experts_decode(x, w1[0].cuda(), w2[0].cuda(), weights, ids, **common))


@pytest.mark.parametrize("kind", R.KINDS)
def test_calls_repeat_overlap_and_replay(kind):
    w1, w2 = experts(kind, 6, 512, 256)
    d1, d2, kw = arguments(kind, w1, w2)
    sets = []
    for s in range(3):
        m = (1, 8, 20)[s]
        weights, ids = routing(m, 6, 2, s)
        x = rows(kind, m, 512, s).cuda()
        sets.append((x, weights.cuda(), ids.cuda(), fused_experts_decode(x, d1, d2, weights.cuda(), ids.cuda(), **kw)))
    for x, weights, ids, want in sets:      # back to back
        assert torch.equal(fused_experts_decode(x, d1, d2, weights, ids, **kw), want)
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    for _ in range(5):
        for (x, weights, ids, want), st in zip(sets, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append((fused_experts_decode(x, d1, d2, weights, ids, **kw), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    x, weights, ids, want = (t.clone() for t in sets[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = fused_experts_decode(x, d1, d2, weights, ids, **kw)
        two = fused_experts_decode(one.to(x.dtype), d1, d2, weights, ids, **kw)
    graph.replay()
    assert torch.equal(one, want)
    assert torch.equal(two, fused_experts_decode(want.to(x.dtype), d1, d2, weights, ids, **kw))
    x.mul_(0.5)
    graph.replay()
    assert torch.equal(one, fused_experts_decode(x, d1, d2, weights, ids, **kw))
    inplace = x.clone()
    assert fused_experts_decode(inplace, d1, d2, weights, ids, **kw, out=inplace) is inplace
    assert torch.equal(inplace, one)


def test_strided_rows_weights_off_the_grid_and_no_tokens():
    w1, w2 = experts("bf16", 6, 256, 128)
    d1, d2 = w1[0].cuda(), w2[0].cuda()
    weights, ids = (t.cuda() for t in routing(4, 6, 2, 1))
    wide = torch.randn(4, 300, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    view = wide[:, 3:259]
    want = fused_experts_decode(view.contiguous(), d1, d2, weights, ids)
    assert torch.equal(fused_experts_decode(view, d1, d2, weights, ids), want)
    flat = torch.empty(d1.numel() + 1, dtype=d1.dtype, device="cuda")
    odd = flat[1:].view(d1.shape).copy_(d1)
    assert torch.equal(fused_experts_decode(view, odd, d2, weights, ids), want)
    assert torch.equal(fused_experts_decode(view, d1, d2.transpose(1, 2).contiguous().transpose(1, 2), weights, ids),
                       want)
    assert fused_experts_decode(view[:0], d1, d2, weights[:0], ids[:0]).shape == (0, 256)


def test_long_rows_many_tokens():
    """Where kept codes do not fit: 8-bit rows are quantised box by box, 4-bit ones go half by half."""
    for m, h in ((8, 32768), (24, 9216)):
        x = rows("fp8_block", m, h, 2) * 0.05
        run("fp8_block", 2, h, 128, m, 1, hout=128, x=x)
        run("int8_channel", 2, h, 128, m, 1, hout=128, x=x)
    for kind, m, h in (("nvfp4", 32, 16384), ("mxfp4", 27, 8192)):
        run(kind, 2, h, 128, m, 1, hout=64, x=rows(kind, m, h, 1) * 0.05)
    w1, w2 = experts("mxfp4", 2, 8192, 128, 64)
    d1, d2, kw = arguments("mxfp4", w1, w2)
    x, logits = rows("mxfp4", 27, 8192, 1).cuda(), torch.randn(27, 2, device="cuda")
    weights, ids = fused_topk(x, logits, 1, True)
    assert torch.equal(fused_moe_decode(x, logits, d1, d2, 1, True, **kw),
                       fused_experts_decode(x, d1, d2, weights, ids, **kw))


def test_many_routes_and_experts():
    """More routes than a warp has lanes, more experts than a block has threads."""
    weights, ids = routing(32, 700, 8, 3)
    for kind in ("bf16", "int8_channel"):
        run(kind, 700, 64, 16, 32, 8, ids=ids, weights=weights)
        run(kind, 700, 64, 16, 5, 7, ids=ids[:5, :7], weights=weights[:5, :7])


def test_situ_and_step_activations():
    def situ(g, u):
        return 2.0 * torch.tanh(g / 2.0) * torch.sigmoid(g) * u

    def step(g, u):
        return (g * torch.sigmoid(g)).clamp(max=0.7) * u.clamp(-0.7, 0.7)
    run("bf16", 4, 256, 128, 5, 2, activation="situ", activation_situ_beta=2.0, act=situ)
    run("f16", 4, 256, 128, 5, 2, activation="swiglustep", gemm1_limit=0.7, act=step)


@pytest.mark.parametrize("kind", ["bf16", "fp8_channel", "int8_channel", "nvfp4", "mxfp4"])
@pytest.mark.parametrize("hout", [1, 3, 7, 33])
def test_output_sizes_below_and_beside_a_unit(kind, hout):
    run(kind, 4, 256, 128, 1, 2, hout=hout, output_dtype=torch.float32)
    run(kind, 4, 256, 128, 19, 2, hout=hout)


@pytest.mark.parametrize("m", [1, 3, 20])
def test_router_of_all_experts_of_one_and_of_views(m):
    """Every expert chosen; one expert; logits in a wider array; logits that are NaN or infinite."""
    for e, topk in ((8, 8), (1, 1), (5, 4)):
        w1, w2 = experts("bf16", e, 64, 16)
        x = rows("bf16", m, 64, m).cuda()
        wide = torch.randn(m, e + 3, generator=torch.Generator().manual_seed(m)).cuda()
        view = wide[:, 2:2 + e]
        sick = view.clone()
        sick[0, 0], sick[-1, -1] = float("nan"), float("-inf")
        for logits in (view, sick, torch.full_like(sick, float("nan"))):
            weights, ids = fused_topk(x, logits.contiguous(), topk, True)
            got = fused_moe_decode(x, logits, w1[0].cuda(), w2[0].cuda(), topk, True)
            want = fused_experts_decode(x, w1[0].cuda(), w2[0].cuda(), weights, ids)
            assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_calls_with_reserved_sms_and_without_alternate():
    """The second kernel starts early in one and waits in the other; both on two streams, and in a graph."""
    w1, w2 = experts("int8_channel", 6, 512, 256)
    d1, d2, kw = arguments("int8_channel", w1, w2)
    weights, ids = (t.cuda() for t in routing(12, 6, 2, 3))
    x = rows("int8_channel", 12, 512, 4).cuda()

    def call(reserve):
        ops.set_gemm_sm_reserve(reserve)
        try:
            return fused_experts_decode(x, d1, d2, weights, ids, **kw)
        finally:
            ops.set_gemm_sm_reserve(0)
    want = {r: call(r) for r in (0, 40)}
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            streams[i % 2].wait_stream(torch.cuda.default_stream())
            got.append((call(40 * (i % 3 == 0)), want[40 * (i % 3 == 0)]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [call(r) for r in (40, 0, 40)]
    graph.replay()
    assert torch.equal(ys[0], want[40]) and torch.equal(ys[1], want[0]) and torch.equal(ys[2], want[40])
