"""The 4-bit calls and the few-token layer without a GPU: argument structures, refusals in Python and at the
C entries, and the reference arithmetic the GPU tests rely on."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import fp4_reference as R

ROOT = Path(__file__).resolve().parent.parent


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: everything in front of the first launch can be run."""
    is_cuda = True


def gpu(t):
    return t.as_subclass(_OnGpu)


@pytest.fixture(scope="module")
def lib():
    from boltops_b200 import _cabi, build
    build.build()
    return _cabi.load()


@pytest.mark.parametrize("name,struct", [("bolt_fp4_tile_job", "Fp4TileJob"), ("bolt_fp4_tile_args", "Fp4TileArgs"),
                                         ("bolt_fp4_gemm_args", "Fp4GemmArgs"), ("bolt_fp4_few_args", "Fp4FewArgs"),
                                         ("bolt_decode_args", "DecodeArgs")])
def test_structures_match_the_header(name, struct, tmp_path):
    from boltops_b200 import _cabi
    cls = getattr(_cabi, struct)
    fields = [f[0] for f in cls._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "boltops_b200.h"}"',
            "int main(void){", f'printf("%zu\\n", sizeof({name}));']
    prog += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]
    (tmp_path / "a.c").write_text("\n".join(prog))
    subprocess.run(["gcc", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    nums = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True,
                                           check=True).stdout.split()]
    assert nums[0] == ctypes.sizeof(cls)
    assert [getattr(cls, f).offset for f in fields] == nums[1:]


def test_enumerations_match_the_header():
    from boltops_b200 import _cabi
    header = (ROOT / "include" / "boltops_b200.h").read_text()
    value = lambda n: int(re.search(rf"\b{n} = (\d+)", header).group(1))  # noqa: E731
    assert (value("BOLT_FP4_NV"), value("BOLT_FP4_MX")) == (_cabi.FP4_NV, _cabi.FP4_MX)
    for n in ("BF16", "F16", "FP8_BLOCK", "INT8_CHANNEL", "FP8_CHANNEL", "INT8_BLOCK", "NVFP4", "MXFP4"):
        assert value("BOLT_DECODE_" + n) == getattr(_cabi, "DECODE_" + n)


# ---- refusals at the C entries: an error code, no launch -----------------------------------
def test_c_entries_refuse(lib):
    from boltops_b200 import _cabi
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf)
    at += -at % 256
    q = lib.bolt_fp4_quant
    assert q(at, _cabi.BF16, 1, 24, _cabi.FP4_NV, None, at, at, None) == 1          # a block and a half
    assert q(at, _cabi.BF16, 1, 48, _cabi.FP4_MX, None, at, at, None) == 1
    assert q(at, _cabi.BF16, 1, 32, 2, None, at, at, None) == 1                     # format
    assert q(at, _cabi.INT8, 1, 32, _cabi.FP4_NV, None, at, at, None) == 1          # type
    assert q(at + 2, _cabi.BF16, 1, 32, _cabi.FP4_NV, None, at, at, None) == 1      # alignment
    assert q(None, _cabi.BF16, 1, 32, _cabi.FP4_NV, None, at, at, None) == 1
    assert q(at, _cabi.BF16, 1, 32, _cabi.FP4_MX, at, at, at, None) == 1            # MX has no whole scale
    assert q(None, _cabi.BF16, 0, 32, _cabi.FP4_NV, None, None, None, None) == 0    # nothing to do
    assert lib.bolt_fp4_dequant(at, at, 1, 24, _cabi.FP4_NV, None, at, _cabi.BF16, None) == 1
    assert lib.bolt_fp4_gemm(None, None) == 1 and lib.bolt_fp4_gemm_few(None, None) == 1
    assert lib.bolt_fp4_tile_scales(None, None) == 1 and lib.bolt_moe_decode(None, None) == 1

    few = dict(format=_cabi.FP4_NV, rows=1, n=8, k=64, x=at, x_scale=at, w=at, w_scale=at, out=at, out_dtype=_cabi.BF16,
               out_ld=8)
    for bad in (dict(rows=33), dict(k=96), dict(k=0), dict(x=None), dict(w=at + 8), dict(out_ld=7), dict(format=5),
                dict(out_dtype=_cabi.INT8), dict(out=at + 1)):
        assert lib.bolt_fp4_gemm_few(_cabi.Fp4FewArgs(**{**few, **bad}), None) == 1, bad
    assert lib.bolt_fp4_gemm_few(_cabi.Fp4FewArgs(**{**few, "rows": 0, "x": None}), None) == 0

    gemm = dict(format=_cabi.FP4_NV, rows=128, n=8, k=64, num_experts=1, a=at, a_tiles=at, b=at, b_tiles=at, c=at,
                c_dtype=_cabi.BF16, c_ld=8)
    for bad in (dict(k=32), dict(format=_cabi.FP4_MX), dict(epilogue=_cabi.EPI_SILU_MUL), dict(num_experts=2),
                dict(epilogue=_cabi.EPI_SILU_MUL_QUANT), dict(a=None), dict(b_tiles=at + 4), dict(c_ld=4),
                dict(sorted_expert_ids=at), dict(sorted_weights=at)):
        assert lib.bolt_fp4_gemm(_cabi.Fp4GemmArgs(**{**gemm, **bad}), None) == 1, bad

    layer = dict(kind=_cabi.DECODE_BF16, x_dtype=_cabi.BF16, out_dtype=_cabi.BF16, num_tokens=1, topk=1, hidden=64,
                 inter=64, model_dim=64, num_experts=2, global_num_experts=2, hidden_states=at, w1=at, w2=at,
                 topk_weights=at, topk_ids=at, out=at, workspace=at, workspace_bytes=1 << 20)
    for bad in (dict(kind=8), dict(num_tokens=33), dict(num_tokens=-1), dict(topk=0), dict(topk=33), dict(hidden=60),
                dict(num_experts=1025), dict(x_dtype=_cabi.F16), dict(kind=_cabi.DECODE_FP8_BLOCK),
                dict(kind=_cabi.DECODE_INT8_CHANNEL), dict(w1=None), dict(topk_ids=None), dict(workspace_bytes=8),
                dict(w1=at + 8), dict(gating=at, gating_dtype=_cabi.INT8), dict(gating=at, topk=3),
                dict(out_dtype=_cabi.INT8)):
        assert lib.bolt_moe_decode(_cabi.DecodeArgs(**{**layer, **bad}), None) == 1, bad
    assert lib.bolt_moe_decode_workspace_bytes(_cabi.DecodeArgs(**layer)) >= 128
    assert lib.bolt_moe_decode_workspace_bytes(_cabi.DecodeArgs(**{**layer, "hidden": 60})) == 0
    assert lib.bolt_moe_decode(_cabi.DecodeArgs(**{**layer, "num_tokens": 0, "out": None}), None) == 0


# ---- refusals in Python ---------------------------------------------------------------------
def test_no_cpu_path():
    from boltops_b200.fp4 import fp4_dequant, fp4_quant
    from boltops_b200.fused_moe import fused_experts_decode, fused_experts_fp4, fused_moe_decode
    from boltops_b200.gemm import gemm_a4w4
    x, c, s = torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 4).to(R.FP8)
    w, ids = torch.zeros(2, 4, 64), torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: fp4_quant(x), lambda: fp4_dequant(c, s), lambda: gemm_a4w4(c, c, s, s),
                 lambda: fused_experts_decode(x, w, w, ids.float(), ids), lambda: fused_moe_decode(x, x, w, w, 1, True),
                 lambda: fused_experts_fp4(x, w, w, ids.float(), ids, s, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_fp4_quant_and_dequant_refuse():
    from boltops_b200.fp4 import fp4_dequant, fp4_quant
    x = gpu(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="format"):
        fp4_quant(x, "fp4")
    with pytest.raises(TypeError):
        fp4_quant(gpu(torch.zeros(2, 64, dtype=torch.int8)))
    with pytest.raises(ValueError, match="whole blocks"):
        fp4_quant(gpu(torch.zeros(2, 40)))
    with pytest.raises(ValueError, match="whole blocks"):
        fp4_quant(gpu(torch.zeros(2, 48)), "mxfp4")
    with pytest.raises(ValueError, match="whole tensor"):
        fp4_quant(x, "mxfp4", torch.ones(1))
    for bad in (torch.ones(2), torch.ones(1, dtype=torch.float64)):
        with pytest.raises(ValueError, match="float32"):
            fp4_quant(x, "nvfp4", bad)
    with pytest.raises(ValueError, match="is on meta"):
        fp4_quant(x, "nvfp4", torch.ones(1, device="meta"))
    c = gpu(torch.zeros(2, 32, dtype=torch.uint8))
    with pytest.raises(TypeError, match="scales"):
        fp4_dequant(c, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="do not belong"):
        fp4_dequant(c, torch.zeros(2, 2).to(R.FP8))
    with pytest.raises(ValueError, match="do not belong"):
        fp4_dequant(c, torch.zeros(2, 4, dtype=torch.uint8))
    with pytest.raises(TypeError):
        fp4_dequant(c, torch.zeros(2, 4).to(R.FP8), dtype=torch.int8)


def test_gemm_a4w4_refuses():
    from boltops_b200.gemm import gemm_a4w4
    x, w = gpu(torch.zeros(3, 64, dtype=torch.uint8)), torch.zeros(5, 64, dtype=torch.uint8)
    xs, ws = torch.zeros(3, 8).to(R.FP8), torch.zeros(5, 8).to(R.FP8)
    good = dict(x=x, w=w, x_scale=xs, w_scale=ws)
    for bad, error in ((dict(w=w.float()), TypeError), (dict(w_scale=torch.zeros(5, 4, dtype=torch.uint8)), TypeError),
                       (dict(x_scale=torch.zeros(3, 8)), TypeError), (dict(dtype=torch.int8), TypeError),
                       (dict(w=torch.zeros(5, 32, dtype=torch.uint8)), ValueError),
                       (dict(w_scale=torch.zeros(5, 4).to(R.FP8)), ValueError),
                       (dict(alpha=torch.ones(2)), ValueError), (dict(alpha=torch.ones(1, device="meta")), ValueError),
                       (dict(w=w.to("meta")), ValueError), (dict(out=torch.zeros(3, 5)), ValueError),
                       (dict(out=torch.zeros(5, 3, dtype=torch.bfloat16).t()), ValueError),
                       (dict(out=torch.zeros(3, 4, dtype=torch.bfloat16)), ValueError)):
        with pytest.raises(error):
            gemm_a4w4(**{**good, **bad})
    with pytest.raises(NotImplementedError, match="multiple of 64"):
        gemm_a4w4(gpu(torch.zeros(3, 16, dtype=torch.uint8)), torch.zeros(5, 16, dtype=torch.uint8),
                  torch.zeros(3, 2).to(R.FP8), torch.zeros(5, 2).to(R.FP8))


def _layer(kind="bf16", m=2, e=2, h=128, i=128):
    gen = torch.Generator().manual_seed(0)
    w1, w2 = R.make_weights(kind, e, 2 * i, h, gen), R.make_weights(kind, e, h, i, gen)
    kw = dict(hidden_states=gpu(torch.zeros(m, h, dtype=torch.bfloat16)), w1=w1[0], w2=w2[0],
              topk_weights=torch.ones(m, 1), topk_ids=torch.zeros(m, 1, dtype=torch.int32))
    if w1[1] is not None:
        kw.update(w1_scale=w1[1], w2_scale=w2[1])
    return kw


def test_fused_experts_decode_refuses():
    from boltops_b200.fused_moe import fused_experts_decode, fused_moe_decode
    good = _layer()
    fp8, fp4 = dict(use_fp8_w8a8=True), dict(use_fp4_w4a4=True)
    cases = [
        (dict(hidden_states=gpu(torch.zeros(33, 128, dtype=torch.bfloat16))), NotImplementedError),
        (dict(hidden_states=gpu(torch.zeros(2, 128))), ValueError),
        (dict(hidden_states=gpu(torch.zeros(2, 128, dtype=torch.float16))), TypeError),
        (dict(hidden_states=gpu(torch.zeros(2, 64, dtype=torch.bfloat16))), ValueError),
        (dict(w2=good["w2"][:1]), ValueError), (dict(w1=good["w1"].to("meta")), ValueError),
        (dict(topk_ids=torch.zeros(3, 1, dtype=torch.int32)), ValueError),
        (dict(topk_ids=torch.zeros(2, 33, dtype=torch.int32), topk_weights=torch.zeros(2, 33)), ValueError),
        (dict(topk_weights=torch.ones(2, 1, device="meta")), ValueError),
        (dict(activation="relu2"), NotImplementedError), (dict(activation="swigluoai"), NotImplementedError),
        (dict(activation="nothing"), ValueError), (dict(output_dtype=torch.int8), ValueError),
        (dict(out=torch.zeros(2, 128)), ValueError), (dict(w1_scale=torch.ones(2), w2_scale=torch.ones(2)), ValueError),
        (dict(a1_global_scale=torch.ones(1)), ValueError), (dict(**fp8), ValueError), (dict(**fp4), ValueError),
        (dict(**fp8, **fp4, w1_scale=torch.ones(2), w2_scale=torch.ones(2)), ValueError),
        (dict(expert_map=torch.zeros(1, dtype=torch.int32), global_num_experts=4), ValueError),
        (dict(expert_map=torch.zeros(2, 2, dtype=torch.int32)), ValueError),
    ]
    for bad, error in cases:
        with pytest.raises(error):
            fused_experts_decode(**{**good, **bad})
    block = {**_layer("fp8_block"), **fp8}
    with pytest.raises(NotImplementedError, match="per-tensor"):
        fused_experts_decode(**block)
    with pytest.raises(NotImplementedError, match="block_shape"):
        fused_experts_decode(**block, block_shape=[64, 64])
    with pytest.raises(ValueError, match="expected"):
        fused_experts_decode(**{**block, "w1_scale": torch.ones(2, 3)}, block_shape=[128, 128])
    four = {**_layer("nvfp4"), **fp4}
    with pytest.raises(ValueError, match="block_shape"):
        fused_experts_decode(**four, block_shape=[1, 32])
    with pytest.raises(TypeError):
        fused_experts_decode(**{**four, "w2_scale": four["w2_scale"].view(torch.uint8)})
    with pytest.raises(ValueError, match="float32"):
        fused_experts_decode(**four, w1_global_scale=torch.ones(3))
    with pytest.raises(ValueError, match="whole tensor"):
        fused_experts_decode(**{**_layer("mxfp4"), **fp4}, a1_global_scale=torch.ones(1))
    with pytest.raises(NotImplementedError, match="multiples of 128"):
        fused_experts_decode(**{**_layer("mxfp4", h=96, i=128), **fp4})
    route = {k: v for k, v in good.items() if not k.startswith("topk")}
    for bad in (dict(gating_output=torch.zeros(2, 3)), dict(gating_output=torch.zeros(1, 2)),
                dict(gating_output=torch.zeros(2, 2, dtype=torch.int32)), dict(topk=3), dict(topk=0)):
        with pytest.raises(ValueError):
            fused_moe_decode(**{**route, "gating_output": torch.zeros(2, 2), "topk": 1, "renormalize": True, **bad})


@pytest.mark.parametrize("kind", ["fp8_block", "int8_block", "nvfp4", "mxfp4"])
def test_scales_in_another_order_are_refused(kind):
    from boltops_b200.fused_moe import fused_experts_decode, fused_experts_fp4
    good = _layer(kind, h=256, i=384)
    flags = dict(use_fp4_w4a4=True) if kind.endswith("fp4") else \
        {f"use_{kind[:-6]}_w8a8": True, "block_shape": [128, 128]}
    for name in ("w1_scale", "w2_scale"):
        turned = {**good, name: good[name].transpose(1, 2)}
        with pytest.raises(ValueError, match=name):
            fused_experts_decode(**turned, **flags)
        if kind.endswith("fp4"):
            with pytest.raises(ValueError, match=name):
                fused_experts_fp4(**turned)


def test_fused_experts_fp4_refuses():
    from boltops_b200.fused_moe import fused_experts_fp4
    good = _layer("nvfp4")
    for bad, error in ((dict(hidden_states=gpu(torch.zeros(2, 128))), ValueError), (dict(w1_scale=None), ValueError),
                       (dict(w1_scale=torch.zeros(2, 256, 8)), TypeError),
                       (dict(w2_scale=good["w2_scale"][:, :64]), ValueError),
                       (dict(w1=good["w1"].float()), TypeError), (dict(topk_ids=torch.zeros(2, dtype=torch.int32)), ValueError),
                       (dict(w2=good["w2"].to("meta")), ValueError), (dict(activation="relu2"), NotImplementedError),
                       (dict(output_dtype=torch.float64), ValueError), (dict(a1_global_scale=torch.ones(2)), ValueError),
                       (dict(global_num_experts=3), ValueError),
                       (dict(expert_map=torch.zeros(1, dtype=torch.int32), global_num_experts=4), ValueError)):
        with pytest.raises(error):
            fused_experts_fp4(**{**good, **bad})
    with pytest.raises(NotImplementedError, match="multiples of 64"):
        fused_experts_fp4(**_layer("nvfp4", h=96))
    gen = torch.Generator().manual_seed(0)
    odd = R.make_weights("nvfp4", 2, 100, 128, gen)
    with pytest.raises(NotImplementedError, match="16 bytes"):
        fused_experts_fp4(**{**good, "w2": odd[0], "w2_scale": odd[1]})


# ---- the reference arithmetic ------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_reference_quantiser_is_the_nearest_code(fmt):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(64, 8 * R.BLOCK[fmt], generator=gen)
    codes, scales, values = R.fp4_quant(fmt, x)
    assert torch.equal(values, R.fp4_values(fmt, codes, scales))
    s = (scales.view(R.FP8).double() if fmt == "nvfp4" else torch.exp2(scales.double() - 127))[..., None]
    grid = torch.cat((R.E2M1, -R.E2M1))
    best = ((grid * s[..., None]) - x.double().unflatten(-1, (-1, R.BLOCK[fmt]))[..., None]).abs().amin(-1)
    off = (values - x.double()).abs().unflatten(-1, (-1, R.BLOCK[fmt]))
    assert torch.allclose(off, best, rtol=0, atol=1e-12)
    if fmt == "mxfp4":      # nothing saturates: the largest magnitude is at most 6 scales
        assert (x.double().abs().unflatten(-1, (-1, 32)) <= 6 * s).all()


@pytest.mark.parametrize("shape", [(2, 4), (1, 2), ()])
def test_an_expert_map_of_several_rows_is_refused(shape):
    """The tiles' experts are looked up in it by one index: a map of two rows would be read past its end."""
    from boltops_b200.fused_moe import fused_experts_decode, fused_experts_fp4
    good = {**_layer("nvfp4"), "expert_map": torch.zeros(shape, dtype=torch.int32)}
    for call, more in ((fused_experts_fp4, {}), (fused_experts_decode, dict(use_fp4_w4a4=True))):
        with pytest.raises(ValueError, match="one row"):
            call(**good, **more)


@pytest.fixture
def calls(monkeypatch):
    """The C entries that a call reaches, with their argument structures: nothing is launched."""
    from boltops_b200 import _cabi
    from boltops_b200.fused_moe import ops
    made = []

    class Lib:
        def __getattr__(self, name):
            def entry(*args):
                made.append((name, args))
                return 64 if name.endswith("_bytes") else 0
            return entry

    monkeypatch.setattr(_cabi, "load", lambda: Lib())
    monkeypatch.setattr(_cabi, "stream_of", lambda t: 0)
    monkeypatch.setattr(_cabi, "call", lambda device, fn, *args: fn(*args))
    monkeypatch.setattr(ops, "stream_of", lambda t: 0)
    monkeypatch.setattr(ops, "device_status", lambda d: torch.zeros(1, dtype=torch.int32))
    return made


@pytest.mark.parametrize("kind", ["bf16", "nvfp4"])
def test_few_token_layer_leaves_the_reserved_sms_free(calls, monkeypatch, kind):
    from types import SimpleNamespace
    from boltops_b200.fused_moe import fused_experts_decode, ops
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda d: SimpleNamespace(multi_processor_count=148))
    flags = dict(use_fp4_w4a4=True) if kind == "nvfp4" else {}
    for reserve, used in ((0, 0), (20, 128)):
        monkeypatch.setattr(ops, "_gemm_sm_reserve", reserve)
        calls.clear()
        fused_experts_decode(**_layer(kind), **flags)
        assert [args[0].sm_count for name, args in calls if name == "bolt_moe_decode"] == [used]


@pytest.mark.parametrize("fmt,m,n,k,few", [
    ("nvfp4", 32, 4096, 7168, True), ("nvfp4", 16, 8192, 8192, True), ("nvfp4", 8, 16384, 8192, True),
    ("nvfp4", 17, 8192, 8192, False), ("nvfp4", 32, 16384, 8192, False), ("nvfp4", 33, 128, 128, False),
    ("mxfp4", 32, 4096, 4096, True), ("mxfp4", 16, 4096, 7168, True), ("mxfp4", 8, 8192, 8192, True),
    ("mxfp4", 32, 4096, 7168, False), ("mxfp4", 9, 8192, 8192, False), ("mxfp4", 1, 16384, 8192, False)])
def test_the_form_of_a_4bit_product_goes_by_rows_and_weights(calls, fmt, m, n, k, few):
    """On which side the measured times of the two forms lie, per format."""
    from boltops_b200.fp4 import FORMATS
    from boltops_b200.gemm import gemm_a4w4
    _, block, scale_dtype = FORMATS[fmt]
    rows = lambda r: (torch.empty(r, k // 2, dtype=torch.uint8), torch.empty(r, k // block, dtype=scale_dtype))  # noqa: E731
    (x, xs), (w, ws) = rows(m), rows(n)
    gemm_a4w4(gpu(x), w, xs, ws)
    assert [name for name, _ in calls] == (["bolt_fp4_gemm_few"] if few else ["bolt_fp4_tile_scales", "bolt_fp4_gemm"])


def test_few_token_layer_says_how_many_kernels_it_launches(lib):
    """Two; one more where 8-bit rows, or activations, are quantised by a kernel of their own; as many again for
    every part of a batch whose 4-bit rows do not fit together."""
    from boltops_b200 import _cabi

    def count(kind, m, h, i, k=8):
        a = _cabi.DecodeArgs(kind=getattr(_cabi, "DECODE_" + kind), num_tokens=m, topk=k, hidden=h, inter=i, model_dim=1024,
                             num_experts=8, global_num_experts=8, sm_count=148)
        return lib.bolt_moe_decode_kernel_count(a)
    assert count("BF16", 0, 1024, 512) == 0 and count("BF16", 32, 1024, 512) == 2
    for kind in ("FP8_BLOCK", "INT8_BLOCK", "FP8_CHANNEL", "INT8_CHANNEL"):
        assert count(kind, 8, 1024, 512) == 2
        assert count(kind, 8, 16384, 256) == 3      # the rows
        assert count(kind, 8, 1024, 2176) == 3      # the activations
        assert count(kind, 9, 1024, 512) == 4       # both
    assert count("NVFP4", 32, 1024, 512) == 2 and count("NVFP4", 32, 16384, 512) == 8       # four times eight tokens
    assert count("BF16", 33, 1024, 512) == -1 and count("BF16", 1, 1020, 512) == -1
    assert lib.bolt_moe_decode_kernel_count(None) == -1


@pytest.mark.parametrize("kernels", [2, 4])
def test_few_token_layer_counts_its_launches(calls, monkeypatch, kernels):
    from boltops_b200 import _cabi
    from boltops_b200.fused_moe import fused_experts_decode, ops
    lib = _cabi.load()
    type(lib).bolt_moe_decode_kernel_count = lambda self, args: kernels
    monkeypatch.setattr(_cabi, "load", lambda: lib)
    before = ops.launch_count()
    fused_experts_decode(**_layer())
    assert ops.launch_count() - before == kernels


def test_a_sort_counts_one_kernel_or_two(calls):
    from boltops_b200.fused_moe import ops
    ids = gpu(torch.zeros(4, 2, dtype=torch.int32))
    weights = gpu(torch.ones(4, 2))
    for sort in (lambda: ops.moe_sorting_ck(ids, weights, 4), lambda: ops.moe_align_block_size(ids, 32, 4)):
        before = ops.launch_count()
        sort()      # (a workspace of 64 bytes: the form for many routes, which has no scan kernel)
        assert ops.launch_count() - before == 2


def test_expired_waits_are_named(monkeypatch):
    """Every code that the 4-bit kernels can leave has a meaning in the header and in the error."""
    from boltops_b200 import _cabi
    from boltops_b200.fused_moe import ops
    header = (ROOT / "include" / "boltops_b200.h").read_text()
    codes = set()
    for source in ("few_tokens.cu", "fp4_gemm.cu"):
        text = (ROOT / "boltops_b200" / "csrc" / source).read_text()
        codes |= {int(c) for c in re.findall(r"\bstatus, (\d+)\)", text)}
    assert codes == {30, 40, 41, 42, 43}
    for code in codes:
        assert f"set to {code} by a wait" in header or f"{code} for " in header
        word = torch.tensor([code], dtype=torch.int32)
        monkeypatch.setattr(ops, "device_status", lambda d: word)
        with pytest.raises(_cabi.BoltError, match="30 few-token layer" if code == 30 else "40-43 tiled 4-bit product"):
            ops.check_device_status(torch.device("cuda"))
        assert not word.any()
