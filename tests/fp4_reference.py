"""The 4-bit formats and the expert layer in 64 bits, with bounds of what fp32 kernels may be off by.

A layer's bound is propagated term by term: a sum of n products in fp32, in any order, is off by at
most n * 2^-23 of the sum of magnitudes (2^-24 for each of the two roundings of a product and an
addition); a quantiser may pick another code only where its input's error reaches across a border,
so its output lies between what it gives for both ends of the input's interval.
"""
from __future__ import annotations

import torch

FP8 = torch.float8_e4m3fn
E2M1 = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), dtype=torch.float64)
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def e2m1(t: torch.Tensor) -> torch.Tensor:
    """Index 0..7 of the nearest magnitude, of two as near the even one, for t >= 0."""
    code = torch.zeros(t.shape, dtype=torch.long)
    for i in range(7):
        middle = (E2M1[i] + E2M1[i + 1]) / 2
        code += (t >= middle) if i % 2 else (t > middle)
    return code


def fp4_scales(fmt: str, y: torch.Tensor):
    """Stored scales and their values for blocks [..., n, block] of finite doubles."""
    amax = y.abs().amax(-1)
    if fmt == "nvfp4":
        # (the recipe multiplies in fp32 with the rounded 1/6)
        s = (amax.float() * torch.tensor(1 / 6, dtype=torch.float32)).clamp(max=448).to(FP8)
        return s, s.double()
    # smallest 2^e >= amax / 6; frexp: amax = part * 2^e', part in [0.5, 1)
    part, e = torch.frexp(amax)
    e = e - torch.where(part <= 0.75, 3, 2)
    byte = torch.where(amax == 0, 0, (e + 127).clamp(0, 254))
    return byte.to(torch.uint8), torch.exp2(byte.double() - 127)


def fp4_quant(fmt: str, x: torch.Tensor, g=None):
    """(packed codes, stored scales, values) of x [..., K] (CPU); a block with a NaN or an infinity
    gets the NaN scale and codes 0."""
    y = x.double()
    if g is not None:       # the recipe multiplies with the rounded reciprocal, in fp32
        y = (x.float() * (1.0 / g.float())).double()
    y = y.unflatten(-1, (-1, BLOCK[fmt]))
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    stored, s = fp4_scales(fmt, y)
    t = torch.where(s[..., None] > 0, y.abs() / s[..., None].clamp_min(2.0 ** -140), 0.0)
    idx = e2m1(t)
    neg = torch.signbit(y) & (s[..., None] > 0) & ~bad[..., None]
    codes = (idx + 8 * neg.long()).flatten(-2).to(torch.uint8)
    stored = stored.view(torch.uint8).clone()
    stored[bad] = 0x7F if fmt == "nvfp4" else 0xFF
    values = torch.where(neg, -E2M1[idx], E2M1[idx]) * s[..., None]
    values = torch.where(bad[..., None], float("nan"), values).flatten(-2)
    if g is not None:
        values = values * g.double()
    return codes[..., 0::2] + codes[..., 1::2] * 16, stored, values


def fp4_values(fmt: str, codes: torch.Tensor, scales: torch.Tensor, g=None) -> torch.Tensor:
    """Packed codes and stored scales as doubles (g: one scale, or one per matrix of [E, N, K])."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = torch.where(c >= 8, -E2M1[c & 7], E2M1[c & 7])
    b = scales.view(torch.uint8)
    s = b.view(FP8).double() if fmt == "nvfp4" else torch.exp2(b.double() - 127)
    if g is not None:
        s = s * g.double().view(-1, *[1] * (s.dim() - 1))
    return (v.unflatten(-1, (-1, BLOCK[fmt])) * s[..., None]).flatten(-2)


# ---- experts -----------------------------------------------------------------------------
KINDS = ("bf16", "f16", "fp8_block", "int8_block", "fp8_channel", "int8_channel", "nvfp4", "mxfp4")


def make_weights(kind: str, e: int, n: int, k: int, gen, spread=0.05):
    """(stored weights, stored scales or None, whole-matrix scales or None, values in 64 bits)."""
    w = torch.randn(e, n, k, generator=gen) * spread
    if kind in ("bf16", "f16"):
        w = w.to(torch.bfloat16 if kind == "bf16" else torch.float16)
        return w, None, None, w.double()
    if kind in BLOCK:
        g = None
        if kind == "nvfp4":
            g = w.abs().amax((1, 2)) / (448 * 6)
            w = w / g[:, None, None]
        codes, stored, _ = fp4_quant(kind, w)
        scales = stored.view(FP8) if kind == "nvfp4" else stored
        return codes, scales, g, fp4_values(kind, codes, stored, g)
    largest, dtype = (448.0, FP8) if kind.startswith("fp8") else (127.0, torch.int8)
    to = (lambda v: v.to(FP8)) if dtype == FP8 else (lambda v: v.round().clamp(-127, 127).to(torch.int8))
    if kind.endswith("block"):
        v = w.view(e, n // 128, 128, k // 128, 128)
        s = v.abs().amax((2, 4)) / largest
        q = to(v / s[:, :, None, :, None])
        return q.view(e, n, k), s, None, (q.double() * s.double()[:, :, None, :, None]).view(e, n, k)
    s = w.abs().amax(-1) / largest
    q = to(w / s[..., None])
    return q, s, None, q.double() * s.double()[..., None]


def quant_rows(kind: str, v: torch.Tensor, g=None, scale_of=None) -> torch.Tensor:
    """Rows after the activation quantiser, as doubles.  `scale_of`: rows that the scales come from."""
    src = v if scale_of is None else scale_of
    if kind in ("bf16", "f16"):
        return v.double()
    if kind in BLOCK:
        inv = 1.0 if g is None else (1.0 / g.float()).double()
        y = (v.double() * inv).unflatten(-1, (-1, BLOCK[kind]))
        z = (src.double() * inv).unflatten(-1, (-1, BLOCK[kind]))
        _, s = fp4_scales(kind, z)
        t = torch.where(s[..., None] > 0, y.abs() / s[..., None].clamp_min(2.0 ** -140), 0.0)
        q = E2M1[e2m1(t)] * s[..., None]
        return (torch.where(y < 0, -q, q)).flatten(-2) * (1.0 if g is None else g.double())
    group = 128 if kind.endswith("block") else v.shape[-1]
    largest = 448.0 if kind.startswith("fp8") else 127.0
    z = src.float().unflatten(-1, (-1, group))
    s = z.abs().amax(-1, keepdim=True).clamp_min(1e-10) * torch.tensor(1 / largest, dtype=torch.float32)
    y = v.float().unflatten(-1, (-1, group)) * (1.0 / s)      # the recipe scales in fp32
    q = y.clamp(-448, 448).to(FP8).double() if largest == 448 else y.round().clamp(-128, 127).double()
    return (q * s.double()).flatten(-2)


def _quant_interval(kind, a, err, g):
    """Quantised rows and how far a quantiser may get from them when its input is off by `err`."""
    mid = quant_rows(kind, a, g)
    far = torch.zeros_like(mid)
    for src in (a, a.sign() * (a.abs() + err), a.sign() * (a.abs() - err).clamp_min(0)):
        for v in (a - err, a + err):
            far = torch.maximum(far, (quant_rows(kind, v, g, scale_of=src) - mid).abs())
    return mid, far


def layer(kind, x, w1, w2, ids, weights, out_dtype, *, a1=None, a2=None, act=None, scale=1.0, emap=None,
          round_routes=None):
    """The layer in 64 bits and the bound of an fp32 implementation, both [M, H].  `w1`, `w2` values;
    `act(gate, up)` with slopes at most 1.2 in |gate| and |up| (default SiLU); `round_routes`: type
    that each route's result is rounded to before the sum over routes."""
    m, topk = ids.shape
    xq = quant_rows(kind, x, a1)
    out = torch.zeros(m, w2.shape[1], dtype=torch.float64)
    bound = torch.zeros_like(out)
    inter = w1.shape[1] // 2
    act = act or (lambda gate, up: gate * torch.sigmoid(gate) * up)
    for i in range(m):
        for j in range(topk):
            e = int(ids[i, j])
            if emap is not None:
                e = int(emap[e]) if 0 <= e < emap.numel() else -1
            if not 0 <= e < w1.shape[0]:
                continue
            both = w1[e] @ xq[i]
            # sums, and the few products with scales around them
            err = (w1[e].abs() @ xq[i].abs()) * (xq.shape[1] + 16) * 2.0 ** -23
            gate, up = both[:inter], both[inter:]
            a = act(gate, up)
            da = 1.2 * (up.abs() + err[inter:]) * err[:inter] + 1.2 * (gate.abs() + err[:inter]) * err[inter:] \
                + a.abs() * 2.0 ** -20
            if kind in ("bf16", "f16"):
                q, dq = a, da + (a.abs() + da) * half_step(x.dtype)
            else:
                q, dq = _quant_interval(kind, a[None], da[None], a2)
                q, dq = q[0], dq[0]
            y = w2[e] @ q
            mag = w2[e].abs() @ (q.abs() + dq)
            dy = w2[e].abs() @ dq + mag * (inter + 16) * 2.0 ** -23
            if round_routes is not None:
                dy = dy + (y.abs() + dy) * half_step(round_routes)
            wt = float(weights[i, j]) * scale
            out[i] += wt * y
            bound[i] += abs(wt) * (dy + (y.abs() + dy) * 2.0 ** -20)
    bound += (out.abs() + bound) * half_step(out_dtype)
    # below the normal range a half step is absolute
    return out, bound + torch.finfo(out_dtype).tiny * half_step(out_dtype) * 2
