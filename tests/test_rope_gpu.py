"""Rotary positions on the GPU against the formula in 64 bits.

Tolerance per element: the result is rounded once to its type (half a step,
eps / 2 relative).  Before that, in steps of 2^-24 of the amplitude times
|x0| + |x1|: the fraction of a turn rounded to fp32 (at most pi steps of
angle), sine and cosine (2), their product with the amplitude (1), the two
products and the sum (2): 8.2, taken as 12.
"""
import math

import pytest
import torch

import bwpp
from test_operators_cpu import frequencies

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def call(ctx, dtype):
    return {"bf16": ctx.rope_bf16, "f16": ctx.rope_f16, "f32": ctx.rope_f32}[dtype]


def turned(x, pos, f, interleaved, sign, amp):
    """x [tokens, heads, head_dim] in 64 bits, and sum |x0| + |x1| per element."""
    R = 2 * len(f)
    a = pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    cos, sin = a.cos()[:, None] * amp, a.sin()[:, None] * (sign * amp)
    x = x.double()
    y, mag = x.clone(), x.abs() * 0
    i0 = slice(0, R, 2) if interleaved else slice(0, R // 2)
    i1 = slice(1, R, 2) if interleaved else slice(R // 2, R)
    y[..., i0] = x[..., i0] * cos - x[..., i1] * sin
    y[..., i1] = x[..., i1] * cos + x[..., i0] * sin
    mag[..., i0] = mag[..., i1] = x[..., i0].abs() + x[..., i1].abs()
    return y, mag


def check(got, x, pos, f, interleaved, sign=1.0, amp=1.0):
    want, mag = turned(x, pos, f, interleaved, sign, amp)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 12 * 2.0**-24 * amp * mag
    if x.dtype == torch.float16:
        tol = tol + 2.0**-25  # half a step of the subnormals
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,hq,hk,hd,R", [(1, 16, 16, 128, 128), (1, 1, 1, 2, 2), (3, 4, 1, 64, 64),
                                               (37, 3, 3, 96, 64), (5, 2, 1, 80, 40), (7, 5, 0, 6, 6),
                                               (129, 8, 2, 256, 256), (11, 2, 2, 34, 18), (9, 0, 3, 20, 12),
                                               (300, 32, 8, 128, 128)])
def test_rope(ctx, dtype, interleaved, tokens, hq, hk, hd, R):
    t = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(tokens * hd + R)
    q = torch.randn(tokens, max(hq, 1), hd, device="cuda", generator=g).to(t)
    k = torch.randn(tokens, max(hk, 1), hd, device="cuda", generator=g).to(t)
    pos = torch.randint(-5, 2**31 - 1, (tokens,), device="cuda", generator=g).int()
    pos[0] = 2**31 - 1
    for positions, inverse in ((None, 0), (pos, 1)):
        qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
        call(ctx, dtype)(q, k, qo, ko, bwpp.rope_table(R), tokens, hq, hk, hd, max(hq, 1) * hd, max(hk, 1) * hd,
                         max(hq, 1) * hd, max(hk, 1) * hd, positions=positions, pos0=70000, interleaved=interleaved,
                         inverse=inverse)
        ctx.sync()
        p = pos if positions is not None else 70000 + torch.arange(tokens, device="cuda")
        for o, x, h in ((qo, q, hq), (ko, k, hk)):
            if h:
                check(o, x, p, frequencies(R), interleaved, -1.0 if inverse else 1.0)
            else:
                assert bool(torch.isnan(o).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,hq,hk,hd,R", [(40000, 5, 3, 64, 32), (30000, 3, 11, 10, 10), (20000, 24, 24, 96, 64),
                                               (90000, 1, 1, 20, 12), (70000, 2, 1, 34, 34), (30000, 0, 2, 128, 128)])
def test_many_tokens(ctx, dtype, interleaved, tokens, hq, hk, hd, R):
    """Batches of heads, and one or two heads a token; per sequence of 10000 and
    from token-major to head-major."""
    t, seq = TYPES[dtype], 10000
    g = torch.Generator(device="cuda").manual_seed(tokens + hd)
    q = torch.randn(tokens, max(hq, 1), hd, device="cuda", generator=g).to(t)
    k = torch.randn(tokens, max(hk, 1), hd, device="cuda", generator=g).to(t)
    qo, ko = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    call(ctx, dtype)(q, k, qo, ko, bwpp.rope_table(R), tokens, hq, hk, hd, max(hq, 1) * hd, max(hk, 1) * hd, hd, hd,
                     seq=seq, pos0=3, interleaved=interleaved, head_major_out=1)
    ctx.sync()
    pos = 3 + torch.arange(tokens, device="cuda") % seq
    for o, x, h in ((qo, q, hq), (ko, k, hk)):
        if h:
            o = o.view(tokens // seq, h, seq, hd).transpose(1, 2).reshape(tokens, h, hd)
            check(o, x, pos, frequencies(R), interleaved)


@pytest.mark.parametrize("scaling,factor,amp", [("linear", 4.0, 1.0), ("base", 8.0, 1.0), ("parts", 16.0, 1.277)])
def test_scaled_for_long_contexts(ctx, scaling, factor, amp):
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(50, 4, 128, device="cuda", generator=g)
    o = torch.empty_like(q)
    table = bwpp.rope_table(128, scaling=scaling, factor=factor, context=4096.0, amplitude=amp)
    ctx.rope_f32(q, None, o, None, table, 50, 4, 0, 128, 512, 0, 512, 0, pos0=65000)
    ctx.sync()
    check(o, q, 65000 + torch.arange(50, device="cuda"), frequencies(128, scaling=scaling, factor=factor), 0,
          amp=table.amplitude)


def test_in_place_inside_a_fused_product_and_back(ctx):
    """q and k of a [tokens, 3 D] product turn in place; v and the columns
    behind rotary_dim keep their bits; turning back is the inverse."""
    T, H, hd, R = 77, 3, 64, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(T, 3 * H * hd, device="cuda", generator=g)
    before = qkv.clone()
    k = qkv.data_ptr() + H * hd * 4
    table = bwpp.rope_table(R)
    for inverse in (0, 1):
        ctx.rope_f32(qkv, k, qkv, k, table, T, H, H, hd, 3 * H * hd, 3 * H * hd, 3 * H * hd, 3 * H * hd, seq=11,
                     inverse=inverse)
        if not inverse:
            ctx.sync()
            a, b = qkv.view(T, 3, H, hd), before.view(T, 3, H, hd)
            assert torch.equal(a[:, 2], b[:, 2]) and torch.equal(a[..., R:], b[..., R:])
            pos = torch.arange(T, device="cuda") % 11
            for i in (0, 1):
                check(a[:, i].contiguous(), b[:, i].contiguous(), pos, frequencies(R), 0)
    ctx.sync()
    # two turns, each within 12 steps of |x0| + |x1|
    assert float((qkv - before).abs().max()) <= 2 * 12 * 2.0**-24 * 2 * float(before.abs().max())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,S,hq,hk,hd", [(2, 33, 4, 2, 64), (1, 1, 2, 2, 128), (3, 5, 3, 1, 10)])
def test_layouts_convert(ctx, dtype, B, S, hq, hk, hd):
    t = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(S)
    q = torch.randn(B * S, hq, hd, device="cuda", generator=g).to(t)
    k = torch.randn(B * S, hk, hd, device="cuda", generator=g).to(t)
    table = bwpp.rope_table(hd)

    def run(xq, xk, hin, hout):
        pad = 8 if hout else 0  # head-major rows with a pitch
        oq = torch.zeros((B, hq, S, hd + pad) if hout else (B * S, hq, hd), dtype=t, device="cuda")
        ok = torch.zeros((B, hk, S, hd + pad) if hout else (B * S, hk, hd), dtype=t, device="cuda")
        call(ctx, dtype)(xq, xk, oq, ok, table, B * S, hq, hk, hd, hd if hin else hq * hd, hd if hin else hk * hd,
                         hd + pad if hout else hq * hd, hd + pad if hout else hk * hd, seq=S, pos0=9,
                         head_major_in=hin, head_major_out=hout)
        ctx.sync()
        if hout:
            assert not bool(oq[..., hd:].any()) and not bool(ok[..., hd:].any())
            return oq[..., :hd].transpose(1, 2).reshape(B * S, hq, hd), ok[..., :hd].transpose(1, 2).reshape(B * S, hk, hd)
        return oq, ok

    want = run(q, k, 0, 0)
    major = [x.view(B, S, -1, hd).transpose(1, 2).contiguous() for x in (q, k)]
    for hin, hout in ((0, 1), (1, 0), (1, 1)):
        got = run(*(major if hin else (q, k)), hin, hout)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (hin, hout)
    check(want[0], q, 9 + torch.arange(B * S, device="cuda") % S, frequencies(hd), 0)


def test_odd_addresses_and_pitches(ctx):
    """An address that is off by one element, odd pitches: padding stays."""
    T, H, hd = 13, 2, 32
    g = torch.Generator(device="cuda").manual_seed(4)
    buf = torch.randn(T * 71 + 9, device="cuda", generator=g).bfloat16()
    out = torch.zeros(T * 67 + 9, device="cuda").bfloat16()
    ctx.rope_bf16(buf.data_ptr() + 2, None, out.data_ptr() + 6, None, bwpp.rope_table(hd), T, H, 0, hd, 71, 0, 67, 0,
                  interleaved=1)
    ctx.sync()
    x = buf[1:1 + T * 71].view(T, 71)[:, :H * hd].reshape(T, H, hd)
    o = out[3:3 + T * 67].view(T, 67)
    check(o[:, :H * hd].reshape(T, H, hd), x, torch.arange(T, device="cuda"), frequencies(hd), 1)
    assert not bool(o[:, H * hd:].any()) and not bool(out[:3].any())


def test_offsets_past_32_bits(ctx):
    ld = 2**31
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(2 * ld + 256, dtype=torch.bfloat16, device="cuda")
    rows = torch.as_strided(x, (3, 2, 128), (ld, 128, 1))
    rows.copy_(torch.randn(3, 2, 128, device="cuda", generator=g))
    src = rows.clone()
    ctx.rope_bf16(x, None, x, None, bwpp.rope_table(128), 3, 2, 0, 128, ld, 0, ld, 0, pos0=5)
    ctx.sync()
    check(rows.clone(), src, 5 + torch.arange(3, device="cuda"), frequencies(128), 0)


def test_gradient_is_the_transpose(ctx):
    """<rope(x), g> == <x, rope_inverse(g)>, and the derivative by differences."""
    T, H, hd, R = 40, 2, 96, 64
    g = torch.Generator(device="cuda").manual_seed(6)
    x, gy, d = (torch.randn(T, H, hd, device="cuda", generator=g) for _ in range(3))
    table = bwpp.rope_table(R, amplitude=1.2)
    y, gx, yp, ym = (torch.empty_like(x) for _ in range(4))
    for src, dst, inv in ((x, y, 0), (gy, gx, 1), (x + 0.5 * d, yp, 0), (x - 0.5 * d, ym, 0)):
        ctx.rope_f32(src, None, dst, None, table, T, H, 0, hd, H * hd, 0, H * hd, 0, pos0=1000, inverse=inv)
    ctx.sync()
    n = T * H * hd
    # each side: n products whose factors are 12 steps off, magnitudes about 1
    tol = 4 * 12 * 2.0**-24 * n
    assert abs(float((y.double() * gy.double()).sum() - (x.double() * gx.double()).sum())) <= tol
    diff = ((yp.double() - ym.double()) * gy.double()).sum()
    assert abs(float(diff - (d.double() * gx.double()).sum())) <= tol


def test_captured_and_replayed_on_another_stream(ctx):
    stream = torch.cuda.Stream()
    c = bwpp.Ctx(0, stream.cuda_stream)
    x = torch.randn(64, 4, 128, device="cuda")
    o, want = torch.empty_like(x), torch.empty_like(x)
    table = bwpp.rope_table(128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.rope_f32(x, None, o, None, table, 64, 4, 0, 128, 512, 0, 512, 0)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        o.zero_()
        graph.replay()
        ctx.rope_f32(x, None, want, None, table, 64, 4, 0, 128, 512, 0, 512, 0)
        torch.cuda.synchronize()
        assert torch.equal(o, want)
    del graph
    c.close()


def test_refusals(ctx):
    x = torch.zeros(4, 64, device="cuda")
    ok = dict(q=x, k=None, q_out=x, k_out=None, table=bwpp.rope_table(32), tokens=4, heads_q=2, heads_k=0,
              head_dim=32, ldq=64, ldk=0, ldq_out=64, ldk_out=0)
    ctx.rope_f32(**ok)
    bad = [dict(head_dim=16), dict(ldq=63), dict(ldq_out=60), dict(q=None), dict(q_out=None),
           dict(table=bwpp.RopeTable()), dict(ldq_out=65), dict(seq=3, head_major_in=1, head_major_out=1),
           dict(seq=2, head_major_out=1), dict(heads_k=1, ldk=32, ldk_out=32)]
    for b in bad:
        with pytest.raises(bwpp.BwppError) as e:
            ctx.rope_f32(**{**ok, **b})
        assert e.value.status == bwpp.ERR_ARG, b
    ctx.rope_f32(**{**ok, "tokens": 0})
    ctx.sync()


@pytest.mark.parametrize("heads", [2**31, 2**32 - 1])
def test_2_31_heads_are_refused(ctx, heads):
    """Head major, where no pitch grows with the heads."""
    x = torch.zeros(16, device="cuda")
    for hq, hk in ((heads, 0), (0, heads), (1, heads)):
        with pytest.raises(bwpp.BwppError) as e:
            ctx.rope_f32(x, x, x, x, bwpp.rope_table(2), 1, hq, hk, 2, 2, 2, 2, 2, head_major_in=1, head_major_out=1)
        assert e.value.status == bwpp.ERR_ARG
    ctx.sync()
