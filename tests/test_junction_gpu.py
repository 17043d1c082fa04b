"""The junction between decoder blocks (norm after, gate, scaled residual, norm
before) on the GPU, forward and gradient, against the formula in 64 bits.

Tolerances (relative Frobenius).  All arithmetic is fp32: a row's sum of squares
adds at most 16 terms in a thread, then 10 levels of a tree, and each element
sees about a dozen more roundings, 40 * 2^-24 = 2.4e-6; a result that is rounded
to its type adds half a step, eps / 2.  h' and dh are sums whose parts may
cancel, so their error is taken relative to the parts.  A column sum over n rows
adds its terms one after the other in a chunk of ceil(n / (4 * 148)) rows, then
ceil(chunks / 32) + 32 partial sums: that many steps, plus 40, of 2^-24 of the sum
of the terms' magnitudes.
"""
import math

import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
STEP = 2.0**-24
ROW = 40 * STEP


def fwd(ctx, dtype):
    return {"bf16": ctx.junction_fwd_bf16, "f16": ctx.junction_fwd_f16, "f32": ctx.junction_fwd_f32}[dtype]


def bwd(ctx, dtype):
    return {"bf16": ctx.junction_bwd_bf16, "f16": ctx.junction_bwd_f16, "f32": ctx.junction_bwd_f32}[dtype]


def wide(t):
    return None if t is None else t.double()


def rms(x, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def after(b, gain_post, gate, rows, gate_rows, norm_after, eps):
    """gate * u in 64 bits."""
    u = rms(b, eps) if norm_after else b
    if norm_after and gain_post is not None:
        u = u * gain_post
    if gate is not None:
        at = torch.arange(rows, device=b.device) // gate_rows
        u = u * gate[at]
    return u


def make(dtype, rows, cols, gate_rows, norm_after, seed, pad=0, gains=True):
    t = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = {"h": rnd(rows, cols + pad) * 3, "b": (rnd(rows, cols + pad) * 0.5).to(t),
         "dh_out": rnd(rows, cols + pad), "dy": rnd(rows, cols + pad).to(t),
         "gain_post": 1 + 0.1 * rnd(cols) if norm_after and gains else None,
         "gain_pre": 1 + 0.1 * rnd(cols) if gains else None, "gate": None}
    if gate_rows is not None:
        x["gate"] = 0.5 + 0.3 * rnd(-(-rows // (gate_rows or rows)), cols + pad)
    return x


def close(got, want, parts, rel):
    """|got - want|_F <= rel |parts|_F."""
    err, size = float((got.double() - want).norm()), float(parts.norm())
    assert err <= rel * size, (err / max(size, 1e-300), rel)


SHAPES = [(1, 1), (1, 2048), (3, 5), (2, 8), (7, 33), (33, 256), (5, 257), (9, 512), (4, 1000), (13, 1003),
          (6, 1024), (10, 2048), (3, 2500), (5, 4096), (3, 5001), (2, 8192), (2, 9001), (2, 16384), (1, 20000),
          (2, 16400)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(ctx, dtype, rows, cols):
    for gate_rows, norm_after, sh, sb in ((None, 1, 1.0, 1.0), (0, 1, 0.7, 1.3), (1, 0, 1.0, -0.5), (2, 1, 2.0, 1.0)):
        x = make(dtype, rows, cols, gate_rows, norm_after, rows + cols)
        ho, y = torch.full_like(x["h"], float("nan")), torch.full_like(x["b"], float("nan"))
        fwd(ctx, dtype)(x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"], ho, y, rows, cols,
                        gate_rows=gate_rows or 0, norm_after=norm_after, scale_h=sh, scale_b=sb, eps_post=1e-6)
        ctx.sync()
        u = after(wide(x["b"]), wide(x["gain_post"]), wide(x["gate"]), rows, gate_rows or rows, norm_after, 1e-6)
        sh, sb = float(torch.tensor(sh)), float(torch.tensor(sb))
        want = sh * wide(x["h"]) + sb * u
        parts = (sh * wide(x["h"])).abs() + (sb * u).abs()
        close(ho, want, parts, ROW)
        wy = rms(want, 1e-5) * wide(x["gain_pre"])
        # y carries h's error, relative to the parts h' is the sum of
        close(y, wy, wy.abs() + rms(parts, 1e-5), 2 * ROW + torch.finfo(y.dtype).eps / 2)


def check_backward(ctx, dtype, rows, cols, gate_rows, norm_after, sh=1.0, sb=1.0, pad=0, gains=True, use_dh=True,
                   use_dy=True):
    x = make(dtype, rows, cols, gate_rows, norm_after, rows * 3 + cols, pad, gains)
    groups = 0 if x["gate"] is None else x["gate"].shape[0]
    out = {"dh": torch.full_like(x["h"], 7.0), "db": torch.full_like(x["b"], 7.0),
           "dgain_post": torch.full((cols,), 7.0, device="cuda") if norm_after else None,
           "dgate": torch.full((groups, cols + pad), 7.0, device="cuda") if groups else None,
           "dgain_pre": torch.full((cols,), 7.0, device="cuda")}
    ld = cols + pad
    bwd(ctx, dtype)(x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"], x["dh_out"] if use_dh else None,
                    x["dy"] if use_dy else None, out["dh"], out["db"], out["dgain_post"], out["dgate"],
                    out["dgain_pre"], rows, cols, gate_rows=gate_rows or 0, norm_after=norm_after, scale_h=sh,
                    scale_b=sb, eps_post=1e-6, ldh=ld, ldb=ld, ldy=ld, ldgate=ld)
    ctx.sync()
    if pad:
        for k in ("dh", "db", "dgate"):
            if out[k] is not None:
                assert bool((out[k][:, cols:] == 7.0).all()), k
    cut = {k: v[:, :cols] if v is not None and v.dim() == 2 else v for k, v in {**x, **out}.items()}
    h, b, gate = (wide(cut[k]) for k in ("h", "b", "gate"))
    gp = wide(x["gain_post"]) if x["gain_post"] is not None else torch.ones(cols, dtype=torch.float64, device="cuda")
    gq = wide(x["gain_pre"]) if x["gain_pre"] is not None else torch.ones(cols, dtype=torch.float64, device="cuda")
    sh, sb = float(torch.tensor(sh)), float(torch.tensor(sb))
    leaf = {"h": h.requires_grad_(), "gq": gq.requires_grad_()}
    dH = cut["dh_out"].double() if use_dh else torch.zeros_like(h)
    parts = dH.abs()
    if use_dy:
        (rms(leaf["h"], 1e-5) * leaf["gq"]).backward(wide(cut["dy"]))
        dH = dH + h.grad
        r = (h.detach().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        g = (gq.detach() * wide(cut["dy"])).abs()
        hat = (h.detach() * r).abs()
        parts = parts + r * (g + hat * (g * hat).mean(-1, keepdim=True))
    b, gp = b.requires_grad_(), gp.requires_grad_()
    gate = gate.requires_grad_() if gate is not None else None
    (sb * after(b, gp, gate, rows, gate_rows or rows, norm_after, 1e-6)).backward(dH.detach())
    close(cut["dh"], sh * dH.detach(), sh * parts, ROW)
    # db: the same steps once more on e = scale_b dH, whose parts are `parts`
    bd, gd = b.detach(), torch.ones_like(b) if gate is None else gate.detach()[torch.arange(rows, device="cuda") // (gate_rows or rows)]
    du = (sb * gd).abs() * parts
    rb = (bd.square().mean(-1, keepdim=True) + 1e-6).rsqrt() if norm_after else torch.ones_like(bd[:, :1])
    bh = (bd * rb).abs()
    gu = gp.detach().abs() * du if norm_after else du
    db_parts = rb * (gu + bh * (gu * bh).mean(-1, keepdim=True)) if norm_after else du
    close(cut["db"], b.grad, b.grad.abs() + db_parts * (2 * ROW / (2 * ROW + torch.finfo(TYPES[dtype]).eps / 2)),
          2 * ROW + torch.finfo(TYPES[dtype]).eps / 2)
    chunk = -(-rows // (4 * 148))
    depth = chunk + -(-rows // chunk) // 32 + 1 + 32 + 80
    if norm_after:
        close(out["dgain_post"], gp.grad, (du * bh).sum(0), depth * STEP)
    if use_dy:
        close(out["dgain_pre"], gq.grad, (wide(cut["dy"]).abs() * hat).sum(0), depth * STEP)
    else:
        assert not bool(out["dgain_pre"].any())
    if gate is not None:
        u = bh * (gp.detach().abs() if norm_after else 1.0)
        size = torch.zeros_like(gate)
        size.index_add_(0, torch.arange(rows, device="cuda") // (gate_rows or rows), sb * parts * u)
        close(cut["dgate"], gate.grad, size.detach(), depth * STEP)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(ctx, dtype, rows, cols):
    check_backward(ctx, dtype, rows, cols, 0, 1, 0.7, 1.3)


@pytest.mark.parametrize("cols", [96, 257, 1024, 2048, 17000])
@pytest.mark.parametrize("rows,gate_rows", [(700, 0), (700, 1), (700, 64), (701, 100), (40, 7), (3, 1000), (1, 1)])
@pytest.mark.parametrize("norm_after", [0, 1])
def test_backward_gates(ctx, cols, rows, gate_rows, norm_after):
    if cols == 17000 and rows > 100:
        rows //= 10
    check_backward(ctx, "bf16", rows, cols, gate_rows, norm_after)


@pytest.mark.parametrize("cols,pad", [(256, 8), (1000, 3), (2048, 64)])
@pytest.mark.parametrize("kw", [dict(gate_rows=None, norm_after=1, gains=False), dict(gate_rows=None, norm_after=0),
                                dict(gate_rows=0, norm_after=1, use_dh=False),
                                dict(gate_rows=5, norm_after=1, use_dy=False),
                                dict(gate_rows=1, norm_after=0, use_dy=False)])
def test_backward_without_parts_and_with_pitches(ctx, cols, pad, kw):
    check_backward(ctx, "f16", 23, cols, pad=pad, **kw)


def test_many_rows(ctx):
    check_backward(ctx, "f32", 9001, 136, 3000, 1)
    check_backward(ctx, "bf16", 4099, 2048, 0, 1)


@pytest.mark.parametrize("cols", [64, 2048, 3001, 20000])
def test_in_place_and_repeatable(ctx, cols):
    rows = 37
    x = make("bf16", rows, cols, 0, 1, cols)
    ho, y = torch.empty_like(x["h"]), torch.empty_like(x["b"])
    args = (x["b"], x["gain_post"], x["gate"], x["gain_pre"])
    ctx.junction_fwd_bf16(x["h"], *args, ho, y, rows, cols)
    h2, y2 = x["h"].clone(), torch.empty_like(y)
    ctx.junction_fwd_bf16(h2, *args, h2, y2, rows, cols)
    ctx.junction_fwd_bf16(x["h"], *args, x["h"], None, rows, cols)  # without y
    ctx.sync()
    assert torch.equal(h2, ho) and torch.equal(y2, y) and torch.equal(x["h"], ho)
    outs = []
    for place in (False, True, False):
        dho = x["dh_out"].clone()
        dh = dho if place else torch.empty_like(dho)
        o = [dh, torch.empty_like(y), *(torch.empty(cols, device="cuda") for _ in range(3))]
        ctx.junction_bwd_bf16(ho, *args, dho, x["dy"], *o[:2], o[2], o[3], o[4], rows, cols)
        ctx.sync()
        outs.append(o)
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_gradient_by_differences(ctx):
    """d sum(h' G + y K) along random directions, by central differences of the
    64-bit formula (error h^2 times the third derivative, below 1e-7 here)."""
    rows, cols, gr = 12, 160, 4
    x = make("f32", rows, cols, gr, 1, 77)
    G, K = x["dh_out"], x["dy"]
    ho, y = torch.empty_like(x["h"]), torch.empty_like(x["b"])
    ctx.junction_fwd_f32(x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"], ho, y, rows, cols, gate_rows=gr,
                         scale_h=0.9, scale_b=1.1)
    out = [torch.empty_like(t) for t in (x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"])]
    ctx.junction_bwd_f32(ho, x["b"], x["gain_post"], x["gate"], x["gain_pre"], G, K, *out, rows, cols, gate_rows=gr,
                         scale_h=0.9, scale_b=1.1)
    ctx.sync()

    def f(h, b, gp, gate, gq):
        h2 = float(torch.tensor(0.9)) * h + float(torch.tensor(1.1)) * after(b, gp, gate, rows, gr, 1, 1e-5)
        return float((h2 * wide(G)).sum() + (rms(h2, 1e-5) * gq * wide(K)).sum())

    at = [wide(x[k]) for k in ("h", "b", "gain_post", "gate", "gain_pre")]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(5):
        d = torch.randn(at[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        step = 1e-4
        up, dn = list(at), list(at)
        up[i], dn[i] = at[i] + step * d, at[i] - step * d
        num = (f(*up) - f(*dn)) / (2 * step)
        ana = float((out[i].double() * d).sum())
        size = float((out[i].double() * d).abs().sum())
        assert abs(num - ana) <= 4 * ROW * size + 1e-6 * abs(num) + 1e-5, (i, num, ana)


def test_zero_rows_and_refusals(ctx):
    z = torch.zeros(4, 16, device="cuda")
    g = torch.full((16,), 5.0, device="cuda")
    ctx.junction_fwd_f32(z, z, None, None, None, z, z, 0, 16)
    ctx.junction_bwd_f32(z, z, g, None, g, z, z, z, z.clone(), g, None, g, 0, 16)
    ctx.sync()
    assert not bool(g.any())
    ctx.junction_fwd_f32(z, z, None, None, None, z, z, 4, 0)

    def refused(fn, *a, **kw):
        with pytest.raises(bwpp.BwppError) as e:
            fn(*a, **kw)
        assert e.value.status == bwpp.ERR_ARG

    f, b = ctx.junction_fwd_f32, ctx.junction_bwd_f32
    refused(f, None, z, None, None, None, z, z, 4, 16)
    refused(f, z, None, None, None, None, z, z, 4, 16)
    refused(f, z, z, None, None, None, None, z, 4, 16)
    refused(f, z, z, None, None, None, z, z, 4, 16, ldh=15)
    refused(f, z, z, None, None, None, z, z, 4, 16, ldy=8)
    refused(f, z, z, None, z, None, z, z, 4, 16, ldgate=8)
    refused(f, z, z, None, None, None, z, z, 2**31, 16)
    refused(b, z, z, None, None, None, z, z, z, z, None, None, None, 4, 16)  # db is b
    refused(b, z, None, None, None, None, z, z, z, z, None, None, None, 4, 16)
    refused(b, None, z, None, None, None, z, z, z, None, None, None, None, 4, 16)
    refused(b, z, z, None, None, None, z, z, z, None, None, z, None, 4, 16)  # dgate without a gate
    refused(b, z, z, None, None, None, z, z, z, None, g, None, None, 4, 16, norm_after=0)
    with pytest.raises(bwpp.BwppError) as e:  # 32 columns a block, 65535 blocks
        b(z, z, None, None, None, None, z, None, None, None, None, g, 1, 32 * 65535 + 1)
    assert e.value.status == bwpp.ERR_UNSUPPORTED


def test_zero_rows_of_b_and_eps_zero(ctx):
    """A row of zeros with eps > 0 stays zero; NaN and infinities stay in their row."""
    rows, cols = 5, 2048
    x = make("bf16", rows, cols, None, 1, 8)
    x["b"][1] = 0
    x["b"][3, 7] = float("nan")
    x["h"][4, 9] = float("inf")
    ho, y = torch.empty_like(x["h"]), torch.empty_like(x["b"])
    ctx.junction_fwd_bf16(x["h"], x["b"], x["gain_post"], None, x["gain_pre"], ho, y, rows, cols)
    ctx.sync()
    assert torch.equal(ho[1], x["h"][1])
    assert bool(torch.isfinite(ho[:3]).all()) and bool(torch.isfinite(y[:3].float()).all())
    assert bool(torch.isnan(y[3].float()).all()) and bool(torch.isinf(ho[4, 9]))


def test_offsets_past_32_bits(ctx):
    ld = 2**31
    cols = 264
    h = torch.empty(2 * ld + cols, device="cuda")
    rows = torch.as_strided(h, (3, cols), (ld, 1))
    rows.copy_(torch.randn(3, cols, device="cuda"))
    b = torch.randn(3, cols, device="cuda").bfloat16()
    small, want = rows.clone(), torch.empty(3, cols, device="cuda")
    y, wy = torch.empty_like(b), torch.empty_like(b)
    ctx.junction_fwd_bf16(h, b, None, None, None, h, y, 3, cols, ldh=ld)
    ctx.junction_fwd_bf16(small, b, None, None, None, want, wy, 3, cols)
    ctx.sync()
    assert torch.equal(rows, want) and torch.equal(y, wy)


def test_captured_replayed_and_the_workspace(ctx):
    """Under capture the column sums need a caller's workspace; replays agree
    with eager calls on the same inputs."""
    rows, cols = 300, 512
    stream = torch.cuda.Stream()
    c = bwpp.Ctx(0, stream.cuda_stream)
    x = make("bf16", rows, cols, 0, 1, 21)
    shapes = [x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"]]
    out, want = ([torch.empty_like(t) for t in shapes] for _ in range(2))
    run = lambda k, o: k.junction_bwd_bf16(x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"],  # noqa: E731
                                           x["dh_out"], x["dy"], *o, rows, cols)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    need = bwpp.load().bwpp_cuda_junction_bwd_workspace_size(c.handle, rows, cols, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(bwpp.BwppError) as e:
            run(c, out)
        assert e.value.status == bwpp.ERR_UNSUPPORTED
        c.set_workspace(ws, need)
        run(c, out)
    for seed in (1, 2, 3):
        x["dy"].copy_(torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        run(ctx, want)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    c.set_workspace(ws, need - 1)
    with pytest.raises(bwpp.BwppError) as e:
        run(c, out)
    assert e.value.status == bwpp.ERR_NOMEM
    del graph
    c.close()


@pytest.mark.parametrize("cols", [2**31, 2**32 - 1])
def test_rows_of_2_31_columns_are_refused(ctx, cols):
    z = torch.zeros(16, device="cuda")
    for call in (lambda: ctx.junction_fwd_f32(z, z, None, None, None, z, z, 1, cols),
                 lambda: ctx.junction_bwd_f32(z, z, None, None, None, z, z, z, z.clone(), None, None, None, 1, cols)):
        with pytest.raises(bwpp.BwppError) as e:
            call()
        assert e.value.status == bwpp.ERR_ARG
    assert bwpp.load().bwpp_cuda_junction_bwd_workspace_size(ctx.handle, 4, cols, 0) == 0
    ctx.sync()


@pytest.mark.parametrize("gate_rows", [0, 3])
def test_no_rows_leave_no_gradient(ctx, gate_rows):
    """One gate for all rows has a gradient of zero where there are no rows; a
    gate for every three rows has none."""
    z = torch.zeros(1, 16, device="cuda")
    gate, dgate = torch.ones(1, 24, device="cuda"), torch.full((1, 24), 5.0, device="cuda")
    gains = torch.full((2, 16), 5.0, device="cuda")
    ctx.junction_bwd_f32(z, z, None, gate, None, z, z, None, None, gains[0], dgate, gains[1], 0, 16,
                         gate_rows=gate_rows, ldgate=24)
    ctx.sync()
    assert not bool(gains.any())
    assert bool((dgate[0, 16:] == 5.0).all()) and bool((dgate[0, :16] == (5.0 if gate_rows else 0.0)).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gate_rows", [0, 1])
@pytest.mark.parametrize("rows,cols", [(2000, 264), (1800, 512), (700, 520), (350, 2560), (301, 5632), (301, 5800),
                                       (301, 5808), (151, 7168), (151, 7248), (151, 7256), (150, 8192)])
def test_backward_of_staged_rows(ctx, dtype, gate_rows, rows, cols):
    """Widths on both sides of what two stages of a row leave room for, with more
    chunks of rows than an SM holds at a time, and with one."""
    check_backward(ctx, dtype, rows, cols, gate_rows, 1, 0.7, 1.3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [40, 264, 1003])
def test_many_gate_groups(ctx, dtype, cols):
    """A gate for every two rows of twenty thousand.  Column sums over all rows add
    a group's two rows, then ceil(groups / 32) partial rows and 32 warps' sums; a
    gate's gradient its two rows and what one partial row passes."""
    rows, gate_rows = 20001, 2
    x = make(dtype, rows, cols, gate_rows, 1, cols)
    groups = x["gate"].shape[0]
    assert groups == 10001
    dh, db = torch.empty_like(x["h"]), torch.empty_like(x["b"])
    dgp, dgate, dgq = torch.full((cols,), 7.0, device="cuda"), torch.full_like(x["gate"], 7.0), torch.full((cols,), 7.0, device="cuda")
    bwd(ctx, dtype)(x["h"], x["b"], x["gain_post"], x["gate"], x["gain_pre"], x["dh_out"], x["dy"], dh, db, dgp, dgate,
                    dgq, rows, cols, gate_rows=gate_rows)
    ctx.sync()
    h, b, gp, gate, gq = (wide(x[k]).requires_grad_() for k in ("h", "b", "gain_post", "gate", "gain_pre"))
    (rms(h, 1e-5) * gq).backward(wide(x["dy"]))
    dH = wide(x["dh_out"]) + h.grad
    after(b, gp, gate, rows, gate_rows, 1, 1e-5).backward(dH)
    at = torch.arange(rows, device="cuda") // gate_rows
    r = (h.detach().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    g = (gq.detach() * wide(x["dy"])).abs()
    hat = (h.detach() * r).abs()
    parts = wide(x["dh_out"]).abs() + r * (g + hat * (g * hat).mean(-1, keepdim=True))  # of dH
    bh = (b.detach() * (b.detach().square().mean(-1, keepdim=True) + 1e-5).rsqrt()).abs()
    close(dh, dH, parts, ROW)
    depth = gate_rows + -(-groups // 32) + 32 + 80
    close(dgp, gp.grad, (gate.detach()[at].abs() * parts * bh).sum(0), depth * STEP)
    close(dgq, gq.grad, (wide(x["dy"]).abs() * hat).sum(0), depth * STEP)
    size = torch.zeros_like(gate.detach()).index_add_(0, at, parts * bh * gp.detach().abs())
    close(dgate, gate.grad, size, (gate_rows + 32 + 80) * STEP)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("gate_rows", [0, 1])
@pytest.mark.parametrize("cols", [64, 520, 2048, 4104])
def test_odd_addresses(ctx, dtype, gate_rows, cols):
    """Each tensor one element off its 16 bytes, in turn, with pitches in eights:
    what aligned tensors give, up to both sides' errors (2 * ROW and half a step of
    the type each, of parts that are at most three times the result here), and
    nothing written around the outputs."""
    rows = 9
    x = make(dtype, rows, cols, gate_rows, 1, cols)
    names = ["h", "b", "gain_post", "gate", "gain_pre", "dh_out", "dy"]
    outs = {"ho": x["h"], "y": x["b"], "dh": x["h"], "db": x["b"], "dgain_post": x["gain_post"], "dgate": x["gate"],
            "dgain_pre": x["gain_pre"]}

    def at(like, off):
        buf = torch.full((like.numel() + 16,), 7.0, device="cuda", dtype=like.dtype)
        return buf, buf[off:off + like.numel()].view(like.shape)

    def run(odd):
        t = {k: at(x[k], odd == k)[1].copy_(x[k]) for k in names}
        o = {k: at(v, odd == k) for k, v in outs.items()}
        g = {k: v[1] for k, v in o.items()}
        fwd(ctx, dtype)(t["h"], t["b"], t["gain_post"], t["gate"], t["gain_pre"], g["ho"], g["y"], rows, cols,
                        gate_rows=gate_rows)
        bwd(ctx, dtype)(t["h"], t["b"], t["gain_post"], t["gate"], t["gain_pre"], t["dh_out"], t["dy"], g["dh"], g["db"],
                        g["dgain_post"], g["dgate"], g["dgain_pre"], rows, cols, gate_rows=gate_rows)
        ctx.sync()
        for k, (buf, v) in o.items():
            off = int(odd == k)
            assert bool((buf[:off] == 7.0).all()) and bool((buf[off + v.numel():] == 7.0).all()), (odd, k)
        return g

    want = run(None)
    for odd in names + list(outs):
        for k, v in run(odd).items():
            close(v, want[k].double(), want[k].double(), 3 * 2 * (2 * ROW + torch.finfo(v.dtype).eps / 2))
