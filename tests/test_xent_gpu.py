"""Softmax cross entropy over a vocabulary on the GPU, forward and gradient,
against the formula in 64 bits.

Tolerances, per element.  A logit is a sum of D bf16 products in fp32 on the
tensor cores, 16 at a time: D / 16 + 1 additions, each off by at most 2^-22 of
sum |x w| (the adder keeps at least 22 bits), DL = (D / 16 + 1) 2^-22 sum |x w|.
lse and loss are off by DL, and by 2^-20 (|value| + |target's logit| + 1) for
the exponentials, their sum and the logarithm.  dlogit = g (p - hit) is off by
g p (2 DL + 2^-20) and rounded to bf16, half a step 2^-8; the products with it
add (K / 16 + 1) 2^-22 of the sum of magnitudes, once more for each piece's
sum in fp32; a bf16 gradient adds half a step of its own.
"""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu
HALF = 2.0**-8  # half a step of bf16


def make(T, V, D, vocab_major, seed, ignored=0.2, sharp=2.0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, D, device="cuda", generator=g) * (sharp / D**0.5)).bfloat16()
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    lift = 4.0 * torch.rand(T, 1, device="cuda", generator=g)
    x = (torch.randn(T, D, device="cuda", generator=g) + lift * w[target].float()).bfloat16()
    keep = torch.rand(T, device="cuda", generator=g) >= ignored
    target = torch.where(keep, target, -1 - target).int()
    dloss = torch.rand(T, device="cuda", generator=g) + 0.5
    xs = torch.full((T, D + pad), float("nan"), device="cuda").bfloat16()
    xs[:, :D] = x
    ws = torch.full((V, D + pad) if vocab_major else (D, V + pad), float("nan"), device="cuda").bfloat16()
    ws[:, :D if vocab_major else V] = w if vocab_major else w.t()
    return x, w, target, dloss, xs, ws


def formula(x, w, target, scale):
    """logits, lse, loss, DL per row, all in 64 bits."""
    x, w = x.double(), w.double()
    logits = scale * (x @ w.t())
    lse = torch.logsumexp(logits, 1)
    hit = logits.gather(1, target.long().clamp(min=0)[:, None])[:, 0]
    loss = torch.where(target >= 0, lse - hit, torch.zeros_like(lse))
    dl = (x.shape[1] // 16 + 2) * 2.0**-22 * abs(scale) * (x.abs() @ w.abs().t()).amax(1)
    return logits, lse, loss, hit, dl


def within(got, want, tol):
    most = torch.finfo(got.dtype).max  # a sum beyond it is an infinity
    beyond = want.abs() > most
    assert torch.equal(got[beyond].double(), want[beyond] * float("inf"))
    err = torch.where(beyond, 0.0, (got.double() - want).abs())
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))


def check(ctx, T, V, D, vocab_major, scale=1.0, bf16=1, pad=0, seed=0, ones=False, sharp=2.0, ignored=0.2,
          step=HALF, each_dloss=None):
    x, w, target, dloss, xs, ws = make(T, V, D, vocab_major, seed + T + V, ignored, sharp, pad)
    if each_dloss is not None:
        dloss = torch.where(target >= 0, torch.full_like(dloss, each_dloss), dloss)
    ldw = ws.shape[1]
    scale = float(torch.tensor(scale))
    loss, lse = (torch.full((T,), float("nan"), device="cuda") for _ in range(2))
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D + pad, ldw, w_vocab_major=vocab_major, scale=scale)
    ctx.sync()
    logits, wlse, wloss, hit, dl = formula(x, w, target, scale)
    tol = 2 * dl + 2.0**-20 * (wlse.abs() + hit.abs() + 1)
    within(lse, wlse, tol)
    within(loss, wloss, tol)
    assert not bool(loss[target < 0].any())

    t = torch.bfloat16 if bf16 else torch.float32
    dx = torch.full((T, D + pad), 7.0, device="cuda", dtype=t)
    dw = torch.full(tuple(ws.shape), 7.0, device="cuda", dtype=t)
    ctx.xent_bwd(xs, ws, target, lse, None if ones else dloss, dx, dw, T, V, D, D + pad, ldw, D + pad, ldw,
                 w_vocab_major=vocab_major, scale=scale, grads_bf16=bf16)
    ctx.sync()
    g = torch.where(target >= 0, torch.ones_like(wlse) if ones else dloss.double(), torch.zeros_like(wlse))
    p = (logits - wlse[:, None]).exp()
    d = p.clone()
    d[torch.arange(T, device="cuda"), target.long().clamp(min=0)] -= 1.0
    d, off = d * g[:, None] * scale, p * (g * abs(scale) * (4 * dl + 2.0**-20 * (wlse.abs() + 2)))[:, None]
    each = off + step * d.abs()
    xd, wd = x.double(), w.double()
    out = HALF if bf16 else 2.0**-24
    pieces = 66  # 2^-22 of a sum of magnitudes for each piece, at most 64 here
    add = lambda K: (K // 16 + pieces) * 2.0**-22  # noqa: E731
    within(dx[:, :D], d @ wd, (each + add(V) * d.abs()) @ wd.abs() * (1 + HALF) + out * (d @ wd).abs() + 1e-30)
    want = d.t() @ xd
    tol = (each + add(T) * d.abs()).t() @ xd.abs() * (1 + HALF) + out * want.abs() + 1e-30
    got = dw[:, :D] if vocab_major else dw[:, :V].t()
    within(got, want, tol)
    if pad:
        assert bool((dx[:, D:] == 7.0).all()) and bool((dw[:, D if vocab_major else V:] == 7.0).all())


@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 2, 8), (1, 1000, 64), (3, 257, 16), (5, 255, 33), (64, 256, 64),
                                   (127, 1000, 72), (128, 512, 128), (129, 513, 65), (200, 3001, 100),
                                   (257, 770, 256), (300, 5000, 520), (1, 32000, 256), (777, 1009, 101),
                                   (140, 700, 1096), (33, 1500, 2500), (260, 300, 4096),
                                   (2, 333, 40), (2, 1001, 129), (1, 130, 264), (2, 4097, 1000), (2, 600, 7000),
                                   (1, 50000, 16), (7, 20000, 8), (1, 200, 30000), (2, 90, 50000),
                                   (5000, 300, 40), (4001, 700, 136), (2100, 64, 520)])
def test_sizes(ctx, T, V, D, vocab_major):
    check(ctx, T, V, D, vocab_major, ignored=0.0 if T == 1 else 0.2)


@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("kw", [dict(scale=0.125), dict(scale=0.0), dict(scale=-3.0), dict(bf16=0), dict(pad=8), dict(pad=3),
                                dict(pad=3, bf16=0), dict(ones=True), dict(sharp=30.0), dict(ignored=1.0)])
def test_options(ctx, vocab_major, kw):
    check(ctx, 150, 1111, 136, vocab_major, **kw)
    check(ctx, 40, 300, 31, vocab_major, **kw)


@pytest.mark.parametrize("vocab_major", [0, 1])
def test_several_pieces(ctx, vocab_major):
    """Enough rows that the vocabulary goes by in several pieces, the last short."""
    check(ctx, 9000, 9003 if vocab_major else 9000, 64, vocab_major, bf16=vocab_major)


def test_ignored_rows_may_hold_anything(ctx):
    T, V, D = 70, 520, 96
    x, w, target, dloss, xs, ws = make(T, V, D, 1, 5)
    target[::3] = -100
    good = xs.clone()
    xs[::3] = float("nan")
    xs[3, 5] = float("inf")
    outs = []
    for src in (good, xs):
        loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ctx.xent_fwd(src, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
        ctx.xent_bwd(src, ws, target, lse, dloss, dx, dw, T, V, D, D, D, D, D, w_vocab_major=1, grads_bf16=1)
        ctx.sync()
        outs.append((loss, dx, dw))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not bool(outs[1][1][::3].any())


def test_target_outside_the_vocabulary_is_reported(ctx):
    T, V, D = 20, 100, 32
    x, w, target, dloss, xs, ws = make(T, V, D, 1, 6, ignored=0.0)
    want_dw, dw = torch.empty_like(w), torch.empty_like(w)
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    dx = torch.empty_like(x)
    target[4] = -1
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
    ctx.xent_bwd(xs, ws, target, lse, dloss, dx, want_dw, T, V, D, D, D, D, D, w_vocab_major=1, grads_bf16=1)
    ctx.sync()
    for bad in (V, 2**31 - 1):
        target[4] = bad
        ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
        with pytest.raises(bwpp.BwppError) as e:
            ctx.sync()
        assert e.value.status == bwpp.ERR_ARG
        assert bool(torch.isnan(loss[4])) and int(torch.isnan(loss).sum()) == 1
        ctx.xent_bwd(xs, ws, target, lse, dloss, dx, dw, T, V, D, D, D, D, D, w_vocab_major=1, grads_bf16=1)
        with pytest.raises(bwpp.BwppError) as e:
            ctx.sync()
        assert e.value.status == bwpp.ERR_ARG
        assert torch.equal(dw, want_dw) and not bool(dx[4].any())
    ctx.sync()


def test_large_logits_and_infinities(ctx):
    """Logits of +-3000 neither overflow nor lose the sum; -inf logits drop out;
    a NaN row stays alone."""
    T, V, D = 9, 600, 8
    x, w, target, _, xs, ws = make(T, V, D, 1, 7, ignored=0.0)
    xs[0] *= 2000
    xs[1] *= -2000
    xs[2, 3] = float("nan")
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
    ctx.sync()
    _, wlse, wloss, hit, dl = formula(xs, w, target, 1.0)
    rows = [0, 1, 3, 4, 5, 6, 7, 8]
    tol = 2 * dl + 2.0**-20 * (wlse.abs() + hit.abs() + 1)
    within(lse[rows], wlse[rows], tol[rows])
    within(loss[rows], wloss[rows], tol[rows])
    assert bool(torch.isnan(loss[2]))
    ws[5] = float("-inf")  # with positive x: a logit of -inf
    xs[:] = xs.abs().nan_to_num(1.0)
    target[:] = 7
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
    ctx.sync()
    keep = [v for v in range(V) if v != 5]
    _, wlse, _, _, dl = formula(xs, w[keep], torch.zeros_like(target), 1.0)
    within(lse, wlse, 2 * dl + 2.0**-20 * (wlse.abs() + 1))


def test_one_output_at_a_time(ctx):
    T, V, D = 130, 700, 64
    x, w, target, dloss, xs, ws = make(T, V, D, 0, 9)
    loss, lse, l1, l2 = (torch.empty(T, device="cuda") for _ in range(4))
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, V)
    ctx.xent_fwd(xs, ws, target, l1, None, T, V, D, D, V)
    ctx.xent_fwd(xs, ws, None, None, l2, T, V, D, D, V)
    dx, dw, d1, d2 = torch.empty_like(x), torch.empty_like(ws), torch.empty_like(x), torch.empty_like(ws)
    a = (T, V, D, D, V, D, V)
    ctx.xent_bwd(xs, ws, target, lse, dloss, dx, dw, *a, grads_bf16=1)
    ctx.xent_bwd(xs, ws, target, lse, dloss, d1, None, *a, grads_bf16=1)
    ctx.xent_bwd(xs, ws, target, lse, dloss, None, d2, *a, grads_bf16=1)
    ctx.sync()
    assert torch.equal(loss, l1) and torch.equal(lse, l2) and torch.equal(dx, d1) and torch.equal(dw, d2)


@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D", [(1, 1000, 64), (3, 1237, 100), (1, 5000, 300), (64, 900, 64), (50, 3000, 136)])
def test_few_rows_keep_more_than_one_rounding(ctx, T, V, D, vocab_major):
    """Up to 64 rows, dlogit is two bf16: half a step of half a step is left."""
    check(ctx, T, V, D, vocab_major, bf16=0, step=HALF * HALF, ignored=0.0 if T == 1 else 0.2)


@pytest.mark.parametrize("each_dloss", [1.0 / 300.0, 1e-30, 3e38, 0.0, -0.7])
def test_rows_that_share_their_dloss(ctx, each_dloss):
    """A mean loss: one dloss for all live rows, any others in ignored ones."""
    check(ctx, 300, 700, 72, 1, each_dloss=each_dloss, bf16=0, scale=0.25)
    check(ctx, 300, 700, 72, 0, each_dloss=each_dloss, scale=0.25)


def test_a_dloss_that_is_not_a_number_stays_in_its_row(ctx):
    T, V, D = 200, 300, 64
    x, w, target, dloss, xs, ws = make(T, V, D, 1, 13, ignored=0.0)
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1)
    dx = torch.empty(T, D, device="cuda")
    for bad in (float("nan"), float("inf")):
        for rest in (0.5, None):  # one value in the other rows, or their own
            g = dloss.clone() if rest is None else torch.full_like(dloss, rest)
            g[77] = bad
            ctx.xent_bwd(xs, ws, target, lse, g, dx, None, T, V, D, D, D, D, D, w_vocab_major=1)
            ctx.sync()
            off = ~torch.isfinite(dx).all(1)
            assert bool(off[77]) and int(off.sum()) == 1


@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D", [(1, 1000, 64), (3, 700, 100), (2, 1300, 1000), (60, 1000, 2500), (64, 999, 64)])
def test_loss_of_sure_targets(ctx, T, V, D, vocab_major):
    """Few rows whose target has nearly all of the probability: losses down to
    1e-7 keep their digits."""
    g = torch.Generator(device="cuda").manual_seed(T + D)
    w = (torch.randn(V, D, device="cuda", generator=g) / D**0.5).bfloat16()
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    a = 15 + 8 * torch.rand(T, 1, device="cuda", generator=g)
    x = (a * w[target].float() / w[target].float().square().sum(1, keepdim=True)).bfloat16()
    ws = w if vocab_major else w.t().contiguous()
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ctx.xent_fwd(x, ws, target.int(), loss, lse, T, V, D, D, ws.shape[1], w_vocab_major=vocab_major)
    ctx.sync()
    logits = x.double() @ w.double().t()
    hit = logits.gather(1, target[:, None])[:, 0]
    logits.scatter_(1, target[:, None], float("-inf"))
    others = torch.logsumexp(logits, 1)
    want = torch.log1p((others - hit).exp())
    assert float(want.min()) < 1e-3
    # d loss = p' d(others - hit): the logits' errors (a truncation of 2^-22 per 16
    # of up to 256 and per sum of 128, of the terms' magnitudes), roundings of numbers in
    # powers of two up to 1.45 hit, and a few of the loss itself
    dl = (min(D, 256) // 16 + D // 128 + 2) * 2.0**-22 * (x.double().abs() @ w.double().abs().t()).amax(1)
    tol = want * (2 * dl + 2.0**-21 * (hit.abs() + others.abs() + 4))
    within(loss, want, tol)


def test_gradient_by_differences(ctx):
    """d sum(dloss loss) along random directions, by central differences of the
    64-bit formula; the kernel's gradient carries bf16's half step twice."""
    T, V, D = 24, 400, 64
    x, w, target, dloss, xs, ws = make(T, V, D, 1, 11)
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    dx, dw = torch.empty(T, D, device="cuda"), torch.empty(V, D, device="cuda")
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, D, w_vocab_major=1, scale=0.5)
    ctx.xent_bwd(xs, ws, target, lse, dloss, dx, dw, T, V, D, D, D, D, D, w_vocab_major=1, scale=0.5)
    ctx.sync()

    def f(x, w):
        return float((formula(x, w, target, 0.5)[2] * dloss.double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(3)
    for arg, grad in ((0, dx), (1, dw)):
        at = [x.double(), w.double()]
        d = torch.randn(at[arg].shape, device="cuda", generator=gen, dtype=torch.float64)
        up, dn = list(at), list(at)
        up[arg], dn[arg] = at[arg] + 1e-4 * d, at[arg] - 1e-4 * d
        num = (f(*up) - f(*dn)) / 2e-4
        terms = grad.double() * d
        # each element is within half a step of bf16 of the sum of its terms'
        # magnitudes, at most sqrt(V) or sqrt(T) times its own size; the
        # directions are random, so elements' errors add as a root
        tol = 4 * HALF * float(terms.square().sum().sqrt()) * max(V, T) ** 0.5 + 1e-5
        assert abs(num - float(terms.sum())) <= tol, (arg, num, float(terms.sum()), tol)


def test_no_rows_and_refusals(ctx):
    z = torch.zeros(16, 16, device="cuda").bfloat16()
    t = torch.zeros(16, device="cuda").int()
    f = torch.zeros(16, device="cuda")
    dw = torch.full((16, 16), 3.0, device="cuda").bfloat16()
    ctx.xent_fwd(z, z, t, f, f, 0, 16, 16, 16, 16)
    ctx.xent_bwd(z, z, t, f, None, z, dw, 0, 16, 8, 8, 16, 8, 16, grads_bf16=1)
    ctx.sync()
    assert not bool(dw[:8].any()) and bool((dw[8:] == 3.0).all())

    def refused(fn, *a, **kw):
        with pytest.raises(bwpp.BwppError) as e:
            fn(*a, **kw)
        assert e.value.status == bwpp.ERR_ARG

    fw, bw = ctx.xent_fwd, ctx.xent_bwd
    refused(fw, z, z, t, f, f, 16, 0, 16, 16, 16)
    refused(fw, z, z, t, f, f, 16, 16, 0, 16, 16)
    refused(fw, z, z, t, f, f, 16, 16, 16, 15, 16)
    refused(fw, z, z, t, f, f, 16, 16, 16, 16, 15)
    refused(fw, z, z, t, f, f, 16, 16, 16, 16, 16, scale=float("nan"))
    refused(fw, None, z, t, f, f, 16, 16, 16, 16, 16)
    refused(fw, z, None, t, f, f, 16, 16, 16, 16, 16)
    refused(fw, z, z, None, f, f, 16, 16, 16, 16, 16)
    refused(fw, z, z, t, None, None, 16, 16, 16, 16, 16)
    refused(bw, z, z, t, f, None, z, dw, 16, 16, 16, 16, 16, 15, 16)
    refused(bw, z, z, t, f, None, z, dw, 16, 16, 16, 16, 16, 16, 15)
    refused(bw, z, z, None, f, None, z, dw, 16, 16, 16, 16, 16, 16, 16)
    refused(bw, z, z, t, None, None, z, dw, 16, 16, 16, 16, 16, 16, 16)
    ctx.xent_bwd(z, z, t, f, None, None, None, 16, 16, 16, 16, 16, 16, 16)
    ctx.sync()


def test_rows_past_32_bits(ctx):
    ld = 2**31
    T, V, D = 3, 300, 64
    x, w, target, dloss, _, ws = make(T, V, D, 1, 13, ignored=0.0)
    far = torch.empty(2 * ld + D, dtype=torch.bfloat16, device="cuda")
    torch.as_strided(far, (T, D), (ld, 1)).copy_(x)
    got, want = [], []
    for src, pitch, out in ((x, D, want), (far, ld, got)):
        loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ctx.xent_fwd(src, ws, target, loss, lse, T, V, D, pitch, D, w_vocab_major=1)
        ctx.xent_bwd(src, ws, target, lse, dloss, dx, dw, T, V, D, pitch, D, D, D, w_vocab_major=1, grads_bf16=1)
        ctx.sync()
        out += [loss, lse, dx, dw]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 30, 400])
def test_captured_and_replayed(ctx, T):
    """Forward and gradient in one graph with a caller's workspace, replayed on
    new inputs; without a workspace the capture is refused."""
    V, D = 2100, 128
    stream = torch.cuda.Stream()
    c = bwpp.Ctx(0, stream.cuda_stream)
    x, w, target, dloss, xs, ws = make(T, V, D, 0, 15)
    need = max(bwpp.xent_workspace_size(T, V, D, D, ws.shape[1], 0, b, 1) for b in (0, 1))
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    bufs = [[torch.empty(T, device="cuda"), torch.empty(T, device="cuda"), torch.empty_like(x), torch.empty_like(ws)]
            for _ in range(2)]

    def run(k, o):
        k.xent_fwd(xs, ws, target, o[0], o[1], T, V, D, D, V)
        k.xent_bwd(xs, ws, target, o[1], dloss, o[2], o[3], T, V, D, D, V, D, V, grads_bf16=1)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(bwpp.BwppError) as e:
            run(c, bufs[0])
        assert e.value.status == bwpp.ERR_UNSUPPORTED
        c.set_workspace(room, need)
        run(c, bufs[0])
    k = bwpp.Ctx(0)
    other = torch.empty(need, dtype=torch.uint8, device="cuda")
    k.set_workspace(other, need)
    for seed in (1, 2, 3):
        xs.copy_(make(T, V, D, 0, seed)[4])
        graph.replay()
        torch.cuda.synchronize()
        run(k, bufs[1])
        k.sync()
        assert all(torch.equal(a, b) for a, b in zip(*bufs))
    c.set_workspace(room, 256)
    with pytest.raises(bwpp.BwppError) as e:
        run(c, bufs[0])
    assert e.value.status == bwpp.ERR_NOMEM
    del graph
    c.close()
    k.close()


@pytest.mark.parametrize("captured", [0, 1])
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D", [(3, 1000, 64), (150, 1112, 136), (300, 2104, 256)])
def test_odd_addresses(T, V, D, vocab_major, bf16, captured):
    """x, w, dx and dw one element off their 16 bytes, alone and together, with
    pitches that TMA takes, in a workspace of the queried size: the results of
    aligned buffers bit for bit, nothing written around them."""
    stream = torch.cuda.Stream()
    c = bwpp.Ctx(0, stream.cuda_stream)
    x, w, target, dloss, xs, ws = make(T, V, D, vocab_major, 17)
    ldw = ws.shape[1]
    need = max(bwpp.xent_workspace_size(T, V, D, D, ldw, vocab_major, b, bf16) for b in (0, 1))
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    c.set_workspace(room, need)
    t = torch.bfloat16 if bf16 else torch.float32

    def at(like, off, dtype):
        buf = torch.full((like.numel() + 16,), 7.0, device="cuda", dtype=dtype)
        return buf, buf[off:off + like.numel()].view(like.shape)

    def run(odd):
        x1, w1 = at(xs, odd[0], xs.dtype)[1], at(ws, odd[1], ws.dtype)[1]
        x1.copy_(xs)
        w1.copy_(ws)
        bufs = [at(xs, odd[2], t), at(ws, odd[3], t)]
        (bx, dx), (bw, dw) = bufs
        loss, lse = torch.full((T,), 7.0, device="cuda"), torch.full((T,), 7.0, device="cuda")

        def calls():
            c.xent_fwd(x1, w1, target, loss, lse, T, V, D, D, ldw, w_vocab_major=vocab_major)
            c.xent_bwd(x1, w1, target, lse, dloss, dx, dw, T, V, D, D, ldw, D, ldw, w_vocab_major=vocab_major,
                       grads_bf16=bf16)

        torch.cuda.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                calls()
            graph.replay()
            graph.replay()
            torch.cuda.synchronize()
            del graph
        else:
            calls()
        c.sync()
        for (buf, _), off, n in ((bufs[0], odd[2], dx.numel()), (bufs[1], odd[3], dw.numel())):
            assert bool((buf[:off] == 7.0).all()) and bool((buf[off + n:] == 7.0).all())
        return loss, lse, dx, dw

    want = run((0, 0, 0, 0))
    assert bool(torch.isfinite(want[2].float()).all()) and bool(torch.isfinite(want[3].float()).all())
    for odd in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 3, 5, 7)):
        assert all(torch.equal(a, b) for a, b in zip(run(odd), want)), odd
    c.close()


@pytest.mark.parametrize("T,V,D", [(4, 4, 2**32 - 1), (4, 4, 2**31 - 511), (2**32 - 1, 4, 4), (4, 2**32 - 1, 4)])
@pytest.mark.parametrize("vocab_major", [0, 1])
def test_sizes_past_31_bits_are_refused(ctx, T, V, D, vocab_major):
    z = torch.zeros(16, device="cuda").bfloat16()
    f = torch.zeros(16, device="cuda")
    ldw = D if vocab_major else V
    for call in (lambda: ctx.xent_fwd(z, z, f.int(), f, f, T, V, D, D, ldw, w_vocab_major=vocab_major),
                 lambda: ctx.xent_bwd(z, z, f.int(), f, None, z, z, T, V, D, D, ldw, D, ldw, w_vocab_major=vocab_major,
                                      grads_bf16=1)):
        with pytest.raises(bwpp.BwppError) as e:
            call()
        assert e.value.status == bwpp.ERR_ARG
    ctx.sync()


@pytest.mark.parametrize("T,V,D,vocab_major", [(24, 400, 64, 1), (64, 1000, 136, 0), (65, 700, 96, 0), (300, 900, 264, 1)])
def test_gradient_along_itself_by_differences(ctx, T, V, D, vocab_major):
    """d sum(dloss loss) along the gradient's own direction, by central differences
    of the 64-bit formula, is the gradient's norm: a wrong scale, sign or missing
    term would be off by a large part of it.

    With d = grad / |grad| the sum of terms is |grad|, and an element's error e, at
    most `step` of the sum of its products' magnitudes, enters as d . e.  Each term
    of the sum is rounded on its own: by at most `step` of itself, so d . e is at
    most step * sum over rows and columns of |dlogit| (|d W|) = step * A, A taken
    in 64 bits.  `step` is half a step of bf16, or of what it leaves up to 64 rows,
    and twice that bounds the logits' and sums' errors of fp32 size as well (2^-16).
    The differences are off by the third derivative, 1e-7 of |grad| here."""
    x, w, target, dloss, xs, ws = make(T, V, D, vocab_major, 23)
    ldw = ws.shape[1]
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    dx, dw = torch.empty(T, D, device="cuda"), torch.empty(tuple(ws.shape), device="cuda")
    ctx.xent_fwd(xs, ws, target, loss, lse, T, V, D, D, ldw, w_vocab_major=vocab_major, scale=0.5)
    ctx.xent_bwd(xs, ws, target, lse, dloss, dx, dw, T, V, D, D, ldw, D, ldw, w_vocab_major=vocab_major, scale=0.5)
    ctx.sync()
    dw = dw if vocab_major else dw.t().contiguous()
    x, w = x.double(), w.double()
    step = HALF * HALF if T <= 64 else HALF

    def f(x, w):
        return float((formula(x, w, target, 0.5)[2] * dloss.double()).sum())

    logits, wlse = formula(x, w, target, 0.5)[:2]
    p = (logits - wlse[:, None]).exp()
    p[torch.arange(T, device="cuda"), target.long().clamp(min=0)] -= 1.0
    dlogit = torch.where(target >= 0, dloss.double(), 0.0)[:, None] * p
    for grad, is_x in ((dx, True), (dw, False)):
        norm = float(grad.double().norm())
        d = grad.double() / norm
        h = 1e-3
        at = [(x + s * h * d, w) if is_x else (x, w + s * h * d) for s in (1, -1)]
        num = (f(*at[0]) - f(*at[1])) / (2 * h)
        each = 0.5 * (d @ w.t() if is_x else x @ d.t())  # the derivative of each logit along d
        tol = 2 * (step + 2.0**-16) * float((dlogit * each).abs().sum()) + 1e-6 * norm
        assert abs(num - norm) <= tol, (is_x, num, norm, tol)
        assert tol <= 0.05 * norm  # the bound says something


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("vocab_major", [0, 1])
@pytest.mark.parametrize("T,V,D,pad", [(194, 37, 77, 3), (743, 1, 1, 7), (3, 999, 127, 1), (300, 2099, 83, 5), (500, 258, 66, 6),
                                       (1500, 1284, 516, 4), (130, 1, 1001, 7), (9000, 9003, 67, 5)])
def test_padding_of_rows_that_end_inside_16_bytes(ctx, T, V, D, pad, vocab_major, bf16):
    """Pitches that TMA takes, rows that are no multiple of 16 bytes: what lies
    behind a row is not the gradient's."""
    check(ctx, T, V, D, vocab_major, bf16=bf16, pad=pad)
