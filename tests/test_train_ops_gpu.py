"""The training-step operators as a decoder uses them: block end (junction),
qkv product, rotary positions, attention, output product, block end, vocabulary
cross entropy, and all of it backward, against float64 torch autograd.

The checker rounds to bf16 where the GPU stores bf16 (straight through in the
backward), so the comparison isolates the kernels.  Tolerance: relative
Frobenius <= 3e-2, the bound of the whole training step's gradients (each
activation gradient on the way is rounded to bf16 once more); the loss, one
rounding of the hidden state behind it, 2e-3.
"""
import math

import pytest
import torch

import bwpp
from conftest import rel_fro
from test_junction_gpu import after, rms
from test_operators_cpu import frequencies

pytestmark = pytest.mark.gpu
B, S, H, HD, V = 2, 192, 2, 128, 1500
T, D = B * S, H * HD


def r16(x):
    return x + (x.bfloat16().double() - x).detach()


def rotate(x, f):  # [T, H, HD]
    pos = torch.arange(T, device=x.device).remainder(S).double()
    a = pos[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    cos, sin = a.cos()[:, None], a.sin()[:, None]
    h = HD // 2
    return torch.cat([x[..., :h] * cos - x[..., h:] * sin, x[..., h:] * cos + x[..., :h] * sin], -1)


def make(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    p = {"h0": rnd(T, D), "b0": rnd(T, D).bfloat16(), "wqkv": (rnd(D, 3 * D) / D**0.5).bfloat16(),
         "wo": (rnd(D, D) / D**0.5).bfloat16(), "wv": (2 * rnd(V, D) / D**0.5).bfloat16()}
    for k in ("gp0", "gq0", "gp1", "gq1"):
        p[k] = 1 + 0.1 * rnd(D)
    p["gate0"], p["gate1"] = 0.5 + 0.2 * rnd(B, D), 0.5 + 0.2 * rnd(1, D)
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    target[::7] = -1
    p["target"] = target.int()
    p["dloss"] = (target >= 0).float() / (target >= 0).sum()
    return p


def checker(p):
    q = {k: v.double().requires_grad_() for k, v in p.items() if k not in ("target", "dloss")}
    eps = 1e-5
    h1 = q["h0"] + after(q["b0"], q["gp0"], q["gate0"], T, S, 1, eps)
    y1 = r16(rms(h1, eps) * q["gq0"])
    qkv = r16(y1 @ q["wqkv"]).view(T, 3, H, HD)
    f = frequencies(HD)
    qq, kk, vv = r16(rotate(qkv[:, 0], f)), r16(rotate(qkv[:, 1], f)), qkv[:, 2]
    heads = lambda t: t.reshape(B, S, H, HD).permute(0, 2, 1, 3)  # noqa: E731
    s = heads(qq) @ heads(kk).transpose(-1, -2) / math.sqrt(HD)
    s = s.masked_fill(torch.triu(torch.ones(S, S, dtype=torch.bool, device=s.device), 1), float("-inf"))
    o = r16((torch.softmax(s, -1) @ heads(vv)).permute(0, 2, 1, 3).reshape(T, D))
    b1 = r16(o @ q["wo"])
    h2 = 0.9 * h1 + 1.1 * after(b1, q["gp1"], q["gate1"], T, T, 1, eps)
    y2 = r16(rms(h2, eps) * q["gq1"])
    logp = torch.log_softmax(y2 @ q["wv"].t(), 1)
    t = p["target"].long()
    loss = torch.where(t >= 0, -logp.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros_like(logp[:, 0]))
    (loss * p["dloss"].double()).sum().backward()
    return loss.detach(), {k: v.grad for k, v in q.items()}


class Step:
    """The same through one bwpp.Ctx, buffers kept between steps."""

    def __init__(self, ctx, p):
        self.ctx, self.p, self.table = ctx, p, bwpp.rope_table(HD)
        f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        b16 = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.h1, self.h2, self.dh1 = f32(T, D), f32(T, D), f32(T, D)
        self.y1, self.y2, self.o, self.b1 = b16(T, D), b16(T, D), b16(T, D), b16(T, D)
        self.qkv, self.dqkv = b16(T, 3 * D), b16(T, 3 * D)
        self.alse, self.loss, self.lse = f32(B * H * S), f32(T), f32(T)
        self.dy2, self.db1, self.do, self.dy1 = b16(T, D), b16(T, D), b16(T, D), b16(T, D)
        self.g = {k: torch.empty_like(v) for k, v in p.items() if k not in ("target", "dloss", "wqkv", "wo")}
        self.g["wqkv"], self.g["wo"] = f32(D, 3 * D), f32(D, D)

    def run(self):
        c, p, g, lib = self.ctx, self.p, self.g, self.ctx.lib
        qkv = [self.qkv.data_ptr() + 2 * D * i for i in range(3)]
        dqkv = [self.dqkv.data_ptr() + 2 * D * i for i in range(3)]
        scale = 1.0 / math.sqrt(HD)
        one = dict(gate_rows=S)
        two = dict(gate_rows=T, scale_h=0.9, scale_b=1.1)
        c.junction_fwd_bf16(p["h0"], p["b0"], p["gp0"], p["gate0"], p["gq0"], self.h1, self.y1, T, D, **one)
        c.gemm_ex(self.y1, p["wqkv"], self.qkv, T, 3 * D, D, D, 3 * D, 3 * D, out_bf16=1)
        c.rope_bf16(qkv[0], qkv[1], qkv[0], qkv[1], self.table, T, H, H, HD, *[3 * D] * 4, seq=S)
        c.check(lib.bwpp_cuda_attention_fwd_lse_bf16(c.handle, *qkv, 3 * D, B, H, S, scale, 1, self.o.data_ptr(), D,
                                                     self.alse.data_ptr()), "attention")
        c.gemm_ex(self.o, p["wo"], self.b1, T, D, D, D, D, D, out_bf16=1)
        c.junction_fwd_bf16(self.h1, self.b1, p["gp1"], p["gate1"], p["gq1"], self.h2, self.y2, T, D, **two)
        c.xent_fwd(self.y2, p["wv"], p["target"], self.loss, self.lse, T, V, D, D, D, w_vocab_major=1)
        # backward
        c.xent_bwd(self.y2, p["wv"], p["target"], self.lse, p["dloss"], self.dy2, g["wv"], T, V, D, D, D, D, D,
                   w_vocab_major=1, grads_bf16=1)
        c.junction_bwd_bf16(self.h2, self.b1, p["gp1"], p["gate1"], p["gq1"], None, self.dy2, self.dh1, self.db1,
                            g["gp1"], g["gate1"], g["gq1"], T, D, **two)
        c.gemm_ex(self.db1, p["wo"], self.do, T, D, D, D, D, D, b_mn=0, out_bf16=1)
        c.gemm_ex(self.o, self.db1, g["wo"], D, D, T, D, D, D, a_mn=1)
        c.check(lib.bwpp_cuda_attention_bwd_bf16(c.handle, *qkv, 3 * D, self.o.data_ptr(), D, self.do.data_ptr(), D,
                                                 self.alse.data_ptr(), B, H, S, scale, 1, *dqkv, 3 * D), "attention bwd")
        c.rope_bf16(dqkv[0], dqkv[1], dqkv[0], dqkv[1], self.table, T, H, H, HD, *[3 * D] * 4, seq=S, inverse=1)
        c.gemm_ex(self.dqkv, p["wqkv"], self.dy1, T, D, 3 * D, 3 * D, 3 * D, D, b_mn=0, out_bf16=1)
        c.gemm_ex(self.y1, self.dqkv, g["wqkv"], D, 3 * D, T, D, 3 * D, 3 * D, a_mn=1)
        c.junction_bwd_bf16(self.h1, p["b0"], p["gp0"], p["gate0"], p["gq0"], self.dh1, self.dy1, g["h0"], g["b0"],
                            g["gp0"], g["gate0"], g["gq0"], T, D, **one)

    def outputs(self):
        return {"loss": self.loss, **self.g}


def test_step_against_autograd(ctx):
    p = make(1)
    step = Step(ctx, p)
    step.run()
    ctx.sync()
    loss, grads = checker(p)
    assert rel_fro(step.loss.cpu(), loss.cpu()) <= 2e-3
    for k, want in grads.items():
        assert rel_fro(step.g[k].float().cpu(), want.cpu()) <= 3e-2, k


def test_step_repeats_bit_for_bit(ctx):
    step = Step(ctx, make(2))
    step.run()
    ctx.sync()
    first = {k: v.clone() for k, v in step.outputs().items()}
    step.run()
    ctx.sync()
    assert all(torch.equal(v, first[k]) for k, v in step.outputs().items())


def test_two_steps_at_once_and_captured():
    """Two contexts on two streams run together, eagerly and as replayed graphs,
    and give what one alone gives."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [bwpp.Ctx(0, s.cuda_stream) for s in streams]
    steps = [Step(c, make(3 + i)) for i, c in enumerate(ctxs)]
    torch.cuda.synchronize()
    # a caller's workspace throughout: eager calls and captured ones then take
    # the same variants of the products
    room = [torch.empty(1 << 28, dtype=torch.uint8, device="cuda") for _ in ctxs]
    want = []
    for c, r, s in zip(ctxs, room, steps):
        c.set_workspace(r, r.numel())
        s.run()
        c.sync()
        want.append({k: v.clone() for k, v in s.outputs().items()})
    torch.cuda.synchronize()
    for _ in range(5):
        for s in steps:
            s.run()
    for c in ctxs:
        c.sync()
    for s, w in zip(steps, want):
        assert all(torch.equal(v, w[k]) for k, v in s.outputs().items())
    graphs = []
    for st, s in zip(streams, steps):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            s.run()
        graphs.append(graph)
    torch.cuda.synchronize()
    for s in steps:
        for v in s.outputs().values():
            v.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    for c in ctxs:
        c.sync()
    for s, w in zip(steps, want):
        assert all(torch.equal(v, w[k]) for k, v in s.outputs().items())
    del graphs
    for c in ctxs:
        c.close()
