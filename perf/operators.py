"""The training-step operators around the decoder block, as cases to measure.

  xent   softmax cross entropy over a vocabulary, from hidden states and the
         vocabulary weight, without keeping the logits; its gradient
  rope   rotary positions on q and k together; its gradient
  junction  the norm after a block, its gate and the scaled residual sum, and the
         norm before the next block; its gradient

`run` computes a case with elementary torch operations where `own` is false and
through bwpp.Ctx where it is true.  `exact` is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases -------------------------------------------------------------------

def xent(name, T, V, D, vocab_major, way, ignored=0.0):
    return {"name": name, "op": "xent", "T": T, "V": V, "D": D, "vocab_major": vocab_major,
            "way": way, "ignored": ignored}


def rope(name, dtype, batch, seq, heads_q, heads_k, head_dim, rotary_dim, interleaved=False,
         scaling="none", factor=1.0, start=0, ragged=False, inverse=False, head_major=False):
    return {"name": name, "op": "rope", "type": dtype, "batch": batch, "seq": seq,
            "heads_q": heads_q, "heads_k": heads_k, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "scaling": scaling, "factor": factor, "start": start,
            "ragged": ragged, "inverse": inverse, "head_major": head_major}


def junction(name, dtype, batch, seq, cols, gate, way, norm_after=True, scale_h=1.0, scale_b=1.0):
    return {"name": name, "op": "junction", "type": dtype, "batch": batch, "seq": seq, "cols": cols,
            "gate": gate, "way": way, "norm_after": norm_after, "scale_h": scale_h,
            "scale_b": scale_b}


def listed():
    return [
        # the loss of one sampled token while a model answers: the weight is read once
        xent("xent one token", 1, 32000, 1024, False, "fwd"),
        # evaluation of a batch, the vocabulary head of the decoder example
        xent("xent fwd", 8192, 32000, 1024, False, "fwd"),
        # the loss's backward in a training step, weight tied to the embedding rows
        xent("xent bwd", 8192, 32000, 2048, True, "bwd"),
        # a fine-tuning batch whose prompts are ignored; no size is a multiple of 8
        xent("xent odd fwd+bwd", 777, 10007, 1001, False, "train", ignored=0.3),
        # one new token at a far position
        rope("rope one token", "bf16", 1, 1, 16, 16, 128, 128, start=4097),
        # a training batch, q and k inside the fused qkv product
        rope("rope train", "bf16", 16, 2048, 16, 16, 128, 128),
        # the gradient of a long-context batch: shared k heads, neighbouring pairs, part of
        # the head, packed sequences of their own positions
        rope("rope grad partial", "f16", 3, 2731, 20, 4, 96, 64, interleaved=True, scaling="parts",
             factor=16.0, ragged=True, inverse=True),
        # f32 into the [batch, heads, seq, dim] layout of the attention call
        rope("rope f32 head major", "f32", 4, 1021, 16, 16, 128, 128, scaling="linear", factor=4.0,
             start=100000, head_major=True),
        # one new token through a block's end
        junction("junction one token", "bf16", 1, 1, 2048, "channel", "fwd"),
        # a training batch, forward and backward, a learned gate per channel
        junction("junction fwd", "bf16", 16, 2048, 2048, "channel", "fwd"),
        junction("junction bwd", "bf16", 16, 2048, 2048, "channel", "bwd"),
        # conditioned model: a gate per sequence, odd width, f32 throughout
        junction("junction odd bwd", "f32", 5, 811, 1003, "sequence", "bwd", scale_h=0.7, scale_b=1.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "rope", "junction"])
    if op == "xent":
        while True:
            T, V, D = _log(rng, 1, 16384), _log(rng, 500, 128000), _log(rng, 64, 4096)
            if rng.random() < 0.5:
                V, D = V // 8 * 8, max(64, D // 64 * 64)
            if T * V * D <= 8192 * 32000 * 2048 and T * V <= 8192 * 32000:
                break
        return _unnamed(xent("", T, V, D, rng.random() < 0.5, rng.choice(["fwd", "bwd", "train"]),
                             rng.choice([0.0, 0.1, 0.5])))
    if op == "rope":
        while True:
            head_dim = rng.choice([32, 64, 80, 96, 128, 160, 256, 2 * rng.randint(3, 100)])
            batch, seq = rng.randint(1, 8), _log(rng, 1, 16384)
            hq = rng.choice([1, 4, 8, 16, 24, 32, 40])
            hk = rng.choice([h for h in (1, 2, 4, 8, 16, 24, 32, 40) if hq % h == 0])
            if batch * seq * (hq + hk) * head_dim <= 16 * 2048 * 32 * 128 // 2:
                break
        part = rng.choice([1, 1, 2, 4])
        return _unnamed(rope("", rng.choice(["bf16", "bf16", "f16", "f32"]), batch, seq, hq, hk, head_dim,
                             max(4, head_dim // part // 2 * 2), rng.random() < 0.5,
                             *rng.choice([("none", 1.0), ("linear", 4.0), ("base", 8.0), ("parts", 16.0)]),
                             _log(rng, 1, 1000000), rng.random() < 0.5, rng.random() < 0.4,
                             rng.random() < 0.3))
    while True:
        batch, seq, cols = rng.randint(1, 16), _log(rng, 1, 8192), _log(rng, 32, 16384)
        if rng.random() < 0.5:
            cols = max(32, cols // 32 * 32)
        if batch * seq * cols <= 16 * 2048 * 2048 // 2:
            break
    return _unnamed(junction("", rng.choice(["bf16", "bf16", "f16", "f32"]), batch, seq, cols,
                             rng.choice(["none", "channel", "sequence", "token"]),
                             rng.choice(["fwd", "bwd"]), rng.random() < 0.75,
                             rng.choice([1.0, 0.7]), rng.choice([1.0, 1.3])))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def work(case):
    if case["op"] == "xent":
        T, V, D = case["T"], case["V"], case["D"]
        fwd = {"bytes": 2 * T * D + 2 * V * D + 12 * T, "flops": 2 * T * V * D}
        # the logits are not kept: their product is computed again, then dx and dw
        bwd = {"bytes": 4 * T * D + 4 * V * D + 12 * T, "flops": 6 * T * V * D}
        if case["way"] == "fwd":
            return fwd
        if case["way"] == "bwd":
            return bwd
        return {k: fwd[k] + bwd[k] for k in fwd}
    rows = case["batch"] * case["seq"]
    s = SIZE[case["type"]]
    if case["op"] == "rope":
        n = rows * (case["heads_q"] + case["heads_k"]) * case["head_dim"]
        turned = n * case["rotary_dim"] // case["head_dim"]
        return {"bytes": 2 * s * n + (4 * rows if case["ragged"] else 0), "flops": 3 * turned}
    cols, n = case["cols"], rows * case["cols"]
    gates = {"none": 0, "channel": 1, "sequence": case["batch"], "token": rows}[case["gate"]] * cols
    if case["way"] == "fwd":
        return {"bytes": n * (8 + 2 * s) + 4 * gates + 8 * cols, "flops": 11 * n}
    return {"bytes": n * (12 + 3 * s) + 8 * gates + 16 * cols, "flops": 30 * n}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inv_freq(case):
    """Radians per position of each pair, float64, on the host."""
    R, base, f = case["rotary_dim"], 10000.0, case["factor"]
    i = torch.arange(0, R, 2, dtype=torch.float64)
    if case["scaling"] == "base":
        base = base * f ** (R / (R - 2))
    inv = base ** (-i / R)
    if case["scaling"] == "linear":
        inv = inv / f
    if case["scaling"] == "parts":
        turns = CONTEXT * inv / (2 * math.pi)  # turns over the trained context
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0, 1)
        inv = inv * keep + inv / f * (1 - keep)
    return inv


# "parts": pairs that turn more than HIGH times over the trained context keep their
# frequency, pairs below LOW turns are slowed by the factor
CONTEXT, LOW, HIGH = 4096.0, 1.0, 32.0


def _amplitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0


def prepare(case, seed):
    g = _gen(seed)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "xent":
        T, V, D = case["T"], case["V"], case["D"]
        w = (rnd(V, D) * (2.0 / math.sqrt(D))).bfloat16()
        target = torch.randint(0, V, (T,), device="cuda", generator=g)
        # hidden states as a trained model has them: from unsure to sure of the target
        lift = 4.0 * torch.rand(T, 1, device="cuda", generator=g)
        x = (rnd(T, D) + lift * w[target].float()).bfloat16()
        valid = torch.rand(T, device="cuda", generator=g) >= case["ignored"]
        s["w"] = w if case["vocab_major"] else w.t().contiguous()
        s["x"], s["target"] = x, torch.where(valid, target, -1).int()
        s["dloss"] = valid.float() / valid.sum().clamp(min=1)
        s["loss"], s["lse"] = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        if case["way"] == "bwd":
            s["lse"] = torch.logsumexp(x.float() @ w.float().t(), 1)
        if case["way"] != "fwd":
            s["dx"], s["dw"] = torch.empty_like(x), torch.empty_like(s["w"])
        return s
    t = TYPES[case["type"]]
    rows = case["batch"] * case["seq"]
    if case["op"] == "rope":
        d = case["head_dim"]
        nq, nk = case["heads_q"] * d, case["heads_k"] * d
        s["qkv"] = rnd(rows, nq + 2 * nk).to(t)  # the fused product; v is not touched
        s["positions"] = None
        if case["ragged"]:  # packed sequences: each row has its own position
            s["positions"] = torch.randint(0, case["start"] + case["seq"] + 1, (rows,), device="cuda",
                                           generator=g).int()
        if case["head_major"]:
            s["q"] = torch.empty(case["batch"], case["heads_q"], case["seq"], d, device="cuda", dtype=t)
            s["k"] = torch.empty(case["batch"], case["heads_k"], case["seq"], d, device="cuda", dtype=t)
        else:
            s["q"] = torch.empty(rows, nq, device="cuda", dtype=t)
            s["k"] = torch.empty(rows, nk, device="cuda", dtype=t)
        return s
    c = case["cols"]
    s["h"], s["b"] = rnd(rows, c) * 3.0, (rnd(rows, c) * 0.5).to(t)
    s["gain_post"] = 1 + 0.1 * rnd(c) if case["norm_after"] else None
    s["gain_pre"] = 1 + 0.1 * rnd(c)
    groups = {"none": 0, "channel": 1, "sequence": case["batch"], "token": rows}[case["gate"]]
    s["gate"] = 0.5 + 0.3 * rnd(groups, c) if groups else None
    if case["way"] == "fwd":
        s["h_out"], s["y"] = torch.empty_like(s["h"]), torch.empty_like(s["b"])
    else:  # h is the stream after the block here, dh_out the gradient from above
        s["dh_out"], s["dy"] = rnd(rows, c), rnd(rows, c).to(t)
        s["dh"], s["db"] = torch.empty_like(s["h"]), torch.empty_like(s["b"])
        s["dgain_pre"] = torch.empty(c, device="cuda")
        s["dgain_post"] = torch.empty(c, device="cuda") if case["norm_after"] else None
        s["dgate"] = torch.empty(groups, c, device="cuda") if groups else None
    return s


EPS = 1e-5


def _gate_rows(case):
    rows = case["batch"] * case["seq"]
    return {"none": rows, "channel": rows, "sequence": case["seq"], "token": 1}[case["gate"]]


# ---- one pass ----------------------------------------------------------------

def run(s):
    return _OWN[s["case"]["op"]](s) if own else _PLAIN[s["case"]["op"]](s)


def _plain_xent(s):
    case, x, target = s["case"], s["x"].float(), s["target"].long()
    w = s["w"].float() if case["vocab_major"] else s["w"].float().t()
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    out = {}
    valid = target >= 0
    lse = s["lse"]
    if case["way"] != "bwd":
        lse = (top + (logits - top).exp().sum(1, keepdim=True).log())[:, 0]
        hit = logits.gather(1, target.clamp(min=0)[:, None])[:, 0]
        out["loss"], out["lse"] = torch.where(valid, lse - hit, torch.zeros_like(lse)), lse
    if case["way"] != "fwd":
        d = (logits - lse[:, None]).exp()
        rows = torch.arange(case["T"], device=x.device)
        d[rows, target.clamp(min=0)] -= 1.0
        d = torch.where(valid[:, None], d * s["dloss"][:, None], torch.zeros_like(d))
        out["dx"] = (d @ w).bfloat16()
        out["dw"] = (d.t() @ x if case["vocab_major"] else x.t() @ d).bfloat16()
    return out


def _plain_rope(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    rows, d, R = case["batch"] * case["seq"], case["head_dim"], case["rotary_dim"]
    nq, nk = case["heads_q"] * d, case["heads_k"] * d
    if case["ragged"]:
        pos = s["positions"].double()
    else:
        pos = case["start"] + torch.arange(rows, device="cuda").remainder(case["seq"]).double()
    angle = pos[:, None] * _inv_freq(case).cuda()
    sign = -1.0 if case["inverse"] else 1.0
    cos = (angle.cos() * _amplitude(case)).float()[:, None]
    sin = (angle.sin() * (sign * _amplitude(case))).float()[:, None]

    def turn(x, heads):
        x = x.float().view(rows, heads, d)
        if case["interleaved"]:
            a, b = x[..., 0:R:2], x[..., 1:R:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :R // 2], x[..., R // 2:R]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        y = torch.cat([y, x[..., R:]], -1).to(t)
        if case["head_major"]:
            return y.view(case["batch"], case["seq"], heads, d).transpose(1, 2).contiguous()
        return y.reshape(rows, heads * d)

    return {"q": turn(s["qkv"][:, :nq], case["heads_q"]), "k": turn(s["qkv"][:, nq:nq + nk], case["heads_k"])}


def _plain_junction(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    rows, c = case["batch"] * case["seq"], case["cols"]
    h, b = s["h"], s["b"].float()
    rb = (b.square().mean(1, keepdim=True) + EPS).rsqrt() if case["norm_after"] else None
    u = b * rb * s["gain_post"] if case["norm_after"] else b
    gate = s["gate"].repeat_interleave(_gate_rows(case), 0) if s["gate"] is not None else torch.ones_like(b)
    if case["way"] == "fwd":
        h2 = case["scale_h"] * h + case["scale_b"] * (gate * u)
        y = h2 * (h2.square().mean(1, keepdim=True) + EPS).rsqrt() * s["gain_pre"]
        return {"h_out": h2, "y": y.to(t)}
    dy = s["dy"].float()
    rh = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    hat, gy = h * rh, dy * s["gain_pre"]
    dh2 = s["dh_out"] + rh * (gy - hat * (gy * hat).mean(1, keepdim=True))
    e = case["scale_b"] * dh2
    out = {"dh": case["scale_h"] * dh2, "dgain_pre": (dy * hat).sum(0)}
    du = e * gate
    if s["gate"] is not None:
        out["dgate"] = (e * u).view(-1, _gate_rows(case), c).sum(1)
    if case["norm_after"]:
        bh, gu = b * rb, du * s["gain_post"]
        out["dgain_post"] = (du * bh).sum(0)
        out["db"] = (rb * (gu - bh * (gu * bh).mean(1, keepdim=True))).to(t)
    else:
        out["db"] = du.to(t)
    return out


_PLAIN = {"xent": _plain_xent, "rope": _plain_rope, "junction": _plain_junction}

_KEPT = {}  # the program's context and its rotary tables, one per model configuration


def _bwpp():
    if "ctx" not in _KEPT:
        path = os.path.join(os.getcwd(), "bluewolf-plus-plus_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bwpp
        _KEPT["bwpp"], _KEPT["ctx"] = bwpp, bwpp.Ctx(torch.cuda.current_device())
    return _KEPT["bwpp"], _KEPT["ctx"]


def _own_xent(s):
    _, ctx = _bwpp()
    case, out = s["case"], {}
    T, V, D = case["T"], case["V"], case["D"]
    ldw = D if case["vocab_major"] else V
    if case["way"] != "bwd":
        ctx.xent_fwd(s["x"], s["w"], s["target"], s["loss"], s["lse"], T, V, D, D, ldw,
                     w_vocab_major=case["vocab_major"])
        out["loss"], out["lse"] = s["loss"], s["lse"]
    if case["way"] != "fwd":
        ctx.xent_bwd(s["x"], s["w"], s["target"], s["lse"], s["dloss"], s["dx"], s["dw"], T, V, D, D,
                     ldw, D, ldw, w_vocab_major=case["vocab_major"], grads_bf16=1)
        out["dx"], out["dw"] = s["dx"], s["dw"]
    return out


def _own_rope(s):
    bwpp, ctx = _bwpp()
    case = s["case"]
    key = (case["rotary_dim"], case["scaling"], case["factor"])
    if key not in _KEPT:
        _KEPT[key] = bwpp.rope_table(case["rotary_dim"], base=10000.0, scaling=case["scaling"],
                                     factor=case["factor"], context=CONTEXT, low=LOW, high=HIGH,
                                     amplitude=_amplitude(case))
    d = case["head_dim"]
    nq, nk = case["heads_q"] * d, case["heads_k"] * d
    major = case["head_major"]
    call = {"bf16": ctx.rope_bf16, "f16": ctx.rope_f16, "f32": ctx.rope_f32}[case["type"]]
    k = s["qkv"].data_ptr() + nq * SIZE[case["type"]]
    call(s["qkv"], k, s["q"], s["k"], _KEPT[key], case["batch"] * case["seq"], case["heads_q"],
         case["heads_k"], d, nq + 2 * nk, nq + 2 * nk, d if major else nq, d if major else nk,
         positions=s["positions"], seq=case["seq"], pos0=case["start"], interleaved=case["interleaved"],
         inverse=case["inverse"], head_major_out=major)
    return {"q": s["q"], "k": s["k"]}


def _own_junction(s):
    _, ctx = _bwpp()
    case = s["case"]
    rows, c = case["batch"] * case["seq"], case["cols"]
    how = dict(gate_rows=_gate_rows(case), norm_after=case["norm_after"], scale_h=case["scale_h"],
               scale_b=case["scale_b"], eps_post=EPS, eps_pre=EPS)
    if case["way"] == "fwd":
        call = {"bf16": ctx.junction_fwd_bf16, "f16": ctx.junction_fwd_f16,
                "f32": ctx.junction_fwd_f32}[case["type"]]
        call(s["h"], s["b"], s["gain_post"], s["gate"], s["gain_pre"], s["h_out"], s["y"], rows, c, **how)
        return {"h_out": s["h_out"], "y": s["y"]}
    call = {"bf16": ctx.junction_bwd_bf16, "f16": ctx.junction_bwd_f16,
            "f32": ctx.junction_bwd_f32}[case["type"]]
    call(s["h"], s["b"], s["gain_post"], s["gate"], s["gain_pre"], s["dh_out"], s["dy"], s["dh"], s["db"],
         s["dgain_post"], s["dgate"], s["dgain_pre"], rows, c, **how)
    return {k: s[k] for k in ("dh", "db", "dgain_post", "dgate", "dgain_pre") if s[k] is not None}


_OWN = {"xent": _own_xent, "rope": _own_rope, "junction": _own_junction}


# ---- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"xent": _exact_xent, "rope": _exact_rope, "junction": _exact_junction}[case["op"]](case, s)


def _exact_xent(case, s):
    w = (s["w"] if case["vocab_major"] else s["w"].t()).double()
    out = {"loss": [], "lse": [], "dx": []}
    dw = torch.zeros_like(w)
    for x, target, g in zip(s["x"].split(1024), s["target"].split(1024), s["dloss"].split(1024)):
        x, g = x.double(), g.double()
        logp = torch.log_softmax(x @ w.t(), 1)
        hit = torch.nn.functional.one_hot(target.long().clamp(min=0), case["V"])
        valid = (target >= 0).double()
        loss = -(logp * hit).sum(1) * valid
        out["loss"].append(loss)
        out["lse"].append(torch.logsumexp(x @ w.t(), 1))
        if case["way"] != "fwd":
            d = (logp.exp() - hit) * (g * valid)[:, None]
            out["dx"].append(d @ w)
            dw += d.t() @ x
    if case["way"] == "bwd":
        return {"dx": torch.cat(out["dx"]), "dw": dw if case["vocab_major"] else dw.t().contiguous()}
    fwd = {"loss": torch.cat(out["loss"]), "lse": torch.cat(out["lse"])}
    if case["way"] == "fwd":
        return fwd
    return {**fwd, "dx": torch.cat(out["dx"]), "dw": dw if case["vocab_major"] else dw.t().contiguous()}


def _exact_rope(case, s):
    B, S, d, R = case["batch"], case["seq"], case["head_dim"], case["rotary_dim"]
    pos = s["positions"].double() if case["ragged"] else \
        (case["start"] + torch.arange(S, device="cuda").double()).repeat(B)
    z = torch.polar(torch.full((B * S, R // 2), _amplitude(case), dtype=torch.float64, device="cuda"),
                    torch.outer(pos, _inv_freq(case).cuda()))
    z = z.conj() if case["inverse"] else z
    at = 0
    out = {}
    for name, heads in (("q", case["heads_q"]), ("k", case["heads_k"])):
        x = s["qkv"][:, at:at + heads * d].double().reshape(B * S, heads, d)
        at += heads * d
        shape = (B * S, heads, R // 2, 2) if case["interleaved"] else (B * S, heads, 2, R // 2)
        p = x[..., :R].reshape(shape)
        p = p if case["interleaved"] else p.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z[:, None])
        y = y if case["interleaved"] else y.transpose(-1, -2)
        y = torch.cat([y.reshape(B * S, heads, R), x[..., R:]], -1)
        out[name] = y.view(B, S, heads, d).permute(0, 2, 1, 3).contiguous() if case["head_major"] \
            else y.reshape(B * S, heads * d)
    return out


def _exact_junction(case, s):
    """The forward in 64 bits; the backward as its derivative (torch.autograd)."""
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    h, b, gp, gate, gq = (wide(s[k]) for k in ("h", "b", "gain_post", "gate", "gain_pre"))
    rows, c = h.shape

    def rms(x):
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()

    def after(b, gp, gate):
        u = rms(b) * gp if case["norm_after"] else b
        if gate is not None:
            u = (u.view(gate.shape[0], -1, c) * gate[:, None]).reshape(rows, c)
        return case["scale_b"] * u

    if case["way"] == "fwd":
        h2 = case["scale_h"] * h + after(b, gp, gate)
        return {"h_out": h2, "y": rms(h2) * gq}
    h, gq = h.requires_grad_(), gq.requires_grad_()
    (rms(h) * gq).backward(wide(s["dy"]))
    dh2 = s["dh_out"].double() + h.grad
    b.requires_grad_()
    gp = gp.requires_grad_() if gp is not None else None
    gate = gate.requires_grad_() if gate is not None else None
    after(b, gp, gate).backward(dh2)
    out = {"dh": case["scale_h"] * dh2, "db": b.grad, "dgain_pre": gq.grad}
    if gp is not None:
        out["dgain_post"] = gp.grad
    if gate is not None:
        out["dgate"] = gate.grad
    return out
