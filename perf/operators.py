"""What is measured of the operators of a gradient step: attention with its backward pass, and the
global norm and clipping of the gradients.

Three kinds of case:

* ``step``: attention forward and backward through autograd, as a training loop calls it;
* ``backward``: the backward pass alone, from the outputs and row statistics that a forward kept;
* ``norm`` / ``clip``: the norm over a model's gradients, and the gradients scaled by it.

``own = False`` computes the plain form in elementary torch operations, ``own = True`` calls the
framework.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@functools.lru_cache(maxsize=None)
def _framework():
    root = str(Path(__file__).resolve().parent.parent / "muzo-clip_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import muzo_clip_b200

    return muzo_clip_b200


# ---------------------------------------------------------------- cases


def _attention(name, kind, b, hq, hkv, sq, sk, d, dtype, causal, pad="none", record=False):
    return {"name": name, "kind": kind, "batch": b, "heads": hq, "kv_heads": hkv, "seq_q": sq, "seq_k": sk,
            "head_dim": d, "dtype": dtype, "causal": causal, "pad": pad, "record": record}


def _gradients(name, kind, layers, hidden, kv, mlp, vocab, dtype, out="same"):
    return {"name": name, "kind": kind, "layers": layers, "hidden": hidden, "kv_width": kv, "mlp": mlp,
            "vocab": vocab, "dtype": dtype, "out": out}


def listed():
    return [
        # the tiny Llama of the optimizer's end-to-end run (batch 4 x 64 tokens, 4 heads of 64):
        # a call whose launches cost more than its arithmetic
        _attention("step tiny llama", "step", 4, 4, 4, 64, 64, 64, "bf16", True),
        # one Llama-3-8B-shaped layer on a training sequence
        _attention("step llama-8b layer", "step", 1, 32, 8, 2048, 2048, 128, "bf16", True),
        # one Llama-3-70B-shaped layer with the per-head maxima that QK-Clip records
        _attention("step llama-70b layer", "step", 1, 64, 8, 4096, 4096, 128, "bf16", True, record=True),
        # a batch of sentences padded on the right, every token seeing its whole sentence, fp16
        _attention("step padded batch", "step", 8, 12, 12, 1000, 1000, 64, "fp16", False, pad="right"),
        # a small odd batch padded on the left: the first rows see no key
        _attention("backward small left-padded", "backward", 3, 6, 3, 77, 77, 128, "bf16", True, pad="left"),
        # new tokens after a prefix that needs gradients too (end-aligned causality), heads of 96
        _attention("backward after a prefix", "backward", 2, 16, 4, 300, 2348, 96, "bf16", True),
        # a long sequence whose query heads all share one key head
        _attention("backward long multi-query", "backward", 1, 8, 1, 16384, 16384, 128, "bf16", True),
        # every gradient of the tiny Llama, fp32
        _gradients("norm tiny llama", "norm", 2, 256, 256, 688, 1024, "fp32"),
        # six Llama-3-8B-shaped layers, bf16: many times the L2 cache
        _gradients("norm llama-8b layers", "norm", 6, 4096, 1024, 14336, 0, "bf16"),
        # the same two with the scaled gradients written: in the gradients' type, and to fp32
        _gradients("clip tiny llama", "clip", 2, 256, 256, 688, 1024, "fp32"),
        _gradients("clip odd widths", "clip", 4, 1037, 259, 2751, 1009, "bf16"),
        _gradients("clip llama-8b layers", "clip", 6, 4096, 1024, 14336, 0, "bf16", out="fp32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "backward", "step", "backward", "norm", "clip"])
    if kind in ("norm", "clip"):
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        out = rng.choice(["same", "fp32"]) if kind == "clip" else "same"
        hidden = _log_uniform(rng, 16, 4096)
        case = _gradients("", kind, rng.randint(1, 6), hidden, max(1, hidden // rng.choice([1, 2, 4, 8])),
                          int(hidden * rng.uniform(2.0, 3.5)) + 1, rng.choice([0, _log_uniform(rng, 100, 30000)]), dtype, out)
    else:
        hkv = rng.choice([1, 2, 3, 4, 8])
        sq = _log_uniform(rng, 1, 6000)
        # one query alone comes with more keys than one: a softmax over one key has no gradient
        sk = sq if sq > 1 and rng.random() < 0.75 else sq + _log_uniform(rng, 1, 3000)
        causal = rng.random() < 0.7
        case = _attention("", kind, rng.randint(1, 6), hkv * rng.choice([1, 2, 4, 8]), hkv, sq, sk,
                          rng.choice([64, 128, 64, 128, 32, 80, 96]), rng.choice(["bf16", "bf16", "fp16"]), causal,
                          rng.choice(["none", "none", "right", "left"]), kind == "step" and rng.random() < 0.3)
        # no more work, and no larger probability matrices, than the largest listed cases have
        most = 64 * 4096 * 4096
        while case["batch"] > 1 and case["batch"] * case["heads"] * sq * sk > most // 2:
            case["batch"] -= 1
        while case["heads"] > case["kv_heads"] and case["heads"] * sq * sk > most // 2:
            case["heads"] -= case["kv_heads"]
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs


def _key_range(case):
    """Per batch row the visible keys [lo, hi): lengths spread from a third of the keys to all."""
    sk, b = case["seq_k"], case["batch"]
    lengths = [max(1, sk - (2 * sk * i) // (3 * b)) for i in range(b)]
    if case["pad"] == "right":
        return [0] * b, lengths
    if case["pad"] == "left":
        return [sk - n for n in lengths], [sk] * b
    return None


def _tensor_shapes(case):
    h, kv, mlp, shapes = case["hidden"], case["kv_width"], case["mlp"], []
    if case["vocab"]:
        shapes.append((case["vocab"], h))
    for _ in range(case["layers"]):
        shapes += [(h, h), (kv, h), (kv, h), (h, h), (mlp, h), (mlp, h), (h, mlp), (h,), (h,)]
    return shapes


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["kind"] in ("norm", "clip"):
        # every tensor has a scale of its own, as layers have; the embedding's unused rows are zero
        shapes = _tensor_shapes(case)
        scales = torch.exp(torch.randn(len(shapes), generator=g, device=dev) * 1.5 - 5.0)
        grads = [torch.randn(s, generator=g, device=dev, dtype=dtype).mul_(scales[i]) for i, s in enumerate(shapes)]
        if case["vocab"]:
            grads[0].mul_((torch.rand(case["vocab"], 1, generator=g, device=dev) < 0.3).to(dtype))
        out_dtype = dtype if case["out"] == "same" else DTYPES[case["out"]]
        state.update(grads=grads, max_norm=1.0, destination=[torch.empty_like(x, dtype=out_dtype) for x in grads] if case["kind"] == "clip" else None)
        return state
    b, hq, hkv, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))

    def states(s, h, scale=1.0):
        x = torch.randn((b, s, h, d), generator=g, device=dev, dtype=torch.float32) * scale
        return x.to(dtype).transpose(1, 2)   # the projections' [B, S, H, D], seen as [B, H, S, D]

    q, k, v = states(sq, hq, 1.3), states(sk, hkv, 1.3), states(sk, hkv)
    dout = states(sq, hq, 0.2).transpose(1, 2)
    lo = hi = None
    ranges = _key_range(case)
    if ranges is not None:
        lo, hi = (torch.tensor(r, dtype=torch.int32, device=dev) for r in ranges)
    state.update(q=q, k=k, v=v, dout=dout, lo=lo, hi=hi, scaling=d ** -0.5)
    if case["kind"] == "step":
        for x in (q, k, v):
            x.requires_grad_(True)
    else:
        out, lse, _, _ = _plain_forward(state)
        state.update(out=out.to(dtype), lse=lse)
    return state


# ---------------------------------------------------------------- the plain forms


def _visible(state, sq, sk, device):
    """Boolean [B or 1, 1, Sq, Sk]: the keys that each query sees."""
    j = torch.arange(sk, device=device)
    i = torch.arange(sq, device=device)[:, None] + (sk - sq)
    seen = torch.ones((1, 1, sq, sk), dtype=torch.bool, device=device)
    if state["causal"]:
        seen = seen & (j <= i)
    if state["lo"] is not None:
        seen = seen & ((j >= state["lo"][:, None]) & (j < state["hi"][:, None]))[:, None, None, :]
    return seen


def _grouped(x, hkv):
    """[B, Hq, S, D] as fp32 [B, Hkv, (Hq / Hkv) S, D]: the query heads of one key head in a row."""
    b, h, s, d = x.shape
    return x.float().reshape(b, hkv, (h // hkv) * s, d)


def _plain_probabilities(state, q, k):
    """Scaled logits' row maximum and the normalised probabilities, [B, Hkv, G, Sq, Sk]."""
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    seen = _visible(state, sq, sk, q.device)[:, :, None]
    logits = torch.matmul(_grouped(q, hkv), k.float().transpose(2, 3)).view(b, hkv, hq // hkv, sq, sk)
    raw = logits.masked_fill(~seen, -math.inf) if state["record"] else None
    logits = (logits * state["scaling"]).masked_fill_(~seen, -math.inf)
    top = logits.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)   # a row that sees no key
    p = torch.exp(logits - top)
    total = p.sum(dim=-1, keepdim=True)
    lse = (top + torch.log(total)).view(b, hq, sq)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return p, lse, raw


def _plain_forward(state):
    q, k, v = state["q"].detach(), state["k"].detach(), state["v"].detach()
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    p, lse, raw = _plain_probabilities(state, q, k)
    out = torch.matmul(p.view(b, hkv, -1, sk), v.float()).view(b, hq, sq, d).transpose(1, 2)
    top = None
    if state["record"]:
        # the logits of eager attention: rounded as the product's type, and again after the scaling
        top = raw.amax(dim=(0, 3, 4)).view(hq).to(q.dtype) * state["scaling"]
    return out, lse, p, top


def _plain_backward(state, p, out):
    q, k, v = state["q"].detach(), state["k"].detach(), state["v"].detach()
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    dout = _grouped(state["dout"].transpose(1, 2), hkv)
    delta = (dout * _grouped(out.transpose(1, 2), hkv)).sum(dim=-1, keepdim=True)
    p = p.view(b, hkv, -1, sk)
    dv = torch.matmul(p.transpose(2, 3), dout)
    ds = torch.matmul(dout, v.float().transpose(2, 3)).sub_(delta).mul_(p)
    dq = torch.matmul(ds, k.float()).mul_(state["scaling"]).view(b, hq, sq, d)
    dk = torch.matmul(ds.transpose(2, 3), _grouped(q, hkv)).mul_(state["scaling"])
    return {"dq": dq.to(q.dtype), "dk": dk.to(q.dtype), "dv": dv.to(q.dtype)}


def _plain_norm(grads):
    return torch.stack([torch.sum(x.float().square(), dtype=torch.float64) for x in grads]).sum().sqrt().float()


def _plain_clip(grads, max_norm, destination):
    norm = _plain_norm(grads)
    factor = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    return {"grads": [o.copy_(x.float() * factor) for x, o in zip(grads, destination)], "norm": norm}


# ---------------------------------------------------------------- one pass


def run(state):
    kind = state["kind"]
    if own:
        m = _framework()
        if kind == "norm":
            return m.grad_norm(state["grads"])
        if kind == "clip":
            grads, norm = m.clip_grads(state["grads"], state["max_norm"], out=state["destination"])
            return {"grads": grads, "norm": norm}
        q, k, v = state["q"], state["k"], state["v"]
        if kind == "backward":
            dq, dk, dv = m.attention_max_backward(state["dout"], q, k, v, state["out"], state["lse"], state["scaling"],
                                                  state["causal"], state["lo"], state["hi"])
            return {"dq": dq, "dk": dk, "dv": dv}
        out, smax, _valid = m.attention_max(q, k, v, state["scaling"], state["causal"], state["lo"], state["hi"],
                                            record=state["record"])
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
        got = {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
        if state["record"]:
            got["smax"] = smax.to(q.dtype)   # the maxima are values of this type
        return got
    if kind == "norm":
        return _plain_norm(state["grads"])
    if kind == "clip":
        return _plain_clip(state["grads"], state["max_norm"], state["destination"])
    if kind == "backward":
        p, _, _ = _plain_probabilities(state, state["q"], state["k"])
        return _plain_backward(state, p, state["out"])
    out, _, p, top = _plain_forward(state)
    got = {"out": out.to(state["q"].dtype), **_plain_backward(state, p, out)}
    if state["record"]:
        got["smax"] = top
    return got


# ---------------------------------------------------------------- the least work


def _visible_pairs(case):
    """Pairs of a query and a key that it sees, summed over the batch."""
    sq, sk, total = case["seq_q"], case["seq_k"], 0
    ranges = _key_range(case) or ([0] * case["batch"], [sk] * case["batch"])
    for lo, hi in zip(*ranges):
        if not case["causal"]:
            total += sq * (hi - lo)
        else:
            total += sum(max(0, min(hi, i + sk - sq + 1) - lo) for i in range(sq))
    return total


def work(case):
    if case["kind"] in ("norm", "clip"):
        n = sum(math.prod(s) for s in _tensor_shapes(case))
        size = 4 if case["dtype"] == "fp32" else 2
        out = 0 if case["kind"] == "norm" else 4 if "fp32" in (case["out"], case["dtype"]) else 2
        return {"bytes": n * (size + out) + 4, "flops": n * (2 if case["kind"] == "norm" else 3)}
    b, hq, hkv, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))
    q, kv = b * hq * sq * d * 2, b * hkv * sk * d * 2
    pairs = hq * _visible_pairs(case)
    # products of 2 d operations for each visible pair: 2 forward, 5 backward (the logits again)
    if case["kind"] == "step":
        return {"bytes": 4 * q + 4 * kv, "flops": 7 * 2 * d * pairs}
    return {"bytes": 4 * q + 4 * kv + b * hq * sq * 4, "flops": 5 * 2 * d * pairs}


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("norm", "clip"):
        squares = [float(x.double().pow(2).sum()) for x in state["grads"]]
        norm = math.sqrt(math.fsum(squares))
        top = torch.tensor(norm, dtype=torch.float64)
        if case["kind"] == "norm":
            return top
        factor = min(1.0, state["max_norm"] / (norm + 1e-6))
        return {"grads": [x.double() * factor for x in state["grads"]], "norm": top}
    b, hq, hkv, sq, sk, d = (case[k] for k in ("batch", "heads", "kv_heads", "seq_q", "seq_k", "head_dim"))
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    dev, f64 = q.device, torch.float64
    out = torch.zeros((b, sq, hq, d), dtype=f64, device=dev)
    dq = torch.zeros((b, hq, sq, d), dtype=f64, device=dev)
    dk, dv = (torch.zeros((b, hkv, sk, d), dtype=f64, device=dev) for _ in range(2))
    smax = torch.full((hq,), -math.inf, dtype=f64, device=dev)
    ranges = _key_range(case)
    for bi in range(b):
        lo, hi = (ranges[0][bi], ranges[1][bi]) if ranges is not None else (0, sk)
        hidden = torch.zeros((sq, sk), dtype=torch.bool, device=dev)
        hidden[:, :lo] = True
        hidden[:, hi:] = True
        if case["causal"]:
            hidden |= torch.ones((sq, sk), dtype=torch.bool, device=dev).triu(sk - sq + 1)
        empty = hidden.all(dim=1)
        for h in range(hq):
            n = h // (hq // hkv)
            qh, kh, vh = q[bi, h].double(), k[bi, n].double(), v[bi, n].double()
            gh = state["dout"][bi, :, h].double()
            logits = torch.mm(qh, kh.t()).mul_(state["scaling"]).masked_fill_(hidden, -math.inf)
            smax[h] = torch.maximum(smax[h], logits.max())
            p = torch.softmax(logits, dim=1).masked_fill_(empty[:, None], 0.0)
            del logits
            oh = torch.mm(p, vh)
            out[bi, :, h] = oh
            # d softmax: the row's mean of dP under P is taken from dP itself
            dp = torch.mm(gh, vh.t())
            given = state["out"][bi, :, h].double() if case["kind"] == "backward" else oh
            dv[bi, n] += torch.mm(p.t(), gh)
            ds = dp.sub_((gh * given).sum(dim=1, keepdim=True)).mul_(p)
            dq[bi, h] = torch.mm(ds, kh) * state["scaling"]
            dk[bi, n] += torch.mm(ds.t(), qh) * state["scaling"]
    got = {"dq": dq, "dk": dk, "dv": dv}
    if case["kind"] == "step":
        got["out"] = out
        if case["record"]:
            got["smax"] = smax
    return got
