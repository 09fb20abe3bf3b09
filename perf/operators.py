"""Cases, plain forms and 64-bit results of the fine-tuning operators.

Four operators of a training step on preferences or sampled text:

  policy       the clipped policy loss with a KL term over logits: losses, KL estimates, log-probabilities and
               (unless the case is an evaluation) the gradient of the logits
  preference   the preference loss over pairs of sequences (chosen, rejected): losses, rewards and the gradient
               of the logits
  clip         the norm over all gradient tensors of a model, and the gradients clipped to a largest norm
  adamw        the same norm, and the AdamW update that reads the clipped gradients without storing them

Every position has a weight; a weight of zero (prompt and padding) takes the position out of the loss and of the
gradient. Logits have V columns in rows of `ld` elements; the gradient is zero in the columns from V on.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # fine-tuning on sampled answers, 16 sequences of 1024 (the micro-batch of the 124M training step); the
        # prompts, about half of each sequence, carry no weight
        {"name": "policy-16x1024", "op": "policy", "B": 16, "T": 1024, "V": 50257, "ld": 50304, "dtype": "bf16",
         "live": 0.5, "kl": 0.05, "grad": True},
        # every position live, fp32 logits (the TF32 training mode), half the rows of the GEMM benchmark
        {"name": "policy-fp32-4x1024", "op": "policy", "B": 4, "T": 1024, "V": 50257, "ld": 50304, "dtype": "f32",
         "live": 1.0, "kl": 0.02, "grad": True},
        # the 4 x 64 micro-batch of the parity runs: too few rows to fill the GPU one row at a time
        {"name": "policy-4x64", "op": "policy", "B": 4, "T": 64, "V": 50257, "ld": 50304, "dtype": "bf16",
         "live": 1.0, "kl": 0.05, "grad": True},
        # odd sizes of a small test vocabulary, without a reference model: latency
        {"name": "policy-9x37", "op": "policy", "B": 9, "T": 37, "V": 1001, "ld": 1008, "dtype": "f32",
         "live": 0.6, "kl": 0.0, "grad": True},
        # evaluation: losses and KL over 8 x 1024 positions, no gradient
        {"name": "policy-eval-8x1024", "op": "policy", "B": 8, "T": 1024, "V": 50257, "ld": 50304, "dtype": "bf16",
         "live": 1.0, "kl": 0.05, "grad": False},
        # eight pairs of 1024 positions: a preference step at the training micro-batch; answers are half of each
        {"name": "preference-8x1024", "op": "preference", "B": 8, "T": 1024, "V": 50257, "ld": 50304,
         "dtype": "bf16", "live": 0.5, "smooth": 0.0, "grad": True},
        # ragged lengths, fp32 logits, label smoothing
        {"name": "preference-fp32-3x500", "op": "preference", "B": 3, "T": 500, "V": 50257, "ld": 50304,
         "dtype": "f32", "live": 0.6, "smooth": 0.1, "grad": True},
        # two short pairs: latency
        {"name": "preference-2x64", "op": "preference", "B": 2, "T": 64, "V": 50257, "ld": 50304, "dtype": "bf16",
         "live": 0.6, "smooth": 0.0, "grad": True},
        # all 148 gradient tensors of the 124M model, fp32
        {"name": "clip-124m", "op": "clip", "L": 12, "C": 768, "V": 50304, "maxT": 1024, "dtype": "f32",
         "out": "f32", "scale": 1e-3},
        # a two-layer test model whose bf16 gradients become clipped fp32 ones: latency
        {"name": "clip-bf16-2l", "op": "clip", "L": 2, "C": 128, "V": 1001, "maxT": 128, "dtype": "bf16",
         "out": "f32", "scale": 0.01},
        # the optimizer step of the 124M model
        {"name": "adamw-124m", "op": "adamw", "n": 124475904, "scale": 1e-3},
        # the optimizer step of a two-layer test model
        {"name": "adamw-2l", "op": "adamw", "n": 541312, "scale": 1e-2},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["policy", "policy", "preference", "preference", "clip", "adamw"])
    if op in ("policy", "preference"):
        B = _log_int(rng, 1, 16 if op == "policy" else 8)
        T = _log_int(rng, 1, 1024)
        V = _log_int(rng, 500, 131072)
        ld = -(-V // 8) * 8 + 8 * rng.choice([0, 0, 1, 5, 17])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        rows = B * T * (1 if op == "policy" else 2)
        room = 16384 * 50304 * 2 // (ld * _BYTES[dtype])
        while rows > room:  # no dearer than the largest listed case
            T = max(1, T // 2)
            rows = B * T * (1 if op == "policy" else 2)
        case = {"op": op, "B": B, "T": T, "V": V, "ld": ld, "dtype": dtype, "live": round(rng.uniform(0.2, 1.0), 3)}
        if op == "policy":
            return {**case, "kl": rng.choice([0.0, round(rng.uniform(0.01, 0.1), 3)]), "grad": rng.random() < 0.8}
        return {**case, "smooth": rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]), "grad": rng.random() < 0.8}
    if op == "clip":
        dtype = rng.choice(["f32", "bf16", "f16"])
        C = _log_int(rng, 16, 768)
        return {"op": "clip", "L": rng.randint(1, 12), "C": C, "V": _log_int(rng, 100, 50304),
                "maxT": _log_int(rng, 16, 1024), "dtype": dtype, "out": rng.choice([dtype, "f32"]),
                "scale": round(math.exp(rng.uniform(math.log(1e-4), math.log(0.1))), 7)}
    return {"op": "adamw", "n": 4 * _log_int(rng, 250, 31118976),
            "scale": round(math.exp(rng.uniform(math.log(1e-4), math.log(0.1))), 7)}


def _tensor_sizes(case):
    """Element counts of the tensors of a GPT-2 of this shape, one for each weight and bias."""
    C, sizes = case["C"], [case["V"] * case["C"], case["maxT"] * case["C"]]
    for _ in range(case["L"]):
        sizes += [C, C, 3 * C * C, 3 * C, C * C, C, C, C, 4 * C * C, 4 * C, 4 * C * C, C]
    return sizes + [C, C]


def _live_lengths(case, sequences):
    """Live positions of each sequence: ragged, `live` of all on average."""
    T, live = case["T"], case["live"]
    spread = min(0.5, 1.0 / live - 1.0)  # none where every position is live
    return [min(T, round(T * live * (1.0 + spread * (2.0 * (i + 0.5) / sequences - 1.0)))) for i in range(sequences)]


def work(case):
    op = case["op"]
    if op in ("policy", "preference"):
        sequences = case["B"] * (1 if op == "policy" else 2)
        rows, live = sequences * case["T"], sum(_live_lengths(case, sequences))
        es = _BYTES[case["dtype"]]
        # live logits read once, the gradient (zero rows too) written once, about eight values a position beside it
        return {"bytes": live * case["V"] * es + (rows * case["ld"] * es if case["grad"] else 0) + 32 * rows,
                "flops": live * case["V"] * (8 if case["grad"] else 4)}
    if op == "clip":
        n = sum(_tensor_sizes(case))
        return {"bytes": n * (_BYTES[case["dtype"]] + _BYTES[case["out"]]), "flops": 3 * n}
    return {"bytes": case["n"] * 30, "flops": 18 * case["n"]}


# ----------------------------------------------------------------- inputs
def _weights(case, sequences, seed, dev):
    """1 / live rows at the live positions (a span at a drawn place in each sequence), 0 at the others."""
    T, lengths, rng = case["T"], _live_lengths(case, sequences), random.Random(seed)
    w = np.zeros((sequences, T), np.float32)
    for i, n in enumerate(lengths):
        at = rng.randint(0, T - n)
        w[i, at:at + n] = 1.0
    return torch.from_numpy(w.reshape(-1)).to(dev)


def _logits(rows, case, g, dev):
    """Logits of a trained model's spread, the targets drawn from their softmax, and their log-probabilities."""
    x = torch.empty(rows, case["ld"], dtype=_DTYPES[case["dtype"]], device=dev)
    targets = torch.empty(rows, dtype=torch.int32, device=dev)
    logps = torch.empty(rows, device=dev)
    for r in range(0, rows, 4096):
        n = min(4096, rows - r)
        v = torch.randn(n, case["ld"], generator=g, device=dev) * 2.5
        x[r:r + n] = v
        v = x[r:r + n, :case["V"]].float()
        race = torch.empty_like(v).exponential_(generator=g)
        t = (v - race.log_()).argmax(-1)
        targets[r:r + n] = t.int()
        logps[r:r + n] = v.gather(-1, t[:, None])[:, 0] - v.logsumexp(-1)
    return x, targets, logps


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "policy":
        rows = case["B"] * case["T"]
        s["logits"], s["targets"], logps = _logits(rows, case, g, dev)
        w = _weights(case, case["B"], seed, dev)
        s["weights"] = w / w.sum().clamp(min=1.0)
        s["advantages"] = torch.randn(rows, generator=g, device=dev)
        # the sampling policy is a few updates old; no ratio within 1e-4 of a clipping bound, where the rounding
        # of the inputs alone would decide the gradient
        drift = torch.randn(rows, generator=g, device=dev) * 0.15
        near = ((drift.exp() - 1.2).abs() < 1e-4) | ((drift.exp() - 0.8).abs() < 1e-4)
        s["old"] = logps - torch.where(near, drift * 1.01, drift)
        s["ref"] = logps + torch.randn(rows, generator=g, device=dev) * 0.3 if case["kl"] else None
        s["losses"] = torch.empty(rows, device=dev)
        s["kls"] = torch.empty(rows, device=dev) if case["kl"] else None
        s["logps"] = torch.empty(rows, device=dev)
        s["dlogits"] = torch.empty_like(s["logits"]) if case["grad"] else None
    elif op == "preference":
        pairs, rows = case["B"], 2 * case["B"] * case["T"]
        s["logits"], s["targets"], logps = _logits(rows, case, g, dev)
        s["weights"] = _weights(case, 2 * pairs, seed, dev)
        s["ref"] = (logps * s["weights"]).view(2 * pairs, -1).sum(-1) + torch.randn(2 * pairs, generator=g, device=dev) * 4.0
        s["losses"] = torch.empty(pairs, device=dev)
        s["rewards"] = torch.empty(2 * pairs, device=dev)
        s["dlogits"] = torch.empty_like(s["logits"]) if case["grad"] else None
    elif op == "clip":
        n = sum(_tensor_sizes(case))
        # the tensors lie one behind another, as a model's gradients do
        s["grads"] = (torch.randn(n, generator=g, device=dev) * case["scale"]).to(_DTYPES[case["dtype"]])
        s["out"] = torch.empty(n, dtype=_DTYPES[case["out"]], device=dev)
        s["norm"] = torch.empty(1, device=dev)
    else:
        n = case["n"]
        s["params"] = torch.randn(n, generator=g, device=dev) * 0.02
        s["params_bf16"] = torch.empty(n, dtype=torch.bfloat16, device=dev)
        s["grads"] = torch.randn(n, generator=g, device=dev) * case["scale"]
        s["m"] = torch.randn(n, generator=g, device=dev) * (0.1 * case["scale"])
        s["v"] = torch.rand(n, generator=g, device=dev) * case["scale"] ** 2
        s["norm"] = torch.empty(1, device=dev)
        # lr, beta1, beta2, eps, weight decay, 1 / (1 - beta1^t), 1 / (1 - beta2^t), gradient scale; t = 10
        s["hparams"] = torch.tensor([3e-4, 0.9, 0.999, 1e-8, 0.1, 1 / (1 - 0.9 ** 10), 1 / (1 - 0.999 ** 10), 1.0],
                                    device=dev)
    return s


_MAX_NORM = 1.0
_CLIP = 0.2
_BETA = 0.1


# ------------------------------------------------------------- plain forms
def _rows(logits, targets, V):
    """exp(x - max), their sum and the targets' log-probabilities (the sums and logarithms in 64 bits)."""
    x = logits[:, :V].float()
    e = x - x.amax(-1, keepdim=True)
    at = e.gather(-1, targets.long()[:, None])[:, 0].double()
    e = e.exp_()
    total = e.sum(-1, dtype=torch.float64)
    return e, total, at - total.log()


def _dlogits(e, total, targets, c, live, like):
    """c ([j = target] - softmax_j) in the live rows, 0 in the others and in the padding columns."""
    scale = torch.where(live, -c / total, torch.zeros_like(c)).float()
    e = e.mul_(scale[:, None])
    e.scatter_add_(-1, targets.long()[:, None], torch.where(live, c, torch.zeros_like(c)).float()[:, None])
    out = torch.zeros_like(like)
    out[:, :e.shape[1]] = e
    return out


def _plain_policy(s):
    case, w = s["case"], s["weights"].double()
    live = w != 0
    e, total, lp = _rows(s["logits"], s["targets"], case["V"])
    A = s["advantages"].double()
    ratio = (lp - s["old"].double()).exp()
    s1, s2 = ratio * A, ratio.clamp(1 - _CLIP, 1 + _CLIP) * A
    loss = -torch.minimum(s1, s2)
    c = torch.where(s1 > s2, torch.zeros_like(s1), -s1)
    zero = torch.zeros_like(w)
    out = {}
    if case["kl"]:
        d = s["ref"].double() - lp
        kl = torch.expm1(d) - d
        loss = loss + case["kl"] * kl
        c = c - case["kl"] * torch.expm1(d)
        out["kls"] = torch.where(live, kl, zero).float()
    out["losses"] = torch.where(live, w * loss, zero).float()
    out["logps"] = torch.where(live, lp, zero).float()
    if case["grad"]:
        out["dlogits"] = _dlogits(e, total, s["targets"], c * w, live, s["logits"])
    return out


def _plain_preference(s):
    case, w = s["case"], s["weights"].double()
    live = w != 0
    e, total, lp = _rows(s["logits"], s["targets"], case["V"])
    sums = torch.where(live, lp * w, torch.zeros_like(w)).view(2, case["B"], case["T"]).sum(-1)
    rewards = _BETA * (sums - s["ref"].double().view(2, -1))
    h = rewards[0] - rewards[1]
    smooth = case["smooth"]
    soft = lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    out = {"losses": ((1 - smooth) * soft(-h) + smooth * soft(h)).float(), "rewards": rewards.view(-1).float()}
    if case["grad"]:
        slope = (smooth / (1 + torch.exp(-h)) - (1 - smooth) / (1 + torch.exp(h))) * (_BETA / case["B"])
        c = torch.stack([slope, -slope])[:, :, None].expand(2, case["B"], case["T"]).reshape(-1) * w
        out["dlogits"] = _dlogits(e, total, s["targets"], c, live, s["logits"])
    return out


def _plain_norm(g):
    return g.float().square().sum(dtype=torch.float64).sqrt()


def _plain_clip(s):
    norm = _plain_norm(s["grads"])
    k = (_MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    s["norm"].copy_(norm)
    s["out"].copy_(s["grads"].float() * k)
    return {"norm": s["norm"], "out": s["out"]}


def _plain_adamw(s):
    norm = _plain_norm(s["grads"])
    s["norm"].copy_(norm)
    lr, b1, b2, eps, wd, c1, c2, scale = s["hparams"].unbind()
    g = s["grads"] * (scale * (_MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float())
    s["m"].mul_(b1).add_(g * (1 - b1))
    s["v"].mul_(b2).add_(g * g * (1 - b2))
    s["params"].sub_(lr * ((s["m"] * c1) / ((s["v"] * c2).sqrt() + eps) + wd * s["params"]))
    s["params_bf16"].copy_(s["params"])
    return {k: s[k] for k in ("norm", "params", "params_bf16", "m", "v")}


# -------------------------------------------------- the framework's calls
def _llmk():
    if "llmk" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.cpp_b200"))
    import llmk
    return llmk


def _workspace(s, nbytes):
    """The scratch memory that a program keeps from its first step on."""
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _own_policy(s):
    llmk, case = _llmk(), s["case"]
    ws = s.get("workspace")
    if ws is None:
        ws = _workspace(s, llmk.policy_loss_workspace(s["logits"].shape[0], case["ld"]))
    llmk.policy_loss(s["losses"], s["logits"], s["targets"], s["advantages"], V=case["V"], weights=s["weights"],
                     old_logps=s["old"], ref_logps=s["ref"], kls=s["kls"], logps=s["logps"], dlogits=s["dlogits"],
                     clip_low=_CLIP, clip_high=_CLIP, kl_coef=case["kl"], dscale=1.0, workspace=ws)
    return {k: s[k] for k in ("losses", "kls", "logps", "dlogits") if s[k] is not None}


def _own_preference(s):
    llmk, case = _llmk(), s["case"]
    ws = s.get("workspace")
    if ws is None:
        ws = _workspace(s, llmk.preference_loss_workspace(case["B"], case["T"], case["ld"]))
    llmk.preference_loss(s["losses"], s["logits"], s["targets"], V=case["V"], weights=s["weights"], ref_logps=s["ref"],
                         rewards=s["rewards"], dlogits=s["dlogits"], beta=_BETA, label_smoothing=case["smooth"],
                         dscale=1.0 / case["B"], workspace=ws)
    return {k: s[k] for k in ("losses", "rewards", "dlogits") if s[k] is not None}


def _own_clip(s):
    llmk = _llmk()
    if "tensors" not in s:
        sizes = _tensor_sizes(s["case"])
        s["tensors"] = llmk.TensorList(s["grads"].split(sizes), s["out"].split(sizes))
    ws = s.get("workspace")
    if ws is None:
        ws = _workspace(s, llmk.grad_norm_workspace(s["tensors"]))
    llmk.clip_grad_norm(s["norm"], s["tensors"], _MAX_NORM, workspace=ws)
    return {"norm": s["norm"], "out": s["out"]}


def _own_adamw(s):
    llmk = _llmk()
    if "tensors" not in s:
        s["tensors"] = llmk.TensorList([s["grads"]])
    ws = s.get("workspace")
    if ws is None:
        ws = _workspace(s, llmk.grad_norm_workspace(s["tensors"]))
    llmk.grad_norm(s["norm"], s["tensors"], workspace=ws)
    llmk.adamw_clipped(s["params"], s["grads"], s["m"], s["v"], s["hparams"], s["norm"], _MAX_NORM,
                       params_bf16=s["params_bf16"])
    return {k: s[k] for k in ("norm", "params", "params_bf16", "m", "v")}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"policy": _own_policy, "preference": _own_preference, "clip": _own_clip, "adamw": _own_adamw}[op](state)
    return {"policy": _plain_policy, "preference": _plain_preference, "clip": _plain_clip, "adamw": _plain_adamw}[op](state)


# ------------------------------------------------- the definitions in 64 bits
def _chunk(logits, r, n, V):
    return logits[r:r + n, :V].double().requires_grad_(True)


def _exact_gradient(s, coefficients, live, V):
    """The gradient of sum(coefficients * logp(target)) over the live rows, by differentiation."""
    logits, t = s["logits"], s["targets"].long()
    out = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    for r in range(0, logits.shape[0], 1024):
        x = _chunk(logits, r, 1024, V)
        lp = torch.log_softmax(x, -1).gather(-1, t[r:r + 1024, None])[:, 0]
        keep = live[r:r + 1024]
        (lp[keep] * coefficients[r:r + 1024][keep]).sum().backward()
        out[r:r + 1024, :V] = x.grad
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("policy", "preference"):
        V, t, w = case["V"], s["targets"].long(), s["weights"].double()
        live = w != 0
        lp = torch.cat([torch.log_softmax(_chunk(s["logits"], r, 1024, V).detach(), -1).gather(-1, t[r:r + 1024, None])[:, 0]
                        for r in range(0, t.numel(), 1024)]).requires_grad_(True)
        if op == "policy":
            A = s["advantages"].double()
            ratio = torch.exp(lp - s["old"].double())
            gain = torch.minimum(ratio * A, torch.clamp(ratio, 1 - _CLIP, 1 + _CLIP) * A)
            loss, out = -gain, {}
            if case["kl"]:
                d = s["ref"].double() - lp
                kl = torch.exp(d) - 1 - d
                loss = loss + case["kl"] * kl
                out["kls"] = torch.where(live, kl, 0.0).detach()
            losses = torch.where(live, loss * w, 0.0)
            out |= {"losses": losses.detach(), "logps": torch.where(live, lp, 0.0).detach()}
            total = losses.sum()
        else:
            B = case["B"]
            score = _BETA * (torch.where(live, lp * w, 0.0).reshape(2 * B, -1).sum(-1) - s["ref"].double())
            h = score[:B] - score[B:]
            losses = -(1 - case["smooth"]) * torch.nn.functional.logsigmoid(h) - case["smooth"] * torch.nn.functional.logsigmoid(-h)
            out = {"losses": losses.detach(), "rewards": score.detach()}
            total = losses.mean()
        if case["grad"]:
            (c,) = torch.autograd.grad(total, lp)
            out["dlogits"] = _exact_gradient(s, c, live, V)
        return out
    g = s["grads"].double()
    norm = torch.linalg.vector_norm(g)
    k = min(1.0, _MAX_NORM / (float(norm) + 1e-6))
    if op == "clip":
        return {"norm": norm.reshape(1), "out": g * k}
    lr, b1, b2, eps, wd, c1, c2, scale = s["hparams"].double().tolist()
    g = g * (scale * k)
    m = b1 * s["m"].double() + (1 - b1) * g
    v = b2 * s["v"].double() + (1 - b2) * g * g
    p = s["params"].double()
    p = p - lr * (m * c1 / (torch.sqrt(v * c2) + eps) + wd * p)
    return {"norm": norm.reshape(1), "params": p, "params_bf16": p, "m": m, "v": v}
