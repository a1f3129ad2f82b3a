"""Measured cases of the sequence-policy operators (SwarmACB_isaac.agents.sequence_ops).

Five calls, each with its plain form in elementary torch operations and its definition in 64 bits:

  recurrence   gated_recurrence and its gradients: a policy memory over whole sequences
  step         gated_recurrence_step: the same memory, one decision at a time
  norm         residual_rms_norm, forward alone or with its gradients
  loss         categorical_policy_loss and its gradient: the clipped policy loss with a KL term, from logits
  log_probs    categorical_log_probs: what a rollout keeps of the policy, from logits

Run from the repository's root.
"""

import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
CLIP = 0.2
KL_COEF = 0.05
ENTROPY_COEF = 0.01


def _ops():
    package = os.path.join(os.getcwd(), "swarmacb-isaaclab_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from SwarmACB_isaac.agents import sequence_ops

    return sequence_ops


# --------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one minibatch of the trainers' updates: 16 sequences of 128 steps, memory_size 128 (64 units), float32,
        # the memory cleared where an episode ends
        {"name": "memory_minibatch", "op": "recurrence", "n": 16, "t": 128, "u": 64, "dtype": "f32", "keep": True,
         "ragged": False},
        # one long recorded episode: few channels for the card, so the length has to be split
        {"name": "one_long_sequence", "op": "recurrence", "n": 1, "t": 32768, "u": 1024, "dtype": "bf16", "keep": False,
         "ragged": False},
        # a large batch of a wide memory, padded to its longest sequence
        {"name": "wide_padded_batch", "op": "recurrence", "n": 64, "t": 1024, "u": 2048, "dtype": "bf16", "keep": True,
         "ragged": True},
        # one environment's 20 robots acting: a call of a few microseconds
        {"name": "one_env_step", "op": "step", "rows": 20, "u": 64, "dtype": "f32"},
        # one decision of 4096 environments with 20 robots each
        {"name": "rollout_step", "op": "step", "rows": 81920, "u": 64, "dtype": "f32"},
        # the residual stream of one environment's robots while acting
        {"name": "one_env_norm", "op": "norm", "rows": 20, "d": 128, "dtype": "f32", "train": False},
        # an odd row count and width in half precision, training
        {"name": "odd_norm", "op": "norm", "rows": 5001, "d": 1001, "dtype": "f16", "train": True},
        # a wide residual stream over many tokens, training
        {"name": "wide_norm", "op": "norm", "rows": 16384, "d": 4096, "dtype": "bf16", "train": True},
        # the dandelion / cyclamen module choice over one minibatch: 2048 rows of 6 logits
        {"name": "module_loss", "op": "loss", "rows": 2048, "k": 6, "dtype": "f32"},
        # a large discrete action space (a vocabulary) with an odd row length
        {"name": "vocabulary_loss", "op": "loss", "rows": 4096, "k": 50001, "dtype": "bf16"},
        # scoring a decision of 4096 environments with 20 robots each: a few choices, many rows
        {"name": "rollout_log_probs", "op": "log_probs", "rows": 81920, "k": 18, "dtype": "f32"},
        # scoring a rollout over a large action space
        {"name": "vocabulary_log_probs", "op": "log_probs", "rows": 8192, "k": 32768, "dtype": "bf16"},
    ]


def _log_uniform(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "step", "norm", "norm", "loss", "loss", "log_probs"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    wide = 2 if dtype == "f32" else 1
    if op == "recurrence":
        n, u = _log_uniform(rng, 1, 256), _log_uniform(rng, 8, 4096)
        t = _log_uniform(rng, 1, max(2, min(65536, 134_000_000 // (n * u * wide))))
        return {"op": op, "n": n, "t": t, "u": u if rng.random() < 0.3 else max(8, u // 8 * 8), "dtype": dtype,
                "keep": rng.random() < 0.5, "ragged": rng.random() < 0.3}
    if op == "step":
        return {"op": op, "rows": _log_uniform(rng, 1, 81920), "u": _log_uniform(rng, 8, 1024), "dtype": dtype}
    if op == "norm":
        d = _log_uniform(rng, 16, 16384)
        d = d if rng.random() < 0.3 else max(16, d // 16 * 16)
        return {"op": op, "rows": _log_uniform(rng, 1, 67_000_000 // (d * wide)), "d": d, "dtype": dtype,
                "train": rng.random() < 0.7}
    k = _log_uniform(rng, 2, 150_000)
    return {"op": op, "rows": _log_uniform(rng, 1, min(200_000, 200_000_000 // (k * wide))), "k": k, "dtype": dtype}


# -------------------------------------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]
    op = case["op"]
    if op == "recurrence":
        n, t, u = case["n"], case["t"], case["u"]
        gates = _normal(g, n, t, 3 * u)
        gates[..., :u] += 2.0                                  # a forget gate's bias: memories of tens of steps
        keep = lengths = None
        if case["keep"]:                                       # episodes that end about every 64 steps
            keep = (torch.rand(n, t, device="cuda", generator=g) > 1.0 / 64).float()
        if case["ragged"]:                                     # sequences of half the padded length and more
            lengths = torch.randint((t + 1) // 2, t + 1, (n,), device="cuda", generator=g)
        return {"case": dict(case), "gates": gates.to(dtype), "state": _normal(g, n, u), "keep": keep,
                "lengths": lengths, "d_h": _normal(g, n, t, u).to(dtype), "d_state": _normal(g, n, u)}
    if op == "step":
        rows, u = case["rows"], case["u"]
        gates = _normal(g, rows, 3 * u)
        gates[:, :u] += 2.0
        return {"case": dict(case), "gates": gates.to(dtype), "state": _normal(g, rows, u)}
    if op == "norm":
        rows, d = case["rows"], case["d"]
        return {"case": dict(case), "x": _normal(g, rows, d).to(dtype), "residual": (2.0 * _normal(g, rows, d)).to(dtype),
                "weight": (1.0 + 0.2 * _normal(g, d)).to(dtype), "d_y": _normal(g, rows, d).to(dtype),
                "d_stream": _normal(g, rows, d).to(dtype)}
    rows, k = case["rows"], case["k"]
    logits = (2.0 * _normal(g, rows, k)).to(dtype)
    actions = torch.randint(0, k, (rows,), device="cuda", generator=g)
    if op == "log_probs":
        return {"case": dict(case), "logits": logits, "actions": actions}
    now = (logits.gather(1, actions[:, None]).squeeze(1).float() - torch.logsumexp(logits.float(), 1)).double()
    shift = 0.15 * _normal(g, rows).double()                   # log(new / old) of one policy update
    # the loss has a kink where the ratio meets 1 - CLIP and 1 + CLIP: no row sits on it, as none does in earnest
    for border in (math.log(1 - CLIP), math.log(1 + CLIP)):
        shift = torch.where((shift - border).abs() < 0.01, border + 0.02 * torch.sign(shift - border + 1e-9), shift)
    return {"case": dict(case), "logits": logits, "actions": actions, "old": (now - shift).float(),
            "ref": (now + 0.3 * _normal(g, rows).double()).float(), "advantages": _normal(g, rows),
            "mask": torch.rand(rows, device="cuda", generator=g) < 0.9,
            # half precision trains with a scaled loss
            "d_loss": torch.tensor(float(rows * min(k, 2048) if case["dtype"] == "f16" else 1), device="cuda")}


# ---------------------------------------------------------------------------------------------- runs

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    ops = _ops()
    op = s["case"]["op"]
    if op == "recurrence":
        gates, state = s["gates"].detach().requires_grad_(), s["state"].detach().requires_grad_()
        h, last = ops.gated_recurrence(gates, state, keep=s["keep"], lengths=s["lengths"])
        d_gates, d_state = torch.autograd.grad((h, last), (gates, state), (s["d_h"], s["d_state"]))
        return {"h": h.detach(), "last": last.detach(), "d_gates": d_gates, "d_state": d_state}
    if op == "step":
        h, state = ops.gated_recurrence_step(s["gates"], s["state"])
        return {"h": h, "state": state}
    if op == "norm":
        if not s["case"]["train"]:
            y, stream = ops.residual_rms_norm(s["x"], s["residual"], s["weight"], eps=EPS)
            return {"y": y, "stream": stream}
        x, residual, weight = (s[k].detach().requires_grad_() for k in ("x", "residual", "weight"))
        y, stream = ops.residual_rms_norm(x, residual, weight, eps=EPS)
        dx, dr, dw = torch.autograd.grad((y, stream), (x, residual, weight), (s["d_y"], s["d_stream"]))
        return {"y": y.detach(), "stream": stream.detach(), "dx": dx, "dr": dr, "dw": dw}
    if op == "log_probs":
        log_probs, entropy = ops.categorical_log_probs(s["logits"], s["actions"])
        return {"log_probs": log_probs, "entropy": entropy}
    logits = s["logits"].detach().requires_grad_()
    loss, terms = ops.categorical_policy_loss(logits, s["actions"], s["old"], s["advantages"], clip=CLIP,
                                              ref_log_probs=s["ref"], kl_coef=KL_COEF, entropy_coef=ENTROPY_COEF,
                                              mask=s["mask"])
    (d_logits,) = torch.autograd.grad(loss, logits, s["d_loss"])
    return {"loss": loss.detach(), "terms": terms, "d_logits": d_logits}


def _scan(a, b):
    """x_t = a_t x_{t-1} + b_t over dimension 1 (x_{-1} = 0), by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_recurrence(s):
    u = s["case"]["u"]
    dtype = s["gates"].dtype
    gates = s["gates"].float()
    n, t = gates.shape[:2]
    f = 1 / (1 + torch.exp(-gates[..., :u]))
    g = 1 / (1 + torch.exp(gates[..., :u]))                    # 1 - f
    z = gates[..., u:2 * u]
    o = 1 / (1 + torch.exp(-gates[..., 2 * u:]))
    a, b, d_h = f, g * z, s["d_h"].float()
    before = torch.ones(n, t, 1, device=f.device)              # what the state is multiplied by before step t
    if s["keep"] is not None:
        before[:, 1:] = s["keep"][:, :-1, None]
    a = f * before
    if s["lengths"] is not None:                               # the state stands still behind a sequence's end
        live = torch.arange(t, device=f.device) < s["lengths"][:, None]
        live = live[:, :, None]
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
        o, d_h = torch.where(live, o, 0.0), torch.where(live, d_h, 0.0)
    start = s["state"][:, None]
    c = _scan(a, torch.cat([b[:, :1] + a[:, :1] * start, b[:, 1:]], 1))
    p = torch.cat([start, c[:, :-1]], 1) * before
    back = (o * d_h).flip(1)
    back = torch.cat([back[:, :1] + s["d_state"][:, None], back[:, 1:]], 1)
    ahead = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    d_c = _scan(ahead, back).flip(1)
    d_gates = torch.cat([d_c * (p - z) * f * g, d_c * g, d_h * c * o * (1 - o)], 2)
    if s["lengths"] is not None:
        d_gates = torch.where(live, d_gates, 0.0)
    return {"h": (o * c).to(dtype), "last": c[:, -1], "d_gates": d_gates.to(dtype), "d_state": d_c[:, 0] * a[:, 0]}


def _plain_norm(s):
    dtype = s["x"].dtype
    x, w = s["x"].float() + s["residual"].float(), s["weight"].float()
    inv = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    out = {"y": (x * inv * w).to(dtype), "stream": x.to(dtype)}
    if s["case"]["train"]:
        dy = s["d_y"].float()
        dn, n = dy * w, x * inv
        dx = (inv * (dn - n * (dn * n).mean(1, keepdim=True)) + s["d_stream"].float()).to(dtype)
        out.update(dx=dx, dr=dx, dw=(dy * n).sum(0).to(dtype))
    return out


def _plain_rows(logits, actions):
    """(probabilities, log-probabilities, entropy of each row, log-probability of each action), in 32 bits."""
    z = logits.float()
    z = z - z.max(1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_p = z - torch.log(total)
    p = e / total
    return p, log_p, -(p * log_p).sum(1), log_p.gather(1, actions[:, None]).squeeze(1)


def _plain_loss(s):
    p, log_p, entropy, now = _plain_rows(s["logits"], s["actions"])
    live = s["mask"].float()
    denom = live.sum().clamp(min=1.0)
    adv = s["advantages"]
    ratio = torch.exp((now - s["old"]).clamp(-20, 20))
    plain, clipped = ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv
    policy = -torch.minimum(plain, clipped)
    delta = (s["ref"] - now).clamp(-20, 20)
    kl = torch.exp(delta) - delta - 1
    outside = ((ratio < 1 - CLIP) | (ratio > 1 + CLIP)).float()
    terms = torch.stack([(v * live).sum() / denom for v in (policy, kl, entropy, outside)])
    loss = terms[0] + KL_COEF * terms[1] - ENTROPY_COEF * terms[2]
    d_now = torch.where(plain <= clipped, -plain, 0.0) + KL_COEF * (1 - torch.exp(delta))
    scale = (live * s["d_loss"] / denom)[:, None]
    picked = torch.arange(p.shape[1], device=p.device) == s["actions"][:, None]
    d = scale * (d_now[:, None] * (picked.float() - p) + ENTROPY_COEF * p * (log_p + entropy[:, None]))
    return {"loss": loss, "terms": terms, "d_logits": d.to(s["logits"].dtype)}


def _run_plain(s):
    op = s["case"]["op"]
    if op == "recurrence":
        return _plain_recurrence(s)
    if op == "step":
        u = s["case"]["u"]
        gates = s["gates"].float()
        f = 1 / (1 + torch.exp(-gates[:, :u]))
        state = f * s["state"] + (1 - f) * gates[:, u:2 * u]
        return {"h": (state / (1 + torch.exp(-gates[:, 2 * u:]))).to(s["gates"].dtype), "state": state}
    if op == "norm":
        return _plain_norm(s)
    if op == "log_probs":
        _, _, entropy, now = _plain_rows(s["logits"], s["actions"])
        return {"log_probs": now, "entropy": entropy}
    return _plain_loss(s)


# ------------------------------------------------------------------------------------- work and truth

def work(case):
    op = case["op"]
    e = 4 if case["dtype"] == "f32" else 2
    if op == "recurrence":
        n, t, u = case["n"], case["t"], case["u"]
        read = 0.75 if case["ragged"] else 1.0                 # nothing behind a sequence's end has to be read
        size = n * t * u
        return {"bytes": e * size * (4 + 4 * read) + 16 * n * u + (4 * n * t if case["keep"] else 0), "flops": 35 * size}
    if op == "step":
        size = case["rows"] * case["u"]
        return {"bytes": (4 * e + 8) * size, "flops": 12 * size}
    if op == "norm":
        size = case["rows"] * case["d"]
        if not case["train"]:
            return {"bytes": e * (4 * size + case["d"]), "flops": 5 * size}
        return {"bytes": e * (7 * size + 2 * case["d"]), "flops": 15 * size}
    size = case["rows"] * case["k"]
    if op == "log_probs":
        return {"bytes": e * size + 16 * case["rows"], "flops": 6 * size}
    return {"bytes": 1.9 * e * size + 21 * case["rows"], "flops": 15 * size}   # a tenth of the rows is masked out


def _exact_recurrence(s):
    """Step by step, as the recurrence and the chain rule are written."""
    u = s["case"]["u"]
    gates, d_h = s["gates"].double(), s["d_h"].double()
    n, t = gates.shape[:2]
    f, z, o = torch.sigmoid(gates[..., :u]), gates[..., u:2 * u], torch.sigmoid(gates[..., 2 * u:])
    g = torch.sigmoid(-gates[..., :u])
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((n,), t, device=gates.device)
    live = torch.arange(t, device=gates.device)[None] < lengths[:, None]
    keep = s["keep"].double() if s["keep"] is not None else torch.ones(n, t, dtype=torch.float64, device=gates.device)
    p, c = torch.empty(n, t, u, dtype=torch.float64, device=gates.device), torch.empty_like(f)
    now = s["state"].double()
    gz = g * z
    for i in range(t):
        p[:, i] = now if i == 0 else now * keep[:, i - 1:i]
        now = torch.where(live[:, i:i + 1], f[:, i] * p[:, i] + gz[:, i], now)
        c[:, i] = now
    last = now
    h = torch.where(live[..., None], o * c, 0.0)
    d_gates = torch.zeros_like(gates)
    back = s["d_state"].double()                               # the gradient of the state behind step i
    od = o * d_h
    d_c = torch.zeros_like(c)
    for i in range(t - 1, -1, -1):
        on = live[:, i:i + 1]
        full = back + od[:, i]
        d_c[:, i] = torch.where(on, full, 0.0)
        before = f[:, i] * full if i == 0 else f[:, i] * full * keep[:, i - 1:i]
        back = torch.where(on, before, back)
    d_gates[..., :u] = d_c * (p - z) * f * g
    d_gates[..., u:2 * u] = d_c * g
    d_gates[..., 2 * u:] = torch.where(live[..., None], d_h * c * o * (1 - o), 0.0)
    return {"h": h, "last": last, "d_gates": d_gates, "d_state": back}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "recurrence":
        return _exact_recurrence(s)
    if op == "step":
        f, z, o = s["gates"].double().chunk(3, 1)
        state = torch.sigmoid(f) * s["state"].double() + torch.sigmoid(-f) * z
        return {"h": torch.sigmoid(o) * state, "state": state}
    if op == "norm":
        names = ("x", "residual", "weight")
        x, residual, weight = (s[k].double().requires_grad_() for k in names)
        stream = x + residual
        y = stream * torch.rsqrt(stream.square().mean(-1, keepdim=True) + EPS) * weight
        if not case["train"]:
            return {"y": y.detach(), "stream": stream.detach()}
        dx, dr, dw = torch.autograd.grad((y, stream), (x, residual, weight), (s["d_y"].double(), s["d_stream"].double()))
        return {"y": y.detach(), "stream": stream.detach(), "dx": dx, "dr": dr, "dw": dw}
    logits = s["logits"].double().requires_grad_(op == "loss")
    log_p = torch.log_softmax(logits, 1)
    now = log_p.gather(1, s["actions"][:, None])[:, 0]
    entropy = -(log_p.exp() * log_p).sum(1)
    if op == "log_probs":
        return {"log_probs": now, "entropy": entropy}
    mask, adv = s["mask"], s["advantages"].double()
    count = max(1, int(mask.sum()))
    ratio = (now - s["old"].double()).exp()
    delta = s["ref"].double() - now
    policy = torch.maximum(-ratio * adv, -ratio.clamp(1 - CLIP, 1 + CLIP) * adv)
    outside = ((ratio - 1).abs() > CLIP).double()
    terms = torch.stack([torch.where(mask, v, 0.0).sum() / count for v in (policy, torch.expm1(delta) - delta, entropy, outside)])
    loss = terms[0] + KL_COEF * terms[1] - ENTROPY_COEF * terms[2]
    (d,) = torch.autograd.grad(loss, logits, s["d_loss"].double())
    return {"loss": loss.detach(), "terms": terms.detach(), "d_logits": d}
