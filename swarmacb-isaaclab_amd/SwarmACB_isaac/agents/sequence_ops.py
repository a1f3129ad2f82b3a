"""Operators of sequence policies: a gated linear recurrence, the norm of a residual stream, and the
clipped policy loss with a KL term over any number of choices.

They stand beside what the trainers run (the LSTM memory of ``poca_networks.lstm_sequence``, its
LayerNorms, ``categorical_terms`` and ``trust_region_policy_loss`` of the update) for memories wider than
64 units, sequences of any length, action spaces of more than 64 choices, and bfloat16 / float16 as well
as float32:

``gated_recurrence``         h, c over whole sequences, with gradients
``gated_recurrence_step``    one decision of the same memory (rollouts; no autograd)
``residual_rms_norm``        the residual sum and its root-mean-square norm, with gradients
``categorical_policy_loss``  clipped ratio + KL to a reference + entropy bonus, from logits, with its gradient
``categorical_log_probs``    log-probability of the action and entropy per row (rollouts; no autograd)

On the GPU every call runs the HIP kernels of include/swarmseq.h (through csrc/swarm_torch.cpp, which holds the
backward passes) on the current stream of the tensors' device, captures into graphs, and waits for nothing;
what the kernels do not take raises ValueError, dual tensors of forward-mode differentiation included; differentiating
twice and torch.jit.trace raise RuntimeError. On the CPU the same functions run torch operations (float64 too).
"""

from __future__ import annotations

import torch

from .. import _native
from ._trainer import _BAD_ACTIONS, _bad_action_flag, _flag_key, check_policy_inputs

__all__ = ["gated_recurrence", "gated_recurrence_step", "residual_rms_norm", "categorical_policy_loss",
           "categorical_log_probs", "check_policy_inputs"]

_GPU_TYPES = (torch.float32, torch.bfloat16, torch.float16)   # swarm_dtype_t
RATIO_BOUND = 20.0     # log-ratios are held inside +- this, as in the learned-option trainer's policy loss


def _flat(t: torch.Tensor, n: int) -> torch.Tensor:
    """t as n contiguous values."""
    return (t if t.dim() == 1 else t.reshape(n)).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension contiguous (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _float_type(t: torch.Tensor, what: str):
    if t.is_cuda:
        if t.dtype not in _GPU_TYPES:
            raise ValueError(f"{what}: float32, bfloat16 or float16 is needed on the GPU, got {t.dtype}")
    elif not t.is_floating_point():
        raise ValueError(f"{what}: a floating type is needed, got {t.dtype}")


def _like(t, ref: torch.Tensor, shape, dtypes, what: str):
    """Checks an optional operand against the main one."""
    if t is None:
        return
    if not torch.is_tensor(t):
        raise ValueError(f"{what}: a tensor is needed, got {type(t).__name__}")
    if t.device != ref.device:
        raise ValueError(f"{what} is on {t.device}, not on {ref.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: shape {tuple(shape)} is needed, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what}: {' or '.join(str(d) for d in dtypes)} is needed, got {t.dtype}")


def _no_grad_operand(t, what: str):
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} takes no gradient: detach it")


# -------------------------------------------------------------------------------- gated recurrence

def gated_recurrence(gates: torch.Tensor, state: torch.Tensor | None = None, keep: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None):
    """(h, last state) of a gated linear recurrence over n sequences of T steps.

    gates (n, T, 3U) are the pre-activations of a step's forget, candidate and output blocks, in this order
    (one linear layer of the input); with f, o their sigmoids and z the candidate itself,

        c_t = f_t p_t + (1 - f_t) z_t        p_t = keep_{t-1} c_{t-1},  p_0 = state
        h_t = o_t c_t

    state (n, U) float32 (None: zeros); keep (n, T) float32 within [-1, 1] or bool multiplies the state after step
    t before step t + 1, as in ``lstm_sequence`` (0 where the episode ended); lengths (n,) int64 or int32: steps from
    lengths[i] on are padding, where the state stands still, h is 0, no gradient flows, and the inputs'
    values are not used. Returns h (n, T, U) in the gates' type and the state (n, U) behind the last step in
    float32. Gradients flow to gates and state."""
    if not torch.is_tensor(gates) or gates.dim() != 3 or gates.shape[2] % 3 or gates.shape[2] == 0:
        raise ValueError("gated_recurrence: gates (n, T, 3 units) are needed")
    _float_type(gates, "gated_recurrence: gates")
    n, T, U = gates.shape[0], gates.shape[1], gates.shape[2] // 3
    state_types = (torch.float32,) if gates.is_cuda else (torch.float32, torch.float64)
    _like(state, gates, (n, U), state_types, "gated_recurrence: state")
    _like(keep, gates, (n, T), (torch.float32, torch.bool) + (() if gates.is_cuda else (torch.float64,)),
          "gated_recurrence: keep")
    _like(lengths, gates, (n,), (torch.int64, torch.int32), "gated_recurrence: lengths")
    _no_grad_operand(keep, "gated_recurrence: keep")
    if not gates.is_cuda:
        return _plain_scan(gates, state, keep, lengths)
    if n == 0 or T == 0:
        h = gates[..., :U] * 0
        last = gates.new_zeros(n, U, dtype=torch.float32) if state is None else state.clone()
        return h, last
    if keep is not None:
        keep = keep.to(torch.float32).contiguous()
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    if state is not None:
        state = state.contiguous()
    return _native.seq_ops().gated_scan(_rows(gates), state, keep, lengths)


def _plain_scan(gates, state, keep, lengths):
    dtype, (n, T, U3) = gates.dtype, gates.shape
    U = U3 // 3
    acc = torch.promote_types(gates.dtype, torch.float32)
    gates, before = gates.to(acc), None if keep is None else keep[:, :-1].to(acc)
    live = None
    if lengths is not None:
        # what the padding holds goes before any arithmetic: a selection behind it leaves 0 NaN = NaN to the gradients
        live = torch.arange(T, device=gates.device)[None] < lengths[:, None]
        gates = gates.masked_fill(~live[..., None], 0.0)
        before = None if before is None else before.masked_fill(~live[:, 1:], 1.0)
    xf, z, xo = gates.split(U, dim=2)
    f, g, o = torch.sigmoid(xf), torch.sigmoid(-xf), torch.sigmoid(xo)
    c = torch.zeros(n, U, dtype=acc, device=gates.device) if state is None else state.to(acc)
    hs = []
    for t in range(T):
        p = c if before is None or t == 0 else c * before[:, t - 1, None]
        now = f[:, t] * p + g[:, t] * z[:, t]
        h = o[:, t] * now
        if live is not None:
            on = live[:, t, None]
            now, h = torch.where(on, now, c), torch.where(on, h, torch.zeros_like(h))
        c = now
        hs.append(h)
    h = torch.stack(hs, dim=1) if hs else xf * 0
    return h.to(dtype), (c.clone() if c is state else c)


def gated_recurrence_step(gates: torch.Tensor, state: torch.Tensor, keep: torch.Tensor | None = None,
                          inplace: bool = False):
    """One step of ``gated_recurrence`` for rollouts: gates (rows, 3U), state (rows, U) float32, keep (rows,)
    float32 or bool multiplies the state before the step (0 starts a new episode). Returns h (rows, U) in the
    gates' type and the new state, written over `state` if inplace. No autograd: a training pass runs
    ``gated_recurrence``."""
    if not torch.is_tensor(gates) or gates.dim() != 2 or gates.shape[1] % 3 or gates.shape[1] == 0:
        raise ValueError("gated_recurrence_step: gates (rows, 3 units) are needed")
    _float_type(gates, "gated_recurrence_step: gates")
    rows, U = gates.shape[0], gates.shape[1] // 3
    if state is None:
        raise ValueError("gated_recurrence_step: a state (rows, units) is needed")
    _like(state, gates, (rows, U), (torch.float32,) + (() if gates.is_cuda else (torch.float64,)),
          "gated_recurrence_step: state")
    _like(keep, gates, (rows,), (torch.float32, torch.bool) + (() if gates.is_cuda else (torch.float64,)),
          "gated_recurrence_step: keep")
    if torch.is_grad_enabled() and (gates.requires_grad or state.requires_grad):
        raise ValueError("gated_recurrence_step has no gradient: use gated_recurrence, or torch.no_grad()")
    if inplace and not state.is_contiguous():
        raise ValueError("gated_recurrence_step: a state that is written in place has to be contiguous")
    if not gates.is_cuda:
        acc = torch.promote_types(gates.dtype, torch.float32)
        xf, z, xo = gates.to(acc).split(U, dim=1)
        p = state.to(acc) if keep is None else state.to(acc) * keep[:, None].to(acc)
        now = torch.sigmoid(xf) * p + torch.sigmoid(-xf) * z
        h = (torch.sigmoid(xo) * now).to(gates.dtype)
        return h, (state.copy_(now) if inplace else now.to(state.dtype))
    gates = _rows(gates)
    state = state.contiguous()
    if keep is not None:
        keep = keep.to(torch.float32).contiguous()
    return _native.seq_ops().gated_step(gates, state, keep, inplace)


# ------------------------------------------------------------------------------- residual RMS norm

def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                      eps: float = 1e-6):
    """(y, stream): stream = x + residual and y = stream / sqrt(mean(stream^2) + eps) * weight over the last
    dimension; without a residual the stream is x. x and residual (..., D) and weight (D,) share one type;
    the sum, its norm and y are formed in float32 and rounded once each (y, and the gradients, from the sum
    before its rounding). Gradients flow to all three."""
    if not torch.is_tensor(x) or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("residual_rms_norm: x (..., D) with D >= 1 is needed")
    _float_type(x, "residual_rms_norm: x")
    _like(residual, x, x.shape, (x.dtype,), "residual_rms_norm: residual")
    _like(weight, x, (x.shape[-1],), (x.dtype,), "residual_rms_norm: weight")
    if not eps >= 0.0:
        raise ValueError(f"residual_rms_norm: eps >= 0 is needed, got {eps}")
    if not x.is_cuda:
        acc = torch.promote_types(x.dtype, torch.float32)
        s = x.to(acc) if residual is None else x.to(acc) + residual.to(acc)
        y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)
        y = y if weight is None else y * weight.to(acc)
        return y.to(x.dtype), (x if residual is None else s.to(x.dtype))
    D = x.shape[-1]
    rows = x.numel() // D
    flat = x.dim() == 2
    x2 = _rows(x if flat else x.reshape(rows, D))
    r2 = None if residual is None else _rows(residual if flat else residual.reshape(rows, D))
    w = None if weight is None else weight.contiguous()
    y, stream = _native.seq_ops().residual_norm(x2, r2, w, float(eps))
    if residual is None:
        return (y if flat else y.view(x.shape)), x
    return (y, stream) if flat else (y.view(x.shape), stream.view(x.shape))


# ------------------------------------------------------------------------------------- policy loss

def _flag(device, what: str) -> torch.Tensor:
    """The device's input-check word. A graph must not be what allocates and clears it."""
    if _flag_key(device) not in _BAD_ACTIONS and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: run a policy operator on {device} once before capturing one")
    return _bad_action_flag(device)


def _logit_rows(logits, actions, what: str):
    if not torch.is_tensor(logits) or logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits (..., K) with K >= 1 are needed")
    _float_type(logits, f"{what}: logits")
    _like(actions, logits, logits.shape[:-1], (torch.int64, torch.int32), f"{what}: actions")
    if actions is None:
        raise ValueError(f"{what}: actions are needed")
    K = logits.shape[-1]
    M = logits.numel() // K
    return _rows(logits if logits.dim() == 2 else logits.reshape(M, K)), _flat(actions.to(torch.int64), M), M, K


def categorical_log_probs(logits: torch.Tensor, actions: torch.Tensor):
    """(log-probability of the taken action, entropy) of Categorical(logits) per row, both float32 in the
    shape of actions: logits (..., K), actions (...) int64 or int32. A logit of -inf is a choice that cannot
    be taken. For rollouts and references: no autograd (``categorical_policy_loss`` has the gradient). On the
    GPU an action outside [0, K) gives NaN and raises at the next ``check_policy_inputs``."""
    z, a, M, K = _logit_rows(logits, actions, "categorical_log_probs")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("categorical_log_probs has no gradient: detach the logits, or use torch.no_grad()")
    if not z.is_cuda:
        lp, ent = _plain_log_probs(z, a)
        return lp.reshape(actions.shape), ent.reshape(actions.shape)
    lp, ent = _native.seq_ops().log_probs(z, a, _flag(z.device, "categorical_log_probs"))
    return lp.view(actions.shape), ent.view(actions.shape)


def _plain_log_probs(z, a):
    log_p = torch.log_softmax(z.to(torch.promote_types(z.dtype, torch.float32)), dim=-1)
    p = log_p.exp()
    ent = -(p * log_p.masked_fill(log_p == -torch.inf, 0.0)).sum(-1)
    return log_p.gather(1, a[:, None]).squeeze(1), ent


def categorical_policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_log_probs: torch.Tensor,
                            advantages: torch.Tensor, *, clip=0.2, ref_log_probs: torch.Tensor | None = None,
                            kl_coef: float = 0.0, entropy_coef: float = 0.0, mask: torch.Tensor | None = None,
                            denom: torch.Tensor | None = None):
    """(loss, terms) of the clipped policy objective over rows of logits (..., K), with l the log-probability
    of the row's action (int64 or int32) under softmax(logits) and r = exp(l - old_log_probs):

        pg   = -min(r adv, clamp(r, 1 - clip, 1 + clip) adv)      clip: a number, or (below, above)
        kl   = exp(d) - d - 1,  d = ref_log_probs - l             (0 without a reference)
        loss = sum over active rows of (pg + kl_coef kl - entropy_coef H) / denom

    terms (4,): the means of pg, kl, the entropy H and the clipped share, without gradient. mask (...) bool:
    inactive rows are not looked at (whatever they hold) and get a zero gradient; denom: a float32 scalar
    tensor (the global count of a multi-GPU update), else the number of active rows, at least 1. The
    log-ratios are held inside +-20, without gradient beyond. float32 per-row operands in the rows' shape.
    On the GPU an active row's action outside [0, K) makes the loss NaN and raises at the next
    ``check_policy_inputs``. Gradients flow to the logits alone."""
    what = "categorical_policy_loss"
    z, a, M, K = _logit_rows(logits, actions, what)
    shape = logits.shape[:-1]
    per_row = (torch.float32,) if z.is_cuda else (torch.float32, torch.float64)
    for t, name in ((old_log_probs, "old_log_probs"), (advantages, "advantages"), (ref_log_probs, "ref_log_probs")):
        if t is None and name != "ref_log_probs":
            raise ValueError(f"{what}: {name} are needed")
        _like(t, z, shape, per_row, f"{what}: {name}")
        _no_grad_operand(t, f"{what}: {name}")
    _like(mask, z, shape, (torch.bool,), f"{what}: mask")
    if denom is not None:
        _like(denom, z, denom.shape if torch.is_tensor(denom) and denom.numel() == 1 else (), per_row, f"{what}: denom")
        _no_grad_operand(denom, f"{what}: denom")
    below, above = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    lo, hi = 1.0 - float(below), 1.0 + float(above)
    if not lo <= hi:
        raise ValueError(f"{what}: clip {clip} leaves no interval")
    if kl_coef != 0.0 and ref_log_probs is None:
        raise ValueError(f"{what}: kl_coef needs ref_log_probs")
    old, adv = _flat(old_log_probs, M), _flat(advantages, M)
    ref = None if ref_log_probs is None else _flat(ref_log_probs, M)
    active = None if mask is None else _flat(mask, M)
    d = None if denom is None else denom.reshape(()).contiguous()
    if not z.is_cuda:
        return _plain_policy_loss(z, a, old, adv, ref, active, d, lo, hi, float(kl_coef), float(entropy_coef))
    return _native.seq_ops().policy_loss(z, a, old, adv, ref, active, d, lo, hi, float(kl_coef), float(entropy_coef),
                                         _flag(z.device, what))


def _plain_kl(d):
    """exp(d) - d - 1: by its series where d is small and the difference would cancel (float64 needs 16 terms)."""
    series = torch.ones_like(d)
    for k in range(18, 2, -1):
        series = 1.0 + d / k * series
    return torch.where(d.abs() < 0.5, 0.5 * d * d * series, torch.expm1(d) - d)


def _plain_policy_loss(z, a, old, adv, ref, active, denom, lo, hi, kl_coef, entropy_coef):
    if active is not None:
        z, a, old, adv = z[active], a[active], old[active], adv[active]
        ref = None if ref is None else ref[active]
    lp, ent = _plain_log_probs(z, a)
    n = denom if denom is not None else max(1, z.shape[0])
    r = (lp - old).clamp(-RATIO_BOUND, RATIO_BOUND).exp()
    pg = -torch.min(r * adv, r.clamp(lo, hi) * adv)
    if ref is None:
        kl = torch.zeros_like(pg)
    else:
        kl = _plain_kl((ref - lp).clamp(-RATIO_BOUND, RATIO_BOUND))
    outside = ((r < lo) | (r > hi)).to(pg.dtype)
    terms = torch.stack([v.sum() / n for v in (pg, kl, ent, outside)])
    return terms[0] + kl_coef * terms[1] - entropy_coef * terms[2], terms.detach()
