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

On the GPU every call runs the HIP kernels of include/swarmseq.h on the current stream of the tensors'
device, captures into graphs, and waits for nothing; what the kernels do not take raises ValueError. On the
CPU the same functions run torch operations (float64 too). The forward outputs are not differentiable twice.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from ._trainer import _bad_action_flag, check_policy_inputs

__all__ = ["gated_recurrence", "gated_recurrence_step", "residual_rms_norm", "categorical_policy_loss",
           "categorical_log_probs", "check_policy_inputs"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # swarm_dtype_t
RATIO_BOUND = 20.0     # log-ratios are held inside +- this, as in the learned-option trainer's policy loss


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    """The current stream of t's device, without building a torch.cuda.Stream (2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _once(backward):
    """once_differentiable for a backward whose gradients are new tensors. Its wrapper costs 9 us a call and is
    only needed where a graph of the gradients is asked for, which is when gradients are recorded in here."""
    wrapped = once_differentiable(backward)

    def run(ctx, *grads):
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def _flat(t: torch.Tensor, n: int) -> torch.Tensor:
    """t as n contiguous values."""
    return (t if t.dim() == 1 else t.reshape(n)).contiguous()


def _check(rc: int, what: str):
    if rc != 0:
        _native.check(rc, what)


def _work(words: int, device):
    """A call's own workspace of that many floats, None for none."""
    return torch.empty(words, dtype=torch.float32, device=device) if words > 0 else None


class _on:
    """torch.cuda.device(t.device) that costs nothing when it is the current device already."""

    __slots__ = ("guard",)

    def __init__(self, t: torch.Tensor):
        self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension contiguous (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _float_type(t: torch.Tensor, what: str):
    if t.is_cuda:
        if t.dtype not in _DTYPES:
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

def _scan_forward(gates, state, keep, lengths, save: bool):
    """(h, last state, tile states or None)"""
    n, T, U3 = gates.shape
    U = U3 // 3
    lib = _native.load()
    with _on(gates):
        h = torch.empty(n, T, U, dtype=gates.dtype, device=gates.device)
        last = torch.empty(n, U, dtype=torch.float32, device=gates.device)
        tiles = (torch.empty(n, _native.gated_tiles(T), U, dtype=torch.float32, device=gates.device)
                 if save else None)
        work = _work(lib.swarm_gated_scan_workspace(n, T, U), gates.device)
        _check(lib.swarm_gated_scan_forward(_DTYPES[gates.dtype], n, T, U, _p(gates), gates.stride(0), gates.stride(1),
                                            _p(state), _p(keep), _p(lengths), _p(h), _p(last), _p(tiles), _p(work),
                                            _stream(gates)), "swarm_gated_scan_forward")
    return h, last, tiles


class _GatedScan(torch.autograd.Function):
    """swarm_gated_scan_forward / _backward. The backward forms the states again from one saved state per
    tile of steps, so nothing of the size of the sequence is kept but the inputs."""

    @staticmethod
    def forward(ctx, gates, state, keep, lengths):
        h, last, tiles = _scan_forward(gates, state, keep, lengths, True)
        ctx.save_for_backward(gates, keep, lengths, tiles)
        ctx.has_state = state is not None
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @_once
    def backward(ctx, d_h, d_last):
        gates, keep, lengths, tiles = ctx.saved_tensors
        n, T, U3 = gates.shape
        U = U3 // 3
        lib = _native.load()
        with _on(gates):
            d_gates = torch.empty(n, T, U3, dtype=gates.dtype, device=gates.device)
            d_state = (torch.empty(n, U, dtype=torch.float32, device=gates.device)
                       if ctx.has_state and ctx.needs_input_grad[1] else None)
            if d_h is not None:
                d_h = _rows(d_h)
            if d_last is not None:
                d_last = d_last.contiguous()
            work = _work(lib.swarm_gated_scan_workspace(n, T, U), gates.device)
            _check(lib.swarm_gated_scan_backward(
                _DTYPES[gates.dtype], n, T, U, _p(gates), gates.stride(0), gates.stride(1), _p(keep), _p(lengths),
                _p(tiles), _p(d_h), d_h.stride(0) if d_h is not None else 0, d_h.stride(1) if d_h is not None else 0,
                _p(d_last), _p(d_gates), _p(d_state), _p(work), _stream(gates)), "swarm_gated_scan_backward")
        return d_gates, d_state, None, None


def gated_recurrence(gates: torch.Tensor, state: torch.Tensor | None = None, keep: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None):
    """(h, last state) of a gated linear recurrence over n sequences of T steps.

    gates (n, T, 3U) are the pre-activations of a step's forget, candidate and output blocks, in this order
    (one linear layer of the input); with f, o their sigmoids and z the candidate itself,

        c_t = f_t p_t + (1 - f_t) z_t        p_t = keep_{t-1} c_{t-1},  p_0 = state
        h_t = o_t c_t

    state (n, U) float32 (None: zeros); keep (n, T) float32 or bool multiplies the state after step t before
    step t + 1, as in ``lstm_sequence`` (0 where the episode ended); lengths (n,) int64 or int32: steps from
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
    gates = _rows(gates)
    if torch.is_grad_enabled() and (gates.requires_grad or (state is not None and state.requires_grad)):
        return _GatedScan.apply(gates, state, keep, lengths)
    return _scan_forward(gates, state, keep, lengths, False)[:2]


def _plain_scan(gates, state, keep, lengths):
    n, T, U3 = gates.shape
    U = U3 // 3
    acc = torch.promote_types(gates.dtype, torch.float32)
    xf, z, xo = gates.to(acc).split(U, dim=2)
    f, g, o = torch.sigmoid(xf), torch.sigmoid(-xf), torch.sigmoid(xo)
    c = torch.zeros(n, U, dtype=acc, device=gates.device) if state is None else state.to(acc)
    hs = []
    for t in range(T):
        p = c if keep is None or t == 0 else c * keep[:, t - 1, None].to(acc)
        now = f[:, t] * p + g[:, t] * z[:, t]
        h = o[:, t] * now
        if lengths is not None:
            live = (t < lengths)[:, None]
            now, h = torch.where(live, now, c), torch.where(live, h, torch.zeros_like(h))
        c = now
        hs.append(h)
    h = torch.stack(hs, dim=1) if hs else xf * 0
    return h.to(gates.dtype), (c.clone() if c is state else c)


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
    with _on(gates):
        h = torch.empty(rows, U, dtype=gates.dtype, device=gates.device)
        out = state if inplace else torch.empty_like(state)
        _check(_native.load().swarm_gated_step(_DTYPES[gates.dtype], rows, U, _p(gates), gates.stride(0), _p(state),
                                               _p(keep), _p(h), _p(out), _stream(gates)), "swarm_gated_step")
    return h, out


# ------------------------------------------------------------------------------- residual RMS norm

def _norm_forward(x, residual, weight, eps: float, save: bool):
    """(y, stream or None, rstd or None)"""
    rows, D = x.shape
    with _on(x):
        y = torch.empty(rows, D, dtype=x.dtype, device=x.device)
        out = torch.empty_like(y) if residual is not None else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if save else None
        _check(_native.load().swarm_residual_norm_forward(
            _DTYPES[x.dtype], rows, D, _p(x), x.stride(0), _p(residual),
            residual.stride(0) if residual is not None else 0, _p(weight), eps, _p(y), _p(out), _p(rstd),
            _stream(x)), "swarm_residual_norm_forward")
    return y, out, rstd


class _ResidualNorm(torch.autograd.Function):
    """swarm_residual_norm_forward / _backward over (rows, D); the saved sum is the stream itself."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps: float):
        y, out, rstd = _norm_forward(x, residual, weight, eps, True)
        ctx.save_for_backward(out if out is not None else x, weight, rstd)
        ctx.two = residual is not None
        ctx.set_materialize_grads(False)
        return (y, out) if out is not None else y

    @staticmethod
    @_once
    def backward(ctx, d_y, d_out=None):
        s, weight, rstd = ctx.saved_tensors
        rows, D = s.shape
        if d_y is None:        # only the stream was used: the sum passes its gradient on
            return d_out, (d_out if ctx.two else None), (torch.zeros_like(weight) if weight is not None else None), None
        lib = _native.load()
        with _on(s):
            d_y = _rows(d_y)
            if d_out is not None:
                d_out = _rows(d_out)
            d_x = torch.empty(rows, D, dtype=s.dtype, device=s.device)
            d_w = work = None
            if weight is not None and ctx.needs_input_grad[2]:
                d_w = torch.empty_like(weight)
                work = _work(lib.swarm_residual_norm_workspace(rows, D), s.device)
            _check(lib.swarm_residual_norm_backward(
                _DTYPES[s.dtype], rows, D, _p(s), s.stride(0), _p(weight), _p(rstd), _p(d_y), d_y.stride(0),
                _p(d_out), d_out.stride(0) if d_out is not None else 0, _p(d_x), _p(d_w), _p(work), _stream(s)),
                "swarm_residual_norm_backward")
        return d_x, (d_x if ctx.two else None), d_w, None


def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                      eps: float = 1e-6):
    """(y, stream): stream = x + residual and y = stream / sqrt(mean(stream^2) + eps) * weight over the last
    dimension; without a residual the stream is x. x and residual (..., D) and weight (D,) share one type;
    the sum, its norm and y are formed in float32 and rounded once each (y from the sum before its
    rounding). Gradients flow to all three; the backward reads the stored stream."""
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
    if torch.is_grad_enabled() and (x2.requires_grad or (r2 is not None and r2.requires_grad)
                                    or (w is not None and w.requires_grad)):
        out = _ResidualNorm.apply(x2, r2, w, float(eps))
        y, stream = (out, None) if residual is None else out
    else:
        y, stream, _ = _norm_forward(x2, r2, w, float(eps), False)
    if residual is None:
        return (y if flat else y.view(x.shape)), x
    return (y, stream) if flat else (y.view(x.shape), stream.view(x.shape))


# ------------------------------------------------------------------------------------- policy loss

def _loss_forward(logits, actions, old, adv, ref, mask_u, denom, lo, hi, kl_coef, entropy_coef, save: bool):
    """(loss, terms, row statistics, denominator, gradient for an incoming gradient of 1 or None)"""
    M, K = logits.shape
    dev = logits.device
    with _on(logits):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        terms = torch.empty(4, dtype=torch.float32, device=dev)
        used = torch.empty((), dtype=torch.float32, device=dev)
        work = torch.empty(_native.POLICY_LOSS_PARTIALS + 4 * M, dtype=torch.float32, device=dev)
        unit = torch.empty(M, K, dtype=logits.dtype, device=dev) if save and logits.dtype != torch.float16 else None
        stats = work.data_ptr() + 4 * _native.POLICY_LOSS_PARTIALS
        _check(_native.load().swarm_policy_loss_forward(
            _DTYPES[logits.dtype], M, K, _p(logits), logits.stride(0), _p(actions), _p(old), _p(ref), _p(adv),
            _p(mask_u), _p(denom), lo, hi, kl_coef, entropy_coef, _p(loss), _p(terms), _p(used), stats, _p(unit),
            _p(work), _p(_bad_action_flag(dev)), _stream(logits)), "swarm_policy_loss_forward")
    return loss, terms, work, used, unit


class _PolicyLossFromLogits(torch.autograd.Function):
    """swarm_policy_loss_forward / _backward. The forward call, which has the logits at hand, forms the gradient
    for an incoming gradient of 1 as well (not in float16, where losses are scaled); the first backward call
    hands it out, written anew if the incoming gradient is another one, and later calls form their own."""

    @staticmethod
    def forward(ctx, logits, actions, old, adv, ref, mask_u, denom, lo, hi, kl_coef, entropy_coef):
        loss, terms, work, used, ctx.unit = _loss_forward(logits, actions, old, adv, ref, mask_u, denom, lo, hi,
                                                          kl_coef, entropy_coef, True)
        ctx.save_for_backward(logits, actions, work, used)
        ctx.entropy_coef = entropy_coef
        ctx.mark_non_differentiable(terms)
        return loss, terms

    @staticmethod
    @_once
    def backward(ctx, g, _terms):
        logits, actions, work, used = ctx.saved_tensors
        M, K = logits.shape
        d, ctx.unit = ctx.unit, None
        with _on(logits):
            have = d is not None
            if not have:
                d = torch.empty(M, K, dtype=logits.dtype, device=logits.device)
            g = g.contiguous()
            _check(_native.load().swarm_policy_loss_backward(
                _DTYPES[logits.dtype], M, K, _p(logits), logits.stride(0), _p(actions), ctx.entropy_coef,
                work.data_ptr() + 4 * _native.POLICY_LOSS_PARTIALS, _p(used), _p(g), have, _p(d), _stream(logits)),
                "swarm_policy_loss_backward")
        return (d,) + (None,) * 10


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
    with _on(z):
        lp = torch.empty(M, dtype=torch.float32, device=z.device)
        ent = torch.empty(M, dtype=torch.float32, device=z.device)
        lib = _native.load()
        work = _work(lib.swarm_log_probs_workspace(M, K), z.device)
        _check(lib.swarm_log_probs(_DTYPES[z.dtype], M, K, _p(z), z.stride(0), _p(a), _p(lp), _p(ent), _p(work),
                                   _p(_bad_action_flag(z.device)), _stream(z)), "swarm_log_probs")
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
    args = (z, a, old, adv, ref, None if active is None else active.view(torch.uint8), d, lo, hi, float(kl_coef),
            float(entropy_coef))
    if torch.is_grad_enabled() and z.requires_grad:
        return _PolicyLossFromLogits.apply(*args)
    return _loss_forward(*args, False)[:2]


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
        d = (ref - lp).clamp(-RATIO_BOUND, RATIO_BOUND)
        kl = d.exp() - d - 1.0
    outside = ((r < lo) | (r > hi)).to(pg.dtype)
    terms = torch.stack([v.sum() / n for v in (pg, kl, ent, outside)])
    return terms[0] + kl_coef * terms[1] - entropy_coef * terms[2], terms.detach()
