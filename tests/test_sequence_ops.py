"""Sequence-policy operators without a GPU: the CPU form against the 64-bit reference, gradients against
differences, every refusal (of the Python entry points and of the C ABI), and the header against the binding."""

import ctypes as C
import os
import re

import pytest
import torch

import sequence_reference as R
from conftest import ROOT
from SwarmACB_isaac import _native
from SwarmACB_isaac.agents import (categorical_log_probs, categorical_policy_loss, gated_recurrence,
                                   gated_recurrence_step, residual_rms_norm)


def _randn(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=dtype)


def _text():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "swarmseq.h")).read(), flags=re.S)


def test_header_and_binding_agree():
    assert sorted(set(re.findall(r"\b(swarm_[a-z0-9_]+)\s*\(", _text()))) == sorted(_native.SEQ_EXPORTS)
    lib = _native.load()
    for name in _native.SEQ_EXPORTS:
        assert hasattr(lib, name), name


def test_header_constants_agree():
    tile = int(re.search(r"#define SWARM_GATED_TILE (\d+)", _text()).group(1))
    partials = re.search(r"#define SWARM_POLICY_LOSS_PARTIALS \((\d+) \* (\d+)\)", _text())
    assert tile == _native.GATED_TILE
    assert int(partials.group(1)) * int(partials.group(2)) == _native.POLICY_LOSS_PARTIALS
    assert _native.gated_tiles(1) == 1 and _native.gated_tiles(tile) == 1 and _native.gated_tiles(tile + 1) == 2


def test_torch_module_binds_the_loaded_library():
    ops = _native.seq_ops()
    assert ops is _native.seq_ops() and ops.GATED_TILE == _native.GATED_TILE
    with pytest.raises(RuntimeError):
        ops.bind("/nowhere/libswarmstep.so")


@pytest.mark.parametrize("n,T,U,with_keep,with_lengths", [(1, 1, 1, False, False), (3, 7, 5, True, False),
                                                          (4, 9, 3, True, True), (2, 6, 4, False, True)])
def test_recurrence_cpu(n, T, U, with_keep, with_lengths):
    gates = _randn(n, T, 3 * U, seed=1).requires_grad_()
    state = _randn(n, U, seed=2).requires_grad_()
    keep = (torch.arange(n * T).view(n, T) % 3 != 1).double() if with_keep else None
    lengths = torch.tensor([0, T, T // 2, 1])[:n] if with_lengths else None
    d_h, d_last = _randn(n, T, U, seed=3), _randn(n, U, seed=4)
    h, last = gated_recurrence(gates, state, keep, lengths)
    grads = torch.autograd.grad((h, last), (gates, state), (d_h, d_last))
    ref = R.recurrence(gates, state, keep, lengths, d_h, d_last)
    for got, name in zip((h, last) + grads, ("h", "last", "d_gates", "d_state")):
        R.check(got, ref[name][0], 1e-13 * (1 + ref[name][0].abs()), name)


def test_recurrence_gradient_by_differences():
    keep = torch.tensor([[1.0, 0.0, 1.0, 1.0], [1.0, 1.0, 1.0, 0.0]], dtype=torch.float64)
    lengths = torch.tensor([4, 3])
    gates, state = _randn(2, 4, 6, seed=5).requires_grad_(), _randn(2, 2, seed=6).requires_grad_()
    assert torch.autograd.gradcheck(lambda g, s: gated_recurrence(g, s, keep, lengths), (gates, state))


def test_recurrence_of_steps():
    gates, state = _randn(3, 5, 12, seed=7), _randn(3, 4, seed=8)
    keep = (torch.arange(15).view(3, 5) % 4 != 2).double()
    h, last = gated_recurrence(gates, state, keep)
    c = state
    for t in range(5):
        ht, c = gated_recurrence_step(gates[:, t], c, keep[:, t - 1] if t else None)
        assert torch.allclose(ht, h[:, t], atol=1e-14)
    assert torch.allclose(c, last, atol=1e-14)
    buf = state.clone()
    _, out = gated_recurrence_step(gates[:, 0], buf, inplace=True)
    assert out is buf and not torch.equal(buf, state)


@pytest.mark.parametrize("T,n", [(0, 3), (4, 0), (0, 0)])
def test_recurrence_of_nothing(T, n):
    state = _randn(n, 2, seed=9)
    h, last = gated_recurrence(_randn(n, T, 6), state)
    assert h.shape == (n, T, 2) and torch.equal(last, state)
    assert last.data_ptr() != state.data_ptr() or n == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("keep_type", [torch.float32, torch.bool, None])
def test_padding_holds_anything_cpu(keep_type, dtype):
    """NaN and infinities behind a sequence's end change neither the outputs nor any gradient, which is zero there."""
    n, T, U = 4, 7, 3
    lengths = torch.tensor([0, 1, 4, 7])
    pad = torch.arange(T)[None] >= lengths[:, None]
    clean, state = _randn(n, T, 3 * U, seed=40).to(dtype).masked_fill(pad[..., None], 0.0), _randn(n, U, seed=41).float()
    d_h, d_last = _randn(n, T, U, seed=42).to(dtype).masked_fill(pad[..., None], 0.0), _randn(n, U, seed=43)
    keep = None if keep_type is None else (torch.arange(n * T).view(n, T) % 3 != 1).to(keep_type)
    out = []
    for bad in (None, float("nan"), float("inf")):
        gates, dh, k = clean.clone(), d_h.clone(), None if keep is None else keep.clone()
        if bad is not None:
            gates[pad] = dh[pad] = bad
            if keep_type == torch.float32:
                k[torch.arange(T)[None] >= lengths[:, None] - 1] = bad      # the last step's has no step behind it
        gates, s = gates.requires_grad_(), state.clone().requires_grad_()
        h, last = gated_recurrence(gates, s, k, lengths)
        out.append((h, last) + torch.autograd.grad((h, last), (gates, s), (dh, d_last.to(last.dtype))))
    for got in out[1:]:
        for a, b in zip(got, out[0]):
            assert a.isfinite().all() and torch.equal(a, b)
    assert not out[1][0][pad].any() and not out[1][2][pad].any()
    assert torch.equal(out[1][1][0], state[0].to(out[1][1].dtype))


@pytest.mark.parametrize("with_res,with_w", [(True, True), (False, True), (True, False), (False, False)])
def test_norm_cpu(with_res, with_w):
    x = _randn(3, 2, 7, seed=10).requires_grad_()
    r = _randn(3, 2, 7, seed=11).requires_grad_() if with_res else None
    w = _randn(7, seed=12).requires_grad_() if with_w else None
    inputs = [t for t in (x, r, w) if t is not None]
    assert torch.autograd.gradcheck(lambda *a: residual_rms_norm(x, r, w, eps=1e-3), inputs)
    d_y, d_s = _randn(3, 2, 7, seed=13), _randn(3, 2, 7, seed=14)
    y, s = residual_rms_norm(x, r, w, eps=1e-3)
    ref = R.norm(x, r, w, 1e-3, d_y, d_s)
    grads = dict(zip(("dx", "dr", "dw")[:1] + (("dr",) if with_res else ()) + (("dw",) if with_w else ()),
                     torch.autograd.grad((y, s), inputs, (d_y, d_s))))
    R.check(y, ref["y"][0], 1e-13 * (1 + ref["y"][0].abs()), "y")
    for name, got in grads.items():
        v = ref["dx" if name == "dr" else name][0]
        R.check(got, v, 1e-13 * (1 + v.abs()), name)


def _loss_inputs(M, K, seed=20):
    z = 2 * _randn(M, K, seed=seed)
    a = torch.randint(0, K, (M,), generator=torch.Generator().manual_seed(seed + 1))
    l = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    return z, a, l - 0.3 * _randn(M, seed=seed + 2), _randn(M, seed=seed + 3), l + 0.3 * _randn(M, seed=seed + 4)


@pytest.mark.parametrize("K", [1, 2, 6, 70])
@pytest.mark.parametrize("kind", ["plain", "mask", "none active", "denom"])
def test_policy_loss_cpu(K, kind):
    M = 12
    z, a, old, adv, ref = _loss_inputs(M, K)
    if K > 2:
        z[:, 1] = -torch.inf                    # a choice that cannot be taken
        a[a == 1] = 0
        old, ref = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0] + 0.25, old.clone()
    mask = None if kind == "plain" else torch.arange(M) % 3 != 0 if kind != "none active" else torch.zeros(M, dtype=torch.bool)
    denom = torch.tensor(7.0, dtype=torch.float64) if kind == "denom" else None
    z.requires_grad_()
    loss, terms = categorical_policy_loss(z, a, old, adv, clip=(0.1, 0.3), ref_log_probs=ref, kl_coef=0.2,
                                          entropy_coef=0.05, mask=mask, denom=denom)
    (d,) = torch.autograd.grad(loss, z)
    want = R.policy_loss(z, a, old, adv, ref, mask, denom, 0.9, 1.3, 0.2, 0.05)
    for got, name in ((loss, "loss"), (terms, "terms"), (d, "d_logits")):
        R.check(got, want[name][0], 1e-12 * (1 + want[name][0].abs()), name)
    lp, ent = categorical_log_probs(z.detach(), a)
    l, _, H, _, _, _ = R.rows_of(z, a)
    R.check(lp, l, 1e-12 * (1 + l.abs()), "log_probs")
    R.check(ent, H, 1e-12 * (1 + H.abs()), "entropy")


@pytest.mark.parametrize("dtype,unit", [(torch.float32, 2.0 ** -24), (torch.float64, 2.0 ** -53)])
def test_references_close_by_cpu(dtype, unit):
    """kl = exp d - d - 1 and its gradient where d is small. With one choice left l is 0, so d is the reference itself.
    40 units cover exp d - 1 and its difference to d at |d| = 1 / 2, where they cancel most."""
    d = torch.logspace(-6, 0.5, 60, dtype=dtype)
    d = torch.cat([d, -d])
    n, dd = len(d), d.double()
    exact, term = torch.zeros_like(dd), dd
    for k in range(2, 40):
        term = term * dd / k
        exact = exact + term
    z = torch.tensor([0.0, -30.0], dtype=dtype).expand(n, 2).clone().requires_grad_()
    row = torch.zeros(n, dtype=dtype)
    one = [float(categorical_policy_loss(torch.zeros(1, 1, dtype=dtype), row[:1].long(), row[:1], row[:1],
                                         ref_log_probs=d[k:k + 1], kl_coef=1.0)[1][1]) for k in range(n)]
    assert min(one) > 0.0
    R.check(torch.tensor(one, dtype=torch.float64), exact, 40 * unit * exact, "kl")
    loss, _ = categorical_policy_loss(z, row.long(), row, row, ref_log_probs=d, kl_coef=1.0, denom=torch.ones((), dtype=dtype))
    (dz,) = torch.autograd.grad(loss, z)
    p = torch.sigmoid(torch.tensor(-30.0, dtype=torch.float64))
    want = torch.expm1(dd + torch.log1p(torch.tensor(-30.0, dtype=torch.float64).exp())) * p
    # l = -log(1 + e^-30) moves d by its own rounding: half a step of 1 for the sum and as much for the logarithm, or all
    # of e^-30 = p where that is less; the gradient's slope in d is exp(d) p
    moved = min(2 * unit, float(p)) * dd.exp() * p
    R.check(dz[:, 1], want, 40 * unit * want.abs() + moved, "gradient of the other choice")


def test_policy_loss_gradient_by_differences():
    z, a, old, adv, ref = _loss_inputs(5, 6)
    mask = torch.tensor([True, True, False, True, True])
    z.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda q: categorical_policy_loss(q, a, old, adv, ref_log_probs=ref, kl_coef=0.3, entropy_coef=0.1, mask=mask)[0], (z,))


def test_refusals():
    f = torch.zeros
    bad = [
        lambda: gated_recurrence(f(2, 3, 7)), lambda: gated_recurrence(f(2, 6)), lambda: gated_recurrence(f(2, 3, 0)),
        lambda: gated_recurrence(torch.zeros(2, 3, 6, dtype=torch.int32)),
        lambda: gated_recurrence(f(2, 3, 6), f(2, 3)), lambda: gated_recurrence(f(2, 3, 6), f(2, 2).half()),
        lambda: gated_recurrence(f(2, 3, 6), keep=f(2, 2)), lambda: gated_recurrence(f(2, 3, 6), keep=f(2, 3).int()),
        lambda: gated_recurrence(f(2, 3, 6), keep=f(2, 3).requires_grad_()),
        lambda: gated_recurrence(f(2, 3, 6), lengths=f(2)), lambda: gated_recurrence(f(2, 3, 6), lengths=[3, 3]),
        lambda: gated_recurrence_step(f(2, 7), f(2, 2)), lambda: gated_recurrence_step(f(2, 6), None),
        lambda: gated_recurrence_step(f(2, 6), f(2, 3)), lambda: gated_recurrence_step(f(2, 6).requires_grad_(), f(2, 2)),
        lambda: gated_recurrence_step(f(2, 6), f(2, 4)[:, ::2], inplace=True),
        lambda: residual_rms_norm(f(2, 0)), lambda: residual_rms_norm(f(())), lambda: residual_rms_norm(f(2, 4), f(4)),
        lambda: residual_rms_norm(f(2, 4), f(2, 4).half()), lambda: residual_rms_norm(f(2, 4), weight=f(3)),
        lambda: residual_rms_norm(f(2, 4), eps=-1.0), lambda: residual_rms_norm(f(2, 4), eps=float("nan")),
        lambda: residual_rms_norm(torch.zeros(2, 4, dtype=torch.int64)),
        lambda: categorical_log_probs(f(2, 0), f(2).long()), lambda: categorical_log_probs(f(2, 3), f(3).long()),
        lambda: categorical_log_probs(f(2, 3), f(2)), lambda: categorical_log_probs(f(2, 3), None),
        lambda: categorical_log_probs(f(2, 3).requires_grad_(), f(2).long()),
    ]
    loss = lambda z=f(2, 3), a=f(2).long(), o=f(2), v=f(2), **kw: categorical_policy_loss(z, a, o, v, **kw)  # noqa: E731
    bad += [
        lambda: loss(a=f(2)), lambda: loss(o=f(3)), lambda: loss(o=None), lambda: loss(v=None), lambda: loss(v=f(2).half()),
        lambda: loss(o=f(2).requires_grad_()), lambda: loss(v=f(2).requires_grad_()), lambda: loss(mask=f(2)),
        lambda: loss(mask=f(3).bool()), lambda: loss(denom=f(2)), lambda: loss(denom=3.0), lambda: loss(clip=(-0.5, -0.6)),
        lambda: loss(clip=float("nan")), lambda: loss(kl_coef=0.1), lambda: loss(z=f(2, 0)),
        lambda: loss(ref_log_probs=f(2, 1)), lambda: loss(ref_log_probs=f(2).requires_grad_()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")


def test_c_abi_refusals():
    """The C entry points check before they touch the device: these return without one."""
    lib = _native.load()
    p = C.c_void_p(4096)            # never read: every call below is refused or has nothing to do
    fwd = lambda dt=0, n=1, T=1, U=1, g=p, gn=3, gt=3, h=p, last=p: lib.swarm_gated_scan_forward(  # noqa: E731
        dt, n, T, U, g, gn, gt, None, None, None, h, last, None, None, None)
    assert fwd(n=0, g=None, h=None, last=None) == 0
    for kw in (dict(dt=3), dict(dt=-1), dict(n=-1), dict(T=0), dict(U=0), dict(g=None), dict(h=None), dict(last=None),
               dict(gn=-1), dict(gt=-1), dict(n=1 << 40, T=1 << 30), dict(U=1 << 60)):
        assert fwd(**kw) == -1, kw
    bwd = lambda dt=0, n=1, T=1, U=1, g=p, tiles=p, dg=p, hn=1: lib.swarm_gated_scan_backward(  # noqa: E731
        dt, n, T, U, g, 3, 3, None, None, tiles, p, hn, 1, None, dg, None, None, None)
    assert bwd(n=0) == 0
    for kw in (dict(dt=9), dict(n=-1), dict(T=0), dict(U=0), dict(g=None), dict(tiles=None), dict(dg=None), dict(hn=-1)):
        assert bwd(**kw) == -1, kw
    step = lambda dt=0, rows=1, U=1, g=p, c=p, h=p, out=p, gr=3: lib.swarm_gated_step(  # noqa: E731
        dt, rows, U, g, gr, c, None, h, out, None)
    assert step(rows=0) == 0
    for kw in (dict(dt=5), dict(rows=-1), dict(U=0), dict(g=None), dict(c=None), dict(h=None), dict(out=None), dict(gr=-1)):
        assert step(**kw) == -1, kw
    nf = lambda dt=0, rows=1, D=1, x=p, r=p, y=p, s=p, eps=1e-6: lib.swarm_residual_norm_forward(  # noqa: E731
        dt, rows, D, x, 1, r, 1, None, eps, y, s, None, None)
    assert nf(rows=0) == 0
    for kw in (dict(dt=4), dict(rows=-1), dict(D=0), dict(x=None), dict(y=None), dict(s=None), dict(eps=-1.0),
               dict(eps=float("nan")), dict(rows=1 << 40, D=1 << 30)):
        assert nf(**kw) == -1, kw
    nb = lambda dt=0, rows=1, D=1, x=p, r=p, rr=1, rstd=p, dy=p, dx=p, dw=p, work=p: lib.swarm_residual_norm_backward(  # noqa: E731
        dt, rows, D, x, 1, r, rr, None, rstd, dy, 1, None, 0, dx, dw, work, None)
    assert nb(rows=0, dw=None, work=None) == 0
    for kw in (dict(dt=4), dict(rows=-1), dict(D=0), dict(x=None), dict(rr=-1), dict(rstd=None), dict(dy=None), dict(dx=None),
               dict(work=None)):
        assert nb(**kw) == -1, kw
    assert lib.swarm_residual_norm_workspace(-1, 4) == -1 and lib.swarm_residual_norm_workspace(4, 0) == -1
    assert lib.swarm_gated_scan_workspace(0, 5, 5) >= 0
    lp = lambda dt=0, M=1, K=1, z=p, a=p, o=p, e=p, ld=1: lib.swarm_log_probs(dt, M, K, z, ld, a, o, e, None, None, None)  # noqa: E731
    assert lp(M=0) == 0
    for kw in (dict(dt=7), dict(M=-1), dict(K=0), dict(z=None), dict(a=None), dict(o=None), dict(e=None), dict(ld=-1), dict(K=40000)):
        assert lp(**kw) == -1, kw
    lf = lambda dt=0, M=1, K=1, z=p, a=p, old=p, adv=p, lo=0.8, hi=1.2, loss=p, terms=p, used=p, st=p, part=p: (  # noqa: E731
        lib.swarm_policy_loss_forward(dt, M, K, z, 1, a, old, None, adv, None, None, lo, hi, 0.0, 0.0, loss, terms,
                                      used, st, None, part, None, None))
    for kw in (dict(dt=7), dict(M=-1), dict(K=0), dict(z=None), dict(a=None), dict(old=None), dict(adv=None),
               dict(lo=1.3), dict(lo=float("nan")), dict(loss=None), dict(terms=None), dict(used=None), dict(st=None),
               dict(part=None)):
        assert lf(**kw) == -1, kw
    lb = lambda dt=0, M=1, K=1, z=p, a=p, st=p, used=p, g=p, d=p: lib.swarm_policy_loss_backward(  # noqa: E731
        dt, M, K, z, 1, a, 0.0, st, used, g, 0, d, None)
    assert lb(M=0) == 0
    for kw in (dict(dt=7), dict(M=-1), dict(K=0), dict(z=None), dict(a=None), dict(st=None), dict(used=None),
               dict(g=None), dict(d=None)):
        assert lb(**kw) == -1, kw


def test_a_graph_does_not_make_the_input_check(monkeypatch):
    """The word that reports bad actions is made before a capture, or the capture is refused."""
    from SwarmACB_isaac.agents import _trainer, sequence_ops

    monkeypatch.setattr(_trainer, "_BAD_ACTIONS", {})
    monkeypatch.setattr(sequence_ops, "_BAD_ACTIONS", _trainer._BAD_ACTIONS)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="once before"):
        sequence_ops._flag(torch.device("cuda:0"), "categorical_log_probs")
    flag = _trainer._BAD_ACTIONS["cuda:0"] = torch.zeros(1, dtype=torch.int32)
    assert sequence_ops._flag(torch.device("cuda:0"), "categorical_log_probs") is flag
