"""How exact the sequence-policy kernels are in float32 where values are small: closed and open gates, unlikely choices.

Units of E = 2^-24, half a float32 step, relative to the value. exp is formed as 2^h (1 + d) with h = x log2 e rounded
and d = x - h ln 2 what the rounding left out: 2 for the hardware's 2^h, 1 for the last product, |x| / 20 for ln 2's own
rounding. A sigmoid adds 1 for the sum, 2 for the reciprocal and 1 for a product: at most 7 + |x| / 20. So every bound
here grows with |x| by a twentieth of it or less; exp's argument rounded as one product with log2 e would cost |x|."""

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = 2.0 ** -126        # below it a float32 kernel may give 0, or the smallest normal number


def _ops():
    from SwarmACB_isaac.agents import sequence_ops

    return sequence_ops


def _close(got, ref, units, what):
    off, allowed = (got.detach().double().cpu() - ref).abs(), units * E * ref.abs() + 2 * TINY
    worst = int((off / allowed).argmax())
    assert not (off > allowed).any() and not off.isnan().any(), (
        f"{what}: off by {float(off.reshape(-1)[worst] / ref.abs().reshape(-1)[worst] / E):.1f} units, "
        f"{float(units.expand_as(ref).reshape(-1)[worst]):.1f} allowed, value {float(ref.reshape(-1)[worst]):.4g}")


def _gate_values(n, U):
    far = [100.0, 1e4, 3e38, float("inf")]
    x = torch.linspace(-86.0, 86.0, n * U - 2 * len(far))
    return torch.cat([x, torch.tensor(far), -torch.tensor(far)]).view(n, U)


def _units(x):
    return 8 + x.double().abs().clamp(max=128) / 20


@pytest.mark.parametrize("n,T,U", [(64, 1, 64), (1365, 1, 3), (64, 17, 64), (1365, 40, 3), (2, 1024, 2048)])
def test_gates_of_a_sequence(n, T, U, gpu_device):
    """One live step: the state becomes f with a candidate of 0, 1 - f with a state of 0, and h becomes o. A walked
    thread, tiles, single channels, and a length that is split."""
    x = _gate_values(n, U)
    xd = x.double()
    f, b = torch.sigmoid(xd), torch.sigmoid(-xd)
    lengths = torch.ones(n, dtype=torch.long, device=gpu_device)
    u = _units(x)

    def call(xf, z, xo, state):
        gates = torch.zeros(n, T, 3 * U, device=gpu_device)
        for k, v in enumerate((xf, z, xo)):
            gates[:, 0, k * U:(k + 1) * U] = v
        gates.requires_grad_()
        state = torch.full((n, U), state, device=gpu_device, requires_grad=True)
        return _ops().gated_recurrence(gates, state, None, lengths), (gates, state)

    x = x.to(gpu_device)
    (_, last), leaves = call(x, 0.0, 0.0, 1.0)
    d, d_state = torch.autograd.grad(last.sum(), leaves)
    _close(last, f, u, "f")
    _close(d_state, f, u, "d state")
    _close(d[:, 0, U:2 * U], b, u, "d candidate")
    _close(d[:, 0, :U], f * b, 2 * u + 2, "d forget gate")
    _close(call(x, 1.0, 0.0, 0.0)[0][1], b, u, "1 - f")
    (h, _), leaves = call(torch.full_like(x, 86.0), 0.0, x, 1.0)
    d = torch.autograd.grad(h.sum(), leaves)[0]
    _close(h[:, 0], f, u, "o")
    _close(d[:, 0, 2 * U:], f * b, 2 * u + 2, "d output gate")


def test_gates_of_a_step(gpu_device):
    x = _gate_values(64, 64)
    f, b = torch.sigmoid(x.double()), torch.sigmoid(-x.double())
    one, zero, wide = torch.ones(64, 64, device=gpu_device), torch.zeros(64, 64, device=gpu_device), 86.0 * torch.ones(64, 64)
    call = lambda *g, state: _ops().gated_recurrence_step(torch.cat([t.to(gpu_device) for t in g], 1), state)  # noqa: E731
    _close(call(x, zero, zero, state=one)[1], f, _units(x), "f")
    _close(call(x, one, zero, state=zero)[1], b, _units(x), "1 - f")
    _close(call(wide, zero, x, state=one)[0], f, _units(x), "o")


@pytest.mark.parametrize("grad", [1.0, 2.0])
@pytest.mark.parametrize("K", [2, 65, 700, 5000, 9000, 20000, 40000])
def test_unlikely_choices(K, grad, gpu_device):
    """Two choices y apart, the likely one taken: the other's gradient is its probability, down to 1e-37. Beyond the
    exponential's 3 + y / 20: the sum 1, its reciprocal 2, the ratio 5, three products 3."""
    M = 300
    y = -torch.linspace(0.5, 85.0, M)
    z = torch.full((M, K), -float("inf"))
    g = torch.Generator().manual_seed(K)
    at = torch.stack([torch.randperm(K, generator=g)[:2] for _ in range(M)])
    rows = torch.arange(M)
    z[rows, at[:, 0]], z[rows, at[:, 1]] = 0.0, y
    old = -torch.log1p(y.double().exp())
    leaf = z.to(gpu_device).requires_grad_()
    loss, _ = _ops().categorical_policy_loss(leaf, at[:, 0].to(gpu_device), old.float().to(gpu_device),
                                             torch.ones(M, device=gpu_device), denom=torch.ones((), device=gpu_device))
    (d,) = torch.autograd.grad(loss, leaf, torch.tensor(grad, device=gpu_device))
    p = torch.sigmoid(y.double())
    _close(d[rows, at[:, 1]], grad * p, 16 + y.double().abs() / 20, "gradient of the unlikely choice")
    d = d.detach().clone()
    d[rows, at[:, 0]], d[rows, at[:, 1]] = 0.0, 0.0
    assert not d.any()


def test_references_close_by(gpu_device):
    """kl = exp d - d - 1 and its gradient where d is small, as it is in every update: with one choice left l is 0, so d
    is the reference itself. 40 units cover exp d - 1 and its difference to d at |d| = 1 / 2, where they cancel most."""
    d = torch.logspace(-6, 0.5, 80)
    d = torch.cat([d, -d, torch.zeros(1)])
    dd = d.double()
    kl = torch.where(dd.abs() < 1e-2, dd ** 2 * (0.5 + dd * (1 / 6 + dd * (1 / 24 + dd * (1 / 120 + dd / 720)))),
                     torch.expm1(dd) - dd)
    row = torch.zeros(1, device=gpu_device)
    for k in range(len(d)):
        _, terms = _ops().categorical_policy_loss(torch.zeros(1, 1, device=gpu_device), row.long(), row, row,
                                                  ref_log_probs=d[k:k + 1].to(gpu_device), kl_coef=1.0)
        _close(terms[1], kl[k], torch.tensor(40.0), f"kl of {float(d[k])}")
        assert float(terms[1]) >= 0.0
    d, dd, M = d[:-1], dd[:-1], len(d) - 1          # without 0, where the other choice's own e^-30 is all there is
    z = torch.tensor([0.0, -30.0], device=gpu_device).expand(M, 2).clone().requires_grad_()
    rows = torch.zeros(M, device=gpu_device)
    loss, _ = _ops().categorical_policy_loss(z, rows.long(), rows, rows, ref_log_probs=d.to(gpu_device), kl_coef=1.0,
                                             denom=torch.ones((), device=gpu_device))
    (dz,) = torch.autograd.grad(loss, z)
    p = torch.sigmoid(torch.tensor(-30.0, dtype=torch.float64))
    ref = torch.expm1(dd + torch.log1p(torch.tensor(-30.0, dtype=torch.float64).exp())) * p
    _close(dz[:, 1], ref, 40 + 0 * ref, "gradient of the other choice")
