"""Sequence-policy operators on the GPU against the 64-bit reference (tests/sequence_reference.py derives every
bound), at the sizes, strides, masks and values where they can go wrong; captured, on side streams, together."""

import pytest
import torch

import sequence_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from SwarmACB_isaac.agents import sequence_ops

    return sequence_ops


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


# ------------------------------------------------------------------------------------ gated recurrence

def _recurrence_inputs(dev, n, T, U, dtype, keep, lengths, seed):
    g = _gen(dev, seed)
    gates = torch.randn(n, T, 3 * U, device=dev, generator=g)
    gates[..., :U] += 2.0
    k = (torch.rand(n, T, device=dev, generator=g) > 0.1).float() if keep else None
    ln = None
    if lengths:
        ln = torch.randint(0, T + 1, (n,), device=dev, generator=g)
        ln[0] = 0 if n > 1 else T // 2
        ln[-1] = T if n > 1 else ln[-1]
    return (gates.to(dtype), torch.randn(n, U, device=dev, generator=g), k, ln,
            torch.randn(n, T, U, device=dev, generator=g).to(dtype), torch.randn(n, U, device=dev, generator=g))


def _check_recurrence(gates, state, keep, lengths, d_h, d_last, ref_of=None):
    gates, state = gates.requires_grad_(), state.requires_grad_() if state is not None else None
    h, last = _ops().gated_recurrence(gates, state, keep, lengths)
    leaves = (gates,) if state is None else (gates, state)
    grads = torch.autograd.grad((h, last), leaves, (d_h, d_last))
    assert h.dtype == gates.dtype and last.dtype == torch.float32 and grads[0].dtype == gates.dtype
    ref = R.recurrence(gates, state, keep, lengths, d_h, d_last)
    for got, name in zip((h, last) + grads, ("h", "last", "d_gates", "d_state")):
        R.check(got, *ref[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,T,U,keep,lengths", [
    (1, 1, 1, False, False), (5, 2, 3, True, True), (16, 128, 64, True, False), (2, 129, 65, True, True),
    (3, 257, 72, False, True), (1, 2000, 8, True, False), (2, 700, 200, False, False), (300, 5, 40, True, True),
    (1, 4099, 16, False, True), (40, 31, 264, True, False)])
def test_recurrence(n, T, U, keep, lengths, dtype, gpu_device):
    _check_recurrence(*_recurrence_inputs(gpu_device, n, T, U, dtype, keep, lengths, n * 1000 + T))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 511, 513])
def test_recurrence_at_every_border(T, gpu_device):
    """Around the lengths where the number of tiles, of saved states or of chunks changes, with ragged ends."""
    for U in (3, 8, 67):
        _check_recurrence(*_recurrence_inputs(gpu_device, 3, T, U, torch.bfloat16, True, True, T * 7 + U))


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_of_a_strided_view_without_state(dtype, gpu_device):
    """Rows of a wider, time-major buffer whose start is not aligned; a gradient that is a broadcast view."""
    n, T, U = 3, 150, 20
    g = _gen(gpu_device, 5)
    big = torch.randn(T, n, 3 * U + 7, device=gpu_device, generator=g).to(dtype)
    gates = big[:, :, 5:5 + 3 * U].transpose(0, 1)
    assert not gates.is_contiguous() and gates.stride(2) == 1
    leaf = gates.detach().requires_grad_()
    h, last = _ops().gated_recurrence(leaf)
    d = torch.autograd.grad(h, leaf, torch.ones((), device=gpu_device, dtype=dtype).expand(n, T, U))[0]
    ref = R.recurrence(gates, None, None, None, torch.ones(n, T, U), None)
    R.check(h, *ref["h"], "h")
    R.check(last, *ref["last"], "last")
    R.check(d, *ref["d_gates"], "d_gates")
    d_only_last = torch.autograd.grad(_ops().gated_recurrence(leaf)[1].sum(), leaf)[0]
    ref = R.recurrence(gates, None, None, None, None, torch.ones(n, U))
    R.check(d_only_last, *ref["d_gates"], "d_gates of the last state")


def test_recurrence_time_major_columns(gpu_device):
    """A last dimension that is not contiguous is copied, not misread."""
    base = torch.randn(2, 3 * 24, 40, device=gpu_device, generator=_gen(gpu_device, 6))
    gates = base.transpose(1, 2)
    h, last = _ops().gated_recurrence(gates)
    ref = R.recurrence(gates, None, None, None)
    R.check(h, *ref["h"], "h")
    R.check(last, *ref["last"], "last")


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_holds_anything(dtype, gpu_device):
    """NaN and infinities behind a sequence's end change nothing and get zero gradients."""
    n, T, U = 4, 300, 48
    gates, state, keep, _, d_h, d_last = _recurrence_inputs(gpu_device, n, T, U, dtype, True, False, 7)
    lengths = torch.tensor([0, 1, 137, 300], device=gpu_device, dtype=torch.int32)
    pad = torch.arange(T, device=gpu_device)[None] >= lengths[:, None]
    clean = gates.clone()
    clean[pad] = 0.0
    gates[pad], d_h[pad], keep[pad] = float("nan"), float("inf"), float("nan")
    out = []
    for z, dh, k in ((gates, d_h, keep), (clean, d_h.masked_fill(pad[..., None], 0.0), keep.masked_fill(pad, 0.0))):
        z, s = z.clone().requires_grad_(), state.clone().requires_grad_()
        h, last = _ops().gated_recurrence(z, s, k, lengths)
        out.append((h, last) + torch.autograd.grad((h, last), (z, s), (dh, d_last)))
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not out[0][0][pad].any() and not out[0][2][pad].any()
    assert torch.equal(out[0][1][0], state[0]) and torch.equal(out[0][3][0], d_last[0])


def test_lengths_outside_the_sequence_are_clamped(gpu_device):
    gates, state, keep, _, _, _ = _recurrence_inputs(gpu_device, 3, 50, 16, torch.float32, True, False, 8)
    far = torch.tensor([-3, 1 << 40, 25], device=gpu_device)
    near = torch.tensor([0, 50, 25], device=gpu_device)
    for a, b in zip(_ops().gated_recurrence(gates, state, keep, far), _ops().gated_recurrence(gates, state, keep, near)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_gates(dtype, gpu_device):
    """Closed and open gates (largest and lowest values, infinities) stay finite; a NaN stays in its channel."""
    n, T, U = 2, 200, 32
    gates, state, _, _, d_h, d_last = _recurrence_inputs(gpu_device, n, T, U, dtype, False, False, 9)
    top = torch.finfo(dtype).max
    gates[0, 3, :U], gates[0, 4, :U], gates[0, 5, :U] = top, -top, float("inf")
    gates[0, 6, :U], gates[1, 7, 2 * U:], gates[1, 8, 2 * U:] = -float("inf"), -top, float("inf")
    gates[1, 50, 5] = float("nan")
    gates, state = gates.requires_grad_(), state.requires_grad_()
    h, last = _ops().gated_recurrence(gates, state)
    d_gates, d_state = torch.autograd.grad((h, last), (gates, state), (d_h, d_last))
    bad = torch.zeros(n, T, U, dtype=torch.bool, device=gpu_device)
    bad[1, 50:, 5] = True
    assert torch.equal(h.isnan(), bad)
    assert d_gates[0].isfinite().all() and d_state[0].isfinite().all()
    other = [u for u in range(U) if u != 5]
    assert d_gates[1].view(T, 3, U)[..., other].isfinite().all() and last[1, other].isfinite().all()


def test_offsets_beyond_32_bits(gpu_device):
    """Two sequences 2.3e9 elements apart."""
    T, U, far = 130, 64, 2_300_000_000
    store = torch.empty(far + T * 3 * U, dtype=torch.bfloat16, device=gpu_device)
    gates = store.as_strided((2, T, 3 * U), (far, 3 * U, 1))
    gates.copy_(torch.randn(2, T, 3 * U, device=gpu_device, generator=_gen(gpu_device, 10)))
    ref = R.recurrence(gates, None, None, None, torch.ones(2, T, U), None)
    leaf = gates.detach().requires_grad_()
    h, last = _ops().gated_recurrence(leaf)
    d = torch.autograd.grad(h, leaf, torch.ones_like(h))[0]
    R.check(h, *ref["h"], "h")
    R.check(last, *ref["last"], "last")
    R.check(d, *ref["d_gates"], "d_gates")


def test_recurrence_beyond_32_bits_of_outputs(gpu_device):
    """More than 2^31 gate elements: the last sequence equals the same sequence alone."""
    n, T, U = 9, 4000, 20000
    gates = torch.empty(n, T, 3 * U, dtype=torch.bfloat16, device=gpu_device).normal_(generator=_gen(gpu_device, 11))
    assert gates.numel() > 1 << 31
    d_h = torch.ones((), dtype=torch.bfloat16, device=gpu_device).expand(1, T, U)
    tail = gates[-1:].clone().requires_grad_()
    alone = _ops().gated_recurrence(tail)
    alone_d = torch.autograd.grad(alone[0], tail, d_h)[0]
    gates.requires_grad_()
    h, last = _ops().gated_recurrence(gates)
    d = torch.autograd.grad(h, gates, d_h.expand(n, T, U))[0]
    # how a length is split may go by the number of channels: a bfloat16 step of the largest values
    for a, b in ((h[-1:], alone[0]), (last[-1:], alone[1]), (d[-1:], alone_d)):
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -8 * float(b.float().abs().max())


@pytest.mark.parametrize("T", [1, 17])
def test_more_sequences_than_a_grid_counts(T, gpu_device):
    """More threads than the 2^32 of a launch: sequences at both ends and at the seam equal the same ones alone."""
    n = 268_435_450
    gates = torch.empty(n, T, 3, dtype=torch.bfloat16, device=gpu_device).normal_(generator=_gen(gpu_device, 12))
    d_h = torch.ones((), dtype=torch.bfloat16, device=gpu_device)
    gates.requires_grad_()
    h, last = _ops().gated_recurrence(gates)
    d = torch.autograd.grad(h, gates, d_h.expand(n, T, 1))[0]
    for part in (slice(0, 9), slice(n // 2 - 9, n // 2 + 9), slice(n - 9, n)):
        few = gates.detach()[part].clone().requires_grad_()
        few_h, few_last = _ops().gated_recurrence(few)
        few_d = torch.autograd.grad(few_h, few, d_h.expand(few.shape[0], T, 1))[0]
        for a, b in ((h[part], few_h), (last[part], few_last), (d[part], few_d)):
            # how a length is split may go by the number of channels: a bfloat16 step of the largest values
            assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -8 * float(b.float().abs().max())


def test_more_rows_than_a_grid_counts(gpu_device):
    """The step form and the norm with more than 2^32 threads: rows at both ends and at the seam equal the same
    rows alone."""
    rows, U = (1 << 30) + 5, 4
    parts = (slice(0, 9), slice((1 << 30) - 100, rows))
    gates = torch.empty(rows, 3 * U, dtype=torch.bfloat16, device=gpu_device).normal_(generator=_gen(gpu_device, 13))
    state = torch.ones(rows, U, device=gpu_device)
    h, c = _ops().gated_recurrence_step(gates, state, inplace=True)
    for part in parts:
        few_h, few_c = _ops().gated_recurrence_step(gates[part].clone(), torch.ones_like(c[part]))
        assert torch.equal(h[part], few_h) and torch.equal(c[part], few_c)
    del h, c, state, gates
    x = torch.empty(rows, 8, dtype=torch.bfloat16, device=gpu_device).normal_(generator=_gen(gpu_device, 14))
    y, stream = _ops().residual_rms_norm(x, x)
    for part in parts:
        few_y, few_stream = _ops().residual_rms_norm(x[part].clone(), x[part].clone())
        assert torch.equal(y[part], few_y) and torch.equal(stream[part], few_stream)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,U", [(1, 1), (20, 64), (333, 67), (4096, 64)])
def test_step(rows, U, dtype, gpu_device):
    g = _gen(gpu_device, rows)
    wide = torch.randn(rows, 3 * U + 3, device=gpu_device, generator=g).to(dtype)
    for gates in (wide[:, :3 * U].contiguous(), wide[:, 1:1 + 3 * U]):
        state = torch.randn(rows, U, device=gpu_device, generator=g)
        keep = torch.rand(rows, device=gpu_device, generator=g) > 0.3
        ref = R.recurrence(gates[:, None], state * keep[:, None], None, None)
        kept = state.clone()
        h, out = _ops().gated_recurrence_step(gates, state, keep)
        assert torch.equal(kept, state)
        R.check(h[:, None], *ref["h"], "h")
        R.check(out, *ref["last"], "state")
        h2, out2 = _ops().gated_recurrence_step(gates, state, keep, inplace=True)
        assert out2 is state and torch.equal(out2, out) and torch.equal(h2, h)


def test_step_of_nothing(gpu_device):
    h, c = _ops().gated_recurrence_step(torch.zeros(0, 12, device=gpu_device), torch.zeros(0, 4, device=gpu_device))
    assert h.shape == c.shape == (0, 4)


# ------------------------------------------------------------------------------------------- the norm

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (20, 128), (7, 63), (129, 257), (1000, 512), (33, 1001), (5, 4096),
                                    (64, 5000), (2, 16384), (3, 20011), (2, 70000),
                                    (3000, 16), (777, 31), (1030, 33), (515, 128), (300, 129), (9, 2049), (7, 8193)])
def test_norm(rows, D, dtype, gpu_device):
    g = _gen(gpu_device, rows + D)
    x, r, dy, ds = (torch.randn(rows, D, device=gpu_device, generator=g).to(dtype) for _ in range(4))
    w = (1 + 0.3 * torch.randn(D, device=gpu_device, generator=g)).to(dtype)
    for res, wt, both in ((r, w, True), (None, w, False), (r, None, True), (None, None, False)):
        leaves = [t.detach().requires_grad_() for t in (x, res, wt) if t is not None]
        it = iter(leaves)
        xl, rl, wl = next(it), next(it) if res is not None else None, next(it) if wt is not None else None
        y, s = _ops().residual_rms_norm(xl, rl, wl, eps=1e-5)
        outs, gs = ((y, s), (dy, ds)) if both else ((y,), (dy,))
        grads = torch.autograd.grad(outs, leaves, gs)
        ref = R.norm(x, res, wt, 1e-5, dy, ds if both else None)
        R.check(y, *ref["y"], "y")
        R.check(s, *ref["stream"], "stream")
        R.check(grads[0], *ref["dx"], "dx")
        if res is not None:
            assert torch.equal(grads[0], grads[1])
        if wt is not None:
            R.check(grads[-1], *ref["dw"], "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(1, 3), (600, 1), (70001, 5), (300000, 7), (255, 4)])
def test_norm_of_narrow_rows(rows, D, dtype, gpu_device):
    test_norm(rows, D, dtype, gpu_device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_strided_rows(dtype, gpu_device):
    """Row slices of wider buffers, at offsets that no vector load is aligned to; gradients that are views."""
    rows, D = 37, 200
    g = _gen(gpu_device, 12)
    buf = [torch.randn(rows, D + 9, device=gpu_device, generator=g).to(dtype) for _ in range(4)]
    x, r, dy, ds = (b[:, k:k + D] for b, k in zip(buf, (1, 3, 0, 5)))
    w = torch.randn(D + 1, device=gpu_device, generator=g).to(dtype)[1:]
    xl, rl, wl = (t.detach().requires_grad_() for t in (x, r, w))
    y, s = _ops().residual_rms_norm(xl, rl, wl)
    grads = torch.autograd.grad((y, s), (xl, rl, wl), (dy, ds))
    ref = R.norm(x, r, w, 1e-6, dy, ds)
    for got, name in ((y, "y"), (s, "stream"), (grads[0], "dx"), (grads[2], "dw")):
        R.check(got, *ref[name], name)
    only = torch.autograd.grad(_ops().residual_rms_norm(xl, rl, wl)[1], (xl, rl, wl), ds)
    assert torch.equal(only[0], ds) and torch.equal(only[1], ds) and not only[2].any()
    three = x.reshape(rows, 2, D // 2).transpose(0, 1)
    y3, _ = _ops().residual_rms_norm(three)
    R.check(y3, *R.norm(three, None, None, 1e-6)["y"], "transposed")


@pytest.mark.parametrize("D", [96, 1031])
def test_norm_zero_rows_and_extremes(D, gpu_device):
    """A row of zeros gives zeros with eps, rows of no length give nothing; a NaN stays in its row."""
    x = torch.zeros(3, D, device=gpu_device)
    x[2, 7] = float("nan")
    x[1] = 1e15
    xl = x.requires_grad_()
    y, _ = _ops().residual_rms_norm(xl)
    (d,) = torch.autograd.grad(y, xl, torch.ones_like(y))
    assert not y[0].any() and torch.allclose(y[1], torch.ones_like(y[1])) and y[2].isnan().all()
    assert d[:2].isfinite().all()
    e = torch.zeros(0, D, device=gpu_device, requires_grad=True)
    w = torch.ones(D, device=gpu_device, requires_grad=True)
    y, s = _ops().residual_rms_norm(e, e.detach(), w)
    de, dw = torch.autograd.grad((y.sum() + s.sum()), (e, w))
    assert y.shape == (0, D) and de.shape == (0, D) and not dw.any()


def test_norm_weight_gradient_repeats(gpu_device):
    """No atomics: the same inputs give the same bits."""
    g = _gen(gpu_device, 13)
    x, dy = (torch.randn(3000, 300, device=gpu_device, generator=g) for _ in range(2))
    w = torch.ones(300, device=gpu_device, requires_grad=True)
    runs = [torch.autograd.grad(_ops().residual_rms_norm(x, None, w)[0], w, dy)[0] for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


# -------------------------------------------------------------------------------------- the policy loss

def _loss_inputs(dev, M, K, dtype, seed):
    g = _gen(dev, seed)
    z = (2 * torch.randn(M, K, device=dev, generator=g)).to(dtype)
    a = torch.randint(0, K, (M,), device=dev, generator=g)
    l = torch.log_softmax(z.float(), 1).gather(1, a[:, None])[:, 0]
    shift = 0.3 * torch.randn(M, device=dev, generator=g)
    for border in (0.8, 1.2):        # off the kinks by far more than any rounding
        b = torch.tensor(border).log().item()
        shift = torch.where((shift - b).abs() < 0.01, torch.full_like(shift, b + 0.02), shift)
    return z, a, l - shift, torch.randn(M, device=dev, generator=g), l + 0.3 * torch.randn(M, device=dev, generator=g)


def _check_loss(z, a, old, adv, ref, mask, denom, g=1.0, **kw):
    leaf = z.detach().requires_grad_()
    loss, terms = _ops().categorical_policy_loss(leaf, a, old, adv, clip=0.2, ref_log_probs=ref,
                                                 kl_coef=0.1 if ref is not None else 0.0, entropy_coef=0.02,
                                                 mask=mask, denom=denom, **kw)
    (d,) = torch.autograd.grad(loss, leaf, torch.tensor(float(g), device=z.device))
    assert loss.dtype == torch.float32 and loss.shape == () and d.dtype == z.dtype and not terms.requires_grad
    want = R.policy_loss(z, a, old, adv, ref, mask, denom, 1 - 0.2, 1 + 0.2, 0.1 if ref is not None else 0.0, 0.02, float(g))
    for got, name in ((loss, "loss"), (terms, "terms"), (d, "d_logits")):
        R.check(got, *want[name], name)
    return loss, d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 2), (2048, 6), (700, 18), (65, 64), (130, 65), (50, 333), (9, 1000),
                                 (17, 4096), (6, 5001), (3, 50001), (2, 140000), (5000, 3)])
def test_policy_loss(M, K, dtype, gpu_device):
    z, a, old, adv, ref = _loss_inputs(gpu_device, M, K, dtype, M + K)
    mask = torch.rand(M, device=gpu_device, generator=_gen(gpu_device, 3)) < 0.7
    scale = float(M * min(K, 1024)) if dtype == torch.float16 else 1.0
    _check_loss(z, a, old, adv, ref, mask, None, scale)
    _check_loss(z, a, old, adv, None, None, torch.tensor(3.5, device=gpu_device), scale * 0.75)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [4, 8, 9, 15, 64, 65, 255, 256, 257, 512, 513, 1024, 1025, 2048, 2049, 8192, 8193, 16384,
                               16385, 32768, 32769, 65536, 65537])
def test_rows_at_every_border(K, dtype, gpu_device):
    """Around the row lengths where another layout takes over; the action in the row's first and last places too."""
    M = 5
    z, a, old, adv, ref = _loss_inputs(gpu_device, M, K, dtype, K + 1)
    a[0], a[1], a[2] = K - 1, 0, max(0, K - 3)
    l = torch.log_softmax(z.float(), 1).gather(1, a[:, None])[:, 0]
    old, ref = l - 0.07, l + 0.2
    _check_loss(z, a, old, adv, ref, None, None)
    _check_loss(z, a, old, adv, ref, torch.tensor([True, False, True, True, True], device=gpu_device), None, 0.5)
    lp, ent = _ops().categorical_log_probs(z, a)
    l, le, H, He, _, _ = R.rows_of(z, a)
    R.check(lp, l, le, "log_probs")
    R.check(ent, H, He, "entropy")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [66, 127, 128, 129, 384, 385, 768, 769, 1536, 1537, 2047, 4096, 4097, 8191])
def test_16_bit_rows_at_every_border(K, dtype, gpu_device):
    test_rows_at_every_border(K, dtype, gpu_device)


@pytest.mark.parametrize("M,K", [(1, 20000), (3, 33333), (300, 17000)])
def test_few_long_rows(M, K, gpu_device):
    """Rows that are read in parts: parts without any choice, a NaN, an infinity and a row with nothing to take."""
    z, a, *_ = _loss_inputs(gpu_device, M, K, torch.bfloat16, M + 5)
    z[0, :K // 2] = -float("inf")
    a[0] = K - 2
    if M > 2:
        z[1, K - 1], z[2] = float("nan"), -float("inf")
    if M > 3:
        z[3, 5] = float("inf")
    lp, ent = _ops().categorical_log_probs(z, a)
    l, le, H, He, _, _ = R.rows_of(z, a)
    bad = torch.zeros(M, dtype=torch.bool)
    bad[1:min(M, 4) if M > 3 else min(M, 3)] = M > 1
    nan = torch.full((M,), float("nan"), dtype=torch.float64)
    R.check(lp, torch.where(bad, nan, l), le, "log_probs")
    R.check(ent, torch.where(bad, nan, H), He, "entropy")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (2048, 6), (81, 18), (40, 64), (33, 77), (9, 2000), (4, 5001), (3, 140000),
                                 (70000, 2)])
def test_log_probs(M, K, dtype, gpu_device):
    z, a, *_ = _loss_inputs(gpu_device, M, K, dtype, M * 3 + K)
    lp, ent = _ops().categorical_log_probs(z, a.int())
    l, le, H, He, _, _ = R.rows_of(z, a)
    R.check(lp, l, le, "log_probs")
    R.check(ent, H, He, "entropy")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [5, 64, 130, 3001])
def test_choices_that_cannot_be_taken(K, dtype, gpu_device):
    """-inf and the type's lowest value: probability 0, no gradient; one choice left: l = 0, H = 0."""
    M = 24
    z, a, old, adv, ref = _loss_inputs(gpu_device, M, K, dtype, K)
    z[:, ::2], z[:8, 1::4] = -float("inf"), torch.finfo(dtype).min
    z[:, 3] = 1.0
    z[16:] = -float("inf")
    z[16:, 3] = -5.0
    a[:] = 3
    l = torch.log_softmax(z.float(), 1)[:, 3]
    old, ref = l - 0.1, l + 0.2
    lp, ent = _ops().categorical_log_probs(z, a)
    assert not lp[16:].any() and not ent[16:].any()
    _, d = _check_loss(z, a, old, adv, ref, None, None, float(M) if dtype == torch.float16 else 1.0)
    assert not d[:, ::2].any() and not d[16:].any()


@pytest.mark.parametrize("K", [40000, 50001])
def test_choices_of_long_rows_that_cannot_be_taken(K, gpu_device):
    test_choices_that_cannot_be_taken(K, torch.bfloat16, gpu_device)


@pytest.mark.parametrize("K", [6, 500, 9000])
def test_inactive_rows_are_not_looked_at(K, gpu_device):
    """NaN logits, NaN operands and sentinel actions on inactive rows change nothing and raise nothing."""
    M = 40
    z, a, old, adv, ref = _loss_inputs(gpu_device, M, K, torch.float32, 77)
    mask = torch.arange(M, device=gpu_device) % 3 != 1
    loss, d = _check_loss(z, a, old, adv, ref, mask, None)
    z2, a2 = z.clone(), a.clone()
    z2[~mask], a2[~mask] = float("nan"), -1
    for t in (old, adv, ref):
        t[~mask] = float("nan")
    leaf = z2.requires_grad_()
    loss2, _ = _ops().categorical_policy_loss(leaf, a2, old, adv, clip=0.2, ref_log_probs=ref, kl_coef=0.1,
                                              entropy_coef=0.02, mask=mask)
    (d2,) = torch.autograd.grad(loss2, leaf)
    assert torch.equal(loss, loss2) and torch.equal(d, d2) and not d2[~mask].any()
    _ops().check_policy_inputs(gpu_device)


@pytest.mark.parametrize("K", [6, 300])
def test_nothing_active_and_nothing_at_all(K, gpu_device):
    z, a, old, adv, ref = _loss_inputs(gpu_device, 8, K, torch.float32, 5)
    loss, d = _check_loss(z, a, old, adv, ref, torch.zeros(8, dtype=torch.bool, device=gpu_device), None)
    assert float(loss) == 0.0 and not d.any()
    e = torch.zeros(0, K, device=gpu_device, requires_grad=True)
    n = torch.zeros(0, device=gpu_device)
    loss, terms = _ops().categorical_policy_loss(e, n.long(), n, n)
    (d,) = torch.autograd.grad(loss, e)
    assert float(loss) == 0.0 and not terms.any() and d.shape == (0, K)
    lp, ent = _ops().categorical_log_probs(e.detach(), n.long())
    assert lp.shape == ent.shape == (0,)


@pytest.mark.parametrize("K", [6, 300, 9000])
def test_actions_out_of_range_are_reported(K, gpu_device):
    z, a, old, adv, _ = _loss_inputs(gpu_device, 8, K, torch.float32, 6)
    ops = _ops()
    ops.check_policy_inputs(gpu_device)
    for bad in (-1, K, 1 << 40):
        b = a.clone()
        b[5] = bad
        leaf = z.detach().requires_grad_()
        loss, _ = ops.categorical_policy_loss(leaf, b, old, adv)
        (d,) = torch.autograd.grad(loss, leaf)
        assert loss.isnan() and d[5].isnan().all() and d[:5].isfinite().all() and d[6:].isfinite().all()
        with pytest.raises(IndexError):
            ops.check_policy_inputs(gpu_device)
        lp, ent = ops.categorical_log_probs(z, b)
        assert lp[5].isnan() and lp[:5].isfinite().all() and ent.isfinite().all()
        with pytest.raises(IndexError):
            ops.check_policy_inputs(gpu_device)
    ops.check_policy_inputs(gpu_device)


@pytest.mark.parametrize("K", [6, 300, 9000])
def test_nan_and_infinite_logits_show(K, gpu_device):
    """A NaN or +inf logit, or a row with no choice left, gives NaN in its own row and the loss, as torch does."""
    z, a, old, adv, _ = _loss_inputs(gpu_device, 9, K, torch.float32, 8)
    z[2, 1], z[4, K - 1], z[6] = float("nan"), float("inf"), -float("inf")
    a[4] = 0
    leaf = z.detach().requires_grad_()
    loss, _ = _ops().categorical_policy_loss(leaf, a, old, adv, entropy_coef=0.01)
    (d,) = torch.autograd.grad(loss, leaf)
    rows = torch.tensor([2, 4, 6], device=gpu_device)
    others = torch.tensor([0, 1, 3, 5, 7, 8], device=gpu_device)
    assert loss.isnan() and d[rows].isnan().any(1).all() and d[others].isfinite().all()
    lp, ent = _ops().categorical_log_probs(z, a)
    assert lp[rows].isnan().all() and ent[rows].isnan().all() and lp[others].isfinite().all()


def test_nan_and_infinite_logits_show_in_long_rows(gpu_device):
    test_nan_and_infinite_logits_show(30001, gpu_device)


def test_far_log_ratios_are_bounded(gpu_device):
    """Log-ratios beyond +-20 are held there, without gradient of their own."""
    z, a, old, adv, ref = _loss_inputs(gpu_device, 12, 9, torch.float32, 9)
    old[:4] -= 40.0
    old[4:8] += 40.0
    ref[2:6] += 50.0
    ref[6:9] -= 50.0
    _check_loss(z, a, old, adv.abs() * torch.tensor([1.0, -1.0], device=gpu_device).repeat(6), ref, None, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,lead", [(7, (4, 5)), (200, (3, 2, 3)), (6001, (5,))])
def test_strided_logits(K, lead, dtype, gpu_device):
    """Leading dimensions, and rows of a wider buffer at an odd offset."""
    M = int(torch.tensor(lead).prod())
    z, a, old, adv, ref = _loss_inputs(gpu_device, M, K, dtype, 21)
    wide = torch.zeros(M, K + 11, device=gpu_device, dtype=dtype)
    wide[:, 3:3 + K] = z
    s = float(M) if dtype == torch.float16 else 1.0
    loss, d = _check_loss(wide[:, 3:3 + K], a, old, adv, ref, None, None, s)
    leaf = z.view(*lead, K).requires_grad_()
    loss2, _ = _ops().categorical_policy_loss(leaf, a.view(lead), old.view(lead), adv.view(lead), clip=0.2,
                                              ref_log_probs=ref.view(lead), kl_coef=0.1, entropy_coef=0.02)
    (d2,) = torch.autograd.grad(loss2 * s, leaf)
    want = R.policy_loss(z, a, old, adv, ref, None, None, 0.8, 1.2, 0.1, 0.02, s)
    R.check(loss2, *want["loss"], "loss")
    R.check(d2.reshape(M, K), *want["d_logits"], "d_logits")
    cols = z.detach().t().contiguous().t()
    lp, ent = _ops().categorical_log_probs(cols, a)
    l, le, H, He, _, _ = R.rows_of(z, a)
    R.check(lp, l, le, "log_probs")
    R.check(ent, H, He, "entropy")


def test_logit_rows_beyond_32_bits(gpu_device):
    far, K = 2_300_000_000, 1000
    store = torch.empty(far + K, dtype=torch.bfloat16, device=gpu_device)
    z = store.as_strided((2, K), (far, 1))
    fresh, a, old, adv, ref = _loss_inputs(gpu_device, 2, K, torch.bfloat16, 22)
    z.copy_(fresh)
    _check_loss(z, a, old, adv, ref, None, None)


def test_loss_twice_and_scaled(gpu_device):
    """One graph walked twice, then with another incoming gradient: each gradient is its own."""
    z, a, old, adv, ref = _loss_inputs(gpu_device, 30, 3000, torch.bfloat16, 23)
    leaf = z.requires_grad_()
    loss, _ = _ops().categorical_policy_loss(leaf, a, old, adv, ref_log_probs=ref, kl_coef=0.1)
    (one,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = one.clone()
    (two,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device=gpu_device), retain_graph=True)
    (again,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(one, kept) and torch.equal(again, one) and torch.equal(two, one * 2)
    assert one.data_ptr() != two.data_ptr() != again.data_ptr()


# ------------------------------------------------------------------------------------------- together

def _policy(ops, p, x, state, keep, lengths, a, old, adv, ref, mask):
    """norm -> gates -> recurrence -> output, added to the stream -> norm -> logits -> loss."""
    n, T, D = x.shape
    y, stream = ops.residual_rms_norm(x, None, p["w1"])
    h, last = ops.gated_recurrence(y @ p["w_gates"].t(), state, keep, lengths)
    y, _ = ops.residual_rms_norm(h @ p["w_out"].t(), stream, p["w2"])
    loss, terms = ops.categorical_policy_loss(y @ p["w_head"].t(), a, old, adv, ref_log_probs=ref, kl_coef=0.1,
                                              entropy_coef=0.01, mask=mask)
    return loss + 0.01 * last.sum(), terms


def _policy_inputs(n, T, D, U, K):
    g = torch.Generator().manual_seed(31)
    p = {"w1": 1 + 0.1 * torch.randn(D, generator=g), "w_gates": torch.randn(3 * U, D, generator=g) / D ** 0.5,
         "w_out": torch.randn(D, U, generator=g) / U ** 0.5, "w2": 1 + 0.1 * torch.randn(D, generator=g),
         "w_head": torch.randn(K, D, generator=g) / D ** 0.5}
    x, state = torch.randn(n, T, D, generator=g), torch.randn(n, U, generator=g)
    keep = (torch.rand(n, T, generator=g) > 0.1).float()
    lengths = torch.randint(T // 2, T + 1, (n,), generator=g)
    a = torch.randint(0, K, (n, T), generator=g)
    old = -torch.log(torch.tensor(float(K))) + 0.3 * torch.randn(n, T, generator=g)
    adv, ref = torch.randn(n, T, generator=g), old + 0.1 * torch.randn(n, T, generator=g)
    mask = torch.arange(T)[None] < lengths[:, None]
    return p, (x, state, keep, lengths, a, old, adv, ref, mask)


def test_together_gradients(gpu_device):
    """A sequence policy's loss and all its gradients, float32 on the GPU against float64 on the CPU. A float32
    pass through five layers of sums of at most 96 terms stays within 300 half steps of each tensor's largest
    entry (5 layers x (96 / 2 + 12) roundings, forward and back, none of them amplified: every factor is of
    order one); rows near the loss's kinks are taken out of the mask in advance."""
    ops = _ops()
    p, data = _policy_inputs(4, 60, 48, 96, 40)
    p64 = {k: v.double().requires_grad_() for k, v in p.items()}
    d64 = [t.double() if t.is_floating_point() else t for t in data]
    with torch.no_grad():           # rows within 1e-3 of a clipping border, by the 64-bit pass
        n, T, D = d64[0].shape
        y, stream = ops.residual_rms_norm(d64[0], None, p64["w1"])
        h, _ = ops.gated_recurrence(y @ p64["w_gates"].t(), *d64[1:4])
        y, _ = ops.residual_rms_norm(h @ p64["w_out"].t(), stream, p64["w2"])
        l, _ = ops.categorical_log_probs(y @ p64["w_head"].t(), d64[4])
        r = (l - d64[5]).exp()
        data[8].logical_and_(((r - 0.8).abs() > 1e-3) & ((r - 1.2).abs() > 1e-3))
        d64[8] = data[8]
    x64, s64 = d64[0].requires_grad_(), d64[1].requires_grad_()
    loss64, _ = _policy(ops, p64, *d64)
    names = list(p) + ["x", "state"]
    want = torch.autograd.grad(loss64, list(p64.values()) + [x64, s64])
    pg = {k: v.to(gpu_device).requires_grad_() for k, v in p.items()}
    dg = [t.to(gpu_device) for t in data]
    dg[0].requires_grad_(), dg[1].requires_grad_()
    loss, _ = _policy(ops, pg, *dg)
    got = torch.autograd.grad(loss, list(pg.values()) + [dg[0], dg[1]])
    assert abs(float(loss) - float(loss64)) <= 300 * R.E * max(1.0, abs(float(loss64)))
    for name, a, b in zip(names, got, want):
        b = b.detach()
        assert float((a.cpu().double() - b).abs().max()) <= 300 * R.E * float(b.abs().max()), name


def test_not_differentiable_twice(gpu_device):
    """A graph of a gradient can be asked for, but not walked."""
    ops = _ops()
    x = torch.randn(4, 5, 24, device=gpu_device, requires_grad=True)
    w = torch.ones(24, device=gpu_device, requires_grad=True)
    a = torch.zeros(4, 5, dtype=torch.long, device=gpu_device)
    f = torch.zeros(4, 5, device=gpu_device)
    for call in (lambda: ops.gated_recurrence(x)[0].square().sum(), lambda: ops.residual_rms_norm(x, None, w)[0].square().sum(),
                 lambda: ops.categorical_policy_loss(x, a, f, f)[0]):
        (d,) = torch.autograd.grad(call(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            d.sum().backward()


def test_rollout_equals_sequence(gpu_device):
    """The step form, one decision after another in place, gives the sequence form's outputs."""
    ops = _ops()
    gates, state, keep, _, _, _ = _recurrence_inputs(gpu_device, 20, 90, 64, torch.float32, True, False, 33)
    ref = R.recurrence(gates, state, keep, None)
    c = state.clone()
    hs = []
    for t in range(90):
        h, c = ops.gated_recurrence_step(gates[:, t], c, keep[:, t - 1] if t else None, inplace=True)
        hs.append(h)
    R.check(torch.stack(hs, 1), *ref["h"], "h")
    R.check(c, *ref["last"], "last")


@pytest.mark.parametrize("U,K", [(16, 6), (128, 5000)])
def test_captured_step_replays(U, K, gpu_device):
    """Forward and backward of everything in one graph, replayed on new inputs, with eager work of the same
    operators between the replays, gives the eager results."""
    ops = _ops()
    p, data = _policy_inputs(3, 50, 32, U, K)
    pg = {k: v.to(gpu_device).requires_grad_() for k, v in p.items()}
    dg = [t.to(gpu_device) for t in data]
    leaves = list(pg.values())

    def step(args):
        loss, terms = _policy(ops, pg, *args)
        return [loss, terms] + list(torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        for _ in range(2):
            step(dg)
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(dg)
    for k in range(4):
        g = torch.Generator().manual_seed(50 + k)
        dg[0].copy_(torch.randn(dg[0].shape, generator=g))
        dg[3].copy_(torch.randint(1, 51, dg[3].shape, generator=g))
        graph.replay()
        torch.cuda.synchronize(gpu_device)
        got = [t.clone() for t in out]
        for a, b in zip(got, step(dg)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_captured_without_its_forward(dtype, gpu_device):
    """Every replay of a captured backward call forms the gradient anew, whatever became of the last one."""
    ops = _ops()
    z, a, old, adv, ref = _loss_inputs(gpu_device, 30, 900, dtype, 24)
    ops.categorical_log_probs(z, a)
    g = torch.ones((), device=gpu_device)
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        leaf = z.detach().clone().requires_grad_()
        loss, _ = ops.categorical_policy_loss(leaf, a, old, adv, ref_log_probs=ref, kl_coef=0.1)
    torch.cuda.synchronize(gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (d,) = torch.autograd.grad(loss, leaf, g, retain_graph=True)
    with torch.cuda.stream(side):
        for scale in (1.0, 2.0, 1.0, 1.0, -0.5):
            g.fill_(scale)
            d.fill_(7.0)
            graph.replay()
            (want,) = torch.autograd.grad(loss, leaf, g, retain_graph=True)
            side.synchronize()
            assert torch.equal(d, want)


def test_two_streams_at_once(gpu_device):
    """Calls that overlap on two streams do not share anything."""
    ops = _ops()
    p, data = _policy_inputs(3, 200, 32, 64, 700)
    pg = {k: v.to(gpu_device).requires_grad_() for k, v in p.items()}
    sets = []
    for k in range(2):
        dg = [t.to(gpu_device) for t in data]
        dg[0] = dg[0] * (k + 1)
        sets.append(dg)

    def step(args):
        loss, terms = _policy(ops, pg, *args)
        return [loss.detach(), terms] + list(torch.autograd.grad(loss, list(pg.values())))

    want = [step(s) for s in sets]
    torch.cuda.synchronize(gpu_device)
    streams = [torch.cuda.Stream(gpu_device) for _ in sets]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(s))
        torch.cuda.synchronize(gpu_device)
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_gpu_refusals(gpu_device):
    ops = _ops()
    z = lambda *s, **k: torch.zeros(*s, device=gpu_device, **k)  # noqa: E731
    bad = [lambda: ops.gated_recurrence(z(2, 3, 6, dtype=torch.float64)), lambda: ops.gated_recurrence(z(2, 3, 6), torch.zeros(2, 2)),
           lambda: ops.gated_recurrence(z(2, 3, 6), keep=torch.ones(2, 3)),
           lambda: ops.gated_recurrence_step(z(2, 6, dtype=torch.float64), z(2, 2)),
           lambda: ops.residual_rms_norm(z(2, 4, dtype=torch.float64)), lambda: ops.residual_rms_norm(z(2, 4), torch.zeros(2, 4)),
           lambda: ops.residual_rms_norm(z(2, 4, dtype=torch.bfloat16), weight=z(4)),
           lambda: ops.categorical_log_probs(z(2, 4), torch.zeros(2, dtype=torch.long)),
           lambda: ops.categorical_policy_loss(z(2, 4), z(2).long(), z(2), z(2), denom=z((), dtype=torch.float64)),
           lambda: ops.categorical_policy_loss(z(2, 4), z(2).long(), z(2, dtype=torch.float64), z(2))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
