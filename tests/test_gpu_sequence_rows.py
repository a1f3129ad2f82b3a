"""Sequence-policy operators with more rows than a launch has places for: a workgroup's second turn, counted masks, sums
over several rows of a thread, joined by many workgroups."""

import pytest
import torch

import sequence_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from SwarmACB_isaac.agents import sequence_ops

    return sequence_ops


# ------------------------------------------------------------------------------------- the policy loss

def _loss_inputs(dev, M, K, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = (2 * torch.randn(M, K, device=dev, generator=g)).to(dtype)
    a = torch.randint(0, K, (M,), device=dev, generator=g)
    l = z.gather(1, a[:, None])[:, 0].float() - torch.logsumexp(z.float(), 1)
    shift = 0.3 * torch.randn(M, device=dev, generator=g)
    for border in (0.8, 1.2):        # off the kinks by far more than any rounding
        b = torch.tensor(border).log().item()
        shift = torch.where((shift - b).abs() < 0.01, torch.full_like(shift, b + 0.02), shift)
    mask = torch.rand(M, device=dev, generator=g) < 0.7
    return (z, a, l - shift, torch.randn(M, device=dev, generator=g), l + 0.3 * torch.randn(M, device=dev, generator=g), mask)


def _call(z, a, old, adv, ref, mask, denom, grads):
    """(loss, terms, one gradient for each of the incoming ones, in their order on one graph)"""
    leaf = z.detach().requires_grad_()
    loss, terms = _ops().categorical_policy_loss(leaf, a, old, adv, clip=0.2, ref_log_probs=ref, kl_coef=0.1,
                                                 entropy_coef=0.02, mask=mask, denom=denom)
    ds = [torch.autograd.grad(loss, leaf, torch.tensor(float(g), device=z.device), retain_graph=True)[0] for g in grads]
    return loss.detach(), terms, ds


def _reference(z, a, old, adv, ref, mask, n, grads, part):
    """The reference over parts of the rows, which bounds its memory: (loss, terms, gradients), each with its bound."""
    M, total, ds = z.shape[0], None, [[] for _ in grads]
    for r in range(0, M, part):
        s = slice(r, r + part)
        for k, g in enumerate(grads):
            want = R.policy_loss(z[s], a[s], old[s], adv[s], ref[s], mask[s], n, 0.8, 1.2, 0.1, 0.02, float(g))
            ds[k].append(want["d_logits"])
        here = [want["loss"], want["terms"]]
        total = here if total is None else [tuple(x + y for x, y in zip(p, q)) for p, q in zip(total, here)]
    return total[0], total[1], [tuple(torch.cat(x) for x in zip(*d)) for d in ds]


# A row takes 1, 4 and 8 lanes, part of a wave, a wave, two waves, a workgroup, a workgroup with LDS; rows of the last
# size are gathered in one pass, and the last two sizes of float32 spill.
@pytest.mark.parametrize("M,K,dtype", [
    (20001, 18, torch.float32), (20001, 18, torch.bfloat16), (66001, 6, torch.float32),            # counted masks
    (140003, 18, torch.float32), (140003, 50, torch.float16), (600011, 6, torch.bfloat16),        # second turns
    (70001, 130, torch.float32), (18001, 900, torch.bfloat16), (9001, 2048, torch.float32),
    (2101, 4097, torch.bfloat16), (2101, 4097, torch.float32), (2101, 9000, torch.bfloat16)])
def test_loss_of_many_rows(M, K, dtype, gpu_device):
    z, a, old, adv, ref, mask = _loss_inputs(gpu_device, M, K, dtype, M + K)
    n = int(mask.sum())
    scale = float(n * min(K, 1024)) if dtype == torch.float16 else 1.0
    grads = (scale, 0.5 * scale)
    loss, terms, ds = _call(z, a, old, adv, ref, mask, None, grads)
    want_loss, want_terms, want_ds = _reference(z, a, old, adv, ref, mask, float(n), grads, max(64, 4_000_000 // K))
    R.check(loss, *want_loss, "loss")
    R.check(terms, *want_terms, "terms")
    for d, want, g in zip(ds, want_ds, grads):
        R.check(d, *want, f"d_logits of {g}")


@pytest.mark.parametrize("M,K,dtype", [
    (2300, 16385, torch.bfloat16), (2300, 33000, torch.bfloat16), (2300, 9000, torch.float32), (2300, 20000, torch.float32),
    (2200, 70001, torch.bfloat16), (2200, 40000, torch.float32), (2300, 16385, torch.float16)])
def test_loss_of_many_long_rows(M, K, dtype, gpu_device):
    """Rows of a second turn and those before it equal the same rows alone, bit by bit; those around the border are
    checked themselves."""
    z, a, old, adv, ref, mask = _loss_inputs(gpu_device, M, K, dtype, M + K)
    mask[2040:2060] = torch.arange(20, device=gpu_device) % 3 != 0       # active and inactive ones on both sides
    n = mask.sum().float()
    scale = float(M * 1024) if dtype == torch.float16 else 1.0
    grads = (scale, 0.5 * scale)
    loss, terms, ds = _call(z, a, old, adv, ref, mask, None, grads)
    parts = []
    for r in range(0, M, 500):
        s = slice(r, r + 500)
        parts.append(_call(z[s], a[s], old[s], adv[s], ref[s], mask[s], n, grads))
        for d, alone in zip(ds, parts[-1][2]):
            assert torch.equal(d[s], alone), f"rows from {r} on"
        for d in ds:
            assert not d[s][~mask[s]].any()
    R.check(loss, sum(p[0] for p in parts).double().cpu(), 64 * R.E * sum(p[0].abs() for p in parts).double().cpu() + 64 * R.E, "loss")
    R.check(terms, sum(p[1] for p in parts).double().cpu(), 64 * R.E * sum(p[1].abs() for p in parts).double().cpu() + 64 * R.E, "terms")
    for s in (slice(0, 12), slice(2040, 2060), slice(M - 12, M)):
        for g, d in zip(grads, ds):
            want = R.policy_loss(z[s], a[s], old[s], adv[s], ref[s], mask[s], float(n), 0.8, 1.2, 0.1, 0.02, g)
            R.check(d[s], *want["d_logits"], f"d_logits of {g}")


@pytest.mark.parametrize("M", [1, 15, 16, 17, 65537, 262_147])
def test_masks_are_counted(M, gpu_device):
    """The number of active rows, whichever kernel counts it and wherever the mask begins: exact in every case."""
    for K in (2, 18):
        for offset in (0, 1, 7):
            g = torch.Generator(device=gpu_device).manual_seed(M + offset)
            mask = (torch.rand(M + offset, device=gpu_device, generator=g) < 0.6)[offset:]
            z = torch.zeros(M, K, device=gpu_device, requires_grad=True)
            row = torch.zeros(M, device=gpu_device)
            # every active row has r = 1 and A = -1, so its gradient at the action is (1 - 1 / K) / active rows
            old = torch.full((M,), -float(torch.tensor(float(K)).log()), device=gpu_device)
            loss, _ = _ops().categorical_policy_loss(z, row.long(), old, row - 1.0, mask=mask)
            (d,) = torch.autograd.grad(loss, z)
            n = max(1, int(mask.sum()))
            want = torch.where(mask, (1 - 1 / K) / n, 0.0).double().cpu()
            assert not (d[:, 0].double().cpu() - want).abs().gt(16 * R.E * want).any()


# ------------------------------------------------------------------------------------------- the norm

# A workgroup of the backward pass takes these many rows at a time, and a launch has these many workgroups at most.
def _shape(D, dtype):
    if D < 16 // dtype.itemsize:
        return 256, 1024
    for most, rows, blocks in ((32, 64, 1024), (128, 16, 1024), (512, 4, 1024), (1024, 1, 2048), (2048, 1, 1024),
                               (4096, 1, 512), (16384, 1, 256)):
        if D <= most:
            return rows, blocks
    return 1, 1024


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(1_000_003, 3), (300_000, 7), (70_001, 5), (140_001, 24), (40_001, 100), (9_001, 300),
                                    (4_500, 512), (4_301, 1001), (2_100, 2000), (1_501, 4096), (700, 8000), (600, 16384),
                                    (2_200, 17000)])
def test_weight_gradient_of_many_rows(rows, D, dtype, gpu_device):
    """The sum over rows, against the longest chain of additions that it is formed by: a thread's rows, a workgroup's
    threads, a thirty-second of the workgroups, the last 32. Leaving out one workgroup's rows, or any one of them being
    counted twice, shows: their share is four times the bound and more."""
    g = torch.Generator(device=gpu_device).manual_seed(rows + D)
    x, r, dy, ds = (torch.randn(rows, D, device=gpu_device, generator=g).to(dtype) for _ in range(4))
    w = (1 + 0.3 * torch.randn(D, device=gpu_device, generator=g)).to(dtype).requires_grad_()
    xl = x.requires_grad_()
    y, s = _ops().residual_rms_norm(xl, r, w, eps=1e-5)
    dx, dw = torch.autograd.grad((y, s), (xl, w), (dy, ds))
    want = R.norm(x, r, w, 1e-5, dy, ds)
    R.check(y, *want["y"], "y")
    R.check(s, *want["stream"], "stream")
    R.check(dx, *want["dx"], "dx")
    at_once, most = _shape(D, dtype)
    count = min(-(-rows // at_once), most)
    chain = -(-rows // (at_once * count)) + min(at_once, 64) + count / 32 + 32
    n = x.detach().double().cpu() + r.double().cpu()
    n = n / torch.sqrt((n * n).mean(1, keepdim=True) + 1e-5)
    size = (dy.double().cpu() * n).abs().sum(0)
    value = want["dw"][0]
    # of every term: the sum's rounding, rstd (half the row sum's error and a few of its own), two products
    bound = ((D / 64 + 28) + chain) * R.E * size + R.rounding(value, dtype)
    share = (rows / count) ** 0.5         # of a workgroup's rows, terms of size 1 and either sign
    accumulated = bound - R.rounding(value, dtype)
    assert 4 * float(accumulated.max()) < share * (1 if rows > count else 4), "the bound would hide a workgroup"
    R.check(dw, value, bound, "dw")
