"""What torch's autograd has to see of the sequence-policy operators on the GPU, as it does on the CPU: writes in place,
forward-mode derivatives, traces."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from SwarmACB_isaac.agents import sequence_ops

    return sequence_ops


@pytest.mark.parametrize("device", ["cpu", "gpu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_in_place_is_seen(dtype, device, gpu_device):
    """A state that another operation saved for its backward pass cannot be overwritten unnoticed."""
    dev = gpu_device if device == "gpu" else torch.device("cpu")
    gates, state = torch.randn(5, 12, device=dev).to(dtype), torch.randn(5, 4, device=dev)
    w = torch.ones(5, 4, device=dev, requires_grad=True)
    for view in (False, True):
        saved = state[None] if view else state
        v, before = (saved * w).sum(), state._version
        _ops().gated_recurrence_step(gates, state)
        assert state._version == before
        torch.autograd.grad(v, w, retain_graph=True)
        _, out = _ops().gated_recurrence_step(gates, state, inplace=True)
        assert out is state and state._version > before
        with pytest.raises(RuntimeError, match="inplace operation"):
            v.backward()


def test_a_step_in_place_without_a_version(gpu_device):
    """Tensors made in inference mode, which nothing can save, have none."""
    with torch.inference_mode():
        gates, state = torch.randn(5, 12, device=gpu_device), torch.randn(5, 4, device=gpu_device)
        want = _ops().gated_recurrence_step(gates, state)[1].clone()
        assert torch.equal(_ops().gated_recurrence_step(gates, state.clone(), inplace=True)[1], want)
    with torch.no_grad():
        assert torch.equal(_ops().gated_recurrence_step(gates, state, inplace=True)[1], want)


def _calls(ops, dev):
    """{name: (function of one float operand, that operand)} for every float operand of every operator."""
    z = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    gates, state, keep, x, w = z(2, 3, 12), z(2, 4), torch.ones(2, 3, device=dev), z(6, 8), z(8)
    a, row = torch.zeros(6, dtype=torch.long, device=dev), z(6)
    loss = lambda logits=x, old=row, adv=row, ref=row, denom=None: ops.categorical_policy_loss(  # noqa: E731
        logits, a, old, adv, ref_log_probs=ref, kl_coef=0.1, denom=denom)
    return {
        "scan gates": (lambda t: ops.gated_recurrence(t, state, keep), gates),
        "scan state": (lambda t: ops.gated_recurrence(gates, t, keep), state),
        "scan keep": (lambda t: ops.gated_recurrence(gates, state, t), keep),
        "step gates": (lambda t: ops.gated_recurrence_step(t, state), gates[:, 0]),
        "step state": (lambda t: ops.gated_recurrence_step(gates[:, 0], t), state),
        "step keep": (lambda t: ops.gated_recurrence_step(gates[:, 0], state, t), keep[:, 0]),
        "norm x": (lambda t: ops.residual_rms_norm(t, x, w), x),
        "norm residual": (lambda t: ops.residual_rms_norm(x, t, w), x),
        "norm weight": (lambda t: ops.residual_rms_norm(x, None, t), w),
        "loss logits": (lambda t: loss(logits=t), x),
        "loss old": (lambda t: loss(old=t), row),
        "loss advantages": (lambda t: loss(adv=t), row),
        "loss ref": (lambda t: loss(ref=t), row),
        "loss denom": (lambda t: loss(denom=t), torch.tensor(3.0, device=dev)),
        "log_probs": (lambda t: ops.categorical_log_probs(t, a), x),
    }


NAMES = ["scan gates", "scan state", "scan keep", "step gates", "step state", "step keep", "norm x", "norm residual",
         "norm weight", "loss logits", "loss old", "loss advantages", "loss ref", "loss denom", "log_probs"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, gpu_device):
    """A dual tensor's derivative is not dropped: the CPU form carries it on, the kernels refuse it."""
    import torch.autograd.forward_ad as fa

    for dev in (torch.device("cpu"), gpu_device):
        call, t = _calls(_ops(), dev)[name]
        call(t)
        with fa.dual_level():
            dual = fa.make_dual(t, torch.ones_like(t))
            if dev.type == "cpu":
                assert any(fa.unpack_dual(r).tangent is not None for r in call(dual))
                continue
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            call(fa.unpack_dual(dual).primal)
        call(t)


@pytest.mark.parametrize("name", ["scan gates", "step gates", "norm x", "loss logits", "log_probs"])
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traces_are_refused(name, gpu_device):
    """A trace would record the empty tensors that the kernels write."""
    call, t = _calls(_ops(), gpu_device)[name]
    call(t)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda x: call(x)[0], t, check_trace=False)
    call(t)


@pytest.mark.parametrize("name", ["scan gates", "norm x", "loss logits"])
def test_function_transforms_raise(name, gpu_device):
    call, t = _calls(_ops(), gpu_device)[name]
    for transform in (lambda f: torch.func.grad(lambda x: f(x).sum()), torch.vmap,
                      lambda f: lambda x: torch.func.jvp(f, (x,), (torch.ones_like(x),))):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            transform(lambda x: call(x)[0])(t[None] if transform is torch.vmap else t)
