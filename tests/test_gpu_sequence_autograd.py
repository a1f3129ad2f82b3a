"""What torch's autograd has to see of the sequence-policy operators on the GPU, as it does on the CPU."""

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
