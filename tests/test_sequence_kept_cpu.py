"""CPU: a dense layer that keeps its input in 8 bits does so only where gradients are recorded."""
import pytest
import torch

from slayerpytorch_b200 import layer

NEURON = {"type": "SRMALPHA", "theta": 10, "tauSr": 10.0, "tauRef": 1.0, "scaleRef": 2, "tauRho": 1, "scaleRho": 1}


@pytest.mark.parametrize("off", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_evaluation_is_the_plain_layer(off, dtype, monkeypatch):
    """Any input that the plain layer takes, on any device."""
    net = layer.spikeLayer(NEURON, {"Ts": 1.0, "tSample": 30})
    dense, plain = net.dense((4, 4, 2), 3, checkpoint=True).to(dtype), net.dense((4, 4, 2), 3).to(dtype)
    plain.load_state_dict(dense.state_dict())
    x = torch.randn(2, 2, 4, 4, 6, dtype=dtype)
    calls = []
    compress = layer.slayerCuda.compress8
    monkeypatch.setattr(layer.slayerCuda, "compress8", lambda x: calls.append(x) or compress(x))
    with off():
        assert torch.equal(dense(x), plain(x)) and not calls
        with pytest.raises(ValueError, match="inputs of its own size"):
            dense(torch.zeros(1, 2, 5, 4, 6, dtype=dtype))
    with pytest.raises(RuntimeError, match="CUDA"):
        dense(x)
    assert len(calls) == 1
    dense.weight.requires_grad_(False)      # nothing to keep
    assert torch.equal(dense(x), plain(x)) and len(calls) == 1
