"""The gradient of a layer with experts with respect to its input is one sum, rounded once."""
import pytest

EPS = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,half", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
@pytest.mark.parametrize("tokens,reserved,top,how", [(1, 1, 3, None), (40, 40, 1, "stream"), (64, 300, 6, "handle"), (257, 300, 2, None)])
def test_parts_are_summed_in_f32(dtype, half, tokens, reserved, top, how):
    """Of 2 top + 2 terms: f32 sums in any order, (2 top + 2) eps sum |terms|, rounded to half a step"""
    import torch

    from rocwmma_amd.expert_layer import ExpertLayer

    torch.manual_seed(tokens)
    layer = ExpertLayer(136, 72, 11, top, dtype, seed=tokens)
    layer.reserve(reserved, training=True)
    x, dy = (torch.randn(tokens, 136, device="cuda").to(layer.torch_type) for _ in range(2))
    side = torch.cuda.Stream()
    stream = {None: None, "stream": side, "handle": side.cuda_stream}[how]
    torch.cuda.synchronize()
    layer.forward(x, keep=True, stream=stream)
    dx = layer.backward(x, dy, stream=stream)
    torch.cuda.synchronize()
    at = layer.place[:tokens].long()
    terms = torch.cat([dy[:, None].double(), layer.dxs.double()[at], layer.dxs2.double()[at], layer.dx_router[:tokens, None].double()], 1)
    want, err = terms.sum(1), (2 * top + 2) * EPS * terms.abs().sum(1)
    off, far = (dx.double() - want).abs(), err + half * (want.abs() + err) + 2.0 ** -25
    assert (off <= far).all(), (off / far).max().item()


def test_streams(monkeypatch):
    """None is the default stream, a number a stream's handle"""
    import torch

    from rocwmma_amd import expert_layer

    class Stream:
        pass

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "default_stream", Stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle: ("external", handle))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
    mine = Stream()
    assert expert_layer._on(mine) is mine and isinstance(expert_layer._on(None), Stream) and expert_layer._on(77) == ("external", 77)
    other = type("Other", (), {"cuda_stream": 78})()  # (as the calls take it)
    assert expert_layer._on(other) == ("external", 78)
