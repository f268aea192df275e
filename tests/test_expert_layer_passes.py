"""What passes of a layer with experts leave for one another: backward() takes the buffers of the kept pass just before it, or raises."""
import contextlib

import pytest


def _on_the_host(monkeypatch):
    """The layer with its buffers in host memory and calls that do nothing"""
    import torch

    import rocwmma_amd as R
    from rocwmma_amd import expert_layer

    monkeypatch.setattr(expert_layer, "_on", lambda stream: contextlib.nullcontext())
    for name in ("empty", "arange", "Generator"):
        made = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, _made=made, device=None, **kw: _made(*a, **kw))
    for name in ("linear", "linear_backward", "route", "route_backward", "combine", "dispatch"):
        monkeypatch.setattr(R, name, lambda *a, **kw: None)
    monkeypatch.setattr(R, "_index", lambda name, t, size, count: R._ptr(t))  # (that would want them in device memory)


def _refused_passes():
    import torch

    from rocwmma_amd.expert_layer import ExpertLayer

    layer = ExpertLayer(64, 32, 8, 2, "f16")
    layer.reserve(12, training=True)
    x = torch.randn(12, 64).to(layer.router.device).half()
    dy = torch.ones_like(x)
    with pytest.raises(ValueError):  # no pass
        layer.backward(x, dy)
    layer.forward(x)
    with pytest.raises(ValueError):  # one that was not kept
        layer.backward(x, dy)
    layer.forward(x, keep=True)
    layer.backward(x, dy)
    layer.backward(x, dy)  # (again: nothing that it reads was written to)
    layer.forward(x[:5].contiguous())
    with pytest.raises(ValueError):  # another pass since
        layer.backward(x, dy)
    layer.forward(x[:5].contiguous(), keep=True)
    with pytest.raises(ValueError):  # of other tokens
        layer.backward(x, dy)
    layer.backward(x[:5].contiguous(), dy[:5].contiguous())
    layer.forward(x, keep=True)
    with pytest.raises(ValueError):  # a pass that is refused leaves the kept one
        layer.forward(x.float())
    layer.backward(x, dy)
    layer.reserve(12, training=True)
    with pytest.raises(ValueError):  # new buffers
        layer.backward(x, dy)


def test_refused_passes(monkeypatch):
    _on_the_host(monkeypatch)
    _refused_passes()


@pytest.mark.gpu
def test_refused_passes_on_the_gpu():
    _refused_passes()
