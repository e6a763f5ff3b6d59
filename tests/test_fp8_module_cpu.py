"""The 8-bit layer's module without a GPU: when it builds its weight's 8-bit form and what it keeps of it. Launches are
counted in place of being made, streams are numbers, and the tensors (never filled) are in host memory."""

from __future__ import annotations

import pytest
import torch

BUILD = "mxq_fp8_quantize_tiles"


@pytest.fixture
def host(monkeypatch):
    """The module's calls into the library as a list of names."""
    from mx_qlinear import fp8

    calls = []
    monkeypatch.setattr(fp8, "_launch", lambda dev, name, *args: calls.append(name))
    monkeypatch.setattr(fp8, "_require_gpu", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(fp8, "_workspace", lambda *args: 0)
    monkeypatch.setattr(fp8, "_capturing", lambda device: False)
    return calls


def _layer(frozen=True, **kw):
    from mx_qlinear import Fp8Linear

    layer = Fp8Linear(256, 96, dtype=torch.bfloat16, **kw)
    return layer.requires_grad_(not frozen)


def test_a_form_built_in_inference_mode_serves_a_later_backward_pass(host):
    layer = _layer()
    with torch.inference_mode():
        layer(torch.zeros(4, 256, dtype=torch.bfloat16))
    x = torch.zeros(4, 256, dtype=torch.bfloat16, requires_grad=True)
    layer(x).float().sum().backward()
    assert x.grad.shape == x.shape
    assert host.count(BUILD) == 1
