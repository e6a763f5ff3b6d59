"""The 8-bit layer's module without a GPU: when it builds its weight's 8-bit form and what it keeps of it. Launches are
counted in place of being made, streams are numbers, and the tensors (never filled) are in host memory."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch

BUILD = "mxq_fp8_quantize_tiles"


class _Calls(list):
    pass


@pytest.fixture
def host(monkeypatch):
    """The module's calls into the library as a list of names."""
    from mx_qlinear import fp8

    calls = _Calls()
    monkeypatch.setattr(fp8, "_launch", lambda dev, name, *args: calls.append(name))
    monkeypatch.setattr(fp8, "_require_gpu", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(fp8, "_workspace", lambda *args: 0)
    monkeypatch.setattr(fp8, "_capturing", lambda device: calls.capturing)
    monkeypatch.setattr(fp8, "_synchronize", lambda device: calls.append("synchronize"), raising=False)
    calls.stream, calls.follows, calls.capturing = 0, [], False
    monkeypatch.setattr(fp8, "_raw_stream", lambda index: calls.stream, raising=False)
    monkeypatch.setattr(fp8, "_event", lambda device: ("built on", calls.stream), raising=False)
    monkeypatch.setattr(fp8, "_follow", lambda device, event, tensors: calls.follows.append((calls.stream, event, len(tensors))),
                        raising=False)
    return calls


def _layer(frozen=True, **kw):
    from mx_qlinear import Fp8Linear

    layer = Fp8Linear(256, 96, **{"dtype": torch.bfloat16, **kw})
    return layer.requires_grad_(not frozen)


def test_a_form_built_in_inference_mode_serves_a_later_backward_pass(host):
    layer = _layer()
    with torch.inference_mode():
        layer(torch.zeros(4, 256, dtype=torch.bfloat16))
    x = torch.zeros(4, 256, dtype=torch.bfloat16, requires_grad=True)
    layer(x).float().sum().backward()
    assert x.grad.shape == x.shape
    assert host.count(BUILD) == 1


def test_another_stream_waits_for_the_build(host):
    """A call on a stream that did not build the form waits for the build and holds the form's four tensors; the builder's
    own calls do neither."""
    layer, x = _layer(), torch.zeros(4, 256, dtype=torch.bfloat16)
    with torch.no_grad():
        host.stream = 5
        layer(x)
        layer(x)
        assert host.count(BUILD) == 1 and host.follows == []
        host.stream = 7
        layer(x)
        layer(x)
        assert host.count(BUILD) == 1 and host.follows == [(7, ("built on", 5), 4)] * 2
        layer.weight.mul_(2)
        layer(x)
        assert host.count(BUILD) == 2 and len(host.follows) == 2
        host.stream = 5
        layer(x)
        assert host.follows[2:] == [(5, ("built on", 7), 4)]
    host.stream = 9
    layer(x.clone().requires_grad_())  # (the input's gradient alone)
    assert host.count(BUILD) == 2 and host.follows[3:] == [(9, ("built on", 7), 4)]


def test_copies_and_pickles_leave_the_form_behind(host):
    layer, x = _layer(), torch.zeros(4, 256, dtype=torch.bfloat16)
    layer(x)
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
        assert other._prepared is None and layer._prepared is not None
        assert torch.equal(other.weight, layer.weight)
        other(x)
    assert host.count(BUILD) == 3
    # a pickle of the layer that held the form as an attribute
    old = layer.__getstate__()
    del old["_kept"]
    other = type(layer).__new__(type(layer))
    other.__setstate__({**old, "_prepared": layer._prepared, "_prepared_of": None})
    assert other._prepared is None
    other(x)
    assert host.count(BUILD) == 4


def _pointers(layer):
    f = layer._prepared
    return [t.data_ptr() for t in (f.q, f.scale, f.qt, f.scale_t)]


def test_a_captured_call_builds_its_own_form_unless_asked_before(host):
    """Whether an eager call came first changes nothing: the form is the graph's own, or the one that was asked for."""
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    for eager in (False, True):
        layer = _layer()
        if eager:
            layer(x)
        kept = layer._prepared
        host.capturing = True
        del host[:]
        layer(x)
        host.capturing = False
        assert host.count(BUILD) == 1 and layer._prepared is kept
    layer.prepare()
    host.capturing = True
    del host[:]
    layer(x)
    assert host.count(BUILD) == 0 and host.follows == []
    layer.weight.mul_(2)  # (no longer the weight's)
    layer(x)
    assert host.count(BUILD) == 1
    with pytest.raises(RuntimeError, match="prepare"):
        layer.prepare()


def test_what_a_graph_reads_stays_in_place(host):
    """The memory of a form that a graph reads is neither given back nor moved: later contents are written into it, between
    two synchronizations, and a form that no longer fits is held."""
    layer, x = _layer().prepare(), torch.zeros(4, 256, dtype=torch.bfloat16)
    host.capturing = True
    layer(x)
    host.capturing = False
    at, form = _pointers(layer), layer._prepared
    for change in (lambda: layer.weight.mul_(2), lambda: layer.load_state_dict(layer.state_dict()), layer.float,
                   lambda: setattr(layer, "weight", torch.nn.Parameter(layer.weight.detach() + 1, requires_grad=False))):
        change()
        del host[:]
        layer(x)
        assert host[:3] == ["synchronize", BUILD, "synchronize"]
        assert layer._prepared is form and _pointers(layer) == at
    layer.prepare()
    assert layer._prepared is form and _pointers(layer) == at
    layer.weight = torch.nn.Parameter(torch.zeros(100, 256), requires_grad=False)
    layer.prepare()
    assert layer._prepared is not form and layer._kept.held == (form,)


def test_a_backward_pass_refuses_a_form_that_was_written_over(host):
    """A form that a graph reads is written in place: a backward pass that saved it before does not run on other contents."""
    layer = _layer(bias=False).prepare()
    host.capturing = True
    layer(torch.zeros(4, 256, dtype=torch.bfloat16))
    host.capturing = False
    x = torch.zeros(4, 256, dtype=torch.bfloat16, requires_grad=True)
    y = layer(x)
    layer.weight.mul_(2)
    layer(x.detach())
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.float().sum().backward()
    layer(x).float().sum().backward()


@pytest.mark.parametrize("optimizer", [torch.optim.AdamW, torch.optim.SGD])
def test_a_trainable_weight_is_read_anew_by_every_call(host, optimizer):
    """A fused optimizer changes the parameter without counting it."""
    # (float32: of bfloat16 parameters in host memory torch's fused SGD leaves whole vectors as they are)
    layer, x = _layer(frozen=False, dtype=torch.float32), torch.zeros(4, 256, dtype=torch.bfloat16)
    step = optimizer(layer.parameters(), lr=0.1, fused=True)
    with torch.no_grad():
        layer(x)
    before, state = layer.weight.detach().clone(), layer._state()
    layer.weight.grad, layer.bias.grad = torch.ones_like(layer.weight), torch.ones_like(layer.bias)
    step.step()
    assert not torch.equal(layer.weight, before)
    assert layer._state()[1:] == state[1:], "counted after all: the rule can be looser"
    with torch.no_grad():
        for calls in (2, 3):
            layer(x)
            assert host.count(BUILD) == calls
        form = layer._form()
        assert layer._form() is form and host.count(BUILD) == 5  # (the same memory, written anew)
        assert form.qt is None  # (which only the input's gradient of a frozen layer reads)
    # asked for, it is kept: up to the next forward with gradients, and train() or eval()
    for end in (lambda: layer(x), layer.eval, layer.train, lambda: layer.weight.detach().mul_(2),
                lambda: layer.load_state_dict(layer.state_dict())):
        layer.prepare()
        del host[:]
        with torch.no_grad():
            layer(x)
            layer(x)
        assert host.count(BUILD) == 0
        end()
        del host[:]
        with torch.no_grad():
            layer(x)
        assert host.count(BUILD) == 1
    # frozen after training without a counted change
    layer.requires_grad_(False)
    layer(x)
    layer.requires_grad_(True)
    layer(x)
    layer.requires_grad_(False)
    del host[:]
    layer(x)
    layer(x)
    assert host.count(BUILD) == 1


def test_a_frozen_weight_is_read_anew_once_it_may_have_changed(host):
    layer, x = _layer(), torch.zeros(4, 256, dtype=torch.bfloat16)
    layer(x)
    layer(x)
    assert host.count(BUILD) == 1
    w = layer.weight
    # the state before and after a type and back can be the same: a layer of one value, rounded by it
    for change in (lambda: w.add_(1), lambda: layer.load_state_dict(layer.state_dict()), lambda: layer.float().bfloat16(),
                   layer.half, layer.eval, lambda: setattr(layer, "weight", torch.nn.Parameter(w.detach() + 1, False))):
        change()
        del host[:]
        layer(x.to(layer.weight.dtype))
        layer(x.to(layer.weight.dtype))
        assert host.count(BUILD) == 1
    layer.prepare()
    layer.eval()
    del host[:]
    layer(x.half())
    assert host.count(BUILD) == 0


def test_a_weight_of_inference_mode_is_read_anew_by_every_call(host):
    with torch.inference_mode():
        layer, x = _layer(), torch.zeros(4, 256, dtype=torch.bfloat16)
        assert layer.weight.is_inference()
        layer(x)
        layer.weight.mul_(2)
        layer(x)
        assert host.count(BUILD) == 2
        layer.prepare()
        layer(x)
        assert host.count(BUILD) == 3
        layer.load_state_dict({k: v * 2 for k, v in layer.state_dict().items()})
        layer(x)
        assert host.count(BUILD) == 4


def test_memory_that_others_read_is_not_written_over(host):
    """A form that another stream or a backward pass reads is replaced, not written anew."""
    layer = _layer(bias=False)
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    layer(x)
    first = layer._prepared
    layer.weight.mul_(2)
    layer(x)
    assert layer._prepared is first
    y = layer(x.clone().requires_grad_())
    layer.weight.mul_(2)
    layer(x)
    second = layer._prepared
    assert second is not first
    y.float().sum().backward()
    host.stream = 3
    layer(x)
    host.stream = 0
    layer.weight.mul_(2)
    layer(x)
    third = layer._prepared
    assert third is not second
    host.stream = 3
    layer.weight.mul_(2)
    layer(x)
    assert layer._prepared is not third


def test_a_moved_layer_gives_its_form_back(host):
    layer, x = _layer(), torch.zeros(4, 256, dtype=torch.bfloat16)
    layer(x)
    layer.to(torch.float16)
    assert layer._prepared is None


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("dual", ["x", "weight", "bias"])
@pytest.mark.parametrize("name", ["Fp8Linear", "LayerNorm"])
def test_forward_mode_is_refused(host, name, dual, requires_grad):
    """A tangent is carried on or refused, never dropped."""
    import mx_qlinear
    from torch.autograd import forward_ad

    module = mx_qlinear.Fp8Linear(256, 96) if name == "Fp8Linear" else mx_qlinear.LayerNorm(256)
    module.requires_grad_(requires_grad)
    args = {"x": torch.zeros(4, 256), "weight": module.weight, "bias": module.bias}
    with forward_ad.dual_level():
        args[dual] = forward_ad.make_dual(args[dual].detach(), torch.ones_like(args[dual]))
        with pytest.raises(RuntimeError, match="forward mode"):
            torch.func.functional_call(module, {k: args[k] for k in ("weight", "bias")}, args["x"])
    params = {"weight": module.weight, "bias": module.bias}
    args["x"] = torch.zeros(4, 256)
    start = {**args, **params}[dual].detach().clone()
    with pytest.raises(RuntimeError, match="forward mode"):
        torch.func.jvp(lambda t: torch.func.functional_call(module, {**params, dual: t} if dual != "x" else params, t if dual == "x" else args["x"]),
                       (start,), (torch.ones_like(start),))


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", ["Fp8Linear", "LayerNorm"])
def test_host_tensors_are_refused_by_name(name, requires_grad):
    import mx_qlinear

    module = mx_qlinear.Fp8Linear(256, 96) if name == "Fp8Linear" else mx_qlinear.LayerNorm(256)
    module.requires_grad_(requires_grad)
    with pytest.raises(RuntimeError, match="GPU only"):
        module(torch.zeros(4, 256))
    if name == "Fp8Linear":
        with pytest.raises(RuntimeError, match="GPU only"):
            module.prepare()


def test_memory_written_anew_on_another_stream_is_still_held(host):
    """A form that a graph reads can be written anew on a stream that did not allocate it: that stream's calls hold it too."""
    layer, x = _layer().prepare(), torch.zeros(4, 256, dtype=torch.bfloat16)
    host.capturing = True
    layer(x)
    host.capturing = False
    host.stream = 7
    layer.weight.mul_(2)
    form = layer._prepared
    layer(x)
    layer(x)
    assert layer._prepared is form and host.follows == [(7, ("built on", 7), 4)] * 2
