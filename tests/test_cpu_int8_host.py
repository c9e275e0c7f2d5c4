"""What humanrf_amd.int8's modules hold and hand to the product, on the CPU: the library's calls are replaced, nothing is launched."""
import contextlib

import pytest
import torch


@pytest.fixture
def host(monkeypatch):
    """-> the handles that products were called with."""
    from humanrf_amd import _lib, ops
    chk, handles = ops._chk, []

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0

    def quantize(x):
        x = x.float()
        scale = x.abs().amax(1) / 127.0
        return torch.round(x / scale[:, None]).to(torch.int8), scale

    def linear(x, weight, relu=False, out_dtype=None):
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("linear_int8: no gradient flows")
        handles.append(weight)
        return x.new_zeros(*x.shape[:-1], weight.out_features)
    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(ops, "_chk", lambda t, name, dtype=None, cuda=True: chk(t, name, dtype, False))
    monkeypatch.setattr(ops, "_rows_of", lambda t, name: t)
    monkeypatch.setattr(ops, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "stream_of", lambda index: 0)
    monkeypatch.setattr(ops, "quantize_int8", quantize)
    monkeypatch.setattr(ops, "linear_int8", linear)
    return handles


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_served_layer_has_a_bias_of_its_own(host, dtype):
    from humanrf_amd.int8 import Int8Linear, Int8MLP
    net = torch.nn.Linear(20, 10).to(dtype)
    served = Int8Linear.from_linear(net)
    want = net.bias.detach().float().clone()
    with torch.no_grad():
        net.bias += 1.0                                     # training goes on
    assert torch.equal(served.bias, want) and served.bias.dtype == torch.float32
    trained = net.bias.detach().clone()
    other = Int8Linear.from_linear(torch.nn.Linear(20, 10))
    served.load_state_dict(other.state_dict())              # another checkpoint is loaded into the served layer
    assert torch.equal(net.bias, trained) and torch.equal(served.bias, other.bias)
    strided = torch.arange(20.0)[::2]
    assert Int8Linear(torch.ones(10, 4), strided).bias.tolist() == strided.tolist()
    mlp = Int8MLP.from_sequential(torch.nn.Sequential(net, torch.nn.ReLU()))
    assert mlp[0].bias.data_ptr() != net.bias.data_ptr()


def test_buffers_that_are_replaced_are_the_ones_multiplied_with(host):
    from humanrf_amd.int8 import Int8Linear
    make = lambda: Int8Linear.from_linear(torch.nn.Linear(20, 10))  # noqa: E731
    served, x = make(), torch.zeros(3, 20)

    def used():
        served(x)
        h = host[-1]
        assert h.packed is served.packed and h.scale is served.scale and h.bias is served.bias
        return h
    used()
    used()
    assert host[-1] is host[-2]
    other = make()
    served.load_state_dict(other.state_dict(), assign=True)
    assert torch.equal(used().scale, other.scale)
    for name in ("packed", "scale", "bias"):
        setattr(served, name, getattr(served, name).clone())
        used()
    served.bias = None
    assert used().bias is None
    served.bias = other.bias
    third = make()
    torch.func.functional_call(served, dict(third.named_buffers()), (x,))
    assert host[-1].packed is third.packed and host[-1].scale is third.scale and host[-1].bias is third.bias
    used()


def test_inputs_that_need_a_gradient_are_refused(host):
    from humanrf_amd.int8 import Int8Linear, Int8MLP
    net = torch.nn.Sequential(torch.nn.Linear(20, 10), torch.nn.ReLU(), torch.nn.Linear(10, 4))
    x = torch.zeros(3, 20, requires_grad=True)
    for served in (Int8Linear.from_linear(net[0]), Int8MLP.from_sequential(net)):
        with pytest.raises(RuntimeError, match="no gradient flows"):
            served(x)
        with torch.no_grad():
            assert not served(x).requires_grad
        assert not served(x.detach()).requires_grad


def test_a_checkpoint_of_another_width_is_refused(host):
    """Rows of 100 and of 120 codes are both padded to 128."""
    from humanrf_amd.int8 import Int8Linear, Int8MLP
    make = lambda k: Int8Linear.from_linear(torch.nn.Linear(k, 10))  # noqa: E731
    served, same, wider = make(100), make(100), make(120)
    assert served.packed.shape == wider.packed.shape
    before = served.bias.clone()
    for assign in (False, True):
        with pytest.raises(RuntimeError, match=r"\(120, 10\).*\(100, 10\)"):
            served.load_state_dict(wider.state_dict(), assign=assign)
        assert torch.equal(served.bias, before)
    served.load_state_dict(same.state_dict())
    assert torch.equal(served.bias, same.bias)
    old = {k: v for k, v in make(100).state_dict().items() if k in ("packed", "scale", "bias")}       # without the widths
    served.load_state_dict(old)
    assert torch.equal(served.bias, old["bias"])
    with pytest.raises(RuntimeError, match="Missing"):
        served.load_state_dict({k: v for k, v in old.items() if k != "scale"})
    net = torch.nn.Sequential(torch.nn.Linear(100, 10), torch.nn.ReLU(), torch.nn.Linear(10, 4))
    a, b = Int8MLP.from_sequential(net), Int8MLP.from_sequential(torch.nn.Sequential(torch.nn.Linear(100, 10), torch.nn.Linear(10, 4)))
    assert list(a.load_state_dict(b.state_dict())) == [[], []]
