"""What test_dense8bit_layer.py checks on the CPU and test_gpu_dense8bit_layer.py on the GPU: the layer that answers in 8 bits around its kernel."""
import pytest
import torch


def make(device, dtype=torch.float32, activation="silu", bias=True, inputs=200, units=72):
    import tf_approximate_b200 as ax
    torch.manual_seed(2)
    dense = ax.Dense(inputs, units, activation=activation, use_bias=bias, dtype=dtype).to(device)
    if bias:
        with torch.no_grad():
            dense.bias.normal_()
    return dense


def gradients_are_refused(device):
    """A result of something that is differentiated can be had, and a backward pass through it is an error, not a gradient that is missing."""
    import tf_approximate_b200 as ax
    layer = ax.Dense8bit(make(device))
    x, w, r = torch.randn(5, 200, device=device), torch.randn(200, 200, device=device, requires_grad=True), torch.randn(5, 72, device=device)
    want, beside = layer(x), layer(x, r)
    assert not want.requires_grad
    leaf = x.clone().requires_grad_()
    for y, plain in ((layer(leaf), want), (layer(x, r.clone().requires_grad_()), beside), (layer(leaf, r), beside)):
        assert torch.equal(y.detach(), plain)
        with pytest.raises(ax.InvalidArgumentError):
            y.sum().backward()
    assert leaf.grad is None
    with pytest.raises(ax.InvalidArgumentError):
        (layer(x @ w) + (x @ w).sum()).sum().backward()
    with torch.no_grad():
        assert not layer(leaf).requires_grad and torch.equal(layer(leaf), want)
    with torch.inference_mode():
        assert torch.equal(layer(leaf), want)
    # what does not pass through it has its gradient
    y = layer(leaf.detach()) * leaf[:, :72]
    y.sum().backward()
    assert torch.equal(leaf.grad[:, :72], want)


def casts_of_a_network_leave_the_operands(device):
    """.half(), .bfloat16(), .to(...) and .float() are for the network around the layer: its codes and scales are what they were."""
    import copy
    import tf_approximate_b200 as ax
    layer = ax.Dense8bit(make(device, bias=False))
    # a scale that float16 flushes to 0, and one that it takes for an infinity
    layer.scales[0, 0], layer.scales[0, 1] = 2.0 ** -30, 3.0 * 2.0 ** 17
    bits, lines = layer.scales.view(torch.int32).clone(), layer.lines.clone()
    x = torch.randn(3, 200, device=device)
    net = torch.nn.Sequential(torch.nn.Linear(200, 200).to(device), layer)
    steps = (lambda n: n.half(), lambda n: n.bfloat16(), lambda n: n.to(torch.float16), lambda n: n.to(device, torch.bfloat16), lambda n: n.double(), lambda n: n.type(torch.float16),
             lambda n: n.float())
    want = layer(x)
    for step in steps:
        step(net)
        for which in (layer, copy.deepcopy(layer)):
            assert which.scales.dtype == torch.float32 and torch.equal(which.scales.view(torch.int32), bits)
            assert which.lines.dtype == torch.uint8 and torch.equal(which.lines, lines) and which.kernel.dtype == torch.float8_e4m3fn
    assert torch.equal(layer(x), want) and list(layer.state_dict()) == ["lines", "scales"] and layer.state_dict()["scales"].dtype == torch.float32
    moved = copy.deepcopy(layer).to("meta")
    assert moved.scales.is_meta and moved.lines.is_meta and moved.scales.dtype == torch.float32
    again = moved.to_empty(device=device)
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), want)


def answers_have_the_types_that_the_dense_layers_have(device):
    import tf_approximate_b200 as ax
    types = (torch.float32, torch.bfloat16, torch.float16)
    for dtype in types:
        dense = make(device, dtype)
        layer, x = ax.Dense8bit(dense), torch.randn(4, 200, device=device)
        for given in types + (torch.float64,):
            y = layer(x.to(given))
            # as Dense does: inputs are cast to its type
            assert y.dtype == dtype and torch.equal(y, ax.dense_8bit(x.to(given).to(dtype), layer.kernel, layer.scales, layer.bias, activation="silu"))
            assert layer(x.to(given), torch.zeros(4, 72, device=device, dtype=dtype)).dtype == dtype
        # and it follows a network's casts
        for cast in types:
            assert layer.to(cast)(x).dtype == cast and ax.Dense8bit(dense).to(dtype=cast)(x).dtype == cast
        assert list(layer.state_dict()) == ["lines", "scales", "bias"]
