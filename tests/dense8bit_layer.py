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
