"""GPU: a step tells autograd that it changed the parameters."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_from_before_the_step_is_refused(built, bits):
    import torch
    import tf_approximate_b200 as ax
    params = [torch.ones(n, device="cuda", requires_grad=True) for n in (5, 300)]
    opt = ax.AdamW(params, state_bits=bits)
    loss = sum((p * p).sum() for p in params)
    loss.backward(retain_graph=True)
    versions = [p._version for p in params]
    opt.step([params[0].grad, None])
    assert params[0]._version > versions[0] and params[1]._version == versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode_have_no_version(built):
    import torch
    import tf_approximate_b200 as ax
    with torch.inference_mode():
        p = torch.ones(300, device="cuda")
        opt = ax.AdamW([p], lr=0.5, weight_decay=0.0)
        opt.step([torch.ones(300, device="cuda")])
        assert torch.allclose(p, torch.full_like(p, 0.5))
