"""GPU: a state is loaded as a whole or refused as a whole."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_do_not_fit_change_nothing(built, bits):
    import torch
    import tf_approximate_b200 as ax
    p, q = torch.ones(600, device="cuda"), torch.ones(600, device="cuda")
    one, two = ax.AdamW([p], state_bits=bits), ax.AdamW([q], state_bits=bits)
    one.step([torch.ones_like(p)])
    state, names = one.state_dict(), [k for k in ax.AdamW._STATES if hasattr(one, k)]
    last = names[-1]
    bad = [{k: v for k, v in state.items() if k != last}, {**state, last: state[last][:1]}, {**state, last: state[last].double()}, {**state, last: None}, {**state, "step_count": -1},
           {k: v for k, v in state.items() if k != "step_count"}, None]
    for other in bad:
        with pytest.raises(ax.InvalidArgumentError):
            two.load_state_dict(other)
    assert two.step_count == 0 and not any(bool(getattr(two, k).float().any()) for k in names)
    two.load_state_dict({k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in state.items()})
    for k in names:
        assert torch.equal(getattr(two, k).view(torch.uint8), getattr(one, k).view(torch.uint8))
    assert two.step_count == 1
