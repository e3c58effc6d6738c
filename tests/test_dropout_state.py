"""CPU: what a resumed run needs of a dropout layer is in its state, with a stand-in for the kernel."""
import io

import pytest

import dropout_stand_in


@pytest.fixture(autouse=True)
def stand_in(built, monkeypatch):
    dropout_stand_in.place(monkeypatch)


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("seed", [None, 5, (1 << 64) - 1])
def test_masks_go_on_after_a_state_was_loaded(capturable, seed):
    import torch
    import tf_approximate_b200 as ax
    x = torch.ones(400)
    first = torch.nn.Sequential(torch.nn.Linear(400, 400), ax.Dropout(0.5, seed=seed, capturable=capturable))
    for _ in range(3):
        first[1](x)
    file = io.BytesIO()
    torch.save(first.state_dict(), file)
    file.seek(0)
    second = torch.nn.Sequential(torch.nn.Linear(400, 400), ax.Dropout(0.5, capturable=capturable))
    assert not second.load_state_dict(torch.load(file, weights_only=True)).missing_keys
    assert second[1].seed == first[1].seed and int(second[1].calls) == 3
    for _ in range(2):
        assert torch.equal(first[1](x), second[1](x))
    # from one form to the other
    other = ax.Dropout(0.5, capturable=not capturable)
    other.load_state_dict(first[1].state_dict())
    assert int(other.calls) == 5 and type(other.calls) is type(ax.Dropout(0.5, capturable=not capturable).calls) and torch.equal(other(x), first[1](x))


@pytest.mark.parametrize("capturable", [False, True])
def test_states_without_them(capturable):
    """States saved before the layer had any: they load as they did, and the layer keeps its own seed and count."""
    import torch
    import tf_approximate_b200 as ax
    net = torch.nn.Sequential(torch.nn.Linear(4, 4), ax.Dropout(0.5, seed=9, capturable=capturable))
    net[1](torch.ones(8))
    state = {k: v for k, v in net.state_dict().items() if k.startswith("0.") or capturable and k == "1.calls"}
    assert not net.load_state_dict(state).missing_keys and net[1].seed == 9 and int(net[1].calls) == 1


def test_states_that_are_none():
    import torch
    import tf_approximate_b200 as ax
    layer = ax.Dropout(0.5, seed=9)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(())):
        for name in ("seed", "calls"):
            with pytest.raises(RuntimeError):
                layer.load_state_dict({**layer.state_dict(), name: bad})
    assert layer.seed == 9 and layer.calls == 0


@pytest.mark.parametrize("capturable", [False, True])
def test_copies(capturable):
    """A copy of a layer that was given no seed draws its own (blocks that are copied drop other places); one with a seed keeps it, and its count."""
    import copy
    import pickle
    import torch
    import tf_approximate_b200 as ax
    x = torch.ones(1000)
    block = torch.nn.Sequential(torch.nn.Linear(4, 4), ax.Dropout(0.5, capturable=capturable))
    block[1](x)
    blocks = [block] + [copy.deepcopy(block) for _ in range(3)]
    assert len({b[1].seed for b in blocks}) == 4 and all(int(b[1].calls) == 1 for b in blocks)
    masks = [b[1](x) for b in blocks]
    assert not any(torch.equal(a, b) for i, a in enumerate(masks) for b in masks[:i])
    # a copy is the same layer in every other respect, and a stored one in all
    for other in (pickle.loads(pickle.dumps(block[1])), copy.copy(block[1])):
        assert other.seed == block[1].seed and int(other.calls) == int(block[1].calls)
    given = ax.Dropout(0.5, seed=7, capturable=capturable).eval()
    again = copy.deepcopy(given)
    assert again.seed == 7 and not again.training and again.rate == 0.5 and list(again.state_dict()) == list(given.state_dict())
    if capturable:
        again.calls.add_(1)
        assert int(given.calls) == 0
