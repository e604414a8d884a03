"""reorder_states where beam lies in the memory of a state: it is read while states are written."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    with torch.random.fork_rng():                              # other files' random numbers are those they would have alone
        torch.manual_seed(0)
        yield


def test_a_state_that_holds_beam_is_refused():
    beam = torch.tensor([[1, 0], [0, 0]], device="cuda")
    state = torch.randn(4, 6, device="cuda")
    kept = state.clone()
    for states in ([beam.view(4, 1)], [state, beam.view(4, 1)], [beam.view(torch.uint8).view(4, 8)]):
        with pytest.raises(ValueError, match="beam"):
            m2_b200.reorder_states(states, beam)
    wide = torch.zeros(2, 4, dtype=torch.long, device="cuda")      # rows of a state, entries of beam in between
    with pytest.raises(ValueError, match="beam"):
        m2_b200.reorder_states([wide.view(-1)[:4]], wide.view(-1)[2:6].view(2, 2))
    assert torch.equal(state, kept) and beam.tolist() == [[1, 0], [0, 0]]
    m2_b200.reorder_states([beam.view(4, 1)], beam.clone())         # a copy of it is none of a state's
    assert beam.tolist() == [[0, 1], [0, 0]]
    m2_b200.reorder_states([wide.view(-1)[:4]], torch.zeros(2, 4, dtype=torch.long, device="cuda")[:, ::2])       # copied by the call
    m2_b200.reorder_states([], torch.zeros(2, 2, dtype=torch.long, device="cuda"))
    m2_b200.reorder_states([state[:0]], torch.zeros(0, 2, dtype=torch.long, device="cuda"))
