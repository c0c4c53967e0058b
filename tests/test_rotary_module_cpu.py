"""RotaryPositions as part of a model that is moved, cast, copied and made without memory first."""
import copy
import io

import pytest
import torch


@pytest.mark.parametrize("kw", [{}, {"base": 500.0, "stretch": 4.0, "trained": 64}])
def test_made_without_memory(tpo, kw):
    """A model made on the meta device gets its frequencies with its memory, in 64 bits."""
    want = tpo.RotaryPositions(16, **kw).frequencies
    with torch.device("meta"):
        m = torch.nn.Sequential(torch.nn.Linear(4, 4), tpo.RotaryPositions(16, **kw))
    assert m[1].frequencies.is_meta
    m.half()
    assert m[1].frequencies.is_meta and m[1].frequencies.dtype == torch.float64
    m.to_empty(device="cpu")
    assert torch.equal(m[1].frequencies, want) and m[0].weight.dtype == torch.float16
    m = tpo.RotaryPositions(16, device="meta", **kw).to_empty(device="cpu")
    assert torch.equal(m.frequencies, want)


def test_given_frequencies_have_to_be_there(tpo):
    """Frequencies that were given cannot be made again: what has none is refused."""
    m = tpo.RotaryPositions(6, frequencies=torch.ones(3, device="meta"))
    with pytest.raises(NotImplementedError):
        m.to_empty(device="cpu")
    m = tpo.RotaryPositions(6, frequencies=torch.tensor([1.0, 3.0, 9.0]))
    assert torch.equal(m.to_empty(device="cpu").frequencies, torch.tensor([1.0, 3.0, 9.0]).double())


def test_copies(tpo):
    m = tpo.RotaryPositions(16, base=500.0, interleaved=True, amplitude=1.5).bfloat16()
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    for other in (copy.deepcopy(m), torch.load(file, weights_only=False)):
        assert torch.equal(other.frequencies, m.frequencies)
        assert other.interleaved and other.amplitude == 1.5
    assert not m.state_dict()
    m.load_state_dict({})
