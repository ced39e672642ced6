"""Prompts of a decoder layer start their sequences: what is refused before the layer runs."""
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402


class _Reached(Exception):
    pass


def _layer():
    from oxionnx_amd import decoder

    class Layer(decoder.DecoderLayer):
        def __init__(self):
            pass

        def _append(self, x, slots, positions):
            raise _Reached
    return Layer()


@pytest.mark.parametrize("counts, held", [([3, 2], [0, 4]), ([1], [1]), ([0, 5, 2], [3, 0, 9])])
def test_prompts_behind_tokens_are_refused(counts, held):
    cu = torch.tensor([0] + counts).cumsum(0).int()
    positions = torch.cat([torch.arange(h, h + c) for h, c in zip(held, counts)]).int()
    with pytest.raises(L.OhipError):
        _layer().prefill(torch.zeros(sum(counts), 8), cu, positions, positions)


@pytest.mark.parametrize("counts, held", [([3, 2], [0, 0]), ([0, 2, 0, 4], [7, 0, 1, 0]), ([0], [5])])
def test_prompts_that_start_their_sequences_run(counts, held):
    """(a sequence without a prompt in the batch may hold what it holds)"""
    cu = torch.tensor([0] + counts).cumsum(0).int()
    positions = torch.cat([torch.arange(h, h + c) for h, c in zip(held, counts)]).int()
    with pytest.raises(_Reached):
        _layer().prefill(torch.zeros(sum(counts), 8), cu, positions, positions)
