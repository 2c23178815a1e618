"""What Decoder.beam_search refuses before it touches the GPU."""
from __future__ import annotations

from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from fleet_moe import ops  # noqa: E402


@pytest.mark.parametrize("n, n_steps", [(0, 1), (1, 0), (8, 4), (11, 1), (4, -1)])
def test_prompts_that_do_not_fit(n, n_steps):
    dec = SimpleNamespace(max_pos=10, blob=torch.empty(0))
    with pytest.raises(ValueError, match="positions"):
        ops.Decoder.beam_search(dec, torch.zeros(n, dtype=torch.int32), 2, n_steps)


def test_prompts_that_are_not_rows():
    dec = SimpleNamespace(max_pos=10, blob=torch.empty(0))
    with pytest.raises(ValueError, match="positions"):
        ops.Decoder.beam_search(dec, torch.zeros((1, 4), dtype=torch.int32), 2, 2)
