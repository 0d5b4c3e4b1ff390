"""Calls of the gated linear recurrence at the edge of what its documentation allows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests.test_gpu_recurrence import _check, _close, _inputs, _np
from tests import recurrence_ref as ref

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T", [200, 1500])
def test_a_state_that_lies_in_the_output(T):
    """Chunks through one buffer: the state in front is the last row of the chunk before, which y replaces."""
    from tacotron2_amd import recurrence as R
    from tacotron2_amd._lib import T2Error
    z, f, _, state, _, _ = _inputs(1, T, 96, "f32", False, 3)
    out = torch.empty_like(z)
    for turn in range(3):
        want, final = R.gated_scan(None, z, f, state=state if turn == 0 else want[:, -1].clone())
        got, last = R.gated_scan(None, z, f, state=state if turn == 0 else out[:, -1], out=out)
        assert got is out and torch.equal(out, want) and torch.equal(last, final)
    lens = out.view(torch.int64).view(-1)[:1]
    with pytest.raises(T2Error):
        R.gated_scan(None, z, f, lens=lens, out=out)
