"""Linear attention with infinities in its state, and over many chunks."""
import numpy as np
import pytest

from tests import decoder_cases as dc
from tests.test_gpu_linear_attention import call, check, inputs, tf  # noqa: F401  (tf: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("log_decay", [0.0, -0.5, -1e-3])
def test_an_infinite_state_stays_infinite(tf, n, log_decay):
    """An infinity times a decay is that infinity, and so it leaves in the new state, single tokens and
    prompts alike; the elements beside it keep their values."""
    h, d = 2, 32
    q, k, v, s = inputs(n, 1, h, n, d, d)
    s[0, 0, 3, 5], s[0, 1, 30, 31] = np.inf, -np.inf
    ld = np.full(h, log_decay, np.float32)
    _, got = call(tf, q, k, v, ld, state=s)
    clean = np.where(np.isfinite(s), s, 0).astype(np.float32)
    _, ref, _, off = dc.linear(q, k, v, ld, clean)
    assert got[0, 0, 3, 5] == np.inf and got[0, 1, 30, 31] == -np.inf
    there = np.isfinite(s)
    assert np.all(np.abs(got - ref)[there] <= off[there])
