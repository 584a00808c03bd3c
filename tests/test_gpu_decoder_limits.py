"""The decoder's operators where sizes and values reach their limits."""
import numpy as np
import pytest

from tests import decoder_cases as dc
from tests.test_gpu_paged_cache import run_evict, tf  # noqa: F401  (tf: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [11952, 11968, 12288, 12304, 49152, 49168])
@pytest.mark.parametrize("dim", [8, 6])
def test_evict_around_the_shared_memory_steps(tf, slots, dim):
    """Rows whose keys fill the shared memory that a launch has without asking for more, and what it
    can ask for at most; full rows and short ones in long tables."""
    page = 16
    lengths = [slots, 100] if slots < 20000 else [300, 100]
    cache = dc.Cache(slots + dim, 1, dim, page, lengths, max_pages=slots // page)
    r = np.random.default_rng(slots)
    w = r.random((2, 1, slots)).astype(np.float32)
    ref = dc.evict(cache, w, lengths, 60, 20)
    got = run_evict(tf, cache, w, 60, 20)
    for a, b in zip(got, ref):
        assert a.dtype == b.dtype and np.array_equal(a, b, equal_nan=a.dtype == np.float32)
