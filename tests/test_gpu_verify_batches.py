"""fl_verify_device on large batches of tiny and uneven work, and at the ends of
its inputs' ranges, against the definition in 64 bits (test_gpu_verify.py)."""
from __future__ import annotations

import pytest
import torch

from test_gpu_verify import case, run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [2, 3, 17, 40])
def test_many_sequences_of_almost_no_work(V, probs):
    """2000 clusters whose CTAs have an entry each, or none: sums go around as soon as the CTAs start."""
    run_case(*case(V, V, [2, 1, 3, 0, 2] * 400, probs=probs))
