"""fl_verify_device on large batches of tiny and uneven work, and at the ends of
its inputs' ranges, against the definition in 64 bits (test_gpu_verify.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dotnetfoundryllm_b200.speculate import verify_drafts
from test_gpu_verify import case, run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [2, 3, 17, 40])
def test_many_sequences_of_almost_no_work(V, probs):
    """2000 clusters whose CTAs have an entry each, or none: sums go around as soon as the CTAs start."""
    run_case(*case(V, V, [2, 1, 3, 0, 2] * 400, probs=probs))


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [5, 300, 5000])
def test_temperatures_up_to_infinity(V, probs):
    """All logits weigh the same in the end, masked ones nothing."""
    counts = [1, 3, 2, 4, 2, 5]
    logits, starts, draft, _, ua, us, q = case(V + 3, V, counts, probs=probs)
    ua[::2] *= 1.0 / V                      # small enough for some drafts to be accepted
    accepted = 0
    for t in (1e4, 1e30, torch.finfo(torch.float32).max, math.inf):
        temp = np.full(len(counts), t, np.float32)
        _, n = run_case(logits, starts, draft, temp, ua, us, q)
        accepted += n.sum()
        masked = logits.masked_fill(torch.rand(logits.shape, generator=torch.Generator().manual_seed(2)) < 0.4, -math.inf)
        run_case(masked, starts, draft, np.minimum(temp, torch.finfo(torch.float32).max), ua, us, q)
    assert accepted > 0
    dev = lambda x, dt: torch.as_tensor(np.asarray(x), dtype=dt).cuda()  # noqa: E731
    got = [verify_drafts(masked.cuda(), dev(starts, torch.int32), dev(draft, torch.int32), dev([t] * len(counts), torch.float32),
                         dev(ua, torch.float32), dev(us, torch.float32), None if q is None else q.cuda())
           for t in (torch.finfo(torch.float32).max, math.inf)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
