"""Append and gather of a paged KV cache: rows whose scale is a few units of the
smallest subnormal number, against the formats' definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged import DEV, Setup, quantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("kv", ["q8", "f8"])
def test_rows_of_a_few_units_of_the_smallest_number(kv, hd):
    """Largest magnitudes of 1 .. 1500 x 2^-149: the scale is rounded to 0, 1, 2, ... units, so the largest quotients
    lie up to a factor of 1.5 past the largest code, which stands for them."""
    tops = [*range(1, 700), *range(700, 1500, 7)]
    g = torch.Generator().manual_seed(hd)
    x = torch.randint(-1500, 1501, (len(tops), 1, hd), generator=g)
    for i, t in enumerate(tops):
        x[i] = x[i].clamp(-t, t)
        x[i, 0, :4] = torch.tensor([t, -t, t - 1, 1 - t])
    x = x.float() * 2.0 ** -149
    assert x.abs().amax().item() > 0
    su = Setup(kv, hd, 1, 16, lens=[len(tops)], rows=[len(tops)])
    su.cache.append(su.batch, x.to(DEV), -x.to(DEV))
    k, v = su.cache.gather(su.batch, len(tops), torch.float32)
    elems, scale = quantise(x, kv)
    want = elems.float() * scale[..., None]
    assert torch.equal(k.cpu(), want)
    assert torch.equal(v.cpu(), -want)
