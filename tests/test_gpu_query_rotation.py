"""GPU: rotations of fp32 rows are rounded once."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import QueryBatch, Rotary, install_tokens
from cachebridge_amd.plan import rows_from_stacked
from oracle import queries as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 32), (256, 256), (6, 6), (510, 510)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_fp32_rows_are_rounded_once(dim, rotary, interleaved):
    """Half a step of the result, and what 64 bits leave of the angle: positions below 2^17 turn by at most 2^17
    radians, whose three roundings of 2^-53 move an element by 2^-34 of its pair; the series' error is 2^-45."""
    n = 300
    g = torch.Generator().manual_seed(dim)
    q, k = torch.randn(n, 3, dim, generator=g), torch.randn(n, 1, dim, generator=g)
    pool = torch.zeros(1, n, 1, dim).cuda(), torch.zeros(1, n, 1, dim).cuda()
    batch = QueryBatch(rows_from_stacked(*pool), torch.tensor([0, n]).int().cuda(), torch.tensor([n]).int().cuda(), max_length=n)
    pos = torch.cat([torch.arange(100), torch.randint(0, 1 << 17, (200,), generator=g)])
    spin = Rotary.build(rotary, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32), interleaved=interleaved)
    got = install_tokens(batch, 0, q.cuda(), k.cuda(), k.cuda(), spin, positions=pos.cuda())
    # The magnitude is an fp32 argument.
    magnitude = float(torch.tensor(spin.magnitude, dtype=torch.float32))
    for a, x in ((got, q), (pool[0][0], k)):
        want = oracle.rotate(x, pos, spin.inv_freq.cpu(), magnitude=magnitude, interleaved=interleaved)
        size = x.double().abs().amax(-1, keepdim=True) * 2 * magnitude
        assert ((a.double().cpu() - want).abs() - (2.0 ** -24 * want.abs() + 2.0 ** -33 * size)).max() <= 0
