"""GPU: an 8-bit cache past 2^32 bytes holds, for the same calls, the bits that one of a few pages holds."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import QueryBatch, Rotary, install_tokens, paged_attention, quantize_tokens
from cachebridge_amd.plan import BlockScales, rows_from_stacked
from oracle import quantized as oracle, queries

from . import query_cases
from .quantized_cases import codes_of
from .query_cases import check_attention

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_keys_and_values_past_32_bits(new, dtype):
    """Pages on both sides of 2^32 bytes of a 5 GB layer: stored keys and values, the tokens before them, the answers."""
    kv, dim, page, rows = 16, 256, 64, 5 * (1 << 30) // 4096
    far = (1 << 32) // 4096 // page  # the page that 2^32 bytes lie before
    mine = {rows // page: [3, far - 1, far, rows // page - 1], 4: [0, 1, 2, 3]}
    length = 4 * page - 7
    plain = query_cases.make([length], [new], heads=kv, kv_heads=kv, dim=dim, dtype=dtype, seed=new)
    fused = (torch.randn(new, 3 * kv, dim, generator=torch.Generator().manual_seed(9)) * 0.5).to(dtype)
    spin = Rotary.build(dim, 1e4)
    held = {}
    for pages, place in mine.items():
        k, v = (torch.empty(1, pages * page, kv, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        scales = [torch.full((1, pages, kv), 99, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
        table = torch.tensor(place, dtype=torch.int32).cuda()
        batch = QueryBatch(rows_from_stacked(k, v, block_table=table, page_size=page, scales=BlockScales(*scales, page, dtype)),
                           *plain.batch._keep[:2], request_stride=4 * page, max_length=length)

        def state():
            codes = [torch.cat([codes_of(x[:, p * page:(p + 1) * page]) for p in place], 1)[0, :length].cpu() for x in (k, v)]
            return codes + [codes_of(s)[0, place].cpu() for s in scales]
        got = [quantize_tokens(plain.batch, batch).cpu(), *state()]
        fd = fused.cuda()
        q = install_tokens(batch, 0, fd[:, :kv], fd[:, kv:2 * kv], fd[:, 2 * kv:], spin)
        got += [q.cpu(), *state()]
        got += [x.cpu() for x in paged_attention(batch, 0, q, return_lse=True)]
        held[pages] = got
        del k, v, batch
    for x, y in zip(*held.values()):
        assert torch.equal(x, y)
    lengths, *before = held[4][:5]
    q, *after, out, lse = held[4][5:]
    assert lengths.tolist() == [length]
    at = torch.arange(length - new, length)
    turned = queries.rotate(fused[:, kv:2 * kv], at, spin.inv_freq.cpu())
    for kind, want in enumerate((turned, fused[:, 2 * kv:].double())):
        codes, e = after[kind], after[2 + kind].long() - 127
        values = oracle.values(codes, e, page)
        # Half a step of the code (2^-4 of the value or 2^-10 of the scale), and what an fp32 rotation is off by.
        scale = 2.0 ** e.double()[at // page][..., None]
        slack = 2.0 ** -21 * want.abs().amax() * 2
        assert ((values[at] - want).abs() <= 2.0 ** -4 * (want.abs() + slack) + 2.0 ** -10 * scale + slack).all()
        # Rows of half the cached ones' size: no scale grows, the cached tokens keep their codes.
        assert torch.equal(after[2 + kind], before[2 + kind]) and torch.equal(codes[:length - new], before[kind][:length - new])
        setattr(plain, "kv"[kind], values[None])
    plain.q, plain.slots = q, [torch.arange(length)]
    check_attention(plain, out, lse)
