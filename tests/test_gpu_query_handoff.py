"""GPU: from the handoff to answers. A cohort's histories are mapped into a paged pool, its new tokens are stored,
attend and weigh, long histories are evicted to other pages of the same pool, and the next step answers on those."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd import pool_rows, synthetic
from cachebridge_amd.online.blocks import map_install_batch, map_install_block
from cachebridge_amd.online.queries import QueryBatch, Rotary, add_key_weights, evict_tokens, install_tokens, paged_attention
from cachebridge_amd.plan import RequestSpan
from cachebridge_amd.pool import PagedKVPool
from oracle import queries as oracle

pytestmark = pytest.mark.gpu

LAYERS, PAGE, HISTORY, NEW, BUDGET = 3, 16, [333, 250], [5, 1], 100


class LayerPool:
    """A pool that is no PagedKVPool: one buffer per layer, as MHATokenToKVPool has."""

    def __init__(self, like: PagedKVPool):
        self.layer_num, self.start_layer, self.dtype = like.layer_num, like.start_layer, like.dtype
        self.page_size = like.page_size
        self._k, self._v = ([x.clone() for x in buffers] for buffers in (like.k_buffer, like.v_buffer))

    def _get_key_buffer(self, layer):
        return self._k[layer - self.start_layer]

    def _get_value_buffer(self, layer):
        return self._v[layer - self.start_layer]


def tables(room, order):
    """Flat block table, offsets in index tokens and each request's slots for requests of `room` tokens."""
    flat, offsets, slots = [], [], []
    for n in room:
        pages = [order.pop() for _ in range(math.ceil(n / PAGE))]
        offsets.append(PAGE * len(flat))
        flat += pages
        t = torch.arange(n)
        slots.append(torch.tensor(pages)[t // PAGE] * PAGE + t % PAGE)
    return torch.tensor(flat, dtype=torch.int32).cuda(), torch.tensor(offsets).cuda(), slots


def check(out, q, k, v, dim):
    """Rows of one request against the oracle on the pool's own rows."""
    group = q.shape[1] // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    for h in range(q.shape[1]):
        want, _, mag = oracle.attention(q[:, h], k[:, h // group], v[:, h // group], scale=dim ** -0.5)
        d = oracle.score_error(q[:, h], k[:, h // group], scale=dim ** -0.5)
        tol = u * want.abs() + u * mag + mag * (4 * d + (k.shape[0] + 16) * 2.0 ** -23)
        assert ((out[:, h].double().cpu() - want).abs() - tol).max() <= 0, h


@pytest.mark.parametrize("layers_apart", [False, True])
def test_answers_on_a_handed_off_cohort(layers_apart):
    sh = synthetic.shape("tp4", tokens=sum(HISTORY))
    sh.target_layers = LAYERS
    h = synthetic.make_handoff(sh, target_pages=128)
    pool = LayerPool(h.target_pool) if layers_apart else h.target_pool
    g = torch.Generator().manual_seed(3)
    order = torch.randperm(128, generator=g).tolist()
    table, offsets, slots = tables([n + m for n, m in zip(HISTORY, NEW)], order)
    spans = [RequestSpan(0, int(offsets[0]), HISTORY[0], 0, HISTORY[0]),
             RequestSpan(HISTORY[0], int(offsets[1]), HISTORY[1], 0, HISTORY[1])]
    map_install_batch(h.mapper, h.source_pool, h.source_slots, pool, spans, block_table=table, page_size=PAGE)
    mapped = [(pool._get_key_buffer(l).cpu(), pool._get_value_buffer(l).cpu()) for l in range(LAYERS)]

    kv, dim = pool._get_key_buffer(0).shape[1:]
    heads, dtype = 4 * kv, pool.dtype
    new = torch.randn(LAYERS, sum(NEW), heads + 2 * kv, dim, generator=g).to(dtype).cuda()
    start = torch.tensor([0, NEW[0], sum(NEW)], dtype=torch.int32).cuda()
    lengths = torch.tensor([n + m for n, m in zip(HISTORY, NEW)], dtype=torch.int32).cuda()
    batch = QueryBatch(pool_rows(pool, block_table=table, page_size=PAGE), start, lengths, offsets=offsets,
                       max_length=int(lengths.max()), max_query=max(NEW))
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    spin = Rotary.build(dim, 1e6, device="cuda")
    weights = torch.zeros(2, int(lengths.max())).cuda()
    for layer in range(LAYERS):
        x = new[layer]
        q = install_tokens(batch, layer, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], spin, error_flag=flag)
        out, lse = paged_attention(batch, layer, q, return_lse=True, error_flag=flag)
        add_key_weights(batch, layer, q, lse, weights, error_flag=flag)
        k, v = pool._get_key_buffer(layer).cpu(), pool._get_value_buffer(layer).cpu()
        for b, (n, m) in enumerate(zip(HISTORY, NEW)):
            old = slots[b][:n]
            assert torch.equal(k[old], mapped[layer][0][old]) and torch.equal(v[old], mapped[layer][1][old])
            rows = slice(0, NEW[0]) if b == 0 else slice(NEW[0], None)
            assert torch.equal(v[slots[b][n:]], x[rows, heads + kv:].cpu())
            check(out[rows], q[rows].cpu(), k[slots[b]], v[slots[b]], dim)
    sums = weights.sum(1).cpu()  # each row's weights sum to one: fp32 sums of at most 338 terms
    want = torch.tensor([float(LAYERS * heads * m) for m in NEW])
    assert ((sums - want).abs() <= want * 400 * 2.0 ** -23).all()

    # The kept tokens go to pages of the same pool; the step after answers there, at the tokens' own positions.
    table2, offsets2, slots2 = tables([BUDGET + 1] * 2, order)
    grown = torch.zeros(2, dtype=torch.int32).cuda()
    one = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    smaller = QueryBatch(pool_rows(pool, block_table=table2, page_size=PAGE), one, grown, offsets=offsets2,
                         max_length=BUDGET + 1, max_query=1)
    kept = evict_tokens(batch, weights, smaller, budget=BUDGET, first=4, last=16, error_flag=flag)
    grown.copy_(kept.lengths + 1)
    x = torch.randn(2, heads + 2 * kv, dim, generator=g).to(dtype).cuda()
    for layer in range(LAYERS):
        q = install_tokens(smaller, layer, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], spin,
                           positions=lengths.clone(), error_flag=flag)
        out = paged_attention(smaller, layer, q, error_flag=flag)
        k, v = pool._get_key_buffer(layer).cpu(), pool._get_value_buffer(layer).cpu()
        for b in range(2):
            tokens = kept.tokens[b].cpu().long()
            assert tokens.tolist() == oracle.keep(weights[b, :int(lengths[b])].tolist(), BUDGET, 4, 16)
            assert torch.equal(k[slots2[b][:BUDGET]], k[slots[b][tokens]]) and torch.equal(v[slots2[b][:BUDGET]], v[slots[b][tokens]])
            check(out[b:b + 1], q[b:b + 1].cpu(), k[slots2[b]], v[slots2[b]], dim)
    assert int(flag) == 0 and h.mapper.plan.read_errors() == 0
    # The cohort's rows are those of each request mapped alone.
    if not layers_apart:
        alone = PagedKVPool(layer_num=LAYERS, pages=128, head_num=kv, head_dim=dim, dtype=dtype, fill="zeros")
        pages = table[:math.ceil((HISTORY[0] + NEW[0]) / PAGE)].contiguous()
        map_install_block(h.mapper, h.source_pool, h.source_slots, alone, start=0, stop=HISTORY[0], block_table=pages,
                          page_size=PAGE, prefix_length=HISTORY[0])
        for layer in range(LAYERS):
            at = slots[0][:HISTORY[0]]
            assert torch.equal(alone.k_buffer[layer].cpu()[at], mapped[layer][0][at])
