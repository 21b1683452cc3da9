"""A captured decode step driven by PagedCache: the step's own tables, into which those
of every PagedCache.batch() are copied."""
import pytest
import torch

import moe_infer_amd as m

from .test_gpu_paged import D, gen, norm_weights, randn

pytestmark = pytest.mark.gpu


def test_a_captured_step_takes_the_tables_of_the_cache():
    """Sequences that grow over the ends of pages, one that ends and another in its pages,
    replayed beside the same calls made eagerly over a cache of its own."""
    B, width, most = 3, 8, 8 * 32
    rope, g = m.Rope(64, 1e6), gen(1)
    caches = [m.PagedCache(num_layers=1, num_q_heads=16, num_kv_heads=2, num_pages=20, page_rows=32) for _ in range(2)]
    qw, kw = norm_weights(g), norm_weights(g)
    seqs = [c.add() for c in caches for _ in range(B)]
    mine, other = seqs[:B], seqs[B:]
    past = [30, 95, 5]
    k, v, q = randn(g, sum(past), 2, D), randn(g, sum(past), 2, D), randn(g, sum(past), 16, D)
    for c, ss in zip(caches, (mine, other)):
        t = c.batch(ss, past)
        m.paged_append(c.pages(0), t.block_table, t.kv_len, k, v, rope=rope, cu_q=t.cu_q, k_norm_w=kw)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    kv_len = torch.zeros(B, dtype=torch.int32, device="cuda")
    k, v, q, gate = (randn(g, B, h, D) for h in (2, 2, 16, 16))
    qo, out = torch.empty_like(q), torch.empty_like(q)
    ws = m.paged_workspace(B, B, 1, most)

    def step(pages, table, kv_len, qo, out):
        m.paged_append(pages, table, kv_len, k, v, rope=rope, q=q, q_norm_w=qw, k_norm_w=kw, q_out=qo)
        m.attn_decode_paged(pages, table, kv_len, qo, most, gate=gate, out=out, workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(caches[0].pages(0), table, kv_len, qo, out)  # no rows: writes no page
    torch.cuda.current_stream().wait_stream(s)
    assert torch.all(out == 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0].pages(0), table, kv_len, qo, out)
    for i in range(40):
        if i == 20:  # one sequence ends, a new one takes its place and its pages
            for c, ss in zip(caches, (mine, other)):
                c.remove(ss[1])
                ss[1] = c.add()
        for x in (k, v, q, gate):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        t = caches[0].batch(mine)
        table[:, :t.block_table.shape[1]].copy_(t.block_table)
        table[:, t.block_table.shape[1]:] = -1
        kv_len.copy_(t.kv_len)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        t = caches[1].batch(other)
        want_q, want = torch.empty_like(q), torch.empty_like(q)
        step(caches[1].pages(0), t.block_table, t.kv_len, want_q, want)
        assert torch.equal(got, want) and torch.equal(qo, want_q), f"step {i}"
        assert not torch.any(torch.isnan(got)), f"step {i}"
