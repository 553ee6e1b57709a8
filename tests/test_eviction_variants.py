"""ext.paged_cache_evict's variants at the sizes that choose each: many wide rows in one workgroup a row, the second move, moves
of their own in graphs and beside other calls; bit for bit as test_paged_evict's plain choice and move on the host."""
import pytest
import torch

from paged_cases import E4M3
from test_paged_cache import _bits
from test_paged_evict import NAMES, evict_case, expected, run_and_check

F16, BF16 = torch.float16, torch.bfloat16


def _workspace(a, budget):
    from tris_moe_amd import _lib

    page, heads = a["k_cache"].shape[2], a["k_cache"].shape[1]
    batch, pages = a["block_table"].shape
    return _lib.load().tris_paged_cache_evict_workspace_bytes(batch, heads, pages, page, budget)


def _check_outcome(a, want, got):
    out, sums, new, kept = want
    assert torch.equal(got[0].cpu(), new) and torch.equal(got[1].cpu(), kept)
    assert torch.equal(_bits(a["weight_sum"]), _bits(sums))
    for n in NAMES:
        assert out[n] is None or torch.equal(_bits(a[n]), _bits(out[n])), n


# more than 64 rows on tables of 16385 to 32768 positions: a workgroup each, 32 positions a thread
@pytest.mark.gpu
@pytest.mark.parametrize("cache,page,heads,dim,longest,budget,limit,sink,recent", [
    (F16, 16, 2, 64, 32768, 200, 250, 0, 0),             # (moved by the choosing workgroups: little of a row stays)
    (F16, 16, 2, 64, 32768, 17000, 17000, 3, 500),       # moved by a launch of its own
    (E4M3, 7, 8, 64, 17000, 9000, 9000, 0, 9000),        # more than 160 rows: with the choice; nothing chosen by weight
    (BF16, 5, 8, 128, 16390, 16384, 16384, 0, 0),
    (E4M3, 64, 33, 64, 20000, 12000, 12001, 12000, 0),   # more than 256 rows
], ids=str)
def test_wide_tables_of_many_rows(tris, cuda, cache, page, heads, dim, longest, budget, limit, sink, recent):
    """One sequence fills the table, some have a place less, one is just over the limit, the others are short; in their heads
    all weights are alike, all different, or of both."""
    few = heads == 2
    lengths = [longest, limit + 1, limit, 1, 0, 33] + [7 * i % 30 for i in range(20)] + ([longest - 1] * 8 if few else [])
    a = evict_case(cuda, heads, dim, cache, page, lengths, seed=budget, extra_pages=0)
    rows, positions = len(lengths) * heads, a["block_table"].shape[1] * page
    assert rows > 64 and 16384 < positions <= 32768 and _workspace(a, budget) == 0
    w, g = a["weight_sum"], torch.Generator().manual_seed(rows)
    w[0, 0] = 0.5
    w[0, 1] = torch.randperm(positions, generator=g).to(torch.float32).to(cuda)
    w[1, 0, ::2] = 0.25
    w[1, 1] = torch.randperm(positions, generator=g).to(torch.float32).to(cuda) * 2.0 ** -20
    if few:
        w[-1, 0] = torch.arange(positions, dtype=torch.float32, device=cuda)
        w[-1, 1] = float("nan")
    print(f"[gpu-case] evict wide {cache} rows={rows} positions={positions} budget={budget}", flush=True)
    new, _ = run_and_check(tris, a, budget, limit, sink, recent)
    assert new.tolist()[:3] == [budget, budget, limit]


# budgets past 4096 on tables of twice as many positions: rows past the budget are moved by a launch of their own
@pytest.mark.gpu
@pytest.mark.parametrize("cache,page,heads,dim,order,lengths,budget,extra_pages", [
    (F16, 16, 3, 128, "token", [20000, 300], 5000, 1),   # the choice in segments
    (BF16, 9, 2, 256, "head", [33000], 8200, 1),
    (E4M3, 7, 4, 256, "token", [17000, 9000], 4100, 1),
    (E4M3, 16, 3, 128, "head", [18000], 6001, 1),
    (F16, 16, 2, 128, "token", [12000, 11000], 5000, 0),  # the choice in one workgroup a row
    (E4M3, 7, 4, 256, "head", [9000, 100], 4097, 0),
    (BF16, 64, 4, 256, "token", [16384], 8192, 0),
    (E4M3, 16, 1, 64, "token", [10000], 4500, 100),
], ids=str)
def test_rows_from_past_the_budget(tris, cuda, cache, page, heads, dim, order, lengths, budget, extra_pages):
    a = evict_case(cuda, heads, dim, cache, page, lengths, order, seed=budget, extra=2, extra_pages=extra_pages)
    positions = a["block_table"].shape[1] * page
    assert positions >= 2 * budget and (_workspace(a, budget) > 0) == (positions > 16384)
    for sink, recent in ((4, 64), (0, budget)):
        print(f"[gpu-case] evict far {cache} heads={heads} dim={dim} {order} {lengths} budget={budget} recent={recent}",
              flush=True)
        b = {n: None if t is None else t.clone() for n, t in a.items()}
        if order == "token":                             # (a clone keeps the pool's order)
            assert b["k_cache"].stride() == a["k_cache"].stride()
        new, _ = run_and_check(tris, b, budget, None, sink, recent)
        assert new[0] == budget


SEPARATE = [
    (256, 1, 250, 252, [600, 300], BF16),                # one workgroup a row
    (256, 1, 250, 251, [600, 300], E4M3),
    (256, 2100, 250, 252, [600, 300], E4M3),             # segments
    (128, 1, 4200, 4201, [9000, 4300], F16),             # the second move
    (64, 1100, 4200, 4201, [9000, 4300], BF16),          # both
]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,extra_pages,budget,limit,lengths,cache", SEPARATE, ids=str)
def test_replays_of_separate_moves(tris, cuda, dim, extra_pages, budget, limit, lengths, cache):
    """Captured calls whose moves are launches of their own, with eager calls and other work between the replays."""
    ext = tris["ext"]
    a = evict_case(cuda, 2, dim, cache, 16, lengths, seed=3, extra_pages=extra_pages)
    other = evict_case(cuda, 2, dim, cache, 16, lengths, seed=4, extra_pages=extra_pages)
    args = dict(budget=budget, limit=limit, sink=4, recent=20)
    a["seq_lens"].zero_()
    ext.paged_cache_evict(**a, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ext.paged_cache_evict(**a, **args)
    moved = 0
    for step, lens in enumerate(([limit, limit + 1], lengths, [0, budget], lengths[::-1], [limit + 1, limit + 1])):
        lens = [min(n, m) for n, m in zip(lens, lengths)]
        a["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        want = expected(a, **args)
        graph.replay()
        torch.cuda.synchronize()
        _check_outcome(a, want, got)
        moved += int((want[2] != a["seq_lens"].cpu()).sum())
        ext.paged_cache_evict(**other, budget=lengths[1] - 1 - step)
        a["weight_sum"].add_(torch.rand_like(a["weight_sum"]))
    assert moved >= 4


@pytest.mark.gpu
@pytest.mark.parametrize("dim,extra_pages,budget,limit,lengths,cache", SEPARATE, ids=str)
def test_separate_moves_beside_another_call(tris, cuda, dim, extra_pages, budget, limit, lengths, cache):
    """Two calls of several launches at once, on two streams: keys, values, scales and sums of both."""
    ext = tris["ext"]
    cases = [evict_case(cuda, 2, dim, cache, 16, lengths, seed=s, extra_pages=extra_pages) for s in (1, 2)]
    args = dict(budget=budget, limit=limit, sink=4, recent=100)
    want = [expected(x, **args) for x in cases]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got_b = ext.paged_cache_evict(**cases[1], **args)
    got_a = ext.paged_cache_evict(**cases[0], **args)
    torch.cuda.synchronize()
    for x, w, got in zip(cases, want, (got_a, got_b)):
        _check_outcome(x, w, got)
