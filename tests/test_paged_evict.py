"""ext.paged_cache_evict (tris_paged_cache_evict) against a plain choice and move on the host, bit for bit: types, head
layouts, pages, lengths, budgets, ties and special weights, pages outside the pool, strides, streams, graphs, refusals."""
import ctypes

import pytest
import torch

from paged_cases import E4M3, make_pool, make_table
from test_paged_cache import BAD_CACHES, _bits, c_cache

F16, BF16 = torch.float16, torch.bfloat16
NAMES = ("k_cache", "v_cache", "k_scale", "v_scale")


def evict_case(cuda, heads, dim, cache, page, lengths, order="head", seed=0, extra=0, extra_pages=1):
    """A pool of random bits, sums with zeros, ties and large ones, all of them past the sequences too."""
    gen = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lengths) + 2
    a = dict(zip(NAMES, make_pool(pages, heads, page, dim, cache, cuda, order)))
    a["block_table"] = make_table(lengths, page, pages, cuda, gen, extra_pages)
    a["seq_lens"] = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    for t in (a[n] for n in NAMES):
        if t is None:
            continue
        raw = torch.uint8 if t.element_size() == 1 else torch.int16 if t.element_size() == 2 else torch.int32
        bits = torch.randint(0, 1 << 7, t.shape, generator=gen) if t.element_size() == 1 else \
            torch.randint(0, 1 << 14, t.shape, generator=gen)
        t.copy_(bits.to(raw).to(cuda).view(t.dtype))
    w = torch.rand((len(lengths), heads, a["block_table"].shape[1] * page + extra), generator=gen)
    w[w < 0.1] = 0.0
    near = torch.rand(w.shape, generator=gen) < 0.3
    w[near] = (w[near] * 4).round() / 4
    a["weight_sum"] = w.to(cuda)
    return a


def expected(a, budget, limit=None, sink=0, recent=0):
    """Host copies after the eviction: (caches and scales by name, sums, new_lens, kept)."""
    limit = budget if limit is None else limit
    c = {n: None if a[n] is None else a[n].cpu() for n in NAMES}
    out = {n: None if t is None else t.clone() for n, t in c.items()}
    raw = {n: None if t is None else t.view(torch.uint8) if t.element_size() == 1 else t for n, t in c.items()}
    to = {n: None if t is None else t.view(torch.uint8) if t.element_size() == 1 else t for n, t in out.items()}
    pages, heads, page = c["k_cache"].shape[:3]
    sums, table, lens = a["weight_sum"].cpu().clone(), a["block_table"].cpu().long(), a["seq_lens"].cpu().tolist()
    new, kept = list(lens), torch.full((len(lens), heads, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        n = min(n, table.shape[1] * page)
        used = table[b, : -(-max(n, 0) // page)]
        if n <= limit or bool(((used < 0) | (used >= pages)).any()):
            continue
        new[b] = budget
        for h in range(heads):
            w = sums[b, h].tolist()
            middle = range(sink, n - recent)
            # NaN above all, of equal ones the lowest position
            order = sorted(middle, key=lambda i: (0 if w[i] != w[i] else 1, -w[i] if w[i] == w[i] else 0, i))
            stay = sorted(list(range(sink)) + order[: budget - sink - recent] + list(range(n - recent, n)))
            assert len(stay) == budget
            j = torch.tensor(stay)
            kept[b, h] = j.to(torch.int32)
            i = torch.arange(budget)
            for name in NAMES:
                if raw[name] is not None:
                    to[name][table[b, i // page], h, i % page] = raw[name][table[b, j // page], h, j % page]
            moved = sums[b, h, j].clone()
            sums[b, h, :n] = 0
            sums[b, h, :budget] = moved
    return out, sums, torch.tensor(new, dtype=torch.int32), kept


def run_and_check(tris, a, budget, limit=None, sink=0, recent=0):
    out, sums, new, kept = expected(a, budget, limit, sink, recent)
    lens = a["seq_lens"].clone()
    got_new, got_kept = tris["ext"].paged_cache_evict(**a, budget=budget, limit=limit, sink=sink, recent=recent)
    assert got_new.dtype == got_kept.dtype == torch.int32
    assert torch.equal(a["seq_lens"], lens)
    assert got_new.tolist() == new.tolist()
    assert torch.equal(got_kept.cpu(), kept)
    assert torch.equal(_bits(a["weight_sum"]), _bits(sums))
    for n in NAMES:
        if out[n] is not None:
            assert torch.equal(_bits(a[n]), _bits(out[n])), n
    return got_new, got_kept


LENGTHS = [0, 1, 2, 15, 16, 17, 33, 100, 129, 200]


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, BF16, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,order", [(16, "head"), (7, "token"), (1, "head"), (48, "token"), (256, "head")])
def test_lengths_and_budgets(tris, cuda, cache, dim, page, order):
    for budget, limit, sink, recent in ((1, 1, 0, 0), (16, 16, 4, 6), (33, 100, 0, 33), (100, 128, 100, 0), (130, 150, 1, 0)):
        print(f"[gpu-case] evict {cache} dim={dim} page={page} {order} budget={budget}", flush=True)
        a = evict_case(cuda, 2, dim, cache, page, LENGTHS, order, seed=budget, extra=3)
        run_and_check(tris, a, budget, limit, sink, recent)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("lengths,budget", [([5000, 4097, 4096, 3], 4096), ([9000, 1030], 1025), ([20000], 1500),
                                            ([3000] * 5, 2999), ([2000], 1), ([1500] * 33, 1400)], ids=str)
def test_long_sequences(tris, cuda, heads, lengths, budget):
    for cache, page in ((F16, 16), (E4M3, 5)):
        print(f"[gpu-case] evict long {cache} heads={heads} {lengths} budget={budget}", flush=True)
        a = evict_case(cuda, heads, 64, cache, page, lengths, seed=heads)
        run_and_check(tris, a, budget, None, min(4, budget - 1), budget // 3)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,budget,limit,sink,recent", [
    ([20000, 16385, 15000, 0, 18000], 15000, 16000, 4, 3000), ([40000], 4096, None, 0, 0), ([33000, 40], 9000, None, 4500, 4500),
    ([300000], 20000, None, 64, 1000), ([16384, 16383], 16380, None, 1, 1), ([32768], 20000, None, 9000, 9000),
    ([50000, 49000, 7], 49000, 49500, 100, 100), ([33000], 4097, None, 0, 4097)], ids=str)
def test_long_rows(tris, cuda, lengths, budget, limit, sink, recent):
    """Tables of as many positions as one workgroup takes and more; budgets beside and below half of them."""
    for cache, page in ((BF16, 64), (E4M3, 7)):
        print(f"[gpu-case] evict segments {cache} {lengths} budget={budget}", flush=True)
        a = evict_case(cuda, 1, 64, cache, page, lengths, seed=budget, extra=1)
        run_and_check(tris, a, budget, limit, sink, recent)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16384, 30000, 40000])
def test_ties_over_segments(tris, cuda, n):
    """The border among equal weights that lie in every segment, one segment, or are all there is."""
    a = evict_case(cuda, 4, 64, F16, 16, [n], extra_pages=0)
    w = a["weight_sum"]
    w[0, 0] = 0.5
    w[0, 1] = 0.0
    w[0, 1, 9000:9100] = 1.0
    w[0, 2, ::3], w[0, 2, 1::3], w[0, 2, 2::3] = 2.0, 1.0, 3.0
    w[0, 3] = float("nan")
    w[0, 3, 5::5] = float("inf")
    run_and_check(tris, a, n // 2 + 77, None, 3, 500)


@pytest.mark.gpu
@pytest.mark.parametrize("extra_pages", [1, 300, 1100, 2100])
def test_special_weights_and_ties(tris, cuda, extra_pages):
    """All equal, zeros of both signs, subnormals, negative ones, infinities and NaN of either sign; ties at the border go
    to the lowest positions.  The same in tables of other widths."""
    inf, nan = float("inf"), float("nan")
    lengths = [3000, 500, 300, 64, 200, 400]
    a = evict_case(cuda, 2, 64, F16, 16, lengths, extra_pages=extra_pages)
    w = a["weight_sum"]
    w[0] = 0.25
    w[1, :, ::2], w[1, :, 1::2] = 0.0, -0.0
    w[2, :, 7:60], w[2, :, 100:110] = nan, inf
    w[2, 1, 3] = torch.tensor(-1, dtype=torch.int32).view(torch.float32)     # a NaN with its sign set
    w[3] = -w[3]
    w[3, :, 5] = -inf
    w[4] = (torch.arange(w.shape[2], device=cuda) % 7 * 2.0 ** -149).to(torch.float32)
    w[5] = nan
    run_and_check(tris, a, 50, 60, 3, 4)


@pytest.mark.gpu
def test_neighbouring_weights(tris, cuda):
    """Weights that differ in their last bits alone, and in their first alone."""
    a = evict_case(cuda, 3, 64, F16, 16, [2000, 1500])
    g = torch.Generator().manual_seed(4)
    n = a["weight_sum"].shape[2]
    bits = torch.stack([torch.stack([0x3F800000 + torch.randint(0, 300, (n,), generator=g),
                                     torch.randint(0, 2 ** 31 - 2 ** 24, (n,), generator=g),
                                     torch.randint(0, 120, (n,), generator=g) << 24]) for _ in range(2)])
    a["weight_sum"].copy_(bits.to(torch.int32).view(torch.float32))
    run_and_check(tris, a, 700, None, 0, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 9])
def test_pages_outside_the_pool(tris, cuda, page):
    """A sequence with such a page below its length stays as it is, wherever the page lies; one past it does not matter."""
    lengths = [200, 200, 200, 200, 130]
    a = evict_case(cuda, 2, 64, E4M3, page, lengths)
    last = -(-200 // page) - 1
    for b, i, bad in ((0, 0, -1), (1, last, a["k_cache"].shape[0]), (2, last // 2, 2 ** 31 - 1)):
        a["block_table"][b, i] = bad
    new, kept = run_and_check(tris, a, 100, 120, 4, 20)
    assert new.tolist() == [200, 200, 200, 100, 100] and bool((kept[:3] == -1).all())


@pytest.mark.gpu
def test_lengths_past_the_table_and_negative(tris, cuda):
    a = evict_case(cuda, 2, 64, F16, 16, [64, 40, 0, 64], extra_pages=0)
    a["seq_lens"].copy_(torch.tensor([2 ** 31 - 1, 40, -5, 70], dtype=torch.int32))
    new, _ = run_and_check(tris, a, 32, 40, 1, 2)
    assert new.tolist() == [32, 40, -5, 32]
    run_and_check(tris, a, 2 ** 12, 2 ** 31 - 1)            # more than the table has: nothing is ever due
    none = {**a, "block_table": a["block_table"][:, :0], "weight_sum": a["weight_sum"][..., :0]}
    assert tris["ext"].paged_cache_evict(**none, budget=4)[0].tolist() == a["seq_lens"].tolist()
    empty = {**a, "block_table": a["block_table"][:0], "weight_sum": a["weight_sum"][:0], "seq_lens": a["seq_lens"][:0]}
    new, kept = tris["ext"].paged_cache_evict(**empty, budget=4)
    assert new.shape == (0,) and kept.shape == (0, 2, 4)


@pytest.mark.gpu
def test_strides_of_pool_and_sums(tris, cuda):
    """A pool inside a larger buffer, whose other parts stay; sums whose heads are the outer dimension, at odd offsets."""
    lengths = [300, 90]
    a = evict_case(cuda, 2, 64, E4M3, 16, lengths)
    whole = {}
    for n in ("k_cache", "v_cache"):
        p, h, s, d = a[n].shape
        whole[n] = torch.full((p, h + 1, s, 2 * d), 3, dtype=torch.uint8, device=cuda)
        view = whole[n][:, 1:, :, d:].view(E4M3)
        view.copy_(a[n])
        a[n] = view
    for n in ("k_scale", "v_scale"):
        p, h, s = a[n].shape
        whole[n] = torch.full((s, p + 1, h), 3.0, device=cuda)
        view = whole[n][:, 1:].permute(1, 2, 0)
        view.copy_(a[n])
        a[n] = view
    w = a["weight_sum"]
    sums = torch.full((w.shape[1], w.shape[0], w.shape[2] + 3), 9.0, device=cuda)
    a["weight_sum"] = sums[..., 1: w.shape[2] + 1].transpose(0, 1).copy_(w)
    run_and_check(tris, a, 64, None, 4, 8)
    for n in ("k_cache", "v_cache"):
        d = a[n].shape[3]
        assert bool((whole[n][:, 0] == 3).all()) and bool((whole[n][..., :d] == 3).all())
    assert bool((whole["k_scale"][:, 0] == 3).all()) and bool((sums[..., 0] == 9).all()) and bool((sums[..., -2:] == 9).all())


@pytest.mark.gpu
def test_again_and_again(tris, cuda):
    """An eviction on what an eviction left, down to one position."""
    a = evict_case(cuda, 2, 128, F16, 16, [700, 320, 90])
    for budget, recent in ((300, 100), (299, 0), (64, 63), (2, 1), (1, 0)):
        new, _ = run_and_check(tris, a, budget, None, 0, recent)
        a["seq_lens"].copy_(new)
    assert a["seq_lens"].tolist() == [1, 1, 1]


@pytest.mark.gpu
def test_streams(tris, cuda):
    """Beside another call on another stream."""
    ext = tris["ext"]
    a, b = (evict_case(cuda, 2, 64, BF16, 16, [600, 300], seed=s) for s in (1, 2))
    want = [expected(x, 256, None, 4, 100) for x in (a, b)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got_b = ext.paged_cache_evict(**b, budget=256, sink=4, recent=100)
    got_a = ext.paged_cache_evict(**a, budget=256, sink=4, recent=100)
    torch.cuda.synchronize()
    for x, (out, sums, new, kept), got in ((a, want[0], got_a), (b, want[1], got_b)):
        assert torch.equal(got[0].cpu(), new) and torch.equal(got[1].cpu(), kept)
        assert torch.equal(x["weight_sum"].cpu(), sums) and torch.equal(_bits(x["k_cache"]), _bits(out["k_cache"]))


@pytest.mark.gpu
@pytest.mark.parametrize("extra_pages,budget", [(1, 250), (2100, 250), (1, 40)])
def test_graph_replays(tris, cuda, extra_pages, budget):
    """A captured call over lengths that grow past the limit, with eager calls and other work between its replays; a table
    of one workgroup a row and of several, a move of its own and with the choice."""
    ext = tris["ext"]
    a = evict_case(cuda, 2, 64, BF16, 16, [600, 300], seed=3, extra_pages=extra_pages)
    other = evict_case(cuda, 2, 64, BF16, 16, [500, 450], seed=4, extra_pages=extra_pages)
    args = dict(budget=budget, limit=290, sink=4, recent=20)
    a["seq_lens"].zero_()
    ext.paged_cache_evict(**a, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, kept = ext.paged_cache_evict(**a, **args)
    lens = [289, 295]
    for step in range(5):
        a["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        out, sums, want_new, want_kept = expected(a, **args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(new.cpu(), want_new) and torch.equal(kept.cpu(), want_kept)
        assert torch.equal(a["weight_sum"].cpu(), sums)
        for n in ("k_cache", "v_cache"):
            assert torch.equal(_bits(a[n]), _bits(out[n]))
        ext.paged_cache_evict(**other, budget=300 + step)
        lens = [n + 1 if n > 250 else 289 + i for i, n in enumerate(want_new.tolist())]
        a["weight_sum"].add_(torch.rand_like(a["weight_sum"]))


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    a = dict(evict_case(cuda, 2, 64, F16, 16, [100, 30]), budget=20)
    e = dict(evict_case(cuda, 2, 64, E4M3, 16, [100, 30]), budget=20)
    s, n = a["weight_sum"], a["weight_sum"].shape[2]
    bad = [
        (a, "budget <= limit", dict(budget=0)), (a, "budget <= limit", dict(limit=19)), (a, "budget <= limit", dict(budget=1 << 31)),
        (a, "within the budget", dict(sink=-1)), (a, "within the budget", dict(recent=-1)),
        (a, "within the budget", dict(sink=10, recent=11)), (a, "torch.float32", dict(weight_sum=s.half())),
        (a, "weight_sum must be", dict(weight_sum=s[..., :n - 1])), (a, "weight_sum must be", dict(weight_sum=s[:1])),
        (a, "rows of weight_sum overlap", dict(weight_sum=s[:1].expand(2, 2, n))),
        (a, "rows of weight_sum must be contiguous", dict(weight_sum=s.transpose(1, 2).contiguous().transpose(1, 2))),
        (a, "torch.int32", dict(seq_lens=a["seq_lens"].long())), (a, "CUDA", dict(k_cache=a["k_cache"].cpu())),
        (a, "cache rows overlap", dict(k_cache=a["k_cache"][:, :1].expand(a["k_cache"].shape))),
        (a, "belong to an e4m3 cache", dict(k_scale=torch.ones(1, device=cuda))), (e, "needs k_scale", dict(v_scale=None)),
        (e, "cache scales overlap", dict(k_scale=e["k_scale"][:, :1].expand(e["k_scale"].shape))),
        (a, "float16", dict(k_cache=a["k_cache"].float(), v_cache=a["v_cache"].float())),
        (a, "no gradient", dict(weight_sum=s.clone().requires_grad_())),
        (a, "no gradient", dict(k_cache=a["k_cache"].clone().requires_grad_())),
    ]
    for args, match, kw in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.paged_cache_evict(**{**args, **kw})


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(cache=None, sums=p, seq=96, head=48, budget=8, limit=8, sink=1, recent=2, lens=ctypes.c_void_p(8192), kept=p,
             ws=None, space=0):
        return lib.tris_paged_cache_evict(ctypes.byref(cache or c_cache()), sums, seq, head, budget, limit, sink, recent, lens,
                                          kept, ws, space, None)

    for kw, word in BAD_CACHES:
        if "dtype" not in kw or kw["dtype"] == 3:
            assert call(c_cache(**kw)) == -1 and word in lib.tris_last_error(), kw
    most = 2 ** 31 - 1
    need = lib.tris_paged_cache_evict_workspace_bytes(2, 2, 2049, 16, 8)
    assert need > 4 * 32784 * 4 and lib.tris_paged_cache_evict_workspace_bytes(2, 2, 16, 16, 8) == 0
    wide = dict(cache=c_cache(max_pages=2049, table_stride=2049), seq=65568, head=32784, ws=p, space=need)
    for bad in ((0, 2, 2049, 16, 8), (2, 0, 2049, 16, 8), (2, 2, -1, 16, 8), (2, 2, 2049, 0, 8), (2, 2, 2049, 16, 0)):
        assert lib.tris_paged_cache_evict_workspace_bytes(*bad) == 0
    for kw, word in ((dict(budget=0, limit=0), b"budget"), (dict(limit=7), b"budget"), (dict(sink=-1), b"within"),
                     (dict(recent=-1), b"within"), (dict(sink=7), b"within"), (dict(sink=most, recent=most), b"within"),
                     (dict(sums=None), b"null"), (dict(lens=None), b"null"), (dict(kept=None), b"null"),
                     (dict(lens=p), b"seq_lens"), (dict(seq=95), b"overlap"), (dict(head=47), b"overlap"),
                     (dict(seq=-96), b"overlap"), (dict(cache=c_cache(dtype=2)), b"e4m3"),
                     (dict(cache=c_cache(k_head_stride=0)), b"rows overlap"), (dict(cache=c_cache(v_page_stride=2048)), b"rows overlap"),
                     (dict(cache=c_cache(batch=1 << 26)), b"too many rows"),
                     (dict(wide, ws=None), b"workspace"), (dict(wide, space=need - 1), b"workspace"),
                     (dict(wide, ws=ctypes.c_void_p(4104)), b"workspace")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), (kw, lib.tris_last_error())
    assert call(c_cache(batch=0)) == 0
