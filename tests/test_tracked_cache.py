"""PagedKVCache with sums of attention weights under block tables of fewer rows than it was made for: a serving loop whose
batch shrinks, or whose steps are captured for several batch sizes."""
import pytest
import torch

from paged_cases import E4M3
from test_paged_cache import _bits

F16 = torch.float16


@pytest.mark.parametrize("rows,got", [(4, 4), (3, 3), (1, 1), (0, 0), (5, 4)])
def test_rows_of_the_sums(tris, monkeypatch, rows, got):
    """The first rows are the block table's; of more rows than there are the operators are left to say so."""
    from tris_moe_amd import attention

    seen = []
    monkeypatch.setattr(attention.ext, "paged_attention_decode", lambda *a, **kw: seen.append(kw["weight_sum"]))
    monkeypatch.setattr(attention.ext, "paged_cache_evict", lambda *a, **kw: seen.append(a[4]))
    cache = attention.PagedKVCache(3, 5, 2, 64, F16, device="cpu")
    table, lens = torch.zeros((rows, 3), dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    cache.attend(None, table, lens)
    assert seen.pop() is None
    cache.track_weights(4, 15)
    cache.attend(None, table, lens)
    cache.evict(table, lens, 4)
    for s in seen:
        assert s.shape == (got, 2, 15) and s.data_ptr() == cache.weight_sum.data_ptr() or got == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, E4M3])
def test_smaller_batches(tris, cuda, dtype):
    """Steps of four, two and three rows: sums, evictions and caches as the operators' own calls give them on the rows."""
    from tris_moe_amd import attention

    ext = tris["ext"]
    heads, q_heads, dim, page, pages = 2, 6, 64, 16, 24
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(pages, generator=g).view(4, 6).to(torch.int32).to(cuda)
    cos, sin = attention.rotary_tables(dim, 96, device=cuda)
    cache, plain = (attention.PagedKVCache(pages, page, heads, dim, dtype, cuda) for _ in range(2))
    lens = torch.tensor([40, 33, 20, 7], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 40, 73, 93, 100], dtype=torch.int32, device=cuda)
    k, v = (torch.randn((100, heads, dim), generator=g).to(F16).to(cuda) for _ in range(2))
    for c in (cache, plain):
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t.zero_()
        c.append(None, k, v, cos, sin, table, lens, starts)
    cache.track_weights(4, 96)
    sums = torch.zeros_like(cache.weight_sum)
    scales = dict(k_scale=plain.k_scale, v_scale=plain.v_scale)
    for rows in (4, 2, 3):
        q = torch.randn((rows, q_heads, dim), generator=g).to(F16).to(cuda)
        n, before = lens[:rows], cache.weight_sum.clone()
        y = cache.attend(q, table[:rows], n)
        want = ext.paged_attention_decode(q, plain.k, plain.v, table[:rows], n, **scales, weight_sum=sums[:rows])
        assert torch.equal(y, want) and torch.equal(cache.weight_sum, sums)
        assert torch.equal(sums[rows:], before[rows:]) and not torch.equal(sums[:rows], before[:rows])
        got = cache.evict(table[:rows], n, 24, 30, 2, 5)
        want = ext.paged_cache_evict(plain.k, plain.v, table[:rows], n, sums[:rows], 24, 30, 2, 5, **scales)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for name in ("k", "v", "k_scale", "v_scale", "weight_sum"):
            x, z = getattr(cache, name), sums if name == "weight_sum" else getattr(plain, name)
            assert x is None or torch.equal(_bits(x), _bits(z))
        lens[:rows] = got[0] + 4
    with pytest.raises(RuntimeError, match="weight_sum must be"):
        cache.attend(torch.zeros((5, q_heads, dim), dtype=F16, device=cuda), torch.cat([table, table[:1]]),
                     torch.zeros(5, dtype=torch.int32, device=cuda))
