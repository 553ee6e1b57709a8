"""Given rotary positions, sums of weights and eviction at their borders: tables far wider than sequences, large batches,
offsets past 32 bits, gradients refused on every tensor, sections that are no counts."""
import pytest
import torch

from paged_cases import E4M3, rows_of
from test_attention_weights import _sums, check_sums
from test_paged_attention import _case as attention_case
from test_paged_attention import _check
from test_paged_cache import _case as append_case
from test_paged_evict import NAMES, evict_case, run_and_check
from test_rotary_axes import _positions, _run

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,wide", [([17, 0, 100], 60000), ([2000, 900], 9000), ([(7 * i) % 50 for i in range(1000)], 40)],
                         ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}x{max(v)}")
def test_wide_tables_and_large_batches(tris, cuda, lengths, wide):
    """Entries past a sequence's pages are never followed; sums past it stay as they were, also those that the table has no
    places for."""
    ext = tris["ext"]
    a = attention_case(cuda, 4, 2, 64, BF16, BF16, 16, lengths, seed=len(lengths))
    table = torch.full((len(lengths), wide), -1, dtype=torch.int32, device=cuda)
    table[:, : a["block_table"].shape[1]] = a["block_table"]
    a["block_table"] = table
    sums = _sums(a, 5)
    before = sums.clone()
    y = ext.paged_attention_decode(**a, weight_sum=sums)
    _check(a, lengths, y)
    check_sums(a, lengths, before, sums)
    e = evict_case(cuda, 2, 64, F16, 16, lengths, seed=wide, extra_pages=wide - -(-max(lengths) // 16))
    run_and_check(tris, e, 12, 20, 2, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, E4M3])
def test_offsets_past_32_bits(tris, cuda, cache):
    """Pages 2 GiB and more apart, sums of one sequence 4 GiB after another's."""
    ext = tris["ext"]
    lengths, page, heads, dim = [40, 33], 16, 2, 64
    step = (1 << 30) + 64                                  # elements between pages
    a = attention_case(cuda, 4, heads, dim, BF16 if cache == E4M3 else F16, cache, page, lengths)
    a["block_table"] = torch.tensor([[4, 0, 2], [1, 3, 5]], dtype=torch.int32, device=cuda)
    big = {}
    g = torch.Generator().manual_seed(2)
    for n in ("k_cache", "v_cache"):
        raw = torch.empty(5 * step + heads * page * dim, dtype=torch.uint8 if cache == E4M3 else F16, device=cuda)
        x = torch.randn((6, heads, page, dim), generator=g).to(cache)
        big[n] = raw.view(cache).as_strided((6, heads, page, dim), (step, page * dim, dim, 1))
        for p in range(6):
            big[n][p].copy_(x[p])
    a.update(big)
    if cache == E4M3:
        for n in ("k_scale", "v_scale"):
            a[n] = torch.rand((6, heads, page), generator=g).to(cuda)
    store = torch.zeros((1 << 30) + 256, dtype=torch.float32, device=cuda)
    sums = store.as_strided((2, heads, 48), (1 << 30, 100, 1))
    before = sums.clone()
    y = ext.paged_attention_decode(**a, weight_sum=sums)
    small = {n: a[n].contiguous() for n in ("k_cache", "v_cache")}
    _check({**a, **small}, lengths, y)
    check_sums({**a, **small}, lengths, before, sums)
    e = {n: a[n] for n in (*NAMES, "block_table", "seq_lens")}
    run_and_check(tris, dict(e, weight_sum=sums), 20, None, 2, 5)
    new = append_case(cuda, 4, heads, dim, dim, a["q"].dtype, cache, page, [39, 32], [1, 1])
    new.update({n: a[n] for n in (*NAMES, "block_table")})
    _run(tris, new, [39, 32], [1, 1], _positions(2, 2, new["cos"].shape[0], cuda), (20, 12), False)


@pytest.mark.gpu
def test_gradients_are_refused_on_every_tensor(tris, cuda):
    import torch.autograd.forward_ad as fwd

    ext = tris["ext"]
    append = dict(append_case(cuda, 4, 2, 64, 64, F16, E4M3, 16, [0, 3], [4, 2]), positions=_positions(2, 6, 8, cuda),
                  sections=(20, 12))
    attend = attention_case(cuda, 4, 2, 64, F16, E4M3, 16, [10, 3])
    attend["weight_sum"] = _sums(attend)
    evict = dict(evict_case(cuda, 2, 64, E4M3, 16, [100, 30]), budget=20)
    plain = dict(evict_case(cuda, 2, 64, F16, 16, [100, 30]), budget=20)
    for call, args in ((ext.rotary_append_paged, append), (ext.paged_attention_decode, attend),
                       (ext.paged_cache_evict, evict), (ext.paged_cache_evict, plain)):
        names = [n for n, t in args.items() if isinstance(t, torch.Tensor) and t.dtype in (F16, torch.float32)]
        assert len(names) >= 3
        for n in names:
            leaf = args[n].detach().clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: leaf})
            with torch.no_grad():
                call(**{**args, n: leaf})
            with fwd.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: fwd.make_dual(args[n], torch.ones_like(args[n]))})


def test_sections_are_counts(tris):
    import numpy as np

    def sections(counts):
        return tris["ext"]._sections("op", counts)

    assert list(sections((16, 8, 8))) == [16, 8, 8] and list(sections(tuple(np.array([16, 16])))) == [16, 16]
    for bad in ((16.0, 16), ("a",), (2 ** 32 + 32,), (-(2 ** 40), 32), (None,)):
        with pytest.raises(RuntimeError, match="op: sections"):
            sections(bad)


@pytest.mark.gpu
def test_evicted_cache_is_read_and_appended_to(tris, cuda):
    """What attention reads after an eviction is what stayed, and nothing that the evicted pages still hold."""
    ext = tris["ext"]
    lengths, page, budget = [150, 90], 16, 48
    a = attention_case(cuda, 4, 2, 64, F16, F16, page, lengths)
    sums = _sums(a)
    ext.paged_attention_decode(**a, weight_sum=sums)
    rows = [[rows_of(a[f"{n}_cache"], None, a["block_table"], b, m, page) for n in "kv"] for b, m in enumerate(lengths)]
    caches = {n: a[n] for n in (*NAMES, "block_table", "seq_lens")}
    lens, kept = ext.paged_cache_evict(**caches, weight_sum=sums, budget=budget, sink=4, recent=10)
    a["seq_lens"] = lens
    _check(a, [budget, budget], ext.paged_attention_decode(**a))
    for b in range(2):
        for t, before in zip("kv", rows[b]):
            now = rows_of(a[f"{t}_cache"], None, a["block_table"], b, budget, page)
            for h in range(2):
                assert torch.equal(now[h], before[h][kept[b, h].cpu().long()])
    assert not bool(sums[0, :, budget:150].any()) and not bool(sums[1, :, budget:90].any())


@pytest.mark.gpu
@pytest.mark.parametrize("extra_pages", [1, 1200], ids=["one workgroup", "segments"])
def test_the_largest_budget(tris, cuda, extra_pages):
    """A budget of 2^31 - 1: no sequence is due, nothing moves, and every one of its places says so."""
    a = evict_case(cuda, 1, 64, F16, 16, [200], seed=3, extra_pages=extra_pages)
    before = {n: a[n].clone() for n in ("k_cache", "v_cache", "weight_sum")}
    new, kept = tris["ext"].paged_cache_evict(**a, budget=2 ** 31 - 1)
    assert new.tolist() == [200] and kept.shape == (1, 1, 2 ** 31 - 1)
    for part in kept[0, 0].split(1 << 28):
        assert bool((part == -1).all())
    for n, t in before.items():
        raw = torch.int16 if t.element_size() == 2 else torch.int32
        assert torch.equal(t.view(raw), a[n].view(raw)), n


def test_workspace_of_budgets_past_the_table(tris):
    """No sums move where no sequence can be due."""
    from tris_moe_amd import _lib

    need = _lib.load().tris_paged_cache_evict_workspace_bytes
    assert need(1, 1, 1213, 16, 1213 * 16) == need(1, 1, 1213, 16, 2 ** 31 - 1)
    assert need(1, 1, 1213, 16, 1213 * 16 - 1) == need(1, 1, 1213, 16, 1213 * 16) + 4 * (1213 * 16 - 1)


@pytest.mark.parametrize("kw", [{}, dict(dtype=3, v=8192, k_scale=4096, v_scale=4096)], ids=["rows", "scales"])
def test_keys_that_are_the_values_are_refused(tris, kw):
    """Both would be moved in the same memory at the same time."""
    import ctypes

    from test_paged_cache import c_cache
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)
    c = c_cache(**kw)
    for n in ("k", "v"):
        for field, stride in (("page", 32), ("head", 16), ("slot", 1)):
            setattr(c, f"{n}_scale_{field}_stride", stride)
    rc = lib.tris_paged_cache_evict(ctypes.byref(c), p, 96, 48, 8, 8, 1, 2, ctypes.c_void_p(8192), p, None, 0, None)
    assert rc == -1 and b"share memory" in lib.tris_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cache,shared", [(F16, "cache"), (E4M3, "scale")], ids=["rows", "scales"])
def test_a_pool_given_twice_is_refused(tris, cuda, cache, shared):
    a = evict_case(cuda, 2, 64, cache, 16, [100, 30])
    a[f"v_{shared}"] = a[f"k_{shared}"]
    with pytest.raises(RuntimeError, match="share memory"):
        tris["ext"].paged_cache_evict(**a, budget=20)
