"""The norm, the append and the paged attention at calls that the other files do not make: many query heads a kv head at
every head dimension, pools past 4 GiB, layer and key / value slices of one pool, expanded rows, outputs over inputs,
windows past 32 bits, tensors of another device than the current one, long page tables, calls side by side."""
import ctypes

import pytest
import torch

from paged_cases import E4M3, rows_of
from test_paged_attention import _case, _check
from test_paged_cache import _bits, _case as _append_case, _expected, _same

F16, BF16 = torch.float16, torch.bfloat16


def test_launch_makes_the_tensors_device_current(tris, monkeypatch):
    ext, seen = tris["ext"], []

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            seen.append(("enter", self.i))

        def __exit__(self, *a):
            seen.append(("exit", self.i))

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    assert ext._launch(0, lambda a, b: a + b, 1, 2) == 3 and seen == []
    assert ext._launch(1, lambda a: seen.append("call") or a, 5) == 5
    assert seen == [("enter", 1), "call", ("exit", 1)]


def test_launches_past_their_thread_count_are_refused(tris):
    """A launch has less than 2^32 threads; what would need more is refused before it, with a message."""
    from test_paged_cache import c_cache
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)
    for width, rows in ((128, 1 << 28), (4096, 1 << 24), (32768, 1 << 22), (64, 1 << 32)):
        assert lib.tris_rms_norm(p, 0, width, None, 0, 0, p, 0, 0.0, 1e-6, rows, width, p, 0, width, None, 0, None) == -1
        assert b"too many rows" in lib.tris_last_error()
    c = c_cache(batch=1 << 27)
    assert lib.tris_rotary_append_paged(p, 512, 128, p, 256, 128, p, 256, 128, 0, 1 << 27, 4, p, p, 128, 48, None,
                                        ctypes.byref(c), p, 512, 128, 0, None) == -1
    assert b"too many tokens" in lib.tris_last_error()
    args = (0.1, 0, p, 512, 128, p, 1 << 60, None)
    assert lib.tris_paged_attention_decode(p, 512, 128, 0, 4, ctypes.byref(c), *args) == -1
    assert b"too many rows" in lib.tris_last_error()
    c = c_cache(batch=1 << 20, max_pages=1 << 20)
    assert lib.tris_paged_attention_decode(p, 512, 128, 0, 4, ctypes.byref(c), *args) == -1
    assert b"too many positions" in lib.tris_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F16, E4M3)], ids=str)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("heads", [(16, 1), (40, 2)], ids=str)
@pytest.mark.parametrize("page", [16, 11])
def test_many_query_heads(tris, cuda, types, dim, heads, page):
    print(f"[gpu-case] attention heads={heads} dim={dim} {types} page={page}", flush=True)
    lengths = [700, 0, 33, 1]
    a = _case(cuda, *heads, dim, *types, page, lengths, seed=dim + page)
    _check(a, lengths, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
@pytest.mark.parametrize("types,page", [((F16, F16), 16), ((BF16, BF16), 9), ((F16, E4M3), 16)], ids=str)
def test_pool_past_four_gib(tris, cuda, types, page):
    """Rows whose offset needs more than 32 bits, in elements too: stored and read back.  The pool's other pages hold
    whatever the memory held."""
    ext, heads, dim = tris["ext"], 8, 128
    size = 1 if types[1] == E4M3 else 2
    pages = (5 << 30) // (heads * page * dim * size) * (2 if size == 2 else 1)
    kc, vc = (torch.empty((pages, heads, page, dim), dtype=types[1], device=cuda) for _ in range(2))
    assert kc.numel() > 1 << 32
    ks, vs = (torch.empty((pages, heads, page), device=cuda) if size == 1 else None for _ in range(2))
    lengths, g = [70, 40], torch.Generator().manual_seed(2)
    table = torch.full((2, 8), -1, dtype=torch.int32)
    table[0, : -(-70 // page)] = pages - 1 - torch.arange(-(-70 // page), dtype=torch.int32) * 3
    table[1, : -(-40 // page)] = pages // 2 + torch.arange(-(-40 // page), dtype=torch.int32)
    a = dict(k_cache=kc, v_cache=vc, block_table=table.to(cuda),
             seq_lens=torch.tensor(lengths, dtype=torch.int32, device=cuda), k_scale=ks, v_scale=vs)
    k, v = (torch.randn((110, heads, dim), generator=g).to(types[0]).to(cuda) for _ in range(2))
    cos, sin = torch.ones((8 * page, 64), device=cuda), torch.zeros((8 * page, 64), device=cuda)   # no rotation
    ext.rotary_append_paged(None, k, v, cos, sin, query_start=torch.tensor([0, 70, 110], dtype=torch.int32, device=cuda), **a)
    q = torch.randn((2, 16, dim), generator=g).to(types[0]).to(cuda)
    got = ext.paged_attention_decode(q, **a)
    # the same rows in a small pool
    used = torch.unique(table[table >= 0]).to(cuda)
    small = torch.full_like(a["block_table"], -1)
    for i, p in enumerate(used.tolist()):
        small[a["block_table"] == p] = i
    b = dict(a, q=q, k_cache=kc[used.long()] if size == 2 else kc.view(torch.uint8)[used.long()].view(E4M3),
             v_cache=vc[used.long()] if size == 2 else vc.view(torch.uint8)[used.long()].view(E4M3), block_table=small,
             k_scale=None if ks is None else ks[used.long()], v_scale=None if vs is None else vs[used.long()])
    assert torch.equal(ext.paged_attention_decode(**b), got)
    _check(b, lengths, got)
    if size == 2:
        for s, (lo, n) in enumerate(((0, 70), (70, 40))):
            assert torch.equal(rows_of(b["k_cache"], None, small, s, n, page).permute(1, 0, 2), k[lo: lo + n].cpu().double())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, E4M3])
@pytest.mark.parametrize("page", [16, 5])
def test_slices_of_one_pool(tris, cuda, cache, page):
    """A layer's slice of a pool that holds keys and values side by side: strides of their own for pages, heads and
    slots; the other layer stays as it was."""
    ext, lengths = tris["ext"], [50, 3, 0, 81]
    a = _append_case(cuda, 8, 2, 128, 128, F16, cache, page, [0, 1, 0, 60], [50, 2, 0, 21])
    pages = a["k_cache"].shape[0]
    pool = torch.zeros((pages, 2, 2, 2, page, 128), dtype=torch.uint8 if cache == E4M3 else cache, device=cuda)
    pool = pool.view(E4M3) if cache == E4M3 else pool                            # [page, layer, k / v, head, slot, dim]
    scales = torch.zeros((pages, 2, 2, 2, page), device=cuda)
    b = dict(a, k_cache=pool[:, 1, 0], v_cache=pool[:, 1, 1])
    if cache == E4M3:
        b.update(k_scale=scales[:, 1, 0], v_scale=scales[:, 1, 1])
    want = _expected(a, [0, 1, -1, 60], [50, 2, 0, 21])
    q = ext.rotary_append_paged(**b)
    _same(q, want[0])
    for got, w in ((b["k_cache"], want[1]), (b["v_cache"], want[2])):
        stored = ~torch.isnan(w.float())
        assert torch.equal(_bits(got)[stored], _bits(w)[stored])
    assert bool((pool[:, 0].view(torch.uint8) == 0).all()) and bool((scales[:, 0] == 0).all())
    state = {n: b[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens")}
    state["q"] = torch.randn((4, 8, 128), generator=torch.Generator().manual_seed(4)).to(F16).to(cuda)
    _check(state, lengths, ext.paged_attention_decode(**state))


@pytest.mark.gpu
def test_output_over_the_queries(tris, cuda):
    ext, lengths = tris["ext"], [3000, 40, 0, 1]
    for heads in ((8, 2), (40, 1)):
        a = _case(cuda, *heads, 128, F16, F16, 16, lengths)
        want = ext.paged_attention_decode(**a)
        q = a["q"].clone()
        assert ext.paged_attention_decode(**{**a, "q": q}, out=q) is q
        assert torch.equal(q, want)


@pytest.mark.gpu
def test_window_past_32_bits(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 128, F16, F16, 16, [300, 20])
    want = ext.paged_attention_decode(**a)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 300):
        assert torch.equal(ext.paged_attention_decode(**a, window=window), want)
    for window in (-1, -2 ** 32 + 5):
        with pytest.raises(RuntimeError, match="negative window"):
            ext.paged_attention_decode(**a, window=window)


@pytest.mark.gpu
def test_wide_tables_and_large_batches(tris, cuda):
    """Tables far wider than the sequences are long, and batches over several wavefronts of sequences."""
    for lengths, wide in (([17, 0, 100], 60000), ([(7 * i) % 50 for i in range(1000)], 40)):
        a = _case(cuda, 4, 2, 64, BF16, BF16, 16, lengths, seed=len(lengths))
        table = torch.full((len(lengths), wide), -1, dtype=torch.int32, device=cuda)
        table[:, : a["block_table"].shape[1]] = a["block_table"]
        a["block_table"] = table
        _check(a, lengths, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
def test_norm_of_expanded_and_overlapping_rows(tris, cuda):
    ext, g = tris["ext"], torch.Generator().manual_seed(8)
    w = torch.randn(256, generator=g).to(BF16).to(cuda)
    row = torch.randn((1, 256), generator=g).to(BF16).to(cuda)
    one = ext.rms_norm(row, w, 1e-6)
    assert torch.equal(ext.rms_norm(row.expand(5, 256), w, 1e-6), one.expand(5, 256))
    x = torch.randn((5, 256), generator=g).to(BF16).to(cuda)
    got, stream = ext.rms_norm(x, w, 1e-6, residual=row.expand(5, 256))
    want, want_stream = ext.rms_norm(x, w, 1e-6, residual=row.expand(5, 256).contiguous())
    assert torch.equal(got, want) and torch.equal(stream, want_stream)
    flat = torch.randn(1024, generator=g).to(BF16).to(cuda)
    slid = flat.as_strided((7, 256), (64, 1))                 # rows that share values: inputs may
    assert torch.equal(ext.rms_norm(slid, w, 1e-6), ext.rms_norm(slid.contiguous(), w, 1e-6))


@pytest.mark.gpu
def test_graphs_of_one_pool_and_eager_calls_between(tris, cuda):
    """Two captured calls that share an allocation pool, replayed in turn with eager calls between."""
    ext = tris["ext"]
    a = _case(cuda, 8, 2, 128, BF16, BF16, 16, [2500, 7, 900])
    b = _case(cuda, 4, 4, 64, F16, E4M3, 10, [33, 4000], seed=3)
    want_a, want_b = ext.paged_attention_decode(**a), ext.paged_attention_decode(**b)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got_a = ext.paged_attention_decode(**a)
    with torch.cuda.graph(second, pool=first.pool()):
        got_b = ext.paged_attention_decode(**b)
    for _ in range(3):
        first.replay()
        torch.cuda.synchronize()
        assert torch.equal(got_a, want_a)
        assert torch.equal(ext.paged_attention_decode(**b), want_b)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(got_b, want_b)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("dim,longest", [(64, 900), (128, 470), (256, 230)])
@pytest.mark.parametrize("page", [16, 6])
def test_narrow_tables(tris, cuda, types, dim, longest, page):
    """Block tables narrow enough for one launch without a workspace, and the same sequences with a wider table, which
    are split; small batches and ones with a workgroup for each CU."""
    from tris_moe_amd import _lib

    need = _lib.load().tris_paged_attention_workspace_bytes
    for batch, heads in ((9, (8, 2)), (70, (10, 5))):
        print(f"[gpu-case] attention {types} dim={dim} page={page} batch={batch} narrow and wide", flush=True)
        lengths = [(37 * i * i) % longest for i in range(batch)]
        lengths[1] = longest
        a = _case(cuda, *heads, dim, *types, page, lengths, seed=batch)
        assert need(batch, *heads, dim, a["block_table"].shape[1], page) == 0
        _check(a, lengths, tris["ext"].paged_attention_decode(**a))
        _check(a, lengths, tris["ext"].paged_attention_decode(**a, window=40), window=40)
        wide = torch.full((batch, 3000), -1, dtype=torch.int32, device=cuda)
        wide[:, : a["block_table"].shape[1]] = a["block_table"]
        a["block_table"] = wide
        assert need(batch, *heads, dim, 3000, page) > 0
        _check(a, lengths, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
def test_workspace_too_small_is_refused(tris, cuda):
    from tris_moe_amd import _lib

    lib = _lib.load()
    a = _case(cuda, 4, 2, 128, F16, F16, 16, [3000])
    cache, (batch, pages, page, heads, dim) = tris["ext"]._paged_cache(
        "t", a["k_cache"], a["v_cache"], a["block_table"], a["seq_lens"], None, None, a["q"].get_device())
    need = lib.tris_paged_attention_workspace_bytes(batch, 4, heads, dim, pages, page)
    ws, out = torch.empty(need, dtype=torch.uint8, device=cuda), torch.full_like(a["q"], 7.0)
    stream = torch.cuda.current_stream(cuda).cuda_stream
    for p, size in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 8, need)):
        rc = lib.tris_paged_attention_decode(a["q"].data_ptr(), 512, 128, 0, 4, cache, 0.1, 0, out.data_ptr(), 512, 128, p,
                                             size, stream)
        assert rc == -1 and b"workspace" in lib.tris_last_error()
    torch.cuda.synchronize()
    assert bool((out == 7).all())
