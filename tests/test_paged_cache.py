"""ext.rotary_append_paged (tris_rotary_append_paged): rotation and append against the formula, in 64 bits and bit for
bit in 32, over types, head layouts, page sizes and orders, prompts and decode steps, padded batches, idle sequences,
pages outside the pool, special values, refusals."""
import ctypes

import pytest
import torch

from paged_cases import E4M3, make_pool, make_table

F16, BF16 = torch.float16, torch.bfloat16


def _tables(positions, rot, device):
    freq = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _turn(x, cos, sin, pos, dtype):
    """The formula in dtype, each product rounded; x [tokens, heads, dim]."""
    r = cos.shape[1]
    c, s = cos.to(dtype)[pos][:, None], sin.to(dtype)[pos][:, None]
    a, b = x[..., :r].to(dtype), x[..., r: 2 * r].to(dtype)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * r:].to(dtype)], -1)


def _case(cuda, q_heads, heads, dim, rot, dtype, cache, page, before, new, order="head", pad=0, seed=0, strided=False):
    gen = torch.Generator().manual_seed(seed)
    lengths = [b + n for b, n in zip(before, new)]
    pages = sum(-(-n // page) for n in lengths) + 2
    tokens = sum(new) + pad
    cols = (q_heads + 2 * heads) * dim + (8 if strided else 0)
    x = torch.randn((tokens, cols), generator=gen)
    x[:, torch.randperm(cols, generator=gen)[:8]] *= 20
    x = x.to(dtype).to(cuda)
    if strided:    # views of one projection's output
        q = x[:, : q_heads * dim].view(tokens, q_heads, dim)
        k = x[:, q_heads * dim: (q_heads + heads) * dim].view(tokens, heads, dim)
        v = x[:, (q_heads + heads) * dim: (q_heads + 2 * heads) * dim].view(tokens, heads, dim)
    else:
        q, k, v = (t.contiguous().view(tokens, -1, dim) for t in x.split([q_heads * dim, heads * dim, heads * dim], 1))
    table = make_table(lengths, page, pages, cuda, gen)
    kc, vc, ks, vs = make_pool(pages, heads, page, dim, cache, cuda, order)
    cos, sin = _tables(table.shape[1] * page, rot, cuda)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
    return dict(q=q, k=k, v=v, cos=cos, sin=sin, k_cache=kc, v_cache=vc, block_table=table,
                seq_lens=torch.tensor(lengths, dtype=torch.int32, device=cuda), query_start=starts, k_scale=ks,
                v_scale=vs)


def _expected(a, before, new):
    """Host copies of (q_out, k_cache, v_cache, k_scale, v_scale) after the append, by the formula in fp32."""
    c = {n: t.cpu() if t is not None else None for n, t in a.items()}
    page = c["k_cache"].shape[2]
    out = torch.zeros_like(c["q"])
    kc, vc = c["k_cache"].clone(), c["v_cache"].clone()
    scales = [None if s is None else s.clone() for s in (c["k_scale"], c["v_scale"])]
    at = 0
    for b, (m, n) in enumerate(zip(before, new)):
        rows, pos = slice(at, at + n), torch.arange(m, m + n)
        at += n
        if n == 0 or m < 0:
            continue
        out[rows] = _turn(c["q"][rows], c["cos"], c["sin"], pos, torch.float32).to(out.dtype)
        pg, slot = c["block_table"][b].long()[pos // page], pos % page
        good = (pg >= 0) & (pg < kc.shape[0])
        for x, cache, scale in ((_turn(c["k"][rows], c["cos"], c["sin"], pos, torch.float32), kc, scales[0]),
                                (c["v"][rows].float(), vc, scales[1])):
            x = x[good]
            if scale is not None:
                f = (x.abs().amax(-1) * torch.tensor(1.0 / 448.0, dtype=torch.float32)).clamp_min(2.0 ** -126)
                scale[pg[good], :, slot[good]] = f
                x = x / f[..., None]
            cache[pg[good], :, slot[good]] = x.to(cache.dtype)
    return out, kc, vc, scales[0], scales[1]


def _bits(t):
    t = t.detach().cpu().contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _same(got, want):
    assert got.dtype == want.dtype and got.shape == want.shape
    g, w = got.detach().cpu().float(), want.float()
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    # bit for bit where a number is held (a NaN may be any)
    assert torch.equal(_bits(got)[~torch.isnan(w)], _bits(want)[~torch.isnan(w)])


def _append_and_check(tris, a, before, new):
    want = _expected(a, before, new)          # before the call changes the cache
    q = tris["ext"].rotary_append_paged(**a)
    for got, w in zip((q, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"]), want):
        if w is not None:
            _same(got, w)
    return q


LAYOUTS = [(32, 8, 128, 128), (16, 16, 128, 128), (16, 2, 256, 64), (14, 2, 64, 64), (5, 1, 128, 16), (3, 3, 64, 48),
           (70, 2, 256, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("order,page", [("head", 16), ("token", 7), ("head", 1)])
def test_prompts(tris, cuda, layout, types, order, page):
    """Ragged prompts on caches of different lengths, one sequence without new tokens, padded rows behind."""
    before, new = [0, 5, 33, 17], [9, 1, 0, 40]
    print(f"[gpu-case] append {layout} {types} page={page} {order}", flush=True)
    a = _case(cuda, *layout, *types, page, before, new, order, pad=6, strided=page == 7)
    q = _append_and_check(tris, a, before, new)
    assert bool((q[sum(new):] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, E4M3])
@pytest.mark.parametrize("batch", [1, 3, 64, 130])
def test_decode_step(tris, cuda, batch, cache):
    """One token a sequence without query_start, and with it: the same; idle sequences store nothing."""
    before = [(37 * i) % 101 for i in range(batch)]
    a = _case(cuda, 8, 2, 128, 128, F16, cache, 16, before, [1] * batch, seed=batch)
    if batch > 2:
        a["seq_lens"][1] = 0
        before[1] = -1
    b = {n: t.clone() if n in ("k_cache", "v_cache", "k_scale", "v_scale") and t is not None else t for n, t in a.items()}
    q = _append_and_check(tris, a, before, [1] * batch)
    q2 = tris["ext"].rotary_append_paged(**{**b, "query_start": None})
    assert torch.equal(q, q2)
    for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if a[n] is not None:
            assert torch.equal(_bits(a[n]), _bits(b[n]))


@pytest.mark.gpu
def test_against_64_bits(tris, cuda):
    """Half a step of the type, and three fp32 roundings (two products, their sum) of the products' size; the e4m3
    element half a step (2^-4) or half its smallest step (2^-10), times the scale, which has two fp32 roundings."""
    before, new = [3000, 70000], [5, 64]
    for dtype, cache in ((F16, F16), (BF16, BF16), (BF16, E4M3)):
        a = _case(cuda, 4, 2, 128, 128, dtype, cache, 64, before, new)
        q = tris["ext"].rotary_append_paged(**a)
        c = {n: t.cpu() for n, t in a.items() if t is not None}
        at = 0
        for b, (m, n) in enumerate(zip(before, new)):
            pos, rows = torch.arange(m, m + n), slice(at, at + n)
            at += n
            for name, x in (("q", c["q"][rows]), ("k", c["k"][rows])):
                want = _turn(x, c["cos"], c["sin"], pos, torch.float64)
                size = _turn(x.abs(), c["cos"].abs(), -c["sin"].abs(), pos, torch.float64).abs()
                size = torch.maximum(size, _turn(x.abs(), c["cos"].abs(), c["sin"].abs(), pos, torch.float64).abs())
                bound = torch.finfo(dtype).eps / 2 * (1 + 1e-3) * want.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25
                if name == "q":
                    got = q[rows].cpu().double()
                else:
                    pg, slot = c["block_table"][b].long()[pos // 64], pos % 64
                    got = c["k_cache"].float()[pg, :, slot].double()
                    if cache == E4M3:
                        s = c["k_scale"][pg, :, slot].double()[..., None]
                        got = got * s
                        assert bool(((s[..., 0] / (want.abs().amax(-1) / 448) - 1).abs() < 2.0 ** -20).all())
                        bound = 2.0 ** -4 * (1 + 1e-3) * want.abs() + 2.0 ** -10 * s + 8 * 2.0 ** -24 * size
                assert bool(((got - want).abs() <= bound).all())


@pytest.mark.gpu
def test_pages_outside_the_pool_and_special_values(tris, cuda):
    before, new = [0, 20], [40, 13]
    for cache in (F16, E4M3):
        a = _case(cuda, 4, 2, 128, 128, F16, cache, 16, before, new)
        a["block_table"][0, 1] = a["k_cache"].shape[0]     # one past the pool
        a["block_table"][1, 1] = -3
        a["k"][2, 0, :], a["v"][2, 1, :] = 0.0, 0.0        # rows of zeros
        a["k"][3, 0, 77], a["v"][4, 0, 5] = float("inf"), float("nan")
        want = _expected(a, before, new)
        q = tris["ext"].rotary_append_paged(**a)
        _same(q, want[0])
        for got, w, scale in ((a["k_cache"], want[1], a["k_scale"]), (a["v_cache"], want[2], a["v_scale"])):
            if cache == F16:
                _same(got, w)
            else:   # an infinity: its row reads back as NaN, scale infinite and elements zero or NaN
                g = got.cpu().float() * scale.cpu()[..., None]
                w = w.float() * (want[3] if got is a["k_cache"] else want[4])[..., None]
                assert torch.equal(torch.isnan(g), torch.isnan(w))
                assert torch.equal(g[~torch.isnan(w)], w[~torch.isnan(w)])


@pytest.mark.gpu
def test_queries_in_place_given_and_absent(tris, cuda):
    ext = tris["ext"]
    before, new = [0, 3], [4, 2]
    a = _case(cuda, 6, 2, 64, 64, BF16, BF16, 16, before, new, pad=3)
    want = _expected(a, before, new)[0]
    q_in = a["q"].clone()
    given = torch.full_like(q_in, 7.0)
    assert ext.rotary_append_paged(**a, q_out=given) is given
    _same(given[:6], want[:6])
    assert bool((given[6:] == 7).all())                    # padded rows of a given buffer stay
    a["q"] = q_in
    same = ext.rotary_append_paged(**a, q_out=q_in)
    assert same is q_in
    _same(q_in[:6], want[:6])
    kc = a["k_cache"].clone()
    a["q"] = None
    a["k_cache"].fill_(0)
    assert ext.rotary_append_paged(**a) is None
    good = ~torch.isnan(kc.float())
    assert torch.equal(a["k_cache"][good], kc[good])


@pytest.mark.gpu
def test_graph_replays_with_new_positions(tris, cuda):
    ext = tris["ext"]
    before = [4, 0, 11]
    a = _case(cuda, 4, 2, 128, 128, F16, E4M3, 16, [b + 4 for b in before], [1] * 3)
    a["seq_lens"].sub_(4)
    ext.rotary_append_paged(**a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ext.rotary_append_paged(**a)
    for step in range(4):
        a["seq_lens"].add_(1)
        a["k"].mul_(0.5)
        want = _expected(a, [b + 1 + step for b in before], [1] * 3)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((q, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"]), want):
            _same(got, w)


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 128, 128, F16, F16, 16, [0, 3], [4, 2])
    wide = torch.zeros((6, 2, 192), dtype=F16, device=cuda)
    bad = [
        ("float16", dict(k=a["k"].float())),
        ("head_dim", dict(k=wide)),
        ("kv_heads", dict(k=a["k"][:, :1].contiguous(), v=a["v"][:, :1].contiguous())),
        ("number of tokens", dict(q=a["q"][:3])),
        ("positions", dict(cos=a["cos"][:8].contiguous(), sin=a["sin"][:8].contiguous())),
        ("multiple of 16", dict(cos=a["cos"][:, :12].contiguous(), sin=a["sin"][:, :12].contiguous())),
        ("one shape", dict(sin=a["sin"][:8].contiguous())),
        ("batch \\+ 1", dict(query_start=a["query_start"][:2].contiguous())),
        ("one token a sequence", dict(query_start=None)),
        ("torch.int32", dict(seq_lens=a["seq_lens"].long())),
        ("torch.int32", dict(block_table=a["block_table"].long())),
        ("belong to an e4m3 cache", dict(k_scale=torch.ones((1,), device=cuda))),
        ("needs k_scale", dict(k_cache=a["k_cache"].to(E4M3), v_cache=a["v_cache"].to(E4M3))),
        ("activations' type", dict(k_cache=a["k_cache"].to(BF16), v_cache=a["v_cache"].to(BF16))),
        ("contiguous", dict(k_cache=a["k_cache"].transpose(2, 3).contiguous().transpose(2, 3))),
        ("16-byte", dict(k_cache=torch.zeros(a["k_cache"].numel() + 4, dtype=F16, device=cuda)[4:].view(a["k_cache"].shape))),
        ("no gradient", dict(k=a["k"].clone().requires_grad_())),
    ]
    for match, kw in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.rotary_append_paged(**{**a, **kw})


def c_cache(**kw):
    from tris_moe_amd import _lib

    c = _lib.TrisPagedCache(k=4096, v=4096, block_table=4096, seq_lens=4096, num_pages=4, page_size=16, kv_heads=2,
                            head_dim=128, batch=2, max_pages=3, dtype=0, table_stride=3)
    for n in ("k", "v"):
        for field, s in (("page", 4096), ("head", 2048), ("slot", 128)):
            setattr(c, f"{n}_{field}_stride", s)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


BAD_CACHES = [
    (dict(head_dim=96), b"head_dim"), (dict(page_size=0), b"page_size"), (dict(num_pages=0), b"at least one page"),
    (dict(dtype=1), b"activations' type"), (dict(dtype=3), b"k_scale"), (dict(k_scale=4096), b"k_scale"),
    (dict(k=None), b"null"), (dict(block_table=None), b"null"), (dict(k=4104), b"16-byte"),
    (dict(v_slot_stride=132), b"16-byte"), (dict(max_pages=1 << 30), b"too wide"), (dict(v_page_stride=-8), b"16-byte"),
    (dict(k_slot_stride=1 << 27), b"slot stride"), (dict(table_stride=-1), b"table stride"),
]


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(cache=None, tokens=2, q_heads=4, rot=128, positions=48, starts=None, q_stride=512, act=0, k=p):
        return lib.tris_rotary_append_paged(p, q_stride, 128, k, 256, 128, p, 256, 128, act, tokens, q_heads, p, p, rot,
                                            positions, starts, ctypes.byref(cache or c_cache()), p, 512, 128, 0, None)

    for kw, word in BAD_CACHES:
        assert call(c_cache(**kw)) == -1 and word in lib.tris_last_error(), kw
    for kw, word in ((dict(tokens=3), b"one token a sequence"), (dict(tokens=-1), b"negative"), (dict(rot=24), b"rotary_dim"),
                     (dict(rot=144), b"rotary_dim"), (dict(rot=0), b"rotary_dim"), (dict(positions=47), b"positions"),
                     (dict(q_stride=516), b"16-byte"), (dict(act=2), b"fp16"), (dict(k=None), b"null"),
                     (dict(q_heads=1 << 30), b"heads")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), kw
    assert call(c_cache(batch=0), tokens=0) == 0
    with pytest.raises(RuntimeError, match="CUDA"):
        t = torch.zeros((1, 2, 128), dtype=F16)
        tris["ext"].rotary_append_paged(t, t, t, t, t, t, t, t, t)
