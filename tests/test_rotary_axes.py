"""ext.rotary_append_paged with positions of its own (tris_rotary_axes_append_paged): against the formula bit for bit in
fp32 and in 64 bits, over axes, sections in a row and interleaved, head layouts, types, prompts and decode steps, positions
outside the tables, strides, graphs, refusals."""
import ctypes

import pytest
import torch

from paged_cases import E4M3
from test_paged_cache import BAD_CACHES, LAYOUTS, _bits, _case, _expected, _same, c_cache

F16, BF16 = torch.float16, torch.bfloat16


def pair_axes(sections, interleaved, half):
    """The formula's axis of each pair."""
    if not interleaved:
        return torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    n = len(sections)
    return torch.tensor([i % n if i // n < sections[i % n] else 0 for i in range(half)])


def turn_axes(x, cos, sin, positions, sections, interleaved, dtype):
    """The formula in dtype, each product rounded; x [tokens, heads, dim], positions [axes, tokens]."""
    r = cos.shape[1]
    at, pair = positions.long()[pair_axes(sections, interleaved, r)].T, torch.arange(r)
    c, s = cos.to(dtype)[at, pair][:, None], sin.to(dtype)[at, pair][:, None]
    a, b = x[..., :r].to(dtype), x[..., r: 2 * r].to(dtype)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * r:].to(dtype)], -1)


def _sections(half, axes):
    first = half - (axes - 1) * (half // axes)
    return (first,) + (half // axes,) * (axes - 1)


def expected_axes(a, before, new, positions, sections, interleaved):
    """Host copies of (q_out, k_cache, v_cache, k_scale, v_scale) after the append, by the formula in fp32.  A token with a
    position outside the tables has no place."""
    c = {n: t.cpu() if t is not None else None for n, t in a.items()}
    pos, rows = positions.cpu(), c["cos"].shape[0]
    good = ((pos >= 0) & (pos < rows)).all(0)
    args = (c["cos"], c["sin"], pos.clamp(0, rows - 1), sections, interleaved, torch.float32)
    q, k = turn_axes(c["q"], *args), turn_axes(c["k"], *args)
    out, kc, vc = torch.zeros_like(c["q"]), c["k_cache"].clone(), c["v_cache"].clone()
    scales = [None if s is None else s.clone() for s in (c["k_scale"], c["v_scale"])]
    page, at = kc.shape[2], 0
    for b, (m, n) in enumerate(zip(before, new)):
        rows = torch.arange(at, at + n)
        place = torch.arange(m, m + n)
        at += n
        keep = good[rows] & (place >= 0)
        rows, place = rows[keep], place[keep]
        out[rows] = q[rows].to(out.dtype)
        pg, slot = c["block_table"][b].long()[place // page], place % page
        inside = (pg >= 0) & (pg < kc.shape[0])
        rows, pg, slot = rows[inside], pg[inside], slot[inside]
        for x, cache, scale in ((k[rows], kc, scales[0]), (c["v"][rows].float(), vc, scales[1])):
            if scale is not None:
                f = (x.abs().amax(-1) * torch.tensor(1.0 / 448.0, dtype=torch.float32)).clamp_min(2.0 ** -126)
                scale[pg, :, slot] = f
                x = x / f[..., None]
            cache[pg, :, slot] = x.to(cache.dtype)
    return out, kc, vc, scales[0], scales[1]


def _run(tris, a, before, new, positions, sections, interleaved, **kw):
    want = expected_axes(a, before, new, positions if positions.ndim == 2 else positions[None], sections, interleaved)
    q = tris["ext"].rotary_append_paged(**a, positions=positions, sections=sections, interleaved=interleaved, **kw)
    for got, w in zip((q, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"]), want):
        if w is not None:
            _same(got, w)
    return q


def _positions(axes, tokens, rows, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, rows, (axes, tokens), generator=g, dtype=torch.int32).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
def test_prompts(tris, cuda, layout, types, axes):
    """Ragged prompts, one sequence without new tokens, padded rows behind; tables of other lengths than the cache."""
    before, new = [0, 5, 33, 17], [9, 1, 0, 40]
    half = layout[3] // 2
    for order, page, interleaved in (("head", 16, False), ("token", 7, True)):
        print(f"[gpu-case] axes {layout} {types} axes={axes} page={page} {interleaved}", flush=True)
        a = _case(cuda, *layout, *types, page, before, new, order, pad=6, strided=page == 7)
        if page == 7:
            a["cos"], a["sin"] = a["cos"][:23].contiguous(), a["sin"][:23].contiguous()
        p = _positions(axes, sum(new) + 6, a["cos"].shape[0], cuda, axes)
        q = _run(tris, a, before, new, p, _sections(half, axes), interleaved)
        assert bool((q[sum(new):] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("sections", [(64, 0, 0), (0, 64), (1, 62, 1), (16, 24, 24), (3, 5, 7, 49), (40, 8, 16)], ids=str)
def test_sections_in_a_row(tris, cuda, sections):
    a = _case(cuda, 4, 2, 128, 128, F16, F16, 16, [3, 0], [20, 7])
    _run(tris, a, [3, 0], [20, 7], _positions(len(sections), 27, 32, cuda), sections, False)


@pytest.mark.gpu
@pytest.mark.parametrize("sections", [(64, 0, 0), (32, 32), (22, 21, 21), (24, 20, 20), (40, 3, 21), (16, 16, 16, 16), (60, 4)],
                         ids=str)
def test_interleaved_sections(tris, cuda, sections):
    a = _case(cuda, 4, 2, 128, 128, F16, F16, 16, [3, 0], [20, 7])
    _run(tris, a, [3, 0], [20, 7], _positions(len(sections), 27, 32, cuda), sections, True)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, E4M3])
@pytest.mark.parametrize("batch", [1, 3, 130])
def test_decode_step(tris, cuda, batch, cache):
    """One token a sequence, positions past the cache's places and tables longer than it; one idle sequence; the places
    themselves as positions give what the append without positions gives."""
    before = [(37 * i) % 101 for i in range(batch)]
    a = _case(cuda, 8, 2, 128, 128, F16, cache, 16, before, [1] * batch, seed=batch)
    freq = 1e4 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    angle = torch.arange(5000, dtype=torch.float64)[:, None] * freq
    a.update(cos=angle.cos().float().to(cuda), sin=angle.sin().float().to(cuda), query_start=None)
    if batch > 2:
        a["seq_lens"][1] = 0
        before[1] = -1
    saved = {n: None if a[n] is None else a[n].clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    _run(tris, a, before, [1] * batch, _positions(1, batch, 5000, cuda)[0], (64,), False)
    plain = {**a, **{n: None if t is None else t.clone() for n, t in saved.items()}}
    q = tris["ext"].rotary_append_paged(**plain)
    given = {**a, **saved}
    own = torch.tensor([max(m, 0) for m in before], dtype=torch.int32, device=cuda)
    for p, s in ((own, None), (own[None], None), (own.expand(3, -1), (22, 21, 21))):
        got = tris["ext"].rotary_append_paged(**given, positions=p, sections=s, interleaved=s is not None)
        assert torch.equal(_bits(got), _bits(q))
        for n, t in saved.items():
            if t is not None:
                assert torch.equal(_bits(t), _bits(plain[n]))


@pytest.mark.gpu
def test_against_64_bits(tris, cuda):
    """Half a step of the type, and three fp32 roundings (two products, their sum) of the products' size, at far
    positions."""
    before, new = [30, 700], [5, 64]
    for dtype in (F16, BF16):
        a = _case(cuda, 4, 2, 128, 128, dtype, dtype, 64, before, new)
        freq = 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
        angle = torch.arange(90000, dtype=torch.float64)[:, None] * freq
        a.update(cos=angle.cos().float().to(cuda), sin=angle.sin().float().to(cuda))
        p = 80000 + _positions(3, 69, 10000, "cpu")
        for interleaved in (False, True):
            q = tris["ext"].rotary_append_paged(**a, positions=p.to(cuda), sections=(24, 20, 20), interleaved=interleaved)
            x, cos, sin = a["q"].cpu(), a["cos"].cpu(), a["sin"].cpu()
            want = turn_axes(x, cos, sin, p, (24, 20, 20), interleaved, torch.float64)
            size = turn_axes(x.abs(), cos.abs(), -sin.abs(), p, (24, 20, 20), interleaved, torch.float64).abs()
            size = torch.maximum(size, turn_axes(x.abs(), cos.abs(), sin.abs(), p, (24, 20, 20), interleaved,
                                                 torch.float64).abs())
            bound = torch.finfo(dtype).eps / 2 * (1 + 1e-3) * want.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25
            assert bool(((q.cpu().double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F16, E4M3])
def test_positions_outside_the_tables(tris, cuda, cache):
    """Such a token is not stored, its query zero, or left as it was in a given output; the others are as ever.  A token
    whose page is outside the pool is rotated and not stored."""
    before, new = [0, 20], [40, 13]
    for q_out in (False, True):
        a = _case(cuda, 4, 2, 128, 128, F16, cache, 16, before, new, pad=2)
        a["cos"], a["sin"] = a["cos"][:30].contiguous(), a["sin"][:30].contiguous()
        a["block_table"][1, 1] = -3
        p = _positions(3, 55, 30, cuda)
        p[0, 3], p[1, 17], p[2, 41], p[2, 50], p[0, 9] = 30, -1, 2 ** 31 - 1, -(2 ** 31), 29
        want = expected_axes(a, before, new, p, (22, 21, 21), True)
        given = torch.full_like(a["q"], 7.0) if q_out else None
        got = tris["ext"].rotary_append_paged(**a, positions=p, sections=(22, 21, 21), interleaved=True, q_out=given)
        lost = [3, 17, 41, 50, 53, 54]
        if q_out:
            want[0][lost] = 7.0
        assert bool((want[0][lost] == (7.0 if q_out else 0.0)).all())
        for g, w in zip((got, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"]), want):
            if w is not None:
                _same(g, w)


@pytest.mark.gpu
def test_in_place_without_queries_and_without_tokens(tris, cuda):
    ext = tris["ext"]
    before, new = [0, 3], [4, 2]
    a = _case(cuda, 6, 2, 64, 64, BF16, BF16, 16, before, new, pad=3)
    p = _positions(2, 9, 16, cuda)
    kw = dict(positions=p, sections=(20, 12))
    want = expected_axes(a, before, new, p, (20, 12), False)
    q = a["q"]
    assert ext.rotary_append_paged(**a, **kw, q_out=q) is q
    _same(q[:6], want[0][:6])
    kc = a["k_cache"].clone()
    a["q"] = None
    a["k_cache"].fill_(0)
    assert ext.rotary_append_paged(**a, **kw) is None
    good = ~torch.isnan(kc.float())
    assert torch.equal(a["k_cache"][good], kc[good])
    none = {**a, "q": q[:0], "k": a["k"][:0], "v": a["v"][:0], "query_start": torch.zeros_like(a["query_start"])}
    assert ext.rotary_append_paged(**none, positions=p[:, :0], sections=(20, 12)).shape == (0, 6, 64)


@pytest.mark.gpu
def test_graph_replays_with_new_positions_and_another_stream(tris, cuda):
    ext = tris["ext"]
    before = [4, 0, 11]
    a = _case(cuda, 4, 2, 128, 128, F16, E4M3, 16, [b + 4 for b in before], [1] * 3)
    a["seq_lens"].sub_(4)
    wide = torch.zeros((3, 5), dtype=torch.int32, device=cuda)
    p = wide[:, 1:4]                                        # rows five apart
    kw = dict(positions=p, sections=(24, 20, 20), interleaved=True)
    ext.rotary_append_paged(**a, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ext.rotary_append_paged(**a, **kw)
    side = torch.cuda.Stream()
    for step in range(4):
        a["seq_lens"].add_(1)
        p.copy_(_positions(3, 3, 16, cuda, step))
        want = expected_axes(a, [b + 1 + step for b in before], [1] * 3, p, (24, 20, 20), True)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            again = ext.rotary_append_paged(**a, **kw)
        torch.cuda.synchronize()
        assert torch.equal(_bits(again), _bits(q))
        for got, w in zip((q, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"]), want):
            _same(got, w)


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 128, 128, F16, F16, 16, [0, 3], [4, 2])
    p = _positions(3, 6, 16, cuda)
    good = dict(positions=p, sections=(24, 20, 20))
    bad = [
        ("torch.int32", dict(positions=p.long())), ("CUDA", dict(positions=p.cpu())),
        ("must be a tensor", dict(positions=[0] * 6)), ("axes, tokens", dict(positions=p[None])),
        ("one for each token", dict(positions=p[:, :5])), ("contiguous", dict(positions=p.t().contiguous().t())),
        ("each of the sections", dict(positions=p[:2])), ("each of the sections", dict(positions=p[0])),
        ("each of the sections", dict(sections=None)), ("add up", dict(sections=(24, 20, 21))),
        ("negative section", dict(sections=(44, -4, 24))), ("do not fit", dict(sections=(20, 22, 22), interleaved=True)),
        ("1 to 4 axes", dict(positions=_positions(5, 6, 16, cuda), sections=(60, 1, 1, 1, 1))),
        ("1 to 4 axes", dict(positions=p[:0], sections=())), ("need positions", dict(positions=None)),
        ("without rows", dict(cos=a["cos"][:0], sin=a["sin"][:0])),
        ("need positions", dict(positions=None, sections=None, interleaved=True)),
        ("no gradient", dict(cos=a["cos"].clone().requires_grad_())),
    ]
    saved = a["k_cache"].clone()
    for match, kw in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.rotary_append_paged(**{**a, **good, **kw})
    assert torch.equal(_bits(saved), _bits(a["k_cache"]))
    assert _expected(a, [0, 3], [4, 2])[0].shape == a["q"].shape


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(cache=None, tokens=2, q_heads=4, rot=128, rows=48, act=0, at=p, stride=2, sections=(24, 20, 20), axes=None,
             interleaved=0):
        split = None if sections is None else (ctypes.c_int32 * max(1, len(sections)))(*sections)
        return lib.tris_rotary_axes_append_paged(
            p, 512, 128, p, 256, 128, p, 256, 128, act, tokens, q_heads, p, p, rot, rows, None,
            ctypes.byref(cache or c_cache()), p, 512, 128, 0, at, stride, len(sections or ()) if axes is None else axes, split,
            interleaved, None)

    for kw, word in BAD_CACHES:
        assert call(c_cache(**kw)) == -1 and word in lib.tris_last_error(), kw
    most = 2 ** 31 - 1
    for kw, word in ((dict(at=None), b"null"), (dict(axes=0), b"axes"), (dict(sections=(60, 1, 1, 1, 1)), b"axes"),
                     (dict(axes=-1), b"axes"), (dict(sections=None, axes=3), b"axes"), (dict(stride=-1), b"axes"),
                     (dict(sections=(24, 20, 19)), b"add up"), (dict(sections=(most, most, 66)), b"add up"),
                     (dict(sections=(65, 0, -1)), b"negative"), (dict(sections=(20, 22, 22), interleaved=1), b"fit"),
                     (dict(sections=(0, 64), interleaved=1), b"fit"), (dict(rows=0), b"rows"), (dict(rot=24), b"rotary_dim"),
                     (dict(tokens=3), b"one token a sequence")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), kw
    assert call(c_cache(batch=0), tokens=0, at=None) == 0
