"""ext.paged_attention_decode (tris_paged_attention_decode) against softmax attention in 64 bits: types, head layouts,
lengths from nothing to long ones, page sizes and orders, windows, pages outside the pool, stale slots, special
values, graphs, refusals."""
import ctypes
import math

import pytest
import torch

from paged_cases import E4M3, make_pool, make_table, rows_of
from test_paged_cache import BAD_CACHES, c_cache

F16, BF16 = torch.float16, torch.bfloat16


def _case(cuda, q_heads, heads, dim, dtype, cache, page, lengths, order="head", seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // page) for n in lengths) + 2
    table = make_table(lengths, page, pages, cuda, gen)
    kc, vc, ks, vs = make_pool(pages, heads, page, dim, cache, cuda, order)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        j = torch.arange(n)
        pg, slot = table[b].cpu().long()[j // page].to(cuda), (j % page).to(cuda)
        for t, s, f in ((kc, ks, spread), (vc, vs, 1.0)):
            x = (torch.randn((n, heads, dim), generator=gen) * f).to(cuda)
            if s is not None:
                amax = x.abs().amax(-1) / 448.0
                s[pg, :, slot] = amax
                x = x / amax[..., None]
            t[pg, :, slot] = x.to(t.dtype)
    q = torch.randn((len(lengths), q_heads, dim), generator=gen).to(dtype).to(cuda)
    return dict(q=q, k_cache=kc, v_cache=vc, block_table=table,
                seq_lens=torch.tensor(lengths, dtype=torch.int32, device=cuda), k_scale=ks, v_scale=vs)


def _check(a, lengths, got, scale=None, window=0, keep=None):
    """The error bound, element by element, of fp32 attention with one rounding at the end:
      half a step of the output's type, plus, in units of W = sum_j w_j |v_j| (w the softmax weights),
      2 * 2 (dim + 8) 2^-24 max_j sum_i |q_i k_ij| scale   scores: the dot product's roundings (twice for the matrix
                                                           unit's order) and three scalings, on weights and their sum
      2 * (n + 64) 2^-24                                   the sums over the keys (all weights positive) and rescalings
      2 * 2^-20 (1 + |s|max 2^-2)                          base-2 exponentials of rounded arguments
      2^-13                                                weights held as two 16-bit parts in the value product."""
    q = a["q"].double().cpu()
    batch, q_heads, dim = q.shape
    heads, page = a["k_cache"].shape[1:3]
    scale = dim ** -0.5 if scale is None else scale
    dtype = a["q"].dtype
    assert got.dtype == dtype and got.shape == a["q"].shape
    got, worst = got.double().cpu(), 0.0
    for b, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        at = torch.arange(first, n)
        if keep is not None:
            at = at[keep[b][first:n]]
        if at.numel() == 0:
            assert bool((got[b] == 0).all())
            continue
        k = rows_of(a["k_cache"], a["k_scale"], a["block_table"], b, n, page)[:, at]
        v = rows_of(a["v_cache"], a["v_scale"], a["block_table"], b, n, page)[:, at]
        qb = q[b].view(heads, q_heads // heads, dim)
        s = qb @ k.transpose(1, 2) * scale
        w = torch.softmax(s, -1)
        want = (w @ v).reshape(q_heads, dim)
        size = (w @ v.abs()).reshape(q_heads, dim)
        dots = (qb.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1).reshape(q_heads, 1)
        far = s.abs().amax(-1).reshape(q_heads, 1)
        u = 2.0 ** -24
        part = 4 * (dim + 8) * u * dots + 2 * (at.numel() + 64) * u + 2.0 ** -19 * (1 + far / 4) + 2.0 ** -13
        bound = torch.finfo(dtype).eps / 2 * (1 + 1e-3) * want.abs() + part * size + (2.0 ** -25 if dtype == F16 else 1e-38)
        worst = max(worst, ((got[b] - want).abs() / bound).max().item())
        assert not math.isnan(worst) and bool(torch.isfinite(got[b]).all())
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


TYPES = [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)]
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 200, 513]


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,order", [(16, "head"), (64, "token"), (7, "head"), (1, "token"), (48, "head"), (20, "token")])
def test_ragged_lengths(tris, cuda, types, dim, page, order):
    print(f"[gpu-case] attention {types} dim={dim} page={page} {order}", flush=True)
    a = _case(cuda, 8, 2, dim, *types, page, LENGTHS, order, seed=dim + page)
    _check(a, LENGTHS, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (7, 1), (16, 1), (17, 1), (40, 2), (33, 3), (64, 1)], ids=str)
@pytest.mark.parametrize("types", [(BF16, BF16), (F16, E4M3)], ids=str)
def test_head_layouts(tris, cuda, heads, types):
    lengths = [300, 1, 0, 77]
    for page in (16, 5):
        a = _case(cuda, *heads, 128, *types, page, lengths, seed=heads[0])
        _check(a, lengths, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("lengths", [[70000], [5000, 3, 0, 41, 9000, 1, 128], [33] * 70 + [4000], [1] * 300], ids=lambda v: f"{len(v)}x{max(v)}")
def test_split_over_the_length(tris, cuda, types, lengths):
    print(f"[gpu-case] attention {types} lengths {len(lengths)} x {max(lengths)}", flush=True)
    a = _case(cuda, 4, 1, 128, *types, 32, lengths, seed=len(lengths))
    _check(a, lengths, tris["ext"].paged_attention_decode(**a))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 5, 32, 100, 129, 100000])
@pytest.mark.parametrize("types", [(F16, F16), (BF16, E4M3)], ids=str)
def test_windows(tris, cuda, window, types):
    lengths = [0, 1, 31, 64, 130, 1000]
    for page in (16, 6):
        a = _case(cuda, 4, 2, 64, *types, page, lengths, seed=window)
        # what lies before a window may hold anything, its pages too
        for b, n in enumerate(lengths):
            gone = max(0, n - window) // page
            for p in a["block_table"][b, :gone].tolist():
                a["k_cache"][p].view(torch.uint8).fill_(0x7F if types[1] == E4M3 else 0xFF)
                a["v_cache"][p].view(torch.uint8).fill_(0x7F if types[1] == E4M3 else 0xFF)
            a["block_table"][b, :gone] = -7
        table = a["block_table"]
        got = tris["ext"].paged_attention_decode(**a, window=window)
        a["block_table"] = table.clamp(0, a["k_cache"].shape[0] - 1)   # only for the host's gather
        _check(a, lengths, got, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(BF16, BF16), (F16, E4M3)], ids=str)
@pytest.mark.parametrize("page", [16, 9])
def test_pages_outside_the_pool_are_left_out(tris, cuda, types, page):
    lengths = [200, 40, 16, 300]
    a = _case(cuda, 8, 2, 128, *types, page, lengths, seed=3)
    keep = [torch.ones(n, dtype=torch.bool) for n in lengths]
    for b, i, bad in ((0, 0, -1), (0, 2, 1 << 30), (1, -(-40 // page) - 1, a["k_cache"].shape[0]), (3, 1, -(1 << 31))):
        a["block_table"][b, i] = bad
        keep[b][i * page: (i + 1) * page] = False
    for i in range(-(-16 // page)):
        a["block_table"][2, i] = -1
    keep[2][:] = False
    got = tris["ext"].paged_attention_decode(**a)
    a["block_table"] = a["block_table"].clamp(0, a["k_cache"].shape[0] - 1)
    _check(a, lengths, got, keep=keep)


@pytest.mark.gpu
def test_lengths_past_the_table_and_negative(tris, cuda):
    lengths = [64, 40, 0]
    a = _case(cuda, 4, 2, 128, F16, F16, 16, lengths)
    a["block_table"] = a["block_table"][:, :4].contiguous()
    want = tris["ext"].paged_attention_decode(**a)
    a["seq_lens"].copy_(torch.tensor([2 ** 31 - 1, 40, -5], dtype=torch.int32))
    assert torch.equal(tris["ext"].paged_attention_decode(**a), want)
    _check(a, lengths, want)
    a["block_table"] = a["block_table"][:, :0]
    a["seq_lens"].fill_(9)
    assert bool((tris["ext"].paged_attention_decode(**a) == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_sharp_and_flat_scores(tris, cuda, types):
    """Scores far apart (one key takes everything), all equal, and one key high above a long tail whose values alone
    make the output: the tail's weights are far below the peak's."""
    lengths = [513, 2000]
    a = _case(cuda, 4, 1, 128, *types, 16, lengths, seed=9, spread=30.0)
    _check(a, lengths, tris["ext"].paged_attention_decode(**a))
    _check(a, lengths, tris["ext"].paged_attention_decode(**a, scale=0.0), scale=0.0)
    _check(a, lengths, tris["ext"].paged_attention_decode(**a, scale=-0.01), scale=-0.01)
    n = 30000
    a = _case(cuda, 2, 1, 128, *types, 64, [n], seed=10)
    page0 = int(a["block_table"][0, 0])
    one = a["q"].new_ones(128)
    a["q"][:] = one
    for t in (a["k_cache"], a["v_cache"]):
        good = ~torch.isnan(t.float())
        t[good] = torch.where(good, (torch.rand(t.shape, device=cuda) * 0.5 + 1.0).to(t.dtype).float(), t.float())[good].to(t.dtype)
    a["k_cache"][:, 0] = torch.where(torch.isnan(a["k_cache"][:, 0].float()), a["k_cache"][:, 0].float(), 0.0).to(a["k_cache"].dtype)
    if a["k_scale"] is not None:
        a["k_scale"].copy_(torch.where(torch.isnan(a["k_scale"]), a["k_scale"], 1.0))
        a["v_scale"].copy_(torch.where(torch.isnan(a["v_scale"]), a["v_scale"], 0.25))
    a["k_cache"][page0, 0, 0] = one.to(a["k_cache"].dtype)       # its score: 14 above every other at scale 0.11
    a["v_cache"][page0, 0, 0] = a["q"].new_zeros(128).to(a["v_cache"].dtype)
    for scale in (0.11, 0.14, 0.2):
        _check(a, [n], tris["ext"].paged_attention_decode(**a, scale=scale), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 10])
def test_special_values(tris, cuda, page):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 64, BF16, BF16, page, [50, 50, 50, 50])
    want = ext.paged_attention_decode(**a)
    p = a["block_table"].cpu()
    a["k_cache"][p[0, 0], 0, 3, 5] = float("nan")     # sequence 0, kv head 0: query heads 0 and 1
    a["v_cache"][p[1, 1], 1, 2, 7] = float("inf")     # sequence 1, kv head 1: one value column
    a["k_cache"][p[2, 0], 0, 1] = float("inf")        # scores of +-inf or NaN
    a["q"][2, 0], a["q"][2, 1] = 1.0, -1.0
    got = ext.paged_attention_decode(**a).float()
    assert bool(torch.isnan(got[0, :2]).all()) and torch.equal(got[0, 2:], want[0, 2:].float())
    assert bool(torch.isposinf(got[1, 2:, 7]).all()) and bool(torch.isfinite(got[1, 2:, :7]).all())
    assert torch.equal(got[1, :2], want[1, :2].float()) and torch.equal(got[3], want[3].float())
    assert bool(torch.isnan(got[2, 0]).all())         # exp(inf - inf), as softmax gives it
    assert bool(torch.isfinite(got[2, 1]).all())      # a score of -inf: that key counts nothing


@pytest.mark.gpu
def test_strided_queries_and_output(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 8, 2, 128, F16, F16, 16, [100, 33, 5])
    want = ext.paged_attention_decode(**a)
    wide = torch.zeros((3, 8 * 128 + 64), dtype=F16, device=cuda)
    wide[:, 64:].copy_(a["q"].view(3, -1))
    a["q"] = wide[:, 64:].view(3, 8, 128)
    buf = torch.full((3, 10, 128), 7.0, dtype=F16, device=cuda)
    assert torch.equal(ext.paged_attention_decode(**a, out=buf[:, 1:9]), want)
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, 9] == 7).all())
    odd = torch.zeros(3 * 8 * 128 + 3, dtype=F16, device=cuda)[3:]
    odd.copy_(a["q"].reshape(-1))
    a["q"] = odd.view(3, 8, 128)                      # not 16-byte aligned: copied
    assert torch.equal(ext.paged_attention_decode(**a), want)


@pytest.mark.gpu
def test_repeats_graph_and_streams(tris, cuda):
    """The same bits call after call, on another stream beside another call, and from a graph replayed with other
    lengths and tables."""
    ext = tris["ext"]
    lengths = [3000, 10, 0, 700]
    a = _case(cuda, 8, 2, 128, BF16, BF16, 16, lengths)
    b = _case(cuda, 8, 2, 128, BF16, BF16, 16, lengths, seed=5)
    want, want_b = ext.paged_attention_decode(**a), ext.paged_attention_decode(**b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(side):
            got_b = ext.paged_attention_decode(**b)
        got = ext.paged_attention_decode(**a)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got_b, want_b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ext.paged_attention_decode(**a)
        got_b = ext.paged_attention_decode(**b)
    for lens in ([3000, 10, 0, 700], [1, 0, 0, 5], [2999, 4, 0, 17]):
        a["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        eager = ext.paged_attention_decode(**a)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(got_b, want_b)
        _check(a, lens, got)


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 128, F16, F16, 16, [10, 3])
    bad = [
        ("float16", dict(q=a["q"].float())),
        ("one token for each row", dict(q=a["q"][:1])),
        ("multiple of kv_heads", dict(q=a["q"][:, :3].contiguous())),
        ("head_dim", dict(q=a["q"][..., :64].contiguous())),
        ("activations' type", dict(q=a["q"].to(BF16))),
        ("negative window", dict(window=-1)),
        ("shape of q", dict(out=a["q"][:1])),
        ("shape of k_cache", dict(v_cache=a["v_cache"][:1])),
        ("one length", dict(seq_lens=a["seq_lens"][:1])),
        ("torch.int32", dict(block_table=a["block_table"].long())),
        ("rows of block_table", dict(block_table=a["block_table"].t().contiguous().t())),
        ("no gradient", dict(q=a["q"].clone().requires_grad_())),
    ]
    for match, kw in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.paged_attention_decode(**{**a, **kw})
    empty = {**a, "q": a["q"][:0], "block_table": a["block_table"][:0], "seq_lens": a["seq_lens"][:0]}
    assert ext.paged_attention_decode(**empty).shape == (0, 4, 128)


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(cache=None, q_heads=4, window=0, stride=512, q_type=0, q=p):
        return lib.tris_paged_attention_decode(q, stride, 128, q_type, q_heads, ctypes.byref(cache or c_cache()), 0.1,
                                               window, p, 512, 128, p, 1 << 40, None)

    for kw, word in BAD_CACHES:
        assert call(c_cache(**kw)) == -1 and word in lib.tris_last_error(), kw
    for kw, word in ((dict(q_heads=3), b"multiple"), (dict(q_heads=0), b"multiple"), (dict(window=-2), b"window"),
                     (dict(stride=4), b"16-byte"), (dict(q_type=2), b"fp16"), (dict(q=None), b"null")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), kw
    assert call(c_cache(batch=0)) == 0
    with pytest.raises(RuntimeError, match="CUDA"):
        t = torch.zeros((1, 2, 128), dtype=F16)
        tris["ext"].paged_attention_decode(t, t, t, t, t)
