"""ext.paged_attention_decode with weight_sum (tris_paged_attention_decode_weights): the sums of the keys' weights against
softmax in 64 bits and the output against the call without them, over types, head layouts, lengths, pages, windows, pages
outside the pool, special values, strides, streams, graphs, refusals."""
import ctypes

import pytest
import torch

from paged_cases import E4M3, rows_of
from test_paged_attention import TYPES, _case
from test_paged_cache import BAD_CACHES, _bits, c_cache

F16, BF16 = torch.float16, torch.bfloat16


def _sums(a, extra=0, seed=0):
    """Sums of a sequence's life so far, random everywhere."""
    batch, heads = a["seq_lens"].numel(), a["k_cache"].shape[1]
    positions = a["block_table"].shape[1] * a["k_cache"].shape[2] + extra
    g = torch.Generator().manual_seed(seed)
    return torch.rand((batch, heads, positions), generator=g).to(a["q"].device) * 0.01


def check_sums(a, lengths, before, after, scale=None, window=0, keep=None):
    """The error bound of each sum, position by position.  A weight, relatively:
      4 (dim + 8) 2^-24 max_j sum_i |q_i k_ij| scale   the dot product's roundings (twice for the matrix unit's order) and
                                                       three scalings, on the weight and on the softmax's sum
      2 (n + 64) 2^-24                                 the sum over the keys and its rescalings, the weight's product
      2^-19 (1 + |s|max 2^-2)                          two base-2 exponentials of rounded arguments
    the weights of the kv head's heads added, then to the sum: (group + 1) 2^-24 of the weights and 2^-24 of the result.
    Positions that are not attended to keep their bits."""
    q = a["q"].double().cpu()
    batch, q_heads, dim = q.shape
    heads, page = a["k_cache"].shape[1:3]
    scale = dim ** -0.5 if scale is None else scale
    before, after = before.cpu(), after.cpu()
    u, worst = 2.0 ** -24, 0.0
    for b, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        at = torch.arange(first, n)
        if keep is not None:
            at = at[keep[b][first:n]]
        rest = torch.ones(before.shape[2], dtype=torch.bool)
        rest[at] = False
        assert torch.equal(_bits(after[b][:, rest]), _bits(before[b][:, rest])), f"sequence {b}"
        if at.numel() == 0:
            continue
        k = rows_of(a["k_cache"], a["k_scale"], a["block_table"], b, n, page)[:, at]
        qb = q[b].view(heads, q_heads // heads, dim)
        s = qb @ k.transpose(1, 2) * scale
        w = torch.softmax(s, -1)
        dots = (qb.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
        far = s.abs().amax(-1, keepdim=True)
        part = 4 * (dim + 8) * u * dots + 2 * (at.numel() + 64) * u + 2.0 ** -19 * (1 + far / 4)
        want = before[b][:, at].double() + w.sum(1)
        bound = (w * part).sum(1) + (q_heads // heads + 1) * u * w.sum(1) + u * want.abs() + 2.0 ** -120
        got = after[b][:, at].double()
        assert bool(torch.isfinite(got).all())
        worst = max(worst, ((got - want).abs() / bound).max().item())
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


def _run(tris, a, lengths, scale=None, window=0, keep=None, extra=0):
    ext = tris["ext"]
    want = ext.paged_attention_decode(**a, scale=scale, window=window)
    sums = _sums(a, extra)
    before = sums.clone()
    got = ext.paged_attention_decode(**a, scale=scale, window=window, weight_sum=sums)
    assert torch.equal(_bits(got), _bits(want))
    if keep is not None:
        a = {**a, "block_table": a["block_table"].clamp(0, a["k_cache"].shape[0] - 1)}   # only for the host's gather
    check_sums(a, lengths, before, sums, scale, window, keep)
    return sums


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 200, 513]


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,order", [(16, "head"), (64, "token"), (7, "head"), (1, "token"), (20, "token")])
def test_ragged_lengths(tris, cuda, types, dim, page, order):
    print(f"[gpu-case] weights {types} dim={dim} page={page} {order}", flush=True)
    _run(tris, _case(cuda, 8, 2, dim, *types, page, LENGTHS, order, seed=dim + page), LENGTHS)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (7, 1), (16, 1), (17, 1), (40, 2), (33, 3), (64, 1), (1024, 1)], ids=str)
@pytest.mark.parametrize("types", [(BF16, BF16), (F16, E4M3)], ids=str)
@pytest.mark.parametrize("lengths", [[300, 1, 0, 77], [3000, 1, 0, 77, 1500], [12000]], ids=str)
def test_head_layouts(tris, cuda, heads, types, lengths):
    for page in (16, 5):
        _run(tris, _case(cuda, *heads, 128, *types, page, lengths, seed=heads[0]), lengths, extra=page)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("lengths", [[70000], [5000, 3, 0, 41, 9000, 1, 128], [33] * 70 + [4000], [1] * 300], ids=lambda v: f"{len(v)}x{max(v)}")
def test_split_over_the_length(tris, cuda, types, lengths):
    print(f"[gpu-case] weights {types} lengths {len(lengths)} x {max(lengths)}", flush=True)
    _run(tris, _case(cuda, 4, 1, 128, *types, 32, lengths, seed=len(lengths)), lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 5, 32, 100, 129, 100000])
@pytest.mark.parametrize("types", [(F16, F16), (BF16, E4M3)], ids=str)
def test_windows(tris, cuda, window, types):
    for lengths in ([0, 1, 31, 64, 130, 1000], [0, 1, 31, 64, 130, 2500]):
        for page in (16, 6):
            _run(tris, _case(cuda, 4, 2, 64, *types, page, lengths, seed=window), lengths, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(BF16, BF16), (F16, E4M3)], ids=str)
@pytest.mark.parametrize("page", [16, 9])
def test_pages_outside_the_pool_are_left_out(tris, cuda, types, page):
    for lengths in ([200, 40, 16, 300], [200, 40, 16, 3000]):
        a = _case(cuda, 8, 2, 128, *types, page, lengths, seed=3)
        keep = [torch.ones(n, dtype=torch.bool) for n in lengths]
        for b, i, bad in ((0, 0, -1), (0, 2, 1 << 30), (1, -(-40 // page) - 1, a["k_cache"].shape[0]), (3, 1, -(1 << 31))):
            a["block_table"][b, i] = bad
            keep[b][i * page: (i + 1) * page] = False
        for i in range(-(-16 // page)):
            a["block_table"][2, i] = -1
        keep[2][:] = False
        _run(tris, a, lengths, keep=keep)


@pytest.mark.gpu
def test_lengths_past_the_table_and_negative(tris, cuda):
    ext, lengths = tris["ext"], [64, 40, 0]
    a = _case(cuda, 4, 2, 128, F16, F16, 16, lengths)
    a["block_table"] = a["block_table"][:, :4].contiguous()
    a["seq_lens"].copy_(torch.tensor([2 ** 31 - 1, 40, -5], dtype=torch.int32))
    _run(tris, a, lengths, extra=3)
    a["block_table"] = a["block_table"][:, :0]
    sums = torch.zeros((3, 2, 0), device=cuda)
    assert bool((ext.paged_attention_decode(**a, weight_sum=sums) == 0).all())
    some = torch.ones((3, 2, 5), device=cuda)
    ext.paged_attention_decode(**a, weight_sum=some)
    assert bool((some == 1).all())
    empty = {**a, "q": a["q"][:0], "block_table": a["block_table"][:0], "seq_lens": a["seq_lens"][:0]}
    assert ext.paged_attention_decode(**empty, weight_sum=sums[:0]).shape == (0, 4, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_sharp_and_flat_scores(tris, cuda, types):
    """One key takes everything, all scores equal, small ones of the other sign."""
    lengths = [513, 2000]
    a = _case(cuda, 4, 1, 128, *types, 16, lengths, seed=9, spread=30.0)
    for scale in (None, 0.0, -0.01):
        _run(tris, a, lengths, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("n", [50, 3000])
def test_special_values(tris, cuda, page, n):
    """A NaN in a key, a score of infinity: every sum of that kv head that a key is attended for becomes NaN, as softmax
    is; a score of -infinity adds zero; all of them: nothing is added.  Values do not matter."""
    ext, inf = tris["ext"], float("inf")
    a = _case(cuda, 4, 2, 64, BF16, BF16, page, [n] * 5)
    p = a["block_table"].cpu()
    want = _sums(a)
    ext.paged_attention_decode(**a, weight_sum=want)
    a["k_cache"][p[0, 0], 0, 3, 5] = float("nan")
    a["v_cache"][p[1, 1], 1, 2, 7] = float("nan")
    a["k_cache"][p[2, 0], 0, 1] = inf
    a["q"][2, 0] = 1.0
    a["k_cache"][p[3, 0], 1, 1], a["q"][3, 2:] = inf, -1.0
    for i in range(-(-n // page)):
        a["k_cache"][p[4, i], 0] = inf
    a["q"][4, :2] = -1.0
    before = _sums(a)
    sums = before.clone()
    ext.paged_attention_decode(**a, weight_sum=sums)
    for b in (0, 2):
        assert bool(torch.isnan(sums[b, 0, :n]).all())
        assert torch.equal(sums[b, 0, n:], before[b, 0, n:]) and torch.equal(sums[b, 1], want[b, 1])
    assert torch.equal(sums[1], want[1])
    assert float(sums[3, 1, 1]) == float(before[3, 1, 1]) and bool(torch.isfinite(sums[3]).all())
    total = (sums[3, 1].double() - before[3, 1].double()).sum().item()
    assert abs(total - 2) < 1e-3                    # two heads' weights
    assert torch.equal(sums[4, 0], before[4, 0]) and torch.equal(sums[4, 1], want[4, 1])


@pytest.mark.gpu
def test_strides_and_alignment_of_the_sums(tris, cuda):
    ext = tris["ext"]
    for lengths in ([100, 33, 5], [100, 33, 3000]):
        a = _case(cuda, 8, 2, 128, F16, F16, 16, lengths)
        want = _sums(a)
        n = want.shape[2]
        start = want.clone()
        ext.paged_attention_decode(**a, weight_sum=want)
        by_head = torch.empty((2, 3, n), device=cuda).transpose(0, 1).copy_(start)
        ext.paged_attention_decode(**a, weight_sum=by_head)
        assert torch.equal(by_head, want)
        buf = torch.full((3, 3, n + 7), 5.0, device=cuda)
        view = buf[:, 1:, 3: n + 3]
        view.copy_(start)
        ext.paged_attention_decode(**a, weight_sum=view)
        assert torch.equal(view, want)
        assert bool((buf[:, 0] == 5).all()) and bool((buf[..., :3] == 5).all()) and bool((buf[..., n + 3:] == 5).all())


@pytest.mark.gpu
def test_repeats_graphs_and_streams(tris, cuda):
    """The same bits call after call, beside another call on another stream, and from two graphs with a workspace in one
    pool, replayed with other lengths."""
    ext = tris["ext"]
    lengths = [3000, 10, 0, 700]
    a = _case(cuda, 8, 2, 128, BF16, BF16, 16, lengths)
    b = _case(cuda, 8, 2, 128, BF16, BF16, 16, lengths, seed=5)
    start = _sums(a)

    def eager(x):
        s = start.clone()
        return ext.paged_attention_decode(**x, weight_sum=s), s

    want, want_b = eager(a), eager(b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        s, t = start.clone(), start.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got_b = ext.paged_attention_decode(**b, weight_sum=t)
        got = ext.paged_attention_decode(**a, weight_sum=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want[0]) and torch.equal(s, want[1])
        assert torch.equal(got_b, want_b[0]) and torch.equal(t, want_b[1])
    s, t = start.clone(), start.clone()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got = ext.paged_attention_decode(**a, weight_sum=s)
    with torch.cuda.graph(second, pool=first.pool()):
        got_b = ext.paged_attention_decode(**b, weight_sum=t)
    for lens in (lengths, [1, 0, 0, 5], [2999, 4, 0, 17]):
        a["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        s.copy_(start), t.copy_(start)
        first.replay()
        kept = got.clone()
        second.replay()
        again = eager(a)
        torch.cuda.synchronize()
        assert torch.equal(kept, again[0]) and torch.equal(s, again[1])
        assert torch.equal(got_b, want_b[0]) and torch.equal(t, want_b[1])
        check_sums(a, lens, start, s)


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    a = _case(cuda, 4, 2, 128, F16, F16, 16, [10, 3])
    s = _sums(a)
    n = s.shape[2]
    bad = [
        ("torch.float32", s.half()), ("CUDA", s.cpu()), ("3D", s[0]), ("weight_sum must be", s[:1]),
        ("weight_sum must be", s[:, :1]), ("weight_sum must be", s[..., :n - 1]), ("must be a tensor", 1.0),
        ("rows of weight_sum must be contiguous", s.transpose(1, 2).contiguous().transpose(1, 2)),
        ("rows of weight_sum overlap", s[:, :1].expand(2, 2, n)), ("rows of weight_sum overlap", s[:1].expand(2, 2, n)),
        ("no gradient", s.clone().requires_grad_()),
    ]
    for match, sums in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.paged_attention_decode(**a, weight_sum=sums)


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(cache=None, q_heads=4, window=0, stride=512, q_type=0, q=p, sums=p, seq=96, head=48, ws=p, space=1 << 40):
        return lib.tris_paged_attention_decode_weights(q, stride, 128, q_type, q_heads, ctypes.byref(cache or c_cache()), 0.1,
                                                       window, p, stride, 128, sums, seq, head, ws, space, None)

    for kw, word in BAD_CACHES:
        assert call(c_cache(**kw)) == -1 and word in lib.tris_last_error(), kw
    need = lib.tris_paged_attention_weights_workspace_bytes(2, 4, 2, 128, 3, 16)
    assert need >= 2 * 4 * (48 * 4 + 8)
    most = 1 << 23
    for kw, word in ((dict(q_heads=3), b"multiple"), (dict(window=-2), b"window"), (dict(stride=4), b"16-byte"),
                     (dict(q_type=2), b"fp16"), (dict(q=None), b"null"), (dict(sums=None), b"null"),
                     (dict(seq=95), b"overlap"), (dict(head=47), b"overlap"), (dict(head=0), b"overlap"),
                     (dict(seq=-96), b"overlap"), (dict(ws=None), b"workspace"), (dict(space=need - 1), b"workspace"),
                     (dict(ws=ctypes.c_void_p(4104)), b"workspace"),
                     (dict(q_heads=2 * 1025, stride=2 * 1025 * 128), b"1024 query heads"),
                     (dict(cache=c_cache(max_pages=most, table_stride=most, k_slot_stride=128), q_heads=8, stride=1024,
                           seq=1 << 40, head=1 << 30, space=1 << 33), b"workspace")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), kw
    assert call(c_cache(batch=0)) == 0
    for bad in ((0, 4, 2, 128, 3, 16), (2, 1, 2, 128, 3, 16), (2, 4, 0, 128, 3, 16), (2, 4, 2, 128, 3, 0)):
        assert lib.tris_paged_attention_weights_workspace_bytes(*bad) == 0
    assert lib.tris_paged_attention_weights_workspace_bytes(2 ** 31 - 1, 2 ** 31 - 1, 1, 128, 2 ** 24, 64) == -1
