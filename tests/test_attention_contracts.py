"""What the append and the paged attention promise at their borders: the weights' bits, invalid pages beside a sequence's
end and a window's beginning, infinite and very large values, the cache's descriptor, rows of outputs that overlap,
gradients (the norm's too), slot strides, steps without tokens."""
import ctypes
import struct

import pytest
import torch

from paged_cases import E4M3, rows_of
from test_paged_attention import _case, _check
from test_paged_cache import _case as _append_case, c_cache

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("page", [16, 5])
def test_weights_keep_their_bits(tris, cuda, types, page):
    """Sequences of four keys whose weighted values cancel, so that the output's rounding hides nothing.  Scores are
    exact multiples of 1 / 64 up to 1 / 2.  In units of 2^-24 of sum_j w_j |v_j|, for each weight: the argument of the
    power of two (at most 0.73 in size, seven roundings with the maximum's, times ln 2) 3.6, the power's last bit and
    one more 4, the 8-bit cache's factor 1; twelve additions of products, each off by 2 at most, 24; the sum of the
    weights, its inverse and the products with them 8: together 41."""
    dtype, cache = types
    batch, n, dim, u = 64, 4, 64, 2.0 ** -24
    g = torch.Generator().manual_seed(page)
    score = torch.randint(0, 33, (batch, n), generator=g).double() / 64
    w = torch.softmax(score, -1)
    v, vs = torch.zeros((batch, n, dim), dtype=torch.float64), torch.ones((batch, n))
    rest = torch.zeros((batch, dim), dtype=torch.float64)
    for j in range(n):                     # each key takes back what the ones before it left
        x = torch.randn((batch, dim), generator=g).double() if j == 0 else -rest / w[:, j, None]
        if cache == E4M3:
            vs[:, j] = (x.abs().amax(-1) / 448).clamp_min(2.0 ** -126).float()
            v[:, j] = (x / vs[:, j, None].double()).float().to(E4M3).double()
        else:
            v[:, j] = x.to(cache).double()
        rest += w[:, j, None] * v[:, j] * vs[:, j, None].double()
    kc, vc = (torch.zeros((batch, 1, page, dim)) for _ in range(2))
    ks, kv = (torch.ones((batch, 1, page)) for _ in range(2))
    kc[:, 0, :n, 0] = 1.0 if cache == E4M3 else score.float()
    ks[:, 0, :n], kv[:, 0, :n], vc[:, 0, :n] = score.float(), vs, v.float()
    q = torch.zeros((batch, 1, dim), dtype=dtype)
    q[:, 0, 0] = 1.0
    a = dict(q=q, k_cache=kc.to(cache), v_cache=vc.to(cache), block_table=torch.arange(batch, dtype=torch.int32)[:, None],
             seq_lens=torch.full((batch,), n, dtype=torch.int32))
    if cache == E4M3:
        a.update(k_scale=ks, v_scale=kv)
    got = tris["ext"].paged_attention_decode(**{k: t.to(cuda) for k, t in a.items()}, scale=1.0).cpu().double()[:, 0]
    size = (w[..., None] * v.abs() * vs[..., None].double()).sum(1)
    half = torch.finfo(dtype).eps / 2 * (1 + 1e-3)
    bound = half * rest.abs() + 41 * u * size + (2.0 ** -25 if dtype == F16 else 1e-38)
    worst = ((got - rest).abs() / bound).max().item()
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


def _free_first_page(a, fill):
    """Moves the sequences off page 0, which then holds `fill`: nothing may read it."""
    table, pages = a["block_table"], a["k_cache"].shape[0]
    spare = next(p for p in range(1, pages) if not bool((table == p).any()))
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        t = a[name]
        if t is None:
            continue
        raw = t.view(torch.uint8) if t.dtype == E4M3 else t
        raw[spare] = raw[0]
        t[0].copy_(torch.full(t[0].shape, fill).to(t.dtype))
    table[table == 0] = spare


def _without_pages(tris, a, lengths, bad, page, window=0):
    """Attention with the table's entries (sequence, index) in `bad` outside the pool."""
    keep = [torch.ones(n, dtype=torch.bool) for n in lengths]
    for i, (b, p) in enumerate(bad):
        a["block_table"][b, p] = (-1, a["k_cache"].shape[0], 2 ** 31 - 1)[i % 3]
        keep[b][p * page: (p + 1) * page] = False
    got = tris["ext"].paged_attention_decode(**a, window=window)
    a["block_table"] = a["block_table"].clamp(0, a["k_cache"].shape[0] - 1)   # only for the host's gather
    _check(a, lengths, got, window=window, keep=keep)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("fill", [float("nan"), 1.0])
@pytest.mark.parametrize("page", [10, 7, 3, 16])
def test_invalid_pages_at_a_sequences_end(tris, cuda, types, fill, page):
    """The last page, or every page, of sequences that end anywhere in a tile of 32 keys."""
    lengths = list(range(17, 25)) + [50, 52, 55, 31, 33, 5]
    for every in (False, True):
        a = _case(cuda, 4, 2, 64, *types, page, lengths, seed=page)
        _free_first_page(a, fill)
        if types[1] == E4M3 and page == 16:           # scales that cannot be read four at a time
            for name in ("k_scale", "v_scale"):
                flat = torch.empty(a[name].numel() + 1, device=cuda)[1:]
                a[name] = flat.view(a[name].shape).copy_(a[name])
        last = [-(-n // page) - 1 for n in lengths]
        bad = [(b, p) for b, top in enumerate(last) for p in (range(top + 1) if every else [top])]
        _without_pages(tris, a, lengths, bad, page)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("fill", [float("nan"), 1.0])
@pytest.mark.parametrize("page", [10, 7, 16])
def test_invalid_pages_where_a_window_begins(tris, cuda, types, fill, page):
    lengths = [60, 64, 95, 200, 41]
    for window in (3, 17, 25, 30):
        a = _case(cuda, 4, 2, 64, *types, page, lengths, seed=window)
        _free_first_page(a, fill)
        bad = [(b, min((n - window) // page + 1, (n - 1) // page)) for b, n in enumerate(lengths)]
        _without_pages(tris, a, lengths, bad, page, window)


def _plant(a, b, h, key, column, value):
    page = a["k_cache"].shape[2]
    a["v_cache"][int(a["block_table"][b, key // page]), h, key % page, column] = value


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 10])
def test_infinite_values(tris, cuda, dtype, dim, page):
    """An infinite value makes its column infinite, whatever its key's weight is (above zero for every finite score,
    also where fp32 holds none so small): at the key with the largest weight and at that with the smallest, in sequences
    of one token, a few, and so many that several workgroups share them; of both signs, not a number.  All else keeps
    its bits."""
    ext, inf = tris["ext"], float("inf")
    lengths = [1, 40, 33, 5000]
    a = _case(cuda, 4, 2, dim, dtype, dtype, page, lengths, seed=dim)
    for scale in (dim ** -0.5, 0.0, 6 * dim ** -0.5, 60 * dim ** -0.5):   # the last: weights far below 2^-126
        v = a["v_cache"].clone()
        want = ext.paged_attention_decode(**a, scale=scale).float()
        for b, n in enumerate(lengths):
            k = rows_of(a["k_cache"], None, a["block_table"], b, n, page)
            for h in range(2):
                s = a["q"][b, 2 * h].cpu().double() @ k[h].T * scale
                top, low = int(s.argmax()), int(s.argmin())
                _plant(a, b, h, top, 7, inf)
                _plant(a, b, h, low, 9, -inf)
                _plant(a, b, h, top, 20, -inf)
                _plant(a, b, h, 0, 21, inf)
                _plant(a, b, h, n - 1, 21, inf if n == 1 else -inf)
                _plant(a, b, h, n // 2, 40, float("nan"))
                columns = (0, 1) if h == 0 else (2, 3)
                want[b, columns, 7], want[b, columns, 9], want[b, columns, 20] = inf, -inf, -inf
                want[b, columns, 21] = inf if n == 1 else float("nan")
                want[b, columns, 40] = float("nan")
        for given in (None, a["q"].clone()):              # and over the queries
            q = a["q"] if given is None else given
            got = ext.paged_attention_decode(**{**a, "q": q}, scale=scale, out=given).float()
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])
        a["v_cache"].copy_(v)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 10])
def test_infinite_scales_of_an_8_bit_cache(tris, cuda, page):
    """value = element * scale: an infinite scale makes its row's elements infinite, and zeros not a number."""
    ext, lengths = tris["ext"], [1, 50, 4000]
    a = _case(cuda, 4, 2, 128, BF16, E4M3, page, lengths)
    want = ext.paged_attention_decode(**a).float()
    for b, n in enumerate(lengths):
        key = n // 2
        at = int(a["block_table"][b, key // page]), 1, key % page
        a["v_scale"][at] = float("inf")
        a["v_cache"][at].view(torch.uint8)[5] = 0
        want[b, 2:] = a["v_cache"][at].float() * float("inf")
    got = ext.paged_attention_decode(**a).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(want[:, 2:, 5]).all())
    assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 10])
def test_infinite_values_under_special_weights(tris, cuda, page):
    """A weight of exactly zero (a score of -infinity) or of NaN makes an infinite value NaN; keys that are left out do
    not count, whatever they hold."""
    ext, inf = tris["ext"], float("inf")
    lengths = [50, 50, 50, 45]
    a = _case(cuda, 4, 2, 64, BF16, BF16, page, lengths)
    p = a["block_table"].cpu()
    a["q"][0, :2] = -1.0
    a["k_cache"][p[0, 0], 0, 1] = inf                 # key 1 of sequence 0: a score of -infinity
    a["k_cache"][p[1, 0], 0, 1, 3] = float("nan")     # of sequence 1: NaN
    a["k_cache"][p[2, 0], 0, 1] = inf                 # of sequence 2: +infinity
    a["q"][2, :2] = 1.0
    want = ext.paged_attention_decode(**a).float()
    assert bool(torch.isfinite(want[0]).all()) and bool(torch.isnan(want[1:3, :2]).all())
    for b in range(3):
        _plant(a, b, 0, 1, 7, inf)
        want[b, :2, 7] = float("nan")
        _plant(a, b, 0, 2, 9, -inf)
        want[b, :2, 9] = -inf if b == 0 else float("nan")
    _plant(a, 3, 1, 0, 5, inf)                        # before a window of 40
    for window, columns in ((0, inf), (40, None)):
        got = ext.paged_attention_decode(**a, window=window).float()
        if columns is None:
            assert bool(torch.isfinite(got[3]).all())
            continue
        want[3, 2:, 5] = columns
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 10])
def test_largest_finite_values(tris, cuda, page):
    """Means of bf16 values near the type's largest: their weighted sum would pass fp32's range under weights up to one."""
    lengths = [1, 2, 40, 5000]
    a = _case(cuda, 4, 2, 128, BF16, BF16, page, lengths)
    top = torch.finfo(BF16).max
    v = a["v_cache"]
    good = ~torch.isnan(v.float())
    v[good] = (torch.rand(v.shape, device=cuda).sub_(0.5).sign_() * top).to(BF16)[good]
    v[..., :64][good[..., :64]] = top
    got = tris["ext"].paged_attention_decode(**a)
    assert bool((got[..., :64] == top).all())
    _check(a, lengths, got)


def test_cache_descriptor_is_the_c_struct(tris):
    from tris_moe_amd import _lib

    layout, fields = tris["ext"]._CACHE_LAYOUT, [n for n, _ in _lib.TrisPagedCache._fields_]
    assert layout.size == ctypes.sizeof(_lib.TrisPagedCache)
    values = [(7 * i + 3) << (20 if i < 19 else 0) for i in range(len(fields))]
    c = _lib.TrisPagedCache.from_buffer_copy(layout.pack(*values))
    assert [getattr(c, n) for n in fields] == values
    with pytest.raises(struct.error):
        layout.pack(*values[:-1], 1 << 31)


def test_output_rows_that_overlap_are_refused(tris):
    """Rows of an output that share memory would be written by several wavefronts at once."""
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def append(token, head, heads=4, tokens=2):
        c = c_cache(batch=tokens)
        return lib.tris_rotary_append_paged(p, 512, 128, p, 256, 128, p, 256, 128, 0, tokens, heads, p, p, 128, 48, None,
                                            ctypes.byref(c), p, token, head, 0, None)

    def attend(seq, head, heads=4, batch=2):
        return lib.tris_paged_attention_decode(p, 512, 128, 0, heads, ctypes.byref(c_cache(batch=batch)), 0.1, 0, p, seq,
                                               head, p, 1 << 40, None)

    for call in (append, attend):
        for strides in ((0, 128), (512, 0), (384, 128), (504, 128), (512, 120), (128, 248), (256, 128), (0, 0), (128, 128)):
            assert call(*strides) == -1 and b"output rows overlap" in lib.tris_last_error(), strides
        assert call(8, 120, 4, 1) == -1 and b"output rows overlap" in lib.tris_last_error()
        assert call(120, 8, 2, 2) == -1 and b"output rows overlap" in lib.tris_last_error()


def test_cache_rows_that_overlap_are_not_appended_to(tris):
    """A cache whose heads, pages or slots share memory (an expanded pool) can be read, not written."""
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def append(**kw):
        return lib.tris_rotary_append_paged(p, 512, 128, p, 256, 128, p, 256, 128, 0, 2, 4, p, p, 128, 48, None,
                                            ctypes.byref(c_cache(**kw)), p, 512, 128, 0, None)

    for kw in (dict(k_head_stride=0), dict(v_head_stride=0), dict(k_page_stride=0), dict(v_page_stride=2048),
               dict(k_page_stride=4088), dict(v_head_stride=64)):
        assert append(**kw) == -1 and b"cache rows overlap" in lib.tris_last_error(), kw
    scales = dict(dtype=3, k_scale=4096, v_scale=4096)
    for n in ("k", "v"):
        scales.update({f"{n}_scale_page_stride": 32, f"{n}_scale_head_stride": 16, f"{n}_scale_slot_stride": 1})
    for kw in (dict(k_scale_slot_stride=0), dict(v_scale_head_stride=0), dict(v_scale_page_stride=16)):
        assert append(**{**scales, **kw}) == -1 and b"cache scales overlap" in lib.tris_last_error(), kw
    # reading: refused for its window alone
    for kw in (dict(k_head_stride=0, v_head_stride=0), dict(scales, k_scale_slot_stride=0)):
        assert lib.tris_paged_attention_decode(p, 512, 128, 0, 4, ctypes.byref(c_cache(**kw)), 0.1, -1, p, 512, 128, p,
                                               1 << 40, None) == -1 and b"window" in lib.tris_last_error()


@pytest.mark.gpu
def test_output_strides(tris, cuda):
    """Expanded outputs are refused; ones whose heads are the outer dimension, and ones of one row, are taken."""
    ext = tris["ext"]
    lengths = [30, 3, 77]
    a = _case(cuda, 4, 2, 64, F16, F16, 16, lengths)
    want = ext.paged_attention_decode(**a)
    new = _append_case(cuda, 4, 2, 64, 64, F16, F16, 16, [0, 4, 9], [1, 1, 1])
    q = ext.rotary_append_paged(**new)
    for shape, dims in (((1, 4, 64), (3, 4, 64)), ((3, 1, 64), (3, 4, 64))):
        out = torch.zeros(shape, dtype=F16, device=cuda).expand(dims)
        with pytest.raises(RuntimeError, match="output rows overlap"):
            ext.paged_attention_decode(**a, out=out)
        with pytest.raises(RuntimeError, match="output rows overlap"):
            ext.rotary_append_paged(**new, q_out=out)
    by_head = torch.zeros((4, 3, 64), dtype=F16, device=cuda).transpose(0, 1)
    assert torch.equal(ext.paged_attention_decode(**a, out=by_head), want)
    assert torch.equal(ext.rotary_append_paged(**new, q_out=by_head), q)
    one = {**a, "q": a["q"][:1], "block_table": a["block_table"][:1], "seq_lens": a["seq_lens"][:1]}
    out = torch.zeros((1, 4, 64), dtype=F16, device=cuda).as_strided((1, 4, 64), (0, 64, 1))
    assert torch.equal(ext.paged_attention_decode(**one, out=out), want[:1])


def test_gradients_are_refused_on_any_tensor(tris):
    import torch.autograd.forward_ad as fwd

    refuse = tris["ext"]._refuse_gradient
    t, leaf = torch.ones(3), torch.ones(3, requires_grad=True)
    refuse("op", t, None)
    for tensors in ((leaf,), (t, None, leaf)):
        with pytest.raises(RuntimeError, match="op: no gradient"):
            refuse("op", *tensors)
        with torch.no_grad():
            refuse("op", *tensors)
    with fwd.dual_level():
        refuse("op", t, None)
        dual = fwd.make_dual(t, torch.ones(3))
        with pytest.raises(RuntimeError, match="op: no gradient"):
            refuse("op", t, None, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="op: no gradient"):   # tangents pass through no_grad
            refuse("op", dual)


@pytest.mark.gpu
def test_calls_refuse_gradients_on_every_tensor(tris, cuda):
    import torch.autograd.forward_ad as fwd

    ext = tris["ext"]
    x, w = torch.ones((4, 64), dtype=F16, device=cuda), torch.ones(64, dtype=F16, device=cuda)
    norm = dict(x=x, weight=w, eps=1e-6, residual=x.clone(), out=x.clone(), residual_out=x.clone())
    append = dict(_append_case(cuda, 4, 2, 64, 64, F16, F16, 16, [0, 3], [4, 2]))
    append["q_out"] = torch.zeros_like(append["q"])
    attend = _case(cuda, 4, 2, 64, F16, F16, 16, [10, 3])
    attend["out"] = torch.zeros_like(attend["q"])
    scaled = _case(cuda, 4, 2, 64, F16, E4M3, 16, [10, 3])
    for call, args in ((ext.rms_norm, norm), (ext.rotary_append_paged, append), (ext.paged_attention_decode, attend),
                       (ext.paged_attention_decode, scaled)):
        names = [n for n, t in args.items() if isinstance(t, torch.Tensor) and t.dtype in (F16, torch.float32)]
        assert len(names) > 3 or args is scaled
        for n in names:
            leaf = args[n].detach().clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: leaf})
            with torch.no_grad():
                call(**{**args, n: leaf})
            with fwd.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: fwd.make_dual(args[n], torch.ones_like(args[n]))})


def test_slot_strides_are_bounded_in_bytes(tris):
    """page_size * slot stride stays below 2^31 bytes, whatever the element's size; products that pass 64 bits are caught."""
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(4096)

    def call(**kw):
        rc = lib.tris_paged_attention_decode(p, 512, 128, 0, 4, ctypes.byref(c_cache(**kw)), 0.1, -1, p, 512, 128, p, 1 << 40,
                                             None)
        return rc, lib.tris_last_error()      # (a negative window: nothing is launched)

    e4m3 = dict(dtype=3, k_scale=4096, v_scale=4096)
    most = (1 << 31) // 16
    for kw in (dict(k_slot_stride=most // 2 - 8), dict(v_slot_stride=most // 2 - 8),
               dict(e4m3, k_slot_stride=most - 16), dict(e4m3, k_scale_slot_stride=most // 4 - 1)):
        assert call(**kw) == (-1, b"tris_paged_attention_decode: negative window"), kw
    for kw in (dict(k_slot_stride=most // 2), dict(v_slot_stride=most // 2), dict(e4m3, v_slot_stride=most),
               dict(e4m3, v_scale_slot_stride=most // 4), dict(k_slot_stride=1 << 40), dict(e4m3, k_scale_slot_stride=-1),
               dict(page_size=(1 << 31) - (1 << 17), max_pages=1, k_slot_stride=(1 << 31) - 8),
               dict(page_size=1 << 30, max_pages=1, k_slot_stride=1 << 62)):
        rc, error = call(**kw)
        assert rc == -1 and b"slot stride" in error, (kw, error)


@pytest.mark.gpu
@pytest.mark.parametrize("norms", [None, (64, 64), (512, 128)])
def test_steps_without_tokens(tris, cuda, norms):
    """An empty batch, and prompts of which none has a new token, as the linears and the MoE block take them."""
    from test_attention_layer import _layer
    from tris_moe_amd import attention

    layer = _layer(tris, cuda, 64, 31, norms)
    cache = attention.PagedKVCache(6, 16, 2, 64, F16, cuda)
    cache.k.fill_(3.0), cache.v.fill_(5.0)
    table, lens = torch.zeros((2, 4), dtype=torch.int32, device=cuda), torch.full((2,), 5, dtype=torch.int32, device=cuda)
    x = torch.zeros((0, 512), dtype=F16, device=cuda)
    starts = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert layer.attention.append(x, cache, table, lens, starts).shape == (0, 8, 64)
    assert layer.attention.decode(x, cache, table[:0], lens[:0]).shape == (0, 512)
    for residual in (None, x.to(BF16)):
        out, stream = layer.decode(x.to(BF16), residual, cache, table[:0], lens[:0])
        assert out.shape == stream.shape == (0, 512) and out.dtype == stream.dtype == BF16
    assert bool((cache.k == 3).all()) and bool((cache.v == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_values_under_vanishing_weights(tris, cuda, dim):
    """Keys whose weights fp32 does not hold (2^-1000 and less of the others') do not count, however large their values,
    in pieces of their own too."""
    n, page = 6000, 16
    a = _case(cuda, 4, 2, dim, BF16, BF16, page, [n])
    table = a["block_table"][0].long()
    a["q"].fill_(1.0)
    a["k_cache"][table[: n // page]], a["v_cache"][table[: n // page]] = 0.0, 1.0
    a["k_cache"][table[: n // 2 // page]] = -1000.0 / dim
    a["v_cache"][table[: n // 2 // page]] = torch.finfo(BF16).max
    assert bool((tris["ext"].paged_attention_decode(**a, scale=1.0) == 1.0).all())
