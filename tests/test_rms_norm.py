"""ext.rms_norm (tris_rms_norm) against the formula in 64 bits: types and their mixtures, widths from one value to the
largest, odd widths and strides, the residual stream in place, infinities and NaN, a captured graph, refusals."""
import ctypes

import pytest
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
# offset of a sum, the smallest rounding step of fp16 subnormals, halved
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134}


def _exact(x, w, eps, residual=None, offset=0.0):
    h = x.double().cpu()
    if residual is not None:
        h = h + residual.double().cpu()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (w.double().cpu() + offset), h


def _check(got, want, width, dtype, extra=0.0):
    """One rounding to dtype (half a step: eps / 2 of the value) after fp32 steps: the sum of squares (all terms
    positive: at most width + 1 roundings of 2^-24, halved by the root), the mean, eps, root, two products and the
    weight's offset (2^-23 each at most), and the residual's fp32 addition (extra: its error's share of the value)."""
    half = torch.finfo(dtype).eps / 2
    rel = half * (1 + 1e-3) + (width + 1) * 2.0 ** -25 + 8 * 2.0 ** -23
    err = (got.double().cpu() - want).abs()
    bound = rel * want.abs() + TINY[dtype] + extra
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


def _data(shape, dtype, cuda, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 7, 8, 64, 100, 128, 136, 256, 512, 520, 1000, 1024, 1032, 2048, 4096, 4104, 5001,
                                   8192, 8200, 16384, 32767, 32768])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_widths(tris, cuda, width, dtype):
    for rows in (1, 5, 67):
        print(f"[gpu-case] rms_norm {rows} x {width} {dtype}", flush=True)
        x, w = _data((rows, width), dtype, cuda, width + rows), _data((width,), dtype, cuda, 3)
        got = tris["ext"].rms_norm(x, w, 1e-6)
        assert got.dtype == dtype and got.shape == x.shape
        _check(got, _exact(x, w, 1e-6)[0], width, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [33, 128, 768, 4096, 9000])
@pytest.mark.parametrize("types", [(F16, F16, F16, F16), (BF16, BF16, BF16, BF16), (F16, BF16, F32, F16),
                                   (BF16, F16, F16, BF16), (F16, BF16, BF16, BF16)])
def test_residual_and_types(tris, cuda, width, types):
    tx, tr, tw, to = types
    x, r = _data((9, width), tx, cuda, 1, 3.0), _data((9, width), tr, cuda, 2, 5.0)
    w = _data((width,), tw, cuda, 3)
    got, stream = tris["ext"].rms_norm(x, w, 1e-5, residual=r, weight_offset=1.0, out_dtype=to)
    want, h = _exact(x, w, 1e-5, r, 1.0)
    assert got.dtype == to and stream.dtype == tr
    # h carries one fp32 rounding, relative to itself, and weight + offset one, relative to |w| + 1
    f = want.abs() / (w.double().cpu() + 1.0).abs().clamp_min(1e-12)
    _check(got, want, width, to, extra=2.0 ** -23 * f * (w.double().cpu().abs() + 1.0))
    assert torch.equal(stream, (x.float() + r.float()).to(tr))
    # in place: the stream's own buffer, and the output over x where the types agree
    r2, x2 = r.clone(), x.clone()
    got2, same = tris["ext"].rms_norm(x2, w, 1e-5, residual=r2, weight_offset=1.0, out_dtype=to,
                                      out=x2 if to == tx else None, residual_out=r2)
    assert same is r2 and torch.equal(r2, stream) and torch.equal(got2, got)


@pytest.mark.gpu
@pytest.mark.parametrize("width,stride,start", [(128, 384, 0), (128, 136, 8), (100, 101, 3), (4096, 4100, 4),
                                                (2048, 2056, 1)])
def test_strided_rows(tris, cuda, width, stride, start):
    """Rows inside a wider buffer, 16-byte aligned and not; the output rows leave their neighbours alone."""
    base = _data((7 * stride + 64,), BF16, cuda, 5)
    x = base[start: start + 7 * stride].view(7, stride)[:, :width]
    w = _data((width,), BF16, cuda, 6)
    buf = torch.full((7, stride + 16), 7.0, dtype=BF16, device=cuda)
    got = tris["ext"].rms_norm(x, w, 1e-6, out=buf[:, 8: 8 + width])
    _check(got, _exact(x, w, 1e-6)[0], width, BF16)
    assert bool((buf[:, :8] == 7).all()) and bool((buf[:, 8 + width:] == 7).all())
    heads = _data((3, 5, width), BF16, cuda, 7)
    assert torch.equal(tris["ext"].rms_norm(heads, w, 1e-6).view(15, width),
                       tris["ext"].rms_norm(heads.view(15, width), w, 1e-6))


@pytest.mark.gpu
def test_empty_zero_and_special_rows(tris, cuda):
    ext = tris["ext"]
    w = torch.ones(256, dtype=F16, device=cuda)
    assert ext.rms_norm(torch.empty((0, 256), dtype=F16, device=cuda), w, 1e-6).shape == (0, 256)
    x = torch.zeros((4, 256), dtype=F16, device=cuda)
    x[1, 3], x[2, 5], x[3, :] = float("inf"), float("nan"), 65504.0
    got = ext.rms_norm(x, w, 1e-6).float().cpu()
    assert bool((got[0] == 0).all())
    assert bool(torch.isnan(got[1, 3])) and bool((got[1, :3] == 0).all())      # inf * 0; the others 0 * 0
    assert bool(torch.isnan(got[2]).all())
    assert bool((got[3] == 1).all())


@pytest.mark.gpu
def test_rows_do_not_depend_on_the_batch(tris, cuda):
    ext = tris["ext"]
    for width in (128, 1000, 4096):
        x, w = _data((300, width), BF16, cuda, 11), _data((width,), BF16, cuda, 12)
        whole = ext.rms_norm(x, w, 1e-6)
        assert torch.equal(whole[123:124], ext.rms_norm(x[123:124].contiguous(), w, 1e-6))


@pytest.mark.gpu
def test_graph_and_side_stream(tris, cuda):
    ext = tris["ext"]
    x, r, w = (_data((17, 2048), BF16, cuda, s) for s in (1, 2, 3))
    w = w[0].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ext.rms_norm(x, w, 1e-6, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, stream = ext.rms_norm(x, w, 1e-6, residual=r)
    for seed in (21, 22, 23):
        x.copy_(_data((17, 2048), BF16, cuda, seed))
        graph.replay()
        want, want_stream = ext.rms_norm(x, w, 1e-6, residual=r)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(stream, want_stream)


@pytest.mark.gpu
def test_refusals_on_device(tris, cuda):
    ext = tris["ext"]
    x, w = torch.ones((4, 64), dtype=F16, device=cuda), torch.ones(64, dtype=F16, device=cuda)
    bad = [
        ("float16", dict(x=x.float(), weight=w)),
        ("columns", dict(x=x[:, :32], weight=w)),
        ("contiguous, one stride", dict(x=x.t().contiguous().t(), weight=w)),
        ("contiguous, one stride", dict(x=torch.ones((2, 3, 128), dtype=F16, device=cuda)[:, :2, :64], weight=w)),
        ("shape of x", dict(x=x, weight=w, residual=x[:2])),
        ("needs a residual", dict(x=x, weight=w, residual_out=x)),
        ("weight must be contiguous", dict(x=x, weight=torch.ones(128, dtype=F16, device=cuda)[::2])),
        ("overlap", dict(x=x, weight=w, out=x[:1].expand(4, 64))),
        ("no gradient", dict(x=x, weight=w.clone().requires_grad_())),
    ]
    for match, kw in bad:
        with pytest.raises(RuntimeError, match=match):
            ext.rms_norm(eps=1e-6, **kw)


def test_refusals_without_gpu(tris):
    from tris_moe_amd import _lib

    with pytest.raises(RuntimeError, match="CUDA"):
        tris["ext"].rms_norm(torch.ones((2, 8), dtype=F16), torch.ones(8, dtype=F16), 1e-6)
    lib, p = _lib.load(), ctypes.c_void_p(16)

    def call(rows=2, width=64, x_type=0, r=None, ro=None, out_stride=64, x=p, w_type=0):
        return lib.tris_rms_norm(x, x_type, 64, r, 0, 64, p, w_type, 0.0, 1e-6, rows, width, p, 0, out_stride, ro, 64,
                                 None)

    for kw, word in ((dict(width=0), b"width"), (dict(width=32769), b"width"), (dict(rows=-1), b"rows"),
                     (dict(x_type=2), b"fp16"), (dict(w_type=3), b"fp16"), (dict(x=None), b"null"),
                     (dict(r=p), b"go together"), (dict(ro=p), b"go together"), (dict(out_stride=32), b"overlap")):
        assert call(**kw) == -1 and word in lib.tris_last_error(), kw
    assert call(rows=0, x=None) == 0
