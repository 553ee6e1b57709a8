"""ext.paged_cache_evict on memory that its arguments share: keys and values that overlap are refused wherever they begin, and
parts of one buffer that interleave are not."""
import ctypes

import pytest
import torch

from paged_cases import E4M3
from test_paged_cache import c_cache
from test_paged_evict import evict_case, run_and_check

F16, BF16 = torch.float16, torch.bfloat16


def _evict(c, lens=1 << 40, new_lens=1 << 41, kept=1 << 42):
    """The C entry on addresses that are never read: for calls that it refuses.  (rc, message)"""
    from tris_moe_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(1 << 39)
    c.seq_lens = lens
    rc = lib.tris_paged_cache_evict(ctypes.byref(c), p, 96, 48, 8, 8, 1, 2, ctypes.c_void_p(new_lens),
                                    ctypes.c_void_p(kept), None, 0, None)
    return rc, lib.tris_last_error()


PAGE, HEAD, SLOT = 2 * 4096, 2 * 2048, 2 * 128       # bytes, of c_cache's pool: 4 pages of 2 heads of 16 rows


@pytest.mark.parametrize("to", [16, SLOT - 16, SLOT, HEAD, PAGE, 3 * PAGE + HEAD, 4 * PAGE - 16])
@pytest.mark.parametrize("way", [1, -1])
def test_keys_over_values_are_refused(tris, to, way):
    """Views of one buffer some columns, slots, heads or pages apart."""
    base = 1 << 38
    assert _evict(c_cache(k=base, v=base + way * to)) == (-1, b"tris_paged_cache_evict: keys and values must not share memory")


@pytest.mark.parametrize("to,strides", [
    (PAGE, (2 * 4096, 2048, 128)),                   # every other page, the first of the values one of the keys' later ones
    (HEAD, (2 * 4096, 2 * 2048, 128)),
    (SLOT, (2 * 4096, 2 * 2048, 2 * 128))], ids=["pages", "heads", "slots"])
def test_interleaved_keys_and_values_that_meet_are_refused(tris, to, strides):
    """As the layouts of one buffer below, but the values begin 16 bytes before their place."""
    base = 1 << 38
    c = c_cache(k=base, v=base + to - 16)
    for n in "kv":
        for field, s in zip(("page", "head", "slot"), strides):
            setattr(c, f"{n}_{field}_stride", s)
    assert _evict(c) == (-1, b"tris_paged_cache_evict: keys and values must not share memory")


@pytest.mark.parametrize("to", [4, 16 * 4, 32 * 4, 3 * 32 * 4 + 4])
def test_scales_over_scales_are_refused(tris, to):
    base = 1 << 38
    c = c_cache(k=1 << 36, v=1 << 37, dtype=3, k_scale=base, v_scale=base + to)
    for n in "kv":
        for field, s in (("page", 32), ("head", 16), ("slot", 1)):
            setattr(c, f"{n}_scale_{field}_stride", s)
    assert _evict(c) == (-1, b"tris_paged_cache_evict: keys and values must not share memory")


@pytest.mark.parametrize("batch,to", [(2, 0), (2, 4), (2, -4), (9, 32), (9, -32), (9, 2), (9, -35)])
def test_new_lengths_over_lengths_are_refused(tris, batch, to):
    c = c_cache(k=1 << 36, v=1 << 37, batch=batch)
    rc, message = _evict(c, new_lens=(1 << 40) + to)
    assert rc == -1 and b"new_lens must not overlap seq_lens" in message


@pytest.mark.parametrize("of", ["lens", "new_lens"])
@pytest.mark.parametrize("to", [0, 4, -4, -127, 7 - 4 * 2 * 2 * 8])
def test_kept_over_lengths_is_refused(tris, of, to):
    """Two sequences of two heads keep eight each: 128 bytes."""
    at = dict(lens=1 << 40, new_lens=1 << 41)
    rc, message = _evict(c_cache(k=1 << 36, v=1 << 37), **at, kept=at[of] + to)
    assert rc == -1 and b"kept must not overlap the lengths" in message


# one buffer of keys and values, by its dimensions (c: which of the two; o: a part that the pool leaves out)
LAYOUTS = ["cphsd", "pchsd", "phcsd", "phscd", "pschd", "psdhc", "pcshd", "opchsd"]


def _one_buffer(t, u, layout, letters, device):
    """Copies of t and u as parts of one buffer."""
    sizes = dict(zip(letters, t.shape), c=2, o=3)
    names = [n for n in layout if n in letters + "co"]
    if letters[-1] == "d":                            # rows stay whole
        names = [n for n in names if n != "d"] + ["d"]
    whole = torch.empty([sizes[n] for n in names], dtype=t.dtype, device=device)
    whole.view(torch.uint8).fill_(0x55)
    part = whole.select(names.index("o"), 1) if "o" in names else whole
    names = [n for n in names if n != "o"]
    rest = [n for n in names if n != "c"]
    parts = [part.select(names.index("c"), i).permute([rest.index(n) for n in letters]) for i in range(2)]
    for p, x in zip(parts, (t, u)):
        p.copy_(x)
    return whole, parts


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_one_buffer(tris, cuda, cache, layout):
    """Keys and values of one buffer, one behind the other or interleaved by page, head, slot or row; the scales alike."""
    a = evict_case(cuda, 3, 64, cache, 7, [150, 61, 20], seed=len(layout))
    whole, (a["k_cache"], a["v_cache"]) = _one_buffer(a["k_cache"], a["v_cache"], layout, "phsd", cuda)
    if cache == E4M3:
        _, (a["k_scale"], a["v_scale"]) = _one_buffer(a["k_scale"], a["v_scale"], layout, "phs", cuda)
    print(f"[gpu-case] evict one buffer {cache} {layout}", flush=True)
    run_and_check(tris, a, 40, 60, 3, 11)
    if "o" in layout:
        assert bool((whole[::2].view(torch.uint8) == 0x55).all())


@pytest.mark.gpu
def test_padded_pages(tris, cuda):
    """Interleaved rows in pages whose stride the rows' stride does not divide; keys and values laid out differently within
    a page."""
    a = evict_case(cuda, 2, 64, F16, 8, [100, 33], seed=5)
    pages = a["k_cache"].shape[0]
    raw = torch.zeros(pages * 2056 + 2048, dtype=F16, device=cuda)
    rows = [raw.as_strided((pages, 2, 8, 64), (2056, 1024, 128, 1), 64 * i).copy_(a[n]) for i, n in
            enumerate(("k_cache", "v_cache"))]
    run_and_check(tris, {**a, "k_cache": rows[0], "v_cache": rows[1], "weight_sum": a["weight_sum"].clone()}, 30, None, 2, 5)
    raw = torch.zeros(pages * 2056, dtype=F16, device=cuda)
    k = raw.as_strided((pages, 2, 8, 64), (2056, 512, 64, 1)).copy_(a["k_cache"])
    v = raw.as_strided((pages, 2, 8, 64), (2056, 64, 128, 1), 1024).copy_(a["v_cache"])
    run_and_check(tris, {**a, "k_cache": k, "v_cache": v}, 30, None, 2, 5)


@pytest.mark.gpu
def test_overlapping_views_are_refused(tris, cuda):
    a = evict_case(cuda, 2, 64, F16, 16, [100, 30])
    pages = a["k_cache"].shape[0]
    buffer = torch.zeros((pages + 1, 2, 16, 64), dtype=F16, device=cuda)
    e = evict_case(cuda, 2, 64, E4M3, 16, [100, 30])
    scales = torch.ones((pages + 1, 2, 16), device=cuda)
    for args, kw in ((a, dict(k_cache=buffer[:-1], v_cache=buffer[1:])), (a, dict(k_cache=buffer[1:], v_cache=buffer[:-1])),
                     (e, dict(k_scale=scales[:-1], v_scale=scales[1:]))):
        with pytest.raises(RuntimeError, match="share memory"):
            tris["ext"].paged_cache_evict(**{**args, **kw}, budget=20)
