"""What the append and the paged attention promise at their borders: the weights' bits."""
import pytest
import torch

from paged_cases import E4M3

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
