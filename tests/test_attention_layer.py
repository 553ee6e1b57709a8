"""tris_moe_amd.attention: the paged attention module and the decoder layer's decode step, the new operators and the
compact3 projections and MoE block run together: against the formulas in 64 bits, against the separate calls bit for
bit, over several steps of a ragged batch with an idle place, eager and captured."""
import numpy as np
import pytest
import torch

from paged_cases import E4M3
from test_linear import _modules
from test_paged_attention import _check
from test_paged_cache import _bits, _turn

F16, BF16 = torch.float16, torch.bfloat16
HIDDEN, HEADS, KV, DIM = 512, 8, 2, 64


def test_tables_and_constructors_on_the_cpu():
    from tris_moe_amd import attention

    cos, sin = attention.rotary_tables(64, 70000, 1e6, device="cpu")
    i, p = 7, 69999
    angle = p * 1e6 ** (-2 * i / 64)
    assert cos.shape == (70000, 32) and cos.dtype == torch.float32
    assert abs(float(cos[p, i]) - np.cos(angle)) < 2 ** -24 and abs(float(sin[p, i]) - np.sin(angle)) < 2 ** -24
    for bad in (0, 8, 24, -16):
        with pytest.raises(ValueError, match="rotary_dim"):
            attention.rotary_tables(bad, 4, device="cpu")
    c = attention.PagedKVCache(3, 5, 2, 64, E4M3, device="cpu")
    assert c.k.shape == c.v.shape == (3, 2, 5, 64) and c.k_scale.shape == (3, 2, 5) and c.k.dtype == E4M3
    assert attention.PagedKVCache(3, 5, 2, 64, BF16, device="cpu").k_scale is None
    with pytest.raises(ValueError, match="head_dim"):
        attention.PagedKVCache(3, 5, 2, 96, device="cpu")
    with pytest.raises(ValueError, match="float16"):
        attention.PagedKVCache(3, 5, 2, 64, torch.float32, device="cpu")

    class P:
        def __init__(self, i, o):
            self.infeatures, self.outfeatures = i, o

    good = [P(512, 512), P(512, 128), P(512, 128), P(512, 512)]
    for at, proj, word in ((0, P(512, 256), "q_proj"), (1, P(512, 64), "k_proj"), (2, P(512, 512), "v_proj"),
                           (3, P(256, 512), "o_proj")):
        with pytest.raises(ValueError, match=word):
            attention.TrisPagedAttention(*(good[:at] + [proj] + good[at + 1:]), 8, 2, 64, cos, sin)
    with pytest.raises(ValueError, match="multiple"):
        attention.TrisPagedAttention(*good, 8, 3, 64, cos, sin)


def _linear(qlinear, mod, infeatures, outfeatures, cuda):
    m = qlinear.Compact3Linear(infeatures, outfeatures)
    return m.load_tensors(mod).to(cuda)


def _attention(tris, cuda, positions, heads=HEADS, kv=KV, seed=3, rot=DIM, window=0, norms=None):
    from tris_moe_amd import attention, qlinear

    sizes = [(HIDDEN, heads * DIM), (HIDDEN, kv * DIM), (HIDDEN, kv * DIM), (heads * DIM, HIDDEN)]
    mods = [_modules(tris["ext"], 1, n, k, seed + i)[0][0] for i, (k, n) in enumerate(sizes)]
    lin = [_linear(qlinear, m, k, n, cuda) for m, (k, n) in zip(mods, sizes)]
    cos, sin = attention.rotary_tables(rot, positions, device=cuda)
    q_norm = k_norm = None
    if norms is not None:
        g = torch.Generator().manual_seed(seed)
        q_norm, k_norm = ((1 + 0.1 * torch.randn(n, generator=g)).to(F16).to(cuda) for n in norms)
    return attention.TrisPagedAttention(*lin, heads, kv, DIM, cos, sin, q_norm, k_norm, window=window), mods


def _plan(cuda, page, most, batch):
    g = torch.Generator().manual_seed(9)
    per = -(-most // page)
    table = torch.randperm(batch * per + 2, generator=g)[: batch * per].view(batch, per).to(torch.int32).to(cuda)
    return table, batch * per + 2


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4)])
@pytest.mark.parametrize("window", [0, 9])
def test_attention_against_64_bits(tris, oracle_mod, cuda, heads, kv, window):
    """A prompt appended, then a decode step, all in 64 bits from the dequantised projections, with the error that the
    path's fp16 roundings may make carried through: h = 2^-11 a rounding; projections (their rounding and K 2^-23 of
    their fp32 sums), the rotation's output, the scores' effect on the weights, values, the attention's output."""
    from tris_moe_amd import attention

    page, prompt = 16, 37
    att, mods = _attention(tris, cuda, 64, heads, kv, window=window)
    table, pages = _plan(cuda, page, prompt + 1, 1)
    cache = attention.PagedKVCache(pages, page, kv, DIM, F16, cuda)
    rng = np.random.default_rng(5)
    x = torch.from_numpy((rng.standard_normal((prompt + 1, HIDDEN)) * 0.7).astype(np.float16)).to(cuda)
    starts = torch.tensor([0, prompt], dtype=torch.int32, device=cuda)
    att.append(x[:prompt].contiguous(), cache, table, torch.tensor([prompt], dtype=torch.int32, device=cuda), starts)
    got = att.decode(x[prompt:].contiguous(), cache, table,
                     torch.tensor([prompt + 1], dtype=torch.int32, device=cuda)).cpu().double()[0]

    w = [torch.from_numpy(oracle_mod.dequant_grouped_expert(oracle_mod.module_as_payload(m), 0)).double() for m in mods]
    x64, h = x.cpu().double(), 2.0 ** -11 * (1 + 2 ** -6)
    cos, sin = att.cos.cpu(), att.sin.cpu()
    pos = torch.arange(prompt + 1)

    def project(i, n):
        y = (x64 @ w[i].T).view(prompt + 1, n, DIM)
        return y, h * y.abs() + HIDDEN * 2.0 ** -23 * (x64.abs() @ w[i].abs().T).view(y.shape) + 2.0 ** -25

    def turn(y, e):
        z = _turn(y, cos, sin, pos, torch.float64)
        big = e.view(*e.shape[:2], 2, DIM // 2).sum(2)          # |cos|, |sin| <= 1: both partners' errors
        return z, torch.cat([big, big], -1) + h * z.abs() + 2.0 ** -22 * (z.abs() + 1e-3)

    def far(shift):
        """The largest error in units of its bound; shift 1 plants a mistake in the formula: the values of the
        neighbouring positions.  (With these weights the scores are nearly flat, so that a mistake in the rotation moves
        the output by less than the bound; the append's tests hold the rotation bit for bit.)"""
        (q, dq), (k, dk), (v, dv) = turn(*project(0, heads)), turn(*project(1, kv)), project(2, kv)
        v, dv = v.roll(shift, 0), dv.roll(shift, 0)
        first = max(0, prompt + 1 - window) if window else 0
        q, dq = q[-1], dq[-1]
        k, dk, v, dv = (t[first:].repeat_interleave(heads // kv, 1) for t in (k, dk, v, dv))
        s = torch.einsum("hd,thd->ht", q, k) * DIM ** -0.5
        ds = (torch.einsum("hd,thd->ht", dq, k.abs() + dk) + torch.einsum("hd,thd->ht", q.abs(), dk)) * DIM ** -0.5
        p = torch.softmax(s, -1)
        y = torch.einsum("ht,thd->hd", p, v)
        dy = torch.expm1(2 * ds.amax(-1, keepdim=True) + 2.0 ** -12) * torch.einsum("ht,thd->hd", p, v.abs() + dv)
        dy = dy + torch.einsum("ht,thd->hd", p, dv) + h * y.abs()
        out, dout = w[3] @ y.reshape(-1), w[3].abs() @ dy.reshape(-1)
        dout = dout + h * out.abs() + heads * DIM * 2.0 ** -23 * (w[3].abs() @ y.abs().reshape(-1)) + 2.0 ** -25
        return ((got - out).abs() / dout).max().item()

    assert far(0) <= 1.0
    if window:
        assert far(1) > 1.0     # the bound is narrow enough to see this


def _layer(tris, cuda, positions, seed, norms=None, kv=KV):
    from tris_moe_amd import attention
    from tris_moe_amd.configs import MoELayerSpec

    synthetic, qlinear, moe = tris["synthetic"], tris["qlinear"], tris["moe"]
    spec = MoELayerSpec("t", hidden=HIDDEN, num_experts=8, intermediate=768, top_k=2, rank=256, tokens=(4,))
    data = synthetic.make_layer(spec, seed, tris["ext"].gr_encode)
    payloads = {p: qlinear.payload_to_device(data[p], cuda) for p in ("gate", "up", "down")}
    backbones = {p: torch.from_numpy(data["backbones"][p]).to(cuda) for p in ("gate", "up", "down")}
    g = torch.Generator().manual_seed(seed)
    router = (torch.randn((8, HIDDEN), generator=g) * 0.05).to(BF16)
    block = moe.TrisSparseMoeBlock(HIDDEN, 8, 2, payloads, backbones, router_weight=router).to(cuda)
    att, _ = _attention(tris, cuda, positions, kv=kv, seed=seed, norms=norms)
    w = [(1 + 0.1 * torch.randn(HIDDEN, generator=g)).to(BF16).to(cuda) for _ in range(2)]
    return attention.TrisDecoderLayer(att, block, *w)


def _by_calls(tris, layer, x, residual, cache, table, lens):
    """The layer's step by the separate public calls; also what the attention read and gave."""
    ext, att = tris["ext"], layer.attention
    h = ext.rms_norm(x, layer.input_norm, layer.norm_eps, residual=residual, out_dtype=F16)
    h, residual = (h, x) if residual is None else h
    q, k, v = (p(h).view(len(h), -1, DIM) for p in (att.q_proj, att.k_proj, att.v_proj))
    if att.q_norm is not None:
        q = ext.rms_norm(q, att.q_norm, att.norm_eps) if att.q_norm.numel() == DIM else \
            ext.rms_norm(q.reshape(len(h), -1), att.q_norm, att.norm_eps).view(q.shape)
        k = ext.rms_norm(k, att.k_norm, att.norm_eps) if att.k_norm.numel() == DIM else \
            ext.rms_norm(k.reshape(len(h), -1), att.k_norm, att.norm_eps).view(k.shape)
    kw = dict(k_scale=cache.k_scale, v_scale=cache.v_scale)
    q = ext.rotary_append_paged(q, k, v, att.cos, att.sin, cache.k, cache.v, table, lens, **kw)
    y = ext.paged_attention_decode(q, cache.k, cache.v, table, lens, **kw)
    h, residual = ext.rms_norm(att.o_proj(y.view(len(h), -1)), layer.post_norm, layer.norm_eps, residual=residual,
                               out_dtype=BF16)
    out, _ = layer.block(h[None])
    return (out[0], residual), dict(q=q, k_cache=cache.k, v_cache=cache.v, block_table=table, seq_lens=lens, **kw), y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, E4M3])
@pytest.mark.parametrize("norms,kv", [(None, 2), ((DIM, DIM), 2), ((HEADS * DIM, HEADS * DIM), 8)])
def test_layers_over_several_steps(tris, cuda, dtype, norms, kv):
    from tris_moe_amd import attention

    page, steps = 12, 5
    prompts = [7, 40, 0, 1]
    batch, most = len(prompts), max(prompts) + steps
    table, pages = _plan(cuda, page, most, batch)
    layers = [_layer(tris, cuda, table.shape[1] * page, seed, norms, kv) for seed in (31, 47)]
    caches = [[attention.PagedKVCache(pages, page, kv, DIM, dtype, cuda) for _ in layers] for _ in range(3)]
    g = torch.Generator().manual_seed(1)
    idle = 2
    starts = torch.tensor(np.concatenate([[0], np.cumsum(prompts)]), dtype=torch.int32, device=cuda)
    lens0 = torch.tensor(prompts, dtype=torch.int32, device=cuda)
    for i, layer in enumerate(layers):
        x = torch.randn((sum(prompts) + 2, HIDDEN), generator=g).to(F16).to(cuda)      # two padded rows
        for c in caches:
            layer.attention.append(x, c[i], table, lens0, starts)
    xs = torch.randn((steps, batch, HIDDEN), generator=g).to(BF16).to(cuda)
    lens = lens0.clone()

    def run(cache, x):
        pair = (x, None)
        for layer, c in zip(layers, cache):
            pair = layer.decode(*pair, c, table, lens)
        return pair

    def advance(step):
        n = [p + step + 1 for p in prompts]
        n[idle] = 0
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        return n

    # a captured run of the same steps, on a cache of its own
    x_in = xs[0].clone()
    advance(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(caches[2], x_in)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(caches[2], x_in)
    for step in range(steps):
        n = advance(step)
        out, stream = run(caches[0], xs[step])
        x_in.copy_(xs[step])
        graph.replay()
        pair = (xs[step], None)
        for layer, c in zip(layers, caches[1]):
            pair, state, y = _by_calls(tris, layer, *pair, c, table, lens)
            _check(state, n, y)
        torch.cuda.synchronize()
        assert torch.equal(out, pair[0]) and torch.equal(stream, pair[1])
        assert torch.equal(captured[0], out) and torch.equal(captured[1], stream)
        assert bool(torch.isfinite(out.float()).all())
    for i in range(len(layers)):
        for name in ("k", "v", "k_scale", "v_scale"):
            a, b, c = (getattr(cs[i], name) for cs in caches)
            if a is not None:
                for s, p in enumerate(prompts):
                    if s == idle:
                        continue
                    for j in range(p + steps):
                        at = (int(table[s, j // page]), slice(None), j % page)
                        assert torch.equal(_bits(a[at]), _bits(b[at])) and torch.equal(_bits(a[at]), _bits(c[at]))
