"""Decode loops whose caches are kept within a budget: append with given rotary positions, attention that sums its weights and
eviction together, as ext's calls and through tris_moe_amd.attention, eager and captured."""
import pytest
import torch

from paged_cases import E4M3, make_pool
from test_attention_layer import DIM, HIDDEN, _layer, _plan
from test_attention_weights import check_sums
from test_paged_attention import _check
from test_paged_cache import _bits
from test_paged_evict import NAMES, expected
from test_rotary_axes import expected_axes, turn_axes

F16, BF16 = torch.float16, torch.bfloat16


def test_constructors_on_the_cpu():
    from tris_moe_amd import attention

    c = attention.PagedKVCache(3, 5, 2, 64, F16, device="cpu")
    assert c.weight_sum is None
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(torch.zeros((1, 3), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 4)
    c.track_weights(4, 15)
    assert c.weight_sum.shape == (4, 2, 15) and c.weight_sum.dtype == torch.float32 and not bool(c.weight_sum.any())

    class P:
        def __init__(self, i, o):
            self.infeatures, self.outfeatures = i, o

    proj = [P(512, 512), P(512, 128), P(512, 128), P(512, 512)]
    cos, sin = attention.rotary_tables(64, 10, device="cpu")
    att = attention.TrisPagedAttention(*proj, 8, 2, 64, cos, sin, sections=[12, 10, 10], interleaved=True)
    assert att.sections == (12, 10, 10)
    with pytest.raises(ValueError, match="sections"):
        attention.TrisPagedAttention(*proj, 8, 2, 64, cos, sin, sections=(12, 10, 9))


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F16, F16), (BF16, E4M3)], ids=str)
@pytest.mark.parametrize("page,budget,limit", [(16, 40, 47), (5, 33, 33)])
def test_steps_against_the_formulas(tris, cuda, types, page, budget, limit):
    """Prompts and decode steps of a ragged batch with an idle place: every call against its formula on what it found, and
    the rows that are left against the tokens they were made from, wherever the evictions have put them."""
    ext = tris["ext"]
    dtype, cache = types
    q_heads, heads, dim, sections, sink, recent = 6, 2, 64, (12, 10, 10), 3, 8
    prompts, steps = [30, 45, 0, 5, 1], 40
    batch, idle, most = len(prompts), 2, limit + 1
    g = torch.Generator().manual_seed(page)
    per = -(-max(most, max(prompts) + 1) // page)
    pages = batch * per
    a = dict(zip(NAMES, make_pool(pages, heads, page, dim, cache, cuda)))
    for n in NAMES:                                     # (every page is in a table: the host's copies compare numbers)
        if a[n] is not None:
            a[n].zero_()
    a["block_table"] = torch.randperm(pages, generator=g).view(batch, per).to(torch.int32).to(cuda)
    sums = torch.zeros((batch, heads, per * page), device=cuda)
    freq = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(300, dtype=torch.float64)[:, None] * freq
    cos, sin = angle.cos().float().to(cuda), angle.sin().float().to(cuda)
    length = torch.tensor(prompts)                      # in the cache
    age = torch.tensor(prompts)                         # tokens that the sequence has had
    tokens = {b: [] for b in range(batch)}              # (key, value, positions) of each
    where = torch.full((batch, heads, per * page), -1)  # the token in each place

    def append(new):
        total = sum(new)
        q, k, v = (torch.randn((total, n, dim), generator=g).to(dtype).to(cuda) for n in (q_heads, heads, heads))
        lens = length.to(torch.int32).to(cuda)
        pos = torch.stack([torch.cat([torch.arange(int(age[b]) - n, int(age[b])) * f + e for b, n in enumerate(new)])
                           for f, e in ((1, 0), (1, 7), (2, 1))]).to(torch.int32)
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
        call = dict(a, q=q, k=k, v=v, cos=cos, sin=sin, seq_lens=lens, query_start=starts)
        before = [int(length[b]) - n for b, n in enumerate(new)]
        want = expected_axes(call, before, new, pos, sections, True)
        out = ext.rotary_append_paged(**call, positions=pos.to(cuda), sections=sections, interleaved=True)
        for got, w in zip((out, *(a[n] for n in NAMES)), want):
            assert w is None or torch.equal(_bits(got), _bits(w))
        at = 0
        for b, n in enumerate(new):
            for i in range(n):
                where[b, :, before[b] + i] = len(tokens[b])
                tokens[b].append((k[at].cpu(), v[at].cpu(), pos[:, at]))
                at += 1
        return out, lens

    append(prompts)
    evictions = 0
    for _ in range(steps):
        new = [int(b != idle) for b in range(batch)]
        length += torch.tensor(new)
        age += torch.tensor(new)
        q, lens = append(new)
        full = torch.zeros((batch, q_heads, dim), dtype=dtype, device=cuda)
        full[[b for b in range(batch) if b != idle]] = q
        state = dict(a, q=full, seq_lens=lens)
        before = sums.clone()
        y = ext.paged_attention_decode(**state, weight_sum=sums)
        _check(state, length.tolist(), y)
        check_sums(state, length.tolist(), before, sums)
        call = dict(a, seq_lens=lens, weight_sum=sums)
        out, left, new_lens, kept = expected(call, budget, limit, sink, recent)
        got_lens, got_kept = ext.paged_cache_evict(**call, budget=budget, limit=limit, sink=sink, recent=recent)
        assert torch.equal(got_lens.cpu(), new_lens) and torch.equal(got_kept.cpu(), kept)
        assert torch.equal(sums.cpu(), left)
        for n in NAMES:
            assert out[n] is None or torch.equal(_bits(a[n]), _bits(out[n]))
        for b in range(batch):
            if int(kept[b, 0, 0]) >= 0:
                where[b, :, :budget] = where[b].gather(1, kept[b].long())
                evictions += 1
        length = new_lens.long()
    assert evictions > (20 if budget == limit else 4)
    for b in range(batch):
        n = int(length[b])
        if n == 0:
            continue
        j = torch.arange(n)
        pg, slot = a["block_table"][b].cpu().long()[j // page], j % page
        assert n <= limit and torch.equal(where[b, :, :sink], torch.arange(sink).expand(heads, -1))
        for h in range(heads):
            ids = where[b, h, :n].tolist()
            assert ids == sorted(ids) and ids[-1] == int(age[b]) - 1
            k, v = (torch.stack([tokens[b][i][c][h] for i in ids])[:, None] for c in (0, 1))
            pos = torch.stack([tokens[b][i][2] for i in ids], 1)
            k = turn_axes(k, cos.cpu(), sin.cpu(), pos, sections, True, torch.float32)[:, 0]
            for x, name in ((k, "k"), (v[:, 0].float(), "v")):
                got = a[f"{name}_cache"].cpu()[pg, h, slot]
                if cache == E4M3:
                    f = x.abs().amax(-1) * torch.tensor(1.0 / 448.0, dtype=torch.float32)
                    assert torch.equal(a[f"{name}_scale"].cpu()[pg, h, slot], f)
                    x = x / f[:, None]
                assert torch.equal(_bits(got), _bits(x.to(cache)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, E4M3])
def test_layers_within_a_budget(tris, cuda, dtype):
    """Two decoder layers over steps in which sequences outgrow the budget, their lengths kept on the device: eager and
    captured give the same, and the modules what the separate calls give."""
    from tris_moe_amd import attention

    page, steps, kv = 16, 12, 2
    prompts = [18, 30, 0, 1]
    budget = dict(budget=24, limit=27, sink=2, recent=6)
    batch, idle = len(prompts), 2
    table, pages = _plan(cuda, page, max(prompts) + 1, batch)
    places = table.shape[1] * page
    layers = [_layer(tris, cuda, 200, seed, None, kv) for seed in (31, 47)]
    for layer in layers:
        layer.attention.sections, layer.attention.interleaved = (16, 8, 8), False
    g = torch.Generator().manual_seed(1)
    starts = torch.tensor([0] + prompts).cumsum(0).to(torch.int32).to(cuda)
    lens0 = torch.tensor(prompts, dtype=torch.int32, device=cuda)
    x0 = [torch.randn((sum(prompts), HIDDEN), generator=g).to(F16).to(cuda) for _ in layers]
    p0 = torch.stack([torch.cat([torch.arange(n) + 3 * i for n in prompts]) for i in range(3)]).to(torch.int32).to(cuda)
    xs = torch.randn((steps, batch, HIDDEN), generator=g).to(BF16).to(cuda)
    active = torch.tensor([int(b != idle) for b in range(batch)], dtype=torch.int32, device=cuda)

    class Run:
        def __init__(self):
            self.caches = [attention.PagedKVCache(pages, page, kv, DIM, dtype, cuda) for _ in layers]
            self.lens, self.x = lens0.clone(), xs[0].clone()
            self.age = torch.stack([lens0, lens0 + 3, lens0 + 6]).contiguous()
            for layer, cache, x in zip(layers, self.caches, x0):
                for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
                    if t is not None:
                        t.zero_()
                cache.track_weights(batch, places)
                layer.attention.append(x, cache, table, self.lens, starts, p0)

        def step(self):
            self.lens.add_(active)
            pair = (self.x, None)
            for layer, cache in zip(layers, self.caches):
                pair = layer.decode(*pair, cache, table, self.lens, self.age)
            new = [cache.evict(table, self.lens, **budget)[0] for cache in self.caches]
            self.lens.copy_(new[-1])
            self.age.add_(active)
            return (*pair, *new)

        def tensors(self):
            return [t for c in self.caches for t in (c.k, c.v, c.k_scale, c.v_scale, c.weight_sum) if t is not None] + [
                self.lens, self.age]

    eager, calls = Run(), Run()
    warm = Run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.step()
    torch.cuda.current_stream().wait_stream(side)
    captured = Run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = captured.step()
    assert torch.equal(captured.lens, lens0)
    ext = tris["ext"]
    for step in range(steps):
        for r in (eager, captured, calls):
            r.x.copy_(xs[step])
        want = eager.step()
        graph.replay()
        # the separate calls
        calls.lens.add_(active)
        pair = (calls.x, None)
        for layer, c in zip(layers, calls.caches):
            x, residual = pair
            att = layer.attention
            h = ext.rms_norm(x, layer.input_norm, layer.norm_eps, residual=residual, out_dtype=F16)
            h, residual = (h, x) if residual is None else h
            q, k, v = (p(h).view(batch, -1, DIM) for p in (att.q_proj, att.k_proj, att.v_proj))
            kw = dict(k_scale=c.k_scale, v_scale=c.v_scale)
            q = ext.rotary_append_paged(q, k, v, att.cos, att.sin, c.k, c.v, table, calls.lens, **kw, positions=calls.age,
                                        sections=(16, 8, 8))
            y = ext.paged_attention_decode(q, c.k, c.v, table, calls.lens, **kw, weight_sum=c.weight_sum)
            h, residual = ext.rms_norm(att.o_proj(y.view(batch, -1)), layer.post_norm, layer.norm_eps, residual=residual,
                                       out_dtype=BF16)
            pair = (layer.block(h[None])[0][0], residual)
        new = [ext.paged_cache_evict(c.k, c.v, table, calls.lens, c.weight_sum, **budget, k_scale=c.k_scale,
                                     v_scale=c.v_scale)[0] for c in calls.caches]
        calls.lens.copy_(new[0])
        calls.age.add_(active)
        torch.cuda.synchronize()
        for x, y, z in zip(want, outs, (*pair, *new)):
            assert torch.equal(x, y) and torch.equal(x, z)
        for x, y, z in zip(eager.tensors(), captured.tensors(), calls.tensors()):
            assert torch.equal(_bits(x), _bits(y)) and torch.equal(_bits(x), _bits(z))
        assert bool(torch.isfinite(want[0].float()).all()) and int(eager.lens.max()) <= 27
    assert eager.lens.tolist() == [26, 27, 0, 13]       # 28 becomes 24
