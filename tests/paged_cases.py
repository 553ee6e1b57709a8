"""Paged caches for the append's and the attention's tests: the pool in either order of its dimensions, pages in random
order, and everything outside the sequences NaN."""
import torch

E4M3 = torch.float8_e4m3fn


def nan_fill(t):
    if t.dtype == E4M3:
        t.view(torch.uint8).fill_(0x7F)
    else:
        t.fill_(float("nan"))
    return t


def make_pool(pages, heads, page, dim, dtype, device, order="head"):
    """(k_cache, v_cache, k_scale, v_scale) of NaN; order "token": a [pages, page, heads, dim] buffer, permuted."""
    out = []
    for _ in range(2):
        if order == "head":
            t = torch.empty((pages, heads, page, dim), dtype=dtype, device=device)
        else:
            t = torch.empty((pages, page, heads, dim), dtype=dtype, device=device).permute(0, 2, 1, 3)
        out.append(nan_fill(t))
    for _ in range(2):
        if dtype != E4M3:
            out.append(None)
        elif order == "head":
            out.append(torch.full((pages, heads, page), float("nan"), device=device))
        else:
            out.append(torch.full((pages, page, heads), float("nan"), device=device).permute(0, 2, 1))
    return tuple(out)


def make_table(lengths, page, pages, device, gen, extra=1):
    """int32 [batch, max_pages]: distinct random pages where a sequence has positions, an invalid number elsewhere."""
    need = [-(-n // page) for n in lengths]
    perm = torch.randperm(pages, generator=gen)
    assert sum(need) <= pages
    table = torch.full((len(lengths), max(need + [0]) + extra), -1, dtype=torch.int32)
    table[:, 1::2] = 2 ** 31 - 1
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at: at + n].to(torch.int32)
        at += n
    return table.to(device)


def rows_of(cache, scale, table, b, n, page):
    """Sequence b's first n rows in 64 bits on the host, [heads, n, dim]."""
    j = torch.arange(n)
    pg, slot = table[b].cpu().long()[j // page], j % page
    x = cache.cpu().float().double() if cache.dtype == E4M3 else cache.cpu().double()
    x = x[pg, :, slot].permute(1, 0, 2)
    if scale is not None:
        x = x * scale.cpu().double()[pg, :, slot].permute(1, 0)[..., None]
    return x
