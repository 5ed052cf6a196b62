"""Requests over a 4-bit cache of random codes, on any device, and how exact a result has to be: so that a key more or less, a sink or a soft
cap left out shows."""
import math
from types import SimpleNamespace as NS

import torch

from test_fewer_bits_gpu import values

# lengths of requests: (queries, cached tokens with them)
LENGTHS = {"decode": [(1, 1), (1, 64), (1, 65), (1, 700)], "long": [(1, 5000)], "many": [(1, 97 + 31 * i) for i in range(40)], "portions": [(3, 3), (70, 200), (33, 33)],
           "wide": [(300, 900), (5, 260), (1, 1000), (64, 64)], "mixed": [(1, 300), (40, 100), (1, 1), (0, 17), (129, 129)]}
# (window, soft cap, sinks)
OPTIONS = [(0, 0.0, False), (0, 0.0, True), (50, 0.0, True), (100, 0.0, False), (1, 2.0, False), (100, 1.5, True), (0, 1.5, False)]


def requests(lengths, Hkv, D, page, device, seed=0):
    """(ctx, view, k cache, v cache, [k], [v]): values around zero of about 1, every slot that no request has full of NaN; the lists hold
    what the cached rows stand for, in 64 bits."""
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(seed + sum(m for _, m in lengths) + D)
    B, width = len(lengths), max(1, max(-(-m // page) for _, m in lengths))
    table = (torch.randperm(B * width, generator=g) + 1).int().view(B, width)
    slots = [table[b].long()[torch.arange(m) // page] * page + torch.arange(m) % page for b, (_, m) in enumerate(lengths)]
    caches, rows = [], []
    for _ in range(2):
        codes = torch.randint(0, 256, (B * width + 1, Hkv, page, D // 2), generator=g, dtype=torch.uint8)
        scale = torch.rand(B * width + 1, Hkv, page, generator=g) * 0.25 + 0.125
        pairs = torch.stack([scale, -7.5 * scale * (1 + 0.1 * torch.randn(scale.shape, generator=g))], -1).bfloat16()
        free = torch.ones((B * width + 1) * page, dtype=torch.bool)
        free[torch.cat(slots)] = False
        pairs.transpose(1, 2)[free.view(-1, page)] = math.nan
        cache = ops.Int4Pages(codes.to(device), pairs.to(device))
        dense = values(cache).transpose(1, 2).flatten(0, 1)
        caches.append(cache)
        rows.append([dense[s.to(device)] for s in slots])
    cu = [0]
    for n, _ in lengths:
        cu.append(cu[-1] + n)
    kv = [m for _, m in lengths]
    ctx = NS(cu_q=torch.tensor(cu, dtype=torch.int32, device=device), kv_lens=torch.tensor(kv, dtype=torch.int32, device=device), num_requests=B, num_tokens=cu[-1],
             max_q_len=max(n for n, _ in lengths), max_kv_len=max(kv), host={"cu_q": cu, "kv_lens": kv})
    view = NS(block_table=table.to(device), page_size=page, slot_mapping=None, num_pages=B * width + 1, max_blocks=width)
    return ctx, view, *caches, *rows


def queries(T, H, D, device):
    """(queries, sinks): a sink weighs as much as some hundred keys, so that it shows beside thousands."""
    g = torch.Generator().manual_seed(7)
    return torch.randn(T, H, D, generator=g).bfloat16().to(device), 6 + torch.randn(H, generator=g).to(device)


def of_requests(lengths):
    """Slices of the rows of every request that has some."""
    at = 0
    for n, m in lengths:
        if n and m:
            yield slice(at, at + n)
        at += n


def exact_enough(out, want, dtype):
    """float32: a score of some sqrt(D) in products of size 1 is off by few half steps of 2^-24, and so are the sums over keys: 64 of them.

    bfloat16: inside, everything is rounded to 11 bits or more, an eighth of the result's half step; roots of sums of squares: eight such
    roundings a term add (1 / 8)^2 8 = 1 / 8 to the square of what rounding the exact result makes, a factor of 1.06.  Of N elements
    the sum of the products of both errors is no zero: three times its deviation is 3 sqrt(1 / 8) / sqrt(N) of that square, half as much of the root."""
    off = (out.double() - want).norm()
    if dtype == torch.float32:
        return bool(off <= 2.0 ** -18 * want.norm())
    rounding = (want.bfloat16().double() - want).norm()
    return bool(off <= (1.06 + 1.5 * math.sqrt(1 / 8) * 2 / math.sqrt(want.numel())) * rounding)
