"""Serving in fewer bits: matrix products in 8-bit integers, and attention over a paged cache held in 4 bits.

What a decode step reads is weights and cache; both shrink here.  A case is one call of an operator as a step of the
engine makes it.

Products (``op`` "product"): y = x W^T (+ bias) where every row of W is held as 8-bit codes and one 32-bit scale, and every row
(token) of x is brought to 8 bits in the same way within the call: scale = max|x| / 127, code = round(x / scale), halves to
even, both operations in 32 bits; y = code_x . code_W * scale_x * scale_W, summed in whole numbers.

Cache (``op`` "attention" and "write"): a key or value head of a token is D codes of 4 bits and a pair (scale, zero) of bfloat16:
zero = bfloat16(min x), scale = bfloat16((max x - zero) / 15), code = round((x - zero) / scale) within 0 and 15, in 32 bits; a code
stands for zero + code * scale.  Eight codes fill a 32-bit word, the even columns its lower half, the odd ones its upper half, the
first in the lowest bits.  Codes are [page, kv head, slot, D / 2] bytes, pairs [page, kv head, slot, 2].  "write" brings a step's
keys and values to their slots; "attention" does that and then attends, every query to its request's cached tokens up to itself (with
``window`` W the last W of them), as a layer of the engine does.  Outputs are the attention and the cache's own tensors: codes are
compared bit by bit, which is stricter than by the values that they stand for."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the q/k/v projection of the 0.6B shapes for one decoded token: latency
        {"name": "product 1 x 1024 -> 4096", "op": "product", "M": 1, "K": 1024, "N": 4096, "dtype": "bfloat16", "out32": False, "bias": False, "pad": 0},
        # gate and up of the 8B shapes for eight decoded tokens: the weights are all the traffic
        {"name": "product 8 x 4096 -> 24576", "op": "product", "M": 8, "K": 4096, "N": 24576, "dtype": "bfloat16", "out32": False, "bias": False, "pad": 0},
        # the down projection of the 8B shapes for a full batch of 64
        {"name": "product 64 x 12288 -> 4096", "op": "product", "M": 64, "K": 12288, "N": 4096, "dtype": "bfloat16", "out32": False, "bias": False, "pad": 0},
        # odd sizes throughout, rows that are a slice of wider ones, 32-bit activations and a bias
        {"name": "product 333 x 1501 -> 1003 f32", "op": "product", "M": 333, "K": 1501, "N": 1003, "dtype": "float32", "out32": True, "bias": True, "pad": 11},
        # gate and up of the 8B shapes for a prompt portion that fills the token budget: compute
        {"name": "product 2048 x 4096 -> 24576", "op": "product", "M": 2048, "K": 4096, "N": 24576, "dtype": "bfloat16", "out32": False, "bias": False, "pad": 0},
        # one conversation decodes at the context that the benchmark quotes: latency
        {"name": "decode 1 x 640", "op": "attention", "dtype": "bfloat16", "H": 32, "Hkv": 8, "D": 128, "page": 64, "B": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 640, "kv_hi": 640, "window": 0},
        # a full batch of ragged contexts: the cache is all the traffic
        {"name": "decode 64 x 2000..8192", "op": "attention", "dtype": "bfloat16", "H": 32, "Hkv": 8, "D": 128, "page": 64, "B": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 2000, "kv_hi": 8192, "window": 0},
        # a few long documents: few rows, a long axis
        {"name": "decode 3 x 32000..32768", "op": "attention", "dtype": "bfloat16", "H": 32, "Hkv": 8, "D": 128, "page": 64, "B": 3, "q_lo": 1, "q_hi": 1, "kv_lo": 32000, "kv_hi": 32768, "window": 0},
        # a portion of a long prompt behind the portions before it: compute
        {"name": "portion 2048 of 4096", "op": "attention", "dtype": "bfloat16", "H": 32, "Hkv": 8, "D": 128, "page": 64, "B": 1, "q_lo": 2048, "q_hi": 2048, "kv_lo": 4096, "kv_hi": 4096, "window": 0},
        # ragged portions and single tokens side by side, small pages, a window, seven query heads a key head
        {"name": "mixed 24 x 1..300, window 333", "op": "attention", "dtype": "bfloat16", "H": 14, "Hkv": 2, "D": 64, "page": 16, "B": 24, "q_lo": 1, "q_hi": 300, "kv_lo": 1, "kv_hi": 1500, "window": 333},
        # the true 32-bit path over the same cache
        {"name": "decode 5 x 700..1900 f32", "op": "attention", "dtype": "float32", "H": 16, "Hkv": 8, "D": 128, "page": 16, "B": 5, "q_lo": 1, "q_hi": 1, "kv_lo": 700, "kv_hi": 1900, "window": 0},
        # the keys and values of a whole token budget on their way to the cache
        {"name": "write 4095 tokens", "op": "write", "dtype": "bfloat16", "H": 8, "Hkv": 8, "D": 128, "page": 64, "B": 3, "q_lo": 1000, "q_hi": 1365, "kv_lo": 1400, "kv_hi": 5000, "window": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "decode", "decode", "portion", "mixed", "f32", "write"])
    if kind == "product":
        while True:
            c = {"op": "product", "M": _log(rng, 1, 2500), "K": _log(rng, 64, 12500), "N": _log(rng, 64, 25000), "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]),
                 "bias": rng.random() < 0.3, "pad": rng.choice([0, 0, 8, 13])}
            if rng.random() < 0.6:          # widths of layers are mostly round
                c["K"], c["N"] = -(-c["K"] // 64) * 64, -(-c["N"] // 64) * 64
            c["out32"] = c["dtype"] == "float32" or rng.random() < 0.2
            if c["M"] * c["K"] * c["N"] <= 2048 * 4096 * 24576:
                return c
    while True:
        Hkv = rng.choice([1, 2, 4, 8])
        c = {"op": "write" if kind == "write" else "attention", "dtype": "float32" if kind == "f32" else "bfloat16", "H": Hkv * rng.choice([1, 2, 4, 5, 7, 8]), "Hkv": Hkv,
             "D": rng.choice([64, 128, 128, 128, 96]), "page": rng.choice([16, 32, 64]), "window": rng.choice([0, 0, 0, _log(rng, 16, 4000)])}
        if kind in ("decode", "f32"):
            c.update(B=_log(rng, 1, 64 if kind == "decode" else 6), q_lo=1, q_hi=1, kv_hi=_log(rng, 40, 32768 if kind == "decode" else 2000))
            c["kv_lo"] = _log(rng, 1, c["kv_hi"])
        elif kind == "portion":
            n = _log(rng, 65, 2048)
            c.update(B=1, q_lo=n, q_hi=n, kv_lo=n + _log(rng, 1, 2048) - 1)
            c["kv_hi"] = c["kv_lo"]
        elif kind == "mixed":
            c.update(B=_log(rng, 2, 30), q_lo=1, q_hi=_log(rng, 2, 300), kv_lo=1, kv_hi=_log(rng, 64, 2000))
        else:
            n = _log(rng, 1, 1365)
            c.update(B=_log(rng, 1, 3), q_lo=-(-n // 2), q_hi=n, kv_lo=n, kv_hi=n + _log(rng, 1, 4000))
        rows = c["B"] * (c["kv_lo"] + c["kv_hi"]) / 2
        if rows * c["Hkv"] * c["D"] <= 64 * 5000 * 8 * 128 and c["B"] * c["H"] * c["q_hi"] * c["kv_hi"] <= 2.7e8:
            return c


# ------------------------------------------------------------------------------------------------- inputs
def _lengths(c):
    """(queries, cached tokens with them) of every request: spread over the case's ranges, the same for every seed, so that
    a case is always the same work."""
    import random
    rng = random.Random(c["B"] * 1000003 + c["q_hi"] * 1009 + c["kv_hi"])
    q, kv = [], []
    for b in range(c["B"]):
        n = c["q_lo"] if c["q_lo"] == c["q_hi"] else (1 if c["op"] == "attention" and b % 3 == 0 else _log(rng, c["q_lo"], c["q_hi"]))
        m = c["kv_hi"] if b == 0 else rng.randint(c["kv_lo"], c["kv_hi"])
        q.append(min(n, max(m, 1)) if c["op"] == "attention" else n)
        kv.append(max(m, q[-1]))
    return q, kv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "product":
        M, K, N = case["M"], case["K"], case["N"]
        # a layer's activations: a few columns are much larger than the rest
        columns = torch.exp(0.6 * torch.randn(K, generator=g, device="cuda"))
        x = (torch.randn(M, K + case["pad"], generator=g, device="cuda") * torch.cat([columns, columns[:case["pad"]]])).to(dtype)[:, :K]
        stride = -(-K // 16) * 16          # rows of codes begin on 16 bytes, as the framework's own weights do
        codes = torch.randn(N, stride, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)[:, :K]
        scales = torch.rand(N, generator=g, device="cuda").add_(0.5).mul_(0.02 / 32)
        bias = torch.randn(N, generator=g, device="cuda").to(dtype) if case["bias"] else None
        return SimpleNamespace(op="product", x=x, codes=codes, scales=scales, bias=bias, out32=case["out32"])
    H, Hkv, D, page, B = case["H"], case["Hkv"], case["D"], case["page"], case["B"]
    q_lens, kv_lens = _lengths(case)
    T = sum(q_lens)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g, device="cuda").to(dtype)
    blocks = [-(-n // page) for n in kv_lens]
    pages, width = sum(blocks) + 1, max(blocks)
    order = (torch.randperm(pages - 1, generator=g, device="cuda") + 1).int().tolist()
    table, at = torch.zeros(B, width, dtype=torch.int32), 0
    for b, n in enumerate(blocks):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    slots = torch.cat([table[b].long()[torch.arange(m - n, m) // page] * page + torch.arange(m - n, m) % page for b, (n, m) in enumerate(zip(q_lens, kv_lens))]).int()
    caches = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, Hkv, page, D // 2), generator=g, device="cuda", dtype=torch.uint8)
        scale = torch.rand(pages, Hkv, page, generator=g, device="cuda").add_(0.5).mul_(0.25)
        zero = -7.5 * scale * (1 + 0.1 * torch.randn(pages, Hkv, page, generator=g, device="cuda"))
        caches.append((codes, torch.stack([scale, zero], -1).to(torch.bfloat16)))
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    table = table.cuda()
    view = SimpleNamespace(page_size=page, max_blocks=width, slot_mapping=slots.cuda(), block_table=table, num_pages=pages)
    kv = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    ctx = SimpleNamespace(cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), kv_lens=kv, num_tokens=T, num_requests=B, max_q_len=max(q_lens), max_kv_len=max(kv_lens),
                          host={"cu_q": cu, "kv_lens": kv_lens})
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, Hkv * D, Hkv * D], 1))
    return SimpleNamespace(op=case["op"], q=q.contiguous(), k=k, v=v, k_codes=caches[0][0], k_pairs=caches[0][1], v_codes=caches[1][0], v_pairs=caches[1][1], view=view, ctx=ctx,
                           scale=D ** -0.5, window=case["window"])


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s.op == "product":
        if own:
            from tinyserve_b200.kernels import ops
            return ops.linear(s.x, ops.Int8Rows(s.codes, s.scales), s.bias, out_float32=s.out32)
        return _plain_product(s)
    if own:
        from tinyserve_b200.kernels import ops
        k_cache, v_cache = ops.Int4Pages(s.k_codes, s.k_pairs), ops.Int4Pages(s.v_codes, s.v_pairs)
        ops.int4_kvwrite(s.k, s.v, k_cache, v_cache, s.view.slot_mapping)
        out = ops.paged_attention(s.q, k_cache, v_cache, s.view, s.ctx, s.scale, s.window) if s.op == "attention" else None
    else:
        _plain_write(s.k, s.k_codes, s.k_pairs, s.view)
        _plain_write(s.v, s.v_codes, s.v_pairs, s.view)
        out = _plain_attention(s) if s.op == "attention" else None
    return {"out": out, "k_codes": s.k_codes, "k_pairs": s.k_pairs, "v_codes": s.v_codes, "v_pairs": s.v_pairs}


def _over(x, n):
    """x / n, rounded once (by a number of the host, torch multiplies by its reciprocal)."""
    return x / x.new_full((), n)


def _plain_product(s):
    x = s.x.float()
    scale = _over(x.abs().amax(1, keepdim=True), 127)
    codes = torch.where(scale > 0, (x / scale).round(), 0)
    y = (codes @ s.codes.float().t()) * (scale * s.scales)
    if s.bias is not None:
        y = y + s.bias.float()
    return y if s.out32 else y.to(s.x.dtype)


def _word_shifts(device):
    """Where the eight columns of a word stand in it."""
    i = torch.arange(8, device=device)
    return (i // 2 * 4 + i % 2 * 16).int()


def _plain_write(x, codes, pairs, view):
    x = x.float()
    zero = x.amin(-1, keepdim=True).to(torch.bfloat16).float()
    scale = _over(x.amax(-1, keepdim=True) - zero, 15).to(torch.bfloat16).float()
    c = torch.where(scale > 0, ((x - zero) / scale).round().clamp(0, 15), 0).int()
    words = (c.unflatten(-1, (-1, 8)) << _word_shifts(x.device)).sum(-1).int()          # (the terms share no bit)
    page, slot = (view.slot_mapping // view.page_size).long(), (view.slot_mapping % view.page_size).long()
    codes[page, :, slot] = words.view(torch.uint8)
    pairs[page, :, slot] = torch.cat([scale, zero], -1).to(torch.bfloat16)


def _plain_read(codes, pairs, table):
    """The cached rows of every request as 32-bit numbers: [B, kv head, token, D]."""
    words = codes.view(torch.int32)[table.long()]                            # [B, block, kv head, slot, D / 8]
    pair = pairs[table.long()].float()
    x = ((words.unsqueeze(-1) >> _word_shifts(codes.device)) & 15).flatten(-2) * pair[..., :1] + pair[..., 1:]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    c, q = s.ctx, s.q
    T, H, D = q.shape
    k, v = _plain_read(s.k_codes, s.k_pairs, s.view.block_table), _plain_read(s.v_codes, s.v_pairs, s.view.block_table)
    B, Hkv, kv = k.shape[:3]
    n, m = c.cu_q.diff()[:, None], c.kv_lens[:, None]
    i, j = torch.arange(c.max_q_len, device=q.device), torch.arange(kv, device=q.device)
    rows = (c.cu_q[:-1, None] + torch.minimum(i, n - 1)).long()                # [B, max_q_len]; rows behind a request's last repeat it
    at = m - n + torch.minimum(i, n - 1)                                       # their positions
    qs = q[rows].float().view(B, -1, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = (qs @ k.transpose(-1, -2)).view(B, Hkv, -1, H // Hkv, kv).mul_(s.scale)
    seen = j <= at[..., None]
    if s.window > 0:
        seen = seen & (j > at[..., None] - s.window)
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (p.flatten(2, 3) @ v) / p.sum(-1).flatten(2, 3)[..., None]
    out = out.view(B, Hkv, -1, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, -1, H, D)
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(c.cu_q[1:].contiguous(), t.int(), right=True)
    return out[b, t - c.cu_q[b]].to(q.dtype)


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "product":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": N * K + 4 * N + M * K * e + M * N * (4 if case["out32"] else e) + (N * e if case["bias"] else 0), "flops": 2 * M * K * N}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    q, kv = _lengths(case)
    row = Hkv * (D / 2 + 4)
    new = sum(q) * 2 * (Hkv * D * e + row)
    if case["op"] == "write":
        return {"bytes": new, "flops": 0}
    W = case["window"] or max(kv)
    read = sum(min(m, n + W - 1) - n for n, m in zip(q, kv)) * 2 * row          # (the new rows are at hand)
    pairs = sum(min(m - n + i + 1, W) for n, m in zip(q, kv) for i in range(n))
    return {"bytes": new + read + 2 * sum(q) * H * D * e, "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "product":
        # the codes are defined by 32-bit operations; everything after them is exact
        x = s.x.to(torch.float32)
        top = torch.maximum(x.amax(1), -x.amin(1))
        step = torch.div(top, torch.full_like(top, 127.0))
        codes = torch.nan_to_num(torch.div(x, step[:, None])).round().double()
        y = torch.einsum("mk,nk->mn", codes, s.codes.double()) * step.double()[:, None] * s.scales.double()
        return y if s.bias is None else y + s.bias.double()
    order = [0, 2, 4, 6, 1, 3, 5, 7]                                           # the columns of a word, from its lowest bits on
    tensors = {}
    for name, x in (("k", s.k.float()), ("v", s.v.float())):
        low = x.min(-1).values.bfloat16()
        span = x.max(-1).values - low.float()
        step = torch.div(span, torch.full_like(span, 15.0)).bfloat16()
        c = torch.div(x - low.float()[..., None], step.float()[..., None]).nan_to_num().round().clamp(0, 15).to(torch.uint8)
        c = c.unflatten(-1, (-1, 8))[..., order].flatten(-2)
        codes, pairs = getattr(s, name + "_codes").clone(), getattr(s, name + "_pairs").clone()
        for t, slot in enumerate(s.view.slot_mapping.tolist()):
            at = (slot // s.view.page_size, slice(None), slot % s.view.page_size)
            codes[at] = c[t, :, 0::2] | c[t, :, 1::2] << 4
            pairs[at] = torch.stack([step[t], low[t]], -1)
        tensors[name] = (codes, pairs)
    answer = {"out": None, "k_codes": None, "k_pairs": tensors["k"][1].double(), "v_codes": None, "v_pairs": tensors["v"][1].double()}
    if s.op == "write":
        return answer
    q = s.q.double()
    T, H, D = q.shape
    Hkv = case["Hkv"]
    place = torch.tensor([order.index(i) for i in range(8)], device=q.device)
    out = torch.zeros_like(q)
    cu, kv = s.ctx.host["cu_q"], s.ctx.host["kv_lens"]
    for b in range(case["B"]):
        table = s.view.block_table[b, :-(-kv[b] // s.view.page_size)].long()
        dense = []
        for name in ("k", "v"):
            codes, pairs = tensors[name][0][table], tensors[name][1][table].double()      # [block, kv head, slot, ..]
            nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))[..., place].flatten(-2)
            x = pairs[..., 1:] + nibbles.double() * pairs[..., :1]
            dense.append(x.transpose(0, 1).flatten(1, 2)[:, :kv[b]])
        n = cu[b + 1] - cu[b]
        for g in range(Hkv):
            heads = slice(g * (H // Hkv), (g + 1) * (H // Hkv))
            score = torch.einsum("thd,jd->htj", q[cu[b]:cu[b + 1], heads], dense[0][g]) * s.scale
            at = torch.arange(kv[b] - n, kv[b], device=q.device)[:, None]
            j = torch.arange(kv[b], device=q.device)
            hidden = (j > at) | ((j <= at - s.window) if s.window > 0 else torch.zeros_like(j > at))
            score = score.masked_fill(hidden, -math.inf)
            out[cu[b]:cu[b + 1], heads] = torch.einsum("htj,jd->thd", torch.softmax(score, -1), dense[1][g])
    answer["out"] = out
    return answer
