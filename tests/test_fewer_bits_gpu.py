"""Products in 8-bit integers and attention over a 4-bit cache against their definitions in 64 bits."""
import math
from types import SimpleNamespace as NS

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}          # half a step, relative to the value
COLUMN = [i // 2 * 4 + i % 2 * 16 for i in range(8)]                   # where a word's eight columns stand


def over(x, n):
    """x / n rounded once (by a number of the host, torch multiplies by its reciprocal)."""
    return x / torch.full_like(x, n)


def row_codes(x):
    """(codes, scales) of rows in 8 bits, by the definition: 32-bit operations."""
    x = x.float()
    scale = over(x.abs().amax(1), 127)
    return torch.where(scale[:, None] > 0, (x / scale[:, None]).round(), 0).nan_to_num(), scale


def product(x, rows, bias=None):
    """The product of x and rows in 8 bits, and how far a kernel may be: one rounding each for the sum, the product of the scales,
    their product and the bias, and of the result."""
    codes, scale = row_codes(x)
    y = (codes.double() @ rows.codes.double().T) * scale.double()[:, None] * rows.scales.double()
    err = 4 * 2.0 ** -24 * y.abs()
    if bias is not None:
        err += 2.0 ** -24 * (y.abs() + bias.double().abs())
        y = y + bias.double()
    return y, err


def rows_of(N, K, seed=0):
    from tinyserve_b200.kernels import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ops.quantize_rows(torch.randn(N, K, generator=g, device="cuda") * torch.rand(N, 1, generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K,pad", [(1, 1, 0), (3, 17, 0), (5, 1000, 8), (2, 4096, 0), (130, 257, 3), (1, 20001, 0)])
def test_rows_in_8_bits(dtype, R, K, pad):
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(R + K)
    x = (torch.randn(R, K + pad, generator=g) * torch.exp(torch.randn(R, 1, generator=g))).to(dtype).cuda()[:, :K]
    x[R // 2, : K // 2] = 0
    if R > 2:
        x[0] = 0
        x[1, -1] = math.inf
        x[2, 0] = math.nan
    got = ops.quantize_rows(x)
    codes, scale = row_codes(x)
    bad = ~torch.isfinite(x).all(1)
    assert torch.equal(got.scales.isnan(), bad) and torch.equal(got.scales[~bad], scale[~bad])
    assert torch.equal(got.codes[~bad].float(), codes[~bad]) and not got.codes[bad].any()
    assert got.codes.stride(0) % 16 == 0


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 4096, 1024), (2, 130, 48), (16, 129, 4096), (17, 1000, 333), (33, 64, 2064), (64, 4096, 12288), (65, 257, 1024),
                                   (200, 300, 160), (300, 384, 4096), (1025, 640, 512)])
@pytest.mark.parametrize("kind", ["bf16", "f32", "bf16 out32 bias", "f32 bias16"])
def test_product(M, N, K, kind):
    from tinyserve_b200.kernels import ops
    dtype = torch.bfloat16 if kind.startswith("bf16") else torch.float32
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randn(M, K + 5, generator=g, device="cuda").to(dtype)[:, :K]
    rows = rows_of(N, K)
    bias = torch.randn(N, generator=g, device="cuda").to(torch.bfloat16 if kind.endswith("16") else torch.float32) if "bias" in kind else None
    out = ops.linear(x, rows, bias, out_float32="out32" in kind)
    assert out.dtype == (torch.float32 if "out32" in kind else dtype)
    want, err = product(x, rows, bias)
    assert ((out.double() - want).abs() <= err + HALF[out.dtype] * want.abs() + 1e-30).all()
    assert torch.equal(ops.linear(ops.quantize_rows(x), rows, bias, out_float32=out.dtype == torch.float32), out)
    assert ops.gemm_int8_error() == 0


def test_product_of_extremes():
    """The longest sum of the largest codes, and rows of zeros, infinities and NaN beside ordinary ones."""
    from tinyserve_b200.kernels import ops
    K = ops.INT8_MAX_K
    rows = ops.Int8Rows(torch.full((3, K), -127, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
    x = torch.ones(2, K, device="cuda")
    x[1] = -1
    assert torch.equal(ops.linear(x, rows).double(), (torch.tensor([[-127.0], [127.0]]).double() * K).cuda().expand(2, 3))
    rows = rows_of(70, 96)
    x = torch.randn(4, 96, device="cuda")
    x[0] = 0
    x[1, 3] = math.inf
    x[2, 5] = math.nan
    out = ops.linear(x, rows)
    want, err = product(x[3:], rows)
    assert not out[0].any() and out[1:3].isnan().all() and ((out[3:].double() - want).abs() <= err + HALF[torch.float32] * want.abs()).all()


# ------------------------------------------------------------------------------------------------- the cache
def coded(x):
    """(codes, pair) of heads in 4 bits, by the definition."""
    x = x.float()
    zero = x.amin(-1).bfloat16()
    scale = over(x.amax(-1) - zero.float(), 15).bfloat16()
    s = scale.float()[..., None]
    codes = torch.where(s > 0, ((x - zero.float()[..., None]) / s).round().clamp(0, 15), 0)
    return codes, torch.stack([scale, zero], -1)


def words(codes):
    bits = codes.long().unflatten(-1, (-1, 8)) << torch.tensor(COLUMN, device=codes.device)
    bits = bits.sum(-1)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int().view(torch.uint8)


def values(cache):
    """What a 4-bit cache stands for, in 64 bits: [page, head, slot, D]."""
    w = cache.codes.view(torch.int32)
    codes = ((w[..., None] >> torch.tensor(COLUMN, device=w.device).int()) & 15).flatten(-2).double()
    return cache.pairs[..., 1:].double() + codes * cache.pairs[..., :1].double()


def empty_cache(pages, Hkv, page, D, fill=255):
    """A pool whose every slot is full of codes with a pair of NaN: nothing of it may reach a result."""
    from tinyserve_b200.kernels import ops
    return ops.Int4Pages(torch.full((pages, Hkv, page, D // 2), fill, dtype=torch.uint8, device="cuda"),
                         torch.full((pages, Hkv, page, 2), math.nan, dtype=torch.bfloat16, device="cuda"))


def batch(lengths, Hkv, D, page, dtype, seed=0, spread=1.0):
    """Requests (queries, cached tokens) with a cache that the kernel filled: (ctx, view, k cache, v cache, [k], [v]); the lists hold what
    the cached rows of every request stand for, in 64 bits."""
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(seed + sum(m for _, m in lengths) + D)
    B, width = len(lengths), max(1, max(-(-m // page) for _, m in lengths))
    table = (torch.randperm(B * width, generator=g) + 1).int().view(B, width)
    kc, vc = empty_cache(B * width + 1, Hkv, page, D), empty_cache(B * width + 1, Hkv, page, D)
    slots = torch.cat([table[b].long()[torch.arange(m) // page] * page + torch.arange(m) % page for b, (_, m) in enumerate(lengths)] + [torch.tensor([-1])]).int().cuda()
    fill = [(torch.randn(slots.numel(), Hkv, D, generator=g) * spread + torch.randn(1, Hkv, D, generator=g)).to(dtype).cuda() for _ in range(2)]
    ops.int4_kvwrite(fill[0], fill[1], kc, vc, slots)
    dense = []
    for c in (kc, vc):
        x = values(c).transpose(1, 2).flatten(0, 1)                 # [slot, head, D]
        dense.append([x[slots[a:a + m].long()] for a, m in zip(_starts([m for _, m in lengths]), [m for _, m in lengths])])
    cu = _starts([n for n, _ in lengths]) + [sum(n for n, _ in lengths)]
    ctx = NS(cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), kv_lens=torch.tensor([m for _, m in lengths], dtype=torch.int32).cuda(), num_requests=B,
             num_tokens=cu[-1], max_q_len=max(n for n, _ in lengths), max_kv_len=max(m for _, m in lengths), host={"cu_q": cu, "kv_lens": [m for _, m in lengths]})
    view = NS(block_table=table.cuda(), page_size=page, slot_mapping=None, num_pages=B * width + 1, max_blocks=width)
    return ctx, view, kc, vc, dense[0], dense[1]


def _starts(ns):
    return [sum(ns[:i]) for i in range(len(ns))]


def attention(q, lengths, ks, vs, scale, window=0, softcap=0.0, sinks=None):
    """In 64 bits: (result, largest sum of a score's terms |q| (|zero| + code scale), largest range of a value head and largest value)."""
    H, D = q.shape[1:]
    out, at, top, span = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0, 0.0, 0.0
    for (n, m), k, v in zip(lengths, ks, vs):
        G = H // k.shape[1]
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        s = torch.einsum("thd,jhd->htj", q[at:at + n].double(), k) * scale
        if n and m:
            low = k.amin(-1, keepdim=True)             # (its zero: the least column of a head has code 0)
            top = max(top, float(torch.einsum("thd,jhd->htj", q[at:at + n].double().abs(), low.abs() + (k - low)).max()) * scale)
            span = max(span, float(v.abs().max()) + float((v.amax(-1) - v.amin(-1)).max()))
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        pos, j = torch.arange(m - n, m, device=q.device)[:, None], torch.arange(m, device=q.device)
        s = s.masked_fill((j > pos) | ((j <= pos - window) if window else (j < 0)), -math.inf)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None, None].expand(H, n, 1)], -1)
            v = torch.cat([v, torch.zeros_like(v[:1])]) if m else torch.zeros(1, H, D, dtype=torch.float64, device=q.device)
        p = torch.softmax(s, -1).nan_to_num() if s.shape[-1] else s
        out[at:at + n] = torch.einsum("htj,jhd->thd", p, v)
        at += n
    return out, top, span


def allowed(dtype, want, top, span, D, keys):
    """32 bits, sums in any order, additions that cut off (two half steps): a score of D products is off by 2 (D + 8) half steps of its
    terms' sum, a probability by twice that, a sum over the keys by two a key of terms up to twice the range.  bfloat16: the
    probabilities (times their value's scale) and the result are rounded to at least its bits; what queries as 16-bit integers (2^-16 of a row's largest element
    each) and keys in half precision (2^-11) add to a score is, for these inputs, below a quarter of that."""
    t = 2.0 ** -24 * (4 * (D + 8) * top + 4 * (keys + 64)) * span
    return t if dtype == torch.float32 else t + 2.0 ** -8 * span + HALF[dtype] * want.abs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,Hkv,D,page", [(1, 1, 16, 1), (3, 2, 96, 16), (7, 8, 128, 64), (33, 3, 64, 4), (2, 1, 512, 32), (5, 2, 256, 8),
                                           (300, 2, 128, 64), (257, 3, 64, 16), (256, 1, 512, 32), (259, 5, 96, 1), (300, 1, 16, 8), (256, 2, 160, 16)])
def test_write(dtype, T, Hkv, D, page):
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(T + D)
    pages = -(-T // page) + 2
    # a slice of a fused projection, rows of one value, zeros, a wide range, an infinity, a NaN and a range that overflows
    x = (torch.randn(T, (2 * Hkv + 1) * D, generator=g) * torch.exp(3 * torch.randn(T, 1, generator=g))).to(dtype).cuda()
    k, v = x[:, D:].view(T, 2, Hkv, D).unbind(1)
    k[0, 0] = 0
    if T > 2:
        v[1, 0] = 1.25
        k[2, 0, 3], v[2, 0, 5] = math.inf, math.nan
        v[2, -1, 0], v[2, -1, 1] = 3e38, -3e38
    slots = (torch.randperm(pages * page, generator=g)[:T]).int()
    if T > 4:
        slots[4] = -1
    slots = slots.cuda()
    kc, vc = empty_cache(pages, Hkv, page, D, 170), empty_cache(pages, Hkv, page, D, 170)
    ops.int4_kvwrite(k, v, kc, vc, slots)
    live = slots >= 0
    for y, c in ((k, kc), (v, vc)):
        codes, pair = coded(y)
        bad = ~torch.isfinite(pair.float()).all(-1) | ~torch.isfinite(y.float()).all(-1)
        codes[bad], pair[bad] = 0, math.nan
        flat, pairs = c.codes.transpose(1, 2).reshape(-1, Hkv, D // 2), c.pairs.transpose(1, 2).reshape(-1, Hkv, 2)
        assert torch.equal(flat[slots[live].long()], words(codes[live]))
        got, want = pairs[slots[live].long()], pair[live]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[slots[live].long()] = False
        assert (flat[rest] == 170).all() and pairs[rest].isnan().all()
        # a code is off by half a step of its row's scale; the pair's rounding may clamp the ends of the range
        off = (pair[..., 1:].float() + codes * pair[..., :1].float() - y.float()).abs()[~bad]
        top = y.float().abs().amax(-1)[~bad]
        assert (off <= 0.5 * pair[..., :1].float()[~bad] + (2.0 ** -8 * 3 * top)[:, None] + 1e-30).all()


LENGTHS = {"wide": [(300, 900), (5, 260), (1, 1000), (64, 64)], "one": [(1, 1)], "decode": [(1, 1), (1, 64), (1, 65), (1, 700)], "long": [(1, 5000)], "portions": [(3, 3), (70, 200), (33, 33)], "mixed": [(1, 300), (40, 100), (1, 1), (0, 17), (129, 129)]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 4, 16, 8), (8, 2, 128, 64), (14, 2, 64, 16), (3, 3, 96, 1), (20, 1, 256, 32), (2, 1, 512, 16), (9, 1, 32, 64), (32, 8, 128, 16), (5, 1, 160, 64), (2, 1, 224, 16)])
@pytest.mark.parametrize("name", sorted(LENGTHS))
def test_attention(dtype, H, Hkv, D, page, name):
    from tinyserve_b200.kernels import ops
    lengths = LENGTHS[name]
    ctx, view, kc, vc, ks, vs = batch(lengths, Hkv, D, page, dtype)
    q = torch.randn(ctx.num_tokens, H + 1, D, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()[:, :H]
    sinks = torch.randn(H, device="cuda")
    for window, softcap, sink, splits in ((0, 0.0, None, None), (0, 0.0, None, 3), (50, 0.0, sinks, None), (1, 2.0, None, None), (100, 5.0, sinks, 12)):
        want, top, span = attention(q, lengths, ks, vs, D ** -0.5, window, softcap, sink)
        chosen = ops.int4_attention_backend(dtype, D)
        for backend in {chosen, "simt"} | ({"mma"} if chosen == "tcgen05" else set()):
            out = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, window, sinks=sink, softcap=softcap, num_splits=splits, backend=backend)
            assert ((out.double() - want).abs() <= allowed(dtype, want, top, span, D, max(m for _, m in lengths))).all(), (window, softcap, splits, backend)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_keys_and_behind_the_last(dtype):
    """A request with more queries than cached tokens has rows that see nothing: zeros.  Rows behind the last request change nobody's result."""
    from tinyserve_b200.kernels import ops
    lengths = [(1, 40), (2, 2)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, 64, 16, dtype)
    q = torch.randn(6, 4, 64, device="cuda").to(dtype)
    alone = ops.paged_attention(q[:3], kc, vc, view, ctx, 0.125)
    assert torch.equal(ops.paged_attention(q, kc, vc, view, ctx, 0.125)[:3], alone)
    ctx.kv_lens = torch.tensor([40, 1], dtype=torch.int32).cuda()
    out = ops.paged_attention(q[:3], kc, vc, view, ctx, 0.125)
    assert not out[1].any() and torch.equal(out[0], alone[0]) and out[2].any()
    ctx.kv_lens = torch.tensor([0, 0], dtype=torch.int32).cuda()
    assert not ops.paged_attention(q[:3], kc, vc, view, ctx, 0.125).any()
    assert not ops.paged_attention(q[:3], kc, vc, view, ctx, 0.125, sinks=torch.zeros(4, device="cuda")).any()
    assert ops.paged_attention(q[:0], kc, vc, view, ctx, 0.125).shape == (0, 4, 64)


@pytest.mark.parametrize("H", [8, 6, 2])
@pytest.mark.parametrize("window", [0, 2])
def test_non_finite_rows_reach_who_sees_them(H, window):
    from tinyserve_b200.kernels import ops
    lengths = [(3, 90), (1, 5)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, 128, 16, torch.bfloat16)
    q = torch.randn(4, H, 128, device="cuda").bfloat16()
    clean = ops.paged_attention(q, kc, vc, view, ctx, 0.1, window)
    j = 88                                     # the last query but one sees it, the first does not
    page = int(view.block_table[0, j // 16])
    for c in (kc, vc):
        keep = c.pairs.clone()
        c.pairs[page, 1, j % 16] = math.nan
        out = ops.paged_attention(q, kc, vc, view, ctx, 0.1, window)
        c.pairs.copy_(keep)
        assert torch.equal(out[0], clean[0]) and torch.equal(out[3], clean[3]) and torch.equal(out[:, :H // 2], clean[:, :H // 2])
        assert out[1:3, H // 2:].isnan().all()
    assert ops.int4_attention_error(128) == 0


def test_pages_outside_the_pool_are_reported():
    from tinyserve_b200.kernels import ops
    ctx, view, kc, vc, ks, vs = batch([(1, 40)], 1, 64, 16, torch.bfloat16)
    q = torch.randn(1, 2, 64, device="cuda").bfloat16()
    words_ = ops.status_words()
    assert not words_.any()
    try:
        view.block_table[0, 1] = 10 ** 6
        ops.paged_attention(q, kc, vc, view, ctx, 0.1)
        torch.cuda.synchronize()
        with pytest.raises(ops.DeviceError, match="page"):
            ops.raise_on_device_error()
        words_[:] = 0
        x = torch.randn(1, 1, 64, device="cuda")
        ops.int4_kvwrite(x, x, kc, vc, torch.tensor([10 ** 6], dtype=torch.int32).cuda())
        torch.cuda.synchronize()
        with pytest.raises(ops.DeviceError, match="slot"):
            ops.raise_on_device_error()
    finally:
        words_[:] = 0


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e12, 1e-12, 1e25), (1e-12, 1e12, 1e-25), (1.0, 1.0, 1e-36), (1e-30, 1e30, 1e30)])
@pytest.mark.parametrize("grows", [0.0, 0.02, -0.02])
def test_attention_of_any_magnitude(D, page, q_size, k_size, v_size, grows):
    """Magnitudes that no 16-bit format but bfloat16 holds, and values that grow or shrink 2^10 over a request: a row is as exact as the
    largest value that it sees (two roundings to bfloat16 of what it adds, and the result's)."""
    from tinyserve_b200.kernels import ops
    lengths = [(500, 500), (1, 450), (40, 300)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, D, page, torch.bfloat16)
    # powers of two: the codes stay, the pairs are exact
    k_by, v_by = 2.0 ** round(math.log2(k_size)), 2.0 ** round(math.log2(v_size))
    kc.pairs.mul_(k_by)
    ks = [x * k_by for x in ks]
    q = (torch.randn(ctx.num_tokens, 8, D, generator=torch.Generator().manual_seed(9)) * q_size).bfloat16().cuda()
    bound = []
    for b, (n, m) in enumerate(lengths):
        by = v_by * torch.exp2((torch.arange(m) * grows).round()).double().cuda()
        at = view.block_table[b].long()[torch.arange(m) // page], torch.arange(m) % page
        vc.pairs[at[0], :, at[1]] = (vc.pairs[at[0], :, at[1]].double() * by[:, None, None]).bfloat16()
        vs[b] = vs[b] * by[:, None, None]
        bound.append(vs[b].abs().amax((1, 2)).cummax(0).values[m - n:])
    bound = torch.cat(bound)[:, None, None]
    scale = D ** -0.5 * 0.5 / (q_size * k_by)
    want, _, _ = attention(q, lengths, ks, vs, scale)
    for backend in ("tcgen05", "mma", "simt"):
        out = ops.paged_attention(q, kc, vc, view, ctx, scale, backend=backend)
        assert ((out.double() - want).abs() <= 2 * 2.0 ** -8 * bound + HALF[torch.bfloat16] * want.abs()).all(), backend


@pytest.mark.parametrize("H,Hkv", [(8, 2), (4, 4)])
def test_a_captured_step_serves_other_lengths(H, Hkv):
    """Write and attention captured for requests of one length, replayed for others of as many tokens: offsets, lengths, tables and slots
    are read on the device, the host's numbers are bounds."""
    from tinyserve_b200.kernels import ops
    D, page, T = 128, 16, 66
    ctx, view, kc, vc, _, _ = batch([(33, 400), (33, 400)], Hkv, D, page, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").bfloat16() for h in (H, Hkv, Hkv))
    slots = torch.full((T,), -1, dtype=torch.int32, device="cuda")

    def step():
        ops.int4_kvwrite(k, v, kc, vc, slots)
        return ops.paged_attention(q, kc, vc, view, ctx, 0.1)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lengths in ([(33, 200), (33, 400)], [(1, 7), (65, 400)], [(64, 399), (2, 2)], [(66, 66), (0, 0)], [(5, 100), (30, 30)]):
        ctx.cu_q.copy_(torch.tensor([0, lengths[0][0], lengths[0][0] + lengths[1][0]], dtype=torch.int32))
        ctx.kv_lens.copy_(torch.tensor([m for _, m in lengths], dtype=torch.int32))
        at = [view.block_table[b, j // page].item() * page + j % page for b, (n, m) in enumerate(lengths) for j in range(m - n, m)]
        slots.fill_(-1)
        slots[:len(at)] = torch.tensor(at, dtype=torch.int32)
        out.fill_(-7)
        graph.replay()
        replayed = out.clone()
        dense = [[values(c).transpose(1, 2)[view.block_table[b].long()].flatten(0, 1)[:m] for b, (_, m) in enumerate(lengths)] for c in (kc, vc)]
        want, top, span = attention(q[:len(at)], lengths, dense[0], dense[1], 0.1)
        assert ((replayed[:len(at)].double() - want).abs() <= allowed(torch.bfloat16, want, top, span, D, 400)).all(), lengths
        assert torch.equal(step()[:len(at)], replayed[:len(at)])


def test_calls_on_two_streams_at_once():
    """Products and attention of two streams side by side give what they give alone, bit by bit."""
    from tinyserve_b200.kernels import ops
    rows = rows_of(4096, 2048)
    xs = [torch.randn(m, 2048, generator=torch.Generator().manual_seed(m)).bfloat16().cuda() for m in (3, 40, 700)]
    cases = [batch(lengths, 2, 128, 16, torch.bfloat16, seed=i) for i, lengths in enumerate(([(1, 9000), (1, 50)], [(70, 700)], [(1, 30)] * 9))]
    qs = [torch.randn(c[0].num_tokens, 8, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i, c in enumerate(cases)]

    def run():
        return [ops.linear(x, rows) for x in xs] + [ops.paged_attention(q, c[2], c[3], c[1], c[0], 0.1) for q, c in zip(qs, cases)]

    alone = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for results in got:
        assert all(torch.equal(a, b) for a, b in zip(results, alone))


def test_a_captured_product_serves_other_inputs():
    from tinyserve_b200.kernels import ops
    rows, bias = rows_of(515, 1040), torch.randn(515, device="cuda")
    for M in (1, 20, 130):
        x = torch.randn(M, 1040, device="cuda").bfloat16()
        ops.linear(x, rows, bias)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear(x, rows, bias)
        for seed in range(3):
            x.copy_(torch.randn(M, 1040, generator=torch.Generator().manual_seed(seed)).bfloat16())
            if seed == 2:
                x[M // 2] = math.nan
            graph.replay()
            assert torch.equal(out.nan_to_num(7.0), ops.linear(x, rows, bias).nan_to_num(7.0))


@pytest.mark.parametrize("B,Hkv,D,page,window", [(40, 8, 64, 16, 0), (100, 8, 32, 4, 0), (100, 8, 128, 16, 40), (190, 4, 64, 8, 0), (257, 3, 64, 16, 0), (300, 1, 128, 32, 0), (33, 9, 96, 64, 0)])
def test_attention_of_many_requests(B, Hkv, D, page, window):
    """More blocks than run at once: long requests first, blocks of four warps; two of equal length, one without keys, padding rows behind the last."""
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(B)
    lengths = [(1, int(m)) for m in torch.randint(1, 400, (B,), generator=g)]
    lengths[3], lengths[7], lengths[B // 2] = (1, 900), (1, 900), (0, 12)
    ctx, view, kc, vc, ks, vs = batch(lengths, Hkv, D, page, torch.bfloat16)
    q = torch.randn(B + 5, 2 * Hkv, D, generator=g).bfloat16().cuda()
    out = ops.paged_attention(q, kc, vc, view, ctx, 0.1, window)[:B - 1]
    want, top, span = attention(q[:B - 1], lengths, ks, vs, 0.1, window)
    assert ((out.double() - want).abs() <= allowed(torch.bfloat16, want, top, span, D, 900)).all()
    assert ops.int4_attention_error(D) == 0 and ops.int4_attention_error(48) == 0


def test_products_that_follow_a_product():
    """Int8Rows as the weight of a gated, an activated and a joint product: the plain product, then what follows it."""
    from tinyserve_b200.kernels import ops
    for M in (1, 40, 300):
        x = torch.randn(M, 512, generator=torch.Generator().manual_seed(M)).bfloat16().cuda()
        rows, other = rows_of(768, 512), rows_of(256, 512, 1)
        y = ops.linear(x, rows)
        assert torch.equal(ops.gated_linear(x, rows), ops.gated_activation(y, "silu"))
        assert torch.equal(ops.activated_linear(x, rows, "gelu_tanh" if "gelu_tanh" in ops.PLAIN_ACTIVATIONS else sorted(ops.PLAIN_ACTIVATIONS)[0]),
                           ops.plain_activation_(y.clone(), "gelu_tanh" if "gelu_tanh" in ops.PLAIN_ACTIVATIONS else sorted(ops.PLAIN_ACTIVATIONS)[0]))
        # rows of one row, of none, and a row read again and again
        assert torch.equal(ops.linear(x[:1].expand(3, -1), other), ops.linear(x[:1], other).expand(3, -1))
        assert ops.linear(x[:0], other).shape == (0, 256) and ops.quantize_rows(x[:0]).codes.shape == (0, 512)


@pytest.mark.parametrize("D", [64, 128, 160, 256])
@pytest.mark.parametrize("lengths", [[(1, 3000), (1, 70)], [(200, 700)], [(4, 1500), (1, 20), (90, 300)]])
def test_attention_is_as_exact_as_its_rounding(D, lengths):
    """bfloat16: inside, everything is rounded to 11 bits or more, an eighth of the result's half step.  Roots of sums of squares:
    eight such roundings a term make 1.06 of what rounding the exact result makes."""
    from tinyserve_b200.kernels import ops
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, D, 16, torch.bfloat16)
    q = torch.randn(ctx.num_tokens, 8, D, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    want, _, _ = attention(q, lengths, ks, vs, D ** -0.5)
    rounding = (want.bfloat16().double() - want).norm()
    for splits in (None, 1, 9):
        assert (ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, num_splits=splits).double() - want).norm() <= 1.06 * rounding


def test_what_no_query_sees_does_not_matter():
    """Slots behind a request's last token, in its last page, hold enormous scales, infinities and NaN."""
    from tinyserve_b200.kernels import ops
    lengths = [(1, 37), (1, 300), (70, 90), (3, 200)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, 128, 64, torch.bfloat16)
    q = torch.randn(ctx.num_tokens, 8, 128, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    clean = [ops.paged_attention(q, kc, vc, view, ctx, 0.1, window, num_splits=sp) for window in (0, 50) for sp in (None, 3)]
    for bad in (3e38, math.inf, -math.inf, 1e-38):
        for b, (_, m) in enumerate(lengths):
            page = int(view.block_table[b, (m - 1) // 64])
            for c in (kc, vc):
                c.pairs[page, :, (m - 1) % 64 + 1:] = bad
                c.codes[page, :, (m - 1) % 64 + 1:] = 0x77
        again = [ops.paged_attention(q, kc, vc, view, ctx, 0.1, window, num_splits=sp) for window in (0, 50) for sp in (None, 3)]
        assert all(torch.equal(a, b) for a, b in zip(clean, again)), bad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("D,first", [(128, 1), (64, 3), (96, 8), (512, 5)])
def test_write_and_attention_of_rows_that_begin_anywhere(dtype, T, D, first):
    """Heads that begin on any element and lie any number of elements apart: what their contiguous copies give, bit by bit."""
    from tinyserve_b200.kernels import ops
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(T, 2, D + 11, generator=g).to(dtype).cuda()[:, :, first:first + D] for _ in range(2))
    q = torch.randn(T, 4, D + 13, generator=g).to(dtype).cuda()[:, :, first:first + D]
    slots = torch.randperm(320, generator=g)[:T].int().cuda()
    caches = [[empty_cache(20, 2, 16, D) for _ in range(2)] for _ in range(2)]
    ops.int4_kvwrite(k, v, *caches[0], slots)
    ops.int4_kvwrite(k.contiguous(), v.contiguous(), *caches[1], slots)
    for a, b in zip(*caches):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.pairs.view(torch.int16), b.pairs.view(torch.int16))
    ctx, view, kc, vc, _, _ = batch([(T, T + 40)], 2, D, 16, dtype)
    # (the kernel for long portions takes rows that begin on 16 bytes only: one kernel for both sides here, the usual choice below)
    one = "mma" if dtype == torch.bfloat16 and D in (64, 128) else None
    assert torch.equal(ops.paged_attention(q, kc, vc, view, ctx, 0.1, backend=one), ops.paged_attention(q.contiguous(), kc, vc, view, ctx, 0.1, backend=one))
    want = ops.paged_attention(q.contiguous(), kc, vc, view, ctx, 0.1).double()
    assert (ops.paged_attention(q, kc, vc, view, ctx, 0.1).double() - want).norm() <= (2.0 ** -7 if dtype == torch.bfloat16 else 0.0) * want.norm()
