"""Attention over a 4-bit cache where a loose bound would hide a mistake: how far it is from the definition in 64 bits, measured against what
rounding the exact result makes."""
import math

import pytest
import torch

from test_fewer_bits_gpu import attention, batch, values

pytestmark = pytest.mark.gpu


def queries(T, H, D, dtype=torch.bfloat16, seed=3):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# bfloat16: inside, everything is rounded to 11 bits or more, an eighth of the result's half step; roots of sums of squares: eight
# such roundings a term make 1.06 of what rounding the exact result makes
AS_EXACT_AS_ITS_ROUNDING = 1.06


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [1e7, 1e5, 30.0, 2.0, 0.3])
def test_a_soft_cap_keeps_scores_far_below_it(D, softcap):
    """Portions whose scores are small, near and far above the cap."""
    from tinyserve_b200.kernels import ops
    lengths = [(200, 700), (64, 64)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, D, 16, torch.bfloat16)
    q = queries(ctx.num_tokens, 8, D)
    for window in (0, 50):
        want, _, _ = attention(q, lengths, ks, vs, D ** -0.5, window, softcap)
        rounding = (want.bfloat16().double() - want).norm()
        for backend in ("tcgen05", "mma", "simt"):
            out = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, window, softcap=softcap, backend=backend)
            assert (out.double() - want).norm() <= AS_EXACT_AS_ITS_ROUNDING * rounding, backend


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [48, 64, 128])
def test_a_sink_of_minus_infinity_is_none(dtype, D):
    """exp(-infinity) adds nothing to a head's sum; a row without keys stays zero."""
    from tinyserve_b200.kernels import ops
    lengths = [(70, 60), (40, 300), (1, 0), (1, 9)]
    ctx, view, kc, vc, ks, vs = batch(lengths, 2, D, 16, dtype)
    q = queries(ctx.num_tokens, 8, D, dtype)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(1)).cuda()
    some = torch.where(torch.arange(8, device="cuda") % 3 == 0, -math.inf, sinks)
    chosen = ops.int4_attention_backend(dtype, D)
    for backend in {chosen, "simt"} | ({"mma"} if chosen == "tcgen05" else set()):
        for splits in (1, 3, None):
            attend = lambda s: ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, sinks=s, num_splits=splits, backend=backend)
            without, with_sinks, got = attend(None), attend(sinks), attend(some)
            assert not without[:10].any() and not without[110].any()
            # (none of these heads' sums holds another term: the same operations, but for a factor of 1)
            none = some.isinf()
            assert torch.equal(got[:, none], without[:, none]) and torch.equal(got[:, ~none], with_sinks[:, ~none]), (backend, splits)


def dense(ctx, view, cache):
    """What the cached rows of every request stand for, in 64 bits."""
    x = values(cache).transpose(1, 2).flatten(0, 1)
    kv, page = ctx.kv_lens.tolist(), view.page_size
    at = [view.block_table[b].long()[torch.arange(m) // page] * page + (torch.arange(m) % page).cuda() for b, m in enumerate(kv)]
    return [x[a] for a in at]


def scale_row(view, cache, b, j, by):
    """Key j of request b times a power of two."""
    page = int(view.block_table[b, j // view.page_size])
    cache.pairs[page, :, j % view.page_size] = (cache.pairs[page, :, j % view.page_size].double() * by).bfloat16()


# how much larger than the other values (and keys) a row may be: below and above what half precision holds beside them
LARGER = {backend: (2.0 ** 12, 2.0 ** 20, 2.0 ** 23, 2.0 ** 25, 2.0 ** 40, 2.0 ** 90) for backend in ("mma", "simt", "tcgen05")}


@pytest.mark.parametrize("backend", sorted(LARGER))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[(1, 1000), (3, 300), (1, 40)], [(1, 9000)] * 2, [(40, 700), (2, 64)]])
@pytest.mark.parametrize("where", [0, 37, -1])
def test_a_huge_value_of_no_weight(backend, D, lengths, where):
    """A key that every query gives a probability of nothing, with values far larger than the others': the others keep their bits."""
    from tinyserve_b200.kernels import ops
    ctx, view, kc, vc, _, _ = batch(lengths, 2, D, 16, torch.bfloat16)
    q = queries(ctx.num_tokens, 8, D).abs()
    for b, (n, m) in enumerate(lengths):
        j = where % m
        page = int(view.block_table[b, j // 16])
        kc.codes[page, :, j % 16] = 0
        kc.pairs[page, :, j % 16] = torch.tensor([0.0, -16.0], dtype=torch.bfloat16, device="cuda")          # scores of -16 sum |q| / sqrt(D): below -70
    for by in LARGER[backend]:
        pairs = vc.pairs.clone()
        for b, (n, m) in enumerate(lengths):
            scale_row(view, vc, b, where % m, by)
        ks, vs = dense(ctx, view, kc), dense(ctx, view, vc)
        want, _, _ = attention(q, lengths, ks, vs, D ** -0.5)
        out = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, backend=backend)
        vc.pairs.copy_(pairs)
        at = 0
        for n, m in lengths:
            rows = slice(at, at + n)
            at += n
            rounding = (want[rows].bfloat16().double() - want[rows]).norm()
            assert (out[rows].double() - want[rows]).norm() <= AS_EXACT_AS_ITS_ROUNDING * rounding, (by, n, m)


@pytest.mark.parametrize("backend", sorted(LARGER))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[(3, 300), (2, 33)], [(40, 700), (4, 40)], [(130, 200)]])
@pytest.mark.parametrize("window", [0, 7])
def test_a_huge_key_that_only_later_queries_see(backend, D, lengths, window):
    """The last key of every request, and its value, are far larger than the others: the queries before it give what they gave."""
    from tinyserve_b200.kernels import ops
    ctx, view, kc, vc, _, _ = batch(lengths, 2, D, 16, torch.bfloat16)
    q = queries(ctx.num_tokens, 8, D)
    attend = lambda: ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, window, backend=backend)
    earlier = torch.cat([torch.arange(n) < n - 1 for n, _ in lengths]).cuda()
    clean = attend()[earlier]
    want, _, _ = attention(q, lengths, dense(ctx, view, kc), dense(ctx, view, vc), D ** -0.5, window)
    want = want[earlier]
    rounding = (want.bfloat16().double() - want).norm()
    assert (clean.double() - want).norm() <= AS_EXACT_AS_ITS_ROUNDING * rounding
    for by in LARGER[backend]:
        pairs = kc.pairs.clone(), vc.pairs.clone()
        for b, (_, m) in enumerate(lengths):
            scale_row(view, kc, b, m - 1, by)
            scale_row(view, vc, b, m - 1, by)
        out = attend()[earlier]
        kc.pairs.copy_(pairs[0])
        vc.pairs.copy_(pairs[1])
        assert (out.double() - want).norm() <= AS_EXACT_AS_ITS_ROUNDING * rounding, by


@pytest.mark.parametrize("D,H,Hkv", [(64, 14, 2), (128, 8, 2), (128, 3, 3), (64, 130, 1)])
@pytest.mark.parametrize("lengths", [[(200, 700), (64, 64), (1, 90)], [(130, 100)], [(17, 3000), (40, 41)]])
def test_portions_whose_keys_and_values_are_far_apart(D, H, Hkv, lengths):
    """Values from 2^-40 to 2^40 of what they were, and some keys at 2^-30: with windows, sinks and soft caps, rows without keys, NaN that some rows see."""
    from tinyserve_b200.kernels import ops
    ctx, view, kc, vc, _, _ = batch(lengths, Hkv, D, 16, torch.bfloat16)
    g = torch.Generator().manual_seed(D)
    by = torch.randint(-40, 41, vc.pairs.shape[:3], generator=g).cuda()
    vc.pairs.copy_(torch.ldexp(vc.pairs.float(), by[..., None]).bfloat16())
    kc.pairs.copy_(torch.ldexp(kc.pairs.float(), torch.where(by % 7 == 0, -30, 0)[..., None]).bfloat16())
    q = queries(ctx.num_tokens, H, D)
    sinks = torch.randn(H, generator=g).cuda()
    for window, softcap, sink in ((0, 0.0, None), (50, 0.0, sinks), (0, 2.0, None), (7, 1e5, sinks)):
        want, _, _ = attention(q, lengths, dense(ctx, view, kc), dense(ctx, view, vc), D ** -0.5, window, softcap, sink)
        out = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5, window, softcap=softcap, sinks=sink)
        # (32 bits inside: every element is off by its rounding, and by the sums' share of the largest term)
        rounding = (want.bfloat16().double() - want).norm(dim=(1, 2))
        assert ((out.double() - want).norm(dim=(1, 2)) <= AS_EXACT_AS_ITS_ROUNDING * rounding + 2.0 ** -16 * want.norm(dim=(1, 2))).all(), (window, softcap)
    clean = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5)
    n, m = lengths[0]
    j = min(m, n) // 2 + max(m - n, 0)                       # the queries of the first request from here on see it
    for cache in (kc, vc):
        keep = cache.pairs.clone()
        cache.pairs[int(view.block_table[0, j // 16]), :, j % 16] = math.nan
        out = ops.paged_attention(q, kc, vc, view, ctx, D ** -0.5)
        cache.pairs.copy_(keep)
        sees = torch.arange(ctx.num_tokens, device="cuda") + (m - n) >= j
        sees[n:] = False
        assert out[sees].isnan().all() and torch.equal(out[~sees], clean[~sees])
    assert ops.int4_attention_error(D) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", range(8, 30))
@pytest.mark.parametrize("step", [1, 2, 7, 8, 16])
def test_maxima_a_few_steps_of_32_bits_apart(D, power, step):
    """Scores of 1.5 2^power in the first tile of keys, a few powers of two above them in the next: whatever 32 bits make of the difference, all
    values are the same, and so is the result."""
    from tinyserve_b200.kernels import ops
    n, m, page = 32, 256, 16
    ctx, view, kc, vc, _, _ = batch([(n, m)], 1, D, page, torch.bfloat16)
    for cache, values_of in ((kc, None), (vc, 3.0)):
        cache.codes.zero_()
        cache.pairs[..., 0], cache.pairs[..., 1] = 1.0, values_of or 0.0
    for j in range(m):
        word = 1 | j // 128 << 16          # column 0: 1; column 1: 0 in the first tile, 1 in the second
        kc.codes[int(view.block_table[0, j // page]), 0, j % page, :4] = torch.tensor([word & 255, 0, word >> 16, 0], dtype=torch.uint8)
    q = torch.zeros(n, 4, D, device="cuda", dtype=torch.bfloat16)
    q[..., 0], q[..., 1] = 1.5 * 2.0 ** power, step
    for backend in ("tcgen05", "mma", "simt"):
        out = ops.paged_attention(q, kc, vc, view, ctx, math.log(2.0), backend=backend)
        assert (out.float() - 3.0).abs().max() <= 3.0 * 2.0 ** -8, backend


@pytest.mark.parametrize("backend", sorted(LARGER))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e5, 1e6, 1e8, 1e10, 1e20])
@pytest.mark.parametrize("spread", [3, 20])
def test_scores_of_any_size(backend, D, size, spread):
    """Scores so large that one key has all of the weight, whose values may be far smaller or larger than the others': a row is that key's values.
    (Rows whose two best scores are within 2^-10 of the largest are left out: 32 bits may take either.)"""
    from tinyserve_b200.kernels import ops
    lengths = [(1, 900), (3, 300), (70, 200)]
    ctx, view, kc, vc, _, _ = batch(lengths, 2, D, 16, torch.bfloat16)
    by = torch.randint(-spread, spread + 1, vc.pairs.shape[:3], generator=torch.Generator().manual_seed(D)).cuda()
    vc.pairs.copy_(torch.ldexp(vc.pairs.float(), by[..., None]).bfloat16())
    q = queries(ctx.num_tokens, 8, D)
    scale, ks, vs = D ** -0.5 * size, dense(ctx, view, kc), dense(ctx, view, vc)
    out, at, checked = ops.paged_attention(q, kc, vc, view, ctx, scale, backend=backend).double(), 0, 0
    for (n, m), k, v in zip(lengths, ks, vs):
        scores = torch.einsum("thd,jhd->thj", q[at:at + n].double(), k.repeat_interleave(4, 1)) * scale
        scores = scores.masked_fill(torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None, None], -math.inf)
        best = scores.topk(2, -1)
        clear = (best.values[..., 0] - best.values[..., 1] > 2.0 ** -10 * scores.nan_to_num(neginf=0.0).abs().amax(-1)) & (best.values[..., 0] - best.values[..., 1] > 60)
        want = v.repeat_interleave(4, 1)[best.indices[..., 0], torch.arange(8, device="cuda")]
        # (the least of 2^41 between two values' scales has a weight of e^-60 against it)
        off = (out[at:at + n] - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * want.abs().amax(-1, keepdim=True)
        assert (off | ~clear[..., None]).all(), (n, m)
        checked += int(clear.sum())
        at += n
    assert checked > 300
