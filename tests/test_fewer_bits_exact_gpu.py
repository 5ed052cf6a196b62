"""Attention over a 4-bit cache where a loose bound would hide a mistake: how far it is from the definition in 64 bits, measured against what
rounding the exact result makes."""
import math

import pytest
import torch

from test_fewer_bits_gpu import attention, batch

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
