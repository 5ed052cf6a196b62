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
