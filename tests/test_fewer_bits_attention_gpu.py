"""Attention over a 4-bit cache, request by request, to within what rounding the exact result makes: windows, sinks and soft caps over long
contexts, where a key more or less is a small part of a result (test_fewer_bits_criterion.py shows that it does not pass)."""
import pytest
import torch

from int4_cases import LENGTHS, OPTIONS, exact_enough, of_requests, queries, requests
from test_fewer_bits_gpu import attention

pytestmark = pytest.mark.gpu

SHAPES = [(4, 4, 16, 8), (8, 2, 128, 64), (14, 2, 64, 16), (3, 3, 96, 1), (20, 1, 256, 32), (2, 1, 512, 16), (9, 1, 32, 64), (32, 8, 128, 16), (5, 1, 160, 64), (8, 8, 64, 4),
          (6, 2, 48, 16), (2, 1, 224, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D,page", SHAPES)
@pytest.mark.parametrize("name", sorted(LENGTHS))
def test_attention_to_its_rounding(dtype, H, Hkv, D, page, name):
    from tinyserve_b200.kernels import ops
    lengths = LENGTHS[name]
    ctx, view, kc, vc, ks, vs = requests(lengths, Hkv, D, page, "cuda")
    q, sinks = queries(ctx.num_tokens, H, D, "cuda")
    q, scale = q.to(dtype), D ** -0.5
    chosen = ops.int4_attention_backend(dtype, D)
    for window, softcap, sunk in OPTIONS:
        sink = sinks if sunk else None
        want, _, _ = attention(q, lengths, ks, vs, scale, window, softcap, sink)
        for backend in [chosen] + (["mma"] if chosen == "tcgen05" else []) + (["simt"] if chosen != "simt" else []):
            for splits in (None, 1, 3, 8, 12):
                attend = lambda: ops.paged_attention(q, kc, vc, view, ctx, scale, window, sinks=sink, softcap=softcap, num_splits=splits, backend=backend)
                out = attend()
                for rows, (n, m) in zip(of_requests(lengths), [x for x in lengths if x[0] and x[1]]):
                    assert exact_enough(out[rows], want[rows], dtype), (window, softcap, sunk, backend, splits, n, m)
                assert splits is not None or torch.equal(attend(), out), "the same call twice"
    if chosen != "simt":
        assert ops.int4_attention_error(D) == 0
