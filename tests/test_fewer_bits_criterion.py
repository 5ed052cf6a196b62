"""The criterion that results over a 4-bit cache are held to rejects the mistakes that a kernel could make, rounded as a kernel would."""
import pytest
import torch

from int4_cases import LENGTHS, OPTIONS, exact_enough, of_requests, queries, requests
from test_fewer_bits_gpu import attention

H, HKV, D = 8, 2, 128


def without(rows, first, n):
    """The rows of a request without n of them from ``first`` on."""
    return torch.cat([rows[:first], rows[first + n:]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", sorted(set(LENGTHS) - {"wide"}))
def test_mistakes_do_not_pass(name, dtype):
    lengths = LENGTHS[name]
    ctx, _, _, _, ks, vs = requests(lengths, HKV, D, 16, "cpu")
    q, sinks = queries(ctx.num_tokens, H, D, "cpu")
    scale = D ** -0.5

    def rejected(wrong, want, applies):
        for (n, m), rows in zip([x for x in lengths if x[0] and x[1]], of_requests(lengths)):
            assert exact_enough(want[rows].to(dtype), want[rows], dtype)
            if applies(n, m):
                assert not exact_enough(wrong[rows].to(dtype), want[rows], dtype), (n, m)

    for window, softcap, sunk in OPTIONS:
        sink = sinks if sunk else None
        attend = lambda w=window, c=softcap, s=sink, k=ks, v=vs, ls=lengths: attention(q, ls, k, v, scale, w, c, s)[0]
        want = attend()
        if window > 1:
            for w in (window - 1, window + 1):
                rejected(attend(w=w), want, lambda n, m: m > window)
        if sunk:
            rejected(attend(s=None), want, lambda n, m: True)
        if softcap and window != 1:
            rejected(attend(c=0.0), want, lambda n, m: m > 1)
        if not window:
            # a step of 32 keys that was left out, at the start, in the middle and short of the end
            for where in (lambda m: 0, lambda m: m // 2, lambda m: m - 33):
                short = [(n, m - 32) if m > 65 and n == 1 else (n, m) for n, m in lengths]
                cut = lambda xs: [without(x, where(m), 32) if m > 65 and n == 1 else x for x, (n, m) in zip(xs, lengths)]
                rejected(attend(k=cut(ks), v=cut(vs), ls=short), want, lambda n, m: m > 65 and n == 1)
            # a key too many, a key too few
            for by in (-1, 1):
                moved = [(n, m + by) if m > n and n else (n, m) for n, m in lengths]
                more = lambda xs: [torch.cat([x, x[:1] * -1]) if by > 0 and m > n and n else x[:m + by] if m > n and n else x for x, (n, m) in zip(xs, lengths)]
                rejected(attend(k=more(ks), v=more(vs), ls=moved), want, lambda n, m: m > n)
