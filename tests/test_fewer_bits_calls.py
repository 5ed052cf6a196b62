"""What the entry points over a 4-bit cache hand to their kernels, recorded without a device."""
from types import SimpleNamespace as NS

import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    """[(entry point, its fields)] of what would have been launched."""
    from tinyserve_b200.kernels import ops
    seen = []
    entry = lambda unit, name: (None, lambda *args: seen.append((name, args)))
    monkeypatch.setattr(ops, "_entry", entry)
    monkeypatch.setattr(ops, "_here", lambda what, *tensors: 0)
    monkeypatch.setattr(ops, "_launched", lambda lib, code, n: None)
    return seen


def attend(lengths, H=4, Hkv=2, D=64, page=16, dtype=torch.bfloat16, blocks=None, **kw):
    from tinyserve_b200.kernels import ops
    B, cu = len(lengths), [0]
    for n, _ in lengths:
        cu.append(cu[-1] + n)
    blocks = blocks or max(-(-m // page) for _, m in lengths)
    ctx = NS(num_requests=B, cu_q=torch.tensor(cu, dtype=torch.int32), kv_lens=torch.tensor([m for _, m in lengths], dtype=torch.int32),
             max_q_len=max(n for n, _ in lengths), max_kv_len=max(m for _, m in lengths))
    view = NS(page_size=page, block_table=torch.zeros(B, blocks, dtype=torch.int32))
    caches = [ops.Int4Pages(torch.zeros(2, Hkv, page, D // 2, dtype=torch.uint8), torch.zeros(2, Hkv, page, 2, dtype=torch.bfloat16)) for _ in range(2)]
    return ops.paged_attention(torch.zeros(cu[-1], H, D, dtype=dtype), *caches, view, ctx, 0.1, **kw)


def test_the_device_is_asked_for_its_multiprocessors(calls, monkeypatch):
    """Whether requests are taken by length depends on how many blocks run at once."""
    from tinyserve_b200.kernels import ops
    for sms in (148, 60):
        monkeypatch.setattr(ops, "num_sms", lambda: sms)
        attend([(1, 30)] * 40)
        name, fields = calls.pop()
        assert name == "ts_int4_attention" and fields[-2] == sms
        ops.struct.pack("=" + ops._INT4_ENTRIES[name], *fields)          # (as many as the entry point takes)
    with open(f"{ops.build.CSRC}/attention_int4.cu") as fh:
        assert "148" not in fh.read().split("int attend_mma(")[1].split("\n}")[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[(1, 30), (1, 5)], [(70, 70), (3, 0)]])
def test_a_window_longer_than_the_table_is_none(calls, dtype, lengths):
    """Kernels take a window as a 32-bit integer and subtract it from positions: 2^32 + 5 would be 5, and 2^31 - 1 wraps behind a
    position below zero (a row of a request with fewer keys than queries)."""
    table = 16 * max(-(-m // 16) for _, m in lengths)
    for window, want in ((0, 0), (5, 5), (table - 1, table - 1), (table, 0), (2 ** 31 - 1, 0), (2 ** 31, 0), (2 ** 32 + 5, 0), (2 ** 70, 0)):
        attend(lengths, dtype=dtype, window=window)
        assert calls and all(fields[{"ts_int4_attention": 21, "ts_int4_attention_tcgen05": 20}[name]] == want for name, fields in calls), window
        calls.clear()
