"""The engine in fewer bits where its tiny models do not reach: heads of 64 and 128 (the kernel for long portions beside the one for short requests),
every attention call of mixed steps checked on its own inputs, steps replayed from graphs; and 8-bit weights in every architecture."""
import importlib
import os

import numpy as np
import pytest
import torch

import plain_fewer_bits as fewer
import plain_qwen3 as plain
from helpers import collect_logits, lines_of, max_live_tokens, random_ids, schedule_mixed, schedule_portions, schedule_tail_decode
from int4_cases import exact_enough, of_requests
from test_fewer_bits_engine_gpu import NOISE, distance
from test_fewer_bits_gpu import attention, values

pytestmark = pytest.mark.gpu

WIDE = {
    # heads of 64, four on a key head, a window on the upper layers
    "S": dict(hidden_size=128, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2, head_dim=64, intermediate_size=256, vocab_size=300,
              rms_norm_eps=1e-6, rope_theta=1e5, tie_word_embeddings=False, max_position_embeddings=1024, use_sliding_window=True, sliding_window=70, max_window_layers=1),
    # heads of 128, all on one key head
    "T": dict(hidden_size=160, num_hidden_layers=2, num_attention_heads=6, num_key_value_heads=1, head_dim=128, intermediate_size=320, vocab_size=257,
              rms_norm_eps=1e-5, rope_theta=1e6, tie_word_embeddings=True, max_position_embeddings=1024),
}
LENGTHS = (300, 150, 40, 7)
PORTIONS = (70, 2, 129, 33, 1, 6)


@pytest.fixture(scope="module", params=sorted(WIDE))
def model(request, tmp_path_factory):
    from tinyserve_b200.config import config_from_dict
    from tinyserve_b200.weights import write_random_model
    config = config_from_dict(dict(WIDE[request.param], architectures=["Qwen3ForCausalLM"], model_type="qwen3"))
    folder = write_random_model(config, str(tmp_path_factory.mktemp(f"wide{request.param}")), seed=22, store_dtype="bfloat16")
    cfg, weights = plain.load_folder(folder)
    return {"folder": folder, "cfg": cfg, "weights": weights, "requests": {f"r{i}": random_ids(cfg["vocab_size"], n, seed=200 + i) for i, n in enumerate(LENGTHS)}}


def logits_of(runner, steps, out_dir, vocab):
    from tinyserve_b200.engine import replay
    replay.replay(runner, lines_of(steps), str(out_dir), lambda _: None)
    outputs = {}
    for s in steps:
        wanted = sum(len(e["want"]) for e in s["entries"])
        if wanted:
            outputs[s["step"]] = torch.from_numpy(np.fromfile(os.path.join(str(out_dir), f"{s['step']}.f32"), dtype="<f4").reshape(wanted, vocab))
    return collect_logits(steps, outputs, vocab)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [16, 64])
def test_every_attention_of_mixed_steps(model, dtype, page, tmp_path, monkeypatch):
    """What each call gives, of the cache and the batch that it met, against the definition: portions and single tokens side by side, pages that
    are used again, layer behind layer."""
    from tinyserve_b200.engine import replay
    from tinyserve_b200.kernels import ops
    real, entries = ops.paged_attention, ops._entry
    seen, used = [], set()

    def checked(q, k_cache, v_cache, view, ctx, scale, window=0, **kw):
        out = real(q, k_cache, v_cache, view, ctx, scale, window, **kw)
        cu, kv = ctx.cu_q.tolist(), ctx.kv_lens.tolist()
        lengths = [(cu[b + 1] - cu[b], kv[b]) for b in range(ctx.num_requests)]
        dense = []
        for cache in (k_cache, v_cache):
            rows = []
            for b, (_, m) in enumerate(lengths):
                first = max(0, m - window - lengths[b][0]) // view.page_size if window else 0          # (pages before the window are given back)
                table = view.block_table[b, first:-(-m // view.page_size)].long()
                part = ops.Int4Pages(cache.codes[table], cache.pairs[table])
                x = values(part).transpose(1, 2).flatten(0, 1)
                rows.append(torch.cat([torch.zeros(first * view.page_size, *x.shape[1:], dtype=x.dtype, device=x.device), x])[:m])
            dense.append(rows)
        want, _, _ = attention(q, lengths, *dense, scale, window)
        for rows, (n, m) in zip(of_requests(lengths), [x for x in lengths if x[0] and x[1]]):
            assert exact_enough(out[rows], want[rows], q.dtype), (lengths, window, n, m)
        seen.append((max(n for n, _ in lengths), min(n for n, _ in lengths), len(lengths)))
        return out

    monkeypatch.setattr(ops, "paged_attention", checked)
    monkeypatch.setattr(ops, "_entry", lambda unit, name: (used.add(name), entries(unit, name))[1])
    reqs = {**model["requests"], **{f"{rid}x": ids for rid, ids in model["requests"].items()}}
    steps = schedule_mixed(reqs, max_live=4, seed=3, chunk_sizes=PORTIONS)
    runner = replay.make_runner(model["folder"], dtype, max_live_tokens(steps), block_size=page, weight_dtype="int8", kv_cache_dtype="int4")
    logits_of(runner, steps, tmp_path, model["cfg"]["vocab_size"])
    assert len(seen) == model["cfg"]["num_hidden_layers"] * len(steps) and any(a > 16 and b == 1 for a, b, _ in seen)
    assert dtype == "float32" or used >= {"ts_int4_attention", "ts_int4_attention_tcgen05"}


@pytest.mark.parametrize("mode", ["int4", "both"])
def test_steps_replayed_from_graphs(model, mode, tmp_path):
    """The same mixed schedule three times over one engine: the first runs the steps as they are, later ones replay what was captured, over pages and
    buffers that were used in between."""
    from tinyserve_b200.engine import replay
    cfg, weights, reqs = model["cfg"], model["weights"], model["requests"]
    w8 = mode == "both"
    steps = schedule_mixed(reqs, max_live=4, seed=4, chunk_sizes=PORTIONS)
    ref = {rid: fewer.logits(cfg, weights, ids, w8, True) for rid, ids in reqs.items()}
    moved = max(distance({rid: fewer.logits(cfg, weights, ids, w8, True, NOISE["bfloat16"], seed) for rid, ids in reqs.items()}, ref) for seed in range(3))
    allowed = 2 * moved + 2.0 ** -7 * distance(ref, {r: 0 * x for r, x in ref.items()})
    runner = replay.make_runner(model["folder"], "bfloat16", max_live_tokens(steps), use_cuda_graphs=True, weight_dtype="int8" if w8 else "auto", kv_cache_dtype="int4")
    replays = []
    for turn in range(3):
        off = distance(logits_of(runner, steps, tmp_path / str(turn), cfg["vocab_size"]), ref)
        print(f"{mode} turn {turn}: {off:.2e} of {allowed:.2e}, {runner.mixed_graph_replays} replays")
        assert off <= allowed
        replays.append(runner.mixed_graph_replays)
    assert replays[-1] > replays[0]


# ------------------------------------------------------------------------------------------------- 8-bit weights in every architecture
ARCHITECTURES = ["babadra", "delilorn", "dudatar", "gunulorn", "ronolorn", "tarivik"]


def plain_int8(x, weight, bias, out_float32, constant_weight):
    """``ops._linear_int8`` in torch operations: the same roundings, the sums in 64 bits."""
    from tinyserve_b200.kernels import ops
    if isinstance(x, ops.Int8Rows):
        codes, scale, dtype = x.codes.double(), x.scales, torch.bfloat16
    else:
        x = ops.materialize(x)
        dtype, x = x.dtype, x.float()
        scale = x.abs().amax(1) / torch.full_like(x[:, 0], 127)
        codes = torch.where(scale[:, None] > 0, (x / scale[:, None]).round(), 0).double()
    y = (codes @ weight.codes.double().T).float() * (scale[:, None] * weight.scales[None])
    if bias is not None:
        y = ((codes @ weight.codes.double().T).float().double() * (scale[:, None] * weight.scales[None]).double() + bias.double()).float()          # (one rounding: a fused multiply-add)
    return y if out_float32 else y.to(dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", ["first", "second", "third"])
@pytest.mark.parametrize("name", ARCHITECTURES)
def test_8_bit_weights_in_every_architecture(name, size, dtype, tmp_path, monkeypatch):
    """A model's logits with 8-bit weights are, bit by bit, what they are with each of its products over them made of torch operations."""
    from tinyserve_b200.engine import replay
    from tinyserve_b200.kernels import ops
    from tinyserve_b200.weights import write_random_model
    module = importlib.import_module(f"{name}_configs")
    which = sorted(getattr(module, f"{name.upper()}_TINY"))[["first", "second", "third"].index(size)]
    folder = write_random_model(getattr(module, f"{name}_config")(which), str(tmp_path / "model"), seed=5, store_dtype="bfloat16")
    real, calls = ops._linear_int8, []
    got = []
    for kernel in (real, plain_int8):
        monkeypatch.setattr(ops, "_linear_int8", lambda *args, kernel=kernel: (calls.append(kernel), kernel(*args))[1])
        reqs, runner, out = None, None, []
        for k, schedule in enumerate((schedule_portions, lambda r: schedule_tail_decode(r, 12), lambda r: schedule_mixed(r, max_live=3, seed=2))):
            if runner is None:
                runner = replay.make_runner(folder, dtype, 512, max_live=4, weight_dtype="int8")
                reqs = {f"r{i}": random_ids(runner.model.vocab_size, n, seed=i) for i, n in enumerate((40, 23, 70))}
            out.append(logits_of(runner, schedule(reqs), tmp_path / f"{kernel.__name__}{k}", runner.model.vocab_size))
        got.append(out)
    assert calls.count(real) == calls.count(plain_int8) > 0
    for a, b in zip(*got):
        for rid in a:
            assert a[rid].isfinite().all() and torch.equal(a[rid], b[rid]), rid
