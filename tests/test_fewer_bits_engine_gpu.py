"""The engine with 8-bit weights, with a 4-bit cache and with both, against the plain decoder in which every value is replaced by the
one that its code stands for: whole prompts, portions, single tokens, pages that are used again, captured graphs."""
import os

import numpy as np
import pytest
import torch

import plain_fewer_bits as fewer
import plain_qwen3 as plain
from helpers import TINY, collect_logits, lines_of, make_model_dir, max_live_tokens, random_ids, schedule_mixed, schedule_portions, schedule_tail_decode, schedule_whole

pytestmark = pytest.mark.gpu

MODES = {"int8": ("int8", "auto"), "int4": ("auto", "int4"), "both": ("int8", "int4")}
LENGTHS = {"A": [5, 17, 70], "B": [1, 40, 100], "C": [90, 130, 3], "D": [33, 80, 2]}
# How far the engine's values before a code are from the plain ones, relative to themselves, generously: sums of 32-bit products, and the
# roundings to bfloat16 of the activations.  What that moves (codes next to a border, layer by layer) is measured on the plain side,
# which is shaken by as much; see plain_fewer_bits.
NOISE = {"float32": 2.0 ** -19, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module", params=sorted(TINY))
def model(request, tmp_path_factory):
    name = request.param
    folder = make_model_dir(tmp_path_factory.mktemp(f"few{name}"), name, seed=21)
    cfg, weights = plain.load_folder(folder)
    reqs = {f"r{i}": random_ids(cfg["vocab_size"], n, seed=100 + i) for i, n in enumerate(LENGTHS[name])}
    refs = {m: {rid: fewer.logits(cfg, weights, ids, w == "int8", c == "int4") for rid, ids in reqs.items()} for m, (w, c) in MODES.items()}
    moved = {}
    for m, (w, c) in MODES.items():
        for dtype, noise in NOISE.items():
            moved[m, dtype] = max(distance({rid: fewer.logits(cfg, weights, ids, w == "int8", c == "int4", noise, seed) for rid, ids in reqs.items()}, refs[m])
                                  for seed in range(3))
    return {"folder": folder, "cfg": cfg, "requests": reqs, "refs": refs, "moved": moved}


def distance(got, ref):
    """Root mean square over all logits of all requests."""
    return float(torch.cat([(got[rid].double() - ref[rid]).flatten() for rid in ref]).pow(2).mean().sqrt())


def run(model, dtype, mode, steps, out_dir, page=16, graphs=False, requests=None):
    from tinyserve_b200.engine import replay
    w, c = MODES[mode]
    runner = replay.make_runner(model["folder"], dtype, max_live_tokens(steps), block_size=page, use_cuda_graphs=graphs, weight_dtype=w, kv_cache_dtype=c)
    replay.replay(runner, lines_of(steps), str(out_dir), lambda _: None)
    vocab, outputs = model["cfg"]["vocab_size"], {}
    for s in steps:
        wanted = sum(len(e["want"]) for e in s["entries"])
        if wanted:
            outputs[s["step"]] = torch.from_numpy(np.fromfile(os.path.join(str(out_dir), f"{s['step']}.f32"), dtype="<f4").reshape(wanted, vocab))
    got = collect_logits(steps, outputs, vocab)
    ref = {rid: model["refs"][mode][rid.rstrip("x")] for rid in (requests or model["requests"])}
    off, allowed = distance(got, ref), 2 * model["moved"][mode, dtype] + {"float32": 2e-6, "bfloat16": 2.0 ** -7}[dtype] * distance(ref, {r: 0 * x for r, x in ref.items()})
    print(f"{dtype} {mode}: {off:.2e} of {allowed:.2e}")
    assert off <= allowed
    return runner


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("mode", sorted(MODES))
def test_schedules(model, dtype, mode, tmp_path):
    reqs = model["requests"]
    for name, steps in (("whole", schedule_whole(reqs)), ("tail", schedule_tail_decode(reqs, 32)), ("portions", schedule_portions(reqs))):
        run(model, dtype, mode, steps, tmp_path / name)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs,page", [(False, 8), (True, 16)])
def test_mixed_steps(model, dtype, graphs, page, tmp_path):
    reqs = {**model["requests"], **{f"{rid}x": ids for rid, ids in model["requests"].items()}}
    runner = run(model, dtype, "both", schedule_mixed(reqs, max_live=4, seed=1), tmp_path, page=page, graphs=graphs, requests=reqs)
    pages = runner.device_cache.entries[0]
    D = model["cfg"]["head_dim"]
    assert pages.tensors["k"].dtype == torch.uint8 and pages.tensors["k"].shape[-1] == D // 2
    assert runner.device_cache.bytes_per_page(runner.model, page, 2)[0] == runner.model.group_sizes[0] * 2 * model["cfg"]["num_key_value_heads"] * (D // 2 + 4) * page


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,D,rot,inter,norm", [(4, 2, 128, 128, False, True), (3, 1, 96, 64, False, True), (2, 2, 16, 16, True, False), (5, 5, 512, 0, False, True),
                                                    (6, 2, 64, 32, True, True)])
@pytest.mark.parametrize("T", [9, 300])
def test_norm_rotation_and_write_in_one(dtype, H, Hkv, D, rot, inter, norm, T):
    """The kernel that norms, turns and writes against the ones that do it to a cache of whole numbers, and then its codes."""
    from types import SimpleNamespace as NS
    from tinyserve_b200.kernels import ops
    from tinyserve_b200.parts.rotary import Rotary
    page = 8
    pages = T // page + 1
    g = torch.Generator().manual_seed(D + H)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g).to(dtype).cuda()
    positions = torch.randint(0, 900, (T,), generator=g).int().cuda()
    rotary = None
    if rot:
        cos, sin = Rotary.tables(rot, 1e4, 1000)
        rotary = NS(cos=cos.cuda(), sin=sin.cuda(), rotary_dim=rot, interleaved=inter)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)) if norm else (None, None)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    slots[3] = -1
    slots = slots.cuda()
    plain_caches = [torch.zeros(pages, Hkv, page, D, dtype=dtype, device="cuda") for _ in range(2)]
    caches = [ops.Int4Pages(torch.zeros(pages, Hkv, page, D // 2, dtype=torch.uint8, device="cuda"), torch.zeros(pages, Hkv, page, 2, dtype=torch.bfloat16, device="cuda")) for _ in range(2)]
    args = (qkv, positions, H, Hkv, D, rotary, qw, kw, 1e-6)
    q0 = ops.qk_norm_rope_kvwrite(*args, *plain_caches, slots, page)
    q1 = ops.qk_norm_rope_kvwrite(*args, *caches, slots, page)
    # sums of squares in another order and a fused multiply-add more or less: a few roundings of 32 bits, one step of bfloat16
    half = 2.0 ** -24 * (D + 8) if dtype == torch.float32 else 2.0 ** -7
    assert ((q0.double() - q1.double()).abs() <= half * (q0.double().abs() + q0.double().abs().amax(-1, keepdim=True) * (dtype == torch.float32)) + 1e-30).all()
    for whole, packed in zip(plain_caches, caches):
        w = packed.codes.view(torch.int32)
        codes = ((w[..., None] >> torch.tensor([i // 2 * 4 + i % 2 * 16 for i in range(8)], device="cuda").int()) & 15).flatten(-2).double()
        got = packed.pairs[..., 1:].double() + codes * packed.pairs[..., :1].double()
        # half a step, the pair's own rounding, and what the rows may differ by
        off = (got - whole.double()).abs()
        assert (off <= 0.5 * packed.pairs[..., :1].double() + (3 * 2.0 ** -8 + 2 * half) * whole.double().abs().amax(-1, keepdim=True) + 1e-30).all()
    written = torch.zeros(pages * page, dtype=torch.bool)
    written[slots[slots >= 0].long().cpu()] = True
    assert not caches[0].pairs.transpose(1, 2).reshape(pages * page, -1)[(~written).cuda()].any()
    before = [c.codes.clone() for c in caches]
    ops.qk_norm_rope_kvwrite(*args, *caches, None, page)
    assert all(torch.equal(a, c.codes) for a, c in zip(before, caches))
