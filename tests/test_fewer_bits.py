"""What the 8-bit products and the 4-bit cache refuse, without a device."""
from types import SimpleNamespace as NS

import pytest
import torch


def rows(N=4, K=32):
    from tinyserve_b200.kernels import ops
    return ops.Int8Rows(torch.zeros(N, K, dtype=torch.int8), torch.ones(N))


def pages(P=3, H=2, S=16, D=64):
    from tinyserve_b200.kernels import ops
    return ops.Int4Pages(torch.zeros(P, H, S, D // 2, dtype=torch.uint8), torch.zeros(P, H, S, 2, dtype=torch.bfloat16))


def test_rows_in_8_bits():
    from tinyserve_b200.kernels import ops
    with pytest.raises(TypeError, match="int8"):
        ops.Int8Rows(torch.zeros(4, 32), torch.ones(4))
    with pytest.raises(TypeError, match="float32"):
        ops.Int8Rows(torch.zeros(4, 32, dtype=torch.int8), torch.ones(5))
    with pytest.raises(ValueError, match="16 bytes"):
        ops.Int8Rows(torch.zeros(4, 33, dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError, match="16 bytes"):
        ops.Int8Rows(torch.zeros(32, 32, dtype=torch.int8).t(), torch.ones(32))
    assert ops.Int8Rows(torch.zeros(4, 48, dtype=torch.int8)[:, :33], torch.ones(4)).shape == (4, 33)


@pytest.mark.parametrize("x,error,match", [
    (torch.zeros(2, 31), ValueError, "does not fit"),
    (torch.zeros(2, 32, dtype=torch.float16), TypeError, "float32 or bfloat16"),
    (torch.zeros(2, 2, 32), TypeError, "float32 or bfloat16"),
    (torch.zeros(32, 32).t(), ValueError, "one run"),
    (torch.zeros(2, 32), RuntimeError, "no CPU path"),
])
def test_product(x, error, match):
    from tinyserve_b200.kernels import ops
    with pytest.raises(error, match=match):
        ops.linear(x, rows())


def test_product_of_mixed_operands():
    from tinyserve_b200.kernels import ops
    with pytest.raises(TypeError, match="weight in 8 bits"):
        ops.linear(rows(), torch.zeros(4, 32))
    with pytest.raises(ValueError, match="bias"):
        ops.linear(torch.zeros(2, 32), rows(), torch.zeros(5))
    with pytest.raises(ValueError, match="K is 1 to"):
        ops.quantize_rows(torch.zeros(1, ops.INT8_MAX_K + 1))


def test_cuts_along_k_are_never_empty():
    from tinyserve_b200.kernels import ops
    for M in (1, 17, 64, 65, 5000):
        for N in (1, 128, 1000, 4096, 24576):
            for K in (1, 128, 129, 1000, 4096, 12288, 131072):
                (tile, s), slices = ops.int8_plan(M, N, K), -(-K // 128)
                assert (tile, s) == (256, 0) or (tile in (16, 32, 64, 128) and 1 <= s <= 8 and (s - 1) * -(-slices // s) < slices)


def test_how_keys_are_cut():
    from tinyserve_b200.kernels import ops
    for blocks in (1, 8, 24, 64, 100, 150, 296, 297, 740, 741, 10 ** 6):
        for keys in (0, 1, 160, 2047, 2048, 32768, 10 ** 6):
            splits = ops.int4_decode_splits(blocks, keys)
            assert 1 <= splits <= 32 and (splits == 1 or (splits * 160 <= keys and splits * blocks <= 4 * ops.num_sms()))
            assert splits in (1, 2, 4, 8) or splits > ops.INT4_CLUSTER_SPLITS
            assert 1 <= ops.int4_attention_splits(blocks, keys) <= 32
            for D in (32, 128, 160):
                assert ops.int4_decode_warps(blocks, splits, D) == (4 if splits == 1 and D <= 128 and blocks > 740 else 8)


def test_pages_in_4_bits():
    from tinyserve_b200.kernels import ops
    with pytest.raises(TypeError, match="uint8"):
        ops.Int4Pages(torch.zeros(3, 2, 16, 32), torch.zeros(3, 2, 16, 2, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="pairs"):
        ops.Int4Pages(torch.zeros(3, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 8, 2, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        ops.Int4Pages(torch.zeros(3, 16, 2, 32, dtype=torch.uint8).transpose(1, 2), torch.zeros(3, 2, 16, 2, dtype=torch.bfloat16))


def test_write():
    from tinyserve_b200.kernels import ops
    x, slots = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int32)
    for args, error, match in (((x, x, pages(), torch.zeros(1), slots), TypeError, "Int4Pages"), ((x, x, pages(), pages(P=4), slots), TypeError, "one shape"),
                               ((x, x[:4], pages(), pages(), slots), TypeError, "float32 or bfloat16"), ((x, x.bfloat16(), pages(), pages(), slots), TypeError, "bfloat16"),
                               ((x[..., :32], x[..., :32], pages(), pages(), slots), TypeError, "64"), ((x, x, pages(), pages(), slots[:4]), TypeError, "slot_mapping"),
                               ((x, x, pages(), pages(), slots.long()), TypeError, "int32"), ((x, x, pages(S=12), pages(S=12), slots), ValueError, "power of two"),
                               ((x.transpose(0, 2).contiguous().transpose(0, 2), x, pages(), pages(), slots), ValueError, "one run"),
                               ((x, x, pages(), pages(), slots), RuntimeError, "no CPU path")):
        with pytest.raises(error, match=match):
            ops.int4_kvwrite(*args)


def test_attention():
    from tinyserve_b200.kernels import ops
    q = torch.zeros(3, 4, 64)
    ctx = NS(num_requests=2, max_q_len=2, max_kv_len=20, cu_q=torch.zeros(3, dtype=torch.int32), kv_lens=torch.zeros(2, dtype=torch.int32))
    view = NS(page_size=16, block_table=torch.zeros(2, 2, dtype=torch.int32))

    def call(q=q, k=None, v=None, view=view, ctx=ctx, **kw):
        return ops.paged_attention(q, pages() if k is None else k, pages() if v is None else v, view, ctx, 0.1, **kw)

    other = lambda o, **kw: NS(**{**vars(o), **kw})
    for kw, error, match in ((dict(keep_first=4, window=8), ValueError, "whole numbers"), (dict(chunk=4), ValueError, "whole numbers"),
                             (dict(slopes=torch.zeros(4)), ValueError, "whole numbers"), (dict(k=pages(D=32)), TypeError, "one shape"),
                             (dict(v=torch.zeros(3, 2, 16, 64)), TypeError, "Int4Pages"), (dict(q=torch.zeros(3, 3, 64)), TypeError, "multiple of 2"),
                             (dict(q=torch.zeros(3, 4, 32)), TypeError, "64"), (dict(q=q.half()), TypeError, "bfloat16"), (dict(window=-1), ValueError, "positive"),
                             (dict(softcap=-1.0), ValueError, "positive"), (dict(sinks=torch.zeros(3)), TypeError, "sinks"), (dict(view=other(view, page_size=32)), ValueError, "pages of"),
                             (dict(view=other(view, block_table=torch.zeros(1, 2, dtype=torch.int32))), TypeError, "block table"),
                             (dict(view=other(view, block_table=torch.zeros(2, 2))), TypeError, "int32"), (dict(ctx=other(ctx, cu_q=torch.zeros(2, dtype=torch.int32))), TypeError, "cu_q"),
                             (dict(ctx=other(ctx, kv_lens=torch.zeros(2))), TypeError, "kv_lens"), (dict(backend="tcgen05x"), ValueError, "backend"), (dict(), RuntimeError, "no CPU path")):
        with pytest.raises(error, match=match):
            call(**kw)


def test_engine_options():
    from tinyserve_b200.config.engine_config import EngineConfig
    cfg = EngineConfig(model="", weight_dtype="int8", kv_cache_dtype="int4")
    assert (cfg.weight_dtype, cfg.kv_cache_dtype, EngineConfig(model="").weight_dtype, EngineConfig(model="").kv_cache_dtype) == ("int8", "int4", "auto", "auto")
    for kw in (dict(weight_dtype="int4"), dict(kv_cache_dtype="int8")):
        with pytest.raises(ValueError, match="must be one of"):
            EngineConfig(model="", **kw)


def test_models_with_a_4_bit_cache():
    from helpers import tiny_config
    from tinyserve_b200.parts.model import build_model
    model = build_model(tiny_config("C"), "int4")
    assert [g.kind for g in model.cache_groups] == ["full", "window"]
    for spec in model.cache_groups:
        assert [(t.name, t.heads, t.width, t.dtype) for t in spec.tensors] == [("k", 2, 24, "uint8"), ("k_pairs", 2, 2, "bfloat16"), ("v", 2, 24, "uint8"), ("v_pairs", 2, 2, "bfloat16")]
        assert spec.bytes_per_token(2) == spec.bytes_per_token(4) == 2 * 2 * (24 + 4)
    plain = build_model(tiny_config("C"))
    assert [spec.bytes_per_token(4) for spec in plain.cache_groups] == [2 * 2 * 48 * 4] * 2


def test_models_that_cannot():
    from delilorn_configs import DELILORN_TINY, delilorn_config
    from tinyserve_b200.parts.model import build_model
    for name in DELILORN_TINY:
        config = delilorn_config(name)
        build_model(config)
        with pytest.raises(ValueError, match="4 bits|4-bit"):
            build_model(config, "int4")


def test_which_matrices_may_be_held_in_8_bits():
    from helpers import tiny_config
    from tinyserve_b200.parts.model import build_model
    model = build_model(tiny_config("B"))
    names = {f"{part.path}.{name}" for part in model.named_parts() for name, spec in part.param_specs().items() if spec.int8}
    assert names == {f"model.layers.{i}.{n}" for i in range(3) for n in ("self_attn.qkv_proj.weight", "self_attn.o_proj.weight", "mlp.gate_up_proj.weight", "mlp.down_proj.weight")}
