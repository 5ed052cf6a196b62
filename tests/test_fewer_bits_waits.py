"""What the kernels of the 8-bit products and the 4-bit cache wait for, looked for in their text: a missing wait shows on the device now and
then only."""
import re

import pytest

from test_kernel_sources import kernels

FILES = ("attention_int4.cu", "attention_int4_tcgen05.cu", "gemm_int8.cu", "gemm_int8_pair.cu")
OURS = sorted(name for name in kernels() if name[0] in FILES)


def test_the_kernels_are_found():
    assert {k for _, k in OURS} >= {"quantize_rows_kernel", "gemm_i8_kernel", "gemm_i8_pair_kernel", "int4_kvwrite_kernel", "int4_rope_kvwrite_kernel",
                                    "int4_attend_kernel", "int4_combine_kernel", "int4_mma_kernel", "int4_prefill_kernel"}


@pytest.mark.parametrize("name", [n for n in OURS if n[1] != "gemm_i8_kernel"])
def test_every_thread_waits_before_it_reads(name):
    """One wait, of every block and under no condition, before anything that a predecessor may have written is read.  (The 8-bit product
    fetches constant weights before its wait, see below; a norm's weights are nobody's output.)"""
    body = kernels()[name][1]
    assert body.count("pdl_wait();") == 1
    before = body[:body.index("pdl_wait();")]
    assert re.search(r"[;}]\s*$", before) and before.count("{") - before.count("}") == 1
    assert not re.search(r"p\.(q|k|v|x|kc|vc|kp|vp|cu_q|kv_lens|block_table|slot_mapping|sx|sw)\b|rp\.(qkv|positions)\b", before)


def test_codes_of_weights_are_fetched_early_only_where_they_are_constant():
    """What stands between the kernel that made a weight's codes and the product (the rows' codes, say) does not make them visible to the
    product: only the caller's word that they are constant lets it read them before its wait."""
    from test_kernel_sources import CSRC
    with open(f"{CSRC}/gemm_int8.cu") as fh:
        text = re.sub(r"//[^\n]*", "", fh.read())
    body = kernels()[("gemm_int8.cu", "gemm_i8_kernel")][1]
    loader = body[body.index("if (threadIdx.x == 0) {", body.index("pdl_trigger")):]
    assert loader.index("if (!p.w_ready) pdl_wait();") < loader.index("tma_load_2d") < loader.index("    pdl_wait();\n") < loader.index("&map_x")
    made = re.search(r"I8Params p = \{([^;]*)\};", text).group(1)
    assert made.split(",")[-1].strip() == "w_constant"


def test_bulk_copies_come_behind_the_ranking_of_requests():
    """The ranking uses the ring's memory by ordinary stores; a copy by the other proxy into the same bytes needs a fence, then a barrier."""
    body = re.sub(r"\s+", " ", kernels()[("attention_int4.cu", "int4_mma_kernel")][1])
    between = body[body.index("nth_longest<"):body.index("bulk_copy(")]
    assert "if (p.ordered) { fence_async_shared(); __syncthreads(); }" in between


def test_what_a_launch_keeps_for_its_device_is_atomic():
    """Calls through ctypes run side by side on several host threads: the word that says which devices a kernel is set up for is shared."""
    from test_kernel_sources import CSRC
    with open(f"{CSRC}/common.cuh") as fh:
        text = fh.read()
    struct = re.search(r"struct SmemSet \{(.*?)\n\};", text, re.S).group(1)
    assert "std::atomic<unsigned long long> done{0};" in struct and "done.fetch_or(" in struct
    assert not re.search(r"\bdone\s*(\||=)", struct)
