"""CPU gate: the attention kernels' launches count on two (D 128) or three
(D 64) four-wave workgroups sharing a CU -- the kernel for few rows on one or
two -- so their registers and LDS must allow that.  Reads only metadata of the
library built in this tree."""
import os

import resource_gate as gate


def test_attention_workgroups_share_a_cu():
    assert os.path.exists(gate.LIB_PATH), "make -C flash-attention3_amd"
    kernels, bad = gate.check(gate.LIB_PATH)
    assert bad == []
    for what, counts, number in (("attn_fwd_kernel", {64: 3, 128: 2}, 32),
                                 ("attn_bwd_kernel", {64: 3, 128: 2}, 48),
                                 ("attn_token_kernel", {64: 2, 128: 1}, 16)):
        found = [k for k in kernels if what in k[".name"]]
        assert len(found) == number, what
        for k in found:
            n = counts[64 if "ILi64E" in k[".name"] else 128]
            assert k[".max_flat_workgroup_size"] == 256
            assert k[".vgpr_count"] + k[".agpr_count"] <= 512 // n // 8 * 8, k[".name"]
            assert n * k[".group_segment_fixed_size"] <= gate.LDS_BYTES, k[".name"]
    for what in ("attn_join_kernel", "attn_sum_kernel", "attn_delta_kernel", "attn_ranges_kernel",
                 "rotary_kernel"):
        assert any(what in k[".name"] for k in kernels), what
