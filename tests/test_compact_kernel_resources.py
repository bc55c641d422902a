"""What the compiler made of the kernels of the 4-bit cache, the gathered weights and eviction: none keeps registers in
scratch memory, and those that hide memory behind several wavefronts fit as many."""
import os

import pytest

from tests.test_kernel_resources import HIPCC, resource_usage

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
LEAST_WAVES = {      # part of the mangled name -> wavefronts per SIMD
    "paged_attention_fp4_kernelILi4E": 1, "attention_weights_one_tile_fp4_kernelILi4E": 5, "attention_weights_one_tile_fp4_kernelILi8E": 3,
    "attention_weights_mfma_kernelILi4ELi1ELi2E": 2, "choose_tokens_kernelILi32E": 4, "fp4_store_kernel": 4, "move_tokens": 4}


@pytest.mark.parametrize("name", ["cache_fp4", "attention_fp4", "attention_weights", "evict", "rope_kv"])
def test_the_kernels_keep_their_registers(name, tmp_path):
    usage = resource_usage(name, tmp_path)
    assert usage, "no kernel was reported"
    for kernel, fields in usage.items():
        assert fields["ScratchSize [bytes/lane]"] == 0, f"{kernel} spills {fields['ScratchSize [bytes/lane]']} bytes per lane"
        for part, least in LEAST_WAVES.items():
            assert part not in kernel or fields["Occupancy [waves/SIMD]"] >= least, (kernel, fields)
