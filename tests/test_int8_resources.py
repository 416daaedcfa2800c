"""Registers and LDS of the built kernels of 8-bit integer products and of the
balance loss: none spills, and as many work-groups fit a CU as their tiles were
chosen for."""
import os
import re

import pytest

from chimere_amd import _lib
from test_kernel_resources import LDS, VGPRS, kernels


@pytest.fixture(scope="module")
def built():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return {n: m for n, m in kernels().items() if re.search(r"k_i8_|k_balance_", n)}


def test_no_spills(built):
    assert len(built) > 60
    for name, m in built.items():
        assert m[".vgpr_spill_count"] == 0 and m[".sgpr_spill_count"] == 0, name


def test_expert_tiles_per_cu(built):
    """Tiles of 64 pairs (four waves): three work-groups per CU; of 128 (eight waves): two."""
    seen = 0
    for name, m in built.items():
        k = re.match(r"_ZN7chimere\d+k_i8_(?:gate_up|down)ILi(64|128)", name)
        if not k:
            continue
        waves_per_simd = int(k[1]) // 64
        by_registers = VGPRS // ((m[".vgpr_count"] + 7) // 8 * 8) // waves_per_simd
        assert min(LDS // m[".group_segment_fixed_size"], by_registers) >= {"64": 3, "128": 2}[k[1]], name
        seen += 1
    assert seen == 6
