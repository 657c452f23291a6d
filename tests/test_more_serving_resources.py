"""What the compiler gave the kernels of shared prefixes, rotary positions and copies: like those of
test_serving_resources.py, none keeps a vector register, or an array, in scratch memory."""

import os

import pytest

from test_serving_resources import READELF, kernels  # noqa: F401 (a fixture)

KERNELS = {"shared_plan_kernel": 1, "shared_tasks_kernel": 6, "shared_join_kernel": 6, "rotate_kernel": 2, "turn_rows_kernel": 2,
           "turn_pages_kernel": 2, "copy_pages_kernel": 1}


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
@pytest.mark.parametrize("name", sorted(KERNELS))
def test_no_scratch_memory(kernels, name):  # noqa: F811
    of = {symbol: fields for symbol, fields in kernels.items() if name in symbol}
    assert len(of) == KERNELS[name], sorted(kernels)
    for symbol, fields in of.items():
        assert int(fields["vgpr_spill_count"]) == 0 and int(fields["private_segment_fixed_size"]) == 0, (symbol, fields)
