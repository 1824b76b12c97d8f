"""CPU: registers, LDS and scratch of the row cache's kernels, read from the built objects: a spill or a wavefront less a SIMD fails no
test of results."""
import os
import re

import pytest

from .test_kernel_resources_cpu import KR

REGISTERS, LDS = 512, 160 * 1024     # of a SIMD's lane, of a CU


@pytest.fixture(scope="module")
def kernels():
    if not os.path.isdir(KR.OBJDIR) or not any(f.startswith("partition_") for f in os.listdir(KR.OBJDIR)):
        pytest.skip("objects not built (python -m redisearch_amd.build)")
    return [k for k in KR.all_kernels() if re.match(r"(partition_few|partition_many|row_write|row_read|row_copy_in|adjust_scores)", k["name"])]


def waves(k):
    """Wavefronts a SIMD: by registers, and by the workgroups that LDS has room for."""
    by_registers = REGISTERS // (-(-k["vgpr"] // 8) * 8)
    by_lds = LDS // max(k["lds"], 1) * (k["wg"] // 64) // 4
    return min(by_registers, by_lds, 8)


def test_nothing_spills(kernels):
    assert len(kernels) > 150
    assert not [k["name"] for k in kernels if k["vgpr_spill"] or k["sgpr_spill"] or k["scratch"]]


def test_partition_scores_keep_their_wavefronts(kernels):
    few = [k for k in kernels if k["name"].startswith("partition_few_kernel<")]
    many = [k for k in kernels if k["name"].startswith("partition_many_kernel<")]
    assert few and many
    for k in few:      # eight and sixteen wavefronts a workgroup: four a SIMD; four (small calls): one workgroup a CU at the least
        assert waves(k) >= (4 if k["wg"] >= 512 else 1), k
    for k in many:     # two workgroups a CU, one's products behind the other's scores
        assert waves(k) >= 2 and 2 * k["lds"] <= LDS, k


def test_rows_and_rules_keep_their_wavefronts(kernels):
    for k in kernels:
        if k["name"].startswith(("row_", "adjust_")):
            assert waves(k) >= 5, k
