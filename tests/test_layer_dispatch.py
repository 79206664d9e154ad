"""The workgroups that gemm_i8 queues, counted on the host by the program of
test_layer_launches.py, which stands in for the HIP calls that launch a kernel."""
import pytest

import bmb
from test_layer_launches import launches, program  # noqa: F401 (a fixture)

FEW_LANES = 1024  # of a workgroup of the few-rows kernel where K is long
MOST = ((1 << 32) - 1) // FEW_LANES // 8 * 8  # workgroups of a launch, the same of each XCD


@pytest.mark.parametrize("type", [bmb.F32, bmb.F16, bmb.BF16])
@pytest.mark.parametrize("M,N", [(1, 16384), (4, 16385), (1, (1 << 26) - 16), (1, 1 << 26),
                                 (4, (1 << 26) + 1), (1, (1 << 28) - 17), (1, 1 << 28)])
def test_few_rows(program, type, M, N):  # noqa: F811
    """16 columns a workgroup; more of them than a dispatch has lanes for come in several
    launches."""
    got = launches(program, "gemm", type, M, N, 8193)
    assert {lanes for _, lanes in got} == {FEW_LANES}
    assert sum(blocks for blocks, _ in got) == -(-N // 16)
    assert len(got) == (-(-N // 16) + MOST - 1) // MOST
