"""The workgroups that gemm_i8 and rotary_forward queue, counted on the host by the program of
test_layer_launches.py, which stands in for the HIP calls that launch a kernel."""
import pytest

import bmb
from test_layer_launches import ROWS, launches, program  # noqa: F401 (a fixture)

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


@pytest.mark.parametrize("M,N,K,want", [
    (1, 1, 0, [(1, 64)]), (16, 4096, 768, [(256, 256)]), (32, 100, 8192, [(7, 1024)]),
    (1, 1 << 20, 64, [(1 << 14, 256)]), (1, 1 << 28, 16, [(1 << 22, 256)]),
    (33, 65, 128, [(2, 256)]), (512, 4096, 4096, [(512, 256)]), (1000, 4096, 4096, [(256, 256)]),
    (1000, 50257, 768, [(788, 512)]), (1 << 17, 1 << 17, 128, [(1 << 18, 512)]),
    (1 << 28, 1, 16, [(1 << 20, 512)]),
    # ranges of 11 stages of 128 k, and what joins them: 1024 sums a workgroup
    (64, 64, 131071, [(94, 256), (4, 256)]), (65, 63, 131071, [(2 * 94, 256), (4, 256)])])
def test_products(program, M, N, K, want):  # noqa: F811
    """A workgroup for each tile, or for each of a tile's ranges of K."""
    for type in (bmb.F32, bmb.BF16):
        assert launches(program, "gemm", type, M, N, K) == want


@pytest.mark.parametrize("type,piece", [(bmb.F32, 4), (bmb.F16, 8), (bmb.BF16, 8)])
@pytest.mark.parametrize("tokens", [2, 255, 4097] + ROWS)
@pytest.mark.parametrize("heads,hs", [(1, 2), (1, 6), (1, 64), (3, 32), (8, 64), (40, 128),
                                      (1000, 256)])
def test_tokens(program, type, piece, tokens, heads, hs):  # noqa: F811
    """As many tokens a workgroup as it has threads for their pieces, or one; every token once."""
    pairs = hs // 2
    while pairs % piece:
        piece //= 2
    each = max(1, 256 // (heads * (pairs // piece)))
    got = launches(program, "rotary", type, tokens, heads, hs)
    assert {lanes for _, lanes in got} == {256}
    assert sum(blocks for blocks, _ in got) == -(-tokens // each)
