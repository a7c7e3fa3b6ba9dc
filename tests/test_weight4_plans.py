"""How the products with weights in 4 bits are cut (CPU), and every form of the kernel for 17 and more rows (GPU)."""

import pytest

from fastgen_amd.kernels import ops, weight4

ROWS = (*range(17, 97), 100, 127, 128, 129, 192, 257, 700, 2048, 8192)
COLUMNS = (16, 48, 1000, 1024, 4096, 6144, 11264, 14336, 25600, 28672, 29536, 57344, 128000)
DEPTHS = (32, 128, 160, 512, 1024, 2080, 4096, 8192, 14336, 15360, 28672)


@pytest.fixture
def units(monkeypatch, request):
    monkeypatch.setattr(ops, "compute_units", lambda: request.param)
    weight4.w4_plan.cache_clear()
    weight4.w4_large_plan.cache_clear()
    yield request.param
    weight4.w4_plan.cache_clear()
    weight4.w4_large_plan.cache_clear()


def _forms(group):
    """Blocks of 16 rows of x a workgroup and of w a wave that the kernel is built with."""
    return {(mb, nt) for mb in (2, 3, 4) for nt in (1, 2) if nt == 1 or group == 128 or (group == 64 and mb < 4)}


@pytest.mark.parametrize("units", [256, 64, 304], indirect=True)
@pytest.mark.parametrize("group", weight4.GROUPS)
def test_plans_of_17_and_more_rows(units, group):
    """No cut is empty, the form is one that there is, and the sums of the cuts fit what a model sets aside for them, for this many rows and for a
    step of more (a model knows its longest step only)."""
    for M in ROWS:
        for N in COLUMNS:
            for K in DEPTHS:
                if K % group:
                    continue
                mb, nt, splits = weight4.w4_plan(M, N, K, group)
                blocks = -(-K // 128)
                assert (mb, nt) in _forms(group)
                assert 1 <= splits <= weight4._MAX_SPLITS and -(-blocks // splits) * (splits - 1) < blocks
                if splits > 1:
                    sums = splits * M * (-(-N // 16) * 16) * 4
                    for most in (M, M + 1, 96, 2048):
                        assert most < M or sums <= weight4.w4_scratch(most, -(-N // 16) * 16), (M, N, K, mb, nt, splits, most)


@pytest.mark.parametrize("units", [256], indirect=True)
def test_sums_of_two_blocks_a_wave(units):
    """Two cuts of 64 rows of 28,672 columns: workgroups of 256 columns."""
    assert weight4.w4_plan(64, 28672, 4096, 128) == (4, 2, 2)
    assert weight4.w4_scratch(64, 28672) >= 2 * 64 * 28672 * 4
