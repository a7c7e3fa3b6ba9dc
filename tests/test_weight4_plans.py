"""How the products with weights in 4 bits are cut (CPU), and every form of the kernel for 17 and more rows (GPU)."""

import pytest
import torch

from test_weight4 import DEV, _in_64, _matrix, _to, _x, gpu

from fastgen_amd.kernels import ops, weight4
from fastgen_amd.kernels.weight4 import gemm_w4, pack_w4

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


# ------------------------------------------------------------------------------- GPU
# columns: a wave's second block partly or wholly behind the end, a last block of 8 rows; k of whole and of cut blocks of 128
SHAPES = {32: [(1000, 1184), (48, 800)], 64: [(1000, 1088), (272, 1024)], 128: [(1000, 1280), (272, 1152), (48, 1024)]}


@gpu
@pytest.mark.parametrize("group,mb,nt", [(g, mb, nt) for g in weight4.GROUPS for mb, nt in sorted(_forms(g))])
def test_every_form(monkeypatch, group, mb, nt):
    """Rows of one workgroup and of several, the last of them full, of one row and of all but one; K whole and cut; every kind of result."""
    for n, k in SHAPES[group]:
        w = pack_w4(*_matrix(n + k + group, n, k, group))
        blocks = -(-k // 128)
        for m in (17, 16 * mb - 1, 16 * mb, 16 * mb + 1, 96):
            x = _x(m, m, k, 8)[:, :k]
            want, tol = _in_64(x, w, out_half=0.0)
            gated, gated_tol = _in_64(x, w, gated=True) if n % 16 == 0 else (None, None)
            x = x.to(DEV)
            for splits in (1, 2, 3, blocks):
                if -(-blocks // splits) * (splits - 1) >= blocks:
                    continue
                monkeypatch.setattr(weight4, "w4_plan", lambda *a: (mb, nt, splits))
                where = f"[{m}, {k}] x [{n}, {k}] in {splits} cuts"
                for out, half in ((torch.bfloat16, 2.0**-8), (torch.float32, 2.0**-24)):
                    got = gemm_w4(x, _to(w, DEV), out)
                    assert got.dtype == out and got.shape == (m, n)
                    assert ((got.cpu().double() - want).abs() <= tol + half * (want.abs() + tol)).all(), f"{where}: {out}"
                if n % 16:
                    continue
                sums = gemm_w4(x, _to(w, DEV), leave_sums=True)
                assert sums.shape == ((splits, m, n) if splits > 1 else (m, n))
                if splits > 1:
                    assert ((sums.cpu().double().sum(0) - want).abs() <= tol).all(), f"{where}: sums"
                got = gemm_w4(x, _to(w, DEV), silu_mul_epilogue=True)
                assert got.shape == (m, n // 2) and ((got.cpu().double() - gated).abs() <= gated_tol).all(), f"{where}: gated"


@gpu
@pytest.mark.parametrize("n,k,group", [(4096, 160, 32), (12288, 96, 32), (12304, 160, 32), (4096, 192, 64), (4112, 320, 64), (16400, 128, 64), (4096, 256, 128), (4112, 512, 128),
                                       (5120, 384, 128), (16384, 256, 128)])
def test_up_to_16_rows_on_both_sides_of_a_border(n, k, group):
    """A workgroup has one, two or four blocks of 16 rows of w by their number alone: stored, gated, and into the residual stream."""
    w, g = pack_w4(*_matrix(n, n, k, group)), torch.Generator().manual_seed(n)
    found = []
    for m in (1, 16):
        x = _x(7, 16, k)[:m]
        want, tol = _in_64(x, w, out_half=0.0)
        for out, half in ((torch.bfloat16, 2.0**-8), (torch.float32, 2.0**-24)):
            got = gemm_w4(x.to(DEV), _to(w, DEV), out)
            assert ((got.cpu().double() - want).abs() <= tol + half * (want.abs() + tol)).all()
        found.append(got)
        gated, gated_tol = _in_64(x, w, gated=True)
        assert ((gemm_w4(x.to(DEV), _to(w, DEV), silu_mul_epilogue=True).cpu().double() - gated).abs() <= gated_tol).all()
        h, norm = torch.randn(m, n, generator=g), 1 + 0.1 * torch.randn(n, generator=g)
        stream = h.to(DEV)
        rows = weight4.gemm_w4_residual(x.to(DEV), _to(w, DEV), stream, norm.to(DEV), 1e-5).rows
        want, tol = h.double() + want, tol + 2.0**-24 * (h.double() + want).abs()
        assert ((stream.cpu().double() - want).abs() <= tol).all()
        assert ((rows.cpu().double() - want * norm.double()).abs() <= norm.double().abs() * (tol * 1.01 + want.abs() * 1.01 * 2.0**-8)).all()
    assert torch.equal(found[0], found[1][:1])  # whatever is beside it


@gpu
@pytest.mark.parametrize("group", [64, 128])
def test_two_blocks_a_wave_have_the_bits_of_one(monkeypatch, group):
    n, k = 1008, 1280
    w, x = _to(pack_w4(*_matrix(group, n, k, group)), DEV), _x(5, 48, k).to(DEV)
    found = []
    for nt in (1, 2):
        monkeypatch.setattr(weight4, "w4_plan", lambda *a: (3, nt, 2))
        found.append([gemm_w4(x, w, torch.float32), gemm_w4(x, w, silu_mul_epilogue=True), gemm_w4(x, w, leave_sums=True)])
    assert all(torch.equal(a, b) for a, b in zip(*found))


@gpu
@pytest.mark.parametrize("n,k,group,m", [(28672, 256, 128, 60), (28672, 256, 64, 33), (28672, 256, 32, 64), (28672, 2176, 128, 64)])
def test_wide_matrices_as_they_are_planned(n, k, group, m):
    """Of so many columns a wave takes two blocks, with groups of 32 one."""
    w = pack_w4(*_matrix(n, n, k, group))
    assert weight4.w4_plan(m, n, k, group)[1] == (1 if group == 32 else 2)
    x = _x(m, m, k)
    want, tol = _in_64(x, w, gated=True)
    assert ((gemm_w4(x.to(DEV), _to(w, DEV), silu_mul_epilogue=True).cpu().double() - want).abs() <= tol).all()


@gpu
def test_cut_products_in_two_graphs_and_on_another_stream():
    """Sums of a cut K, x in fp16 and its exponents are a call's own: two graphs replayed in turns with eager work between them, and calls on two streams at once."""
    n, k = 528, 4096
    w = _to(pack_w4(*_matrix(3, n, k, 128)), DEV)
    calls = {"wide": (48, lambda x: gemm_w4(x, w)), "large": (200, lambda x: gemm_w4(x, w)), "gated": (40, lambda x: gemm_w4(x, w, silu_mul_epilogue=True)),
             "sums": (64, lambda x: gemm_w4(x, w, leave_sums=True)), "one row": (1, lambda x: gemm_w4(x, w, torch.float32))}
    assert weight4.w4_plan(48, n, k, 128)[2] > 1 and weight4.w4_large_plan(200, n, k)[1] > 1
    xs = {name: [_x(i, m, k).to(DEV) for i in range(3)] for name, (m, _) in calls.items()}
    want = {name: [call(x).clone() for x in xs[name]] for name, (_, call) in calls.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for name, (_, call) in calls.items():
        with torch.cuda.stream(side):
            there = call(xs[name][1])
        here = call(xs[name][2])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(there, want[name][1]) and torch.equal(here, want[name][2]), name
    torch.cuda.synchronize()
    graphs = []
    for name, (_, call) in calls.items():
        static, graph = xs[name][0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(static)
        graphs.append((name, static, graph, y))
    for i in (1, 2, 0, 1):
        for name, static, graph, y in graphs:
            static.copy_(xs[name][i])
            y.zero_()
        for name, static, graph, y in graphs:
            graph.replay()
            gemm_w4(xs["wide"][0], w)  # eager work in between
        torch.cuda.synchronize()
        for name, static, graph, y in graphs:
            assert torch.equal(y, want[name][i]), (name, i)


@gpu
@pytest.mark.parametrize("m", [1, 33, 130])
def test_the_first_rows_are_a_matrix(m):
    """A view of a packed matrix multiplies as one that was packed from these rows."""
    n, first, k = 208, 96, 256
    codes, scales, zeros = _matrix(5, n, k, 64)
    part, x = _to(pack_w4(codes, scales, zeros), DEV).first_rows(first), _x(m, m, k).to(DEV)
    whole = _to(pack_w4(codes[:first], scales[:first], zeros[:first]), DEV)
    assert part.data.data_ptr() and torch.equal(gemm_w4(x, part), gemm_w4(x, whole))
    assert torch.equal(gemm_w4(x, part, torch.float32), gemm_w4(x, whole, torch.float32))
