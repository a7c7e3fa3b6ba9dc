"""Weight matrices in 4 bits: ``w = (code - zero) * scale`` with codes of 0 to 15 and a scale and a zero for each row's group of 32, 64 or 128
of ``k``.  A product of few rows then reads a quarter of the bytes that a bfloat16 matrix has.

:func:`pack_w4` lays codes, scales and zeros out as the kernels read them (``csrc/gemm_w4.hip`` states the order), :func:`quantize_w4` makes
them from a matrix, :func:`gemm_w4` multiplies.  (The reference has no weights of fewer bits than its activations'.)
"""

from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib, ops
from .ops import _check, _code, _gpu, _need, _on_current_device, _ptr, _refuse, _stream

GROUPS = (32, 64, 128)
# Products of more rows than this whose result is bfloat16 go through the large tiles.  us without and with them (x made fp16 and sums added), of 64, 96, 128 and 256
# rows: 28,672 x 4,096 33.5 / 33.2, 44.5 / 38.8, 53 / 41, 103 / 64; 4,096 x 14,336 24.7 / 27.8, 30.4 / 33.4, 38 / 36, 66 / 50; 11,264 x 2,048 16.7 / 20.1, 17.0 / 20.4,
# 22.6 / 20.5, 32.6 / 25.8; 6,144 x 4,096 17.5 / 20.3, 19.8 / 25.0, 25.0 / 26.2, 38 / 32.
DIRECT_ROWS = 96
_MAX_SPLITS = 16


@dataclass
class Weight4:
    """A matrix ``[n, k]`` in 4 bits as the kernels read it: ``data``, int32 ``[ceil(n / 16), ceil(k / 128), 64, 4]``, lane ``16 g + r`` of a
    block of 16 rows x 128 k has row ``r``, its word ``s`` the ``k`` ``32 s + 8 g + i`` at nibble ``i // 2 + 4 (i % 2)``; ``words``, int32
    ``[ceil(n / 16), ceil(k / 128) * 128 / group, 16]``, a group's scale in bfloat16 above ``16 + zero`` in bfloat16.  What is behind the
    last row or ``k`` is zero words."""

    data: torch.Tensor
    words: torch.Tensor
    n: int
    k: int
    group: int

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.n, self.k)

    def nbytes(self) -> int:
        return 4 * (self.data.numel() + self.words.numel())

    def first_rows(self, n: int) -> "Weight4":
        """The matrix of the first ``n`` rows (a multiple of 16, or all): a view."""
        _need(0 < n <= self.n and (n % 16 == 0 or n == self.n), "a matrix in 4 bits is cut at multiples of 16 rows")
        return Weight4(self.data[: -(-n // 16)], self.words[: -(-n // 16)], n, self.k, self.group)


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> Weight4:
    """``codes [n, k]`` (an integer type, 0 to 15), ``scales [n, k / group]`` (rounded to bfloat16) and ``zeros`` (integers 0 to 15 of the scales'
    shape; None: 8) as :class:`Weight4`, on the codes' device.  The values are looked at: on a GPU the call waits for it."""
    _need(codes.dim() == 2 and scales.dim() == 2 and not codes.is_floating_point() and scales.is_floating_point(),
          "codes are integers [n, k], scales are numbers [n, k / group]")
    n, k = codes.shape
    group = k // max(1, scales.shape[1])
    (group in GROUPS and scales.shape == (n, k // group) and k % group == 0 and n > 0) or _refuse(
        f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)}: groups of 32, 64 or 128 of k")
    _need(zeros is None or (zeros.shape == scales.shape and not zeros.is_floating_point()), "zeros are integers of the scales' shape")
    for t, name in ((codes, "codes"), (zeros, "zeros")):
        _need(t is None or (int(t.min()) >= 0 and int(t.max()) <= 15), f"{name} are 0 to 15")
    _need(bool(torch.isfinite(scales.to(torch.bfloat16)).all()), "scales must be finite in bfloat16")
    dev = codes.device
    nb, kb = -(-n // 16), -(-k // 128)
    full = torch.zeros((nb * 16, kb * 128), dtype=torch.uint8, device=dev)
    full[:n, :k] = codes.to(torch.uint8)
    # nibbles i // 2 + 4 (i % 2): byte b of a word is elements 4b % 8 ... as (low, high) = nibbles 2b, 2b + 1
    eight = full.view(nb, 16, kb, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)  # block, k block, g, r, s, i
    at = eight[..., [0, 2, 4, 6, 1, 3, 5, 7]]  # by nibble
    data = (at[..., 0::2] | (at[..., 1::2] << 4)).contiguous().view(torch.int32).view(nb, kb, 64, 4)
    words = torch.zeros((nb * 16, kb * 128 // group), dtype=torch.int32, device=dev)
    zero = torch.full_like(scales, 8) if zeros is None else zeros
    words[:n, : k // group] = ((scales.to(torch.bfloat16).view(torch.int16).int() << 16)
                               | (16 + zero.float()).to(torch.bfloat16).view(torch.int16).int())
    return Weight4(data, words.view(nb, 16, -1).transpose(1, 2).contiguous(), n, k, group)


def unpack_w4(w: Weight4):
    """``(codes uint8 [n, k], scales bfloat16 [n, k / group], zeros uint8)`` as :func:`pack_w4` was given them."""
    nb, kb = w.data.shape[:2]
    at = w.data.contiguous().view(torch.uint8).view(nb, kb, 4, 16, 4, 4)
    at = torch.stack([at & 15, at >> 4], -1).view(nb, kb, 4, 16, 4, 8)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    codes = at.permute(0, 3, 1, 4, 2, 5).reshape(nb * 16, kb * 128)[: w.n, : w.k].contiguous()
    words = w.words.transpose(1, 2).reshape(nb * 16, -1)[: w.n, : w.k // w.group]
    scales, zeros = (t.to(torch.int16).view(torch.bfloat16) for t in (words >> 16, words << 16 >> 16))
    return codes, scales, (zeros.float() - 16).to(torch.uint8)


def quantize_w4(w: torch.Tensor, group: int = 128) -> Weight4:
    """``w [n, k]`` rounded to 4 bits, each row's group of ``group`` by itself: the scale is a 15th of the span of the group's numbers and 0, in
    bfloat16, the zero the code nearest to 0's, a code the nearest number's.  (A group of zeros has the scale 1.)"""
    _need(w.dim() == 2 and w.is_floating_point(), "quantize_w4 takes a matrix of numbers")
    n, k = w.shape
    (group in GROUPS and k % group == 0 and n > 0 and k > 0) or _refuse(f"[{n}, {k}] in groups of {group}: 32, 64 or 128, a divisor of k")
    _need(bool(torch.isfinite(w).all()), "the matrix has numbers that are not finite")
    x = w.float().view(n, k // group, group)
    low, high = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    scale = ((high - low) / 15).to(torch.bfloat16)
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / scale.float()).clamp(0, 15)
    codes = (torch.round(x / scale.float()[..., None]) + zero[..., None]).clamp(0, 15)
    return pack_w4(codes.view(n, k).to(torch.uint8), scale, zero.to(torch.uint8))


_LAYOUT = "the matrix in 4 bits is not laid out as pack_w4 does it"


@functools.lru_cache(maxsize=4096)
def _sizes(x: Tuple[int, ...], x_stride: Tuple[int, ...], data: Tuple[int, ...], words: Tuple[int, ...], n: int, k: int, group: int) -> Tuple[int, int, int]:
    """Rows, K and the rows' distance of a product whose sizes fit, worked out once for them: a launch of a few us waits for the host."""
    _need(len(x) == 2, "a product in 4 bits takes bfloat16 x [M, K]")
    (M, K), (ldx, unit) = x, x_stride
    nb, kb = -(-n // 16), -(-k // 128)
    (n > 0 and k == K and group in GROUPS and K % group == 0) or _refuse(f"a matrix [{n}, {k}] in groups of {group} does not fit x [M, {K}]")
    _need(data == (nb, kb, 64, 4) and words == (nb, kb * 128 // group, 16), _LAYOUT)
    _need(unit == 1 and ldx % 8 == 0 and ldx >= K, "rows of x must be 16-byte aligned")
    return M, K, ldx


@functools.lru_cache(maxsize=4096)
def w4_plan(M: int, N: int, K: int, group: int) -> Tuple[int, int, int]:
    """How a product is cut: ``(0, 0, 1)`` for the kernel of up to 16 rows, else blocks of 16 rows of x a workgroup, of ``w`` a wave, and cuts of K.

    More than 64 rows go in equal parts of at most 64.  Two blocks of ``w`` a wave halve what the waves read of x: they are taken where that leaves 100 workgroups (64
    rows of 28,672 x 4,096, 112 workgroups in two cuts, 34.5 us, one block 37.7; 64 of 4,096 x 14,336, 16 in sixteen, 24.0 / 23.1; 48 of them 21.5 /
    19.6).  K is cut until there is a workgroup for every compute unit, not into less than 512 of k (64 rows of 4,096 x 4,096, us with 1, 2, 4 and 8 cuts: 31 /
    20.1 / 15.4 / 15.2)."""
    if M <= 16:
        return 0, 0, 1
    parts = -(-M // 64)
    mb = max(2, -(-M // (16 * parts)))
    nt = 2 if group >= (128 if mb == 4 else 64) and -(-N // 256) * parts >= 100 else 1  # (smaller groups' words do not fit the registers twice)
    workgroups, blocks = -(-N // (128 * nt)) * -(-M // (16 * mb)), -(-K // 128)
    splits = max(1, min(_MAX_SPLITS, ops.compute_units() // workgroups, blocks // 4))
    stages = -(-blocks // splits)
    return mb, nt, -(-blocks // stages)  # (none of them empty)


# What a round of the large tiles takes, as ops._LARGE_COST says it: fitted to 824 products (17 to 2,048 rows, 1,024 to 28,672 columns, 1,024 to 14,336 of
# k, 1 to 8 cuts) to 5 to 8 %; the plan that is the fastest by them takes 0.8 % longer than the fastest one on average, 11 % at most.
_LARGE_COST = {256256: ((0.983, 0.408, 14.4),), 128128: ((0.39, 0.119, 6.0), (0.601, 0.156, 8.8)),
               64128: ((0.315, 0.083, 4.5), (0.364, 0.201, 6.7), (0.526, 0.169, 9.0))}
_LARGE_HALVES = (0.592, 0.14, 5.9)


@functools.lru_cache(maxsize=4096)
def w4_large_plan(M: int, N: int, K: int, leave_sums: bool = False) -> Tuple[int, int, int]:
    """Tile, cuts of K and whole tiles (:func:`~fastgen_amd.kernels.ops.large_whole_tiles`) of a product through the large tiles; the sums of cuts are written and
    read at 4 TB/s, by a kernel of 3 us where they are not left."""
    units, best = ops.compute_units(), None
    for tile, costs in _LARGE_COST.items():
        tiles = -(-M // (tile // 1000)) * -(-N // (tile % 1000))
        for splits in (1, 2, 4, 8):
            steps = -(-(K // 64) // splits)
            steps += steps % 2  # a cut is whole blocks of 128 k
            if splits > 1 and (steps < 5 or steps * (splits - 1) >= K // 64 or tiles * splits > len(costs) * units):
                continue
            took = lambda cost, fill: steps * (cost[0] + cost[1] * fill) + cost[2]
            whole = ops.large_whole_tiles(tile, M, N) if splits == 1 else 0
            rounds, left = divmod(whole or tiles * splits, len(costs) * units)
            last = 0.0
            if whole:
                last = took(_LARGE_HALVES, 2 * (tiles - whole) / units)
            elif left:
                each = -(-left // units)
                last = took(costs[each - 1], left / (each * units))
            sums = (0.0 if leave_sums else 3.0) + (4 * splits + 2) * M * N / 4e6 if splits > 1 else 0.0
            cost = rounds * took(costs[-1], 1.0) + last + sums
            if best is None or cost < best[0]:
                best = (cost, tile, splits, whole)
    return best[1:]


def w4_cuts(M: int, w: Weight4, ldx: int) -> int:
    """Sums that :func:`gemm_w4` leaves of ``M`` bfloat16 rows with ``leave_sums``; 1: the product itself comes."""
    return w4_large_plan(M, w.n, w.k, True)[1] if _goes_large(M, w.n, w.k, ldx) else w4_plan(M, w.n, w.k, w.group)[2]


def _goes_large(M: int, N: int, K: int, ldx: int) -> bool:
    return M > DIRECT_ROWS and ops.gemm_large_takes(M, N, K, ldx)


def w4_scratch(M: int, N: int) -> int:
    """Bytes that the sums of cuts of K take at most for up to ``M`` rows: 16 cuts, a workgroup (up to 256 columns x 64 rows, :func:`w4_plan`) a compute unit, or
    those of the large tiles."""
    return max(min(_MAX_SPLITS * M * N, 256 * 64 * ops.compute_units()) * 4, ops.gemm_large_scratch(M, N) if M > DIRECT_ROWS else 0)


def gemm_w4(x, w: Weight4, out_dtype: Optional[torch.dtype] = None, silu_mul_epilogue: bool = False, leave_sums: bool = False) -> torch.Tensor:
    """``x @ w.T`` for bfloat16 ``x [M, K]`` and a matrix in 4 bits, bfloat16 or float32 out.  With ``silu_mul_epilogue`` ``w`` is a gate and an up matrix
    ordered by :func:`~fastgen_amd.kernels.ops.interleave_gate_up` and the result is ``silu(gate) * up`` ``[M, N / 2]`` in bfloat16.  ``x`` may be
    :class:`~fastgen_amd.kernels.ops.ScaledRows` (at most 16 rows): the result rows are scaled.  With ``leave_sums`` a product whose K is cut over
    workgroups comes as fp32 ``[cuts, M, N]`` sums (``N`` a multiple of 16), which the caller hands to a norm that adds them in order.

    Up to ``DIRECT_ROWS`` rows, for float32 results and where ``K`` is no multiple of 64 the weights enter the product as they are; more rows of a bfloat16 result are
    multiplied with the weights rounded to fp16 (csrc/tile_product.h; groups of a row whose scale is below 2^-25 of the row's largest lose digits there, as do
    numbers of ``x`` below 2^-29 of their row's largest).  A row's result depends on how many other rows there are in
    this and in the order of its sums only, and up to 16 rows not at all.
    A row of ``x`` with a number that is not finite has no finite results, and they need not be the infinities that a product of the
    numbers themselves has (a group's codes are multiplied 16 too large, and the sum of ``x`` 16 times taken off again)."""
    ssq, n_parts, dim, eps = None, 0, 0, 0.0
    if isinstance(x, ops.ScaledRows):
        _need(x.rows.shape[0] <= 16, "gemm_w4 scales at most 16 rows")
        ssq, n_parts, dim, eps = ops._row_scale_args(x, x.rows.shape[0])
        x = x.rows
    M, K, ldx, x_at = _checked(x, w)
    out_dtype = out_dtype or torch.bfloat16
    n = w.n
    large, cols, ld = _way(M, n, K, ldx, out_dtype, bool(silu_mul_epilogue), bool(leave_sums))
    if large:
        tile, splits, whole = w4_large_plan(M, n, K, leave_sums)
    else:
        mb, nt, splits = w4_plan(M, n, K, w.group)
    part = x.new_empty((splits, M, ld), dtype=torch.float32) if splits > 1 else None
    y = None if part is not None and leave_sums else x.new_empty((M, cols)) if out_dtype == torch.bfloat16 else x.new_empty((M, cols), dtype=out_dtype)
    if M == 0:
        return y
    if large:
        to, to_ld = (y, cols) if part is None else (part, ld)
        half, exponents = x.new_empty((M, K), dtype=torch.float16), x.new_empty(M + 3 + ld, dtype=torch.int32)
        st = _lib.load("gemm_w4").fg_w4_half(x_at, ldx, half.data_ptr(), exponents.data_ptr(), w.words.data_ptr(), M, n, K, w.group, _stream(x))
        st = st or _lib.load(f"gemm_large_w4@{w.group}").fg_gemm_large_w4(
            half.data_ptr(), K, w.data.data_ptr(), w.words.data_ptr(), exponents.data_ptr(), to.data_ptr(), to_ld, M * to_ld, splits, M, n, K, _code(to),
            int(silu_mul_epilogue and part is None), tile, whole, _stream(x))
        if not st and part is not None and y is not None:
            st = _lib.load("gemm_w4").fg_w4_add(part.data_ptr(), splits, ld, y.data_ptr(), cols, M, n, int(silu_mul_epilogue), _code(y), _stream(x))
        if st:
            _check(st, "gemm_w4")
        return y if y is not None else part
    st = _lib.load("gemm_w4").fg_gemm_w4(x_at, ldx, w.data.data_ptr(), w.words.data_ptr(), _ptr(y), cols, M, n, K, w.group, int(silu_mul_epilogue),
                                         ops._DTYPE_CODE[out_dtype], mb, nt, splits, _ptr(part), ssq, n_parts, dim, eps, _stream(x))
    if st:
        _check(st, "gemm_w4")
    return y if y is not None else part


@functools.lru_cache(maxsize=4096)
def _way(M: int, n: int, K: int, ldx: int, out_dtype: torch.dtype, gated: bool, leave_sums: bool) -> Tuple[bool, int, int]:
    """What the sizes of a product decide, worked out once for them: whether it goes through the large tiles, the result's columns and those of the sums of
    a cut; a refusal raises."""
    _need(out_dtype in (torch.bfloat16, torch.float32), "gemm_w4 gives bfloat16 or float32")
    _need(not gated or (n % 16 == 0 and out_dtype == torch.bfloat16), "the gate/up epilogue needs N % 16 == 0 and bf16 output")
    _need(not leave_sums or (n % 16 == 0 and not gated), "sums are left of a plain product, N % 16 == 0")
    return out_dtype == torch.bfloat16 and _goes_large(M, n, K, ldx), n // 2 if gated else n, -(-n // 16) * 16


def gemm_w4_residual(x, w: Weight4, h: torch.Tensor, norm_weight: torch.Tensor, eps: float) -> ops.ScaledRows:
    """For at most 16 rows: ``h += x @ w.T`` on the fp32 residual stream ``h [M, N]`` and, in the same kernel, what the RMSNorm that follows needs, as
    :func:`~fastgen_amd.kernels.ops.gemm_skinny_residual` does it.  ``x`` may itself be :class:`~fastgen_amd.kernels.ops.ScaledRows`."""
    rows = x.rows if isinstance(x, ops.ScaledRows) else x
    M, K, ldx, x_at = _checked(rows, w)
    N = w.n
    _gpu(rows, h, norm_weight)
    _need(0 < M <= 16, "gemm_w4_residual takes 1 to 16 rows")
    _need(h.dtype == torch.float32 and h.shape == (M, N) and h.stride(1) == 1 and h.stride(0) >= N, "h must be float32 [M, N]")
    _need(norm_weight.shape == (N,) and norm_weight.is_contiguous() and norm_weight.dtype in (torch.float32, torch.bfloat16),
          "norm_weight must be [N], float32 or bfloat16")
    x_out, ssq_out = rows.new_empty((M, N)), h.new_empty((M, -(-N // 16)))
    st = _lib.load("gemm_w4").fg_gemm_w4_residual(
        x_at, ldx, w.data.data_ptr(), w.words.data_ptr(), M, N, K, w.group, *ops._row_scale_args(x, M), h.data_ptr(), h.stride(0),
        norm_weight.data_ptr(), _code(norm_weight), x_out.data_ptr(), N, ssq_out.data_ptr(), _stream(rows))
    if st:
        _check(st, "gemm_w4_residual")
    return ops.ScaledRows(x_out, ssq_out, N, float(eps))


def _checked(x: torch.Tensor, w: Weight4) -> Tuple[int, int, int, int]:
    """Rows, K, the rows' distance and address of ``x``, which goes with ``w``."""
    data, words, x_at = w.data, w.words, x.data_ptr()
    _gpu(x, data, words)
    _on_current_device(x)
    M, K, ldx = _sizes(x.shape, x.stride(), data.shape, words.shape, w.n, w.k, w.group)
    _need(x.dtype == torch.bfloat16, "a product in 4 bits takes bfloat16 x [M, K]")
    _need(data.dtype == words.dtype == torch.int32 and data.is_contiguous() and words.is_contiguous() and (data.data_ptr() | words.data_ptr()) % 16 == 0, _LAYOUT)
    _need(x_at % 16 == 0, "rows of x must be 16-byte aligned")
    return M, K, ldx, x_at
