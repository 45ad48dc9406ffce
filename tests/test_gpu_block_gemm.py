"""Products of 8-bit floats with a scale for each block of 128 terms, and the quantisation that makes their operands, against
their definitions in 64 bits.

Tolerances.  Products of two 8-bit floats are exact in f32.  The sum of a block's 128 terms on the tensor core and the sum of
the blocks are f32 sums of at most 128 + blocks + 2 additions and multiplications (the scales' product, its product with the
block), each off by at most one unit of 2^-23 (additions may truncate) of the sum of absolute values; the result is then
rounded to out_dtype, half a step.  Quantisation is defined to the bit."""

import numpy as np
import pytest
import torch

from gpu_util import TORCH_OF
from plaidml_b200 import kernels as K

pytestmark = pytest.mark.gpu

F8 = {K.F8E4M3: torch.float8_e4m3fn, K.F8E5M2: torch.float8_e5m2}
LARGEST = {K.F8E4M3: 448.0, K.F8E5M2: 57344.0}
HALF_STEP = {K.F32: 2.0 ** -24, K.BF16: 2.0 ** -8, K.F16: 2.0 ** -11}


def blocks(n):
    return (n + 127) // 128


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bits(shape, dtype, g, spread=1.0):
    x = torch.randn(shape, device="cuda", generator=g) * (LARGEST[dtype] / 6) * spread
    return x.clamp(-LARGEST[dtype], LARGEST[dtype]).to(F8[dtype])


def scales(shape, g):
    """Over twelve binary orders, as blocks of unlike sizes have."""
    return torch.exp2(torch.rand(shape, device="cuda", generator=g) * 12 - 12)


def expect(a, sa, b, sb, b_rows):
    """(the product, the same with absolute values) in 64 bits: a [m, k], sa [blocks, m], b [n, k], sb as b_rows says."""
    n, k = b.shape
    fa = a.double() * sa.double().t().repeat_interleave(128, 1)[:, :k]
    fb = sb.double().t() if b_rows == 1 else sb.double().repeat_interleave(128, 0)[:n]
    fb = b.double() * fb.repeat_interleave(128, 1)[:, :k]
    return fa @ fb.t(), fa.abs() @ fb.abs().t()


def check(c, want, size, k, out):
    tol = (130 + blocks(k)) * 2.0 ** -23 * size + HALF_STEP[out] * want.abs()
    tol += {K.F16: 2.0 ** -25}.get(out, 1e-300)     # half of f16's smallest step
    bad = (c.double() - want).abs() > tol
    if out == K.F16:    # rounding to nearest gives an infinity of the sign from 65520 on, which is half a step above the largest number
        bad = torch.where(torch.isinf(c), (want * c.sign() + tol < 65520), bad)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by {float(((c.double() - want).abs() / tol).max()):.1f} tolerances"


def padded(t, ld):
    """The same values in rows `ld` apart, NaN bits in between."""
    wide = torch.full((*t.shape[:-1], ld), 0x7f, dtype=torch.uint8, device="cuda").view(t.dtype)
    wide[..., : t.shape[-1]] = t
    return wide


def make(m, n, k, a=K.F8E4M3, b=K.F8E4M3, b_rows=128, each=(), seed=1):
    g = gen(seed)
    ld = (k + 15) // 16 * 16
    x = {"a": padded(bits((m, k), a, g), ld), "b": padded(bits(each + (n, k), b, g), ld), "ld": ld}
    x["sa"] = scales((blocks(k), m), g)
    x["sb"] = scales(each + ((blocks(n), blocks(k)) if b_rows == 128 else (blocks(k), n)), g)
    return x


def run(plan, x, c, offsets=None, stream=0):
    plan.block_gemm(x["a"].data_ptr(), x["sa"].data_ptr(), x["b"].data_ptr(), x["sb"].data_ptr(), c.data_ptr(),
                    None if offsets is None else offsets.data_ptr(), stream=stream)


SIZES = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (3, 130, 257), (16, 256, 1024), (17, 520, 384), (33, 127, 130), (64, 1000, 640),
         (65, 128, 128), (100, 64, 3001), (128, 128, 64), (129, 257, 1000), (300, 1001, 520), (777, 2050, 515), (513, 384, 128),
         (1000, 40, 2049), (2050, 1100, 1030)]


@pytest.mark.parametrize("out", [K.BF16, K.F32, K.F16])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_product(m, n, k, out):
    x = make(m, n, k, seed=m + n + k)
    c = torch.empty((m, n), dtype=TORCH_OF[out], device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, out, m, n, k, lda=x["ld"], ldb=x["ld"]))
    run(plan, x, c)
    plan.check()
    check(c, *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], 128), k, out)


@pytest.mark.parametrize("a, b", [(K.F8E5M2, K.F8E4M3), (K.F8E4M3, K.F8E5M2), (K.F8E5M2, K.F8E5M2)])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("m, n, k", [(1, 300, 300), (40, 129, 1000), (260, 513, 700)])
def test_product_types_and_scales_of_each_row(m, n, k, a, b, b_rows):
    x = make(m, n, k, a, b, b_rows, seed=m)
    c = torch.empty((m, n), dtype=torch.float32, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(a, b, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"], b_scale_rows=b_rows))
    run(plan, x, c)
    plan.check()
    check(c, *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], b_rows), k, K.F32)


@pytest.mark.parametrize("m", [1, 30, 200])
@pytest.mark.parametrize("out, ldc", [(K.BF16, 304), (K.BF16, 301), (K.F32, 300), (K.F32, 309)])
def test_product_strides(m, out, ldc):
    """Rows of C inside a wider matrix whose other columns stay, scales stored by rows of A and by columns of B."""
    n, k = 300, 400
    x = make(m, n, k, seed=5)
    c = torch.full((m + 1, ldc), 7.0, dtype=TORCH_OF[out], device="cuda")
    d = K.block_gemm_desc(K.F8E4M3, K.F8E4M3, out, m, n, k, lda=x["ld"], ldb=x["ld"], ldc=ldc, a_scale_row=6, a_scale_block=1,
                          b_scale_row=1, b_scale_block=9)
    want = expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], 128)
    sa = torch.full((m, 6), float("nan"), device="cuda")
    sa[:, : blocks(k)] = x["sa"].t()
    sb = torch.full((blocks(k), 9), float("nan"), device="cuda")
    sb[:, : blocks(n)] = x["sb"].t()
    x["sa"], x["sb"] = sa, sb
    plan = K.Plan("block_gemm", d)
    run(plan, x, c)
    plan.check()
    check(c[:m, :n], *want, k, out)
    assert (c[:m, n:] == 7).all() and (c[m] == 7).all()


TILES = [K.BLOCK_TILES_FEW, K.BLOCK_TILES_SINGLE, K.BLOCK_TILES_PAIR]


@pytest.mark.parametrize("tiles", TILES)
@pytest.mark.parametrize("out", [K.BF16, K.F32])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("m, n, k", [(1, 130, 128), (127, 257, 140), (300, 515, 3000), (257, 1000, 1030), (1030, 264, 96), (520, 2051, 257)])
def test_product_by_each_kind_of_tiles(m, n, k, b_rows, out, tiles):
    x = make(m, n, k, b_rows=b_rows, seed=m + n)
    c = torch.full((m + 1, n + 5), 7.0, dtype=TORCH_OF[out], device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, out, m, n, k, lda=x["ld"], ldb=x["ld"], ldc=n + 5, b_scale_rows=b_rows, tiles=tiles))
    run(plan, x, c)
    plan.check()
    check(c[:m, :n], *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], b_rows), k, out)
    assert (c[m] == 7).all() and (c[:, n:] == 7).all()


def test_products_with_k_split_by_any_number_of_ctas():
    """Few tiles and a deep K: the split follows the shape; each is compared with the formula and is the same on every call."""
    for m, n, k in ((20, 128, 4096), (1, 1000, 8192), (128, 128, 8000), (100, 500, 4096), (256, 1024, 8192), (130, 2048, 2048)):
        x = make(m, n, k, seed=k)
        c, again = (torch.empty((m, n), dtype=torch.float32, device="cuda") for _ in range(2))
        plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k))
        run(plan, x, c)
        run(plan, x, again)
        plan.check()
        check(c, *expect(x["a"], x["sa"], x["b"], x["sb"], 128), k, K.F32)
        assert torch.equal(c, again)


GROUPS = {
    "one": [5], "empty": [0, 0, 0], "gaps": [0, 3, 0, 0, 130, 1, 0, 17, 0], "even": [64] * 6, "tails": [1, 127, 128, 129, 255, 256, 257, 0],
    "many": [(7 * i) % 5 for i in range(257)], "long": [700, 0, 900, 2],
}


@pytest.mark.parametrize("tiles", [0] + TILES)
@pytest.mark.parametrize("out", [K.BF16, K.F32])
@pytest.mark.parametrize("name", GROUPS)
def test_groups_of_rows(name, out, tiles):
    counts = GROUPS[name]
    groups, used, n, k = len(counts), sum(counts), 264, 400
    m = used + 9                                    # rows behind the last group
    x = make(m, n, k, each=(groups,), seed=len(name))
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    c = torch.full((m, n), 3.0, dtype=TORCH_OF[out], device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, out, m, n, k, lda=x["ld"], ldb=x["ld"], groups=groups, tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    at = 0
    for g, count in enumerate(counts):
        if count:
            rows = slice(at, at + count)
            check(c[rows], *expect(x["a"][rows, :k], x["sa"][:, rows], x["b"][g, :, :k], x["sb"][g], 128), k, out)
        at += count
    assert (c[used:] == 3).all()


@pytest.mark.parametrize("counts", [[1, 2, 0, 3], [0, 0], [5], [2, 0, 0, 1, 30, 0, 4]])
@pytest.mark.parametrize("m, n", [(1, 200), (100, 300), (500, 129)])
@pytest.mark.parametrize("tiles", [0] + TILES)
def test_groups_of_terms(counts, m, n, tiles):
    groups, k = len(counts), max(1, 128 * sum(counts))
    x = make(m, n, k, b_rows=1, seed=m + groups)
    offsets = (torch.tensor([0] + counts).cumsum(0) * 128).int().cuda()
    c = torch.full((groups, m, n + 3), 3.0, dtype=torch.float32, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"], ldc=n + 3, groups=groups,
                                                  group_dim=K.GROUP_TERMS, b_scale_rows=1, tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    for g in range(groups):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        if hi > lo:
            want = expect(x["a"][:, lo:hi], x["sa"][lo // 128: hi // 128], x["b"][:, lo:hi], x["sb"][lo // 128: hi // 128], 1)
            check(c[g, :, :n], *want, hi - lo, K.F32)
        else:
            assert (c[g, :, :n] == 0).all()
    assert (c[:, :, n:] == 3).all()


@pytest.mark.parametrize("tiles", TILES)
def test_groups_that_share_one_b(tiles):
    m, n, k, counts = 210, 136, 300, [3, 150, 0, 57]
    x = make(m, n, k, seed=3)
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    c = torch.empty((m, n), dtype=torch.float32, device="cuda")
    d = K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"], groups=4, stride_b=0, b_scale_group=0, tiles=tiles)
    plan = K.Plan("block_gemm", d)
    run(plan, x, c, offsets)
    plan.check()
    check(c, *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], 128), k, K.F32)


@pytest.mark.parametrize("out", [K.F16, K.BF16, K.F32])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("a, b", [(K.F8E5M2, K.F8E4M3), (K.F8E4M3, K.F8E5M2)])
@pytest.mark.parametrize("tiles", [0] + TILES)
def test_groups_of_rows_types_and_scales_of_each_row(tiles, a, b, b_rows, out):
    """Each group's scales of B: [blocks][n] or [n / 128][blocks], a set behind the other and, here, a gap behind each."""
    counts = [3, 0, 130, 257, 0, 1, 40]
    groups, m, n, k = len(counts), sum(counts), 200, 600
    x = make(m, n, k, a, b, b_rows, each=(groups,), seed=21)
    sets = x["sb"]
    wide = torch.full((groups, sets[0].numel() + 3), float("nan"), device="cuda")
    wide[:, :-3] = sets.reshape(groups, -1)
    x["sb"] = wide
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    c = torch.full((m, n), 3.0, dtype=TORCH_OF[out], device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(a, b, out, m, n, k, lda=x["ld"], ldb=x["ld"], groups=groups, b_scale_rows=b_rows,
                                                  b_scale_group=wide.shape[1], tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    at = 0
    for g, count in enumerate(counts):
        if count:
            rows = slice(at, at + count)
            check(c[rows], *expect(x["a"][rows, :k], x["sa"][:, rows], x["b"][g, :, :k], sets[g], b_rows), k, out)
        at += count


@pytest.mark.parametrize("out", [K.F16, K.BF16])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("a, b", [(K.F8E5M2, K.F8E4M3), (K.F8E5M2, K.F8E5M2)])
@pytest.mark.parametrize("tiles", [0] + TILES)
def test_groups_of_terms_types_and_scales_of_128_rows(tiles, a, b, b_rows, out):
    counts, m, n = [2, 0, 5, 1], 150, 330
    groups, k = len(counts), 128 * sum(counts)
    x = make(m, n, k, a, b, b_rows, seed=22)
    offsets = (torch.tensor([0] + counts).cumsum(0) * 128).int().cuda()
    c = torch.full((groups, m, n), 3.0, dtype=TORCH_OF[out], device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(a, b, out, m, n, k, groups=groups, group_dim=K.GROUP_TERMS, b_scale_rows=b_rows, tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    for g in range(groups):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        if hi > lo:
            blocks_of = slice(lo // 128, hi // 128)
            sb = x["sb"][blocks_of] if b_rows == 1 else x["sb"][:, blocks_of]
            check(c[g], *expect(x["a"][:, lo:hi], x["sa"][blocks_of], x["b"][:, lo:hi], sb, b_rows), hi - lo, out)
        else:
            assert (c[g] == 0).all()


@pytest.mark.parametrize("stride_c", [0, 4, -8, 1 << 39])
@pytest.mark.parametrize("tiles", [0] + TILES)
def test_one_group_of_terms_whatever_its_stride(tiles, stride_c):
    """A single group has no neighbour: the distance to it counts for nothing."""
    m, n, k, lo, hi = 200, 264, 640, 128, 512
    x = make(m, n, k, b_rows=1, seed=8)
    offsets = torch.tensor([lo, hi], dtype=torch.int32, device="cuda")
    c = torch.full((m, n), 3.0, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, groups=1, group_dim=K.GROUP_TERMS, b_scale_rows=1,
                                                  stride_c=stride_c, tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    check(c, *expect(x["a"][:, lo:hi], x["sa"][1:4], x["b"][:, lo:hi], x["sb"][1:4], 1), hi - lo, K.F32)


@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("tiles", TILES)
def test_groups_that_share_one_b_and_its_scales_by_default(tiles, b_rows):
    m, n, k, counts = 210, 136, 300, [3, 150, 0, 57]
    x = make(m, n, k, b_rows=b_rows, seed=6)
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    c = torch.empty((m, n), dtype=torch.float32, device="cuda")
    d = K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"], groups=4, stride_b=0, b_scale_rows=b_rows, tiles=tiles)
    plan = K.Plan("block_gemm", d)
    run(plan, x, c, offsets)
    plan.check()
    check(c, *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], b_rows), k, K.F32)


def again_and_again(plan, x, c, offsets=None, calls=40):
    """Calls into a matrix that is wiped before each: every one gives the bits of the first."""
    first, bad = c.clone(), torch.zeros((), dtype=torch.bool, device="cuda")
    for _ in range(calls):
        c.fill_(3.0)
        run(plan, x, c, offsets)
        bad |= (c != first).any()
    plan.check()
    assert not bad


@pytest.mark.parametrize("tiles", [K.BLOCK_TILES_SINGLE, K.BLOCK_TILES_PAIR])
@pytest.mark.parametrize("k", [100, 700])
@pytest.mark.parametrize("n", [45, 66, 93, 173, 207, 301, 335, 366])
@pytest.mark.parametrize("m", [1, 257, 20001])
def test_f32_rows_that_end_inside_a_box(m, n, k, tiles):
    """f32 results leave in boxes of 32 columns, in two places by turns: whole ones by TMA, one that ends inside 16 bytes by plain
    stores, those behind the last column not at all, on rows that start on 16 bytes all the same."""
    x = make(m, n, k, seed=n)
    ldc = (n + 3) // 4 * 4 + 4
    c = torch.full((m + 1, ldc), 3.0, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"], ldc=ldc, tiles=tiles))
    run(plan, x, c)
    plan.check()
    check(c[:m, :n], *expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], 128), k, K.F32)
    assert (c[:, n:] == 3).all() and (c[m] == 3).all()
    again_and_again(plan, x, c)


@pytest.mark.parametrize("tiles", [K.BLOCK_TILES_SINGLE, K.BLOCK_TILES_PAIR])
@pytest.mark.parametrize("n", [264, 512, 2048])
@pytest.mark.parametrize("whole", [128, 256])
def test_f32_groups_whose_tails_follow_whole_tiles(whole, n, tiles):
    """Boxes of whole tiles leave by TMA, those of a group's last rows by plain stores from the same places."""
    counts = [whole * (g % 3) + (11 * g) % 32 for g in range(96)]
    groups, m, k = len(counts), sum(counts), 128
    x = make(m, n, k, each=(groups,), seed=n)
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    c = torch.full((m, n), 3.0, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, groups=groups, tiles=tiles))
    run(plan, x, c, offsets)
    plan.check()
    at = 0
    for g, count in enumerate(counts):
        if count:
            rows = slice(at, at + count)
            check(c[rows], *expect(x["a"][rows], x["sa"][:, rows], x["b"][g], x["sb"][g], 128), k, K.F32)
        at += count
    again_and_again(plan, x, c, offsets)


def test_offsets_outside_the_rows_are_taken_as_the_edge():
    m, n, k = 40, 130, 256
    x = make(m, n, k, each=(4,), seed=2)
    offsets = torch.tensor([-7, 10, 5, 30, 1000], dtype=torch.int32, device="cuda")     # (10, 5): empty, and no row twice
    c = torch.full((m, n), 3.0, dtype=torch.float32, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k, groups=4))
    run(plan, x, c, offsets)
    plan.check()
    for g, lo, hi in ((0, 0, 10), (2, 10, 30), (3, 30, 40)):
        check(c[lo:hi], *expect(x["a"][lo:hi], x["sa"][:, lo:hi], x["b"][g], x["sb"][g], 128), k, K.F32)


@pytest.mark.parametrize("m", [2, 200])
def test_a_nan_and_an_infinity_stay_in_their_rows_and_columns(m):
    n, k = 256, 300
    x = make(m, n, k, K.F8E5M2, K.F8E4M3, seed=4)
    x["a"][1, 290] = float("nan")
    x["b"][77, 3] = float("nan")
    x["a"][0, 5] = float("inf")
    c = torch.empty((m, n), dtype=torch.float32, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E5M2, K.F8E4M3, K.F32, m, n, k, lda=x["ld"], ldb=x["ld"]))
    run(plan, x, c)
    plan.check()
    want, size = expect(x["a"][:, :k], x["sa"], x["b"][:, :k], x["sb"], 128)
    assert torch.equal(torch.isnan(c), torch.isnan(want)) and torch.equal(torch.isinf(c), torch.isinf(want))
    fine = torch.isfinite(want)
    check(c[fine], want[fine], size[fine], k, K.F32)


@pytest.mark.parametrize("m", [3, 300, 5000])
def test_calls_are_alike_on_streams_and_in_graphs(m):
    """One plan on two streams at once, captured and replayed with other inputs in the same place: bits of the plain call."""
    n, k = 512, 2048
    x, y = make(m, n, k, seed=1), make(m, n, k, seed=2)
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, m, n, k))
    cx, cy = (torch.empty((m, n), dtype=torch.float32, device="cuda") for _ in range(2))
    run(plan, x, cx)
    run(plan, y, cy)
    want_x, want_y = cx.clone(), cy.clone()
    cx.zero_(), cy.zero_()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        run(plan, x, cx, stream=s1.cuda_stream)
        run(plan, y, cy, stream=s2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(cx, want_x) and torch.equal(cy, want_y)
    g = torch.cuda.CUDAGraph()
    cx.zero_()
    with torch.cuda.graph(g):
        run(plan, x, cx, stream=torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cx, want_x)
    for name in ("a", "b", "sa", "sb"):
        x[name].view(torch.uint8).copy_(y[name].view(torch.uint8))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cx, want_y)
    plan.check()


def test_products_of_no_rows():
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.BF16, 0, 64, 64))
    plan.block_gemm(None, None, None, None, None)


def test_arguments_that_a_product_refuses():
    x = make(4, 64, 64)
    c = torch.empty((4, 64), dtype=torch.float32, device="cuda")
    plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, 4, 64, 64))
    at = [x["a"].data_ptr(), x["sa"].data_ptr(), x["b"].data_ptr(), x["sb"].data_ptr(), c.data_ptr()]
    for i in range(5):
        for bad in (None, at[i] + 1):
            with pytest.raises(K.KernelError) as e:
                plan.block_gemm(*at[:i], bad, *at[i + 1:])
            assert e.value.status == K.ERR_INVALID
    with pytest.raises(K.KernelError):
        plan.block_gemm(*at, offsets=x["sa"].data_ptr())        # no groups
    with pytest.raises(K.KernelError):
        K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.F32, 4, 64, 64, groups=1)).block_gemm(*at)
    with pytest.raises(K.KernelError):
        plan.quant(at[0], at[1], at[2])


# ---------------------------------------------------------------------------------------- quantisation


def to_8_bits(v, dtype):
    """f32 values rounded to the nearest 8-bit float (ties to even) and saturated, as f32: from the format, 3 or 2 bits of fraction."""
    fraction, low = (3, -6) if dtype == K.F8E4M3 else (2, -14)
    v = v.astype(np.float64)
    _, e = np.frexp(v)
    step = np.exp2(np.maximum(e - 1, low) - fraction)
    return np.clip(np.round(v / step) * step, -LARGEST[dtype], LARGEST[dtype]).astype(np.float32)


def quantised(x, dtype, tall, wide):
    """(q as f32, scales) of x [r, c] f32 in blocks of tall x wide, by f32 arithmetic."""
    r, c = x.shape
    nr, nc = -(-r // tall), -(-c // wide)
    size = np.abs(np.where(np.isnan(x), 0, x))
    full = np.zeros((nr * tall, nc * wide), np.float32)
    full[:r, :c] = size
    amax = full.reshape(nr, tall, nc, wide).max((1, 3))
    scale = np.maximum(amax, np.float32(2.0 ** -100)) / np.float32(LARGEST[dtype])
    inverse = np.float32(1) / scale
    with np.errstate(invalid="ignore"):
        v = x * inverse.repeat(tall, 0)[:r].repeat(wide, 1)[:, :c]
    return to_8_bits(v, dtype), scale


def host_values(rows, cols, dtype, seed):
    g = np.random.Generator(np.random.PCG64(seed))
    x = (g.standard_normal((rows, cols)) * np.exp2(g.integers(-10, 10, (rows, 1)))).astype(np.float32)
    x[g.random((rows, cols)) < 0.05] = 0
    return torch.from_numpy(x).to(TORCH_OF[dtype])


def form_of(q, form):
    return q.T if form in (K.QUANT_COLUMNS, K.QUANT_TILES_TRANSPOSED) else q


@pytest.mark.parametrize("out", [K.F8E4M3, K.F8E5M2])
@pytest.mark.parametrize("dtype", [K.BF16, K.F32, K.F16])
@pytest.mark.parametrize("form", range(4))
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 128), (5, 700), (128, 128), (129, 130), (257, 515), (300, 1028)])
def test_quantisation(rows, cols, form, dtype, out):
    host = host_values(rows, cols, dtype, rows + cols)
    turned, tiles = form in (K.QUANT_COLUMNS, K.QUANT_TILES_TRANSPOSED), form >= K.QUANT_TILES
    tall, wide = (128, 128) if tiles else ((128, 1) if turned else (1, 128))
    q, s = quantised(host.float().numpy(), out, tall, wide)
    r, c = (cols, rows) if turned else (rows, cols)
    ldq = (c + 15) // 16 * 16
    dev = host.cuda()
    got = torch.full((r, ldq), 0x5a, dtype=torch.uint8, device="cuda")
    scale = torch.full((blocks(r) if tiles else blocks(c), blocks(c) if tiles else r), -1.0, device="cuda")
    K.Plan("quant", K.quant_desc(dtype, out, rows, cols, form, ldq=ldq)).quant(dev.data_ptr(), got.data_ptr(), scale.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(scale.cpu().numpy(), s if form == K.QUANT_TILES else s.T if form != K.QUANT_COLUMNS else s)
    assert np.array_equal(got[:, :c].view(F8[out]).float().cpu().numpy(), form_of(q, form))
    assert (got[:, c:] == 0x5a).all()


@pytest.mark.parametrize("form", range(4))
def test_quantisation_in_place_strides_and_batches(form):
    """Batch entries, rows apart, an odd first element and odd strides of both matrices, scales in another order."""
    rows, cols, batch, ldx, ldq = 140, 133, 3, 141, 150
    host = torch.stack([host_values(rows, cols, K.BF16, 40 + b) for b in range(batch)])
    turned, tiles = form in (K.QUANT_COLUMNS, K.QUANT_TILES_TRANSPOSED), form >= K.QUANT_TILES
    tall, wide = (128, 128) if tiles else ((128, 1) if turned else (1, 128))
    r, c = (cols, rows) if turned else (rows, cols)
    x = torch.full((batch * (rows + 2) * ldx + 1,), 1e30, dtype=torch.bfloat16, device="cuda")
    view = x[1:].view(batch, rows + 2, ldx)
    view[:, :rows, :cols] = host.cuda()
    got = torch.full((batch * (r + 1) * ldq + 3,), 0x5a, dtype=torch.uint8, device="cuda")
    sr, sc = (blocks(r) if tiles else r), blocks(c)
    scale = torch.full((batch, sr, sc + 1), -1.0, device="cuda")
    d = K.quant_desc(K.BF16, K.F8E4M3, rows, cols, form, ldx=ldx, ldq=ldq, batch=batch, stride_x=(rows + 2) * ldx, stride_q=(r + 1) * ldq,
                     scale_row=sc + 1, scale_block=1, stride_scale=sr * (sc + 1))
    K.Plan("quant", d).quant(x.data_ptr() + 2, got.data_ptr() + 3, scale.data_ptr())
    torch.cuda.synchronize()
    out = got[3:].view(batch, r + 1, ldq)
    for b in range(batch):
        q, s = quantised(host[b].float().numpy(), K.F8E4M3, tall, wide)
        assert np.array_equal(scale[b, :, :sc].cpu().numpy(), form_of(s, form))
        assert np.array_equal(out[b, :r, :c].view(torch.float8_e4m3fn).float().cpu().numpy(), form_of(q, form))
    assert (out[:, r:] == 0x5a).all() and (out[:, :, c:] == 0x5a).all() and (scale[:, :, sc] == -1).all() and (got[:3] == 0x5a).all()


def test_quantisation_of_rows_by_index():
    sources, cols, div = 20, 300, 4
    host = host_values(sources, cols, K.BF16, 3)
    at = torch.tensor([5, 0, -1, 79, 80, 33, 33, -2147483648, 2147483647, 1], dtype=torch.int32)
    picked = torch.stack([host[i // div] if 0 <= i // div < sources else torch.zeros(cols, dtype=host.dtype) for i in at.tolist()])
    q, s = quantised(picked.float().numpy(), K.F8E4M3, 1, 128)
    dev, rows = host.cuda(), at.cuda()
    got = torch.empty((len(at), 304), dtype=torch.uint8, device="cuda")
    scale = torch.empty((3, len(at)), device="cuda")
    d = K.quant_desc(K.BF16, K.F8E4M3, len(at), cols, K.QUANT_ROWS, ldq=304, source_rows=sources, source_div=div)
    plan = K.Plan("quant", d)
    plan.quant(dev.data_ptr(), got.data_ptr(), scale.data_ptr(), rows=rows.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(scale.cpu().numpy(), s.T)
    assert np.array_equal(got[:, :cols].view(torch.float8_e4m3fn).float().cpu().numpy(), q)
    with pytest.raises(K.KernelError):
        plan.quant(dev.data_ptr(), got.data_ptr(), scale.data_ptr())


@pytest.mark.parametrize("form", range(4))
def test_quantisation_of_numbers_at_the_edges(form):
    """Zeros, subnormals, the largest numbers, ties, NaN (stays, does not count) and infinities (their block stands for NaN)."""
    x = np.zeros((256, 384), np.float32)
    x[0, :8] = [448, 447.9, 17, 19, 21, 232, 2.0 ** -10, 3 * 2.0 ** -10]      # ties between neighbours
    x[1, 128:132] = [1e-45, -1e-40, 2.0 ** -126, 0]
    x[2, 256:260] = [3.4028235e38, -3.4028235e38, 1, -0.0]
    x[130, 3:6] = [1, np.nan, -2]
    x[131, 200] = np.inf
    turned, tiles = form in (K.QUANT_COLUMNS, K.QUANT_TILES_TRANSPOSED), form >= K.QUANT_TILES
    tall, wide = (128, 128) if tiles else ((128, 1) if turned else (1, 128))
    q, s = quantised(x, K.F8E4M3, tall, wide)
    r, c = form_of(x, form).shape
    dev = torch.from_numpy(x).cuda()
    got = torch.empty((r, c), dtype=torch.uint8, device="cuda")
    scale = torch.empty((blocks(r) if tiles else r, blocks(c)), device="cuda")
    d = K.quant_desc(K.F32, K.F8E4M3, 256, 384, form, scale_row=blocks(c), scale_block=1)
    K.Plan("quant", d).quant(dev.data_ptr(), got.data_ptr(), scale.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(scale.cpu().numpy(), form_of(s, form), equal_nan=True)
    assert np.array_equal(got.view(torch.float8_e4m3fn).float().cpu().numpy(), form_of(q, form), equal_nan=True)
