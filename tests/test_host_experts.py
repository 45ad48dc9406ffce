"""Descriptors that block products, quantisation, routing and combination refuse, and the helpers that fill them in.  Every
refusal is made from the descriptor alone, before a device is looked for."""

import pytest

from plaidml_b200 import kernels as K


def problem(kind, desc):
    """The message that the library refuses `desc` with (None: it does not; without a device it says so)."""
    try:
        K.Plan(kind, desc)
    except K.KernelError as e:
        if e.status == K.ERR_UNSUPPORTED and ("no CUDA device" in str(e) or "compute capability" in str(e)):
            return None
        assert e.status == K.ERR_INVALID
        return str(e)
    return None


def changed(desc, **fields):
    for name, value in fields.items():
        setattr(desc, name, value)
    return desc


def product(**fields):
    return changed(K.block_gemm_desc(K.F8E4M3, K.F8E5M2, K.BF16, 100, 200, 256), **fields)


@pytest.mark.parametrize("fields, word", [
    (dict(a_dtype=K.BF16), "8-bit"), (dict(b_dtype=K.I8), "8-bit"), (dict(out_dtype=K.I32), "result"), (dict(m=-1), "positive"),
    (dict(n=0), "positive"), (dict(k=0), "positive"), (dict(lda=255), "smaller"), (dict(ldb=240), "smaller"), (dict(ldc=199), "smaller"),
    (dict(lda=264), "multiples of 16"), (dict(ldb=257), "multiples of 16"), (dict(groups=1025), "groups"), (dict(groups=-1), "groups"),
    (dict(groups=4, group_dim=2), "dimension"), (dict(groups=4, stride_b=200 * 256 + 8), "multiple of 16"),
    (dict(groups=4, stride_b=256), "overlap"), (dict(groups=4, group_dim=K.GROUP_TERMS, stride_c=200), "overlap"),
    (dict(b_scale_rows=64), "scale"), (dict(a_scale_row=-1), "negative"), (dict(b_scale_group=-4), "negative"),
    (dict(m=(1 << 30) + 1), "2^30"), (dict(tiles=4), "tiles"), (dict(tiles=-1), "tiles"),
])
def test_products_that_are_refused(fields, word):
    assert word in problem("block_gemm", product(**fields))


def test_products_that_are_taken():
    assert problem("block_gemm", product()) is None
    assert problem("block_gemm", product(m=0)) is None
    assert problem("block_gemm", product(groups=1024, group_dim=K.GROUP_TERMS)) is None
    assert problem("block_gemm", product(groups=3, stride_b=0)) is None       # one B for all groups


def quant(**fields):
    return changed(K.quant_desc(K.BF16, K.F8E4M3, 300, 200, fields.pop("form", K.QUANT_ROWS), batch=fields.pop("batch", 1)), **fields)


@pytest.mark.parametrize("fields, word", [
    (dict(in_dtype=K.I8), "input"), (dict(out_dtype=K.F16), "8-bit"), (dict(form=4), "form"), (dict(rows=-1), "positive"),
    (dict(cols=0), "positive"), (dict(batch=0), "positive"), (dict(ldx=199), "smaller"), (dict(ldq=199), "smaller"),
    (dict(form=K.QUANT_COLUMNS, ldq=299), "smaller"), (dict(scale_row=-1), "negative"), (dict(batch=2, stride_x=-1), "negative"),
    (dict(form=K.QUANT_TILES, source_rows=4, source_div=1), "index"), (dict(batch=2, source_rows=4, source_div=1), "index"),
    (dict(source_rows=4, source_div=0), "source_div"), (dict(source_rows=-4), "source_rows"), (dict(batch=65536), "launch"),
])
def test_quantisations_that_are_refused(fields, word):
    assert word in problem("quant", quant(**fields))


def test_quantisations_that_are_taken():
    for form in range(4):
        assert problem("quant", quant(form=form)) is None
    assert problem("quant", quant(rows=0)) is None
    assert problem("quant", quant(source_rows=7, source_div=8)) is None


def route(**fields):
    return changed(K.route_desc(K.F32, 100, 64, 8, K.ROUTE_SIGMOID, groups=8, top_groups=4, rows=2048, align=16), **fields)


@pytest.mark.parametrize("fields, word", [
    (dict(dtype=K.I32), "logits"), (dict(tokens=-1), "positive"), (dict(experts=0), "positive"), (dict(top_k=0), "positive"),
    (dict(experts=1032, groups=8, ld=1032), "1024"), (dict(top_k=33), "32"), (dict(experts=66), "divide"), (dict(groups=0), "divide"),
    (dict(top_groups=9), "top_groups"), (dict(top_groups=0), "top_groups"), (dict(top_groups=1, top_k=9), "choose"), (dict(ld=63), "smaller"),
    (dict(score=2), "score"), (dict(scale=float("inf")), "finite"), (dict(tokens=(1 << 21) + 1), "2^24"), (dict(align=0), "align"),
    (dict(align=1025), "align"), (dict(rows=1743), "fewer rows"), (dict(rows=-1), "negative"),
])
def test_routings_that_are_refused(fields, word):
    assert word in problem("route", route(**fields))


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, float("nan")])
def test_scales_of_weights_that_f32_cannot_hold_are_refused(scale):
    assert "finite" in problem("route", route(scale=scale))


def test_the_largest_scale_of_weights_is_taken():
    assert problem("route", route(scale=3.4028234e38)) is None
    assert problem("route", route(scale=-3.4028234e38)) is None and problem("route", route(scale=0.0)) is None


def test_routings_that_are_taken():
    assert problem("route", route()) is None
    assert problem("route", route(rows=K.route_rows(100, 64, 8, 16) // 16 * 16)) is None
    assert problem("route", route(rows=0, align=0)) is None
    assert problem("route", route(tokens=0)) is None


def combine(**fields):
    return changed(K.combine_desc(K.BF16, 10, 4, 64, 40), **fields)


@pytest.mark.parametrize("fields, word", [
    (dict(dtype=K.I8), "rows"), (dict(tokens=-1), "positive"), (dict(top_k=0), "positive"), (dict(width=0), "positive"),
    (dict(rows=-1), "negative"), (dict(ldy=63), "smaller"), (dict(ldo=63), "smaller"), (dict(tokens=1 << 29), "2^30"),
])
def test_combinations_that_are_refused(fields, word):
    assert word in problem("combine", combine(**fields))


def test_combinations_that_are_taken():
    assert problem("combine", combine()) is None
    assert problem("combine", combine(tokens=0, rows=0)) is None


def test_defaults_of_the_helpers_fit_one_another():
    rows = K.quant_desc(K.BF16, K.F8E4M3, 300, 520, K.QUANT_ROWS)
    columns = K.quant_desc(K.BF16, K.F8E4M3, 300, 520, K.QUANT_COLUMNS)
    tiles = K.quant_desc(K.BF16, K.F8E4M3, 700, 520, K.QUANT_TILES)
    p = K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.BF16, 300, 700, 520, lda=528, ldb=528)
    assert (rows.scale_row, rows.scale_block) == (p.a_scale_row, p.a_scale_block) == (1, 300)
    assert (tiles.scale_row, tiles.scale_block) == (p.b_scale_row, p.b_scale_block) == (5, 1)
    assert (columns.scale_row, columns.scale_block, columns.ldq) == (1, 520, 300)
    assert K.route_rows(10, 64, 4, 128) == 40 + 40 * 127


@pytest.mark.parametrize("b_scale_rows", [1, 128])
def test_groups_that_share_one_b_share_its_scales(b_scale_rows):
    def desc(**how):
        return K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.BF16, 300, 700, 512, groups=4, b_scale_rows=b_scale_rows, **how)

    whole = 700 * 4 if b_scale_rows == 1 else 6 * 4
    assert desc(stride_b=0).b_scale_group == 0
    assert desc().b_scale_group == whole and desc(stride_b=700 * 512 + 16).b_scale_group == whole
    assert desc(stride_b=0, b_scale_group=5).b_scale_group == 5


def test_null_arguments():
    lib = K.load()
    for kind in ("block_gemm", "quant", "route", "combine"):
        assert getattr(lib, f"pmlb_{kind}_dispatch")(None, None) == K.ERR_INVALID
    assert lib.pmlb_block_gemm_invoke(*[None] * 8) == K.ERR_INVALID
    assert lib.pmlb_quant_invoke(*[None] * 6) == K.ERR_INVALID
    assert lib.pmlb_route_invoke(*[None] * 9) == K.ERR_INVALID
    assert lib.pmlb_route_order(*[None] * 6) == K.ERR_INVALID
    assert lib.pmlb_route_grad(*[None] * 6) == K.ERR_INVALID
    assert lib.pmlb_combine_invoke(*[None] * 6) == K.ERR_INVALID
    assert lib.pmlb_combine_grad(*[None] * 9) == K.ERR_INVALID
