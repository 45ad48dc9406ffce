"""Routing of tokens to experts, its gradient, the experts' order of rows, and the combination of the experts' rows, against
their definitions in 64 bits; and a whole layer of experts, forward and backward, as these operators are used together.

Tolerances.  u = 2^-24.  Routing weights are quotients of exponentials (two units of 2u each, and the rounding of the exponent:
less than u, relative to the largest), sums of at most 1024 of them in chains of 32 and a tree of 5, three more operations:
64 u of the weight.  The gradient adds a product sum over at most 32 choices, another 70 u of the sum of absolute
values.  Sums over rows: one u per term of the sum of absolute values.  Results in 16 bits: half a step more."""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from gpu_util import TORCH_OF
from plaidml_b200 import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {K.F32: U, K.BF16: 2.0 ** -8, K.F16: 2.0 ** -11}


def logits_of(tokens, experts, dtype, seed, ties=False):
    g = np.random.Generator(np.random.PCG64(seed))
    z = g.standard_normal((tokens, experts)).astype(np.float32) * 2
    if ties:
        z = np.round(z * 2) / 2
    return torch.from_numpy(z).to(TORCH_OF[dtype])


def score64(z, score):
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max)).astype(np.float64)
    if score == K.ROUTE_SIGMOID:
        with np.errstate(over="ignore"):
            return z, 1 / (1 + np.exp(-z))
    m = z.max(1, keepdims=True)
    e = np.where(np.isneginf(z), 0, np.exp(z - np.where(np.isneginf(m), 0, m)))
    total = e.sum(1, keepdims=True)
    return z, np.divide(e, total, out=np.zeros_like(e), where=total > 0)


def routed(z, bias, top_k, score, groups, top_groups, renormalise, scale):
    """(weights, ids) in 64 bits."""
    z, s = score64(z, score)
    rank = z.copy() if bias is None and groups == 1 else s + (0 if bias is None else bias.astype(np.float64))
    if groups > 1:
        inside = rank.reshape(len(rank), groups, -1)
        value = -np.sort(-inside, 2)[:, :, :2].sum(2)
        order = np.argsort(-value, 1, kind="stable")
        for t in range(len(rank)):
            for g in order[t, top_groups:]:
                inside[t, g] = -np.inf
    ids = np.argsort(-rank, 1, kind="stable")[:, :top_k]
    w = np.take_along_axis(s, ids, 1)
    if renormalise:
        if score == K.ROUTE_SOFTMAX:      # shares of the choice, also where the scores themselves underflow
            zc = np.take_along_axis(z, ids, 1)
            m = zc.max(1, keepdims=True)
            w = np.where(np.isneginf(zc), 0, np.exp(zc - np.where(np.isneginf(m), 0, m)))
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return w * scale, ids


def route(z, bias, top_k, score, groups=1, top_groups=1, renormalise=True, scale=1.0, dtype=K.F32, ld=None):
    tokens, experts = z.shape
    ld = ld or experts
    dev = torch.full((tokens, ld), 99.0, dtype=z.dtype, device="cuda")
    dev[:, :experts] = z.cuda()
    b = None if bias is None else torch.from_numpy(bias).cuda()
    w = torch.full((tokens, top_k), -1.0, device="cuda")
    ids = torch.full((tokens, top_k), -7, dtype=torch.int32, device="cuda")
    plan = K.Plan("route", K.route_desc(dtype, tokens, experts, top_k, score, ld=ld, groups=groups, top_groups=top_groups,
                                        renormalise=renormalise, scale=scale))
    plan.route(dev.data_ptr(), None if b is None else b.data_ptr(), w.data_ptr(), ids.data_ptr())
    torch.cuda.synchronize()
    return w.cpu().numpy().astype(np.float64), ids.cpu().numpy()


def check_route(z, bias, top_k, score, dtype=K.F32, **how):
    w, ids = route(z, bias, top_k, score, dtype=dtype, **how)
    how.pop("ld", None)
    want_w, want_ids = routed(z.float().numpy(), bias, top_k, score, how.get("groups", 1), how.get("top_groups", 1),
                              how.get("renormalise", True), how.get("scale", 1.0))
    assert np.array_equal(ids, want_ids)
    assert (np.abs(w - want_w) <= 64 * U * np.abs(want_w) + 1e-37).all()


SHAPES = [(1, 8, 2), (3, 1, 1), (7, 60, 4), (33, 64, 6), (130, 128, 8), (50, 160, 6), (65, 256, 8), (9, 384, 8), (10, 1024, 32), (5, 33, 32)]


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("tokens, experts, top_k", SHAPES)
def test_route(tokens, experts, top_k, with_bias, renormalise, score):
    z = logits_of(tokens, experts, K.F32, tokens * experts)
    bias = np.random.Generator(np.random.PCG64(1)).standard_normal(experts).astype(np.float32) * 0.05 if with_bias else None
    check_route(z, bias, top_k, score, renormalise=renormalise, scale=2.5, ld=experts + 3)


@pytest.mark.parametrize("dtype", [K.BF16, K.F16])
@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("experts, groups, top_groups, top_k", [(256, 8, 4, 8), (64, 4, 1, 3), (60, 4, 2, 5), (32, 32, 7, 7), (1024, 2, 1, 32), (16, 1, 1, 16)])
def test_route_by_groups(experts, groups, top_groups, top_k, score, dtype):
    for with_bias in (False, True):
        bias = np.random.Generator(np.random.PCG64(2)).standard_normal(experts).astype(np.float32) * 0.05 if with_bias else None
        check_route(logits_of(70, experts, dtype, experts), bias, top_k, score, groups=groups, top_groups=top_groups, dtype=dtype)


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("groups", [1, 4])
def test_equal_scores_go_to_the_lowest_index(score, groups):
    z = logits_of(200, 64, K.F32, 3, ties=True)
    z[7] = 0.25
    top = dict(groups=groups, top_groups=max(1, groups // 2))
    check_route(z, None, 8, score, **top)
    check_route(z, np.zeros(64, np.float32), 8, score, **top)
    check_route(z, np.full(64, -0.3, np.float32), 8, score, **top)


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("groups", [1, 8])
def test_scores_that_32_bits_cannot_tell_apart(score, groups):
    """Biases that nearly cancel what the scores differ by: the order is that of 64 bits."""
    g = np.random.Generator(np.random.PCG64(8))
    z = torch.from_numpy((1 + g.standard_normal((400, 64)) * 1e-7).astype(np.float32))
    bias = (g.integers(-3, 4, 64) * 2.0 ** -26).astype(np.float32)
    check_route(z, bias, 8, score, groups=groups, top_groups=max(1, groups // 2))
    one = torch.from_numpy(np.tile(g.standard_normal((400, 1)), (1, 64)).astype(np.float32))     # the bias alone decides, below 32 bits' step
    check_route(one, bias, 8, score, groups=groups, top_groups=max(1, groups // 2))


@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
def test_masked_and_extreme_logits(score, renormalise):
    z = logits_of(12, 64, K.F32, 9)
    z[0] = -np.inf                                # nothing left: the first experts, without weight
    z[1, 3:] = -np.inf                            # fewer left than choices
    z[2, 10] = np.inf
    z[3, 5] = np.nan
    z[4] = torch.finfo(torch.float32).min         # the lowest value as a mask
    z[4, 20] = 1.5
    z[5] = -200.0                                 # sigmoids of zero
    z[6] *= 100
    z[7] = torch.finfo(torch.float32).min
    z[8] = np.nan
    check_route(z, None, 6, score, renormalise=renormalise)
    w, ids = route(z, None, 6, score, renormalise=renormalise)
    assert (w[0] == 0).all() and list(ids[0]) == [0, 1, 2, 3, 4, 5] and (w[8] == 0).all() and (w[1, 3:] == 0).all()


def test_experts_that_a_bias_takes_out():
    z = logits_of(90, 64, K.F32, 10)
    bias = np.zeros(64, np.float32)
    bias[::3] = -np.inf
    bias[1] = np.nan
    b = np.where(np.isnan(bias), -np.inf, bias)
    w, ids = route(z, bias, 8, K.ROUTE_SIGMOID)
    want_w, want_ids = routed(z.numpy(), b, 8, K.ROUTE_SIGMOID, 1, 1, True, 1.0)
    assert np.array_equal(ids, want_ids) and (np.abs(w - want_w) <= 64 * U * want_w).all()


@pytest.mark.parametrize("score, renormalise", [(K.ROUTE_SOFTMAX, True), (K.ROUTE_SOFTMAX, False), (K.ROUTE_SIGMOID, True)])
@pytest.mark.parametrize("experts", [2, 3])
def test_weights_of_experts_far_below_the_first(experts, score, renormalise):
    """Small weights are as accurate as large ones.  An exponential is within one last place of the rounded one (3 u) and takes
    what its argument's rounding left out (2 u more); of sigmoids it is divided by a sum (3 u and u), and u for that: 10 u; the sum
    of two or three of them 10 u of a weighted mean, two u for additions, u for the quotient: 23 u."""
    g = np.random.Generator(np.random.PCG64(experts))
    first = -g.random((20000, 1)) * 3 - 0.1
    z = np.concatenate([first, first - g.random((20000, experts - 1)) * 80], 1).astype(np.float32)
    w, ids = route(torch.from_numpy(z), None, experts, score, renormalise=renormalise)
    want, want_ids = routed(z, None, experts, score, 1, 1, renormalise, 1.0)
    assert np.array_equal(ids, want_ids)
    assert (np.abs(w - want) <= 23 * U * want).all(), (np.abs(w - want) / want).max() / U


def routed_among_the_groups_that_stay(z, bias, top_k, score, groups, top_groups, renormalise=True):
    """(weights, ids) in 64 bits, each token's choice made among the experts of its groups alone."""
    _, s = score64(z, score)
    ids = np.empty((len(z), top_k), np.int64)
    rank = s + np.where(np.isnan(bias), -np.inf, bias.astype(np.float64))
    size = z.shape[1] // groups
    for t in range(len(z)):
        value = np.array([np.sort(rank[t, g * size: (g + 1) * size])[::-1][:2].sum() for g in range(groups)])
        stay = np.sort(np.argsort(-value, kind="stable")[:top_groups])
        among = np.concatenate([np.arange(g * size, (g + 1) * size) for g in stay])
        ids[t] = among[np.argsort(-rank[t, among], kind="stable")[:top_k]]
    w = np.take_along_axis(s, ids, 1)
    return (w / w.sum(1, keepdims=True) if renormalise else w), ids


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("out", [-np.inf, np.nan])
@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("experts, groups, top_groups, top_k", [(8, 2, 1, 4), (64, 4, 1, 16), (64, 8, 2, 12), (60, 4, 2, 28), (160, 4, 1, 32),
                                                                (256, 8, 1, 32), (32, 32, 5, 5), (1024, 16, 1, 32)])
def test_experts_that_a_bias_takes_out_make_no_room_for_other_groups(experts, groups, top_groups, top_k, near, out, score):
    """Fewer experts with a finite score than choices in the groups that stay: the others of these groups, not of the rest.
    `near`: scores that 32 bits cannot tell apart, so that the choice is made in 64."""
    g = np.random.Generator(np.random.PCG64(experts + top_k))
    z = (g.standard_normal((50, experts)) * (1e-7 if near else 2)).astype(np.float32)
    bias = (g.integers(-3, 4, experts) * 2.0 ** -26).astype(np.float32)
    size = experts // groups
    for e in range(groups):       # of each group at least one stays, and where it has them two, so that its value is finite
        at = e * size + g.permutation(size)
        bias[at[2 if size > 2 else size:][: (2 * size) // 3]] = out
    w, ids = route(torch.from_numpy(z), bias, top_k, score, groups=groups, top_groups=top_groups)
    want_w, want_ids = routed_among_the_groups_that_stay(z, bias, top_k, score, groups, top_groups)
    assert np.array_equal(ids, want_ids)
    assert (np.abs(w - want_w) <= 64 * U * want_w).all()


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("tokens", [5, 100])
def test_a_group_that_a_bias_takes_out_whole(tokens, score):
    """All experts of the groups that stay are taken out (no group has a finite value): the first groups', in their order."""
    experts, groups, top_groups, top_k = 64, 4, 2, 20
    z = logits_of(tokens, experts, K.F32, 12)
    w, ids = route(z, np.full(experts, -np.inf, np.float32), top_k, score, groups=groups, top_groups=top_groups)
    want_w, want_ids = routed_among_the_groups_that_stay(z.numpy(), np.full(experts, -np.inf, np.float32), top_k, score, groups, top_groups)
    assert np.array_equal(ids, want_ids) and (ids == np.arange(top_k)).all()
    assert (np.abs(w - want_w) <= 64 * U * want_w).all()
    bias = np.zeros(experts, np.float32)
    bias[:16] = -np.inf            # the first group's: it never stays
    w, ids = route(z, bias, top_k, score, groups=groups, top_groups=3)
    _, want_ids = routed_among_the_groups_that_stay(z.numpy(), bias, top_k, score, groups, 3)
    assert np.array_equal(ids, want_ids) and (ids >= 16).all()


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("experts, groups", [(16, 4), (60, 4), (256, 8), (15, 5)])
def test_groups_whose_values_32_bits_cannot_hold(experts, groups, score):
    """Biases of the largest numbers, as masks have them: the sum of two is infinite in 32 bits, but not in 64."""
    low, high, size = np.finfo(np.float32).min, np.finfo(np.float32).max, experts // groups
    z = logits_of(40, experts, K.F32, 13)
    rising = (high * (0.55 + 0.4 * np.arange(experts) / experts)).astype(np.float32)     # all sums of two are infinite in 32 bits
    for first, others in ((-np.inf, low), (high / 2, high), (high * 0.75, high), (None, None)):
        bias = np.zeros(experts, np.float32)
        bias[:size], bias[size: (groups - 1) * size] = first or 0, others or 0
        if first is None:
            bias = rising
        for top_groups in (1, 2, 3):
            top_k = min(32, top_groups * size - 1)
            w, ids = route(z, bias, top_k, score, groups=groups, top_groups=top_groups)
            want_w, want_ids = routed_among_the_groups_that_stay(z.numpy(), bias, top_k, score, groups, top_groups)
            assert np.array_equal(ids, want_ids)
            assert (np.abs(w - want_w) <= 64 * U * want_w).all()


# ---------------------------------------------------------------------------------------- gradient


def grad64(z, ids, dw, score, renormalise, scale):
    """The formulas, and the sums of the absolute values of their terms."""
    z64, s = score64(z, score)
    there = (ids >= 0) & (ids < z.shape[1])
    at = np.where(there, ids, 0)
    g = np.where(there, dw.astype(np.float64) * scale, 0)
    sc = np.where(there, np.take_along_axis(s, at, 1), 0)
    if renormalise:
        if score == K.ROUTE_SOFTMAX:
            zc = np.where(there, np.take_along_axis(z64, at, 1), -np.inf)
            m = zc.max(1, keepdims=True)
            sc = np.where(np.isneginf(zc), 0, np.exp(zc - np.where(np.isneginf(m), 0, m)))
        total = sc.sum(1, keepdims=True)
        sc = np.divide(sc, total, out=np.zeros_like(sc), where=total > 0)
    dot, size = (g * sc).sum(1, keepdims=True), np.abs(g * sc).sum(1, keepdims=True)
    out, tol = np.zeros(z.shape), np.zeros(z.shape)
    rest = 1 - np.take_along_axis(s, at, 1) if score == K.ROUTE_SIGMOID else 1.0
    if not renormalise and score == K.ROUTE_SIGMOID:
        dot, size = 0 * dot, 0 * size
    if not renormalise and score == K.ROUTE_SOFTMAX:
        out, tol = -s * dot, s * size
    for t, j in zip(*np.nonzero(there)):
        r = rest if np.isscalar(rest) else rest[t, j]
        out[t, ids[t, j]] = sc[t, j] * r * (g[t, j] - dot[t, 0])
        tol[t, ids[t, j]] = sc[t, j] * r * (abs(g[t, j]) + size[t, 0])
    return out, tol


@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("tokens, experts, top_k", SHAPES)
def test_route_grad(tokens, experts, top_k, renormalise, score, dtype):
    z = logits_of(tokens, experts, dtype, tokens + experts)
    if tokens > 5:
        z[3, 1:] = -np.inf
        z[4] = -np.inf
    _, ids = route(z, None, top_k, score, renormalise=renormalise, dtype=dtype)
    if tokens > 5:
        ids[2, 0], ids[5, top_k - 1] = -1, experts
    g = np.random.Generator(np.random.PCG64(4))
    dw = g.standard_normal((tokens, top_k)).astype(np.float32)
    ld = experts + 5
    dev = torch.full((tokens, ld), 99.0, dtype=TORCH_OF[dtype], device="cuda")
    dev[:, :experts] = z.cuda()
    dz = torch.full((tokens, ld), 3.0, dtype=TORCH_OF[dtype], device="cuda")
    plan = K.Plan("route", K.route_desc(dtype, tokens, experts, top_k, score, ld=ld, renormalise=renormalise, scale=2.5))
    di, dd = torch.from_numpy(ids).cuda(), torch.from_numpy(dw).cuda()
    plan.route_grad(dev.data_ptr(), di.data_ptr(), dd.data_ptr(), dz.data_ptr())
    torch.cuda.synchronize()
    want, size = grad64(z.float().numpy(), ids, dw, score, renormalise, 2.5)
    got = dz[:, :experts].double().cpu().numpy()
    assert (np.abs(got - want) <= 140 * U * size + HALF_STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == K.F16 else 1e-37)).all()
    assert (dz[:, experts:] == 3).all()


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_grad_is_the_slope_of_the_weights(score, renormalise):
    """Central differences of the 64-bit weights at a fixed choice: a step of 1e-5 leaves 1e-9 of curvature and 1e-11 of rounding."""
    tokens, experts, top_k = 6, 24, 4
    z = logits_of(tokens, experts, K.F32, 6).numpy()
    g = np.random.Generator(np.random.PCG64(5))
    dw = g.standard_normal((tokens, top_k)).astype(np.float32)
    _, ids = routed(z, None, top_k, score, 1, 1, renormalise, 1.5)

    def value(v):
        _, s = score64(v, score)
        w = np.take_along_axis(s, ids, 1)
        return ((w / w.sum(1, keepdims=True) if renormalise else w) * 1.5 * dw).sum(1)

    slope = np.zeros_like(z, np.float64)
    for e in range(experts):
        up, down = z.astype(np.float64), z.astype(np.float64)
        up[:, e] += 1e-5
        down[:, e] -= 1e-5
        slope[:, e] = (value(up) - value(down)) / 2e-5
    dev, di, dd = torch.from_numpy(z).cuda(), torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(dw).cuda()
    dz = torch.empty((tokens, experts), device="cuda")
    K.Plan("route", K.route_desc(K.F32, tokens, experts, top_k, score, renormalise=renormalise, scale=1.5)).route_grad(
        dev.data_ptr(), di.data_ptr(), dd.data_ptr(), dz.data_ptr())
    torch.cuda.synchronize()
    assert np.abs(dz.cpu().numpy() - slope).max() < 1e-5


# ---------------------------------------------------------------------------------------- order


def ordered(ids, experts, align, rows):
    offsets, source, position = [0], np.full(rows, -1, np.int32), np.full(ids.shape, -1, np.int32)
    flat, at = ids.reshape(-1), 0
    for e in range(experts):
        pairs = np.nonzero(flat == e)[0]
        source[at: at + len(pairs)] = pairs
        position.reshape(-1)[pairs] = at + np.arange(len(pairs))
        at += -(-len(pairs) // align) * align
        offsets.append(at)
    return np.array(offsets, np.int32), source, position


def check_order(ids, experts, align, spare=0, stream=None):
    tokens, top_k = ids.shape
    rows = K.route_rows(tokens, experts, top_k, align) // align * align + spare
    dev = torch.from_numpy(ids.astype(np.int32)).cuda()
    offsets, source, position = (torch.full(s, -9, dtype=torch.int32, device="cuda") for s in ((experts + 1,), (max(rows, 1),), (tokens, top_k)))
    plan = K.Plan("route", K.route_desc(K.F32, tokens, experts, top_k, K.ROUTE_SOFTMAX, rows=rows, align=align))
    plan.route_order(dev.data_ptr(), offsets.data_ptr(), source.data_ptr(), position.data_ptr())
    torch.cuda.synchronize()
    want = ordered(ids, experts, align, rows)
    for got, w in zip((offsets, source[:rows], position), want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("align", [1, 16, 128, 1000])
@pytest.mark.parametrize("tokens, experts, top_k", [(1, 8, 1), (1, 64, 6), (5, 3, 2), (31, 60, 4), (600, 128, 8), (3000, 256, 8), (10001, 1024, 3), (700, 32, 32)])
def test_order(tokens, experts, top_k, align):
    g = np.random.Generator(np.random.PCG64(tokens))
    ids = np.argsort(g.random((tokens, experts)) * (1 + np.arange(experts) % 7), 1)[:, :top_k]
    check_order(ids, experts, align, spare=align * 2 + 5)


@pytest.mark.parametrize("experts, top_k", [(64, 8), (700, 6)])
def test_order_of_more_pairs_than_fit_in_registers(experts, top_k):
    g = np.random.Generator(np.random.PCG64(experts))
    ids = g.integers(-1, experts, (60000, top_k))
    check_order(ids, experts, 1)
    check_order(ids, experts, 128, spare=77)


@pytest.mark.parametrize("tokens", [10, 5000])
def test_order_of_a_padded_batch(tokens):
    """Pairs without an expert have no row; all of one expert; none at all."""
    g = np.random.Generator(np.random.PCG64(tokens))
    ids = g.integers(-2, 40, (tokens, 4))
    ids[tokens // 2:] = -1
    ids[0, 0], ids[1, 1] = 2147483647, -2147483648
    check_order(ids, 37, 8)
    check_order(np.full((tokens, 4), 36), 37, 8)
    check_order(np.full((tokens, 4), -1), 37, 8, spare=3)
    check_order(np.zeros((tokens, 1), int), 1, 1)


def test_order_without_tokens():
    offsets, source = torch.full((9,), -9, dtype=torch.int32, device="cuda"), torch.full((6,), -9, dtype=torch.int32, device="cuda")
    w = torch.empty(1, device="cuda")
    plan = K.Plan("route", K.route_desc(K.F32, 0, 8, 2, K.ROUTE_SOFTMAX, rows=6))
    plan.route(None, None, None, None, offsets.data_ptr(), source.data_ptr(), None)
    torch.cuda.synchronize()
    assert (offsets == 0).all() and (source == -1).all()
    with pytest.raises(K.KernelError):
        plan.route(None, None, None, None, None, source.data_ptr(), None)
    with pytest.raises(K.KernelError):
        K.Plan("route", K.route_desc(K.F32, 4, 8, 2, K.ROUTE_SOFTMAX)).route_order(w.data_ptr(), w.data_ptr(), w.data_ptr(), w.data_ptr())


@pytest.mark.parametrize("score", [K.ROUTE_SOFTMAX, K.ROUTE_SIGMOID])
@pytest.mark.parametrize("experts, groups, top_groups, top_k", [(160, 4, 2, 6), (60, 4, 1, 5), (250, 5, 3, 8), (96, 32, 7, 8), (9, 3, 2, 4)])
@pytest.mark.parametrize("tokens", [1, 33, 64, 65])
def test_few_tokens_chosen_in_64_bits_by_groups_of_any_size(tokens, experts, groups, top_groups, top_k, score):
    """Choice and order of few tokens (one launch up to 64), groups that are no runs of whole lanes, scores that 32 bits cannot tell apart."""
    g = np.random.Generator(np.random.PCG64(experts))
    z = (1 + g.standard_normal((tokens, experts)) * 1e-7).astype(np.float32)
    z[::3] = g.standard_normal((len(z[::3]), experts))
    bias = (g.integers(-3, 4, experts) * 2.0 ** -26).astype(np.float32)
    rows = K.route_rows(tokens, experts, top_k, 8)
    dev, b = torch.from_numpy(z).cuda(), torch.from_numpy(bias).cuda()
    w, ids = torch.full((tokens, top_k), -1.0, device="cuda"), torch.full((tokens, top_k), -7, dtype=torch.int32, device="cuda")
    offsets, source, position = (torch.full(s, -9, dtype=torch.int32, device="cuda") for s in ((experts + 1,), (rows,), (tokens, top_k)))
    plan = K.Plan("route", K.route_desc(K.F32, tokens, experts, top_k, score, groups=groups, top_groups=top_groups, rows=rows, align=8))
    plan.route(dev.data_ptr(), b.data_ptr(), w.data_ptr(), ids.data_ptr(), offsets.data_ptr(), source.data_ptr(), position.data_ptr())
    torch.cuda.synchronize()
    want_w, want_ids = routed(z, bias, top_k, score, groups, top_groups, True, 1.0)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(w.cpu().numpy() - want_w) <= 64 * U * want_w).all()
    for got, want in zip((offsets, source, position), ordered(want_ids, experts, 8, rows)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("align", [0, -5, 1 << 30])
def test_order_without_tokens_and_rows(align):
    """Nothing to put in order: the offsets alone, whatever the alignment of rows that there are not."""
    offsets = torch.full((10,), -9, dtype=torch.int32, device="cuda")
    plan = K.Plan("route", K.route_desc(K.F32, 0, 8, 2, K.ROUTE_SOFTMAX, rows=0, align=align))
    plan.route_order(None, offsets.data_ptr(), None, None)
    torch.cuda.synchronize()
    assert offsets.tolist() == [0] * 9 + [-9]


@pytest.mark.parametrize("tokens", [6, 2000])
def test_routing_in_streams_and_graphs(tokens):
    """Two graphs of one plan, replayed at the same time: each gives what the plain call gives."""
    experts, top_k, rows = 64, 6, K.route_rows(tokens, 64, 6, 128)
    plan = K.Plan("route", K.route_desc(K.F32, tokens, experts, top_k, K.ROUTE_SIGMOID, groups=8, top_groups=4, rows=rows, align=128))

    def fresh(seed):
        return {"z": logits_of(tokens, experts, K.F32, seed).cuda(), "w": torch.zeros((tokens, top_k), device="cuda"),
                "ids": torch.zeros((tokens, top_k), dtype=torch.int32, device="cuda"),
                "offsets": torch.zeros(experts + 1, dtype=torch.int32, device="cuda"),
                "source": torch.zeros(rows, dtype=torch.int32, device="cuda"),
                "position": torch.zeros((tokens, top_k), dtype=torch.int32, device="cuda")}

    def call(x, stream=0):
        plan.route(x["z"].data_ptr(), None, x["w"].data_ptr(), x["ids"].data_ptr(), x["offsets"].data_ptr(), x["source"].data_ptr(),
                   x["position"].data_ptr(), stream=stream)

    sets = [fresh(s) for s in (1, 2)]
    want = []
    for x in sets:
        call(x)
        want.append({k: v.clone() for k, v in x.items()})
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(x, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        for k in ("w", "ids", "offsets", "source", "position"):
            x[k].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, y in zip(sets, want):
        assert all(torch.equal(x[k], y[k]) for k in x)


FIRST_CALL = """
import torch
from plaidml_b200 import kernels as K
z, w, ids = torch.randn((TOKENS, 64), device="cuda"), torch.zeros((TOKENS, 4), device="cuda"), torch.zeros((TOKENS, 4), dtype=torch.int32, device="cuda")
offsets, source, position = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (65, 4 * TOKENS, 4 * TOKENS))
x, y = (torch.randn((4 * TOKENS, 256), device="cuda").bfloat16() for _ in range(2))
q = torch.zeros((4 * TOKENS, 256), dtype=torch.uint8, device="cuda")
s, sb = torch.ones((2, 4 * TOKENS), device="cuda"), torch.ones((64, 2, 2), device="cuda")
b = torch.zeros((64, 256, 256), dtype=torch.uint8, device="cuda")
c, out = torch.zeros((4 * TOKENS, 256), dtype=torch.bfloat16, device="cuda"), torch.zeros((TOKENS, 256), dtype=torch.bfloat16, device="cuda")
dz, dw, dy = torch.zeros_like(z), torch.zeros_like(w), torch.zeros_like(x)

def all_of_it(stream):
    plans = [K.Plan("route", K.route_desc(K.F32, TOKENS, 64, 4, K.ROUTE_SOFTMAX, rows=4 * TOKENS)),
             K.Plan("quant", K.quant_desc(K.BF16, K.F8E4M3, 4 * TOKENS, 256, K.QUANT_ROWS)),
             K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, K.BF16, 4 * TOKENS, 256, 256, groups=64)),
             K.Plan("combine", K.combine_desc(K.BF16, TOKENS, 4, 256, 4 * TOKENS))]
    at = [t.data_ptr() for t in (z, w, ids, offsets, source, position)]
    plans[0].route(at[0], None, *at[1:], stream=stream)
    plans[1].quant(x.data_ptr(), q.data_ptr(), s.data_ptr(), stream=stream)
    plans[2].block_gemm(q.data_ptr(), s.data_ptr(), b.data_ptr(), sb.data_ptr(), c.data_ptr(), offsets=at[3], stream=stream)
    plans[3].combine(y.data_ptr(), at[1], at[5], out.data_ptr(), stream=stream)
    plans[3].combine_grad(out.data_ptr(), y.data_ptr(), at[1], at[5], at[4], dy.data_ptr(), dw.data_ptr(), stream=stream)
    plans[0].route_grad(at[0], at[2], dw.data_ptr(), dz.data_ptr(), stream=stream)
    return plans

results = (w, ids, offsets, source, position, q, s, c, out, dy, dw, dz)
b.copy_(torch.randint(0, 100, b.shape, dtype=torch.uint8, device="cuda"))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    plans = all_of_it(torch.cuda.current_stream().cuda_stream)
del plans
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in results]
for t in results:
    t.zero_()
plans = all_of_it(0)
torch.cuda.synchronize()
assert all(torch.equal(a, t) for a, t in zip(got, results)) and float(out.abs().max()) > 0
print("alike")
"""


@pytest.mark.parametrize("tokens", [8, 1000])
def test_plans_made_and_called_for_the_first_time_under_capture(tokens):
    """In a process of its own: nothing of the library has run on the device before the capture, and the plans are gone before the replay."""
    done = subprocess.run([sys.executable, "-c", FIRST_CALL.replace("TOKENS", str(tokens))], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0 and "alike" in done.stdout, done.stderr[-2000:]


# ---------------------------------------------------------------------------------------- combination


@pytest.mark.parametrize("dtype", [K.BF16, K.F32, K.F16])
@pytest.mark.parametrize("tokens, top_k, width, spare", [(1, 1, 1, 0), (1, 8, 2048, 0), (7, 2, 130, 3), (40, 6, 1000, 200), (33, 5, 4100, 1), (3, 32, 64, 0)])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(tokens, top_k, width, spare, dtype, weighted):
    g = np.random.Generator(np.random.PCG64(tokens * width))
    rows = tokens * top_k + spare
    source = np.full(rows, -1, np.int32)
    place = g.permutation(rows)[: tokens * top_k]
    source[place] = np.arange(tokens * top_k)
    position = place.astype(np.int32).reshape(tokens, top_k).copy()
    if tokens > 2:                                   # pairs without a row
        for t, j, v in ((0, 0, -1), (2, top_k - 1, rows)):
            source[position[t, j]] = -1 if v < 0 else tokens * top_k
            position[t, j] = v
    ldy, ldo = width + 8, width + 16
    y = torch.from_numpy(g.standard_normal((rows, ldy)).astype(np.float32)).to(TORCH_OF[dtype])
    dout = torch.from_numpy(g.standard_normal((tokens, ldo)).astype(np.float32)).to(TORCH_OF[dtype])
    w = g.standard_normal((tokens, top_k)).astype(np.float32)
    y64, d64 = y.double().numpy()[:, :width], dout.double().numpy()[:, :width]
    w64 = w.astype(np.float64) if weighted else np.ones(w.shape)
    there = (position >= 0) & (position < rows)
    picked = np.where(there[:, :, None], y64[np.where(there, position, 0)], 0)
    dev = {k: torch.from_numpy(v).cuda() for k, v in (("w", w), ("position", position), ("source", source))}
    dy, dd = y.cuda(), dout.cuda()
    out = torch.full((tokens + 1, ldo), 3.0, dtype=TORCH_OF[dtype], device="cuda")
    plan = K.Plan("combine", K.combine_desc(dtype, tokens, top_k, width, rows, ldy=ldy, ldo=ldo))
    weights = dev["w"].data_ptr() if weighted else None
    plan.combine(dy.data_ptr(), weights, dev["position"].data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    want, size = (picked * w64[:, :, None]).sum(1), np.abs(picked * w64[:, :, None]).sum(1)
    tiny = 2.0 ** -25 if dtype == K.F16 else 1e-37
    assert (np.abs(out[:tokens, :width].double().cpu().numpy() - want) <= top_k * U * size + HALF_STEP[dtype] * np.abs(want) + tiny).all()
    assert (out[:, width:] == 3).all() and (out[tokens] == 3).all()

    want_dy = np.zeros((rows, width))
    for t in range(tokens):
        for j in range(top_k):
            if there[t, j]:
                want_dy[position[t, j]] = w64[t, j] * d64[t]
    want_dw, size_dw = (picked * d64[:, None]).sum(2), np.abs(picked * d64[:, None]).sum(2)
    for ask_y, ask_w in ((True, True), (True, False), (False, True)):
        gy = torch.full((rows + 1, ldy), 3.0, dtype=TORCH_OF[dtype], device="cuda")
        gw = torch.full((tokens, top_k), 3.0, device="cuda")
        plan.combine_grad(dd.data_ptr(), dy.data_ptr() if ask_w else None, weights, dev["position"].data_ptr(),
                          dev["source"].data_ptr() if ask_y else None, gy.data_ptr() if ask_y else None, gw.data_ptr() if ask_w else None)
        torch.cuda.synchronize()
        if ask_y:
            assert (np.abs(gy[:rows, :width].double().cpu().numpy() - want_dy) <= (U + HALF_STEP[dtype]) * np.abs(want_dy) + tiny).all()
            assert (gy[:, width:] == 3).all() and (gy[rows] == 3).all()
        else:
            assert (gy == 3).all()
        if ask_w:
            assert (np.abs(gw.double().cpu().numpy() - want_dw) <= width * U * size_dw + 1e-37).all()
        else:
            assert (gw == 3).all()


def test_combine_of_nothing_and_refusals():
    x = torch.zeros(64, device="cuda")
    at = x.data_ptr()
    out = torch.full((3, 8), 5.0, device="cuda")
    position = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    K.Plan("combine", K.combine_desc(K.F32, 0, 2, 8, 6)).combine(None, None, None, None)
    K.Plan("combine", K.combine_desc(K.F32, 3, 2, 8, 0)).combine(None, None, position.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert (out == 0).all()
    gy, source = torch.full((4, 8), 5.0, device="cuda"), torch.full((4,), -1, dtype=torch.int32, device="cuda")
    K.Plan("combine", K.combine_desc(K.F32, 0, 2, 8, 4)).combine_grad(None, None, None, None, source.data_ptr(), gy.data_ptr(), None)
    torch.cuda.synchronize()
    assert (gy == 0).all()
    plan = K.Plan("combine", K.combine_desc(K.F32, 3, 2, 8, 6))
    for bad in ((None, at, at, at), (at, at, None, at), (at, at, at, None), (at + 2, at, at, at), (at, at + 1, at, at)):
        with pytest.raises(K.KernelError) as e:
            plan.combine(*bad)
        assert e.value.status == K.ERR_INVALID
    for bad in ((at, at, at, at, at, None, None), (None, at, at, at, at, at, at), (at, None, at, at, at, at, at), (at, at, at, at, None, at, at)):
        with pytest.raises(K.KernelError) as e:
            plan.combine_grad(*bad)
        assert e.value.status == K.ERR_INVALID


# ---------------------------------------------------------------------------------------- all of it


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_a_layer_of_experts_forward_and_backward(tokens):
    """Routing, rows gathered and quantised, the experts' products, their rows combined; then every gradient: of the routing
    weights and logits, of the rows (products with the transposed weights, gathered back) and of the weights (products over
    the terms of each expert).  Each operator gets what the one before it gave, and is compared with its own definition on that."""
    experts, top_k, width, inner, align = 8, 2, 256, 384, 128
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rows = K.route_rows(tokens, experts, top_k, align) // align * align
    x = torch.randn((tokens, width), device="cuda", generator=g).bfloat16()
    z = torch.randn((tokens, experts), device="cuda", generator=g)
    w = (torch.randn((experts, inner, width), device="cuda", generator=g) * width ** -0.5).bfloat16()
    i32, f32 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.float32, device="cuda")

    def quantise(t, r, c, form, batch=1, source=None, div=1, sources=0):
        turned, tiles = form in (K.QUANT_COLUMNS, K.QUANT_TILES_TRANSPOSED), form >= K.QUANT_TILES
        qr, qc = (c, r) if turned else (r, c)
        q = torch.zeros((batch, qr, qc), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        s = torch.zeros((batch, qr // 128, qc // 128) if tiles else (batch, (qc + 127) // 128, qr), **f32)
        K.Plan("quant", K.quant_desc(K.BF16, K.F8E4M3, r, c, form, batch=batch, source_rows=sources, source_div=div)).quant(
            t.data_ptr(), q.data_ptr(), s.data_ptr(), rows=None if source is None else source.data_ptr())
        v = s.repeat_interleave(128, 1).repeat_interleave(128, 2) if tiles else s.transpose(1, 2).repeat_interleave(128, 2)[:, :, :qc]
        return q, s, q.double() * v.double()

    def product(a, b, m, n, k, offsets, dim=K.GROUP_ROWS, b_rows=128, out=K.BF16):
        shape = (experts, m, n) if dim == K.GROUP_TERMS else (m, n)
        c = torch.full(shape, 0.0, dtype=TORCH_OF[out], device="cuda")
        plan = K.Plan("block_gemm", K.block_gemm_desc(K.F8E4M3, K.F8E4M3, out, m, n, k, groups=experts, group_dim=dim, b_scale_rows=b_rows))
        plan.block_gemm(a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), c.data_ptr(), offsets=offsets.data_ptr())
        plan.check()
        return c

    def close(got, want, size, steps, dtype):
        assert ((got.double() - want).abs() <= steps * 2 * U * size + HALF_STEP[dtype] * want.abs() + 1e-30).all()

    weights, ids = torch.empty((tokens, top_k), **f32), torch.empty((tokens, top_k), **i32)
    offsets, source, position = torch.empty(experts + 1, **i32), torch.empty(rows, **i32), torch.empty((tokens, top_k), **i32)
    router = K.Plan("route", K.route_desc(K.F32, tokens, experts, top_k, K.ROUTE_SOFTMAX, rows=rows, align=align))
    router.route(z.data_ptr(), None, weights.data_ptr(), ids.data_ptr(), offsets.data_ptr(), source.data_ptr(), position.data_ptr())
    want_w, want_ids = routed(z.cpu().numpy(), None, top_k, K.ROUTE_SOFTMAX, 1, 1, True, 1.0)
    assert np.array_equal(ids.cpu().numpy(), want_ids) and np.allclose(weights.cpu().numpy(), want_w, rtol=64 * U, atol=0)
    for got, want in zip((offsets, source, position), ordered(want_ids, experts, align, rows)):
        assert np.array_equal(got.cpu().numpy(), want)
    o = offsets.tolist()

    xq = quantise(x, rows, width, K.QUANT_ROWS, source=source, div=top_k, sources=tokens)
    wq = quantise(w, inner, width, K.QUANT_TILES, batch=experts)
    y = product(xq, wq, rows, inner, width, offsets)
    for e in range(experts):
        a, b = xq[2][0, o[e]: o[e + 1]], wq[2][e]
        close(y[o[e]: o[e + 1]], a @ b.t(), a.abs() @ b.abs().t(), 140, K.BF16)
    out = torch.empty((tokens, inner), dtype=torch.bfloat16, device="cuda")
    mix = K.Plan("combine", K.combine_desc(K.BF16, tokens, top_k, inner, rows))
    mix.combine(y.data_ptr(), weights.data_ptr(), position.data_ptr(), out.data_ptr())
    terms = y.double()[position.long()] * weights.double()[:, :, None]
    close(out, terms.sum(1), terms.abs().sum(1), top_k, K.BF16)

    dout = torch.randn((tokens, inner), device="cuda", generator=g).bfloat16()
    dy, dweights, dz = torch.empty((rows, inner), dtype=torch.bfloat16, device="cuda"), torch.empty((tokens, top_k), **f32), torch.empty_like(z)
    mix.combine_grad(dout.data_ptr(), y.data_ptr(), weights.data_ptr(), position.data_ptr(), source.data_ptr(), dy.data_ptr(), dweights.data_ptr())
    there = (source >= 0)[:, None]
    pair = source.clamp(min=0).long()
    close(dy, torch.where(there, dout.double()[pair // top_k] * weights.double().reshape(-1)[pair][:, None], 0.0), torch.zeros_like(dy).double(), 0, K.BF16)
    router.route_grad(z.data_ptr(), ids.data_ptr(), dweights.data_ptr(), dz.data_ptr())
    want, size = grad64(z.cpu().numpy(), ids.cpu().numpy(), dweights.cpu().numpy(), K.ROUTE_SOFTMAX, True, 1.0)
    assert (np.abs(dz.cpu().numpy() - want) <= 140 * U * size + U * np.abs(want)).all()

    # rows: dx = dy * W, with the transposed weights; a token's rows add up
    dyq, wt = quantise(dy, rows, inner, K.QUANT_ROWS), quantise(w, inner, width, K.QUANT_TILES_TRANSPOSED, batch=experts)
    drows = product(dyq, wt, rows, width, inner, offsets)
    for e in range(experts):
        a, b = dyq[2][0, o[e]: o[e + 1]], wt[2][e]
        close(drows[o[e]: o[e + 1]], a @ b.t(), a.abs() @ b.abs().t(), 140, K.BF16)
    dx = torch.empty_like(x)
    K.Plan("combine", K.combine_desc(K.BF16, tokens, top_k, width, rows)).combine(drows.data_ptr(), None, position.data_ptr(), dx.data_ptr())
    back = drows.double()[position.long()]
    close(dx, back.sum(1), back.abs().sum(1), top_k, K.BF16)

    # weights: dW[e] = dy^T * x over the expert's rows
    gathered = torch.where(there, x[pair // top_k], 0.0).contiguous()
    dyt, xt = quantise(dy, rows, inner, K.QUANT_COLUMNS), quantise(gathered, rows, width, K.QUANT_COLUMNS)
    dw = product(dyt, xt, inner, width, rows, offsets, dim=K.GROUP_TERMS, b_rows=1, out=K.F32)
    for e in range(experts):
        a, b = dyt[2][0][:, o[e]: o[e + 1]], xt[2][0][:, o[e]: o[e + 1]]
        close(dw[e], a @ b.t(), a.abs() @ b.abs().t(), 130 + rows // 128, K.F32)
