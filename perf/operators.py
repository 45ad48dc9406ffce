"""Cases that the speed of the operators of sparse language models is measured on: products of 8-bit floats with a scale for
each block of 128 terms (dense, by groups of rows, by groups of terms), the quantisation that makes their operands, the
routing of tokens to experts with its gradient, and the combination of the experts' rows with its gradient.

Each case runs in its plain form (elementary torch operations) or, where ``own`` is true, through the kernel C ABI
(``plaidml_b200.kernels.Plan``) as a user's program calls it.  ``kind`` names the operator:

  product    C = sum over blocks of scale_a * scale_b * (A * B^T)          (``Plan("block_gemm")``)
  quant      values in 8 bits and the scales of their blocks               (``Plan("quant")``)
  route      weights and experts of each token, the experts' order of rows (``Plan("route")``)
  unroute    the gradient of the routing weights to the logits             (``Plan("route")``)
  combine    weighted sum of each token's rows                             (``Plan("combine")``)
  uncombine  its gradients to the rows and to the weights                  (``Plan("combine")``)
"""

import functools
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
         "e5m2": torch.float8_e5m2}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "e5m2": 1}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
BLOCK = 128


def _product(m, n, k, a="e4m3", out="bf16", groups=0, by="none", b_rows=128):
    return {"kind": "product", "m": m, "n": n, "k": k, "a": a, "out": out, "groups": groups, "by": by, "b_rows": b_rows}


def _quant(rows, cols, form, dtype="bf16", to="e4m3", batch=1, div=0):
    return {"kind": "quant", "rows": rows, "cols": cols, "form": form, "dtype": dtype, "to": to, "batch": batch, "div": div}


def _route(tokens, experts, top_k, score, dtype="f32", groups=1, top_groups=1, bias=False, renormalise=True, align=1, kind="route"):
    return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "dtype": dtype, "groups": groups,
            "top_groups": top_groups, "bias": bias, "renormalise": renormalise, "align": align}


def _combine(tokens, top_k, width, dtype="bf16", align=1, kind="combine"):
    return {"kind": kind, "tokens": tokens, "top_k": top_k, "width": width, "dtype": dtype, "align": align}


def listed():
    return [
        # a dense layer over a batch of 4096 tokens
        {"name": "product_4096", **_product(4096, 4096, 4096)},
        # the same layer for one token: reads the weights once
        {"name": "product_one_token", **_product(1, 4096, 4096)},
        # a dense layer's weight gradient: both operands scaled along an odd number of tokens, f32 sums
        {"name": "product_weight_gradient", **_product(4096, 2048, 8190, a="e5m2", out="f32", b_rows=1)},
        # experts' products over a long batch: 4096 tokens to 8 of 64 experts, groups of uneven lengths
        {"name": "experts_long", **_product(32768, 2048, 2048, groups=64, by="rows")},
        # experts' products while tokens are generated: 16 tokens to 8 of 128 experts, most groups of a row or two
        {"name": "experts_few", **_product(128, 2048, 2048, groups=128, by="rows")},
        # activations before a product
        {"name": "quant_rows", **_quant(8192, 4096, "rows")},
        # gradients before a weight gradient: blocks along the tokens, the result transposed; an odd number of tokens
        {"name": "quant_columns", **_quant(8190, 2048, "columns", to="e5m2")},
        # routing of a long batch by sigmoid scores with a balance bias and expert groups
        {"name": "route_long", **_route(16384, 256, 8, "sigmoid", groups=8, top_groups=4, bias=True)},
        # routing while tokens are generated
        {"name": "route_few", **_route(8, 64, 6, "softmax", dtype="bf16", renormalise=False)},
        # the routing's gradient over a long batch
        {"name": "unroute_long", **_route(16384, 128, 8, "softmax", renormalise=False, kind="unroute")},
        # the experts' rows back to their tokens
        {"name": "combine_long", **_combine(8192, 8, 2048)},
        # gradients of that, segments padded as a weight gradient wants them
        {"name": "uncombine_long", **_combine(4096, 8, 2048, align=128, kind="uncombine")},
    ]


def _log(rng, lo, hi, multiple=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(multiple, (v + multiple // 2) // multiple * multiple)


def draw(rng):
    kind = rng.choice(["product", "product", "experts", "experts", "quant", "route", "unroute", "combine", "uncombine"])
    if kind == "product":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192, rng.choice([1, 8, 64])), _log(rng, 64, 8192, rng.choice([1, 16, 128]))
        while m * n * k > 4096 ** 3:
            m = (m + 1) // 2
        return _product(m, n, k, a=rng.choice(["e4m3", "e4m3", "e5m2"]), out=rng.choice(["bf16", "bf16", "f16", "f32"]),
                        b_rows=rng.choice([128, 128, 1]))
    if kind == "experts":
        groups, n, k = rng.choice([8, 16, 60, 64, 128]), _log(rng, 128, 2048, 8), _log(rng, 128, 2048, 8)
        if rng.random() < 0.25:
            return _product(_log(rng, 128, 2048), n, _log(rng, 512, 8192, 128), out="f32", groups=min(groups, 16), by="terms", b_rows=1)
        return _product(_log(rng, 1, 16384), n, k, out=rng.choice(["bf16", "bf16", "f32"]), groups=groups, by="rows")
    if kind == "quant":
        form = rng.choice(["rows", "rows", "columns", "tiles", "tiles_transposed"])
        rows, cols, batch = _log(rng, 1, 16384), _log(rng, 64, 8192, rng.choice([1, 8, 128])), 1
        while rows * cols > 8192 * 4096:
            rows = (rows + 1) // 2
        if "tiles" in form and rng.random() < 0.5:
            batch = rng.choice([2, 8])
            rows = max(1, rows // batch)
        div = rng.choice([1, 8]) if form == "rows" and rng.random() < 0.4 else 0
        return _quant(rows, cols, form, dtype=rng.choice(["bf16", "f16", "f32"]), to=rng.choice(["e4m3", "e4m3", "e5m2"]),
                      batch=batch, div=div)
    if kind in ("route", "unroute"):
        experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 384])
        groups = rng.choice([1, 4, 8]) if experts % 32 == 0 and kind == "route" else 1
        top_k = rng.choice([1, 2, 4, 6, 8])
        return _route(_log(rng, 1, 16384), experts, top_k, rng.choice(["softmax", "sigmoid"]), dtype=rng.choice(["f32", "bf16"]),
                      groups=groups, top_groups=max(1, groups // 2), bias=rng.random() < 0.5, renormalise=rng.random() < 0.6,
                      align=rng.choice([1, 128]), kind=kind)
    tokens, top_k, width = _log(rng, 1, 16384), rng.choice([1, 2, 4, 6, 8]), _log(rng, 128, 7168, rng.choice([1, 8, 64]))
    while tokens * top_k * width > 4096 * 8 * 2048:
        tokens = (tokens + 1) // 2
    return _combine(tokens, top_k, width, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), align=rng.choice([1, 128]), kind=kind)


# ---------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _bits(shape, dtype, g):
    """8-bit values of unit variance at half of the type's range below the largest, as quantised activations have."""
    x = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=g)
    return (x * (LARGEST[dtype] / 5)).clamp_(-LARGEST[dtype], LARGEST[dtype]).to(TORCH[dtype])


def _scales(shape, dtype, g, size=1.0):
    """The scales that blocks of values of about `size` have: their largest value, between three and five, over the type's."""
    return (torch.rand(shape, dtype=torch.float32, device="cuda", generator=g) * 2 + 3) * (size / LARGEST[dtype])


def _counts(case, seed):
    """Uneven lengths of the groups, the same for every caller: shares that fall off, in an order that the seed gives."""
    groups, total = case["groups"], case["m"] if case["by"] == "rows" else case["k"] // BLOCK
    g = torch.Generator().manual_seed(int(seed))
    share = torch.rand(groups, generator=g).add_(0.15)
    at = torch.multinomial(share, total, replacement=True, generator=g)
    counts = torch.bincount(at, minlength=groups)
    return counts if case["by"] == "rows" else counts * BLOCK


def _placed(tokens, top_k, align, seed):
    """Positions of the (token, choice) pairs among the experts' rows and the pairs of the rows: 64 experts' segments, each
    padded to a multiple of `align`."""
    experts, g = 64, torch.Generator().manual_seed(int(seed))
    ids = torch.rand(tokens, experts, generator=g).topk(top_k, 1).indices.reshape(-1)
    counts = torch.bincount(ids, minlength=experts)
    padded = (counts + align - 1) // align * align
    start = torch.cumsum(padded, 0) - padded
    order = torch.sort(ids, stable=True).indices
    inside = torch.arange(len(ids)) - (torch.cumsum(counts, 0) - counts)[ids[order]]
    row = start[ids[order]] + inside
    rows = _rows(tokens * top_k, experts, align)
    source = torch.full((rows,), -1, dtype=torch.int32)
    source[row] = order.int()
    position = torch.empty(tokens * top_k, dtype=torch.int32)
    position[order] = row.int()
    return source.cuda(), position.view(tokens, top_k).cuda(), rows


def _rows(pairs, experts, align):
    """Rows that `pairs` pairs take at most when each of the experts' segments is padded to a multiple of `align`."""
    return pairs if align == 1 else (pairs + min(experts, pairs) * (align - 1)) // align * align


def prepare(case, seed):
    kind, g = case["kind"], _generator(10 * seed + 1)
    s = {"case": case, "plan": {}}
    if kind == "product":
        m, n, k, groups = case["m"], case["n"], case["k"], case["groups"]
        ld = (k + 15) // 16 * 16  # rows of 8-bit matrices start on 16 bytes
        by_rows = groups and case["by"] == "rows"
        each = (groups,) if by_rows else ()
        s["a"], s["b"] = _bits((m, ld), case["a"], g), _bits(each + (n, ld), "e4m3", g)
        s["a_scale"] = _scales((_blocks(k), m), case["a"], g)
        s["b_scale"] = _scales(each + ((_blocks(n), _blocks(k)) if case["b_rows"] == BLOCK else (_blocks(k), n)), "e4m3", g, k ** -0.5)
        each = (groups,) if groups and case["by"] == "terms" else ()
        s["c"] = torch.zeros(each + (m, n), dtype=TORCH[case["out"]], device="cuda")
        s["offsets"] = None
        if groups:
            counts = _counts(case, seed)
            s["most"] = int(counts.max())
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]).int().cuda()
    elif kind == "quant":
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        sources = max(1, rows // case["div"]) if case["div"] else rows
        x = torch.randn((batch, sources, cols), dtype=torch.float32, device="cuda", generator=g)
        x *= torch.exp(torch.randn((batch, sources, 1), dtype=torch.float32, device="cuda", generator=g))  # rows of unlike sizes
        s["x"] = x.to(TORCH[case["dtype"]])
        s["rows"] = None
        if case["div"]:  # rows in the experts' order: pairs of a token and a choice
            s["rows"] = torch.randint(0, sources * case["div"], (rows,), dtype=torch.int32, device="cuda", generator=g)
        out = (batch, cols, rows) if case["form"] in ("columns", "tiles_transposed") else (batch, rows, cols)
        ld = (out[2] + 15) // 16 * 16
        s["q"] = torch.zeros((out[0], out[1], ld), dtype=torch.uint8, device="cuda").view(TORCH[case["to"]])
        shape = (_blocks(out[1]), _blocks(out[2])) if "tiles" in case["form"] else (_blocks(out[2]), out[1])
        s["scale"] = torch.zeros((batch,) + shape, dtype=torch.float32, device="cuda")
    elif kind in ("route", "unroute"):
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        s["logits"] = (torch.randn((t, e), dtype=torch.float32, device="cuda", generator=g) * 1.5).to(TORCH[case["dtype"]])
        s["bias"] = torch.randn((e,), dtype=torch.float32, device="cuda", generator=g) * 0.02 if case["bias"] else None
        if kind == "unroute":
            s["ids"] = _choose(s["logits"], s["bias"], case)[1]
            s["dweights"] = torch.randn((t, k), dtype=torch.float32, device="cuda", generator=g)
            s["dlogits"] = torch.empty((t, e), dtype=TORCH[case["dtype"]], device="cuda")
        else:
            s["capacity"] = _rows(t * k, e, case["align"])
            s["weights"] = torch.empty((t, k), dtype=torch.float32, device="cuda")
            s["ids"], s["position"] = (torch.empty((t, k), dtype=torch.int32, device="cuda") for _ in range(2))
            s["offsets"] = torch.empty((e + 1,), dtype=torch.int32, device="cuda")
            s["source"] = torch.empty((s["capacity"],), dtype=torch.int32, device="cuda")
    else:
        t, k, w, dt = case["tokens"], case["top_k"], case["width"], TORCH[case["dtype"]]
        s["source"], s["position"], s["rows"] = _placed(t, k, case["align"], seed)
        s["y"] = torch.randn((s["rows"], w), dtype=dt, device="cuda", generator=g)
        s["weights"] = torch.rand((t, k), dtype=torch.float32, device="cuda", generator=g)
        s["weights"] /= s["weights"].sum(1, keepdim=True)
        if kind == "combine":
            s["out"] = torch.empty((t, w), dtype=dt, device="cuda")
        else:
            s["dout"] = torch.randn((t, w), dtype=dt, device="cuda", generator=g)
            s["dy"] = torch.empty((s["rows"], w), dtype=dt, device="cuda")
            s["dweights"] = torch.empty((t, k), dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------- plain forms


def _spread(scale, n):
    """[..., blocks] -> [..., n]: each block's scale at each of its terms."""
    return scale.repeat_interleave(BLOCK, -1)[..., :n]


def _dense(s, number):
    """Both operands of a product as the values they stand for, [m, k] and [(groups,) n, k]."""
    case = s["case"]
    k, n = case["k"], case["n"]
    a = s["a"][:, :k].to(number) * _spread(s["a_scale"].t(), k).to(number)
    sb = s["b_scale"].transpose(-1, -2) if case["b_rows"] == 1 else s["b_scale"].repeat_interleave(BLOCK, -2)[..., :n, :]
    return a, s["b"][..., :k].to(number) * _spread(sb, k).to(number)


def _plain_product(s):
    case = s["case"]
    a, b = _dense(s, torch.float32)
    dt = TORCH[case["out"]]
    if not case["groups"]:
        return (a @ b.t()).to(dt)
    # groups of unequal lengths side by side, each padded with zeros to the longest one
    along = torch.arange(case["m"] if case["by"] == "rows" else int(case["k"]), device="cuda")
    group = torch.searchsorted(s["offsets"][1:].long(), along, right=True)
    inside = along - s["offsets"].long()[group]
    if case["by"] == "rows":
        wide = a.new_zeros(case["groups"], s["most"], case["k"])
        wide[group, inside] = a
        return (wide @ b.transpose(1, 2))[group, inside].to(dt)
    wa, wb = a.new_zeros(case["groups"], s["most"], case["m"]), a.new_zeros(case["groups"], s["most"], case["n"])
    wa[group, inside], wb[group, inside] = a.t(), b.t()
    return (wa.transpose(1, 2) @ wb).to(dt)


def _by_blocks(x, number):
    """x [batch, r, c] padded with zeros to whole blocks of columns, as [batch, r, blocks, 128]."""
    b, r, c = x.shape
    return torch.nn.functional.pad(x.to(number), (0, _blocks(c) * BLOCK - c)).view(b, r, _blocks(c), BLOCK)


def _plain_quant(s):
    case, top = s["case"], LARGEST[s["case"]["to"]]
    x = s["x"]
    if s["rows"] is not None:
        x = x[:, (s["rows"] // case["div"]).long()]
    if case["form"] in ("columns", "tiles_transposed"):
        x = x.transpose(1, 2)
    v = _by_blocks(x, torch.float32)
    most = v.abs().amax(3)
    if "tiles" in case["form"]:
        most = _by_blocks(most.transpose(1, 2), torch.float32).amax(3).transpose(1, 2)  # [batch, row blocks, column blocks]
    scale = most.clamp(min=2.0 ** -100) / top
    inverse = 1.0 / scale
    if "tiles" in case["form"]:
        inverse = inverse.repeat_interleave(BLOCK, 1)[:, : v.shape[1]]
    q = (v * inverse[..., None]).clamp(-top, top).to(TORCH[case["to"]])
    q = q.view(v.shape[0], v.shape[1], -1)[:, :, : x.shape[2]]
    return [q.contiguous(), (scale if "tiles" in case["form"] else scale.transpose(1, 2)).contiguous()]


def _score(logits, case, number):
    z = logits.to(number)
    if case["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    z = torch.exp(z - z.amax(1, keepdim=True))
    return z / z.sum(1, keepdim=True)


def _choose(logits, bias, case):
    """Scores and the chosen experts of each token, in 64 bits: what is chosen hangs on which of two near values is larger."""
    score = _score(logits, case, torch.float64)
    if case["groups"] > 1:
        rank = score if bias is None else score + bias
        inside = rank.view(len(rank), case["groups"], -1)
        best = inside.sort(dim=2, descending=True, stable=True).values[:, :, :2].sum(2)
        stay = best.sort(dim=1, descending=True, stable=True).indices[:, : case["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, stay, True)
        rank = inside.masked_fill(~kept[:, :, None], -math.inf).reshape(rank.shape)
    else:
        rank = logits.double() if bias is None else score + bias
    return score, rank.sort(dim=1, descending=True, stable=True).indices[:, : case["top_k"]].int()


SCALE = 2.5  # what the routing weights are multiplied by


def _plain_route(s):
    case = s["case"]
    score, ids = _choose(s["logits"], s["bias"], case)
    w = score.gather(1, ids.long())
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    flat, experts = ids.reshape(-1).long(), case["experts"]
    counts = torch.zeros(experts, dtype=torch.int64, device="cuda").scatter_add_(0, flat, torch.ones_like(flat))
    padded = (counts + case["align"] - 1) // case["align"] * case["align"]
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    offsets, before = torch.cat([zero, torch.cumsum(padded, 0)]), torch.cat([zero, torch.cumsum(counts, 0)])
    order = torch.sort(flat, stable=True).indices
    row = offsets[flat[order]] + torch.arange(len(flat), device="cuda") - before[flat[order]]
    source = torch.full((s["capacity"],), -1, dtype=torch.int32, device="cuda")
    source[row] = order.int()
    position = torch.empty(len(flat), dtype=torch.int32, device="cuda")
    position[order] = row.int()
    return [(w * SCALE).float(), ids, offsets.int(), source, position.view(ids.shape)]


def _plain_unroute(s):
    case = s["case"]
    score, ids = _score(s["logits"], case, torch.float32), s["ids"].long()
    chosen, dw = score.gather(1, ids), s["dweights"] * SCALE
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True)
        dw = (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(score).scatter_(1, ids, dw)
    if case["score"] == "sigmoid":
        return (ds * score * (1 - score)).to(TORCH[case["dtype"]])
    return (score * (ds - (dw * chosen).sum(1, keepdim=True))).to(TORCH[case["dtype"]])


def _plain_combine(s):
    rows = s["y"][s["position"].reshape(-1).long()].float().view(*s["position"].shape, -1)
    return (rows * s["weights"][:, :, None]).sum(1).to(s["y"].dtype)


def _plain_uncombine(s):
    k, at = s["position"].shape[1], s["position"].reshape(-1).long()
    dout = s["dout"].float()
    dweights = (s["y"][at].float().view(-1, k, dout.shape[1]) * dout[:, None]).sum(2)
    there = (s["source"] >= 0)[:, None]
    pair = s["source"].clamp(min=0).long()
    dy = torch.where(there, dout[pair // k] * s["weights"].reshape(-1)[pair][:, None], 0.0)
    return [dy.to(s["dout"].dtype), dweights]


# ---------------------------------------------------------------------------------------- the framework's calls


def _kept(s, make):
    """The plan that a user's program makes once for a layer of these sizes."""
    plan = s["plan"].get("it")
    if plan is None:
        from plaidml_b200 import kernels
        code = {"f32": kernels.F32, "bf16": kernels.BF16, "f16": kernels.F16, "e4m3": kernels.F8E4M3, "e5m2": kernels.F8E5M2}
        plan = s["plan"]["it"] = make(kernels, code, s["case"])
    return plan


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _at(t):
    return None if t is None else t.data_ptr()


def _make_product(K, code, c):
    ld = (c["k"] + 15) // 16 * 16
    return K.Plan("block_gemm", K.block_gemm_desc(
        code[c["a"]], code["e4m3"], code[c["out"]], c["m"], c["n"], c["k"], lda=ld, ldb=ld, groups=c["groups"],
        group_dim=K.GROUP_TERMS if c["by"] == "terms" else K.GROUP_ROWS, b_scale_rows=c["b_rows"]))


def _own_product(s):
    _kept(s, _make_product).block_gemm(_at(s["a"]), _at(s["a_scale"]), _at(s["b"]), _at(s["b_scale"]), _at(s["c"]),
                                       offsets=_at(s["offsets"]), stream=_stream())
    return s["c"]


def _make_quant(K, code, c):
    form = {"rows": K.QUANT_ROWS, "columns": K.QUANT_COLUMNS, "tiles": K.QUANT_TILES, "tiles_transposed": K.QUANT_TILES_TRANSPOSED}
    across = c["rows"] if c["form"] in ("columns", "tiles_transposed") else c["cols"]
    return K.Plan("quant", K.quant_desc(
        code[c["dtype"]], code[c["to"]], c["rows"], c["cols"], form[c["form"]], ldq=(across + 15) // 16 * 16, batch=c["batch"],
        source_rows=max(1, c["rows"] // c["div"]) if c["div"] else 0, source_div=max(1, c["div"])))


def _own_quant(s):
    c = s["case"]
    _kept(s, _make_quant).quant(_at(s["x"]), _at(s["q"]), _at(s["scale"]), rows=_at(s["rows"]), stream=_stream())
    return [s["q"][:, :, : c["rows"] if c["form"] in ("columns", "tiles_transposed") else c["cols"]], s["scale"]]


def _make_route(K, code, c):
    return K.Plan("route", K.route_desc(
        code[c["dtype"]], c["tokens"], c["experts"], c["top_k"], K.ROUTE_SIGMOID if c["score"] == "sigmoid" else K.ROUTE_SOFTMAX,
        groups=c["groups"], top_groups=c["top_groups"], renormalise=c["renormalise"], scale=SCALE,
        rows=_rows(c["tokens"] * c["top_k"], c["experts"], c["align"]), align=c["align"]))


def _own_route(s):
    _kept(s, _make_route).route(_at(s["logits"]), _at(s["bias"]), _at(s["weights"]), _at(s["ids"]), offsets=_at(s["offsets"]),
                                source=_at(s["source"]), position=_at(s["position"]), stream=_stream())
    return [s["weights"], s["ids"], s["offsets"], s["source"], s["position"]]


def _own_unroute(s):
    _kept(s, _make_route).route_grad(_at(s["logits"]), _at(s["ids"]), _at(s["dweights"]), _at(s["dlogits"]), stream=_stream())
    return s["dlogits"]


def _make_combine(K, code, c):
    return K.Plan("combine", K.combine_desc(code[c["dtype"]], c["tokens"], c["top_k"], c["width"],
                                            _rows(c["tokens"] * c["top_k"], 64, c["align"])))


def _own_combine(s):
    _kept(s, _make_combine).combine(_at(s["y"]), _at(s["weights"]), _at(s["position"]), _at(s["out"]), stream=_stream())
    return s["out"]


def _own_uncombine(s):
    _kept(s, _make_combine).combine_grad(_at(s["dout"]), _at(s["y"]), _at(s["weights"]), _at(s["position"]), _at(s["source"]),
                                         _at(s["dy"]), _at(s["dweights"]), stream=_stream())
    return [s["dy"], s["dweights"]]


PLAIN = {"product": _plain_product, "quant": _plain_quant, "route": _plain_route, "unroute": _plain_unroute,
         "combine": _plain_combine, "uncombine": _plain_uncombine}
OWN = {"product": _own_product, "quant": _own_quant, "route": _own_route, "unroute": _own_unroute, "combine": _own_combine,
       "uncombine": _own_uncombine}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------- work and exact values


def work(case):
    kind = case["kind"]
    if kind == "product":
        m, n, k, groups = case["m"], case["n"], case["k"], case["groups"]
        by_rows = groups and case["by"] == "rows"
        # (experts without rows are not read: of `groups`, m rows drawn with replacement meet at most min(groups, m); about
        # groups * (1 - exp(-m / groups)) of them)
        read = groups * (1 - math.exp(-m / groups)) if by_rows else 1
        scales = _blocks(k) * (m + read * (_blocks(n) if case["b_rows"] == BLOCK else n)) * 4
        out = m * n * (groups if groups and not by_rows else 1) * BYTES[case["out"]]
        return {"bytes": int(m * k + read * n * k + scales + out), "flops": 2 * m * n * k}
    if kind == "quant":
        cells, sources = case["batch"] * case["rows"] * case["cols"], case["rows"] // max(1, case["div"])
        read = case["batch"] * max(1, sources) * case["cols"] * BYTES[case["dtype"]] + (4 * case["rows"] if case["div"] else 0)
        return {"bytes": int(read + cells + 4 * cells / BLOCK), "flops": 2 * cells}
    if kind in ("route", "unroute"):
        cells, pairs = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        if kind == "unroute":
            return {"bytes": 2 * cells * BYTES[case["dtype"]] + 8 * pairs, "flops": 8 * cells}
        rows = _rows(pairs, case["experts"], case["align"])
        return {"bytes": cells * BYTES[case["dtype"]] + 12 * pairs + 4 * rows + 4 * case["experts"], "flops": 8 * cells}
    pairs, b = case["tokens"] * case["top_k"], BYTES[case["dtype"]]
    if kind == "combine":
        return {"bytes": (pairs + case["tokens"]) * case["width"] * b + 8 * pairs, "flops": 2 * pairs * case["width"]}
    rows = _rows(pairs, 64, case["align"])
    return {"bytes": (pairs + case["tokens"] + rows) * case["width"] * b + 12 * pairs + 4 * rows, "flops": 3 * pairs * case["width"]}


def _rounded(v, dtype):
    """64-bit values to the nearest 8-bit ones (ties to even), from the format alone: 3 or 2 bits of fraction."""
    bits, low = (3, -6) if dtype == "e4m3" else (2, -14)
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=low).double() - bits)
    return torch.clamp(torch.round(v / step) * step, -LARGEST[dtype], LARGEST[dtype])


def _exact_product(case, s):
    k, n = case["k"], case["n"]
    sa = s["a_scale"].double()
    sb = s["b_scale"].double()

    def one(rows, terms, b, scale):
        """The block sums one after another, each with its scales."""
        c = torch.zeros((rows.stop - rows.start, n), dtype=torch.float64, device="cuda")
        for t in range(terms.start, terms.stop, BLOCK):
            blk, to = t // BLOCK, min(t + BLOCK, terms.stop, k)
            part = s["a"][rows, t:to].double() @ b[:, t:to].double().t()
            col = scale[blk] if case["b_rows"] == 1 else scale[:, blk][torch.arange(n, device="cuda") // BLOCK]
            c += part * sa[blk, rows][:, None] * col
        return c

    if not case["groups"]:
        return one(slice(0, case["m"]), slice(0, k), s["b"], sb)
    o = s["offsets"].tolist()
    if case["by"] == "rows":
        return torch.cat([one(slice(o[e], o[e + 1]), slice(0, k), s["b"][e], sb[e]) for e in range(case["groups"])])
    return torch.stack([one(slice(0, case["m"]), slice(o[e], o[e + 1]), s["b"], sb) for e in range(case["groups"])])


def _exact_quant(case, s):
    x = s["x"].double()
    if s["rows"] is not None:
        x = x[:, torch.div(s["rows"], case["div"], rounding_mode="floor").long()]
    if case["form"] in ("columns", "tiles_transposed"):
        x = x.permute(0, 2, 1)
    batch, r, c = x.shape
    tall = BLOCK if "tiles" in case["form"] else 1
    scale = torch.zeros(batch, -(-r // tall), _blocks(c), dtype=torch.float64, device="cuda")
    q = torch.empty_like(x)
    if tall == 1:
        for j in range(_blocks(c)):
            part = x[:, :, j * BLOCK:(j + 1) * BLOCK]
            scale[:, :, j] = torch.clamp(part.abs().amax(2), min=2.0 ** -100) / LARGEST[case["to"]]
            q[:, :, j * BLOCK:(j + 1) * BLOCK] = _rounded(part / scale[:, :, j, None], case["to"])
        return [q, scale.permute(0, 2, 1)]
    for i in range(scale.shape[1]):
        for j in range(scale.shape[2]):
            at = (slice(None), slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
            scale[:, i, j] = torch.clamp(x[at].abs().amax((1, 2)), min=2.0 ** -100) / LARGEST[case["to"]]
            q[at] = _rounded(x[at] / scale[:, i, j, None, None], case["to"])
    return [q, scale]


def _softmax64(z):
    return torch.exp(z - torch.logsumexp(z, 1, keepdim=True))


def _exact_route(case, s):
    z = s["logits"].double()
    p = torch.sigmoid(z) if case["score"] == "sigmoid" else _softmax64(z)
    rank = p + (s["bias"].double() if s["bias"] is not None else 0)
    if case["groups"] > 1:
        size = case["experts"] // case["groups"]
        two = torch.stack([rank[:, i * size:(i + 1) * size].topk(min(2, size), 1).values.sum(1) for i in range(case["groups"])], 1)
        out = two.argsort(1, descending=True)[:, case["top_groups"]:]
        for i in range(case["groups"]):
            rank[:, i * size:(i + 1) * size][(out == i).any(1)] = -math.inf
    w = p.gather(1, rank.topk(case["top_k"], 1).indices)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return [w * SCALE, None, None, None, None]


def _exact_unroute(case, s):
    z = s["logits"].double().requires_grad_()
    p = torch.sigmoid(z) if case["score"] == "sigmoid" else _softmax64(z)
    w = p.gather(1, s["ids"].long())
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return torch.autograd.grad((w * SCALE * s["dweights"].double()).sum(), z)[0]


def _exact_combine(case, s):
    out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        out += s["weights"][:, j, None].double() * s["y"][s["position"][:, j].long()].double()
    return out


def _exact_uncombine(case, s):
    dy = torch.zeros(s["rows"], case["width"], dtype=torch.float64, device="cuda")
    dweights = []
    for j in range(case["top_k"]):
        at = s["position"][:, j].long()
        dy[at] = s["weights"][:, j, None].double() * s["dout"].double()
        dweights.append((s["y"][at].double() * s["dout"].double()).sum(1))
    return [dy, torch.stack(dweights, 1)]


def exact(case, seed):
    at = {"product": _exact_product, "quant": _exact_quant, "route": _exact_route, "unroute": _exact_unroute,
          "combine": _exact_combine, "uncombine": _exact_uncombine}[case["kind"]]
    return functools.partial(at, case)(prepare(case, seed))
