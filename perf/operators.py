"""Workloads of the W8A8 product and of the expert path: plain forms, library calls, exact values.

Four operators and their chain:

  product   D = bf16(sa[m] sb[n] sum_k A[m,k] B[n,k]) on int8 codes, one scale per token (row of A)
            and per channel (row of B); A is given as codes, or as bf16 rows that the call quantises
  grouped   the same product for rows sorted by expert, row offsets on the device, optionally with
            the gated epilogue (even rows of B up, odd rows gate)
  route     logits -> the top_k experts of every token and their weights; with the gradient where a
            router is trained
  rows      expert ids -> rows sorted by expert: row maps, gathered rows, weighted sum back; with the
            gradients of the sum where a router is trained
  layer     route, rows, gated product, quantisation, product, weighted sum in one pass

``own`` false: elementary torch operations.  ``own`` true: the calls of the library.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_DEV = "cuda"


# --------------------------------------------------------------------------------- cases
def listed():
    return [
        # One token through one projection: the latency of a decode step at batch one.
        dict(name="product_token", op="product", m=1, n=4096, k=4096, acts="bf16"),
        # The decode shape of the benchmark (MLP up-projection) for a batch of sixteen requests.
        dict(name="product_decode", op="product", m=16, n=28672, k=8192, acts="bf16"),
        # The ragged shape of the benchmark, activations as the layer before hands them over.
        dict(name="product_ragged", op="product", m=4095, n=12289, k=4160, acts="bf16"),
        # The square shape of the benchmark on codes: a prefill batch, bound by the tensor cores.
        dict(name="product_square", op="product", m=8192, n=8192, k=8192, acts="codes"),
        # 32 tokens in decode, 8 experts each, gated projection: bound by reading the experts' weights.
        dict(name="grouped_decode", op="grouped", rows=256, groups=128, n=1536, k=2048, gated=True, skew=0.7),
        # A prefill batch of 4096 tokens, 8 experts each, gated projection: bound by the tensor cores.
        dict(name="grouped_prefill", op="grouped", rows=32768, groups=64, n=4096, k=2048, gated=True, skew=0.4),
        # One token, group-limited sigmoid routing with a balance bias: latency.
        dict(name="route_token", op="route", tokens=1, experts=256, top_k=8, n_groups=8, top_groups=4, sigmoid=True,
             renorm=True, top2=True, bias=True, bf16=False, padded=0.0, grad=False),
        # The same routing for a prefill batch with padding rows.
        dict(name="route_prefill", op="route", tokens=16384, experts=256, top_k=8, n_groups=8, top_groups=4,
             sigmoid=True, renorm=True, top2=True, bias=True, bf16=False, padded=0.1, grad=False),
        # A training step of a softmax router: weights and the gradient of the logits.
        dict(name="route_train", op="route", tokens=16384, experts=64, top_k=6, n_groups=1, top_groups=1, sigmoid=False,
             renorm=False, top2=False, bias=False, bf16=True, padded=0.0, grad=True),
        # A decode batch: sort the rows, quantise them into place, sum the experts' outputs.
        dict(name="rows_decode", op="rows", tokens=16, top_k=8, experts=256, width=4096, codes=True, align=1,
             dropped=0.1, grad=False),
        # A training batch in bf16, rows padded to the tiles of the bf16 grouped product, with gradients.
        dict(name="rows_train", op="rows", tokens=8192, top_k=8, experts=64, width=2048, codes=False, align=256,
             dropped=0.02, grad=True),
        # A whole int8 expert layer for 512 tokens.
        dict(name="layer_chunk", op="layer", tokens=512, experts=64, top_k=8, width=2048, hidden=1024),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["product", "product", "grouped", "route", "rows", "layer"])
    if op == "product":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 16, 28672), _log(rng, 32, 8192)
            if m * n * k <= 8192 ** 3:
                return dict(op=op, m=m, n=n, k=k, acts=rng.choice(["bf16", "codes"]))
    if op == "grouped":
        while True:
            gated = rng.random() < 0.5
            rows, groups = _log(rng, 1, 32768), _log(rng, 2, 128)
            n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
            if gated:
                n = (n + 15) // 16 * 16
            if groups * n * k <= 64 * 4096 * 2048 and rows * n * k <= 32768 * 4096 * 2048:
                return dict(op=op, rows=rows, groups=groups, n=n, k=k, gated=gated, skew=round(rng.uniform(0, 1.2), 2))
    if op == "route":
        n_groups = rng.choice([1, 1, 2, 4, 8])
        experts = n_groups * max(1, _log(rng, 8, 512) // n_groups)
        top_groups = rng.randint(1, n_groups)
        top_k = rng.randint(1, min(8, experts // n_groups * top_groups))
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts, top_k=top_k, n_groups=n_groups,
                    top_groups=top_groups, sigmoid=rng.random() < 0.5, renorm=rng.random() < 0.5,
                    top2=rng.random() < 0.5, bias=rng.random() < 0.5, bf16=rng.random() < 0.5,
                    padded=rng.choice([0.0, 0.1]), grad=rng.random() < 0.5)
    if op == "rows":
        while True:
            tokens, top_k, width = _log(rng, 1, 8192), rng.randint(1, 8), _log(rng, 64, 4096)
            if tokens * top_k * width <= 8192 * 8 * 2048:
                return dict(op=op, tokens=tokens, top_k=top_k, experts=_log(rng, 4, 512), width=width,
                            codes=rng.random() < 0.5, align=rng.choice([1, 1, 256]),
                            dropped=rng.choice([0.0, 0.1]), grad=rng.random() < 0.5)
    experts = _log(rng, 8, 64)
    return dict(op=op, tokens=_log(rng, 1, 512), experts=experts, top_k=rng.randint(1, 8),
                width=8 * _log(rng, 16, 256), hidden=8 * _log(rng, 8, 128))


# --------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=_DEV)


def _pitch(k, unit):
    return (k + unit - 1) // unit * unit


def _activations(g, rows, k):
    """bf16 rows as a normalised hidden state looks: tokens of different size, a few large channels."""
    size = torch.exp(0.5 * _randn(g, rows, 1))
    channel = torch.where(torch.rand(k, generator=g, device=_DEV) < 0.01, 8.0, 1.0)
    return (_randn(g, rows, k) * size * channel).bfloat16()


def _pitched(codes):
    """int8 rows at a pitch of 16 bytes, as a program lays its weights out once."""
    rows, k = codes.shape
    out = torch.zeros(rows, _pitch(k, 16), dtype=torch.int8, device=_DEV)
    out[:, :k] = codes
    return out


def _weights(g, rows, k):
    """Codes of Gaussian weights with one scale per channel, at a pitch of 16 bytes."""
    out = torch.zeros(rows, _pitch(k, 16), dtype=torch.int8, device=_DEV)
    for r0 in range(0, rows, 1 << 15):
        r1 = min(rows, r0 + (1 << 15))
        out[r0:r1, :k] = (_randn(g, r1 - r0, k) * 33.0).round_().clamp_(-127, 127).to(torch.int8)
    return out, torch.exp(0.3 * _randn(g, rows)) * (0.02 / 33.0)


def _sizes(rows, groups, skew):
    """Rows per expert: weights falling as 1 / rank^skew, whole numbers that add up to `rows`."""
    share = [1.0 / (i + 1) ** skew for i in range(groups)]
    total = sum(share)
    want = [rows * s / total for s in share]
    have = [int(w) for w in want]
    order = sorted(range(groups), key=lambda i: want[i] - have[i], reverse=True)
    for i in order[:rows - sum(have)]:
        have[i] += 1
    return have


def _max_rows(tokens, top_k, experts, align):
    n = tokens * top_k
    return (n + min(experts, n) * (align - 1)) // align * align


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["b"], s["sb"] = _weights(g, n, k)
        s["x"] = _activations(g, m, k)
        if case["acts"] == "codes":
            codes, s["sa"] = _quantize(s.pop("x"))
            s["a"] = _pitched(codes)
        s["d"] = torch.zeros(m, n, dtype=torch.bfloat16, device=_DEV)
    elif op == "grouped":
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        sizes = _sizes(rows, groups, case["skew"])
        perm = torch.randperm(groups, generator=g, device=_DEV).tolist()
        s["sizes"] = [sizes[i] for i in perm]
        ends = [0]
        for c in s["sizes"]:
            ends.append(ends[-1] + c)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=_DEV)
        s["b"], s["sb"] = _weights(g, groups * n, k)
        codes, s["sa"] = _quantize(_activations(g, rows, k))
        s["a"] = _pitched(codes)
        s["d"] = torch.zeros(rows, n // 2 if case["gated"] else n, dtype=torch.bfloat16, device=_DEV)
    elif op == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        logits = 1.5 * _randn(g, tokens, experts) + 0.5 * _randn(g, experts)
        if case["padded"]:
            logits[torch.rand(tokens, generator=g, device=_DEV) < case["padded"]] = -math.inf
        s["logits"] = logits.bfloat16() if case["bf16"] else logits
        s["bias"] = 0.1 * _randn(g, experts) if case["bias"] else None
        s["ids"] = torch.zeros(tokens, top_k, dtype=torch.int32, device=_DEV)
        s["weights"] = torch.zeros(tokens, top_k, device=_DEV)
        if case["grad"]:
            s["grad_weights"] = _randn(g, tokens, top_k)
            s["grad_logits"] = torch.zeros_like(s["logits"])
    elif op == "rows":
        tokens, top_k, experts, width = case["tokens"], case["top_k"], case["experts"], case["width"]
        # Experts with popularities of their own; dropped slots as capacity limits and padding leave them.
        pop = torch.softmax(0.7 * _randn(g, experts), 0)
        ids = torch.multinomial(pop.expand(tokens, experts), min(top_k, experts), generator=g)
        ids = torch.cat([ids, ids.new_zeros(tokens, top_k - ids.shape[1])], 1).int()
        ids[torch.rand(tokens, top_k, generator=g, device=_DEV) < case["dropped"]] = -1
        s["ids"] = ids.contiguous()
        s["x"] = _activations(g, tokens, width)
        s["weights"] = torch.rand(tokens, top_k, generator=g, device=_DEV)
        cap = _max_rows(tokens, top_k, experts, case["align"])
        s["cap"] = cap
        s["out"] = _randn(g, cap, width).bfloat16()
        i32 = dict(dtype=torch.int32, device=_DEV)
        s["offsets"] = torch.zeros(experts + 1, **i32)
        s["row_of_slot"] = torch.zeros(tokens, top_k, **i32)
        s["slot_of_row"] = torch.zeros(cap, **i32)
        s["mtile_group"] = torch.zeros(cap // 256, **i32) if case["align"] == 256 else None
        if case["codes"]:
            s["codes"] = torch.zeros(cap, _pitch(width, 16), dtype=torch.int8, device=_DEV)
            s["scales"] = torch.zeros(cap, device=_DEV)
        else:
            s["gathered"] = torch.zeros(cap, width, dtype=torch.bfloat16, device=_DEV)
        s["y"] = torch.zeros(tokens, width, dtype=torch.bfloat16, device=_DEV)
        if case["grad"]:
            s["grad_y"] = _randn(g, tokens, width).bfloat16()
            s["grad_out"] = torch.zeros(cap, width, dtype=torch.bfloat16, device=_DEV)
            s["grad_weights"] = torch.zeros(tokens, top_k, device=_DEV)
    else:
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        width, hidden = case["width"], case["hidden"]
        s["x"] = _activations(g, tokens, width)
        s["logits"] = 1.5 * _randn(g, tokens, experts) + 0.5 * _randn(g, experts)
        s["b1"], s["sb1"] = _weights(g, experts * 2 * hidden, width)
        s["b2"], s["sb2"] = _weights(g, experts * width, hidden)
        cap = tokens * top_k
        i32 = dict(dtype=torch.int32, device=_DEV)
        s["ids"] = torch.zeros(tokens, top_k, **i32)
        s["weights"] = torch.zeros(tokens, top_k, device=_DEV)
        s["offsets"] = torch.zeros(experts + 1, **i32)
        s["row_of_slot"] = torch.zeros(tokens, top_k, **i32)
        s["slot_of_row"] = torch.zeros(cap, **i32)
        s["a1"] = torch.zeros(cap, _pitch(width, 16), dtype=torch.int8, device=_DEV)
        s["sa1"] = torch.zeros(cap, device=_DEV)
        s["h"] = torch.zeros(cap, hidden, dtype=torch.bfloat16, device=_DEV)
        s["a2"] = torch.zeros(cap, _pitch(hidden, 16), dtype=torch.int8, device=_DEV)
        s["sa2"] = torch.zeros(cap, device=_DEV)
        s["out"] = torch.zeros(cap, width, dtype=torch.bfloat16, device=_DEV)
        s["y"] = torch.zeros(tokens, width, dtype=torch.bfloat16, device=_DEV)
    if own:
        _plans(s)
    return s


# --------------------------------------------------------------------------------- library calls
def _smb():
    return importlib.import_module("strata-masonry_b200")


def _plans(s):
    """The plans a program keeps: tensor maps and tile choice for its buffers."""
    smb, case = _smb(), s["case"]
    static, gated = smb.capi.FLAG_WEIGHTS_STATIC, smb.capi.FLAG_EPILOGUE_SWIGLU
    plan = smb.gemm.I8Plan
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        if case["acts"] == "bf16":
            s["plan"] = plan.from_bf16_activations(s["x"], s["b"], s["sb"], s["d"], m, n, k, ldb=s["b"].shape[1],
                                                   flags=static)
        else:
            s["plan"] = plan(s["a"], s["sa"], s["b"], s["sb"], s["d"], m, n, k, lda=s["a"].shape[1],
                             ldb=s["b"].shape[1], flags=static)
    elif case["op"] == "grouped":
        s["plan"] = plan.grouped(s["a"], s["sa"], s["b"], s["sb"], s["d"], case["rows"], case["n"], case["k"],
                                 case["groups"], s["offsets"], lda=s["a"].shape[1], ldb=s["b"].shape[1],
                                 flags=static | (gated if case["gated"] else 0))
    elif case["op"] == "layer":
        cap, experts, width, hidden = s["out"].shape[0], case["experts"], case["width"], case["hidden"]
        s["plan1"] = plan.grouped(s["a1"], s["sa1"], s["b1"], s["sb1"], s["h"], cap, 2 * hidden, width, experts,
                                  s["offsets"], lda=s["a1"].shape[1], ldb=s["b1"].shape[1], flags=static | gated)
        s["plan2"] = plan.grouped(s["a2"], s["sa2"], s["b2"], s["sb2"], s["out"], cap, width, hidden, experts,
                                  s["offsets"], lda=s["a2"].shape[1], ldb=s["b2"].shape[1], flags=static)


def _route_flags(smb, case):
    c = smb.capi
    return ((c.ROUTE_SIGMOID if case["sigmoid"] else 0) | (c.ROUTE_RENORM if case["renorm"] else 0) |
            (c.ROUTE_GROUP_TOP2 if case["top2"] else 0))


def _run_own(s):
    smb, case, st = _smb(), s["case"], torch.cuda.current_stream().cuda_stream
    moe, op = smb.moe, case["op"]
    if op in ("product", "grouped"):
        s["plan"].run(st)
        return dict(d=s["d"])
    if op == "route":
        dtype = smb.capi.DTYPE_BF16 if case["bf16"] else smb.capi.DTYPE_F32
        flags, dims = _route_flags(smb, case), (case["tokens"], case["experts"], case["top_k"])
        moe.route_device(s["logits"], s["ids"], s["weights"], *dims, dtype=dtype, bias=s["bias"],
                         n_groups=case["n_groups"], top_groups=case["top_groups"], flags=flags, scale=2.5, stream=st)
        out = dict(ids=s["ids"], weights=s["weights"])
        if case["grad"]:
            moe.route_backward_device(s["logits"], s["ids"], s["grad_weights"], s["grad_logits"], *dims, dtype=dtype,
                                      flags=flags, scale=2.5, stream=st)
            out["grad_logits"] = s["grad_logits"]
        return out
    if op == "rows":
        tokens, top_k, experts, width = case["tokens"], case["top_k"], case["experts"], case["width"]
        moe.dispatch_device(s["ids"], s["offsets"], s["row_of_slot"], s["slot_of_row"], tokens, top_k, experts,
                            s["cap"], align=case["align"], mtile_group=s["mtile_group"], stream=st)
        out = {n: s[n] for n in ("offsets", "row_of_slot", "slot_of_row")}
        if s["mtile_group"] is not None:
            out["mtile_group"] = s["mtile_group"]
        if case["codes"]:
            moe.gather_i8_device(s["x"], s["row_of_slot"], s["codes"], s["scales"], tokens, top_k, width, s["cap"],
                                 ld_bytes=s["codes"].shape[1], stream=st)
            out.update(codes=s["codes"], scales=s["scales"])
        else:
            moe.gather_bf16_device(s["x"], s["row_of_slot"], s["gathered"], tokens, top_k, width, s["cap"], stream=st)
            out["gathered"] = s["gathered"]
        moe.combine_device(s["out"], s["row_of_slot"], s["weights"], s["y"], tokens, top_k, width, s["cap"], stream=st)
        out["y"] = s["y"]
        if case["grad"]:
            moe.combine_backward_device(s["grad_y"], s["out"], s["row_of_slot"], s["weights"], s["grad_out"],
                                        s["grad_weights"], tokens, top_k, width, s["cap"], stream=st)
            out.update(grad_out=s["grad_out"], grad_weights=s["grad_weights"])
        return out
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    width, hidden, cap = case["width"], case["hidden"], s["out"].shape[0]
    moe.route_device(s["logits"], s["ids"], s["weights"], tokens, experts, top_k, flags=smb.capi.ROUTE_RENORM, stream=st)
    moe.dispatch_device(s["ids"], s["offsets"], s["row_of_slot"], s["slot_of_row"], tokens, top_k, experts, cap, stream=st)
    moe.gather_i8_device(s["x"], s["row_of_slot"], s["a1"], s["sa1"], tokens, top_k, width, cap,
                         ld_bytes=s["a1"].shape[1], stream=st)
    s["plan1"].run(st)
    smb.gemm.quantize_i8_bf16_device(s["h"], s["a2"], s["sa2"], cap, hidden, ld_bytes=s["a2"].shape[1], stream=st)
    s["plan2"].run(st)
    moe.combine_device(s["out"], s["row_of_slot"], s["weights"], s["y"], tokens, top_k, width, cap, stream=st)
    return dict(ids=s["ids"], weights=s["weights"], y=s["y"])


# --------------------------------------------------------------------------------- plain forms
def _quantize(x):
    """One scale per row: scale = amax / 127, code = round_half_even(x * (127 / amax)), in 32 bits."""
    v = x.float()
    amax = v.abs().amax(1).clamp_min(2.0 ** -100)
    top = torch.full_like(amax, 127.0)
    return (v * (top / amax).unsqueeze(1)).round().clamp(-127, 127).to(torch.int8), amax / top


def _product(a, sa, b, sb):
    return (a.float() @ b.float().t()) * sa.unsqueeze(1) * sb


def _gate(acc):
    up, gate = acc[:, 0::2], acc[:, 1::2]
    return gate / (1.0 + torch.exp(-gate)) * up


def _route(logits, bias, case):
    """Selection in 64 bits (scores next to a border), weights in 32."""
    top_k, n_groups, top_groups = case["top_k"], case.get("n_groups", 1), case.get("top_groups", 1)
    sigmoid, renorm = case.get("sigmoid", False), case.get("renorm", True)
    l = logits.double()
    tokens, experts = l.shape
    open_ = l > -math.inf
    top = torch.where(open_, l, torch.full_like(l, -1e300)).amax(1, keepdim=True)
    if sigmoid:
        p = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.where(open_, torch.exp(l - top), torch.zeros_like(l))
        p = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    closed = torch.full_like(l, -math.inf)
    score = torch.where(open_, p + bias.double() if bias is not None else (p if n_groups > 1 else l), closed)
    pick = score
    if n_groups > 1:
        by_group = score.view(tokens, n_groups, experts // n_groups)
        best = by_group.sort(dim=2, descending=True).values
        group = best[:, :, 0]
        if case["top2"] and best.shape[2] > 1:
            second = best[:, :, 1]
            group = group + torch.where(second > -math.inf, second, torch.zeros_like(second))
        keep = group.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        kept = torch.zeros_like(group, dtype=torch.bool).scatter_(1, keep, True)
        kept = kept & (group > -math.inf)
        mask = kept.unsqueeze(2).expand_as(by_group).reshape(tokens, experts)
        # Without a bias the logits themselves are compared inside the kept groups.
        pick = torch.where(mask, score if bias is not None else torch.where(open_, l, closed), closed)
    order = pick.sort(dim=1, descending=True, stable=True)
    ids, have = order.indices[:, :top_k], order.values[:, :top_k] > -math.inf
    chosen = p.gather(1, ids).float() * have
    if renorm:
        chosen = chosen / chosen.sum(1, keepdim=True).clamp_min(1e-30)
    return torch.where(have, ids, torch.full_like(ids, -1)).int(), chosen * case.get("scale", 2.5)


def _route_grad(logits, ids, grad, case):
    """Gradient of the logits for fixed ids; w = scale p (or scale p / sum of the chosen p)."""
    l = logits.float()
    have = ids >= 0
    at = ids.clamp_min(0).long()
    g = torch.where(have, grad * 2.5, torch.zeros_like(grad))
    out = torch.zeros_like(l)
    if case["sigmoid"]:
        p = 1.0 / (1.0 + torch.exp(-l))
        pk = p.gather(1, at) * have
        if case["renorm"]:
            q = pk / pk.sum(1, keepdim=True).clamp_min(1e-30)
            d = (1.0 - pk) * q * (g - (g * q).sum(1, keepdim=True))
        else:
            d = g * pk * (1.0 - pk)
        return out.scatter_add_(1, at, d * have).to(logits.dtype)
    open_ = l > -math.inf
    top = torch.where(open_, l, torch.full_like(l, -1e30)).amax(1, keepdim=True)
    e = torch.where(open_, torch.exp(l - top), torch.zeros_like(l))
    p = e / e.sum(1, keepdim=True).clamp_min(1e-30)
    pk = p.gather(1, at) * have
    if case["renorm"]:
        q = pk / pk.sum(1, keepdim=True).clamp_min(1e-30)
        return out.scatter_add_(1, at, q * (g - (g * q).sum(1, keepdim=True))).to(logits.dtype)
    out.scatter_add_(1, at, g * pk)
    return (out - p * (g * pk).sum(1, keepdim=True)).to(logits.dtype)


def _dispatch(ids, experts, align, cap):
    """Stable sort of the slots by expert, every expert's rows padded to a multiple of `align`."""
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < experts)
    key = torch.where(ok, flat, torch.full_like(flat, experts))
    hot = torch.zeros(experts + 1, dtype=torch.int64, device=_DEV).scatter_add_(0, key, torch.ones_like(key))
    padded = (hot[:experts] + align - 1) // align * align
    offsets = torch.cat([padded.new_zeros(1), padded.cumsum(0)])
    order = key.sort(stable=True).indices
    before = hot.cumsum(0) - hot
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device=_DEV) - before[key[order]]
    row = torch.where(ok, offsets[key.clamp_max(experts - 1)] + rank, torch.full_like(flat, -1))
    slot = torch.full((cap + 1,), -1, dtype=torch.int64, device=_DEV)
    slot[torch.where(ok, row, torch.full_like(row, cap))] = torch.arange(flat.numel(), device=_DEV)
    out = dict(offsets=offsets.int(), row_of_slot=row.view(ids.shape).int(), slot_of_row=slot[:cap].int())
    if align == 256:
        tile = torch.arange(cap // 256, device=_DEV) * 256
        out["mtile_group"] = (torch.searchsorted(offsets, tile, right=True) - 1).clamp_max(experts - 1).int()
    return out


def _rows_of(row, values, cap, fill):
    """values[t, j] to row row[t, j]; rows nobody names keep `fill`."""
    out = fill.new_zeros((cap + 1,) + values.shape[2:]) + fill
    at = torch.where(row >= 0, row, torch.full_like(row, cap)).reshape(-1).long()
    out[at] = values.reshape((-1,) + values.shape[2:])
    return out[:cap]


def _combine(rows, row_of_slot, weights):
    have = (row_of_slot >= 0).unsqueeze(2)
    picked = rows[row_of_slot.clamp_min(0).long()].float()
    return (torch.where(have, picked, torch.zeros_like(picked)) * weights.unsqueeze(2)).sum(1)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "product":
        k = case["k"]
        a, sa = (s["a"][:, :k], s["sa"]) if case["acts"] == "codes" else _quantize(s["x"])
        return dict(d=_product(a, sa, s["b"][:, :k], s["sb"]).bfloat16())
    if op == "grouped":
        n, k, parts, r0 = case["n"], case["k"], [], 0
        for g, rows in enumerate(s["sizes"]):
            if rows:
                acc = _product(s["a"][r0:r0 + rows, :k], s["sa"][r0:r0 + rows], s["b"][g * n:(g + 1) * n, :k],
                               s["sb"][g * n:(g + 1) * n])
                parts.append((_gate(acc) if case["gated"] else acc).bfloat16())
                r0 += rows
        return dict(d=torch.cat(parts))
    if op == "route":
        ids, weights = _route(s["logits"], s["bias"], case)
        out = dict(ids=ids, weights=weights)
        if case["grad"]:
            out["grad_logits"] = _route_grad(s["logits"], ids, s["grad_weights"], case)
        return out
    if op == "rows":
        top_k, cap = case["top_k"], s["cap"]
        out = _dispatch(s["ids"], case["experts"], case["align"], cap)
        row = out["row_of_slot"]
        if case["codes"]:
            codes, scales = _quantize(s["x"])
            codes = torch.nn.functional.pad(codes, (0, s["codes"].shape[1] - case["width"]))
            out["codes"] = _rows_of(row, codes.unsqueeze(1).expand(-1, top_k, -1), cap, codes.new_zeros(1))
            out["scales"] = _rows_of(row, scales.unsqueeze(1).expand(-1, top_k), cap, scales.new_zeros(1))
        else:
            out["gathered"] = _rows_of(row, s["x"].unsqueeze(1).expand(-1, top_k, -1), cap, s["x"].new_zeros(1))
        out["y"] = _combine(s["out"], row, s["weights"]).bfloat16()
        if case["grad"]:
            gy = s["grad_y"].float().unsqueeze(1)
            out["grad_out"] = _rows_of(row, (gy * s["weights"].unsqueeze(2)).bfloat16(), cap, s["x"].new_zeros(1))
            picked = s["out"][row.clamp_min(0).long()].float()
            out["grad_weights"] = (picked * gy).sum(2) * (row >= 0)
        return out
    experts, width, hidden = case["experts"], case["width"], case["hidden"]
    ids, weights = _route(s["logits"], None, dict(case, scale=1.0))
    a1, sa1 = _quantize(s["x"])
    y = torch.zeros(case["tokens"], width, device=_DEV)
    for e in range(experts):
        share = torch.where(ids == e, weights, torch.zeros_like(weights)).sum(1, keepdim=True)
        rows1, rows2 = slice(e * 2 * hidden, (e + 1) * 2 * hidden), slice(e * width, (e + 1) * width)
        h = _gate(_product(a1, sa1, s["b1"][rows1, :width], s["sb1"][rows1])).bfloat16()
        a2, sa2 = _quantize(h)
        y += share * _product(a2, sa2, s["b2"][rows2, :hidden], s["sb2"][rows2]).bfloat16().float()
    return dict(ids=ids, weights=weights, y=y.bfloat16())


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k * 2 if case["acts"] == "bf16" else m * k + 4 * m
        return dict(bytes=a + n * k + 4 * n + 2 * m * n, flops=2 * m * n * k)
    if op == "grouped":
        rows, n, k = case["rows"], case["n"], case["k"]
        hit = sum(1 for c in _sizes(rows, case["groups"], case["skew"]) if c)
        wide = n // 2 if case["gated"] else n
        return dict(bytes=rows * (k + 4) + hit * n * (k + 4) + 4 * (case["groups"] + 1) + 2 * rows * wide,
                    flops=2 * rows * n * k)
    if op == "route":
        t, e, k, size = case["tokens"], case["experts"], case["top_k"], 2 if case["bf16"] else 4
        grad = (t * k * 4 + t * e * size) if case["grad"] else 0
        return dict(bytes=t * e * size + (4 * e if case["bias"] else 0) + 8 * t * k + grad,
                    flops=4 * t * e * (2 if case["grad"] else 1))
    if op == "rows":
        t, k, w = case["tokens"], case["top_k"], case["width"]
        n = t * k
        kept = int(n * (1 - case["dropped"]))
        cap = _max_rows(t, k, case["experts"], case["align"])
        maps = 4 * n + 4 * (case["experts"] + 1) + 4 * n + 4 * cap
        moved = 2 * t * w + kept * (w + 4 if case["codes"] else 2 * w) + 2 * kept * w + 4 * n + 2 * t * w
        grad = (2 * t * w + 2 * kept * w + 4 * n) if case["grad"] else 0
        return dict(bytes=maps + moved + grad, flops=2 * n * w * (3 if case["grad"] else 1))
    t, e, k, w, h = case["tokens"], case["experts"], case["top_k"], case["width"], case["hidden"]
    hit = min(e, t * min(k, e))
    return dict(bytes=t * e * 4 + 4 * t * w + hit * (2 * h * (w + 4) + w * (h + 4)) + 8 * t * k,
                flops=2 * t * min(k, e) * 3 * w * h)


# --------------------------------------------------------------------------------- exact values
def _f32(x):
    return x.float().double()


def _exact_codes(x):
    """The quantiser's definition, its 32-bit roundings written out on 64-bit values."""
    v = x.double()
    amax = torch.maximum(v.abs().max(dim=1).values, torch.tensor(2.0 ** -100, device=_DEV, dtype=torch.float64))
    inverse = _f32(127.0 / amax)
    return torch.round(_f32(v * inverse[:, None])), _f32(amax / 127.0)


def _exact_product(a, sa, b, sb):
    return torch.matmul(a.double(), b.double().T) * (sa.double()[:, None] * sb.double()[None, :])


def _exact_silu_pair(acc):
    gate = acc[:, 1::2]
    return acc[:, 0::2] * gate * torch.sigmoid(gate)


def _exact_selection(logits, bias, case):
    """ids by repeated maximum (lowest index on a tie), and the probabilities, in 64 bits."""
    x = logits.double()
    tokens, experts = x.shape
    lowest = torch.tensor(-math.inf, device=_DEV, dtype=torch.float64)
    if case.get("sigmoid", False):
        p = torch.reciprocal(1.0 + torch.exp(-x))
    else:
        p = torch.nan_to_num(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), nan=0.0)
    closed = torch.isneginf(x)
    groups = case.get("n_groups", 1)
    key = p + bias.double() if bias is not None else x
    key = torch.where(closed, lowest, key)
    if groups > 1:
        base = torch.where(closed, lowest, p + bias.double()) if bias is not None else torch.where(closed, lowest, p)
        size = experts // groups
        value = []
        for g in range(groups):
            part = base[:, g * size:(g + 1) * size].clone()
            first = part.max(1)
            total = first.values.clone()
            if case["top2"] and size > 1:
                part.scatter_(1, first.indices[:, None], -math.inf)
                second = part.max(1).values
                total = torch.where(torch.isneginf(second), total, total + second)
            value.append(total)
        value = torch.stack(value, 1)
        allowed = torch.zeros(tokens, groups, dtype=torch.bool, device=_DEV)
        number = torch.arange(groups, device=_DEV)
        for _ in range(case["top_groups"]):
            best = value.max(1, keepdim=True).values
            first = torch.where(value == best, number, groups).min(1, keepdim=True).values
            allowed.scatter_(1, first, ~torch.isneginf(best))
            value.scatter_(1, first, -math.inf)
        key = torch.where(allowed.repeat_interleave(size, 1), key, lowest)
    else:
        key = key.clone()
    number = torch.arange(experts, device=_DEV)
    ids = []
    for _ in range(case["top_k"]):
        if len(ids) >= experts:
            ids.append(torch.full_like(ids[0], -1))
            continue
        best = key.max(1, keepdim=True).values
        first = torch.where(key == best, number, experts).min(1, keepdim=True).values
        ids.append(torch.where(torch.isneginf(best), -1, first))
        key.scatter_(1, first, -math.inf)
    return torch.cat(ids, 1), p


def _exact_weights(ids, p, case, scale):
    w = torch.where(ids >= 0, p.gather(1, ids.clamp(min=0)), 0.0)
    if case.get("renorm", True):
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return w * scale


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "product":
        k = case["k"]
        a, sa = (s["a"][:, :k], s["sa"]) if case["acts"] == "codes" else _exact_codes(s["x"])
        return dict(d=_exact_product(a, sa, s["b"][:, :k], s["sb"]))
    if op == "grouped":
        n, k = case["n"], case["k"]
        out = torch.empty(s["d"].shape, dtype=torch.float64, device=_DEV)
        ends = s["offsets"].tolist()
        for g in range(case["groups"]):
            lo, hi = ends[g], ends[g + 1]
            if hi > lo:
                acc = _exact_product(s["a"][lo:hi, :k], s["sa"][lo:hi], s["b"][g * n:(g + 1) * n, :k],
                                     s["sb"][g * n:(g + 1) * n])
                out[lo:hi] = _exact_silu_pair(acc) if case["gated"] else acc
        return dict(d=out)
    if op == "route":
        ids, p = _exact_selection(s["logits"], s["bias"], case)
        w = _exact_weights(ids, p, case, 2.5)
        out = dict(ids=ids.int(), weights=w)
        if case["grad"]:
            # Row by row Jacobian product: dw_i/dl_e written out per chosen expert.
            g = torch.where(ids >= 0, s["grad_weights"].double(), 0.0)
            grad = torch.zeros_like(p)
            pick = torch.zeros_like(p)
            for j in range(case["top_k"]):
                here = (ids[:, j:j + 1] == torch.arange(case["experts"], device=_DEV)).double()
                grad += here * g[:, j:j + 1]
                pick += here
            # grad: dL/dw per expert.  w = 2.5 r(p), r(p) = p or p / sum of the chosen p.
            if case["renorm"]:
                total = (p * pick).sum(1, keepdim=True)
                inner = (grad * p * pick).sum(1, keepdim=True)
                dp = torch.where(total > 0, pick * (grad - inner / total) / total, 0.0)
            else:
                dp = grad
            dp = 2.5 * dp
            if case["sigmoid"]:
                out["grad_logits"] = dp * p * (1.0 - p)
            else:
                out["grad_logits"] = p * (dp - (dp * p).sum(1, keepdim=True))
        return out
    if op == "rows":
        ids, cap, align, top_k = s["ids"].cpu().numpy(), s["cap"], case["align"], case["top_k"]
        experts, width, tokens = case["experts"], case["width"], case["tokens"]
        lists = [[] for _ in range(experts)]
        for slot, e in enumerate(ids.reshape(-1).tolist()):
            if 0 <= e < experts:
                lists[e].append(slot)
        offsets, row_of_slot, slot_of_row, tiles = [0], [-1] * (tokens * top_k), [-1] * cap, []
        for e, slots in enumerate(lists):
            for i, slot in enumerate(slots):
                row_of_slot[slot] = offsets[-1] + i
                slot_of_row[offsets[-1] + i] = slot
            padded = (len(slots) + align - 1) // align * align
            tiles += [e] * (padded // 256)
            offsets.append(offsets[-1] + padded)
        i32 = dict(dtype=torch.int32, device=_DEV)
        out = dict(offsets=torch.tensor(offsets, **i32), row_of_slot=torch.tensor(row_of_slot, **i32).view(tokens, top_k),
                   slot_of_row=torch.tensor(slot_of_row, **i32))
        if align == 256:
            out["mtile_group"] = torch.tensor(tiles + [experts - 1] * (cap // 256 - len(tiles)), **i32)
        slots = out["slot_of_row"].long()
        live = torch.nonzero(slots >= 0)[:, 0]
        token = slots[live] // top_k
        if case["codes"]:
            codes, scales = _exact_codes(s["x"])
            full = torch.zeros(cap, s["codes"].shape[1], dtype=torch.int8, device=_DEV)
            full[live, :width] = codes.to(torch.int8)[token]
            scale = torch.zeros(cap, dtype=torch.float64, device=_DEV)
            scale[live] = scales[token]
            out.update(codes=full, scales=scale)
        else:
            gathered = torch.zeros(cap, width, dtype=torch.float64, device=_DEV)
            gathered[live] = s["x"].double()[token]
            out["gathered"] = gathered
        w = s["weights"].double().reshape(-1)[slots[live]]
        y = torch.zeros(tokens, width, dtype=torch.float64, device=_DEV)
        y.index_add_(0, token, s["out"].double()[live] * w[:, None])
        out["y"] = y
        if case["grad"]:
            gy = s["grad_y"].double()
            grad_out = torch.zeros(cap, width, dtype=torch.float64, device=_DEV)
            grad_out[live] = gy[token] * w[:, None]
            grad_w = torch.zeros(tokens * top_k, dtype=torch.float64, device=_DEV)
            grad_w[slots[live]] = (gy[token] * s["out"].double()[live]).sum(1)
            out.update(grad_out=grad_out, grad_weights=grad_w.view(tokens, top_k))
        return out
    experts, width, hidden = case["experts"], case["width"], case["hidden"]
    ids, p = _exact_selection(s["logits"], None, case)
    w = _exact_weights(ids, p, case, 1.0)
    a1, sa1 = _exact_codes(s["x"])
    y = torch.zeros(case["tokens"], width, dtype=torch.float64, device=_DEV)
    for e in range(experts):
        at = torch.nonzero(ids == e)
        if len(at) == 0:
            continue
        t = at[:, 0]
        up = _exact_product(a1[t], sa1[t], s["b1"][e * 2 * hidden:(e + 1) * 2 * hidden, :width],
                            s["sb1"][e * 2 * hidden:(e + 1) * 2 * hidden])
        # The hidden state is stored in bf16 before it is quantised again.
        a2, sa2 = _exact_codes(_exact_silu_pair(up).bfloat16())
        down = _exact_product(a2, sa2, s["b2"][e * width:(e + 1) * width, :hidden], s["sb2"][e * width:(e + 1) * width])
        y.index_add_(0, t, down * w[at[:, 0], at[:, 1]][:, None])
    return dict(ids=ids.int(), weights=w, y=y)
