"""Routing, row sorting, gathers and weighted sums on the GPU against plain 64-bit implementations.

Tolerances (half a step of fp32 is u = 2^-24).  Router weights: exp is within 2 u plus |argument| u from
the rounded argument (logits here stay within 40), sums of at most 512 terms over lanes of 16 add 21 u,
the divisions and the scale a handful: below 128 u = 2^-17 relative.  Gradients are sums of such terms,
so 2^-16 of the sum of the terms' magnitudes, plus 2^-8 relative where they are stored in bf16.
Weighted sums: top_k fused multiply-adds (u each of the running magnitude) and one rounding to bf16.
"""
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _torch():
    import torch
    return torch


# ------------------------------------------------------------------ routing, plain
def _probabilities(l, sigmoid):
    """float64 p; closed experts 0."""
    open_ = l > -np.inf
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            return np.where(open_, 1.0 / (1.0 + np.exp(-l)), 0.0)
        top = np.where(open_, l, -1e300).max(1, keepdims=True)
        e = np.where(open_, np.exp(l - top), 0.0)
    return e / np.maximum(e.sum(1, keepdims=True), 1e-300)


def _route_plain(l, bias, top_k, n_groups, top_groups, sigmoid, renorm, top2, scale):
    tokens, experts = l.shape
    l = np.where(l > -np.inf, l, -np.inf)   # NaN closes too
    p = _probabilities(l, sigmoid)
    base = p + (0.0 if bias is None else bias.astype(np.float64))
    base = np.where(l > -np.inf, base, -np.inf)
    key = base if bias is not None else l
    ids = np.full((tokens, top_k), -1)
    weights = np.zeros((tokens, top_k))
    size = experts // n_groups
    for t in range(tokens):
        open_ = key[t] > -np.inf
        if top_groups < n_groups:
            value = []
            for g in range(n_groups):
                best = np.sort(base[t, g * size:(g + 1) * size])[::-1]
                v = best[0]
                if top2 and size > 1 and best[1] > -np.inf:
                    v = v + best[1]
                value.append(v)
            kept = [g for g in sorted(range(n_groups), key=lambda g: (-value[g], g))[:top_groups] if value[g] > -np.inf]
            open_ = open_ & np.isin(np.arange(experts) // size, kept)
        order = sorted(np.nonzero(open_)[0].tolist(), key=lambda e: (-key[t, e], e))[:top_k]
        ids[t, :len(order)] = order
        w = p[t, order]
        if renorm and len(order):
            # Relative to the largest, so that tiny probabilities keep their ratio.
            ref = (np.minimum(l[t, order], 0) if sigmoid else l[t, order])
            q = np.exp(ref - ref.max())
            if sigmoid:
                q = q / (1.0 + np.exp(-np.abs(l[t, order])))
            w = q / q.sum()
        weights[t, :len(order)] = w * scale
    return ids, weights


def _logits(rng, tokens, experts, spread=1.5):
    return (spread * rng.standard_normal((tokens, experts))).astype(np.float32)


def _route(smb, torch, l, dtype, top_k, bias=None, n_groups=1, top_groups=1, flags=0, scale=1.0, pad=0):
    tokens, experts = l.shape
    buf = torch.full((tokens, experts + pad), 50.0, device="cuda")   # what lies behind a row would win
    buf[:, :experts] = torch.from_numpy(l)
    if dtype == smb.capi.DTYPE_BF16:
        buf = buf.bfloat16()
    ids = torch.full((tokens, top_k), 77, device="cuda", dtype=torch.int32)
    weights = torch.full((tokens, top_k), float("nan"), device="cuda")
    b = None if bias is None else torch.from_numpy(bias).cuda()
    smb.moe.route_device(buf, ids, weights, tokens, experts, top_k, dtype=dtype, bias=b, n_groups=n_groups,
                         top_groups=top_groups, flags=flags, scale=scale, ld=experts + pad)
    torch.cuda.synchronize()
    return buf, ids, weights


CASES = [
    # tokens, experts, top_k, n_groups, top_groups
    (1, 1, 1, 1, 1), (3, 7, 2, 1, 1), (130, 32, 4, 1, 1), (65, 64, 6, 1, 1), (40, 100, 5, 4, 2), (33, 160, 6, 8, 3),
    (200, 256, 8, 8, 4), (17, 512, 32, 16, 8), (5, 512, 1, 32, 1), (50, 96, 8, 32, 9), (9, 8, 8, 2, 2),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_route_against_plain(smb, cuda_device, case, sigmoid, with_bias, bf16):
    torch = _torch()
    tokens, experts, top_k, n_groups, top_groups = case
    rng = np.random.default_rng(tokens * 1000 + experts + sigmoid)
    l = _logits(rng, tokens, experts)
    if tokens > 2:
        l[1] = -np.inf                           # padding row
        l[2, rng.random(experts) < 0.7] = -np.inf
        l[0, experts // 2] = np.nan
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if with_bias else None
    if bias is not None and experts > 8:
        bias[3] = -np.inf
    c = smb.capi
    for renorm in (False, True):
        for top2 in (False, True):
            flags = ((c.ROUTE_SIGMOID if sigmoid else 0) | (c.ROUTE_RENORM if renorm else 0) |
                     (c.ROUTE_GROUP_TOP2 if top2 else 0))
            buf, ids, weights = _route(smb, torch, l, c.DTYPE_BF16 if bf16 else c.DTYPE_F32, top_k, bias, n_groups,
                                       top_groups, flags, 2.5, pad=3)
            want_ids, want = _route_plain(buf[:, :experts].float().cpu().numpy().astype(np.float64), bias, top_k, n_groups,
                                          top_groups, sigmoid, renorm, top2, 2.5)
            np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
            assert np.all(np.abs(weights.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -17)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_ties_go_to_the_lowest_index(smb, cuda_device, sigmoid):
    torch = _torch()
    c = smb.capi
    flags = c.ROUTE_SIGMOID if sigmoid else 0
    l = np.zeros((4, 64), dtype=np.float32)
    l[1, 40:] = 1.0
    l[2, ::3] = -2.0
    l[3] = np.repeat(np.arange(16, dtype=np.float32), 4)
    for bias in (None, np.zeros(64, dtype=np.float32), np.full(64, 0.25, dtype=np.float32)):
        _, ids, _ = _route(smb, torch, l, c.DTYPE_F32, 8, bias, 4, 2, flags)
        want, _ = _route_plain(l.astype(np.float64), bias, 8, 4, 2, sigmoid, False, False, 1.0)
        np.testing.assert_array_equal(ids.cpu().numpy(), want)


def test_route_near_ties_are_decided_in_64_bits(smb, cuda_device):
    # Scores that fp32 cannot tell apart: bias moves them by less than the rounding of p.
    torch = _torch()
    rng = np.random.default_rng(8)
    tokens, experts = 500, 64
    base = _logits(rng, tokens, 1, 1.0)
    l = (base + 1e-6 * rng.standard_normal((tokens, experts))).astype(np.float32)
    bias = (1e-7 * rng.standard_normal(experts)).astype(np.float32)
    for flags in (0, smb.capi.ROUTE_SIGMOID):
        for groups, top_groups in ((1, 1), (8, 3)):
            _, ids, _ = _route(smb, torch, l, smb.capi.DTYPE_F32, 6, bias, groups, top_groups,
                               flags | smb.capi.ROUTE_GROUP_TOP2)
            want, _ = _route_plain(l.astype(np.float64), bias, 6, groups, top_groups, bool(flags), False, True, 1.0)
            np.testing.assert_array_equal(ids.cpu().numpy(), want)


def test_route_extreme_logits(smb, cuda_device):
    torch = _torch()
    c = smb.capi
    l = np.full((5, 16), -300.0, dtype=np.float32)
    l[0, 5] = np.inf                    # an infinite logit takes everything
    l[1, [2, 9]] = np.inf               # two share
    l[2] = -np.arange(16) * 50 - 200.0  # all probabilities underflow in fp32, their ratios do not
    l[3] = np.float32(3e38)
    l[4, :] = -np.float32(3e38)
    _, ids, w = _route(smb, torch, l, c.DTYPE_F32, 2, flags=c.ROUTE_RENORM)
    assert ids[0, 0] == 5 and ids[1].tolist() == [2, 9] and ids[3].tolist() == [0, 1] and ids[4].tolist() == [0, 1]
    np.testing.assert_allclose(w.cpu().numpy(), [[1, 0], [0.5, 0.5], [1, np.exp(-50)], [0.5, 0.5], [0.5, 0.5]], rtol=2 ** -17)
    _, ids, w = _route(smb, torch, l[2:3], c.DTYPE_F32, 2, flags=c.ROUTE_RENORM | c.ROUTE_SIGMOID)
    np.testing.assert_allclose(w.cpu().numpy(), [[1, np.exp(-50)]], rtol=2 ** -17)


# Groups that are no whole number of a lane's experts, and one whose lanes do not suffice for lanes of their own.
GROUP_CASES = [(70, 36, 8, 2, 1), (300, 160, 6, 8, 3), (65, 144, 6, 8, 3), (40, 48, 6, 8, 1), (33, 16, 2, 8, 3), (20, 304, 4, 8, 2),
               (31, 240, 7, 12, 5), (29, 510, 8, 17, 6), (50, 21, 3, 7, 3), (17, 62, 9, 31, 8), (12, 12, 6, 4, 2)]


@pytest.mark.parametrize("case", GROUP_CASES, ids=str)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_route_groups_of_any_size(smb, cuda_device, case, bf16, pad):
    torch = _torch()
    tokens, experts, top_k, n_groups, top_groups = case
    rng = np.random.default_rng(experts + pad)
    l = _logits(rng, tokens, experts)
    l[1] = -np.inf
    l[2, :experts // 2] = np.nan
    l[3:8] = np.round(l[3:8])                    # ties inside and between groups
    c = smb.capi
    for bias in (None, (0.1 * rng.standard_normal(experts)).astype(np.float32)):
        for sigmoid in (False, True):
            for top2 in (False, True):
                flags = ((c.ROUTE_SIGMOID if sigmoid else 0) | c.ROUTE_RENORM | (c.ROUTE_GROUP_TOP2 if top2 else 0))
                buf, ids, weights = _route(smb, torch, l, c.DTYPE_BF16 if bf16 else c.DTYPE_F32, top_k, bias, n_groups,
                                           top_groups, flags, 2.5, pad=pad)
                want_ids, want = _route_plain(buf[:, :experts].float().cpu().numpy().astype(np.float64), bias, top_k, n_groups,
                                              top_groups, sigmoid, True, top2, 2.5)
                np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
                assert np.all(np.abs(weights.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -17)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("experts", [16, 64, 256, 512])
def test_route_zeros_of_either_sign_tie(smb, cuda_device, sigmoid, bf16, experts):
    """Logits masked by a product are zeros of both signs; they are equal, so the lowest index comes first."""
    torch = _torch()
    c = smb.capi
    rng = np.random.default_rng(experts)
    l = np.where(rng.random((40, experts)) < 0.5, np.float32(0.0), np.float32(-0.0))
    l[1:20, 3::7] = 1.0                       # some above, the rest of the choices among the zeros
    l[5:30, 5::9] = -1.0
    flags = (c.ROUTE_SIGMOID if sigmoid else 0) | c.ROUTE_RENORM
    for groups in (1, 8):
        _, ids, _ = _route(smb, torch, l, c.DTYPE_BF16 if bf16 else c.DTYPE_F32, 8, n_groups=groups, top_groups=max(1, groups // 2),
                           flags=flags)
        want, _ = _route_plain(l.astype(np.float64), None, 8, groups, max(1, groups // 2), sigmoid, True, False, 1.0)
        np.testing.assert_array_equal(ids.cpu().numpy(), want)


# ------------------------------------------------------------------ routing, gradient
def _weights_of(l, ids, sigmoid, renorm, scale):
    """Weights as a function of the logits for fixed ids (float64), for differences."""
    p = _probabilities(l, sigmoid)
    w = np.where(ids >= 0, np.take_along_axis(p, np.maximum(ids, 0), 1), 0.0)
    if renorm:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return w * scale


def _grad_plain(l, ids, g, sigmoid, renorm, scale):
    """Gradient and, for the tolerance, the sum of its terms' magnitudes."""
    p = _probabilities(l, sigmoid)
    tokens, experts = l.shape
    grad, size = np.zeros_like(p), np.zeros_like(p)
    for t in range(tokens):
        js = [j for j in range(ids.shape[1]) if ids[t, j] >= 0]
        e = ids[t, js]
        gj, pj = g[t, js] * scale, p[t, e]
        if renorm:
            q = pj / max(pj.sum(), 1e-300)
            rest = (1 - pj) if sigmoid else np.ones_like(pj)
            np.add.at(grad[t], e, rest * q * (gj - (gj * q).sum()))
            np.add.at(size[t], e, rest * q * (np.abs(gj) + np.abs(gj * q).sum()))
        elif sigmoid:
            np.add.at(grad[t], e, gj * pj * (1 - pj))
            np.add.at(size[t], e, np.abs(gj) * pj * (1 - pj))
        else:
            np.add.at(grad[t], e, gj * pj)
            grad[t] -= p[t] * (gj * pj).sum()
            np.add.at(size[t], e, np.abs(gj) * pj)
            size[t] += p[t] * np.abs(gj * pj).sum()
    return grad, size


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("case", [(1, 1, 1), (6, 40, 3), (70, 64, 6), (33, 256, 8), (9, 500, 32)], ids=str)
def test_route_gradient(smb, cuda_device, case, sigmoid, renorm, bf16):
    torch = _torch()
    tokens, experts, top_k = case
    c = smb.capi
    rng = np.random.default_rng(experts)
    l = _logits(rng, tokens, experts)
    if tokens > 3:
        l[1] = -np.inf
        l[2, experts // 3:] = -np.inf
    flags = (c.ROUTE_SIGMOID if sigmoid else 0) | (c.ROUTE_RENORM if renorm else 0)
    dtype = c.DTYPE_BF16 if bf16 else c.DTYPE_F32
    buf, ids, _ = _route(smb, torch, l, dtype, top_k, flags=flags, scale=1.5, pad=5)
    g = rng.standard_normal((tokens, top_k)).astype(np.float32)
    out = torch.full((tokens, experts + 2), float("nan"), device="cuda", dtype=buf.dtype)
    smb.moe.route_backward_device(buf, ids, torch.from_numpy(g).cuda(), out, tokens, experts, top_k, dtype=dtype, flags=flags,
                                  scale=1.5, ld=experts + 5, ld_grad=experts + 2)
    torch.cuda.synchronize()
    l64 = buf[:, :experts].float().cpu().numpy().astype(np.float64)
    ids_np = ids.cpu().numpy()
    want, size = _grad_plain(l64, ids_np, g.astype(np.float64), sigmoid, renorm, 1.5)
    got = out[:, :experts].float().cpu().numpy()
    assert np.all(np.abs(got - want) <= 2.0 ** -16 * size + (2.0 ** -8 * np.abs(want) if bf16 else 0.0) + 1e-38)
    assert bool(torch.isnan(out[:, experts:].float()).all())
    # The formula itself against central differences.
    for e in rng.integers(0, experts, 3):
        h = 1e-5
        up, down = l64.copy(), l64.copy()
        up[:, e] += h
        down[:, e] -= h
        diff = ((_weights_of(up, ids_np, sigmoid, renorm, 1.5) - _weights_of(down, ids_np, sigmoid, renorm, 1.5)) * g).sum(1) / (2 * h)
        np.testing.assert_allclose(want[:, e], diff, atol=1e-8 * (1 + np.abs(g).sum(1).max()), rtol=1e-6)


def test_route_gradient_same_expert_twice(smb, cuda_device):
    # ids that a caller made itself: an expert named twice gets both shares, ids outside are ignored.
    torch = _torch()
    c = smb.capi
    l = _logits(np.random.default_rng(1), 2, 48)
    ids = np.array([[5, 5, 7], [-1, 47, 99]], dtype=np.int32)
    g = np.array([[1, 2, 3], [4, 5, 6]], dtype=np.float32)
    for flags in (0, c.ROUTE_RENORM, c.ROUTE_SIGMOID, c.ROUTE_SIGMOID | c.ROUTE_RENORM):
        out = torch.full((2, 48), float("nan"), device="cuda")
        smb.moe.route_backward_device(torch.from_numpy(l).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(g).cuda(), out,
                                      2, 48, 3, flags=flags)
        kept = np.where(ids >= 48, -1, ids)
        want, size = _grad_plain(l.astype(np.float64), kept, g.astype(np.float64), bool(flags & c.ROUTE_SIGMOID),
                                 bool(flags & c.ROUTE_RENORM), 1.0)
        assert np.all(np.abs(out.cpu().numpy() - want) <= 2.0 ** -16 * size)


# ------------------------------------------------------------------ rows
def _dispatch_plain(ids, groups, align, cap):
    flat = ids.reshape(-1)
    offsets, row_of_slot, slot_of_row, tiles = [0], np.full(flat.size, -1), np.full(cap, -1), []
    for g in range(groups):
        slots = np.nonzero(flat == g)[0]
        row_of_slot[slots] = offsets[-1] + np.arange(slots.size)
        slot_of_row[offsets[-1]:offsets[-1] + slots.size] = slots
        size = -(-slots.size // align) * align
        tiles += [g] * (size // 256)
        offsets.append(offsets[-1] + size)
    return np.array(offsets), row_of_slot.reshape(ids.shape), slot_of_row, tiles


def _dispatch(smb, torch, ids, groups, align=1, extra=0, tile_map=False):
    tokens, top_k = ids.shape
    cap = smb.moe.max_rows(tokens, top_k, groups, align) + extra
    i32 = dict(device="cuda", dtype=torch.int32)
    offsets = torch.full((groups + 1,), 55, **i32)
    row_of_slot = torch.full((tokens, top_k), 55, **i32)
    slot_of_row = torch.full((max(cap, 1),), 55, **i32)
    tiles = torch.full((max(cap // 256, 1),), 55, **i32) if tile_map else None
    smb.moe.dispatch_device(torch.from_numpy(ids).cuda(), offsets, row_of_slot, slot_of_row, tokens, top_k, groups, cap,
                            align=align, mtile_group=tiles)
    torch.cuda.synchronize()
    return cap, offsets, row_of_slot, slot_of_row, tiles


@pytest.mark.parametrize("case", [
    # tokens, top_k, groups, align
    (1, 1, 1, 1), (1, 8, 256, 1), (16, 8, 256, 1), (5, 3, 7, 4), (100, 2, 16, 128), (333, 6, 64, 256), (1000, 8, 1024, 1),
    (4097, 8, 128, 1), (8192, 8, 64, 256), (20000, 4, 512, 16), (40, 32, 5, 256), (0, 4, 9, 1), (0, 4, 9, 256)], ids=str)
@pytest.mark.parametrize("skew", [0.0, 1.0])
def test_dispatch_against_plain(smb, cuda_device, case, skew):
    torch = _torch()
    tokens, top_k, groups, align = case
    rng = np.random.default_rng(tokens + groups)
    share = np.ones(groups) if skew == 0 else 1.0 / (1 + rng.permutation(groups)) ** 1.5
    ids = rng.choice(groups, size=(tokens, top_k), p=share / share.sum()).astype(np.int32)   # repeats included
    drop = rng.random(ids.shape) < 0.1
    ids = np.where(drop, rng.choice([-1, groups, 2 ** 31 - 1, -2 ** 31], size=ids.shape), ids).astype(np.int32)
    tile_map = align % 256 == 0
    cap, offsets, row_of_slot, slot_of_row, tiles = _dispatch(smb, torch, ids, groups, align, 300, tile_map)
    w_off, w_row, w_slot, w_tiles = _dispatch_plain(ids, groups, align, cap)
    np.testing.assert_array_equal(offsets.cpu().numpy(), w_off)
    np.testing.assert_array_equal(row_of_slot.cpu().numpy(), w_row)
    np.testing.assert_array_equal(slot_of_row.cpu().numpy(), w_slot)
    if tile_map:
        got = tiles.cpu().numpy()
        np.testing.assert_array_equal(got[:len(w_tiles)], w_tiles)
        assert (got[len(w_tiles):cap // 256] == groups - 1).all()


@pytest.mark.parametrize("case", [(10, 6, 388, 256), (3, 2, 1024, 512), (700, 4, 1024, 128), (1, 1, 1, 65536), (60, 1, 33, 4096)],
                         ids=str)
def test_dispatch_with_more_rows_than_slots(smb, cuda_device, case):
    """Few slots, many padded rows and groups: warps without slots help to walk them."""
    torch = _torch()
    tokens, top_k, groups, align = case
    rng = np.random.default_rng(groups)
    ids = rng.integers(-1, groups, size=(tokens, top_k)).astype(np.int32)
    tile_map = align % 256 == 0
    cap, offsets, row_of_slot, slot_of_row, tiles = _dispatch(smb, torch, ids, groups, align, 7000, tile_map)
    w_off, w_row, w_slot, w_tiles = _dispatch_plain(ids, groups, align, cap)
    np.testing.assert_array_equal(offsets.cpu().numpy(), w_off)
    np.testing.assert_array_equal(row_of_slot.cpu().numpy(), w_row)
    np.testing.assert_array_equal(slot_of_row.cpu().numpy(), w_slot)
    if tile_map:
        got = tiles.cpu().numpy()
        np.testing.assert_array_equal(got[:len(w_tiles)], w_tiles)
        assert (got[len(w_tiles):cap // 256] == groups - 1).all()


def _bf16(torch, *shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


ROWS = [(1, 1, 4, 8, 0), (16, 8, 64, 4096, 0), (37, 3, 5, 130, 0), (50, 2, 9, 1, 0), (20, 4, 6, 1024, 8), (9, 6, 30, 1500, 3),
        (300, 8, 16, 768, 0), (11, 32, 40, 2056, 0), (5, 2, 3, 9000, 0)]


def _map(smb, torch, tokens, top_k, groups, seed, extra=5):
    rng = np.random.default_rng(seed)
    ids = rng.integers(-1, groups, size=(tokens, top_k)).astype(np.int32)
    if tokens > 3:
        ids[2] = -1                     # a token without experts
    cap, offsets, row_of_slot, slot_of_row, _ = _dispatch(smb, torch, ids, groups, 1, extra)
    return cap, offsets, row_of_slot, slot_of_row


@pytest.mark.parametrize("case", ROWS, ids=str)
def test_gathers(smb, cuda_device, case):
    torch = _torch()
    tokens, top_k, groups, width, pad = case
    cap, _, row_of_slot, slot_of_row = _map(smb, torch, tokens, top_k, groups, width)
    x = _bf16(torch, tokens, width + pad, seed=width)
    out = torch.full((cap, width + pad), 9.0, device="cuda", dtype=torch.bfloat16)
    smb.moe.gather_bf16_device(x, row_of_slot, out, tokens, top_k, width, cap, ld_x=width + pad, ld_out=width + pad)
    codes = torch.full((cap, width + pad), 55, device="cuda", dtype=torch.int8)
    scales = torch.full((cap,), 55.0, device="cuda")
    smb.moe.gather_i8_device(x, row_of_slot, codes, scales, tokens, top_k, width, cap, ld_x=width + pad, ld_bytes=width + pad)
    torch.cuda.synchronize()
    want_c, want_s = smb.gemm.quantize_i8_host(x[:, :width].float().cpu().numpy())
    slots = slot_of_row.cpu().numpy()
    live = slots >= 0
    token = slots[live] // top_k
    np.testing.assert_array_equal(out.float().cpu().numpy()[live, :width], x.float().cpu().numpy()[token, :width])
    np.testing.assert_array_equal(codes.cpu().numpy()[live, :width], want_c[token])
    np.testing.assert_array_equal(scales.cpu().numpy()[live], want_s[token])
    assert bool((out[~torch.from_numpy(live)] == 9).all()) and bool((out[:, width:] == 9).all())
    assert bool((codes[~torch.from_numpy(live)] == 55).all()) and bool((codes[:, width:] == 55).all())
    assert bool((scales[~torch.from_numpy(live)] == 55).all())


@pytest.mark.parametrize("case", ROWS, ids=str)
@pytest.mark.parametrize("weighted", [True, False])
def test_combine_and_its_gradients(smb, cuda_device, case, weighted):
    torch = _torch()
    tokens, top_k, groups, width, pad = case
    cap, _, row_of_slot, slot_of_row = _map(smb, torch, tokens, top_k, groups, width + 1)
    rows = _bf16(torch, cap, width + pad, seed=1)
    rows[torch.from_numpy(slot_of_row.cpu().numpy() < 0).cuda()] = float("nan")   # rows nobody names are not read
    weights = torch.rand(tokens, top_k, device="cuda") if weighted else None
    y = torch.full((tokens, width + pad), 9.0, device="cuda", dtype=torch.bfloat16)
    smb.moe.combine_device(rows, row_of_slot, weights, y, tokens, top_k, width, cap, ld_rows=width + pad, ld_y=width + pad)
    gy = _bf16(torch, tokens, width + pad, seed=2)
    g_rows = torch.full((cap, width + pad), 9.0, device="cuda", dtype=torch.bfloat16)
    g_w = torch.full((tokens, top_k), 9.0, device="cuda")
    smb.moe.combine_backward_device(gy, rows, row_of_slot, weights, g_rows, g_w, tokens, top_k, width, cap, ld_grad_y=width + pad,
                                    ld_rows=width + pad, ld_grad_rows=width + pad)
    torch.cuda.synchronize()
    at = row_of_slot.long()
    have = at >= 0
    w = torch.where(have, weights.double() if weighted else torch.ones_like(at).double(), torch.zeros_like(at).double())
    picked = torch.where(have[:, :, None], rows[at.clamp_min(0)][:, :, :width].double(), 0.0)
    ref = (picked * w[:, :, None]).sum(1)
    size = (picked * w[:, :, None]).abs().sum(1)
    assert bool(((y[:, :width].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (top_k + 1) * U * size).all())
    assert bool((y[:, width:] == 9).all())
    gyd = gy[:, None, :width].double()
    ref_w = (picked * gyd).sum(2)
    size_w = (picked * gyd).abs().sum(2)
    # A lane adds width / 32 products (+ 8 in the ragged end), five more additions join the lanes.
    assert bool(((g_w.double() - ref_w).abs() <= (width / 32 + 16) * U * size_w).all())
    live = slot_of_row >= 0
    slot = slot_of_row[live].long()
    ref_r = gy[:, :width].double()[slot // top_k] * w.reshape(-1)[slot][:, None]
    got = g_rows[:cap][live[:cap]][:, :width].double()
    assert bool(((got - ref_r).abs() <= (2.0 ** -8 + 2 * U) * ref_r.abs()).all())
    assert bool((g_rows[~live[:cap]] == 9).all()) and bool((g_rows[:, width:] == 9).all())


@pytest.mark.parametrize("width,shift,pad", [(2048, 0, 0), (2048, 1, 0), (2048, 0, 2), (2046, 0, 0), (2046, 2, 0), (2047, 0, 0),
                                             (2047, 0, 1), (700, 4, 4), (33, 3, 0), (5000, 1, 1)])
def test_rows_of_any_alignment(smb, cuda_device, width, shift, pad):
    """Rows in words of 16, 4 and 2 bytes: bases shifted by elements, odd pitches and widths."""
    torch = _torch()
    tokens, top_k, groups = 19, 9, 7
    cap, _, row_of_slot, slot_of_row = _map(smb, torch, tokens, top_k, groups, width + shift)
    ld = width + pad

    def rows(n, fill=None, seed=0):
        buf = torch.full((n * ld + shift,), 9.0, device="cuda", dtype=torch.bfloat16) if fill else _bf16(torch, n * ld + shift, seed=seed)
        return buf[shift:].view(n, ld)

    x, out, e, y, g = rows(tokens, seed=1), rows(cap, fill=True), rows(cap, seed=2), rows(tokens, fill=True), rows(cap, fill=True)
    weights, gw = torch.rand(tokens, top_k, device="cuda"), torch.full((tokens, top_k), 9.0, device="cuda")
    codes = torch.full((cap, ld), 55, device="cuda", dtype=torch.int8)
    scales = torch.full((cap,), 55.0, device="cuda")
    args = (tokens, top_k, width, cap)
    smb.moe.gather_bf16_device(x, row_of_slot, out, *args, ld_x=ld, ld_out=ld)
    smb.moe.gather_i8_device(x, row_of_slot, codes, scales, *args, ld_x=ld, ld_bytes=ld)
    smb.moe.combine_device(e, row_of_slot, weights, y, *args, ld_rows=ld, ld_y=ld)
    smb.moe.combine_backward_device(x, e, row_of_slot, weights, g, gw, *args, ld_grad_y=ld, ld_rows=ld, ld_grad_rows=ld)
    torch.cuda.synchronize()
    live = slot_of_row >= 0
    slot = slot_of_row[live].long()
    token = slot // top_k
    assert torch.equal(out[live[:cap]][:, :width], x[token][:, :width])
    assert bool((out[~live[:cap]] == 9).all()) and bool((out[:, width:] == 9).all())
    want_c, want_s = smb.gemm.quantize_i8_host(x[:, :width].float().cpu().numpy())
    np.testing.assert_array_equal(codes[live[:cap]].cpu().numpy()[:, :width], want_c[token.cpu().numpy()])
    np.testing.assert_array_equal(scales[live[:cap]].cpu().numpy(), want_s[token.cpu().numpy()])
    have = row_of_slot >= 0
    picked = torch.where(have[:, :, None], e[row_of_slot.long().clamp_min(0)][:, :, :width].double(), 0.0)
    terms = picked * weights.double()[:, :, None]
    assert bool(((y[:, :width].double() - terms.sum(1)).abs() <= 2.0 ** -8 * terms.sum(1).abs() + (top_k + 1) * U * terms.abs().sum(1)).all())
    prod = picked * x[:, None, :width].double()
    assert bool(((gw.double() - prod.sum(2)).abs() <= (width / 32 + 16) * U * prod.abs().sum(2)).all())
    ref = x[token][:, :width].double() * weights.reshape(-1)[slot].double()[:, None]
    assert bool(((g[live[:cap]][:, :width].double() - ref).abs() <= (2.0 ** -8 + 2 * U) * ref.abs()).all())
    assert bool((g[~live[:cap]] == 9).all()) and bool((y[:, width:] == 9).all())


def test_rows_outside_the_buffer_are_skipped(smb, cuda_device):
    torch = _torch()
    tokens, top_k, width, cap = 4, 2, 64, 6
    row_of_slot = torch.tensor([[0, 6], [5, -3], [2 ** 31 - 1, 1], [-1, 700]], device="cuda", dtype=torch.int32)
    x = _bf16(torch, tokens, width, seed=3)
    out = torch.zeros(cap, width, device="cuda", dtype=torch.bfloat16)
    smb.moe.gather_bf16_device(x, row_of_slot, out, tokens, top_k, width, cap)
    y = torch.ones(tokens, width, device="cuda", dtype=torch.bfloat16)
    smb.moe.combine_device(out, row_of_slot, None, y, tokens, top_k, width, cap)
    torch.cuda.synchronize()
    assert torch.equal(out[0], x[0]) and torch.equal(out[5], x[1]) and torch.equal(out[1], x[2])
    assert not bool(out[2:5].any())
    assert torch.equal(y[:3], x[:3]) and not bool(y[3].any())


def test_gather_gradient_is_the_plain_sum(smb, cuda_device):
    torch = _torch()
    tokens, top_k, groups, width = 30, 4, 6, 200
    cap, _, row_of_slot, slot_of_row = _map(smb, torch, tokens, top_k, groups, 3)
    g = _bf16(torch, cap, width, seed=4)
    gx = torch.zeros(tokens, width, device="cuda", dtype=torch.bfloat16)
    smb.moe.combine_device(g, row_of_slot, None, gx, tokens, top_k, width, cap)
    live = slot_of_row >= 0
    ref = torch.zeros(tokens, width, device="cuda", dtype=torch.float64)
    ref.index_add_(0, (slot_of_row[live] // top_k).long(), g[:cap][live[:cap]].double())
    size = torch.zeros_like(ref).index_add_(0, (slot_of_row[live] // top_k).long(), g[:cap][live[:cap]].double().abs())
    assert bool(((gx.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 5 * U * size).all())


# ------------------------------------------------------------------ the operators together
class _Layer:
    """An int8 expert layer as a program holds it: weights, buffers and two grouped plans."""

    def __init__(self, smb, torch, tokens, experts, top_k, width, hidden, flags=0):
        self.smb, self.torch = smb, torch
        self.dims = (tokens, experts, top_k, width, hidden)
        g = torch.Generator(device="cuda")
        g.manual_seed(2)

        def weights(rows, k):
            w = torch.randn(rows, k, generator=g, device="cuda") / k ** 0.5
            codes = torch.zeros(rows, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)
            scales = torch.zeros(rows, device="cuda")
            smb.gemm.quantize_i8_device(w, codes, scales, rows, k, ld_bytes=codes.shape[1])
            return codes, scales

        self.b1, self.sb1 = weights(experts * 2 * hidden, width)
        self.b2, self.sb2 = weights(experts * width, hidden)
        self.cap = cap = smb.moe.max_rows(tokens, top_k, experts)
        i32 = dict(device="cuda", dtype=torch.int32)
        bf = dict(device="cuda", dtype=torch.bfloat16)
        self.x = torch.zeros(tokens, width, **bf)
        self.logits = torch.zeros(tokens, experts, device="cuda")
        self.ids, self.w = torch.zeros(tokens, top_k, **i32), torch.zeros(tokens, top_k, device="cuda")
        self.offsets, self.row, self.slot = (torch.zeros(experts + 1, **i32), torch.zeros(tokens, top_k, **i32),
                                             torch.zeros(cap, **i32))
        self.a1 = torch.zeros(cap, (width + 15) // 16 * 16, device="cuda", dtype=torch.int8)
        self.a2 = torch.zeros(cap, (hidden + 15) // 16 * 16, device="cuda", dtype=torch.int8)
        self.s1, self.s2 = torch.zeros(cap, device="cuda"), torch.zeros(cap, device="cuda")
        self.h, self.out = torch.zeros(cap, hidden, **bf), torch.zeros(cap, width, **bf)
        self.y = torch.zeros(tokens, width, **bf)
        plan = smb.gemm.I8Plan.grouped
        self.p1 = plan(self.a1, self.s1, self.b1, self.sb1, self.h, cap, 2 * hidden, width, experts, self.offsets,
                       lda=self.a1.shape[1], ldb=self.b1.shape[1], flags=flags | smb.capi.FLAG_EPILOGUE_SWIGLU)
        self.p2 = plan(self.a2, self.s2, self.b2, self.sb2, self.out, cap, width, hidden, experts, self.offsets,
                       lda=self.a2.shape[1], ldb=self.b2.shape[1], flags=flags)

    def run(self, stream=None):
        tokens, experts, top_k, width, hidden = self.dims
        moe, c = self.smb.moe, self.smb.capi
        moe.route_device(self.logits, self.ids, self.w, tokens, experts, top_k, flags=c.ROUTE_RENORM, stream=stream)
        moe.dispatch_device(self.ids, self.offsets, self.row, self.slot, tokens, top_k, experts, self.cap, stream=stream)
        moe.gather_i8_device(self.x, self.row, self.a1, self.s1, tokens, top_k, width, self.cap, ld_bytes=self.a1.shape[1],
                             stream=stream)
        self.p1.run(stream)
        self.smb.gemm.quantize_i8_bf16_device(self.h, self.a2, self.s2, self.cap, hidden, ld_bytes=self.a2.shape[1],
                                              stream=stream)
        self.p2.run(stream)
        moe.combine_device(self.out, self.row, self.w, self.y, tokens, top_k, width, self.cap, stream=stream)

    def expected(self):
        """float64 chain with the stored roundings (codes, bf16 hidden state) and the error it allows."""
        torch = self.torch
        tokens, experts, top_k, width, hidden = self.dims

        def codes(x):
            c, s = self.smb.gemm.quantize_i8_host(x.float().cpu().numpy())
            return torch.from_numpy(c).cuda().double(), torch.from_numpy(s).cuda().double()

        ids, w = _route_plain(self.logits.cpu().numpy().astype(np.float64), None, top_k, 1, 1, False, True, False, 1.0)
        c1, s1 = codes(self.x)
        y = torch.zeros(tokens, width, device="cuda", dtype=torch.float64)
        size = torch.zeros_like(y)
        for e in range(experts):
            t, j = np.nonzero(ids == e)
            if t.size == 0:
                continue
            t = torch.from_numpy(t).cuda()
            wt = torch.from_numpy(w[t.cpu().numpy(), j]).cuda()[:, None]
            sl1, sl2 = slice(e * 2 * hidden, (e + 1) * 2 * hidden), slice(e * width, (e + 1) * width)
            z = (c1[t] @ self.b1[sl1, :width].double().t()) * s1[t][:, None] * self.sb1[sl1].double()
            h = (z[:, 0::2] * z[:, 1::2] / (1 + torch.exp(-z[:, 1::2]))).bfloat16()
            c2, s2 = codes(h)
            b2 = self.b2[sl2, :hidden].double()
            scale = s2[:, None] * self.sb2[sl2].double()
            o = (c2 @ b2.t()) * scale
            y.index_add_(0, t, o * wt)
            # A hidden value next to a rounding border may move by one bf16 step and with it by one code.
            size.index_add_(0, t, (o.abs() * 2.0 ** -8 + scale * b2.abs().amax(1)) * wt)
        return ids, w, y, size


@pytest.mark.parametrize("case", [(1, 8, 2, 128, 64), (40, 16, 4, 256, 136), (300, 8, 3, 520, 200), (64, 64, 8, 512, 256)], ids=str)
def test_expert_layer_eager_and_captured(smb, cuda_device, case):
    torch = _torch()
    layer = _Layer(smb, torch, *case)
    tokens, experts, top_k, width, hidden = case
    stream = torch.cuda.Stream()
    graph = None
    for trial in range(3):
        g = torch.Generator(device="cuda")
        g.manual_seed(trial)
        layer.x.copy_(torch.randn(tokens, width, generator=g, device="cuda"))
        layer.logits.copy_(torch.randn(tokens, experts, generator=g, device="cuda"))
        if trial == 2 and tokens > 4:
            layer.logits[1:4] = -float("inf")    # a batch that ends in padding
        torch.cuda.synchronize()
        if trial == 0:
            layer.run(stream)
            layer.p1.check(stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                layer.run(stream)
        else:
            graph.replay()
            torch.cuda.synchronize()
        if trial == 0:
            layer.p2.check(stream)
        ids, w, y, size = layer.expected()
        np.testing.assert_array_equal(layer.ids.cpu().numpy(), ids)
        # Two hidden values of a row may sit on a border; one more rounding of y.
        err = (layer.y.double() - y).abs()
        assert bool((err <= 2.0 ** -8 * y.abs() + 2 * size + 1e-30).all())
    layer.p1.check(stream)
    layer.p2.check(stream)


def test_router_feeds_the_bf16_grouped_plan(smb, cuda_device):
    # The layout with 256-row groups and the tile map is what Bf16Plan.grouped takes.
    torch = _torch()
    tokens, experts, top_k, width, n = 500, 6, 2, 192, 264
    logits = torch.randn(tokens, experts, device="cuda")
    ids = torch.zeros(tokens, top_k, device="cuda", dtype=torch.int32)
    w = torch.zeros(tokens, top_k, device="cuda")
    smb.moe.route_device(logits, ids, w, tokens, experts, top_k, flags=smb.capi.ROUTE_RENORM)
    cap, offsets, row, slot, tiles = _dispatch(smb, torch, ids.cpu().numpy(), experts, 256, 0, True)
    x = _bf16(torch, tokens, width, seed=1)
    a = torch.zeros(cap, width, device="cuda", dtype=torch.bfloat16)
    b = _bf16(torch, experts * n, width, seed=2)
    d = torch.zeros(cap, n, device="cuda", dtype=torch.bfloat16)
    smb.moe.gather_bf16_device(x, row, a, tokens, top_k, width, cap)
    plan = smb.gemm.Bf16Plan.grouped(a, b, d, cap, n, width, experts, tiles)
    plan.run()
    plan.check()
    y = torch.zeros(tokens, n, device="cuda", dtype=torch.bfloat16)
    smb.moe.combine_device(d, row, w, y, tokens, top_k, n, cap)
    torch.cuda.synchronize()
    ref = torch.zeros(tokens, n, device="cuda", dtype=torch.float64)
    size = torch.zeros_like(ref)
    for j in range(top_k):
        per = torch.stack([b[int(e) * n:(int(e) + 1) * n].double() for e in range(experts)])[ids[:, j].long()]
        term = torch.einsum("tk,tnk->tn", x.double(), per) * w[:, j:j + 1].double()
        mags = torch.einsum("tk,tnk->tn", x.double().abs(), per.abs()) * w[:, j:j + 1].double()
        ref += term
        # bf16 rounding of the stored product, fp32 sums of width products.
        size += term.abs() * 2.0 ** -8 + mags * (width * U)
    assert bool(((y.double() - ref).abs() <= size * 1.01 + 2.0 ** -8 * ref.abs() + 4 * U * size).all())


def test_rows_on_another_stream(smb, cuda_device):
    torch = _torch()
    stream = torch.cuda.Stream()
    tokens, top_k, groups, width = 64, 4, 12, 512
    x = _bf16(torch, tokens, width, seed=6)
    logits = torch.randn(tokens, groups, device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    ids, w = torch.zeros(tokens, top_k, **i32), torch.zeros(tokens, top_k, device="cuda")
    cap = smb.moe.max_rows(tokens, top_k, groups)
    offsets, row, slot = torch.zeros(groups + 1, **i32), torch.zeros(tokens, top_k, **i32), torch.zeros(cap, **i32)
    a, y = torch.zeros(cap, width, device="cuda", dtype=torch.bfloat16), torch.zeros_like(x)
    torch.cuda.synchronize()
    smb.moe.route_device(logits, ids, w, tokens, groups, top_k, flags=smb.capi.ROUTE_RENORM, stream=stream)
    smb.moe.dispatch_device(ids, offsets, row, slot, tokens, top_k, groups, cap, stream=stream)
    smb.moe.gather_bf16_device(x, row, a, tokens, top_k, width, cap, stream=stream)
    smb.moe.combine_device(a, row, w, y, tokens, top_k, width, cap, stream=stream)
    stream.synchronize()
    # Weights add up to one, every copy is the token itself.
    assert bool(((y.double() - x.double()).abs() <= 2.0 ** -8 * x.double().abs() + 64 * U * x.double().abs()).all())


@pytest.mark.parametrize("case", [(500, 256, 8, 8, 4), (300, 160, 6, 8, 3), (200, 510, 8, 17, 6), (400, 64, 4, 4, 2)], ids=str)
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("size", [1.0, 16.0, 64.0])
def test_route_group_sums_that_cancel(smb, cuda_device, case, sigmoid, size):
    """Biases of either sign: a group's two best scores are +-size + p and all but cancel, so their sum is far smaller
    than what its rounding goes by.  The 64-bit sums differ by 1e-5 and are off by 2^-45."""
    torch = _torch()
    tokens, experts, top_k, n_groups, top_groups = case
    rng = np.random.default_rng(int(size) + experts + sigmoid)
    l = _logits(rng, tokens, experts, 1e-3 if sigmoid else 1e-2)
    bias = np.full(experts, -size, dtype=np.float32)
    per = experts // n_groups
    bias[np.arange(n_groups) * per + rng.integers(0, per, n_groups)] = size
    flags = smb.capi.ROUTE_GROUP_TOP2 | (smb.capi.ROUTE_SIGMOID if sigmoid else 0)
    _, ids, _ = _route(smb, torch, l, smb.capi.DTYPE_F32, top_k, bias, n_groups, top_groups, flags)
    want, _ = _route_plain(l.astype(np.float64), bias, top_k, n_groups, top_groups, sigmoid, False, True, 1.0)
    np.testing.assert_array_equal(ids.cpu().numpy(), want)


def test_dispatch_histograms_just_below_the_default_shared_memory(tmp_path):
    """Histograms of 47.9 to 48 KB, in a process whose first calls they are: nothing has raised the kernel's limit
    before.  The last case sorts on a cluster."""
    import subprocess
    import sys
    script = tmp_path / "first_calls.py"
    script.write_text("""
import sys
sys.path[:0] = [%r, %r]
import numpy as np, torch
import conftest, test_moe_gpu as t
smb = conftest.load_package()
for tokens, top_k, groups in [(84, 8, 512), (81, 8, 512), (116, 8, 384), (36, 8, 1024), (48, 8, 768), (128, 8, 351), (2500, 8, 351)]:
    ids = np.random.default_rng(groups).integers(-1, groups, size=(tokens, top_k)).astype(np.int32)
    cap, offsets, rows, slots, _ = t._dispatch(smb, torch, ids, groups)
    want = t._dispatch_plain(ids, groups, 1, cap)
    for got, ref in zip((offsets, rows, slots), want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
print("all equal")
""" % (str(ROOT), str(ROOT / "tests")))
    run = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all equal" in run.stdout, run.stdout + run.stderr


def test_route_of_bf16_without_a_word_about_the_type(smb, cuda_device):
    torch = _torch()
    c = smb.capi
    l = torch.from_numpy(_logits(np.random.default_rng(3), 50, 64)).cuda().bfloat16()
    out = []
    for dtype in (None, c.DTYPE_BF16):
        ids, w = torch.zeros(50, 4, device="cuda", dtype=torch.int32), torch.zeros(50, 4, device="cuda")
        grad = torch.zeros_like(l)
        smb.moe.route_device(l, ids, w, 50, 64, 4, dtype=dtype)
        smb.moe.route_backward_device(l, ids, w, grad, 50, 64, 4, dtype=dtype)
        out.append((ids, w, grad))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert torch.equal(out[0][0].long(), l.float().sort(descending=True, stable=True).indices[:, :4])


def test_router_feeds_the_fp4_grouped_plan(smb, cuda_device):
    """Routed rows, quantised to FP4 in groups of whole 256-row tiles, against a dense FP4 product of all tokens with
    every expert: the same codes and scales, so the same bits in every row that a slot names."""
    torch = _torch()
    tokens, experts, top_k, width, n = 300, 5, 2, 256, 384
    lib, u8 = smb.capi.lib(), dict(device="cuda", dtype=torch.uint8)

    def quantised(rows):
        codes = torch.empty(rows.shape[0], width // 2, **u8)
        scales = torch.empty(smb.gemm.sf_packed_bytes(rows.shape[0], width), **u8)
        smb.capi.check(lib.smb_quantize_mx_bf16_device(rows.data_ptr(), width, codes.data_ptr(), width // 2, scales.data_ptr(),
                                                       None, rows.shape[0], width, None))
        return codes, scales

    logits = torch.randn(tokens, experts, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    logits[7] = float("-inf")           # a padding token goes nowhere
    ids = torch.zeros(tokens, top_k, device="cuda", dtype=torch.int32)
    w = torch.zeros(tokens, top_k, device="cuda")
    smb.moe.route_device(logits, ids, w, tokens, experts, top_k, flags=smb.capi.ROUTE_RENORM)
    cap, offsets, row, slot, tiles = _dispatch(smb, torch, ids.cpu().numpy(), experts, 256, 0, True)
    x, weights = _bf16(torch, tokens, width, seed=1), _bf16(torch, experts * n, width, seed=2)
    a = torch.zeros(cap, width, device="cuda", dtype=torch.bfloat16)
    smb.moe.gather_bf16_device(x, row, a, tokens, top_k, width, cap)
    qa, qb, qx = quantised(a), quantised(weights), quantised(x)
    d = torch.zeros(cap, n, device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.Fp4Plan.grouped(*qa, *qb, d, cap, n, width, experts, tiles)
    plan.run()
    plan.check()
    y = torch.zeros(tokens, n, device="cuda", dtype=torch.bfloat16)
    smb.moe.combine_device(d, row, w, y, tokens, top_k, n, cap)
    dense = []
    for e in range(experts):
        qe, out = quantised(weights[e * n:(e + 1) * n].contiguous()), torch.zeros(tokens, n, device="cuda", dtype=torch.bfloat16)
        one = smb.gemm.Fp4Plan(*qx, *qe, out, tokens, n, width)
        one.run()
        one.check()
        dense.append(out)
    dense = torch.stack(dense)
    ref, size = torch.zeros(tokens, n, device="cuda", dtype=torch.float64), 0.0
    for j in range(top_k):
        live = ids[:, j] >= 0
        assert bool((live == (row[:, j] >= 0)).all()) and int((~live).sum()) == 1
        part = dense[ids[live, j].long(), live.nonzero()[:, 0]]
        assert torch.equal(d[row[live, j].long()], part)
        ref[live] += part.double() * w[live, j:j + 1].double()
        size = size + (dense.abs().amax(0).double() * w[:, j:j + 1].double())
    # Two fused multiply-adds and one rounding to bf16.
    assert bool(((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 4 * U * size).all())
    assert not bool(y[7].any())
