"""int8 GEMM and quantiser on the GPU against 64-bit arithmetic.

Tolerances.  The int32 sum is exact, so the product has three fp32 roundings (int to float, two scale
products: 2^-24 each) and one to bf16 (2^-8): the plain product is compared bit for bit with the same
roundings applied to the exact sum, and with the float64 value within 2^-8 + 4 * 2^-24 relative.  The
gated form adds exp and a division: a relative error r of z changes silu(z) by (1 + |z|) r, and the
hardware exponential and divide are within (|z| + 4) * 2^-23, together below (|z| + 8) * 2^-21.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _codes(torch, rows, k, seed, ld=None):
    """int8 codes over the whole range at a pitch of 16 bytes; what lies behind a row is not zero."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ld = (k + 15) // 16 * 16 if ld is None else ld
    return torch.randint(-128, 128, (rows, ld), generator=g, device="cuda", dtype=torch.int8)


def _scales(torch, rows, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.exp(torch.randn(rows, generator=g, device="cuda")) * 0.01


def _sums(torch, a, b, k):
    return a[:, :k].double() @ b[:, :k].double().t()


def _expect_bits(torch, acc, sa, sb):
    """bf16 with the kernels' roundings, from the exact sum."""
    return (acc.float() * sa[:, None] * sb[None, :]).bfloat16()


def _check(torch, d, acc, sa, sb):
    want = _expect_bits(torch, acc, sa, sb)
    assert torch.equal(d.view(torch.int16), want.view(torch.int16))
    ref = acc * sa.double()[:, None] * sb.double()[None, :]
    assert bool(((d.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -22)).all())


def _check_gated(torch, d, acc, sa, sb):
    z = acc * sa.double()[:, None] * sb.double()[None, :]
    up, gate = z[:, 0::2], z[:, 1::2]
    ref = up * gate / (1.0 + torch.exp(-gate))
    bound = ref.abs() * (2.0 ** -8 + (gate.abs() + 8) * 2.0 ** -21) + up.abs() * 2.0 ** -100
    assert bool(((d.double() - ref).abs() <= bound).all())


def _run(smb, torch, m, n, k, flags=0, ldd=None, group_m=0, clusters=0, seed=3):
    a, b = _codes(torch, m, k, seed), _codes(torch, n, k, seed + 1)
    sa, sb = _scales(torch, m, seed + 2), _scales(torch, n, seed + 3)
    wide = n // 2 if flags & smb.capi.FLAG_EPILOGUE_SWIGLU else n
    ldd = wide if ldd is None else ldd
    d = torch.full((m, ldd), float("nan"), device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k, lda=a.shape[1], ldb=b.shape[1], ldd=ldd, flags=flags)
    if group_m or clusters:
        plan.tune(group_m, clusters)
    plan.run()
    plan.check()
    plan.close()
    return a, sa, b, sb, d


SHAPES = [(1, 1, 1), (1, 4096, 4096), (16, 28672, 512), (7, 130, 17), (33, 257, 1000), (256, 256, 128), (300, 512, 384),
          (1000, 777, 1040), (129, 2048, 2048), (2048, 96, 640), (4095, 1229, 416), (64, 4096, 8192), (128, 1000, 300),
          (200, 3000, 96)]


@pytest.mark.parametrize("shape", SHAPES)
def test_i8_shapes_bit_for_bit(smb, cuda_device, shape):
    torch = _torch()
    m, n, k = shape
    a, sa, b, sb, d = _run(smb, torch, m, n, k)
    _check(torch, d, _sums(torch, a, b, k), sa, sb)


@pytest.mark.parametrize("flags_name", ["FLAG_TILE_N_128", "FLAG_TILE_N_256", "FLAG_TILE_N_512"])
@pytest.mark.parametrize("store", ["FLAG_NONE", "FLAG_FORCE_PLAIN_STORE"])
@pytest.mark.parametrize("walk", [(0, 0), (3, 2)])
def test_i8_every_tile_configuration(smb, cuda_device, flags_name, store, walk):
    torch = _torch()
    m, n, k = 1100, 1600, 1300
    flags = getattr(smb.capi, flags_name) | getattr(smb.capi, store) | smb.capi.FLAG_NO_DECODE
    a, sa, b, sb, d = _run(smb, torch, m, n, k, flags=flags, group_m=walk[0], clusters=walk[1])
    _check(torch, d, _sums(torch, a, b, k), sa, sb)


def test_i8_extreme_codes_do_not_wrap(smb, cuda_device):
    # The largest sum there is, 131071 products of -128 * -128 = 2^31 - 2^14; and one of opposite sign.
    torch = _torch()
    m, n, k = 3, 5, 131071
    ld = 131072
    a = torch.full((m, ld), -128, device="cuda", dtype=torch.int8)
    b = torch.full((n, ld), -128, device="cuda", dtype=torch.int8)
    b[1] = 127
    sa, sb = _scales(torch, m, 1), _scales(torch, n, 2)
    d = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k, lda=ld, ldb=ld)
    plan.run()
    plan.check()
    _check(torch, d, _sums(torch, a, b, k), sa, sb)


@pytest.mark.parametrize("shape", [(209, 43, 5141), (1024, 256, 8192), (296, 189, 3759), (48, 1024, 512), (64, 1024, 1024),
                                   (100, 512, 1024), (33, 2048, 2048), (1, 1024, 512), (16, 1024, 640), (555, 7452, 190),
                                   (1151, 4039, 90), (150, 2694, 1972)])
def test_i8_choice_of_kernel_and_split(smb, cuda_device, shape):
    """On either side of the rules that cut the K loop or pick a tile width; forced the other way, the bits agree."""
    torch = _torch()
    m, n, k = shape
    a, sa, b, sb, d = _run(smb, torch, m, n, k)
    _check(torch, d, _sums(torch, a, b, k), sa, sb)
    for flag in (smb.capi.FLAG_NO_DECODE, smb.capi.FLAG_DECODE_SINGLE):
        assert torch.equal(_run(smb, torch, m, n, k, flags=flag)[4].view(torch.int16), d.view(torch.int16))


@pytest.mark.parametrize("n", [64, 130, 191, 256, 321])
@pytest.mark.parametrize("pad", [0, 1, 2, 3])
@pytest.mark.parametrize("tile", ["FLAG_TILE_N_128", "FLAG_TILE_N_256", "FLAG_TILE_N_512"])
def test_i8_plain_store_alignments(smb, cuda_device, n, pad, tile):
    """Whole boxes by pairs and by elements, boxes that end inside M or N, from a base of odd elements too."""
    torch = _torch()
    m, k = 301, 160
    a, b = _codes(torch, m, k, 7), _codes(torch, n, k, 8)
    sa, sb = _scales(torch, m, 9), _scales(torch, n, 10)
    want = _expect_bits(torch, _sums(torch, a, b, k), sa, sb)
    ldd = n + pad
    for shift in (0, 1, 2):
        buf = torch.full((shift + m * ldd + 8,), 9.0, device="cuda", dtype=torch.bfloat16)
        d = buf[shift:shift + m * ldd].view(m, ldd)
        flags = getattr(smb.capi, tile) | smb.capi.FLAG_FORCE_PLAIN_STORE
        plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k, lda=a.shape[1], ldb=b.shape[1], ldd=ldd, flags=flags)
        plan.run()
        plan.check()
        plan.close()
        assert torch.equal(d[:, :n].view(torch.int16), want.view(torch.int16))
        assert bool((d[:, n:] == 9).all()) and bool((buf[:shift] == 9).all()) and bool((buf[shift + m * ldd:] == 9).all())


@pytest.mark.parametrize("n", [1, 7, 30, 66, 130, 381, 514])
@pytest.mark.parametrize("tile", ["FLAG_NONE", "FLAG_TILE_N_128", "FLAG_TILE_N_256", "FLAG_TILE_N_512", "FLAG_DECODE_SINGLE"])
@pytest.mark.parametrize("gated", [False, True])
def test_i8_columns_of_a_wider_matrix(smb, cuda_device, n, tile, gated):
    """D is the left part of a matrix whose other columns belong to someone else: a row that ends inside 16
    bytes ends there, in tiles and in ragged groups."""
    torch = _torch()
    n += n % 2 if gated else 0
    wide, k, groups = n // 2 if gated else n, 96, 3
    ldd = (wide + 7) // 8 * 8 + 8
    flags = getattr(smb.capi, tile) | (smb.capi.FLAG_EPILOGUE_SWIGLU if gated else 0)
    for m, cuts in ((40, None), (300, None), (333, [0, 70, 71, 330])):
        a, b = _codes(torch, m, k, 11), _codes(torch, groups * n, k, 12)
        sa, sb = _scales(torch, m, 13), _scales(torch, groups * n, 14)
        d = torch.full((m, ldd), 7.0, device="cuda", dtype=torch.bfloat16)
        args = dict(lda=a.shape[1], ldb=b.shape[1], ldd=ldd, flags=flags)
        if cuts is None:
            plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k, **args)
        else:
            offsets = torch.tensor(cuts, device="cuda", dtype=torch.int32)
            plan = smb.gemm.I8Plan.grouped(a, sa, b, sb, d, m, n, k, groups, offsets, **args)
        plan.run()
        plan.check()
        plan.close()
        for g, (lo, hi) in enumerate(zip(*((cuts[:-1], cuts[1:]) if cuts else ([0], [m])))):
            acc = _sums(torch, a[lo:hi], b[g * n:(g + 1) * n], k)
            check = _check_gated if gated else _check
            check(torch, d[lo:hi, :wide], acc, sa[lo:hi], sb[g * n:(g + 1) * n])
        assert bool((d[:, wide:] == 7).all()) and (cuts is None or bool((d[cuts[-1]:] == 7).all()))


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("ldd", [104, 101])
def test_i8_pitched_output_keeps_its_padding(smb, cuda_device, m, ldd):
    torch = _torch()
    n, k = 96, 256
    a, sa, b, sb, d = _run(smb, torch, m, n, k, ldd=ldd)
    _check(torch, d[:, :n].contiguous(), _sums(torch, a, b, k), sa, sb)
    assert bool(torch.isnan(d[:, n:].float()).all())


@pytest.mark.parametrize("shape", [(1, 64, 48), (16, 4096, 2048), (300, 512, 256), (1030, 1552, 640), (100, 2064, 1000)])
@pytest.mark.parametrize("tile", ["FLAG_NONE", "FLAG_TILE_N_512", "FLAG_DECODE_SINGLE"])
def test_i8_gated_epilogue(smb, cuda_device, shape, tile):
    torch = _torch()
    m, n, k = shape
    flags = smb.capi.FLAG_EPILOGUE_SWIGLU | getattr(smb.capi, tile)
    a, b = _codes(torch, m, k, 5), _codes(torch, n, k, 6)
    # Gates of a few units of either sign, some far out where silu is almost 0 or almost the identity.
    sa = torch.ones(m, device="cuda")
    sb = torch.full((n,), 4.0 / (74 * 74 * k ** 0.5), device="cuda") * torch.where(
        torch.arange(n, device="cuda") % 7 == 1, 30.0, 1.0)
    d = torch.full((m, n // 2), float("nan"), device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k, lda=a.shape[1], ldb=b.shape[1], flags=flags)
    plan.run()
    plan.check()
    _check_gated(torch, d, _sums(torch, a, b, k), sa, sb)


def _run_grouped(smb, torch, sizes, n, k, flags=0, slack=0, seed=9):
    groups, rows = len(sizes), int(sum(sizes))
    cap = max(1, rows + slack)
    ends = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    offsets = torch.tensor(ends, device="cuda")
    a, b = _codes(torch, cap, k, seed), _codes(torch, groups * n, k, seed + 1)
    gated = bool(flags & smb.capi.FLAG_EPILOGUE_SWIGLU)
    sa = _scales(torch, cap, seed + 2)
    sb = _scales(torch, groups * n, seed + 3)
    if gated:
        sa, sb = torch.ones_like(sa), torch.full_like(sb, 4.0 / (74 * 74 * k ** 0.5))
    wide = n // 2 if gated else n
    d = torch.full((cap, wide), float("nan"), device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan.grouped(a, sa, b, sb, d, cap, n, k, groups, offsets, lda=a.shape[1], ldb=b.shape[1], flags=flags)
    return plan, ends, offsets, a, sa, b, sb, d


def _check_grouped(torch, ends, n, k, a, sa, b, sb, d, gated):
    for g in range(len(ends) - 1):
        lo, hi = int(ends[g]), int(ends[g + 1])
        if hi > lo:
            acc = _sums(torch, a[lo:hi], b[g * n:(g + 1) * n], k)
            (_check_gated if gated else _check)(torch, d[lo:hi], acc, sa[lo:hi], sb[g * n:(g + 1) * n])
    assert bool(torch.isnan(d[int(ends[-1]):].float()).all()), "rows behind the last group were written"


GROUPS = [((300, 0, 77, 512, 1), 384, 256), ((0, 0, 1), 130, 100), ((1,) * 40, 264, 528), ((0, 5, 0, 2000, 3), 520, 130),
          ((17, 33, 64, 65, 128, 129, 255, 256, 257), 256, 384), ((3, 0, 9, 0, 0, 31, 2, 1), 1544, 2048),
          (tuple(i % 5 for i in range(512)), 24, 40), ((700, 600), 2056, 1100)]


@pytest.mark.parametrize("case", GROUPS, ids=lambda c: f"{len(c[0])}x{c[1]}x{c[2]}")
@pytest.mark.parametrize("mode", ["plain", "gated", "no_decode", "wide", "plain_store", "decode", "decode_gated", "tiled_gated",
                                  "tiled_plain_store"])
def test_i8_grouped_ragged(smb, cuda_device, case, mode):
    torch = _torch()
    sizes, n, k = case
    c = smb.capi
    flags = {"plain": 0, "gated": c.FLAG_EPILOGUE_SWIGLU, "no_decode": c.FLAG_NO_DECODE,
             "wide": c.FLAG_NO_DECODE | c.FLAG_TILE_N_512, "plain_store": c.FLAG_FORCE_PLAIN_STORE,
             "tiled_gated": c.FLAG_NO_DECODE | c.FLAG_EPILOGUE_SWIGLU,
             "tiled_plain_store": c.FLAG_NO_DECODE | c.FLAG_FORCE_PLAIN_STORE, "decode": c.FLAG_DECODE_SINGLE, "decode_gated": c.FLAG_DECODE_SINGLE | c.FLAG_EPILOGUE_SWIGLU}[mode]
    if mode.endswith("gated"):
        n = (n + 15) // 16 * 16
    plan, ends, offsets, a, sa, b, sb, d = _run_grouped(smb, torch, sizes, n, k, flags, slack=40)
    plan.run()
    plan.check()
    _check_grouped(torch, ends, n, k, a, sa, b, sb, d, mode.endswith("gated"))


@pytest.mark.parametrize("mode", ["FLAG_DECODE_SINGLE", "FLAG_NO_DECODE"])
def test_i8_grouped_plan_follows_its_offsets(smb, cuda_device, mode):
    # One plan, captured once: every replay reads the offsets that are there then, the empty batch too.
    torch = _torch()
    n, k, groups, cap = 272, 208, 6, 900
    plan, _, offsets, a, sa, b, sb, d = _run_grouped(smb, torch, (150,) * groups, n, k, getattr(smb.capi, mode))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    plan.run(stream)
    plan.check(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.run(stream)
    for sizes in [(900, 0, 0, 0, 0, 0), (0, 0, 0, 0, 0, 0), (1, 2, 3, 4, 5, 6), (0, 300, 1, 299, 0, 17)]:
        ends = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        offsets.copy_(torch.tensor(ends))
        d.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        _check_grouped(torch, ends, n, k, a, sa, b, sb, d, False)
    plan.check(stream)


@pytest.mark.parametrize("flags_name", ["FLAG_NONE", "FLAG_WEIGHTS_STATIC"])
@pytest.mark.parametrize("shape", [(1, 4096, 4096), (16, 4096, 2048), (100, 1000, 1056), (129, 300, 520), (700, 600, 1000),
                                   (3, 130, 77), (64, 28672, 1024), (8, 28672, 1024), (5, 301, 8200), (7, 1000, 12296),
                                   (2, 20000, 12288), (8, 8, 8), (1, 2048, 136)])
def test_i8_plan_fed_with_bf16_activations(smb, cuda_device, shape, flags_name):
    torch = _torch()
    m, n, k = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = (torch.randn(m, k, generator=g, device="cuda") * 3).bfloat16()
    b, sb = _codes(torch, n, k, 7), _scales(torch, n, 8)
    d = torch.full((m, n), float("nan"), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    plan = smb.gemm.I8Plan.from_bf16_activations(x, b, sb, d, m, n, k, ldb=b.shape[1], flags=getattr(smb.capi, flags_name))
    for _ in range(3):
        plan.run()
    plan.check()
    codes = torch.zeros(m, k, device="cuda", dtype=torch.int8)
    scales = torch.zeros(m, device="cuda")
    smb.gemm.quantize_i8_bf16_device(x, codes, scales, m, k)
    _check(torch, d, _sums(torch, codes, b, k), scales, sb)
    # The rows are read by every run, not kept.
    x.mul_(0.5).add_(1.0)
    plan.run()
    plan.check()
    smb.gemm.quantize_i8_bf16_device(x, codes, scales, m, k)
    _check(torch, d, _sums(torch, codes, b, k), scales, sb)


@pytest.mark.parametrize("m", [1, 6, 8, 9])
def test_i8_gated_plan_fed_with_bf16_activations(smb, cuda_device, m):
    torch = _torch()
    n, k = 1552, 2048
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    x = torch.randn(m, k + 8, generator=g, device="cuda").bfloat16()
    if m > 2:
        x[1] = 0.0
    b = _codes(torch, n, k, 7)
    sb = torch.full((n,), 0.05 / 74, device="cuda")
    d = torch.full((m, n // 2), float("nan"), device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan.from_bf16_activations(x, b, sb, d, m, n, k, ldx=k + 8, ldb=b.shape[1],
                                                 flags=smb.capi.FLAG_EPILOGUE_SWIGLU | smb.capi.FLAG_WEIGHTS_STATIC)
    plan.run()
    plan.check()
    codes, scales = torch.zeros(m, k, device="cuda", dtype=torch.int8), torch.zeros(m, device="cuda")
    smb.gemm.quantize_i8_bf16_device(x, codes, scales, m, k, ld_src=k + 8)
    _check_gated(torch, d, _sums(torch, codes, b, k), scales, sb)


def test_i8_nan_token_in_the_fused_quantiser(smb, cuda_device):
    torch = _torch()
    m, n, k = 4, 300, 1024
    x = torch.randn(m, k, device="cuda").bfloat16()
    x[2, 1000] = float("inf")
    b, sb = _codes(torch, n, k, 1), _scales(torch, n, 2)
    d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan.from_bf16_activations(x, b, sb, d, m, n, k)
    assert "fused" in plan.describe()
    plan.run()
    plan.check()
    bad = torch.isnan(d.float())
    assert bool(bad[2].all()) and int(bad.sum()) == n


def test_i8_two_plans_on_two_streams(smb, cuda_device):
    torch = _torch()
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for i, (m, n, k) in enumerate([(24, 3000, 2048), (600, 900, 512)]):
        a, b = _codes(torch, m, k, 20 + i), _codes(torch, n, k, 30 + i)
        sa, sb = _scales(torch, m, 40 + i), _scales(torch, n, 50 + i)
        d = torch.full((m, n), float("nan"), device="cuda", dtype=torch.bfloat16)
        plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k)
        work.append((plan, a, sa, b, sb, d, k))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, w in zip(streams, work):
            w[0].run(s)
    for s, (plan, a, sa, b, sb, d, k) in zip(streams, work):
        plan.check(s)
        _check(torch, d, _sums(torch, a, b, k), sa, sb)


def test_i8_host_entry_points(smb, cuda_device):
    torch = _torch()
    rng = np.random.default_rng(5)
    m, n, k = 37, 53, 101
    x = rng.standard_normal((m, k)).astype(np.float32)
    w = rng.standard_normal((n, k)).astype(np.float32)
    a, sa = smb.gemm.quantize_i8_host(x)
    b, sb = smb.gemm.quantize_i8_host(w)
    d = torch.from_numpy(smb.gemm.dense_gemm_i8_host(a, sa, b, sb).view(np.int16)).view(torch.bfloat16)
    acc = torch.from_numpy(a).double() @ torch.from_numpy(b).double().t()
    _check(torch, d, acc, torch.from_numpy(sa), torch.from_numpy(sb))


@pytest.mark.parametrize("case", [(1, 1, 0), (5, 8, 0), (3, 1000, 0), (9, 1024, 8), (4, 1030, 0), (33, 4096, 0), (2, 8192, 16),
                                  (3, 8200, 0), (2, 20001, 0), (7, 777, 3)])
@pytest.mark.parametrize("bf16", [True, False])
def test_i8_quantizer_matches_host(smb, cuda_device, case, bf16):
    torch = _torch()
    rows, k, extra = case
    rng = np.random.default_rng(rows * k)
    x = rng.standard_normal((rows, k + extra)).astype(np.float32) * np.exp(rng.standard_normal((rows, 1))).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    if bf16:
        t = t.bfloat16()
    t[0, 0] = 0.0
    if rows > 2:
        t[1] = 0.0                       # zero row
        t[2] = t[2] * 1e-36              # far below the floor of amax
    if rows > 4:
        t[3, k // 2] = float("inf")
        t[4, k - 1] = float("nan")
    codes = torch.full((rows, k + extra), 99, device="cuda", dtype=torch.int8)
    scales = torch.full((rows,), 7.0, device="cuda")
    fn = smb.gemm.quantize_i8_bf16_device if bf16 else smb.gemm.quantize_i8_device
    fn(t, codes, scales, rows, k, ld_src=k + extra, ld_bytes=k + extra)
    torch.cuda.synchronize()
    want, want_scales = smb.gemm.quantize_i8_host(t.float().cpu().numpy()[:, :k])
    np.testing.assert_array_equal(codes[:, :k].cpu().numpy(), want)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    assert bool((codes[:, k:] == 99).all())


def test_i8_quantizer_takes_unaligned_rows(smb, cuda_device):
    torch = _torch()
    buf = torch.randn(2000, device="cuda").bfloat16()
    codes = torch.zeros(600, device="cuda", dtype=torch.int8)
    scales = torch.zeros(2, device="cuda")
    # Both rows start at odd elements of their buffers.
    smb.gemm.quantize_i8_bf16_device(buf.data_ptr() + 2, codes.data_ptr() + 1, scales, 2, 257, ld_src=901, ld_bytes=259)
    torch.cuda.synchronize()
    x = torch.stack([buf[1:258], buf[902:1159]]).float().cpu().numpy()
    want, want_scales = smb.gemm.quantize_i8_host(x)
    got = codes.cpu().numpy()
    np.testing.assert_array_equal(got[1:258], want[0])
    np.testing.assert_array_equal(got[260:517], want[1])
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    assert got[0] == 0 and not got[258:260].any() and not got[517:].any()


def test_i8_nan_row_stays_in_its_row(smb, cuda_device):
    torch = _torch()
    m, n, k = 40, 64, 128
    x = torch.randn(m, k, device="cuda").bfloat16()
    x[7, 3] = float("nan")
    b, sb = _codes(torch, n, k, 1), _scales(torch, n, 2)
    d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan.from_bf16_activations(x, b, sb, d, m, n, k)
    plan.run()
    plan.check()
    bad = torch.isnan(d.float())
    assert bool(bad[7].all()) and int(bad.sum()) == n


def test_i8_wait_probe_reports_and_recovers(smb, cuda_device):
    torch = _torch()
    m, n, k = 64, 128, 128
    a, b = _codes(torch, m, k, 1), _codes(torch, n, k, 2)
    sa, sb = _scales(torch, m, 3), _scales(torch, n, 4)
    d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    plan = smb.gemm.I8Plan(a, sa, b, sb, d, m, n, k)
    plan.wait_probe(100_000)
    with pytest.raises(smb.SmbError) as e:
        plan.check()
    assert e.value.code == smb.capi.SMB_ERR_DEVICE and "bounded-wait probe" in str(e.value)
    plan.run()
    plan.check()
    _check(torch, d, _sums(torch, a, b, k), sa, sb)


@pytest.mark.parametrize("seed", [1, 2])
def test_i8_random_shapes_all_schedules_agree(smb, cuda_device, seed):
    torch = _torch()
    rng = np.random.default_rng(seed)
    c = smb.capi
    for _ in range(6):
        m, n, k = int(rng.integers(1, 200)), int(rng.integers(1, 1500)), int(rng.integers(1, 3000))
        outs = []
        for flags in [0, c.FLAG_NO_DECODE, c.FLAG_NO_DECODE | c.FLAG_TILE_N_128, c.FLAG_NO_DECODE | c.FLAG_TILE_N_512,
                      c.FLAG_FORCE_PLAIN_STORE, c.FLAG_WEIGHTS_STATIC, c.FLAG_DECODE_SINGLE]:
            a, sa, b, sb, d = _run(smb, torch, m, n, k, flags=flags, seed=seed)
            outs.append(d)
        _check(torch, outs[0], _sums(torch, a, b, k), sa, sb)
        for d in outs[1:]:
            assert torch.equal(d.view(torch.int16), outs[0].view(torch.int16)), (m, n, k)


@pytest.mark.parametrize("case", [(5, 33), (7, 511), (3, 1023), (700, 1025), (2, 8190), (900, 2046), (9, 16500), (601, 8195), (4100, 66), (5000, 1022)])
@pytest.mark.parametrize("bf16", [True, False])
def test_i8_quantizer_rows_without_vectors(smb, cuda_device, case, bf16):
    torch = _torch()
    rows, k = case
    g = torch.Generator(device="cuda")
    g.manual_seed(k)
    x = torch.randn(rows, k, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    x = x.bfloat16() if bf16 else x
    x[1, k - 1] = float("inf")
    codes = torch.full((rows, k + 3), 55, device="cuda", dtype=torch.int8)
    scales = torch.empty(rows, device="cuda")
    call = smb.gemm.quantize_i8_bf16_device if bf16 else smb.gemm.quantize_i8_device
    call(x, codes, scales, rows, k, ld_bytes=k + 3)
    torch.cuda.synchronize()
    want_c, want_s = smb.gemm.quantize_i8_host(x.float().cpu().numpy())
    np.testing.assert_array_equal(codes[:, :k].cpu().numpy(), want_c)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    assert bool((codes[:, k:] == 55).all())
