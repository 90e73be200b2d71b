"""int8 product, routing and row sorting without a GPU: host quantiser, descriptor bits, refusals."""
import ctypes as C

import numpy as np
import pytest


def test_host_quantizer_matches_numpy(smb):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((60, 333)) * np.exp(rng.standard_normal((60, 1)))).astype(np.float32)
    x[0] = 0.0
    x[1] = np.float32(1e-38)                  # below the floor of amax: codes 0
    x[2, :5] = [127, -127, 0.5, 1.5, 2.5]     # ties go to the even code
    x[2, 5:] = 0
    x[3, 7] = np.inf
    x[4, 8] = -np.nan
    x[5] *= np.float32(1e30)
    codes, scales = smb.gemm.quantize_i8_host(x)
    amax = np.maximum(np.abs(x).max(1), np.float32(2.0 ** -100)).astype(np.float32)
    bad = ~np.isfinite(x).all(1)
    with np.errstate(all="ignore"):
        want = np.rint(x * (np.float32(127) / amax)[:, None])
    want[bad] = 0
    np.testing.assert_array_equal(codes, want.astype(np.int8))
    np.testing.assert_array_equal(scales[~bad], (amax / np.float32(127))[~bad])
    assert np.isnan(scales[bad]).all()
    np.testing.assert_array_equal(codes[2, :5], [127, -127, 0, 2, 2])
    ok = ~bad
    # Half a code, and the rounding of x * inv at the top of the range (127 steps of 2^-24).
    err = np.abs(codes[ok].astype(np.float64) * scales[ok, None].astype(np.float64) - x[ok])
    assert (err <= scales[ok, None].astype(np.float64) * (0.5 + 3 * 127 * 2.0 ** -24)).all()


def test_max_rows(smb):
    f = smb.moe.max_rows
    assert f(16, 8, 256) == 128 and f(0, 8, 4, 256) == 0
    assert f(1, 1, 8, 256) == 256 and f(3, 2, 4, 256) == 4 * 256
    assert f(100, 2, 4, 128) == (200 + 4 * 127) // 128 * 128
    rng = np.random.default_rng(0)
    for _ in range(200):
        t, k, g, a = int(rng.integers(1, 60)), int(rng.integers(1, 9)), int(rng.integers(1, 20)), int(rng.choice([1, 4, 128, 256]))
        counts = rng.multinomial(t * k, rng.dirichlet(np.full(g, 0.3)))
        assert sum(-(-c // a) * a for c in counts) <= f(t, k, g, a)


P = C.c_void_p(0x10000)        # stands for a device address; nothing here gets as far as using it
ODD = C.c_void_p(0x10001)


def _refused(smb, rc, text, code=None):
    assert rc in ((code,) if code is not None else (smb.capi.SMB_ERR_INVALID, smb.capi.SMB_ERR_UNSUPPORTED)), rc
    assert text in smb.capi.last_error(), smb.capi.last_error()


@pytest.mark.parametrize("change,text", [
    (dict(a=None), "null operand"), (dict(sa=None), "null operand"), (dict(b=None), "null operand"),
    (dict(sb=None), "null operand"), (dict(d=None), "null operand"), (dict(M=0), "positive"), (dict(N=-1), "positive"),
    (dict(K=0), "positive"), (dict(K=131072, lda=131072, ldb=131072), "int32"), (dict(lda=120), "lda"), (dict(lda=136), "lda"),
    (dict(ldb=127), "ldb"), (dict(ldd=255), "ldd"), (dict(d=ODD), "2-byte"), (dict(sa=C.c_void_p(0x10002)), "4-byte"),
    (dict(sb=C.c_void_p(0x10002)), "4-byte"), (dict(flags=256), "no int8 form"), (dict(flags=32), "no int8 form"),
    (dict(flags=8192, N=255), "even N"),
])
def test_i8_plan_refusals(smb, change, text):
    args = dict(a=P, sa=P, b=P, sb=P, d=P, M=64, N=256, K=128, lda=128, ldb=128, ldd=256, flags=0)
    args.update(change)
    h = C.c_void_p()
    rc = smb.capi.lib().smb_i8_plan_create(C.byref(h), *args.values())
    _refused(smb, rc, text)
    assert not h.value


@pytest.mark.parametrize("change,text", [
    (dict(off=None), "null offsets"), (dict(off=C.c_void_p(0x10002)), "4-byte"), (dict(groups=0), "groups"),
    (dict(groups=513), "groups"), (dict(rows=0), "positive"), (dict(rows=(8 << 20) + 1), "max_rows"),
    (dict(groups=512, N=1 << 23, ldd=1 << 23), "too large"),
])
def test_i8_grouped_plan_refusals(smb, change, text):
    args = dict(a=P, sa=P, b=P, sb=P, d=P, rows=64, N=256, K=128, lda=128, ldb=128, ldd=256, groups=4, off=P, flags=0)
    args.update(change)
    if args["ldd"] < args["N"]:
        args["ldd"] = args["N"]
    h = C.c_void_p()
    rc = smb.capi.lib().smb_i8_grouped_plan_create(C.byref(h), *args.values())
    _refused(smb, rc, text)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null activations"), (dict(ldx=100), "pitch"), (dict(x=ODD), "2-byte"), (dict(K=131072, ldb=131072), "int32"),
])
def test_i8_activation_plan_refusals(smb, change, text):
    args = dict(x=P, ldx=131072, b=P, sb=P, d=P, M=64, N=256, K=128, ldb=128, ldd=256, flags=0)
    args.update(change)
    h = C.c_void_p()
    rc = smb.capi.lib().smb_i8_plan_create_bf16_activations(C.byref(h), *args.values())
    _refused(smb, rc, text)


def test_i8_null_handles_and_host_refusals(smb):
    lib = smb.capi.lib()
    inv = smb.capi.SMB_ERR_INVALID
    assert lib.smb_i8_plan_run(None, None) == inv and lib.smb_i8_plan_check(None, None) == inv
    assert lib.smb_i8_plan_tune(None, 0, 0) == inv and lib.smb_i8_plan_destroy(None) == 0
    assert lib.smb_i8_plan_create(None, P, P, P, P, P, 1, 1, 16, 16, 16, 8, 0) == inv
    assert lib.smb_dense_gemm_i8_host(None, P, P, P, P, 1, 1, 1) == inv
    with pytest.raises(ValueError):
        smb.gemm.dense_gemm_i8_host(np.zeros((2, 3), np.int8), np.zeros(2, np.float32), np.zeros((2, 4), np.int8),
                                    np.zeros(2, np.float32))
    x = np.zeros((2, 8), np.float32)
    c, s = np.zeros((2, 8), np.int8), np.zeros(2, np.float32)
    q = lib.smb_quantize_i8_host
    assert q(None, 8, c.ctypes.data, 8, s.ctypes.data, 2, 8) == inv
    assert q(x.ctypes.data, 7, c.ctypes.data, 8, s.ctypes.data, 2, 8) == inv
    assert q(x.ctypes.data, 8, c.ctypes.data, 7, s.ctypes.data, 2, 8) == inv
    assert q(x.ctypes.data, 8, c.ctypes.data, 8, s.ctypes.data, 2, 0) == inv
    assert q(x.ctypes.data, 8, c.ctypes.data, 8, s.ctypes.data, 0, 8) == 0
    assert lib.smb_quantize_i8_bf16_device(ODD, 8, P, 8, P, 2, 8, None) == inv


@pytest.mark.parametrize("change,text", [
    (dict(logits=None), "null logits"), (dict(dtype=2), "dtype"), (dict(logits=C.c_void_p(0x10002)), "aligned"),
    (dict(tokens=-1), "negative"), (dict(experts=513), "experts"), (dict(experts=0), "experts"), (dict(top_k=0), "top_k"),
    (dict(top_k=33), "top_k"), (dict(experts=4, n_groups=1, top_groups=1, top_k=5), "top_k"), (dict(ld=63), "pitch"),
    (dict(n_groups=3), "groups"), (dict(n_groups=64), "groups"), (dict(n_groups=0), "groups"), (dict(top_groups=0), "top_groups"),
    (dict(top_groups=9), "top_groups"), (dict(top_groups=1, top_k=9), "open groups"), (dict(flags=8), "flags"),
    (dict(ids=None), "null output"), (dict(weights=None), "null output"), (dict(ids=ODD), "4-byte"),
    (dict(weights=C.c_void_p(0x10002)), "4-byte"), (dict(bias=C.c_void_p(0x10002)), "4-byte"),
])
def test_route_refusals(smb, change, text):
    args = dict(logits=P, dtype=0, ld=64, bias=None, tokens=8, experts=64, top_k=4, n_groups=8, top_groups=4, flags=0, scale=1.0,
                ids=P, weights=P, stream=None)
    args.update(change)
    _refused(smb, smb.capi.lib().smb_moe_route_device(*args.values()), text)


def test_empty_calls_are_valid(smb):
    lib = smb.capi.lib()
    assert lib.smb_moe_route_device(P, 0, 64, None, 0, 64, 4, 1, 1, 0, 1.0, P, P, None) == 0
    assert lib.smb_moe_route_backward_device(P, 0, 64, P, P, 0, 64, 4, 0, 1.0, P, 64, None) == 0
    assert lib.smb_moe_gather_bf16_device(P, 8, P, 0, 1, 8, 4, P, 8, None) == 0
    assert lib.smb_moe_gather_i8_device(P, 8, P, 0, 1, 8, 4, P, 8, P, None) == 0
    assert lib.smb_moe_combine_device(P, 8, P, P, 0, 1, 8, 4, P, 8, None) == 0
    # The address of an empty tensor is null.
    assert lib.smb_moe_route_device(None, 0, 64, None, 0, 64, 4, 1, 1, 0, 1.0, None, None, None) == 0
    assert lib.smb_moe_gather_bf16_device(None, 8, None, 0, 1, 8, 0, None, 8, None) == 0
    assert lib.smb_quantize_i8_bf16_device(None, 8, None, 8, None, 0, 8, None) == 0
    assert lib.smb_moe_combine_backward_device(P, 8, P, 8, P, P, 0, 1, 8, 4, P, 8, P, None) == 0


@pytest.mark.parametrize("change,text", [
    (dict(ids=None), "null"), (dict(offsets=None), "null"), (dict(row_of_slot=None), "null"), (dict(slot_of_row=None), "null"),
    (dict(ids=C.c_void_p(0x10002)), "4-byte"), (dict(groups=0), "groups"), (dict(groups=1025), "groups"), (dict(tokens=-1), "extents"),
    (dict(top_k=0), "extents"), (dict(top_k=33), "extents"), (dict(align=0), "alignment"), (dict(max_rows=63), "room"),
    (dict(align=256, max_rows=1023), "room"), (dict(tiles=P), "256"), (dict(tokens=1 << 29, max_rows=1 << 31), "slots"),
])
def test_dispatch_refusals(smb, change, text):
    args = dict(ids=P, tokens=16, top_k=4, groups=4, align=1, max_rows=64, offsets=P, row_of_slot=P, slot_of_row=P, tiles=None,
                stream=None)
    args.update(change)
    _refused(smb, smb.capi.lib().smb_moe_dispatch_device(*args.values()), text)


def test_row_copy_refusals(smb):
    lib = smb.capi.lib()
    base = dict(x=P, ld_x=64, row=P, tokens=4, top_k=2, width=64, max_rows=8, out=P, ld_out=64, stream=None)
    for change, text in [(dict(x=None), "null"), (dict(out=None), "null"), (dict(row=None), "null"), (dict(ld_x=63), "pitch"),
                         (dict(ld_out=63), "pitch"), (dict(width=0), "width"), (dict(top_k=33), "top_k"), (dict(max_rows=0), "capacity"),
                         (dict(x=ODD), "2-byte"), (dict(tokens=-1), "token count"), (dict(row=ODD), "4-byte")]:
        args = dict(base, **change)
        _refused(smb, lib.smb_moe_gather_bf16_device(*args.values()), text)
        _refused(smb, lib.smb_moe_combine_device(args["x"], args["ld_x"], args["row"], P, args["tokens"], args["top_k"],
                                                 args["width"], args["max_rows"], args["out"], args["ld_out"], None), text)
    _refused(smb, lib.smb_moe_gather_i8_device(P, 64, P, 4, 2, 64, 8, P, 63, P, None), "pitch")
    _refused(smb, lib.smb_moe_gather_i8_device(P, 64, P, 4, 2, 64, 8, P, 64, None, None), "null")
    _refused(smb, lib.smb_moe_combine_backward_device(P, 64, None, 64, P, P, 4, 2, 64, 8, P, 64, P, None), "needs the rows")
    _refused(smb, lib.smb_moe_combine_backward_device(P, 64, P, 64, P, P, 4, 2, 64, 8, None, 64, P, None), "null")
    _refused(smb, lib.smb_moe_combine_backward_device(P, 64, P, 64, P, P, 4, 2, 64, 8, P, 60, P, None), "pitch")
    _refused(smb, lib.smb_moe_route_backward_device(P, 0, 64, None, P, 4, 64, 2, 0, 1.0, P, 64, None), "null")
    _refused(smb, lib.smb_moe_route_backward_device(P, 0, 64, P, P, 4, 64, 2, 0, 1.0, P, 63, None), "pitch")


def test_extents_that_leave_31_bits_are_refused(smb):
    lib = smb.capi.lib()
    inv, uns = smb.capi.SMB_ERR_INVALID, smb.capi.SMB_ERR_UNSUPPORTED
    big = (1 << 30) + 1
    h = C.c_void_p()
    assert lib.smb_i8_plan_create(C.byref(h), P, P, P, P, P, big, 8, 16, 16, 16, 8, 0) == uns
    assert lib.smb_i8_plan_create(C.byref(h), P, P, P, P, P, 8, big, 16, 16, 16, big + 7, 0) == uns
    assert lib.smb_quantize_i8_device(P, big, P, big, P, 1, big, None) == inv
    assert lib.smb_quantize_i8_bf16_device(P, big, P, big, P, 1, big, None) == inv


def test_calls_by_words_take_the_same_arguments(smb):
    """Every argument lands in its own parameter: one bad value at a time comes back as that refusal."""
    moe, gemm, err = smb.moe, smb.gemm, smb.SmbError
    p, odd = P.value, ODD.value
    route = dict(logits=p, ids=p, weights=p, tokens=8, experts=64, top_k=4, n_groups=8, top_groups=4)
    moe.route_device(**dict(route, tokens=0))
    for change, text in [(dict(logits=odd), "logits are not aligned"), (dict(dtype=2), "dtype 2"), (dict(ld=63), "pitch"),
                         (dict(bias=odd), "4-byte"), (dict(tokens=-1), "negative"), (dict(tokens=1 << 40), "does not fit"),
                         (dict(experts=513), "513 experts"), (dict(top_k=33), "top_k=33"), (dict(n_groups=7), "7 groups"),
                         (dict(top_groups=9), "top_groups=9"), (dict(flags=64), "0x40"), (dict(flags=-1), "does not fit"),
                         (dict(ids=None), "null output"), (dict(weights=odd), "4-byte")]:
        with pytest.raises(err, match=text):
            moe.route_device(**dict(route, **change))
    grad = dict(logits=p, ids=p, grad_weights=p, grad_logits=p, tokens=8, experts=64, top_k=4)
    moe.route_backward_device(**dict(grad, tokens=0))
    for change, text in [(dict(ids=odd), "ids and gradients"), (dict(grad_weights=None), "null"), (dict(grad_logits=odd), "gradient is not"),
                         (dict(ld_grad=63), "gradient pitch"), (dict(ld=63), "pitch"), (dict(top_k=0), "top_k=0"), (dict(flags=8), "0x8")]:
        with pytest.raises(err, match=text):
            moe.route_backward_device(**dict(grad, **change))
    sort = dict(ids=p, offsets=p, row_of_slot=p, slot_of_row=p, tokens=8, top_k=2, groups=4, max_rows=16)
    for change, text in [(dict(offsets=None), "null"), (dict(slot_of_row=odd), "4-byte"), (dict(tokens=-1), "tokens=-1"),
                         (dict(top_k=33), "top_k=33"), (dict(groups=1025), "1025 groups"), (dict(max_rows=15), "room for 15 rows"),
                         (dict(align=0), "alignment 0"), (dict(mtile_group=p), "tile map")]:
        with pytest.raises(err, match=text):
            moe.dispatch_device(**dict(sort, **change))
    for call, args in [(moe.gather_bf16_device, dict(x=p, row_of_slot=p, out=p)),
                       (moe.gather_i8_device, dict(x=p, row_of_slot=p, codes=p, scales=p)),
                       (moe.combine_device, dict(rows=p, row_of_slot=p, weights=p, y=p)),
                       (moe.combine_backward_device, dict(grad_y=p, rows=p, row_of_slot=p, weights=p, grad_rows=p, grad_weights=p))]:
        dims = dict(tokens=4, top_k=2, width=64, max_rows=8)
        call(**args, **dict(dims, tokens=0))
        pitches = [n for n in call.__code__.co_varnames if n.startswith("ld_")]
        assert pitches
        for change, text in [(dict(tokens=-1), "token count"), (dict(top_k=33), "top_k=33"), (dict(width=0), "width 0"),
                             (dict(max_rows=0), "capacity")] + [({n: 63}, "pitch") for n in pitches]:
            with pytest.raises(err, match=text):
                call(**args, **dict(dims, **change))
        for n in args:
            if args[n] == p and n not in ("codes",):
                with pytest.raises(err, match="aligned"):
                    call(**dict(args, **{n: odd}), **dims)
    for call in (gemm.quantize_i8_device, gemm.quantize_i8_bf16_device):
        call(p, p, p, 0, 64)
        for args, kw, text in [((None, p, p, 2, 64), {}, "null"), ((p, p, p, -1, 64), {}, "rows=-1"), ((p, p, p, 2, 0), {}, "K=0"),
                               ((p, p, p, 2, 64), dict(ld_src=63), "pitch"), ((p, p, p, 2, 64), dict(ld_bytes=63), "pitch"),
                               ((odd, p, p, 2, 64), {}, "aligned"), ((p, p, odd, 2, 64), {}, "aligned")]:
            with pytest.raises(err, match=text):
                call(*args, **kw)


def test_calls_by_words_refusals(smb):
    words = smb.capi.lib().smb_call_words
    _refused(smb, words(99, b"\0" * 64, 8), "unknown call 99")
    _refused(smb, words(smb.capi.CALL_QUANTIZE_I8, b"\0" * 56, 7), "7 words for 8 arguments")
    _refused(smb, words(smb.capi.CALL_QUANTIZE_I8, None, 8), "no words")
    _refused(smb, words(smb.capi.CALL_QUANTIZE_I8, b"\0" * 120, 15), "no words")
    _refused(smb, words(smb.capi.CALL_QUANTIZE_I8, b"\0" * 8, -1), "no words")


def _words_of(smb, monkeypatch, fn, *args, **kw):
    """The argument words that a wrapper would hand to the library."""
    seen = []
    monkeypatch.setattr(smb.capi, "call_words", lambda call, words, count: seen.append(np.frombuffer(words, np.int64)))
    fn(*args, **kw)
    return seen[-1]


def test_route_takes_the_type_of_its_buffers(smb, monkeypatch):
    """Without a word about the type a bf16 buffer is read as one, not four bytes an element to past its end."""
    torch = pytest.importorskip("torch")
    f32, bf16 = torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.bfloat16)
    ids, w = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    m, c = smb.moe, smb.capi
    for x, kind in ((f32, c.DTYPE_F32), (bf16, c.DTYPE_BF16), (bf16.view(torch.int16), c.DTYPE_BF16), (f32.numpy(), c.DTYPE_F32),
                    (np.zeros((2, 8), np.uint16), c.DTYPE_BF16), (0x10000, c.DTYPE_F32)):
        assert _words_of(smb, monkeypatch, m.route_device, x, ids, w, 2, 8, 2)[1] == kind
        assert _words_of(smb, monkeypatch, m.route_device, x, ids, w, 2, 8, 2, dtype=kind)[1] == kind
        assert _words_of(smb, monkeypatch, m.route_backward_device, x, ids, w, x, 2, 8, 2)[1] == kind
    # Integers hold the bits of whatever the caller says, as raw addresses do.
    for x in (0x10000, torch.zeros(64, dtype=torch.uint8), f32.view(torch.int32), bf16.view(torch.int16)):
        for kind in (c.DTYPE_F32, c.DTYPE_BF16):
            assert _words_of(smb, monkeypatch, m.route_device, x, ids, w, 2, 8, 2, dtype=kind)[1] == kind
            assert _words_of(smb, monkeypatch, m.route_backward_device, x, ids, w, x, 2, 8, 2, dtype=kind)[1] == kind
    assert _words_of(smb, monkeypatch, m.route_device, f32.view(torch.int32), ids, w, 2, 8, 2)[1] == c.DTYPE_F32
    for x, kind in ((f32, c.DTYPE_BF16), (bf16, c.DTYPE_F32), (f32, 7)):
        with pytest.raises(ValueError, match="agree"):
            m.route_device(x, ids, w, 2, 8, 2, dtype=kind)
        with pytest.raises(ValueError, match="agree"):
            m.route_backward_device(x, ids, w, x, 2, 8, 2, dtype=kind)
    with pytest.raises(ValueError, match="agree"):
        m.route_backward_device(bf16, ids, w, f32, 2, 8, 2)
    for t in (torch.float16, torch.float64, torch.complex64):
        with pytest.raises(ValueError, match="fp32 or bf16"):
            m.route_device(torch.zeros(2, 8, dtype=t), ids, w, 2, 8, 2)
        with pytest.raises(ValueError, match="fp32 or bf16"):
            m.route_backward_device(f32, ids, w, torch.zeros(2, 8, dtype=t), 2, 8, 2)


def test_calls_by_words_refuse_a_scale_beyond_fp32(smb):
    def route(scale):     # no tokens: valid and without effect
        smb.moe.route_device(0x10000, 0x10000, 0x10000, 0, 8, 2, scale=scale)
    for scale in (1.0, 0.1, 3.4e38, -3.4e38, 1e-60, float("inf"), float("nan")):
        route(scale)
    for scale in (1e39, -1e300):
        with pytest.raises(smb.SmbError, match="does not fit"):
            route(scale)
