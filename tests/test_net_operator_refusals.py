"""Arguments that gated layers, log probabilities and 4-bit products refuse, before any launch (CPU only)."""
import ctypes

import pytest

from test_operator_refusals import BAD, LARGE, MISALIGNED, UNSUPPORTED, Fake, refused


def test_log_probs(sb):
    def go(logits=0x1000, ld=8, dt=0, rows=4, cols=8, mask=None, prefix=-1, scale=1.0, tokens=0x2000, it=4, out=0x3000, h=None, stats=None, top=0,
           tv=None, tt=None):
        return ("sb_log_probs", logits, ld, dt, rows, cols, mask, prefix, scale, tokens, it, out, h, stats, top, tv, tt, None)
    refused(sb, BAD, *go(logits=None))
    refused(sb, BAD, *go(rows=-1))
    refused(sb, BAD, *go(cols=-1))
    refused(sb, BAD, *go(ld=7))
    refused(sb, BAD, *go(prefix=9))
    refused(sb, BAD, *go(tokens=None))
    refused(sb, BAD, *go(top=-1))
    refused(sb, BAD, *go(top=2))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(sb, BAD, *go(scale=scale))
    refused(sb, LARGE, *go(top=65, tv=0x4000))
    refused(sb, UNSUPPORTED, *go(dt=1))
    refused(sb, UNSUPPORTED, *go(it=0))
    refused(sb, MISALIGNED, *go(logits=0x1002))
    refused(sb, MISALIGNED, *go(tokens=0x2004, it=6))
    refused(sb, MISALIGNED, *go(out=0x3002))
    refused(sb, MISALIGNED, *go(stats=0x3002))
    refused(sb, MISALIGNED, *go(top=1, tt=0x3002))


def test_log_probs_grad(sb):
    def go(logits=0x1000, ld=8, dt=2, rows=4, cols=8, prefix=-1, scale=1.0, tokens=0x2000, it=4, stats=0x3000, dout=0x4000, h=0x5000, dh=0x6000,
           d=0x7000, ldd=8):
        return ("sb_log_probs_grad", logits, ld, dt, rows, cols, None, prefix, scale, tokens, it, stats, dout, h, dh, d, ldd, None)
    refused(sb, BAD, *go(d=None))
    refused(sb, BAD, *go(stats=None))
    refused(sb, BAD, *go(tokens=None))
    refused(sb, BAD, *go(h=None))
    refused(sb, BAD, *go(ldd=7))
    refused(sb, BAD, *go(prefix=9))
    refused(sb, BAD, *go(scale=-2.0))
    refused(sb, UNSUPPORTED, *go(dt=7))
    refused(sb, MISALIGNED, *go(d=0x7001))
    refused(sb, MISALIGNED, *go(dh=0x6002))


def test_log_probs_arrays(sb):
    p = sb.primitives
    x, t, v = Fake((4, 8)), Fake((4,), "int32"), Fake((4,))
    with pytest.raises(ValueError):
        p.log_probs(x, Fake((5,), "int32"), v)
    with pytest.raises(TypeError):
        p.log_probs(x, Fake((4,), "float32"), v)
    with pytest.raises(TypeError):
        p.log_probs(Fake((4, 8), "int32"), t, v)
    with pytest.raises(ValueError):
        p.log_probs(x, t, Fake((3,)))
    with pytest.raises(ValueError):
        p.log_probs(x, t, v, mask=Fake((4, 7), "uint8"))
    with pytest.raises(ValueError):
        p.log_probs(x, t, v, mask=Fake((4, 8), "float32"))
    with pytest.raises(ValueError):
        p.log_probs(x, t, v, top=Fake((4, 2)), top_tokens=Fake((4, 3), "int32"))
    with pytest.raises(ValueError):
        p.log_probs(x, t, v, top_tokens=Fake((4, 2), "int64"))
    with pytest.raises(ValueError):
        p.log_probs(x, t, v, stats=Fake((4,)))
    with pytest.raises(ValueError):
        p.log_probs_grad(x, t, Fake((4, 2)), Fake((4, 7)), dout=v)
    with pytest.raises(ValueError):
        p.log_probs_grad(x, t, Fake((4, 2)), Fake((4, 8), "bfloat16"), dout=v)


def test_gated(sb):
    def go(x=0x1000, ldx=16, w=0x2000, ldw=16, h=0x3000, ldh=8, saved=None, lds=16, m=4, f=8, k=16, dt=2, act=0):
        return ("sb_gated", x, ldx, w, ldw, h, ldh, saved, lds, m, f, k, dt, act, None)
    for null in ("x", "w", "h"):
        refused(sb, BAD, *go(**{null: None}))
    for size in ("m", "f", "k"):
        refused(sb, BAD, *go(**{size: -1}))
    for pitch in ("ldx", "ldw", "ldh"):
        refused(sb, BAD, *go(**{pitch: 7}))
    refused(sb, BAD, *go(saved=0x4000, lds=15))
    for place in ("x", "w"):
        refused(sb, BAD, *go(**{place: 0x3000, "h": 0x3000}))
    refused(sb, UNSUPPORTED, *go(dt=0))
    refused(sb, UNSUPPORTED, *go(act=3))
    refused(sb, LARGE, *go(f=1 << 22, ldh=1 << 22))
    for p in ("x", "w", "h", "saved"):
        refused(sb, MISALIGNED, *go(**{p: 0x1001}))


def test_gated_grad(sb):
    def go(dh=0x1000, lddh=8, x=0x2000, ldx=16, w=0x3000, ldw=16, saved=0x4000, lds=16, dx=0x5000, lddx=16, dw=0x6000, lddw=16, dwt=2, m=4, f=8, k=16,
           dt=2, act=0, ws=0x10000, nws=1 << 20):
        return ("sb_gated_grad", dh, lddh, x, ldx, w, ldw, saved, lds, dx, lddx, dw, lddw, dwt, 0, m, f, k, dt, act, ws, nws, None)
    for null in ("dh", "x", "w", "saved", "ws"):
        refused(sb, BAD, *go(**{null: None}))
    for pitch in ("lddh", "ldx", "ldw", "lds", "lddx", "lddw"):
        refused(sb, BAD, *go(**{pitch: 7}))
    refused(sb, BAD, *go(nws=100))
    refused(sb, BAD, *go(dx=0x2000))
    refused(sb, BAD, *go(dw=0x3000))
    refused(sb, BAD, *go(m=-1))
    refused(sb, UNSUPPORTED, *go(dwt=3))
    refused(sb, UNSUPPORTED, *go(dt=1))
    refused(sb, MISALIGNED, *go(ws=0x10010))
    refused(sb, MISALIGNED, *go(dw=0x6002, dwt=0))
    need = ctypes.c_size_t(0)
    from spiral_b200 import _lib
    refused(sb, BAD, "sb_gated_grad_workspace_bytes", 1, -1, 1, ctypes.byref(need))
    refused(sb, BAD, "sb_gated_grad_workspace_bytes", 1, 1, 1, None)
    _lib.call("sb_gated_grad_workspace_bytes", 100, 64, 32, ctypes.byref(need))
    assert need.value >= 100 * 128 * 2


def test_gated_arrays(sb):
    b = "bfloat16"
    x, w, h = Fake((4, 16), b), Fake((16, 16), b), Fake((4, 8), b)
    with pytest.raises(TypeError):
        sb.gated(Fake((4, 16)), w, h)
    with pytest.raises(ValueError):
        sb.gated(x, Fake((15, 16), b), h)
    with pytest.raises(ValueError):
        sb.gated(x, Fake((16, 8), b), h)
    with pytest.raises(ValueError):
        sb.gated(x, Fake((16, 16), "float16"), h)
    with pytest.raises(ValueError):
        sb.gated(x, w, Fake((4, 16), b))
    with pytest.raises(ValueError):
        sb.gated(x, w, h, saved=Fake((4, 8), b))
    with pytest.raises(ValueError):
        sb.gated(x, w, h, activation="tanh")
    with pytest.raises(ValueError):
        sb.gated_grad(h, x, w, Fake((4, 16), b), dx=Fake((4, 8), b))
    with pytest.raises(TypeError):
        sb.gated_grad(h, x, w, Fake((4, 16), b), dw=Fake((16, 16), "float16"))


def test_int4(sb):
    def quantize(x=0x1000, ldx=64, dt=0, n=4, k=64, group=32, codes=0x2000, ldc=32, scales=0x3000, st=2):
        return ("sb_quantize_int4", x, ldx, dt, n, k, group, codes, ldc, scales, st, None)
    refused(sb, BAD, *quantize(x=None))
    refused(sb, BAD, *quantize(n=-1))
    refused(sb, BAD, *quantize(ldc=31))
    refused(sb, BAD, *quantize(ldx=63))
    refused(sb, UNSUPPORTED, *quantize(group=16))
    refused(sb, UNSUPPORTED, *quantize(dt=7))
    refused(sb, UNSUPPORTED, *quantize(st=0))
    refused(sb, MISALIGNED, *quantize(scales=0x3001))
    refused(sb, LARGE, *quantize(n=1 << 31))

    def dequantize(codes=0x1000, ldw=32, scales=0x2000, st=2, out=0x3000, ldo=64, ot=2, n=4, k=64, group=64):
        return ("sb_dequantize_int4", codes, ldw, scales, st, out, ldo, ot, n, k, group, None)
    refused(sb, BAD, *dequantize(out=None))
    refused(sb, BAD, *dequantize(ldo=63))
    refused(sb, BAD, *dequantize(ldw=31))
    refused(sb, UNSUPPORTED, *dequantize(ot=5))
    refused(sb, UNSUPPORTED, *dequantize(group=48))
    refused(sb, MISALIGNED, *dequantize(out=0x3001))

    def product(a=0x1000, lda=64, dt=2, codes=0x2000, ldw=32, scales=0x3000, st=2, c=0x4000, ldc=8, m=2, n=8, k=64, group=64, ot=0, epi=0, bias=None):
        return ("sb_matmul_int4", a, lda, dt, codes, ldw, scales, st, c, ldc, m, n, k, group, ot, epi, bias, None)
    for null in ("a", "codes", "scales", "c"):
        refused(sb, BAD, *product(**{null: None}))
    for pitch in ("lda", "ldw", "ldc"):
        refused(sb, BAD, *product(**{pitch: 7}))
    refused(sb, BAD, *product(epi=1))
    refused(sb, BAD, *product(m=-1))
    refused(sb, UNSUPPORTED, *product(epi=8))
    refused(sb, UNSUPPORTED, *product(dt=0))
    refused(sb, UNSUPPORTED, *product(ot=7))
    refused(sb, MISALIGNED, *product(c=0x4002))
    refused(sb, MISALIGNED, *product(a=0x1001))


def test_int4_arrays(sb):
    codes, scales = Fake((8, 32), "uint8"), Fake((1, 8), "bfloat16")
    a, c = Fake((2, 64), "bfloat16"), Fake((2, 8))
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, c, group=48)
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, c, group=32)
    with pytest.raises(ValueError):
        sb.matmul_int4(a, Fake((8, 31), "uint8"), scales, c, group=64)
    with pytest.raises(TypeError):
        sb.matmul_int4(a, Fake((8, 32), "int32"), scales, c, group=64)
    with pytest.raises(TypeError):
        sb.matmul_int4(Fake((2, 64)), codes, scales, c, group=64)
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, Fake((2, 7)), group=64)
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, c, group=64, epilogue=("bias",))
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, c, group=64, epilogue=("tanh",))
    with pytest.raises(ValueError):
        sb.quantize_int4(Fake((7, 64)), codes, scales, group=64)
    with pytest.raises(ValueError):
        sb.dequantize_int4(codes, scales, Fake((7, 64)), group=64)


@pytest.mark.parametrize("places", [{"dx": 0x3000}, {"dx": 0x3000, "dw": None}, {"dw": 0x2000}, {"dw": 0x2000, "dx": None}, {"dx": 0x2000}, {"dw": 0x3000},
                                    {"dx": 0x6000}, {"ws": 0x1000}, {"ws": 0x2000}, {"ws": 0x3000}, {"ws": 0x4000}, {"ws": 0x5000}, {"ws": 0x6000}])
def test_gradients_of_gated_layers_in_the_place_of_what_they_are_made_from(sb, places):
    """m = 2 f: dx is as large as w, and dw as x."""
    a = dict(dh=0x1000, x=0x2000, w=0x3000, saved=0x4000, dx=0x5000, dw=0x6000, ws=0x10000)
    a.update(places)
    refused(sb, BAD, "sb_gated_grad", a["dh"], 8, a["x"], 16, a["w"], 16, a["saved"], 16, a["dx"], 16, a["dw"], 16, 2, 0, 16, 8, 16, 2, 0, a["ws"],
            1 << 20, None)


def test_4_bit_outputs_in_the_place_of_what_they_are_made_from(sb):
    for c in (0x1000, 0x2000, 0x3000, 0x5000):
        refused(sb, BAD, "sb_matmul_int4", 0x1000, 64, 2, 0x2000, 32, 0x3000, 2, c, 8, 2, 8, 64, 64, 0, 1, 0x5000, None)
    for codes, scales in ((0x1000, 0x3000), (0x2000, 0x1000), (0x2000, 0x2000)):
        refused(sb, BAD, "sb_quantize_int4", 0x1000, 64, 0, 4, 64, 32, codes, 32, scales, 2, None)
    for out in (0x1000, 0x2000):
        refused(sb, BAD, "sb_dequantize_int4", 0x1000, 32, 0x2000, 2, out, 64, 2, 4, 64, 64, None)


def test_matrices_that_are_turned_over(sb):
    """The right number of values in the wrong layout."""
    b, p = "bfloat16", sb.primitives
    codes, scales, a, c = Fake((8, 64), "uint8"), Fake((8, 4), b), Fake((2, 128), b), Fake((2, 8))          # scales are [4, 8]
    with pytest.raises(ValueError):
        sb.matmul_int4(a, codes, scales, c, group=32)
    with pytest.raises(ValueError):
        sb.quantize_int4(Fake((8, 128)), codes, scales, group=32)
    with pytest.raises(ValueError):
        sb.dequantize_int4(codes, scales, Fake((8, 128)), group=32)
    x, t, v = Fake((4, 8)), Fake((4,), "int32"), Fake((4,))
    for more in ({"mask": Fake((8, 4), "uint8")}, {"stats": Fake((2, 4))}):
        with pytest.raises(ValueError):
            p.log_probs(x, t, v, **more)
    with pytest.raises(ValueError):
        p.log_probs_grad(x, t, Fake((2, 4)), Fake((4, 8)), dout=v)
    with pytest.raises(ValueError):
        p.log_probs_grad(x, t, Fake((4, 2)), Fake((4, 8)), dout=v, mask=Fake((8, 4), "uint8"))


def test_matrices_in_one_dimension(sb):
    """Row by row is what they are: accepted."""
    from spiral_b200.device import array_ptr
    assert array_ptr(Fake((32,), "uint8"), 32, "u8", "mask", 8) == array_ptr(Fake((4, 8), "uint8"), 32, "u8", "mask", 8) == 0x1000
    assert array_ptr(Fake((2, 2, 8), "uint8"), 32, "u8", "mask", 8) == 0x1000 and array_ptr(None, 32, "u8", "mask", 8) is None


def test_log_probs_in_the_place_of_what_they_are_made_from(sb):
    for place in (0x1000, 0x8000):
        for name in range(5):
            outs = [0x3000, 0x4000, 0x5000, 0x6000, 0x7000]
            outs[name] = place
            out, h, stats, values, places = outs
            refused(sb, BAD, "sb_log_probs", 0x1000, 8, 0, 4, 8, 0x8000, -1, 1.0, 0x2000, 4, out, h, stats, 2, values, places, None)
    for d, ldd in ((0x1000, 16), (0x2000, 8), (0x3000, 8), (0x4000, 8), (0x5000, 8), (0x6000, 8), (0x8000, 8)):
        refused(sb, BAD, "sb_log_probs_grad", 0x1000, 8, 2, 4, 8, 0x8000, -1, 1.0, 0x2000, 4, 0x3000, 0x4000, 0x5000, 0x6000, d, ldd, None)


def test_workspaces_of_exact_gradients(sb):
    from spiral_b200 import _lib
    need, exact = ctypes.c_size_t(0), ctypes.c_size_t(0)
    _lib.call("sb_gated_grad_workspace_bytes", 1000, 64, 32, ctypes.byref(need))
    _lib.call("sb_gated_grad_exact_workspace_bytes", 1000, 64, 32, ctypes.byref(exact))
    assert exact.value >= need.value + 1000 * 128 * 2 and sb.gated_grad_workspace(1000, 64, 32, exact=True) == exact.value
    refused(sb, BAD, "sb_gated_grad_exact_workspace_bytes", 1, -1, 1, ctypes.byref(need))
    args = [0x1000000, 64, 0x2000000, 32, 0x3000000, 32, 0x4000000, 128, 0x5000000, 32, 0x6000000, 32, 2, 0, 1000, 64, 32, 2]
    refused(sb, BAD, "sb_gated_grad", *args, _lib.GATED_EXACT, 0x10000000, exact.value - 1, None)
    refused(sb, UNSUPPORTED, "sb_gated_grad", *args, 32, 0x10000000, exact.value, None)
    refused(sb, UNSUPPORTED, "sb_gated", 0x1000, 16, 0x2000, 16, 0x3000, 8, None, 16, 4, 8, 16, 2, _lib.GATED_EXACT, None)
