"""Arguments that the operators of token-reading nets refuse, before any launch (CPU only)."""
import ctypes

import numpy as np
import pytest


class Fake:
    """Something with a device address, a type and a shape."""

    def __init__(self, shape, dtype="float32", ptr=0x1000, strides=None):
        self.shape, self.dtype, self.ptr = shape, dtype, ptr
        self._strides = strides

    def data_ptr(self):
        return self.ptr

    def is_contiguous(self):
        return self._strides is None

    def stride(self):
        if self._strides is not None:
            return self._strides
        out, at = [], 1
        for n in reversed(self.shape):
            out.append(at)
            at *= n
        return tuple(reversed(out))


def refused(sb, code, call, *args):
    from spiral_b200 import _lib
    with pytest.raises(sb.SpiralError) as e:
        _lib.call(call, *args)
    assert e.value.code == code, str(e.value)


BAD, MISALIGNED, UNSUPPORTED, LARGE = -1, -2, -3, -6


def test_embedding(sb):
    def go(tokens=0x1000, index=4, n=4, table=0x2000, ldt=8, tt=0, vocab=5, dim=8, out=0x3000, ldo=8, ot=0):
        return ("sb_embedding", tokens, index, n, table, ldt, tt, vocab, dim, 1.0, out, ldo, ot, None)
    refused(sb, BAD, *go(tokens=None))
    refused(sb, BAD, *go(table=None))
    refused(sb, BAD, *go(out=None))
    refused(sb, BAD, *go(n=-1))
    refused(sb, BAD, *go(ldt=7))
    refused(sb, BAD, *go(ldo=7))
    refused(sb, UNSUPPORTED, *go(index=0))
    refused(sb, UNSUPPORTED, *go(tt=1))
    refused(sb, UNSUPPORTED, *go(ot=5))
    refused(sb, MISALIGNED, *go(tokens=0x1002))
    refused(sb, MISALIGNED, *go(tokens=0x1004, index=6))
    refused(sb, MISALIGNED, *go(out=0x3002))


def test_embedding_grad(sb):
    def go(tokens=0x1000, index=4, n=4, dout=0x2000, ldd=8, dt=0, dtable=0x3000, ldt=8, vocab=5, dim=8, ws=0x4000, nws=1 << 30):
        return ("sb_embedding_grad", tokens, index, n, dout, ldd, dt, 1.0, dtable, ldt, vocab, dim, 0, ws, nws, None)
    for k in ("tokens", "dout", "dtable", "ws"):
        refused(sb, BAD, *go(**{k: None}))
    refused(sb, BAD, *go(nws=64))
    refused(sb, BAD, *go(ldd=7))
    refused(sb, BAD, *go(vocab=-1))
    refused(sb, UNSUPPORTED, *go(index=1))
    refused(sb, UNSUPPORTED, *go(dt=7))
    refused(sb, MISALIGNED, *go(ws=0x4008))
    refused(sb, MISALIGNED, *go(dout=0x2002))
    refused(sb, LARGE, *go(n=(1 << 30) + 1))
    need = ctypes.c_size_t(0)
    refused(sb, BAD, "sb_embedding_grad_workspace_bytes", 4, 4, 4, None)
    refused(sb, BAD, "sb_embedding_grad_workspace_bytes", -4, 4, 4, ctypes.byref(need))


def test_layer_norm(sb):
    def go(x=0x1000, ldx=8, y=0x2000, ldy=8, eps=1e-5, rows=3, cols=8, dt=0, w=None, mean=None):
        return ("sb_layer_norm", x, ldx, y, ldy, w, None, eps, mean, None, rows, cols, dt, None)
    refused(sb, BAD, *go(x=None))
    refused(sb, BAD, *go(y=None))
    refused(sb, BAD, *go(ldx=7))
    refused(sb, BAD, *go(rows=-1))
    refused(sb, BAD, *go(eps=-1.0))
    refused(sb, BAD, *go(eps=float("nan")))
    refused(sb, UNSUPPORTED, *go(dt=4))
    refused(sb, MISALIGNED, *go(x=0x1002))
    refused(sb, MISALIGNED, *go(w=0x1002))
    refused(sb, MISALIGNED, *go(mean=0x1001))


def test_layer_norm_grad(sb):
    def go(dy=0x1000, x=0x2000, mean=0x3000, rstd=0x4000, dx=0x5000, ld=8, dw=0x6000, db=0x7000, rows=3, cols=8, dt=0, ws=0x8000, nws=1 << 30):
        return ("sb_layer_norm_grad", dy, ld, x, ld, mean, rstd, None, dx, ld, dw, db, 0, rows, cols, dt, ws, nws, None)
    for k in ("dy", "x", "mean", "rstd", "ws"):
        refused(sb, BAD, *go(**{k: None}))
    refused(sb, BAD, *go(nws=8))
    refused(sb, BAD, *go(ld=7))
    refused(sb, BAD, *go(rows=-1))
    refused(sb, UNSUPPORTED, *go(dt=6))
    refused(sb, MISALIGNED, *go(dy=0x1001))
    refused(sb, MISALIGNED, *go(db=0x7002))


def test_adamw(sb):
    from spiral_b200 import _lib

    def go(n=1, tensor=None, state=0, grad=0, copy=0, step=1, b1=0.9, eps=1e-8, table=True, **fields):
        t = _lib.AdamwTensor(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, None, 10)
        for k, v in fields.items():
            setattr(t, k, v)
        h = _lib.AdamwHyper(1e-3, b1, 0.999, eps, 0.01, 1.0, step, 0)
        return ("sb_adamw_step", n, (_lib.AdamwTensor * 1)(t) if table else None, state, grad, copy, ctypes.byref(h), None)
    for k in ("param", "grad_", "exp_avg", "exp_avg_sq"):
        refused(sb, BAD, *go(**{k.rstrip("_"): None}) if k != "grad_" else go_null_grad(go))
    refused(sb, BAD, *go(n=-1))
    refused(sb, BAD, *go(table=False))
    refused(sb, BAD, *go(step=0))
    refused(sb, BAD, *go(b1=1.0))
    refused(sb, BAD, *go(b1=float("nan")))
    refused(sb, BAD, *go(eps=-1.0))
    refused(sb, BAD, *go(state=7, exp_avg_scale=None))
    refused(sb, UNSUPPORTED, *go(state=2))
    refused(sb, UNSUPPORTED, *go(grad=1))
    refused(sb, UNSUPPORTED, *go(copy=4))
    refused(sb, MISALIGNED, *go(param=0x1002))
    refused(sb, MISALIGNED, *go(exp_avg=0x3001))
    refused(sb, MISALIGNED, *go(state=7, exp_avg_sq_scale=0x6001))


def go_null_grad(go):
    call = list(go())
    call[2][0].grad = None
    return call


def test_fp8(sb):
    def q(x=0x1000, ldx=16, dt=0, rows=3, cols=16, block=1, codes=0x2000, ldc=16, scales=0x3000):
        return ("sb_quantize_fp8", x, ldx, dt, rows, cols, block, codes, ldc, scales, None)
    for k in ("x", "codes", "scales"):
        refused(sb, BAD, *q(**{k: None}))
    refused(sb, BAD, *q(ldx=15))
    refused(sb, BAD, *q(rows=-1))
    refused(sb, UNSUPPORTED, *q(block=64))
    refused(sb, UNSUPPORTED, *q(dt=7))
    refused(sb, MISALIGNED, *q(x=0x1002))
    refused(sb, MISALIGNED, *q(scales=0x3002))
    refused(sb, LARGE, *q(cols=128 * 65536, ldx=128 * 65536, ldc=128 * 65536))

    def mm(a=0x1000, lda=16, sa=0x2000, w=0x3000, ldw=16, sw=0x4000, c=0x5000, ldc=8, m=4, n=8, k=16, out=0, epi=0, bias=None):
        return ("sb_matmul_fp8", a, lda, sa, w, ldw, sw, c, ldc, m, n, k, out, epi, bias, None)
    for k in ("a", "sa", "w", "sw", "c"):
        refused(sb, BAD, *mm(**{k: None}))
    refused(sb, BAD, *mm(epi=1))
    refused(sb, BAD, *mm(lda=15))
    refused(sb, BAD, *mm(ldc=7))
    refused(sb, BAD, *mm(n=-1))
    refused(sb, UNSUPPORTED, *mm(out=7))
    refused(sb, UNSUPPORTED, *mm(epi=8))
    refused(sb, MISALIGNED, *mm(c=0x5002))
    refused(sb, MISALIGNED, *mm(sa=0x2002))


def test_python_side(sb):
    """Shapes, types and strides, before the C boundary."""
    p = sb.primitives
    t, table, out = Fake((4,), "int32"), Fake((5, 8)), Fake((4, 8))
    for bad in (lambda: p.embedding(t, table, Fake((5, 8))), lambda: p.embedding(t, table, Fake((4, 9))),
                lambda: p.embedding(t, Fake((5, 8), strides=(16, 2)), out), lambda: p.embedding(Fake((4,), "int32", strides=(2,)), table, out),
                lambda: p.embedding(t, Fake((5, 8), strides=(4, 1)), out), lambda: p.embedding_grad(t, Fake((3, 8)), table),
                lambda: p.layer_norm(out, Fake((4, 9))), lambda: p.layer_norm(out, out, weight=Fake((9,))),
                lambda: p.layer_norm(out, out, mean=Fake((5,))), lambda: p.layer_norm(Fake((2, 3, 8), strides=(50, 8, 1))),
                lambda: p.layer_norm_grad(Fake((4, 9)), out, Fake((4,)), Fake((4,))),
                lambda: sb.quantize_fp8(out, Fake((4, 9), "uint8"), Fake((1, 4))), lambda: sb.quantize_fp8(out, Fake((4, 8), "uint8"), Fake((2, 4))),
                lambda: sb.quantize_fp8(out, Fake((4, 8), "uint8"), Fake((1, 4)), block_rows=2),
                lambda: sb.matmul_fp8(Fake((4, 8), "uint8"), Fake((1, 4)), Fake((3, 9), "uint8"), Fake((1, 1)), Fake((4, 3))),
                lambda: sb.matmul_fp8(Fake((4, 8), "uint8"), Fake((1, 5)), Fake((3, 8), "uint8"), Fake((1, 1)), Fake((4, 3))),
                lambda: sb.matmul_fp8(Fake((4, 8), "uint8"), Fake((1, 4)), Fake((3, 8), "uint8"), Fake((1, 1)), Fake((4, 3)), epilogue=("argmax",)),
                lambda: sb.matmul_fp8(Fake((4, 8), "uint8"), Fake((1, 4)), Fake((3, 8), "uint8"), Fake((1, 1)), Fake((4, 3)), epilogue=("bias",)),
                lambda: sb.AdamW([Fake((4,))], []), lambda: sb.AdamW([Fake((4,))], [Fake((5,))], [Fake((4,))], [Fake((4,))]),
                lambda: sb.AdamW([Fake((4,))], [Fake((4,))], state="f16")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: p.embedding(Fake((4,), "uint8"), table, out), lambda: p.embedding(t, Fake((5, 8), "int32"), out),
                lambda: p.embedding_grad(t, out, Fake((5, 8), "bfloat16")), lambda: p.layer_norm(Fake((4, 8), "int32")),
                lambda: sb.quantize_fp8(Fake((4, 8), "uint8"), Fake((4, 8), "uint8"), Fake((1, 4))),
                lambda: sb.quantize_fp8(out, Fake((4, 8), "float16"), Fake((1, 4))),
                lambda: sb.matmul_fp8(Fake((4, 8), "uint8"), Fake((1, 4)), Fake((3, 8), "uint8"), Fake((1, 1)), Fake((4, 3), "uint8")),
                lambda: sb.AdamW([Fake((4,), "float16")], [Fake((4,))], [Fake((4,))], [Fake((4,))]),
                lambda: sb.AdamW([Fake((4,))], [Fake((4,), "int32")], [Fake((4,))], [Fake((4,))]),
                lambda: sb.AdamW([Fake((4,))], [Fake((4,))], [Fake((4,), "uint8")], [Fake((4,))])):
        with pytest.raises(TypeError):
            bad()


def test_sizes_of_nothing_need_no_device(sb):
    from spiral_b200 import _lib
    _lib.call("sb_embedding", None, 4, 0, None, 0, 0, 5, 8, 1.0, None, 8, 0, None)
    _lib.call("sb_layer_norm", None, 0, None, 0, None, None, 1e-5, None, None, 0, 8, 0, None)
    _lib.call("sb_adamw_step", 0, None, 0, 0, 0, None, None)
    _lib.call("sb_quantize_fp8", None, 0, 0, 0, 5, 1, None, 0, None, None)
    _lib.call("sb_matmul_fp8", None, 0, None, None, 0, None, None, 0, 0, 8, 16, 0, 0, None, None)


def test_workspaces_of_any_size(sb):
    """Nothing, one of a kind, the limits: an answer, and for more a refusal."""
    p = sb.primitives
    for n, vocab, dim in ((0, 5, 8), (3, 0, 8), (3, 5, 0), (1, 1, 1), (5, 3, 100000), (1 << 30, 1, 1), (1, 1 << 30, 1), (1 << 30, 1 << 30, 1)):
        assert p.embedding_grad_workspace(n, vocab, dim) >= 0
    for rows, cols in ((0, 5), (5, 0), (1, 1), (1 << 40, 3), (1, 1 << 30)):
        assert p.layer_norm_grad_workspace(rows, cols) >= 0
    with pytest.raises(sb.SpiralError):
        p.embedding_grad_workspace((1 << 30) + 1, 4, 4)


def test_e4m3_conversions(sb):
    """All codes there and back; halves go to even; beyond the range the largest value."""
    from spiral_b200 import dtypes
    codes = np.arange(256, dtype=np.uint8)
    values = dtypes.e4m3_bits_to_f32(codes)
    finite = (codes & 127) != 127
    assert np.array_equal(dtypes.f32_to_e4m3_bits(values)[finite], codes[finite]) and np.isnan(values[~finite]).all()
    assert values[0x7e] == 448 and values[1] == 2.0 ** -9 and values[0x08] == 2.0 ** -6 and values[0x38] == 1.0
    mid = (values[8:126].astype(np.float64) + values[9:127]) / 2
    even = np.where(codes[8:126] % 2 == 0, codes[8:126], codes[9:127])
    assert np.array_equal(dtypes.f32_to_e4m3_bits(mid.astype(np.float32)), even)
    assert list(dtypes.f32_to_e4m3_bits(np.float32([1e9, -1e9, np.inf, np.nan]))[:3]) == [0x7e, 0xfe, 0x7e]
