"""GEMM call surface: the reference's ``matmul_tf32 a_trans b_trans alpha a b beta c``.

Reference: ml/matmul/run.spi:21-26 -- M and N come from ``c``'s shape, K from
``a``'s (swapped when ``a_trans``), every tensor is row-major and ``c`` is
updated in place: ``c <- alpha * op(a) @ op(b) + beta * c``.
"""
import ctypes

from . import _lib
from .device import (Workspaces, array_ptr, device_ptr, dtype_tag, keep_tf32, matrix_of, nbytes_of, stream_ptr, stream_workspace, typed_matrix,
                     values_ptr)

EPILOGUE_FLAGS = {
    "bias": _lib.EPI_BIAS, "relu": _lib.EPI_RELU, "relu_grad": _lib.EPI_RELU_GRAD,
    "masked_softmax": _lib.EPI_MASKED_SOFTMAX, "regret_matching": _lib.EPI_REGRET_MATCHING,
    "argmax": _lib.EPI_ARGMAX, "relu_mask_out": _lib.EPI_RELU_MASK_OUT, "relu_grad_mask": _lib.EPI_RELU_GRAD_MASK,
    "colsum_out": _lib.EPI_COLSUM_OUT, "ln_l2": _lib.EPI_LN_L2,
}


def _shape2(x, what):
    shape = tuple(getattr(x, "shape", ()))
    if len(shape) != 2:
        raise ValueError("%s must be a 2-D array, got shape %s" % (what, shape))
    return int(shape[0]), int(shape[1])


def _dims(a_trans, b_trans, a, b, c):
    m, n = _shape2(c, "c")
    ar, ac = _shape2(a, "a")
    br, bc = _shape2(b, "b")
    am, k = (ac, ar) if a_trans else (ar, ac)
    bk, bn = (bc, br) if b_trans else (br, bc)
    if am != m or bn != n or bk != k:
        raise ValueError("shape mismatch: op(a) is %dx%d, op(b) is %dx%d, c is %dx%d" % (am, k, bk, bn, m, n))
    return m, n, k


_F32X3_WORKSPACES = Workspaces()


def _f32x3_aligned(a_trans, b_trans, m, n, k):
    """Contiguous dimensions are multiples of 4 elements (16-byte row pitches for the split operands)."""
    return n % 4 == 0 and (m % 4 == 0 if a_trans else k % 4 == 0) and (k % 4 == 0 if b_trans else n % 4 == 0)


def _f32x3_workspace(m, n, k, stream):
    ws = _F32X3_WORKSPACES.of(stream)
    if ws is not None and ws.nbytes >= 8 * (m + n) * k + 1024:      # no more than this is ever asked for
        return ws
    need = ctypes.c_size_t(0)
    _lib.call("sb_matmul_f32_workspace_bytes", m, n, k, ctypes.byref(need))
    return _F32X3_WORKSPACES.grown(need.value, stream)


def matmul(a_trans, b_trans, alpha, a, b, beta, c, in_dtype=None, epilogue=(), bias=None, mask=None,
           aux_in=None, aux_out=None, stream=None):
    """``c <- alpha * op(a) @ op(b) + beta * c`` with an optional fused epilogue.

    ``in_dtype``: 'f32' (1e-5 class: 3 x TF32 on the tensor cores where the contiguous
    dimensions are multiples of 4 and the epilogue is bias / ReLU, FFMA otherwise), 'tf32'
    (fp32 storage, TF32 multiply), 'bf16', 'f16'; by default fp32 storage runs as 'tf32', the reference's own
    arithmetic.  ``epilogue``: iterable of names from EPILOGUE_FLAGS.
    """
    m, n, k = _dims(bool(a_trans), bool(b_trans), a, b, c)
    storage, storage_b = dtype_tag(a), dtype_tag(b)
    fp32_storage = ("f32", "tf32")                 # 'tf32' tags fp32 storage whose values are TF32-rounded
    if storage != storage_b and not (storage in fp32_storage and storage_b in fp32_storage):
        raise TypeError("a and b must share a storage dtype (%s vs %s)" % (storage, storage_b))
    if in_dtype is None:
        in_dtype = "tf32" if storage in ("f32", "tf32") else storage
    if (in_dtype in ("f32", "tf32")) != (storage in ("f32", "tf32")) or \
            (in_dtype in ("bf16", "f16") and in_dtype != storage):
        raise TypeError("in_dtype %s does not match the storage dtype %s" % (in_dtype, storage))
    out_dtype = dtype_tag(c)   # a 'tf32'-tagged output is fp32 storage rounded to TF32
    epi = 0
    for name in epilogue:
        epi |= EPILOGUE_FLAGS[name]
    if in_dtype == "f32" and out_dtype == "f32" and not (epi & ~(_lib.EPI_BIAS | _lib.EPI_RELU)) and k > 0 \
            and _f32x3_aligned(bool(a_trans), bool(b_trans), m, n, k) and device_ptr(c) % 16 == 0:
        # fp32 class on the tensor cores (3 x TF32); the split operands live in a workspace this host
        # keeps per device, stream and thread and grows on demand (the C ABI itself allocates nothing).
        ws = _f32x3_workspace(m, n, k, stream)
        _lib.call("sb_matmul_f32x3", int(bool(a_trans)), int(bool(b_trans)), ctypes.c_float(alpha), device_ptr(a),
                  device_ptr(b), ctypes.c_float(beta), device_ptr(c), m, n, k, epi, device_ptr(bias), ws.ptr,
                  ws.nbytes, stream_ptr(stream))
        return c
    _lib.call("sb_matmul_ex", int(bool(a_trans)), int(bool(b_trans)), ctypes.c_float(alpha),
              device_ptr(a), device_ptr(b), ctypes.c_float(beta), device_ptr(c), m, n, k,
              _lib.DTYPE_CODES[in_dtype], _lib.DTYPE_CODES[out_dtype], epi, device_ptr(bias),
              device_ptr(mask), device_ptr(aux_in), device_ptr(aux_out), stream_ptr(stream))
    return c


HEAD_FLAGS = {"masked_softmax": _lib.EPI_MASKED_SOFTMAX, "softmax": _lib.EPI_MASKED_SOFTMAX,
              "regret_matching": _lib.EPI_REGRET_MATCHING, "argmax": _lib.EPI_ARGMAX, "sample": _lib.EPI_SAMPLE,
              "binarize": _lib.EPI_BINARIZE}


def head_spec(head=(), prefix=-1, mask=None, argmax_out=None, sample_out=None, hash_out=None, modulo=0,
              seed=0, row_offset=0, position=0):
    """The ctypes ``sb_head_spec`` of a row head: ``head`` names from HEAD_FLAGS; legal columns are
    ``j < prefix`` when ``prefix >= 0`` (the reference's ``masked_softmax size`` etc.), else ``mask``,
    else all; a sampling head draws output ``position`` of the Philox stream (seed, row_offset + row)."""
    flags = 0
    for name in head:
        flags |= HEAD_FLAGS[name]
    return _lib.HeadSpec(flags, int(prefix), device_ptr(mask), device_ptr(argmax_out), device_ptr(sample_out),
                         device_ptr(hash_out), int(modulo), int(seed), int(row_offset), int(position))


def matmul_head(a_trans, b_trans, alpha, a, b, beta, c, spec, in_dtype=None, epilogue=(), bias=None, stream=None):
    """``c <- head(alpha * op(a) @ op(b) + beta * c (+ bias) (relu))`` with the row head ``spec``
    (``head_spec(...)``); fp32 output.  One launch for rows of up to 64 columns, or up to 256 under a
    prefix mask of at most 64 columns; nothing is allocated."""
    m, n, k = _dims(bool(a_trans), bool(b_trans), a, b, c)
    storage = dtype_tag(a)
    if in_dtype is None:
        in_dtype = "tf32" if storage in ("f32", "tf32") else storage
    epi = 0
    for name in epilogue:
        epi |= EPILOGUE_FLAGS[name]
    _lib.call("sb_matmul_head", int(bool(a_trans)), int(bool(b_trans)), ctypes.c_float(alpha), device_ptr(a),
              device_ptr(b), ctypes.c_float(beta), device_ptr(c), m, n, k, _lib.DTYPE_CODES[in_dtype], epi,
              device_ptr(bias), ctypes.byref(spec), stream_ptr(stream))
    return c


def matmul_tf32(a_trans, b_trans, alpha, a, b, beta, c, stream=None):
    """Drop-in for the reference's ``matmul_tf32`` (fp32 storage, TF32 multiply, fp32 accumulate)."""
    m, n, k = _dims(bool(a_trans), bool(b_trans), a, b, c)
    for x, what in ((a, "a"), (b, "b"), (c, "c")):
        if dtype_tag(x) not in ("f32", "tf32"):
            raise TypeError("matmul_tf32: %s must be fp32" % what)
    _lib.call("sb_matmul_tf32", int(bool(a_trans)), int(bool(b_trans)), ctypes.c_float(alpha),
              device_ptr(a), device_ptr(b), ctypes.c_float(beta), device_ptr(c), m, n, k,
              stream_ptr(stream))
    return c


def matmul_plan(a_trans, b_trans, m, n, k, in_dtype="tf32", epilogue=()):
    """Tile plan of the tensor-core path for a product with ``epilogue`` (names as for ``matmul``):
    dict(block_m, block_n, block_k, stages, grid).

    Counterpart of matmul_config_tf32 (ml/matmul/run.spi:8-19); unlike it, no
    divisibility of m, n, k by the tile is demanded (ragged edges are zero-filled).
    """
    plan = (ctypes.c_int * 5)()
    epi = 0
    for name in epilogue:
        epi |= EPILOGUE_FLAGS[name]
    _lib.call("sb_matmul_plan", int(bool(a_trans)), int(bool(b_trans)), int(m), int(n), int(k),
              _lib.DTYPE_CODES[in_dtype], epi, plan)
    return dict(zip(("block_m", "block_n", "block_k", "stages", "grid"), list(plan)))


_FP8_FLOATS = {"f32": _lib.F32, "tf32": _lib.F32, "bf16": _lib.BF16, "f16": _lib.F16}
_FP8_EPILOGUES = {(): 0, ("bias",): _lib.EPI_BIAS, ("relu",): _lib.EPI_RELU, ("bias", "relu"): _lib.EPI_BIAS | _lib.EPI_RELU}


def _fp8_codes(x, what):
    if dtype_tag(x) not in ("e4m3", "u8"):
        raise TypeError("%s must hold e4m3 codes, not %s" % (what, dtype_tag(x)))
    return device_ptr(x)


def quantize_fp8(x, codes, scales, block_rows=1, stream=None):
    """E4M3 ``codes`` of the matrix ``x`` (fp32, bf16, f16) with a scale per block of ``block_rows`` x 128: scale = largest
    magnitude / 448.  ``block_rows`` 1 is for activations, ``scales`` fp32 [ceil(cols / 128), rows]; 128 is for weights,
    ``scales`` fp32 [ceil(rows / 128), ceil(cols / 128)].  Returns (codes, scales)."""
    rows, cols, ldx = matrix_of(x, "x")
    crows, ccols, ldc = matrix_of(codes, "codes")
    if (crows, ccols) != (rows, cols):
        raise ValueError("quantize_fp8: codes are %dx%d, x is %dx%d" % (crows, ccols, rows, cols))
    if block_rows not in (1, 128):
        raise ValueError("quantize_fp8: blocks are 1 x 128 or 128 x 128")
    tag = dtype_tag(x)
    if tag not in _FP8_FLOATS:
        raise TypeError("quantize_fp8: x must hold f32, bf16 or f16, not %s" % tag)
    across = -(-cols // 128)
    _lib.call("sb_quantize_fp8", device_ptr(x), ldx, _FP8_FLOATS[tag], rows, cols, block_rows, _fp8_codes(codes, "codes"), ldc,
              values_ptr(scales, across * (rows if block_rows == 1 else -(-rows // 128)), "scales"), stream_ptr(stream))
    return codes, scales


def matmul_fp8(a, a_scales, b, b_scales, c, epilogue=(), bias=None, stream=None):
    """``c <- a @ b^T`` of E4M3 codes with their scales, fp32 accumulation: a dense layer in 8 bits.

    ``a`` [m, k] with ``a_scales`` [ceil(k / 128), m] (``quantize_fp8`` with block_rows 1), ``b`` [n, k] with ``b_scales``
    [ceil(n / 128), ceil(k / 128)] (block_rows 128), ``c`` [m, n] in fp32, bf16 or f16; ``epilogue``: "bias" (fp32 [n]),
    "relu" (a NaN gives 0, as in ``matmul``).  Rows may have a pitch.  Rows of codes that start on 16 bytes (a pitch of a multiple of 16, whatever k is) run
    on the tensor cores, others on the CUDA cores at about 1 % of their rate."""
    m, k, lda = matrix_of(a, "a")
    n, kb, ldb = matrix_of(b, "b")
    cm, cn, ldc = matrix_of(c, "c")
    if kb != k or cm != m or cn != n:
        raise ValueError("shape mismatch: a is %dx%d, b^T is %dx%d, c is %dx%d" % (m, k, kb, n, cm, cn))
    tag = dtype_tag(c)
    if tag not in _FP8_FLOATS:
        raise TypeError("matmul_fp8: c must hold f32, bf16 or f16, not %s" % tag)
    epi = _FP8_EPILOGUES.get(tuple(epilogue))
    if epi is None:
        raise ValueError("matmul_fp8: the epilogue is made of bias and relu, got %r" % (epilogue,))
    if epi & _lib.EPI_BIAS and bias is None:
        raise ValueError("matmul_fp8: bias must be %d fp32 values" % n)
    across = -(-k // 128)
    _lib.call("sb_matmul_fp8", _fp8_codes(a, "a"), lda, values_ptr(a_scales, across * m, "a_scales"), _fp8_codes(b, "b"), ldb,
              values_ptr(b_scales, -(-n // 128) * across, "b_scales"), device_ptr(c), ldc, m, n, k, _FP8_FLOATS[tag], epi,
              values_ptr(bias, n, "bias") if epi & _lib.EPI_BIAS else None, stream_ptr(stream))
    return keep_tf32(c, stream)


def matmul_fp8_plan(m, n, k):
    """Tile plan of ``matmul_fp8`` on the tensor cores: dict(block_m, block_n, splits).  ``block_m`` below 128 is the form
    for few rows, ``splits`` the CTAs of a cluster that share k."""
    plan = (ctypes.c_int * 3)()
    _lib.call("sb_matmul_fp8_plan", int(m), int(n), int(k), plan)
    return dict(zip(("block_m", "block_n", "splits"), list(plan)))


ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU}
_GATED = {"bf16": _lib.BF16, "f16": _lib.F16}


def _gated_matrix(who, x, what, tag, rows, cols):
    """Address and pitch of a matrix of the layer's storage type and the given shape."""
    r, c, ld, ptr, own = typed_matrix(x, what)
    if r != rows or c != cols or own != tag:
        raise ValueError("%s: %s must be %s, %dx%d" % (who, what, tag, rows, cols))
    return ptr, ld


def _gated_sizes(who, x, w, activation):
    m, k, ldx, x, tag = typed_matrix(x, "x")
    f2, kw, ldw, w, w_tag = typed_matrix(w, "w")
    if tag not in _GATED:
        raise TypeError("%s: x must hold bf16 or f16, not %s" % (who, tag))
    if f2 % 2 or kw != k or w_tag != tag:
        raise ValueError("%s: w must be %s, an even number of rows of %d" % (who, tag, k))
    if activation not in ACTIVATIONS:
        raise ValueError("%s: the activation is one of %s, got %r" % (who, ", ".join(sorted(ACTIVATIONS)), activation))
    return m, f2 // 2, k, x, ldx, w, ldw, tag, ACTIVATIONS[activation]


def gated(x, w, out, activation="silu", saved=None, stream=None):
    """A gated layer in one kernel: ``out = act(x @ w[:f]^T) * (x @ w[f:]^T)``.

    ``x`` [m, k], ``w`` [2 f, k] (the gate's rows, then the other projection's), ``out`` [m, f] in bf16 or f16, one type; rows may have a
    pitch.  ``activation``: "silu", "gelu" (of the normal distribution) or "relu".  ``saved`` [m, 2 f]: where given, both projections are left there for
    ``gated_grad``.  Rows of x and w that start on 16 bytes run on the tensor cores, others on the CUDA cores at about 1 % of their rate."""
    m, f, k, x, ldx, w, ldw, tag, act = _gated_sizes("gated", x, w, activation)
    h, ldh = _gated_matrix("gated", out, "out", tag, m, f)
    lds = 2 * f
    if saved is not None:
        saved, lds = _gated_matrix("gated", saved, "saved", tag, m, 2 * f)
    _lib.call("sb_gated", x, ldx, w, ldw, h, ldh, saved, lds, m, f, k, _GATED[tag], act, stream_ptr(stream))
    return out


def gated_grad(dout, x, w, saved, dx=None, dw=None, activation="silu", accumulate=False, workspace=None, stream=None, exact=False):
    """Gradient of ``gated`` from ``dout`` [m, f] and what it ``saved``: ``dx`` (like ``x``) and ``dw`` (like ``w``, or fp32), each where given;
    ``accumulate`` adds to the old ``dw``.  The projections' gradients are rounded to the storage type for the products, which is as large an error
    as the rounding of a 16-bit gradient itself and all of that of an fp32 ``dw``; up to 64 rows, and with ``exact`` for any number, what that
    rounding leaves off is multiplied too (with many rows at about twice the time).  ``workspace``: device memory of ``gated_grad_workspace`` bytes; by
    default one is kept per device, stream and host thread.  ``dx`` may not be ``w``, nor ``dw`` ``x``; where both are wanted ``dx`` may not be ``x`` either, nor ``dw`` ``w``.
    Returns (dx, dw)."""
    m, f, k, x, ldx, w, ldw, tag, act = _gated_sizes("gated_grad", x, w, activation)
    dh, lddh = _gated_matrix("gated_grad", dout, "dout", tag, m, f)
    saved, lds = _gated_matrix("gated_grad", saved, "saved", tag, m, 2 * f)
    dx_ptr, lddx, dw_ptr, lddw, dw_tag = None, k, None, k, tag
    if dx is not None:
        dx_ptr, lddx = _gated_matrix("gated_grad", dx, "dx", tag, m, k)
    if dw is not None:
        rows, cols, lddw, dw_ptr, dw_tag = typed_matrix(dw, "dw")
        if dw_tag not in (tag, "f32", "tf32"):
            raise TypeError("gated_grad: dw must hold %s or f32, not %s" % (tag, dw_tag))
        if rows != 2 * f or cols != k:
            raise ValueError("gated_grad: dw must be like w, %dx%d" % (2 * f, k))
    nbytes = gated_grad_workspace(m, f, k, exact) if workspace is None else nbytes_of(workspace)
    act |= _lib.GATED_EXACT if exact else 0
    if workspace is None:
        workspace = stream_workspace(nbytes, stream)
    _lib.call("sb_gated_grad", dh, lddh, x, ldx, w, ldw, saved, lds, dx_ptr, lddx, dw_ptr, lddw, _GATED.get(dw_tag, _lib.F32),
              int(bool(accumulate)), m, f, k, _GATED[tag], act, device_ptr(workspace), nbytes, stream_ptr(stream))
    return dx, keep_tf32(dw, stream)


def gated_plan(m, f, k):
    """What ``gated`` takes for rows of x and w that start on 16 bytes: rows and columns of h in a tile (8 or 16 rows: the form for few
    rows; 256: a pair of CTAs), tiles, and tiles of half the columns behind them."""
    plan = (ctypes.c_int * 4)()
    _lib.call("sb_gated_plan", int(m), int(f), int(k), plan)
    return dict(zip(("rows", "columns", "tiles", "half_tiles"), list(plan)))


def gated_grad_plan(m, f, k, dx=True, dw=True):
    """What the products of ``gated_grad`` take where rows start on 16 bytes: columns of a tile (of 256 rows), and for dx and dw the tiles of
    all K, those in parts of K, and the parts."""
    plan = (ctypes.c_int * 7)()
    _lib.call("sb_gated_grad_plan", int(m), int(f), int(k), int(bool(dx)) + 2 * int(bool(dw)), plan)
    return {"columns": plan[0], "dx": tuple(plan[1:4]), "dw": tuple(plan[4:7])}


def gated_grad_workspace(m, f, k, exact=False):
    """Bytes of device memory that ``gated_grad`` needs for m rows and a [2 f, k] weight matrix."""
    nbytes = ctypes.c_size_t(0)
    _lib.call("sb_gated_grad_exact_workspace_bytes" if exact else "sb_gated_grad_workspace_bytes", m, f, k, ctypes.byref(nbytes))
    return nbytes.value


def _int4_weights(who, codes, scales, k, group):
    """Rows, address and pitch of 4-bit weights of k columns, address and type of their scales."""
    n, nbytes, ldw, codes, tag = typed_matrix(codes, "codes")
    if tag != "u8":
        raise TypeError("%s: codes must be bytes, not %s" % (who, tag))
    if group not in (32, 64, 128):
        raise ValueError("%s: groups are of 32, 64 or 128" % who)
    if nbytes != (k + 1) // 2:
        raise ValueError("%s: codes of %d columns are %d bytes a row, got %d" % (who, k, (k + 1) // 2, nbytes))
    tag = dtype_tag(scales)
    if tag not in _GATED:
        raise TypeError("%s: scales must hold bf16 or f16, not %s" % (who, tag))
    return n, codes, ldw, array_ptr(scales, -(-k // group) * n, tag, "scales", n), _GATED[tag]


def quantize_int4(x, codes, scales, group=128, stream=None):
    """4-bit ``codes`` (uint8 [n, ceil(k / 2)], two in a byte, the even column in the low half) of the weights ``x`` [n, k] (fp32, bf16,
    f16) with a scale per ``group`` (32, 64, 128) columns of a row: ``scales`` [ceil(k / group), n] in bf16 or f16, the largest
    magnitude / 7.  A weight is ``scale * (code - 8)``.  Returns (codes, scales)."""
    rows, k, ldx, x, tag = typed_matrix(x, "x")
    n, codes_ptr, ldc, scales_ptr, scale_code = _int4_weights("quantize_int4", codes, scales, k, group)
    if tag not in _FP8_FLOATS:
        raise TypeError("quantize_int4: x must hold f32, bf16 or f16, not %s" % tag)
    if n != rows:
        raise ValueError("quantize_int4: codes have %d rows, x has %d" % (n, rows))
    _lib.call("sb_quantize_int4", x, ldx, _FP8_FLOATS[tag], n, k, group, codes_ptr, ldc, scales_ptr, scale_code, stream_ptr(stream))
    return codes, scales


def dequantize_int4(codes, scales, out, group=128, stream=None):
    """The weights [n, k] that 4-bit ``codes`` and ``scales`` stand for, in fp32, bf16 or f16: for products of many rows."""
    rows, k, ldo, out_ptr, tag = typed_matrix(out, "out")
    n, codes, ldw, scales, scale_code = _int4_weights("dequantize_int4", codes, scales, k, group)
    if tag not in _FP8_FLOATS:
        raise TypeError("dequantize_int4: out must hold f32, bf16 or f16, not %s" % tag)
    if n != rows:
        raise ValueError("dequantize_int4: codes have %d rows, out has %d" % (n, rows))
    _lib.call("sb_dequantize_int4", codes, ldw, scales, scale_code, out_ptr, ldo, _FP8_FLOATS[tag], n, k, group, stream_ptr(stream))
    return keep_tf32(out, stream)


def matmul_int4(a, codes, scales, c, group=128, epilogue=(), bias=None, stream=None):
    """``c <- a @ w^T`` with 4-bit weights (``quantize_int4``): a dense layer for few rows, whose time is that of the weights' bytes.

    ``a`` [m, k] in bf16 or f16, ``c`` [m, n] in fp32, bf16 or f16, fp32 accumulation; ``epilogue``: "bias" (fp32 [n]), "relu" (a NaN gives 0, as in
    ``matmul``).  Rows may have a pitch.  Made for up to 64 rows; for many, ``dequantize_int4`` and ``matmul`` are faster."""
    m, k, lda, a, a_tag = typed_matrix(a, "a")
    n, codes, ldw, scales, scale_code = _int4_weights("matmul_int4", codes, scales, k, group)
    cm, cn, ldc, c_ptr, tag = typed_matrix(c, "c")
    if cm != m or cn != n:
        raise ValueError("shape mismatch: a is %dx%d, w^T is %dx%d, c is %dx%d" % (m, k, k, n, cm, cn))
    if a_tag not in _GATED:
        raise TypeError("matmul_int4: a must hold bf16 or f16, not %s" % a_tag)
    if tag not in _FP8_FLOATS:
        raise TypeError("matmul_int4: c must hold f32, bf16 or f16, not %s" % tag)
    epi = _FP8_EPILOGUES.get(tuple(epilogue))
    if epi is None:
        raise ValueError("matmul_int4: the epilogue is made of bias and relu, got %r" % (epilogue,))
    if epi & _lib.EPI_BIAS and bias is None:
        raise ValueError("matmul_int4: bias must be %d fp32 values" % n)
    _lib.call("sb_matmul_int4", a, lda, _GATED[a_tag], codes, ldw, scales, scale_code, c_ptr, ldc, m, n, k, group, _FP8_FLOATS[tag], epi,
              array_ptr(bias, n, "f32", "bias") if epi & _lib.EPI_BIAS else None, stream_ptr(stream))
    return keep_tf32(c, stream)


def matmul_int4_plan(m, n, k, group=128):
    """What ``matmul_int4`` takes for contiguous matrices that start on 16 bytes: rows of a in a block (0: up to 8, through registers
    alone) and blocks that share K."""
    plan = (ctypes.c_int * 2)()
    _lib.call("sb_matmul_int4_plan", int(m), int(n), int(k), int(group), plan)
    return dict(zip(("rows", "blocks"), list(plan)))
