"""Stand-alone row / elementwise operations (reference: ml/primitives.spi:701-780, ml/layers.spi:353-420), and the
operators in front of the dense layers of a net that reads tokens (embedding, layer normalisation)."""
import ctypes

from . import _lib
from .device import device_ptr, dtype_tag, flat_size, keep_tf32, matrix_of, stream_ptr, stream_workspace, values_ptr


def _rows_cols(x):
    shape = tuple(x.shape)
    if len(shape) < 1:
        raise ValueError("row operation on a 0-d array")
    cols = int(shape[-1])
    rows = 1
    for s in shape[:-1]:
        rows *= int(s)
    return rows, cols


def relu(x, out=None, stream=None):
    out = x if out is None else out
    _lib.call("sb_relu", device_ptr(x), device_ptr(out), int(x.size), stream_ptr(stream))
    return out


def softmax(x, out=None, mask=None, prefix=-1, stream=None):
    """Row softmax; `mask` (uint8, same shape) or `prefix` (legal iff j < prefix) restricts it."""
    out = x if out is None else out
    rows, cols = _rows_cols(x)
    _lib.call("sb_row_softmax", device_ptr(x), device_ptr(out), rows, cols, device_ptr(mask), int(prefix),
              stream_ptr(stream))
    return out


def masked_softmax(size, x, out=None, stream=None):
    """layers.masked_softmax size (ml/layers.spi:408-414): legal iff column index < size."""
    return softmax(x, out=out, prefix=size, stream=stream)


def regret_matching(x, out=None, mask=None, prefix=-1, stream=None):
    out = x if out is None else out
    rows, cols = _rows_cols(x)
    _lib.call("sb_row_regret_matching", device_ptr(x), device_ptr(out), rows, cols, device_ptr(mask),
              int(prefix), stream_ptr(stream))
    return out


def masked_regret_matching(size, x, out=None, stream=None):
    """layers.masked_regret_matching size (ml/layers.spi:415-420)."""
    return regret_matching(x, out=out, prefix=size, stream=stream)


def argmax(x, out, stream=None):
    rows, cols = _rows_cols(x)
    _lib.call("sb_row_argmax", device_ptr(x), device_ptr(out), rows, cols, stream_ptr(stream))
    return out


def sample(probs, uniforms, out, stream=None):
    """One index per row drawn from the row's non-negative weights with the caller's uniform numbers
    in (0, 1] (one per row): the reference's discrete sampling head (ml/primitives.spi:782-800)."""
    rows, cols = _rows_cols(probs)
    _lib.call("sb_row_sample", device_ptr(probs), device_ptr(uniforms), device_ptr(out), rows, cols,
              stream_ptr(stream))
    return out


def sample_seeded(probs, out, seed, row_offset=0, position=0, stream=None):
    """The same with the uniform numbers drawn on the device as the reference does: row r uses output
    ``position`` of the Philox4x32-10 stream (seed, row_offset + r)."""
    rows, cols = _rows_cols(probs)
    _lib.call("sb_row_sample_seeded", device_ptr(probs), device_ptr(out), rows, cols, ctypes.c_ulonglong(int(seed)),
              ctypes.c_ulonglong(int(row_offset)), ctypes.c_ulonglong(int(position)), stream_ptr(stream))
    return out


def philox_uniform(out, seed, row_offset=0, position=0, stream=None):
    """Fills the fp32 device array ``out`` with the uniform numbers in (0, 1] a sampling head draws:
    element i = output ``position`` of the stream (seed, row_offset + i)."""
    _lib.call("sb_philox_uniform", device_ptr(out), ctypes.c_longlong(int(out.size)), ctypes.c_ulonglong(int(seed)),
              ctypes.c_ulonglong(int(row_offset)), ctypes.c_ulonglong(int(position)), stream_ptr(stream))
    return out


def binarize(modulo, x, out, stream=None):
    """Row hash: bit j = (x[r, j] > 0), modulo ``modulo`` (ml/primitives.spi:816-821); ``out`` is an int32
    device array [rows] holding the unsigned values."""
    rows, cols = _rows_cols(x)
    _lib.call("sb_row_binarize", device_ptr(x), device_ptr(out), rows, cols, ctypes.c_uint(int(modulo)),
              stream_ptr(stream))
    return out


def ln_l2(x, out=None, stream=None):
    out = x if out is None else out
    rows, cols = _rows_cols(x)
    _lib.call("sb_row_ln_l2", device_ptr(x), device_ptr(out), rows, cols, stream_ptr(stream))
    return out


def encode_states(fields, widths, dense, out, stream=None):
    """Compact game states -> the dense network input ``out`` [rows, sum(widths) + n_dense].

    ``fields``: uint8 device array [rows, len(widths)], value v < widths[j] sets feature v of the
    j-th one-hot group, any other value leaves the group zero (the bounded-int pickler of
    corebase/pickler.spi:20-37, run on the device as ml/models.spi:30-41 does); ``dense``: device
    array [rows, n_dense] in the dtype of ``out`` (or None), copied behind the one-hot groups.
    """
    rows = int(out.shape[0])
    widths = [int(w) for w in widths]
    n_dense = 0 if dense is None else int(dense.shape[1])
    if int(out.shape[1]) != sum(widths) + n_dense:
        raise ValueError("encode_states: out has %d features, the layout describes %d"
                         % (out.shape[1], sum(widths) + n_dense))
    if tuple(fields.shape) != (rows, len(widths)):
        raise ValueError("encode_states: fields must be [%d, %d], got %s" % (rows, len(widths), tuple(fields.shape)))
    if dense is not None and (int(dense.shape[0]) != rows or dense.dtype != out.dtype):
        raise ValueError("encode_states: dense must be [%d, n] in the dtype of out" % rows)
    w_c = (ctypes.c_int * max(1, len(widths)))(*widths)
    _lib.call("sb_encode_states", device_ptr(fields), len(widths), w_c, device_ptr(dense), n_dense,
              device_ptr(out), rows, _lib.DTYPE_CODES[out.dtype], stream_ptr(stream))
    return out


def convert(x, out, stream=None):
    """fp32 device array -> `out` (bf16 / f16 / tf32-rounded fp32 / fp32)."""
    _lib.call("sb_convert", device_ptr(x), device_ptr(out), int(x.size), _lib.DTYPE_CODES[out.dtype],
              stream_ptr(stream))
    return out


_FLOATS = {"f32": _lib.F32, "tf32": _lib.F32, "bf16": _lib.BF16, "f16": _lib.F16}
_INDICES = {"i32": _lib.I32, "i64": _lib.I64}


def _code(x, what, table=_FLOATS):
    tag = dtype_tag(x)
    try:
        return table[tag]
    except KeyError:
        raise TypeError("%s must hold %s, not %s" % (what, " / ".join(table), tag)) from None


def embedding(tokens, table, out, scale=1.0, stream=None):
    """``out[i, :] = scale * table[tokens[i], :]``.

    ``tokens``: int32 or int64, any shape; ``table`` [vocab, dim] and ``out`` [.., dim] (one row per token) in fp32, bf16
    or f16, each its own; rows may have a pitch.  A token outside [0, vocab) is no token and gives a row of zeros, as an
    out-of-range field does in ``encode_states``."""
    n = flat_size(tokens, "tokens")
    vocab, dim, ld_table = matrix_of(table, "table")
    rows, cols, ld_out = matrix_of(out, "out")
    if rows != n or cols != dim:
        raise ValueError("embedding: out is %dx%d for %d tokens and rows of %d" % (rows, cols, n, dim))
    _lib.call("sb_embedding", device_ptr(tokens), _code(tokens, "tokens", _INDICES), n, device_ptr(table), ld_table,
              _code(table, "table"), vocab, dim, scale, device_ptr(out), ld_out, _code(out, "out"), stream_ptr(stream))
    return keep_tf32(out, stream)


def embedding_grad(tokens, dout, dtable, scale=1.0, accumulate=False, workspace=None, stream=None):
    """Gradient of ``embedding``: ``dtable[v, :] = scale * sum of dout[i, :] over tokens[i] == v``, fp32 [vocab, dim]
    (``accumulate``: added to it).  Sums in the order of the positions, the same bits on every call.  ``workspace``: device
    memory of ``embedding_grad_workspace`` bytes; by default one is kept per device, stream and host thread."""
    n = flat_size(tokens, "tokens")
    rows, cols, ld_dout = matrix_of(dout, "dout")
    vocab, dim, ld_dtable = matrix_of(dtable, "dtable")
    if rows != n or cols != dim:
        raise ValueError("embedding_grad: dout is %dx%d for %d tokens and rows of %d" % (rows, cols, n, dim))
    if dtype_tag(dtable) != "f32":
        raise TypeError("dtable must hold f32, not %s" % dtype_tag(dtable))
    nbytes = embedding_grad_workspace(n, vocab, dim) if workspace is None else _nbytes(workspace)
    if workspace is None:
        workspace = stream_workspace(nbytes, stream)
    _lib.call("sb_embedding_grad", device_ptr(tokens), _code(tokens, "tokens", _INDICES), n, device_ptr(dout), ld_dout,
              _code(dout, "dout"), scale, device_ptr(dtable), ld_dtable, vocab, dim, int(bool(accumulate)),
              device_ptr(workspace), nbytes, stream_ptr(stream))
    return dtable


def embedding_grad_workspace(n, vocab, dim):
    """Bytes of device memory that ``embedding_grad`` needs for n tokens and a [vocab, dim] table."""
    nbytes = ctypes.c_size_t(0)
    _lib.call("sb_embedding_grad_workspace_bytes", n, vocab, dim, ctypes.byref(nbytes))
    return nbytes.value


def _nbytes(x):
    n = getattr(x, "nbytes", None)
    return int(n) if n is not None else int(x.numel()) * int(x.element_size())


def layer_norm(x, out=None, weight=None, bias=None, eps=1e-5, mean=None, rstd=None, stream=None):
    """``out = (x - mean) * rstd * weight + bias`` over the last dimension, in the storage type of ``x`` (fp32, bf16, f16;
    rows may have a pitch; ``out`` may be ``x``, the default).  ``weight`` and ``bias``: fp32 [cols] or None.  ``mean``,
    ``rstd``: fp32 [rows], filled where given; ``layer_norm_grad`` reads them."""
    out = x if out is None else out
    rows, cols, ldx = matrix_of(x, "x")
    out_rows, out_cols, ldy = matrix_of(out, "out")
    code = _code(x, "x")
    if out_rows != rows or out_cols != cols or _code(out, "out") != code:
        raise ValueError("layer_norm: out must be like x, %dx%d" % (rows, cols))
    _lib.call("sb_layer_norm", device_ptr(x), ldx, device_ptr(out), ldy, values_ptr(weight, cols, "weight"),
              values_ptr(bias, cols, "bias"), eps, values_ptr(mean, rows, "mean"), values_ptr(rstd, rows, "rstd"), rows, cols, code,
              stream_ptr(stream))
    return keep_tf32(out, stream)


def layer_norm_grad(dy, x, mean, rstd, dx=None, weight=None, dweight=None, dbias=None, accumulate=False, workspace=None,
                    stream=None):
    """Gradient of ``layer_norm``: ``dx`` (like ``x``), ``dweight`` and ``dbias`` (fp32 [cols]), each where given;
    ``accumulate`` adds to the old ``dweight`` and ``dbias``.  Sums in a fixed order, the same bits on every call.
    ``workspace``: device memory of ``layer_norm_grad_workspace`` bytes; by default one is kept per device, stream and thread."""
    rows, cols, ldx = matrix_of(x, "x")
    code = _code(x, "x")
    dy_rows, dy_cols, lddy = matrix_of(dy, "dy")
    if dy_rows != rows or dy_cols != cols or _code(dy, "dy") != code:
        raise ValueError("layer_norm_grad: dy must be like x, %dx%d" % (rows, cols))
    lddx = cols
    if dx is not None:
        dx_rows, dx_cols, lddx = matrix_of(dx, "dx")
        if dx_rows != rows or dx_cols != cols or _code(dx, "dx") != code:
            raise ValueError("layer_norm_grad: dx must be like x, %dx%d" % (rows, cols))
    nbytes = 0
    if workspace is not None:
        nbytes = _nbytes(workspace)
    elif dweight is not None or dbias is not None:
        nbytes = layer_norm_grad_workspace(rows, cols)
        workspace = stream_workspace(nbytes, stream)
    _lib.call("sb_layer_norm_grad", device_ptr(dy), lddy, device_ptr(x), ldx, values_ptr(mean, rows, "mean"),
              values_ptr(rstd, rows, "rstd"), values_ptr(weight, cols, "weight"), device_ptr(dx), lddx,
              values_ptr(dweight, cols, "dweight"), values_ptr(dbias, cols, "dbias"), int(bool(accumulate)), rows, cols, code,
              device_ptr(workspace), nbytes, stream_ptr(stream))
    return keep_tf32(dx, stream)


def layer_norm_grad_workspace(rows, cols):
    """Bytes of device memory that ``layer_norm_grad`` needs when it makes weight gradients."""
    nbytes = ctypes.c_size_t(0)
    _lib.call("sb_layer_norm_grad_workspace_bytes", rows, cols, ctypes.byref(nbytes))
    return nbytes.value
