"""Stand-alone row / elementwise operations (reference: ml/primitives.spi:701-780, ml/layers.spi:353-420), and the
operators around the dense layers of a net that reads tokens (embedding and layer normalisation in front of them, the log
probabilities of its answers behind them)."""
import ctypes

from . import _lib
from .device import (array_ptr, device_ptr, dtype_tag, flat_size, keep_tf32, matrix_of, nbytes_of, stream_ptr, stream_workspace,
                     typed_matrix, values_ptr)


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
    nbytes = embedding_grad_workspace(n, vocab, dim) if workspace is None else nbytes_of(workspace)
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
        nbytes = nbytes_of(workspace)
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


def _row_args(who, logits, tokens, mask):
    """What ``log_probs`` and its gradient share: (address, rows, cols, pitch, type), the mask, the tokens and their type."""
    rows, cols, ld, ptr, tag = typed_matrix(logits, "logits")
    code = _FLOATS.get(tag)
    if code is None:
        raise TypeError("logits must hold %s, not %s" % (" / ".join(_FLOATS), tag))
    if mask is not None:
        mask = array_ptr(mask, rows * cols, "u8", "mask", cols)
    index = _lib.I32
    if tokens is not None:
        tag = dtype_tag(tokens)
        index = _INDICES.get(tag)
        if index is None:
            raise TypeError("tokens must hold %s, not %s" % (" / ".join(_INDICES), tag))
        tokens = array_ptr(tokens, rows, tag, "tokens")
    return ptr, rows, cols, ld, code, mask, tokens, index


def _places(who, x, rows, n, tag, what):
    """Alternatives per row of a matrix that takes them; `n` is that of the other one, if there is one."""
    shape = tuple(x.shape)
    if len(shape) != 2 or shape[0] != rows or (n is not None and shape[1] != n):
        raise ValueError("%s: %s must be [%d, %s], got %s" % (who, what, rows, "n" if n is None else n, shape))
    return shape[1], array_ptr(x, rows * shape[1], tag, what)


def log_probs(logits, tokens=None, out=None, entropy=None, stats=None, top=None, top_tokens=None, mask=None, prefix=-1, scale=1.0,
              stream=None):
    """Log probabilities of the given tokens (or actions) under ``softmax(scale * logits)`` of each row, for a policy gradient
    or a token loss, with the rows' entropy and likeliest alternatives.

    ``logits`` [rows, cols] in fp32, bf16 or f16 (rows may have a pitch); ``tokens`` int32 or int64 [rows]; ``mask`` (uint8, same
    shape) or ``prefix`` (legal iff j < prefix) restricts the columns as in ``softmax``.  Filled where given: ``out`` fp32 [rows] (0 where
    the token is outside [0, cols), -inf where it is not legal), ``entropy`` fp32 [rows], ``stats`` fp32 [rows, 2] (the largest logit and the
    logarithm of the sum over it, for ``log_probs_grad``), ``top`` fp32 and ``top_tokens`` int32 [rows, n], n at most 64: the log
    probabilities and columns of the largest logits, equal ones in the order of their columns, -inf and -1 beyond the legal
    ones.  ``scale`` is one over the temperature.  Returns ``out``."""
    ptr, rows, cols, ld, code, mask, tokens, index = _row_args("log_probs", logits, tokens, mask)
    n = None
    if top is not None:
        n, top = _places("log_probs", top, rows, n, "f32", "top")
    if top_tokens is not None:
        n, top_tokens = _places("log_probs", top_tokens, rows, n, "i32", "top_tokens")
    if not n:
        n, top, top_tokens = 0, None, None
    _lib.call("sb_log_probs", ptr, ld, code, rows, cols, mask, prefix, scale, tokens, index, array_ptr(out, rows, "f32", "out"),
              array_ptr(entropy, rows, "f32", "entropy"), array_ptr(stats, 2 * rows, "f32", "stats", 2), n, top, top_tokens,
              stream_ptr(stream))
    return out


def log_probs_plan(rows, cols, top=0):
    """What ``log_probs`` takes a row with: threads, columns of each in registers (0: in one pass over memory), blocks that share a row."""
    plan = (ctypes.c_int * 3)()
    _lib.call("sb_log_probs_plan", int(rows), int(cols), int(top), plan)
    return dict(zip(("threads", "columns", "blocks"), list(plan)))


def log_probs_grad(logits, tokens, stats, dlogits, dout=None, dentropy=None, entropy=None, mask=None, prefix=-1, scale=1.0, stream=None):
    """Gradient of ``log_probs``: ``dlogits`` (like ``logits``, and may be them) from ``dout`` and ``dentropy``, the gradients of
    ``out`` and ``entropy`` (fp32 [rows], None: none), with the ``stats`` and, for ``dentropy``, the ``entropy`` that the forward call
    left.  Zero in columns that are not legal; a row without a token gets no ``dout``.  None flows through the alternatives."""
    ptr, rows, cols, ld, code, mask, tokens, index = _row_args("log_probs_grad", logits, tokens, mask)
    drows, dcols, ldd, dptr, dtag = typed_matrix(dlogits, "dlogits")
    if drows != rows or dcols != cols or _FLOATS.get(dtag) != code:
        raise ValueError("log_probs_grad: dlogits must be like logits, %dx%d" % (rows, cols))
    _lib.call("sb_log_probs_grad", ptr, ld, code, rows, cols, mask, prefix, scale, tokens, index, array_ptr(stats, 2 * rows, "f32", "stats", 2),
              array_ptr(dout, rows, "f32", "dout"), array_ptr(entropy, rows, "f32", "entropy"), array_ptr(dentropy, rows, "f32", "dentropy"),
              dptr, ldd, stream_ptr(stream))
    return keep_tf32(dlogits, stream)
