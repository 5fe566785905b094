"""Dense policy network on the GPU: the caller of the GEMM path.

Reference: ml/models.spi:9-76 (run a layer graph per decision) and the model
graphs game/leduc/model_cem.spi:41-66, game/nl_hu_holdem/model_cem.spi:71-103
(input -> matmul -> relu ... -> masked head).  ``PolicyMLP`` owns the buffers the
reference keeps in its weight / workspace / adjoint arenas and drives
sb_mlp_forward / sb_mlp_backward / sb_sgd_update.
"""
import ctypes

import numpy as np

from . import _lib, primitives
from .device import DeviceArray, capturing, device_ptr, stream_ptr, values_ptr
from . import dtypes
from .matmul import ACTIVATIONS, gated, gated_grad, matmul, matmul_fp8, matmul_int4, quantize_fp8, quantize_int4
from .optim import AdamW

HEAD_FLAGS = {"masked_softmax": _lib.EPI_MASKED_SOFTMAX, "regret_matching": _lib.EPI_REGRET_MATCHING,
              "argmax": _lib.EPI_ARGMAX}


def param_offsets(sizes):
    """Element offsets [W0, b0, W1, b1, ..., total] of the flat parameter vector."""
    n = len(sizes) - 1
    arr = (ctypes.c_int * len(sizes))(*sizes)
    out = (ctypes.c_longlong * (2 * n + 1))()
    _lib.call("sb_mlp_param_offsets", n, arr, out)
    return list(out)


class PolicyMLP:
    """ReLU MLP with a masked row head; weights W_i stored [out, in] like layers.weight."""

    def __init__(self, sizes, batch, in_dtype="bf16", head=("masked_softmax",), with_bias=True,
                 training=False, grads=None):
        if in_dtype not in ("tf32", "bf16", "f16"):
            raise ValueError("in_dtype must be 'tf32', 'bf16' or 'f16'")
        self.sizes = [int(s) for s in sizes]
        self.n_layers = len(self.sizes) - 1
        self.batch = int(batch)
        self.in_dtype = in_dtype
        self.storage = in_dtype          # 'tf32' = fp32 storage holding TF32-rounded values
        self.head = tuple(head)
        self.head_flags = 0
        for h in self.head:
            self.head_flags |= HEAD_FLAGS[h]
        self.with_bias = bool(with_bias)
        self.offsets = param_offsets(self.sizes)
        self.n_params = self.offsets[-1]
        self._sizes_c = (ctypes.c_int * len(self.sizes))(*self.sizes)
        self.params = DeviceArray.zeros((self.n_params,), "f32")
        self.w_compute = DeviceArray.zeros((self.n_params,), self.storage)
        self.weight_changes = 0          # calls that changed the weights, for what is made from them
        self.activations = [DeviceArray((self.batch, self.sizes[i + 1]), self.storage)
                            for i in range(self.n_layers - 1)]
        self._acts_c = (ctypes.c_void_p * max(1, self.n_layers - 1))(*[a.ptr for a in self.activations])
        self.probs = DeviceArray((self.batch, self.sizes[-1]), "f32")
        self.actions = DeviceArray((self.batch,), "i32") if "argmax" in self.head else None
        self.training = bool(training)
        # ReLU sign bits of every hidden layer (uint32 [width / 32, batch], column-block-major): recorded by the
        # forward pass when training so that backward gates by bits instead of re-reading H.
        self.relu_bits = []
        self._bits_c = None
        if self.training and all(w % 32 == 0 for w in self.sizes[1:-1]) and self.n_layers > 1:
            self.relu_bits = [DeviceArray((self.sizes[i + 1] // 32, self.batch), "i32")
                              for i in range(self.n_layers - 1)]
            self._bits_c = (ctypes.c_void_p * (self.n_layers - 1))(*[b.ptr for b in self.relu_bits])
        self.grads = None
        self.scratch = None
        self.loss = None
        if self.training:
            self.grads = grads if grads is not None else DeviceArray.zeros((self.n_params,), "f32")
            nbytes = ctypes.c_size_t(0)
            _lib.call("sb_mlp_backward_scratch_bytes", self.n_layers, self._sizes_c, self.batch,
                      _lib.DTYPE_CODES[in_dtype], ctypes.byref(nbytes))
            self.scratch = DeviceArray((nbytes.value,), "u8")
            self.loss = DeviceArray.zeros((1,), "f32")

    # -- parameters ----------------------------------------------------------
    def load_weights(self, weights, biases=None):
        """Uploads per-layer [out, in] fp32 weights (and biases) into the flat buffers."""
        flat = np.zeros(self.n_params, np.float32)
        for i, w in enumerate(weights):
            w = np.asarray(w, np.float32)
            if w.shape != (self.sizes[i + 1], self.sizes[i]):
                raise ValueError("layer %d weight shape %s" % (i, w.shape))
            o = self.offsets[2 * i]
            flat[o:o + w.size] = w.ravel()
            if biases is not None:
                b = np.asarray(biases[i], np.float32)
                ob = self.offsets[2 * i + 1]
                flat[ob:ob + b.size] = b
        self.params.upload(flat)
        self.w_compute.upload(flat)       # the upload rounds to the storage type
        self.weight_changes += 1
        return self

    def get_weights(self):
        flat = self.params.numpy()
        ws, bs = [], []
        for i in range(self.n_layers):
            o, ob = self.offsets[2 * i], self.offsets[2 * i + 1]
            n = self.sizes[i + 1] * self.sizes[i]
            ws.append(flat[o:o + n].reshape(self.sizes[i + 1], self.sizes[i]).copy())
            bs.append(flat[ob:ob + self.sizes[i + 1]].copy())
        return ws, bs

    def save(self, path):
        """Checkpoint: the flat fp32 master parameter vector with the layer sizes (NumPy .npz)."""
        np.savez(path, params=self.params.numpy(), sizes=np.asarray(self.sizes, np.int64))

    def load(self, path):
        """Restores a checkpoint written by ``save`` (same architecture) into the master parameters
        and the compute copy."""
        with np.load(path) as ck:
            if [int(v) for v in ck["sizes"]] != self.sizes:
                raise ValueError("checkpoint is for layer sizes %s, the model has %s" % (list(ck["sizes"]), self.sizes))
            flat = np.asarray(ck["params"], np.float32)
        if flat.shape != (self.n_params,):
            raise ValueError("checkpoint holds %d parameters, the model %d" % (flat.size, self.n_params))
        self.params.upload(flat)
        self.w_compute.upload(flat)
        self.weight_changes += 1
        return self

    def split_flat(self, flat):
        """Views of a flat host vector as [(W_i, b_i), ...]."""
        out = []
        for i in range(self.n_layers):
            o, ob = self.offsets[2 * i], self.offsets[2 * i + 1]
            n = self.sizes[i + 1] * self.sizes[i]
            out.append((flat[o:o + n].reshape(self.sizes[i + 1], self.sizes[i]), flat[ob:ob + self.sizes[i + 1]]))
        return out

    # -- execution -----------------------------------------------------------
    def forward(self, x, mask=None, head_flags=None, stream=None, fused=None):
        """probs <- head(MLP(x)); returns the probs DeviceArray (and fills actions for argmax heads).
        A net built for training whose shape the fused kernel takes runs the whole pass as one launch that
        also writes the activations and sign words backward needs (``fused=False``: one GEMM per layer)."""
        flags = self.head_flags if head_flags is None else head_flags
        if fused is None:
            fused = self.training and self.batch > 0 and self._fused_ok()
        if fused:
            _lib.call("sb_mlp_forward_fused_train", self.n_layers, self._sizes_c, self.batch,
                      _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr,
                      self.params.ptr if self.with_bias else None, self._acts_c, self._bits_c, flags, device_ptr(mask),
                      self.probs.ptr, device_ptr(self.actions) if flags & _lib.EPI_ARGMAX else None, stream_ptr(stream))
            return self.probs
        _lib.call("sb_mlp_forward", self.n_layers, self._sizes_c, self.batch, _lib.DTYPE_CODES[self.in_dtype],
                  device_ptr(x), self.w_compute.ptr, self.params.ptr if self.with_bias else None, self._acts_c,
                  self._bits_c, flags, device_ptr(mask), self.probs.ptr, device_ptr(self.actions) if flags & _lib.EPI_ARGMAX else None,
                  stream_ptr(stream))
        return self.probs

    def _fused_ok(self):
        if self.in_dtype not in ("bf16", "f16"):
            return False
        return bool(_lib.load().sb_mlp_fused_supported(self.n_layers, self._sizes_c, _lib.DTYPE_CODES[self.in_dtype]))

    def forward_fused(self, x, mask=None, head_flags=None, stream=None):
        """Forward pass as one persistent kernel (narrow nets: 16-bit class, hidden widths multiples of
        64 up to 256, at most 32 outputs); hidden activations never reach global memory.  Raises
        SpiralError (SB_ERR_UNSUPPORTED) for shapes outside those limits."""
        flags = self.head_flags if head_flags is None else head_flags
        _lib.call("sb_mlp_forward_fused", self.n_layers, self._sizes_c, self.batch,
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr,
                  self.params.ptr if self.with_bias else None, flags, device_ptr(mask), self.probs.ptr,
                  device_ptr(self.actions) if flags & _lib.EPI_ARGMAX else None, stream_ptr(stream))
        return self.probs

    def forward_no_alloc(self, x, out, mask=None, actions=None, head_flags=None, stream=None):
        """Forward pass whose hidden activations use the library's built-in 32 MiB workspace.

        For callers that may not allocate device memory (no allocator of their own, a context where
        allocation is forbidden, inside a stream capture).  `out` (fp32 [batch, actions]) and
        `actions` (int32 [batch], for argmax heads) are caller buffers.  Raises SpiralError
        (SB_ERR_TOO_LARGE) when batch x hidden widths does not fit.  Calls share the one workspace and
        run one after the other on the GPU, whatever streams and threads they come from; only a graph
        that captured such a call must be kept from overlapping with others.
        """
        flags = self.head_flags if head_flags is None else head_flags
        _lib.call("sb_mlp_forward_static", self.n_layers, self._sizes_c, self.batch,
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr,
                  self.params.ptr if self.with_bias else None, flags, device_ptr(mask), device_ptr(out),
                  device_ptr(actions) if flags & _lib.EPI_ARGMAX else None, stream_ptr(stream))
        return out

    def backward(self, x, mask, target, global_batch=None, stream=None):
        """grads <- d(mean cross-entropy)/d(params) for this shard (after a masked-softmax forward)."""
        gb = self.batch if global_batch is None else int(global_batch)
        _lib.call("sb_mlp_backward", self.n_layers, self._sizes_c, self.batch, ctypes.c_float(1.0 / gb),
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr, self._acts_c, self._bits_c,
                  self.probs.ptr,
                  device_ptr(mask), device_ptr(target), device_ptr(self.grads), int(self.with_bias),
                  self.scratch.ptr, self.scratch.nbytes, self.loss.ptr, stream_ptr(stream))
        return self.grads

    def backward_logits(self, x, dlogits, stream=None):
        """grads <- the gradient whose part at the logits is ``dlogits`` (fp32 [batch, n_out]), after ``forward(x, head_flags=0)``,
        which leaves the logits in ``probs``: for losses of the caller's own, a policy gradient among them
        (``primitives.log_probs_grad``)."""
        _lib.call("sb_mlp_backward_logits", self.n_layers, self._sizes_c, self.batch, _lib.DTYPE_CODES[self.in_dtype], device_ptr(x),
                  self.w_compute.ptr, self._acts_c, self._bits_c, values_ptr(dlogits, self.batch * self.sizes[-1], "dlogits"),
                  device_ptr(self.grads), int(self.with_bias), self.scratch.ptr, self.scratch.nbytes, stream_ptr(stream))
        return self.grads

    def backward_dp(self, x, mask, target, grads_table, world_size, rank, global_batch=None, stream=None):
        """The backward pass of a data-parallel step: like ``backward``, but the weight-gradient GEMMs of
        the wide layers add their tiles straight into the gradient buffer of the rank that owns those rows
        (``grads_table``: HOST array of every rank's buffer, ``PeerUpdate.grads_table()``), over peer
        memory -- the reduce-scatter half of the gradient all-reduce done by the GEMM itself."""
        gb = self.batch * int(world_size) if global_batch is None else int(global_batch)
        _lib.call("sb_mlp_backward_dp", self.n_layers, self._sizes_c, self.batch, ctypes.c_float(1.0 / gb),
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr, self._acts_c, self._bits_c,
                  self.probs.ptr, device_ptr(mask), device_ptr(target), grads_table, int(world_size), int(rank),
                  int(self.with_bias), self.scratch.ptr, self.scratch.nbytes, self.loss.ptr, stream_ptr(stream))
        return self.grads

    def backward_layers(self, x, mask, target, first_layer, last_layer, global_batch=None, stream=None):
        """The backward pass of layers first_layer .. last_layer (descending); successive calls covering
        n_layers-1 .. 0 equal one ``backward``."""
        gb = self.batch if global_batch is None else int(global_batch)
        _lib.call("sb_mlp_backward_range", self.n_layers, self._sizes_c, self.batch, ctypes.c_float(1.0 / gb),
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr, self._acts_c, self._bits_c,
                  self.probs.ptr, device_ptr(mask), device_ptr(target), device_ptr(self.grads), int(self.with_bias),
                  self.scratch.ptr, self.scratch.nbytes, self.loss.ptr, int(first_layer), int(last_layer),
                  stream_ptr(stream))
        return self.grads

    def layer_dy(self, layer):
        """View of d(loss)/d(output of layer ``layer``) inside the backward scratch: [batch, width padded
        to 8] in the storage type.  Valid after ``backward_layers`` has processed ``layer`` and until it
        processes ``layer - 2`` (the two dY buffers alternate)."""
        off = ctypes.c_size_t(0)
        _lib.call("sb_mlp_backward_dy_offset", self.n_layers, self._sizes_c, self.batch,
                  _lib.DTYPE_CODES[self.in_dtype], int(layer), ctypes.byref(off))
        width = (self.sizes[layer + 1] + 7) // 8 * 8
        return self.scratch.view((self.batch, width), self.storage, off.value)

    def layer_segment(self, layer):
        """[begin, end) of layer `layer`'s weights and bias inside the flat parameter / gradient vectors."""
        end = self.offsets[2 * layer + 2] if layer + 1 < self.n_layers else self.n_params
        return self.offsets[2 * layer], end

    def sgd(self, lr, stream=None):
        self.weight_changes += 1
        _lib.call("sb_sgd_update", self.params.ptr, device_ptr(self.grads), self.w_compute.ptr,
                  ctypes.c_longlong(self.n_params), ctypes.c_float(lr), _lib.DTYPE_CODES[self.storage],
                  stream_ptr(stream))

    def train_step(self, x, mask, target, lr, stream=None):
        """Forward + backward + SGD on one GPU (no gradient exchange)."""
        self.weight_changes += 1
        _lib.call("sb_mlp_train_step", self.n_layers, self._sizes_c, self.batch, _lib.DTYPE_CODES[self.in_dtype],
                  device_ptr(x), self.params.ptr, self.w_compute.ptr, self._acts_c, self._bits_c, device_ptr(mask),
                  device_ptr(target), self.probs.ptr, device_ptr(self.grads), int(self.with_bias),
                  ctypes.c_float(lr), self.scratch.ptr, self.scratch.nbytes, self.loss.ptr, stream_ptr(stream))

    def flops_per_sample(self, training=False):
        f = sum(2 * self.sizes[i] * self.sizes[i + 1] for i in range(self.n_layers))
        if training:
            f = 3 * f - 2 * self.sizes[0] * self.sizes[1]     # no dgrad into the input
        return f


def to_storage(x, in_dtype):
    """Host fp32 array -> DeviceArray in the storage type of an arithmetic class."""
    return DeviceArray.from_numpy(np.asarray(x, np.float32), in_dtype)


class EnsemblePolicyMLP:
    """An ensemble of ``members`` policy nets of one architecture evaluated on ONE input batch in a
    single launch of the fused kernel (the reference builds such nets with ``layers.matmul_ensemble``,
    ml/layers.spi:468-471, and runs the graph once per member, ml/models.spi:47-49).

    16-bit arithmetic classes and the fused kernel's width limits only (input <= 512, hidden layers
    multiples of 64 up to 256, at most 64 outputs -- or 256 under a prefix mask of at most 64 columns).
    Outputs: ``probs`` fp32 [members, batch, n_out] and, with an argmax head, ``actions`` int32
    [members, batch].

    ``hidden_norm``: ln_l2 before every ReLU, as in the reference's nets (ml/layers.spi:594-603; no bias
    then).  ``decide`` (below) is the reference's per-decision call ml/models.spi:9-76.
    """

    def __init__(self, sizes, batch, members, in_dtype="f16", head=("masked_softmax",), with_bias=True,
                 hidden_norm=False):
        if in_dtype not in ("bf16", "f16"):
            raise ValueError("the fused ensemble forward runs in 'bf16' or 'f16'")
        self.sizes = [int(s) for s in sizes]
        self.n_layers = len(self.sizes) - 1
        self.batch, self.members = int(batch), int(members)
        self.in_dtype = self.storage = in_dtype
        self.head = tuple(head)
        self.head_flags = 0
        for h in self.head:
            self.head_flags |= HEAD_FLAGS[h]
        self.hidden_norm = bool(hidden_norm)
        self.with_bias = bool(with_bias) and not self.hidden_norm
        self.offsets = param_offsets(self.sizes)
        self.n_params = self.offsets[-1]
        self._sizes_c = (ctypes.c_int * len(self.sizes))(*self.sizes)
        self._decide = None
        self.params = DeviceArray.zeros((self.members, self.n_params), "f32")
        self.w_compute = DeviceArray.zeros((self.members, self.n_params), self.storage)
        self.probs = DeviceArray((self.members, self.batch, self.sizes[-1]), "f32")
        self.actions = DeviceArray((self.members, self.batch), "i32") if "argmax" in self.head else None

    def load_weights(self, member_weights, member_biases=None):
        """``member_weights[e][i]`` = layer i's [out, in] fp32 weights of member e (biases alike)."""
        if len(member_weights) != self.members:
            raise ValueError("%d weight sets for %d members" % (len(member_weights), self.members))
        flat = np.zeros((self.members, self.n_params), np.float32)
        for e, weights in enumerate(member_weights):
            for i, w in enumerate(weights):
                w = np.asarray(w, np.float32)
                if w.shape != (self.sizes[i + 1], self.sizes[i]):
                    raise ValueError("member %d layer %d weight shape %s" % (e, i, w.shape))
                o = self.offsets[2 * i]
                flat[e, o:o + w.size] = w.ravel()
                if member_biases is not None:
                    b = np.asarray(member_biases[e][i], np.float32)
                    ob = self.offsets[2 * i + 1]
                    flat[e, ob:ob + b.size] = b
        self.params.upload(flat)
        self.w_compute.upload(flat)       # the upload rounds to the storage type
        return self

    def forward(self, x, mask=None, stream=None):
        """All members on the batch ``x`` [batch, features] (storage type); returns ``probs``."""
        _lib.call("sb_mlp_forward_fused_ensemble", self.n_layers, self._sizes_c, self.batch, self.members,
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr,
                  self.params.ptr if self.with_bias else None, self.head_flags, device_ptr(mask), self.probs.ptr,
                  self.actions.ptr if self.actions is not None else None, stream_ptr(stream))
        return self.probs

    def forward_head(self, x, head=("masked_softmax",), prefix=-1, mask=None, seed=0, row_offset=0, position=0,
                     stream=None):
        """All members with the head given in full: ``head`` names from ``matmul.HEAD_FLAGS`` (softmax,
        regret matching, argmax, sample), legal columns ``j < prefix`` (or ``mask``), sampling from the
        Philox stream (seed, row_offset + row), member e using output ``position + e``.  Fills ``probs``,
        ``actions`` (argmax) and ``indices`` (sample)."""
        from .matmul import head_spec
        if "sample" in head and getattr(self, "indices", None) is None:
            self.indices = DeviceArray((self.members, self.batch), "i32")
        if "argmax" in head and self.actions is None:
            self.actions = DeviceArray((self.members, self.batch), "i32")
        spec = head_spec(tuple(head), prefix=prefix, mask=mask, argmax_out=self.actions if "argmax" in head else None,
                         sample_out=self.indices if "sample" in head else None, seed=seed, row_offset=row_offset,
                         position=position)
        _lib.call("sb_mlp_forward_fused_head", self.n_layers, self._sizes_c, self.batch, self.members,
                  _lib.DTYPE_CODES[self.in_dtype], device_ptr(x), self.w_compute.ptr,
                  self.params.ptr if self.with_bias else None, int(self.hidden_norm), ctypes.byref(spec),
                  self.probs.ptr, stream_ptr(stream))
        return self.probs

    def decide(self, seed, fields=None, widths=None, dense=None, x=None, head=("masked_softmax",), prefix=-1,
               mask=None, row_offset=0, stream=None):
        """One decision per game state: the reference's ``models.run`` (ml/models.spi:9-76).

        The states come either as compact records (``fields`` uint8 [batch, len(widths)] and optional
        ``dense`` values, serialised into the network input on the device) or as a ready input ``x``.
        Every member samples an action per state from its head, a member is drawn per state, and the
        result is a dict of device arrays: ``action`` int32 [batch], ``ensemble_id`` int32 [batch],
        ``sampling_prob_selected`` fp32 [batch], ``sampling_prob_ensemble`` fp32 [batch, members],
        plus the reference's tensors ``output_probs`` [members, batch, n_out] and ``output_indices``
        [members, batch].  Two kernel launches (one when ``x`` is given).  Buffers are created on the
        first call and reused."""
        if self._decide is None:
            b, e = self.batch, self.members
            self._decide = dict(
                x=DeviceArray((b, self.sizes[0]), self.storage), output_indices=DeviceArray((e, b), "i32"),
                ensemble_id=DeviceArray((b,), "i32"), action=DeviceArray((b,), "i32"),
                sampling_prob_selected=DeviceArray((b,), "f32"), sampling_prob_ensemble=DeviceArray((b, e), "f32"),
                tile_counters=DeviceArray.zeros(((b + 127) // 128,), "i32"))
        d = self._decide
        flags = 0
        for name in head:
            flags |= HEAD_FLAGS[name]
        a = _lib.DecideArgs()
        a.n_layers, a.sizes, a.members = self.n_layers, self._sizes_c, self.members
        a.in_dtype = _lib.DTYPE_CODES[self.in_dtype]
        a.w_compute, a.params = self.w_compute.ptr, (self.params.ptr if self.with_bias else None)
        a.hidden_norm, a.rows = int(self.hidden_norm), self.batch
        if fields is not None:
            widths = [int(w) for w in widths]
            self._widths_c = (ctypes.c_int * len(widths))(*widths)
            a.fields, a.n_fields, a.widths = device_ptr(fields), len(widths), self._widths_c
            a.dense, a.n_dense = device_ptr(dense), (0 if dense is None else int(dense.shape[1]))
            a.x = d["x"].ptr
        else:
            a.fields, a.n_fields, a.dense, a.n_dense = None, 0, None, 0
            a.x = device_ptr(x)
        a.head_flags, a.prefix, a.mask = flags, int(prefix), device_ptr(mask)
        a.seed, a.row_offset = int(seed), int(row_offset)
        a.output_probs, a.output_indices = self.probs.ptr, d["output_indices"].ptr
        a.ensemble_id, a.action = d["ensemble_id"].ptr, d["action"].ptr
        a.sampling_prob_selected, a.sampling_prob_ensemble = d["sampling_prob_selected"].ptr, d["sampling_prob_ensemble"].ptr
        a.tile_counters = d["tile_counters"].ptr
        _lib.call("sb_policy_decide", ctypes.byref(a), stream_ptr(stream))
        out = {k: d[k] for k in ("action", "ensemble_id", "sampling_prob_selected", "sampling_prob_ensemble",
                                 "output_indices")}
        out["output_probs"] = self.probs
        return out


class TokenPolicy:
    """A policy net whose states are sequences of ``n_tokens`` small integers (cards, actions, history; anything outside the
    vocabulary means "none"): embedding -> layer normalisation over the whole state -> a ``PolicyMLP`` with a masked-softmax
    head.  ``train_step`` is one AdamW step on the mean cross-entropy; ``forward_8bit`` answers with the dense layers in
    8-bit floating point: ``quantize`` first; ``forward_4bit`` has their weights in 4 bits, for few states: ``quantize_4bit`` first.
    After a step, an upload or a checkpoint the next answer quantises them anew; a caller who writes ``mlp.params`` in another
    way, as a replayed graph of a step does, calls ``quantize`` or ``quantize_4bit`` again.  A graph of an answer quantises in every
    replay if the weights had changed when it was captured, else never: then its caller quantises.

    ``evaluate`` gives the log probabilities of actions that were taken, the entropy and the likeliest actions, and
    ``policy_gradients`` the gradient of a loss of these two: the parts of a policy-gradient step.

    ``gated``: the columns, a multiple of 8, of a gated layer (``activation``) between the normalisation and the MLP, none by default.  Its
    products run on the tensor cores where ``n_tokens * dim`` is a multiple of 8, else on the CUDA cores at about 1 % of their rate.

    Buffers: ``table`` fp32 [vocab, dim], ``norm_weight`` and ``norm_bias`` fp32 [n_tokens * dim], ``gated_weight`` fp32 [2 * gated,
    n_tokens * dim], ``mlp.params``; all are stepped by one ``AdamW`` (``optimizer``, states in fp32 or 'e4m3')."""

    def __init__(self, vocab, n_tokens, dim, hidden, n_actions, batch, in_dtype="bf16", training=False, state="f32", gated=None,
                 activation="silu"):
        if in_dtype not in ("bf16", "f16"):
            raise ValueError("in_dtype must be 'bf16' or 'f16'")
        self.vocab, self.n_tokens, self.dim, self.batch = int(vocab), int(n_tokens), int(dim), int(batch)
        self.width = self.n_tokens * self.dim
        self.in_dtype = in_dtype
        self.scale = self.dim ** -0.5
        self.gated = None if gated is None else int(gated)
        self.activation = activation
        if self.gated is not None and (self.gated < 8 or self.gated % 8 or activation not in ACTIVATIONS):
            raise ValueError("gated must be a multiple of 8 columns (the MLP's rows are on 16 bytes) and its activation one of %s"
                             % ", ".join(sorted(ACTIVATIONS)))
        features = self.width if self.gated is None else self.gated
        self.mlp = PolicyMLP([features] + list(hidden) + [n_actions], batch, in_dtype=in_dtype, training=training)
        self.table = DeviceArray.zeros((self.vocab, self.dim), "f32")
        self.norm_weight = DeviceArray.from_numpy(np.ones(self.width, np.float32))
        self.norm_bias = DeviceArray.zeros((self.width,), "f32")
        self.embedded = DeviceArray((self.batch, self.width), in_dtype)
        self.x = DeviceArray((self.batch, self.width), in_dtype)
        self.mean, self.rstd = DeviceArray((self.batch,), "f32"), DeviceArray((self.batch,), "f32")
        self.features = self.x                    # what the MLP reads
        if self.gated is not None:
            self.gated_weight = DeviceArray.zeros((2 * self.gated, self.width), "f32")
            self.gated_compute = DeviceArray.zeros((2 * self.gated, self.width), in_dtype)
            self.gated_saved = DeviceArray((self.batch, 2 * self.gated), in_dtype) if training else None
            self.features = DeviceArray((self.batch, self.gated), in_dtype)
        self.optimizer = None
        self._codes = self._codes_of = self._codes4 = self._codes4_of = self._evaluated = None
        # Per group, and per number of alternatives: what one call left may be in a caller's graph when the next wants another.
        self._codes4_held, self._alternatives = {}, {}
        self._logits_ready = False                # mlp.probs holds what evaluate() left
        if training:
            self.dx = DeviceArray((self.batch, self.width), in_dtype)
            self.dembedded = DeviceArray((self.batch, self.width), in_dtype)
            self.dtable = DeviceArray((self.vocab, self.dim), "f32")
            self.dnorm_weight, self.dnorm_bias = DeviceArray((self.width,), "f32"), DeviceArray((self.width,), "f32")
            params, grads = [self.mlp.params, self.table, self.norm_weight, self.norm_bias], [self.mlp.grads, self.dtable, self.dnorm_weight, self.dnorm_bias]
            copies = [self.mlp.w_compute.view((self.mlp.n_params,)), None, None, None]
            if self.gated is not None:
                self.dfeatures = DeviceArray((self.batch, self.gated), in_dtype)
                self.dgated_weight = DeviceArray((2 * self.gated, self.width), "f32")
                params, grads, copies = params + [self.gated_weight], grads + [self.dgated_weight], copies + [self.gated_compute]
            self.optimizer = AdamW(params, grads, copies=copies, state=state)

    def load_weights(self, table, weights, biases=None, norm_weight=None, norm_bias=None, gated=None):
        """Uploads fp32 host weights: the table, the layers' [out, in] matrices (and biases), the normalisation's vectors, the
        gated layer's matrix."""
        self.table.upload(np.asarray(table, np.float32))
        self.mlp.load_weights(weights, biases)
        if norm_weight is not None:
            self.norm_weight.upload(np.asarray(norm_weight, np.float32))
        if norm_bias is not None:
            self.norm_bias.upload(np.asarray(norm_bias, np.float32))
        if gated is not None:
            if self.gated is None:
                raise ValueError("the net has no gated layer")
            self.gated_weight.upload(np.asarray(gated, np.float32))
            self.gated_compute.upload(np.asarray(gated, np.float32))
        return self

    def _input(self, tokens, stream):
        self._logits_ready = False
        by_token = (self.batch * self.n_tokens, self.dim)
        primitives.embedding(tokens, self.table, self.embedded.view(by_token), scale=self.scale, stream=stream)
        primitives.layer_norm(self.embedded, self.x, self.norm_weight, self.norm_bias, mean=self.mean, rstd=self.rstd, stream=stream)
        if self.gated is not None:
            gated(self.x, self.gated_compute, self.features, activation=self.activation, saved=self.gated_saved, stream=stream)

    def forward(self, tokens, mask=None, stream=None):
        """Action probabilities fp32 [batch, n_actions] for ``tokens`` (int32 or int64, [batch, n_tokens])."""
        self._input(tokens, stream)
        return self.mlp.forward(self.features, mask, stream=stream)

    def evaluate(self, tokens, actions, mask=None, top=0, scale=1.0, stream=None):
        """Log probabilities of ``actions`` (int32 or int64 [batch]) under the policy at the temperature 1 / ``scale``: a dict of ``log_probs`` and
        ``entropy`` fp32 [batch] and, where ``top`` > 0, ``top_log_probs`` fp32 and ``top_actions`` int32 [batch, top], the likeliest.  The
        logits stay in ``mlp.probs`` for ``policy_gradients``, and what is returned until the next call."""
        if self._evaluated is None:
            self._evaluated = {"log_probs": DeviceArray((self.batch,), "f32"), "entropy": DeviceArray((self.batch,), "f32"),
                               "stats": DeviceArray((self.batch, 2), "f32")}
        held, best, places = self._evaluated, None, None
        if top:
            if top not in self._alternatives:
                self._alternatives[top] = DeviceArray((self.batch, top), "f32"), DeviceArray((self.batch, top), "i32")
            best, places = self._alternatives[top]
        self._input(tokens, stream)
        logits = self.mlp.forward(self.features, head_flags=0, stream=stream)
        primitives.log_probs(logits, actions, held["log_probs"], entropy=held["entropy"], stats=held["stats"], top=best, top_tokens=places,
                             mask=mask, scale=scale, stream=stream)
        self._logits_ready = True
        got = {"log_probs": held["log_probs"], "entropy": held["entropy"]}
        return {**got, "top_log_probs": best, "top_actions": places} if top else got

    def policy_gradients(self, tokens, actions, dlog_probs, dentropy=None, mask=None, scale=1.0, stream=None):
        """Gradient of a loss whose derivatives by the log probabilities and the entropies of ``evaluate`` are ``dlog_probs`` and ``dentropy``
        (fp32 [batch]; a PPO or REINFORCE step's advantages times its ratios, over the batch): fills the gradients that ``optimizer``
        steps by.  Called after ``evaluate`` of the same states, actions, mask and scale, once: the gradient takes the logits' place."""
        if not self.mlp.training:
            raise ValueError("the net was not built for training")
        if not self._logits_ready:
            raise ValueError("evaluate() the states first: the logits are not, or no longer, those of this batch")
        held, self._logits_ready = self._evaluated, False
        primitives.log_probs_grad(self.mlp.probs, actions, held["stats"], self.mlp.probs, dout=dlog_probs, dentropy=dentropy,
                                  entropy=held["entropy"], mask=mask, scale=scale, stream=stream)
        self.mlp.backward_logits(self.features, self.mlp.probs, stream=stream)
        self._input_gradients(tokens, stream)

    def gradients(self, tokens, mask, target, stream=None):
        """Forward and backward pass: fills ``mlp.grads``, ``dtable``, ``dnorm_weight`` and ``dnorm_bias`` with the gradient of
        the mean cross-entropy and adds that to ``mlp.loss``."""
        self.forward(tokens, mask, stream=stream)
        self.mlp.backward(self.features, mask, target, stream=stream)
        self._input_gradients(tokens, stream)

    def _input_gradients(self, tokens, stream):
        # Into the input: what the first layer left behind times its weights (rows padded alike to multiples of 8).
        dy = self.mlp.layer_dy(0)
        w = self.mlp.w_compute.view((dy.shape[1], self.mlp.sizes[0]), self.in_dtype, self.mlp.offsets[0] * 2)
        matmul(False, False, 1.0, dy, w, 0.0, self.dx if self.gated is None else self.dfeatures, stream=stream)
        if self.gated is not None:
            gated_grad(self.dfeatures, self.x, self.gated_compute, self.gated_saved, dx=self.dx, dw=self.dgated_weight, activation=self.activation,
                       stream=stream)
        primitives.layer_norm_grad(self.dx, self.embedded, self.mean, self.rstd, self.dembedded, self.norm_weight,
                                   self.dnorm_weight, self.dnorm_bias, stream=stream)
        primitives.embedding_grad(tokens, self.dembedded.view((self.batch * self.n_tokens, self.dim)), self.dtable,
                                  scale=self.scale, stream=stream)

    def train_step(self, tokens, mask, target, lr, weight_decay=0.01, stream=None):
        """One AdamW step on this batch."""
        self.gradients(tokens, mask, target, stream=stream)
        self.optimizer.step(lr, weight_decay=weight_decay, stream=stream)

    def quantize(self, stream=None):
        """E4M3 codes of the dense layers' weights, a scale per block of 128 x 128, for ``forward_8bit``."""
        sizes = self.mlp.sizes
        if self._codes is None:
            self._codes = [(DeviceArray((o, i), "e4m3"), DeviceArray((-(-o // 128), -(-i // 128)), "f32"),
                            DeviceArray((self.batch, i), "e4m3"), DeviceArray((-(-i // 128), self.batch), "f32"))
                           for i, o in zip(sizes, sizes[1:])]
        for layer, (codes, scales, _, _) in enumerate(self._codes):
            w = self.mlp.params.view((sizes[layer + 1], sizes[layer]), "f32", self.mlp.offsets[2 * layer] * 4)
            quantize_fp8(w, codes, scales, block_rows=128, stream=stream)
        self._codes_of = self._weights_now(stream)
        return self

    def _weight_changes(self):
        return self.mlp.weight_changes, self.optimizer.calls if self.optimizer else 0

    def _weights_now(self, stream):
        """The weights whose codes a call on ``stream`` has just made; none while it is captured, as nothing has been made yet."""
        return None if capturing(stream) else self._weight_changes()

    def forward_8bit(self, tokens, mask=None, stream=None):
        """``forward`` with the dense layers in 8 bits: activations quantised per row and 128 columns, products of codes (on the
        tensor cores where a layer's input width is a multiple of 16)."""
        if self._codes is None:
            raise ValueError("quantize() the weights first")
        if self._codes_of != self._weight_changes():
            self.quantize(stream=stream)
        self._input(tokens, stream)
        x = self.features
        for layer, (codes, scales, x_codes, x_scales) in enumerate(self._codes):
            last = layer == self.mlp.n_layers - 1
            out = self.mlp.probs if last else self.mlp.activations[layer]
            bias = self.mlp.params.view((self.mlp.sizes[layer + 1],), "f32", self.mlp.offsets[2 * layer + 1] * 4)
            quantize_fp8(x, x_codes, x_scales, stream=stream)
            matmul_fp8(x_codes, x_scales, codes, scales, out, epilogue=("bias",) if last else ("bias", "relu"), bias=bias,
                       stream=stream)
            x = out
        return primitives.softmax(self.mlp.probs, mask=mask, stream=stream)

    def quantize_4bit(self, group=128, stream=None):
        """4-bit codes of the dense layers' weights, a scale per ``group`` columns of a row, for ``forward_4bit``."""
        sizes = self.mlp.sizes
        if group not in self._codes4_held:
            self._codes4_held[group] = [(DeviceArray((o, (i + 1) // 2), "u8"), DeviceArray((-(-i // group), o), self.in_dtype)) for i, o in zip(sizes, sizes[1:])]
        self._codes4 = group, self._codes4_held[group]
        for layer, (codes, scales) in enumerate(self._codes4[1]):
            w = self.mlp.params.view((sizes[layer + 1], sizes[layer]), "f32", self.mlp.offsets[2 * layer] * 4)
            quantize_int4(w, codes, scales, group=group, stream=stream)
        self._codes4_of = self._weights_now(stream)
        return self

    def forward_4bit(self, tokens, mask=None, stream=None):
        """``forward`` with the MLP's weights in 4 bits: for few states, whose answer waits for the weights."""
        if self._codes4 is None:
            raise ValueError("quantize_4bit() the weights first")
        group, layers = self._codes4
        if self._codes4_of != self._weight_changes():
            self.quantize_4bit(group, stream=stream)
        self._input(tokens, stream)
        x = self.features
        for layer, (codes, scales) in enumerate(layers):
            last = layer == self.mlp.n_layers - 1
            out = self.mlp.probs if last else self.mlp.activations[layer]
            bias = self.mlp.params.view((self.mlp.sizes[layer + 1],), "f32", self.mlp.offsets[2 * layer + 1] * 4)
            matmul_int4(x, codes, scales, out, group=group, epilogue=("bias",) if last else ("bias", "relu"), bias=bias, stream=stream)
            x = out
        return primitives.softmax(self.mlp.probs, mask=mask, stream=stream)
