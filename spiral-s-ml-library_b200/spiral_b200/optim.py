"""AdamW over all parameter tensors of a net in one launch (the reference trains without gradients; ``PolicyMLP.sgd`` is
the plain step)."""
import ctypes

from . import _lib
from .device import DeviceArray, device_ptr, dtype_tag, flat_size, stream_ptr

STATE_BLOCK = 256                # elements that share a scale when the states are held in 8 bits
_GRADS = {"f32": _lib.F32, "tf32": _lib.F32, "bf16": _lib.BF16, "f16": _lib.F16}


def _one_type(arrays, what):
    tags = {dtype_tag(x) for x in arrays}
    if len(tags) > 1:
        raise TypeError("%s must share one storage type, got %s" % (what, ", ".join(sorted(map(str, tags)))))
    return tags.pop() if tags else "f32"


class AdamW:
    """``p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)`` over lists of device arrays.

    ``params``: fp32, updated in place.  ``grads``: fp32, bf16 or f16, one type.  ``copies``: where given (None per tensor
    allowed), compute copies that receive the new parameters rounded to their type.  ``state``: 'f32' keeps m and v in
    fp32; 'e4m3' keeps m and sqrt(v) as E4M3 codes with an fp32 scale per 256 elements (2.03 instead of 8 bytes per
    parameter), rounded with noise drawn from (element, seed).  The states (``exp_avg``, ``exp_avg_sq``, with 'e4m3' their
    ``exp_avg_scale``, ``exp_avg_sq_scale``: lists) are made and zeroed here unless they are given.  The arrays stay the
    caller's: an ``AdamW`` holds on to them and to their addresses for its lifetime."""

    def __init__(self, params, grads, exp_avg=None, exp_avg_sq=None, exp_avg_scale=None, exp_avg_sq_scale=None, copies=None,
                 state="f32"):
        if state not in ("f32", "e4m3"):
            raise ValueError("state must be 'f32' or 'e4m3'")
        self.params, self.grads = list(params), list(grads)
        self.copies = [None] * len(self.params) if copies is None else list(copies)
        self.state = state
        self.sizes = [flat_size(p, "a parameter tensor") for p in self.params]
        blocks = [-(-n // STATE_BLOCK) for n in self.sizes]
        coded = state == "e4m3"
        nothing = [None] * len(self.params)
        self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale = (
            nothing if x is None else list(x)
            for x in (exp_avg, exp_avg_sq, exp_avg_scale if coded else None, exp_avg_sq_scale if coded else None))
        if any(dtype_tag(p) != "f32" for p in self.params):
            raise TypeError("parameters must be fp32")
        grad_tag = _one_type(self.grads, "gradients")
        if grad_tag not in _GRADS:
            raise TypeError("gradients must hold f32, bf16 or f16, not %s" % grad_tag)
        copy_tag = _one_type([c for c in self.copies if c is not None], "copies")
        if copy_tag not in ("f32", "tf32", "bf16", "f16"):
            raise TypeError("copies must hold f32, tf32, bf16 or f16, not %s" % copy_tag)
        for name, arrays, sizes in (("gradients", self.grads, self.sizes), ("copies", self.copies, self.sizes),
                                    ("exp_avg", self.exp_avg, self.sizes), ("exp_avg_sq", self.exp_avg_sq, self.sizes),
                                    ("exp_avg_scale", self.exp_avg_scale, blocks),
                                    ("exp_avg_sq_scale", self.exp_avg_sq_scale, blocks)):
            if len(arrays) != len(self.params):
                raise ValueError("%d %s for %d parameter tensors" % (len(arrays), name, len(self.params)))
            for i, (x, n) in enumerate(zip(arrays, sizes)):
                if x is not None and flat_size(x, name) != n:
                    raise ValueError("%s %d has %d elements, %d are needed" % (name, i, flat_size(x, name), n))
        for name, arrays, tags in (("exp_avg", self.exp_avg, (state, "u8") if coded else ("f32",)),
                                   ("exp_avg_sq", self.exp_avg_sq, (state, "u8") if coded else ("f32",)),
                                   ("exp_avg_scale", self.exp_avg_scale, ("f32",)),
                                   ("exp_avg_sq_scale", self.exp_avg_sq_scale, ("f32",))):
            if any(x is not None and dtype_tag(x) not in tags for x in arrays):
                raise TypeError("%s must hold %s" % (name, " / ".join(tags)))
        self.exp_avg, self.exp_avg_sq = (self._made(x, self.sizes, state) for x in (self.exp_avg, self.exp_avg_sq))
        if coded:
            self.exp_avg_scale, self.exp_avg_sq_scale = (self._made(x, blocks, "f32")
                                                         for x in (self.exp_avg_scale, self.exp_avg_sq_scale))
        self.steps = self.calls = 0
        self._codes = (_lib.E4M3 if coded else _lib.F32, _GRADS[grad_tag], _lib.DTYPE_CODES[copy_tag])
        self._table = (_lib.AdamwTensor * max(1, len(self.params)))()
        for i, n in enumerate(self.sizes):
            self._table[i] = _lib.AdamwTensor(*[device_ptr(x[i]) for x in (
                self.params, self.grads, self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale,
                self.copies)], n)
        self._hyper = _lib.AdamwHyper()

    @staticmethod
    def _made(states, sizes, tag):
        return [DeviceArray.zeros((n,), tag) if x is None else x for x, n in zip(states, sizes)]

    def step(self, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, step=None, seed=None, grad_scale=1.0, stream=None):
        """One step over all tensors.  ``step`` counts from 1 (default: the calls so far and this one); ``seed`` is that of
        the 8-bit rounding (default: ``step``); gradients are multiplied by ``grad_scale`` first."""
        self.steps = self.steps + 1 if step is None else int(step)
        self.calls += 1
        h = self._hyper
        h.lr, h.eps, h.weight_decay, h.grad_scale = lr, eps, weight_decay, grad_scale
        h.beta1, h.beta2 = betas
        h.step = self.steps
        h.seed = (self.steps if seed is None else int(seed)) & 0xffffffff
        _lib.call("sb_adamw_step", len(self.params), self._table, *self._codes, ctypes.byref(h), stream_ptr(stream))
