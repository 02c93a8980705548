"""AdamW steps over many tensors on the GPU at once, with states in 32 or 8 bits: the update of a student that
:func:`distill_gradients`, :func:`logprob_gradients` and :func:`lookup_gradients` give gradients for."""
from __future__ import annotations

import ctypes as C
from operator import attrgetter

import numpy as np

from .class_scores import _TYPE, _bind, _on, _state, _stream

BLOCK = 256   # values of an 8-bit state that share a scale
_SHAPE, _DTYPE, _DEVICE = attrgetter("shape"), attrgetter("dtype"), attrgetter("device")


class _Tensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("exp_avg_scale", C.c_void_p), ("exp_avg_sq_scale", C.c_void_p), ("copy", C.c_void_p), ("n", C.c_uint64),
                ("param_type", C.c_int32), ("grad_type", C.c_int32), ("copy_type", C.c_int32), ("number", C.c_uint32)]


class _Settings(C.Structure):
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
                ("weight_decay", C.c_double), ("step", C.c_int64), ("step_device", C.c_void_p), ("lr_device", C.c_void_p),
                ("grad_scale", C.c_void_p), ("skip", C.c_void_p), ("seed", C.c_uint32), ("state", C.c_int32)]


class AdamW:
    """Weights ``params`` (torch tensors f32, f16 or bf16 on one GPU, contiguous) with the states that AdamW keeps of
    them; :meth:`step` takes their gradients and updates weights and states in place (``cbh_adamw_step``: the formulas are
    there).  One rate and one weight decay for all of them: what takes others is a handle of its own.

    ``state``: ``"f32"`` (``exp_avg`` and ``exp_avg_sq``, f32 of the weights' shapes) or ``"f8"`` (float8_e4m3fn codes
    of the first moment and of the square root of the second, with the scales ``exp_avg_scale`` and
    ``exp_avg_sq_scale`` f32 of every 256 values; rounded by random bits of ``seed`` and the step).  States of an
    earlier run are given by those names, as lists of tensors, and kept, not copied; with ``steps``, the number of steps
    that they are after.  ``copies``: a list of tensors (or None) that get the new weights rounded to their type: 16-bit
    weights beside f32 ones.  The handle's tuples of weights, states and copies stay; the memory of their tensors may be written
    and may move between steps.  A step with a weight that changed its shape or type is refused.

    ``steps`` is a number, or an i64 tensor of one value on the GPU: then every step adds 1 to it on the stream (not
    where ``skip`` holds a step back), and a step may be captured into a graph.  With a number a capture is refused: the
    graph's replays would all be the same step.

    A step counts as an in-place change of what it writes (the tensors' version counters): the backward pass of a graph that
    was recorded with the weights as they were raises, as after torch's own updates.
    """

    def __init__(self, params, *, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, state="f32", exp_avg=None,
                 exp_avg_sq=None, exp_avg_scale=None, exp_avg_sq_scale=None, copies=None, steps=0, seed=0):
        torch = _state.get("torch") or _bind()
        self._params = tuple(params)
        if state not in ("f32", "f8"):
            raise ValueError("state must be 'f32' or 'f8'")
        for p in self.params:
            if not isinstance(p, torch.Tensor):
                raise ValueError("params must be torch tensors")
        self._shapes, self._types = [p.shape for p in self.params], [p.dtype for p in self.params]
        self._check_weights()
        self.lr, self.beta1, self.beta2, self.eps, self.weight_decay = lr, beta1, beta2, eps, weight_decay
        self.state, self.steps, self.seed = state, steps, int(seed) & 0xFFFFFFFF
        small = self._small = state == "f8"
        if not small and (exp_avg_scale is not None or exp_avg_sq_scale is not None):
            raise ValueError("states in f32 have no scales")
        kind = torch.float8_e4m3fn if small else torch.float32
        blocks = [((p.numel() + BLOCK - 1) // BLOCK,) for p in self.params]
        # what every list of states holds: types and shapes
        self._kinds = {"exp_avg": (kind, self._shapes), "exp_avg_sq": (kind, self._shapes)}
        if small:
            self._kinds.update(exp_avg_scale=(torch.float32, blocks), exp_avg_sq_scale=(torch.float32, blocks))
        self._states = {}
        given = dict(exp_avg=exp_avg, exp_avg_sq=exp_avg_sq, exp_avg_scale=exp_avg_scale, exp_avg_sq_scale=exp_avg_sq_scale)
        for name, x in given.items():
            if name in self._kinds and x is None:
                kind, shapes = self._kinds[name]
                x = [torch.zeros(s, dtype=torch.float32, device=p.device).to(kind) for s, p in zip(shapes, self.params)]
            self._states[name] = None if x is None else tuple(x)
        self._copies = (None,) * len(self.params) if copies is None else tuple(copies)
        if isinstance(steps, torch.Tensor):
            if steps.dtype != torch.int64 or steps.numel() != 1 or (self.params and steps.device != self.params[0].device):
                raise ValueError("steps must be a number, or an int64 tensor of one value beside the weights")
        elif steps < 0:
            raise ValueError("steps must not be negative")
        # what of the library's records of the tensors does not change from step to step
        self._records = np.zeros(len(self.params), np.dtype(_Tensor))
        self._records["param_type"] = [_TYPE[t] for t in self._types]
        self._records["number"] = range(len(self.params))
        self._sizes = np.array([p.numel() for p in self.params], np.uint64)
        self._grad_types = None
        self._look(torch)

    def _check_weights(self):
        for p, shape, dtype in zip(self.params, self._shapes, self._types):
            if p.shape != shape or p.dtype != dtype:
                raise ValueError("a weight is not what it was: its shape or type changed")
            if not p.is_cuda or p.device != self.params[0].device:
                raise ValueError("params must be on one GPU")
            if p.dtype not in _TYPE:
                raise ValueError(f"params must be float32, float16 or bfloat16, not {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("params must be contiguous")

    # what a step writes: tuples, whose tensors may be written and moved
    params = property(lambda self: self._params)
    exp_avg = property(lambda self: self._states["exp_avg"])
    exp_avg_sq = property(lambda self: self._states["exp_avg_sq"])
    exp_avg_scale = property(lambda self: self._states["exp_avg_scale"])
    exp_avg_sq_scale = property(lambda self: self._states["exp_avg_sq_scale"])
    copies = property(lambda self: self._copies)

    def _look(self, torch):
        """Checks weights, states and copies and takes their addresses: at first, and where one of them moved."""
        self._check_weights()
        for what, (dtype, shapes) in self._kinds.items():
            x = self._states[what]
            if len(x) != len(self.params):
                raise ValueError(f"{what} must be a tensor for every weight")
            for t, s, p in zip(x, shapes, self.params):
                if not isinstance(t, torch.Tensor) or t.shape != s or t.dtype != dtype or t.device != p.device or not t.is_contiguous():
                    raise ValueError(f"{what} must be contiguous {dtype} tensors of shape {[list(s) for s in shapes]}")
        if len(self.copies) != len(self.params):
            raise ValueError("copies must be a tensor or None for every weight")
        for c, p in zip(self.copies, self.params):
            if c is not None and (not isinstance(c, torch.Tensor) or c.dtype not in _TYPE or c.shape != p.shape
                                  or c.device != p.device or not c.is_contiguous()):
                raise ValueError("a copy must be a contiguous float32, float16 or bfloat16 tensor of its weight's shape and device")
        self._records["param"] = [p.data_ptr() for p in self.params]
        for name in self._kinds:
            self._records[name] = [t.data_ptr() for t in self._states[name]]
        self._records["copy"] = [0 if c is None else c.data_ptr() for c in self.copies]
        self._records["copy_type"] = [0 if c is None else _TYPE[c.dtype] for c in self.copies]
        lists = [self.params] + [self._states[name] for name in self._kinds]
        self._held = [t for x in lists for t in x] + [c for c in self.copies if c is not None]
        self._addresses = [t.data_ptr() for t in self._held]
        self._memory = [t.untyped_storage() for t in self._held]   # (kept: what moves leaves its memory to nobody else before it is seen)
        self._counters = None

    def _written(self, grads):
        """What a step with these gradients (None: all of them) writes, a tensor for every version counter: views share their
        base's."""
        lists = [self.params, self.copies] + [self._states[name] for name in self._kinds]
        all_ = [t for x in lists for i, t in enumerate(x) if t is not None and (grads is None or grads[i] is not None)]
        return list({id(b): b for b in (t if t._base is None else t._base for t in all_)}.values())

    def _scalar(self, torch, x, dtype, what):
        if not isinstance(x, torch.Tensor) or x.numel() != 1 or x.dtype != dtype or x.device != self.params[0].device:
            raise ValueError(f"{what} must be a {dtype} tensor of one value beside the weights")
        return x.data_ptr()

    def step(self, grads=None, *, lr=None, grad_scale=None, skip=None):
        """One step with ``grads``, a list of tensors (f32, f16 or bf16 of the weights' shapes; None leaves its weight as it
        is), by default the weights' ``.grad``.  ``lr`` replaces the rate for this step: a number, or an f32 tensor of one
        value on the GPU.  ``grad_scale``: an f32 tensor of one value by which gradients are multiplied.
        ``skip``: an i32 tensor of one value; where it is not 0, nothing is changed (a number in ``steps`` still counts
        the step)."""
        torch = _state["torch"]
        params = self.params
        grads = [p.grad for p in params] if grads is None else list(grads)
        if len(grads) != len(params):
            raise ValueError("grads must be a tensor or None for every weight")
        if not params:
            return
        dev, records, some = params[0].device, self._records, None
        # (attribute by attribute over all tensors: a loop over them would cost more than the step of small ones)
        try:
            shapes, records["n"] = list(map(_SHAPE, grads)), self._sizes
        except AttributeError:   # (a weight without a gradient: nothing of it is touched)
            some = grads
            records["n"] = np.where([g is None for g in grads], 0, self._sizes)
            grads = [p if g is None else g for g, p in zip(grads, params)]
            shapes = [getattr(g, "shape", None) for g in grads]
        try:
            same = shapes == self._shapes and set(map(torch.Tensor.get_device, grads)) == {dev.index}
            types = list(map(_DTYPE, grads))
            if types != self._grad_types:
                records["grad_type"] = [_TYPE[t] for t in types]
                self._grad_types = types
        except (KeyError, TypeError, AttributeError):
            same = False
        if not same:
            raise ValueError("a gradient must be a float32, float16 or bfloat16 tensor of its weight's shape and device")
        if not all(map(torch.Tensor.is_contiguous, grads)):
            grads = [g.contiguous() for g in grads]
        # (weights, states or copies that moved, weights of another shape or type in the same place)
        if (list(map(torch.Tensor.data_ptr, self._held)) != self._addresses or list(map(_SHAPE, params)) != self._shapes
                or list(map(_DTYPE, params)) != self._types or not all(map(torch.Tensor.is_contiguous, params))):
            self._look(torch)
        records["grad"] = list(map(torch.Tensor.data_ptr, grads))
        s = _Settings(beta1=self.beta1, beta2=self.beta2, eps=self.eps, weight_decay=self.weight_decay, seed=self.seed,
                      state=1 if self._small else 0)
        lr = self.lr if lr is None else lr
        if isinstance(lr, torch.Tensor):
            s.lr_device = self._scalar(torch, lr, torch.float32, "lr")
        else:
            s.lr = lr
        if grad_scale is not None:
            s.grad_scale = self._scalar(torch, grad_scale, torch.float32, "grad_scale")
        if skip is not None:
            s.skip = self._scalar(torch, skip, torch.int32, "skip")
        with _on(params[0]):
            counted = None
            if isinstance(self.steps, torch.Tensor):
                s.step_device = self._scalar(torch, self.steps, torch.int64, "steps")
                counted = 1 if skip is None else (skip.view(self.steps.shape) == 0)
                self.steps.add_(counted)
            else:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("a step that is captured into a graph needs its number on the GPU: give AdamW steps as an int64 tensor")
                s.step = self.steps + 1
            code = _state["adamw"](records.ctypes.data, len(params), C.byref(s), _stream(params[0]))
            if code and counted is not None:   # (a step that was refused is not counted)
                self.steps.sub_(1 if skip is None else counted.to(torch.int64))
            _state["check"](code)
        if some is None and self._counters is None:
            self._counters = self._written(None)
        torch.autograd.graph.increment_version(self._counters if some is None else self._written(some))
        if counted is None:
            self.steps += 1
