"""Operators on class scores that live on the GPU: the top classes of a row with its
log-sum-exp, distillation of a student from a teacher's top classes (loss and gradient),
classes drawn from given random numbers, and log probabilities of given classes with their gradient.

They take torch tensors on the GPU and enqueue on torch's current stream; what they return
is made by torch on that stream.  Scores are [rows][classes], f32, f16 or bf16, of any
strides.  A trained model's scores ([classes][rows] f64 on the host, from ``Trainer.approx`` or
``apply_oblivious``) go in as f32 on the GPU: ``torch.from_numpy(raw).float().cuda().t()``.

They record no autograd graph, also where the scores require a gradient: a loss is a value to look at, and the
gradient goes on with ``scores.backward(grad)``.

One HIP runtime serves a process: import torch before the first call of this package (a library
that was loaded before torch runs on another copy of the runtime, which cannot take torch's
tensors; these functions then raise).
"""
from __future__ import annotations

from collections import namedtuple

_TYPE = {}      # torch dtype -> CBH_TYPE_*
_state = {}     # the bound library functions, once the runtime was looked at


def _runtimes():
    with open("/proc/self/maps") as f:
        return {l.split()[-1] for l in f if "libamdhip64" in l}


def _bind():
    import torch

    import catboost_rs_amd as cb
    L = cb.load()
    if len(_runtimes()) > 1:
        raise RuntimeError("two HIP runtimes are loaded: import torch before the first call of catboost_rs_amd")
    _TYPE.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    _state.update(torch=torch, lib=L, check=cb._check, error=cb.CbhError, top=L.cbh_top_classes, top_ws=L.cbh_top_classes_workspace,
                  distill=L.cbh_distill_gradients, distill_ws=L.cbh_distill_gradients_workspace,
                  sample=L.cbh_sample_classes, sample_ws=L.cbh_sample_classes_workspace,
                  logprobs=L.cbh_class_logprobs, logprobs_ws=L.cbh_class_logprobs_workspace,
                  logprob_grad=L.cbh_logprob_gradients, lookup=L.cbh_lookup_rows, table_grad=L.cbh_lookup_gradients,
                  table_grad_ws=L.cbh_lookup_gradients_workspace, adamw=L.cbh_adamw_step,
                  raw_stream=getattr(torch._C, "_cuda_getCurrentRawStream", None))
    return torch


def _scores(torch, x, what="scores"):
    """Type, rows, classes and strides of a matrix of scores."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{what} must be a torch tensor [rows][classes]")
    t = _TYPE.get(x.dtype)
    if t is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on the GPU")
    (n, m), (rs, cs) = x.shape, x.stride()
    if m > 1 << 24:   # (before anything of that size is allocated, and before 32 bits cut it off)
        raise _state["error"](-2, f"{what}: classes must be in 1 .. 2^24")
    return t, n, m, rs, cs


def _vector(torch, x, shape, dtype, like, what):
    """`x` as a contiguous tensor of this shape and type beside `like`; its address."""
    if not isinstance(x, torch.Tensor) or x.shape != shape:
        raise ValueError(f"{what} must be a torch tensor of shape {list(shape)}")
    if x.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, not {x.dtype}")
    if x.device != like.device:
        raise ValueError(f"{what} must be on {like.device}, not {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _workspace(torch, n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


def _addr(x):
    return None if x is None else x.data_ptr()


class _Stay:
    def __enter__(self):
        pass

    def __exit__(self, *_):
        pass


_STAY = _Stay()


def _on(x):
    """The device of `x` made current for the call (nothing where it is: the context costs a small call 2 us)."""
    cuda = _state["torch"].cuda
    return _STAY if cuda.current_device() == x.device.index else cuda.device(x.device)


def _stream(x):
    """torch's current stream on the device of `x`, as an address."""
    raw = _state["raw_stream"]
    return raw(x.device.index) if raw else _state["torch"].cuda.current_stream(x.device).cuda_stream


def top_classes(scores, k, temperature=1.0):
    """The ``k`` largest scores of every row (``cbh_top_classes``): ``values`` [rows][k] f32, largest
    first, their classes ``index`` [rows][k] i32 (the lowest first among equal scores), and
    ``lse`` [rows] f32, the row's log-sum-exp of ``scores / temperature``: what
    :func:`distill_gradients` takes of a teacher.  1 <= k <= min(classes, 1024); 1e-38 <= temperature <= 1e36."""
    torch = _state.get("torch") or _bind()
    t, n, m, rs, cs = _scores(torch, scores)
    k = int(k)
    k = k if 1 <= k <= 1024 else 0   # (0: refused below)
    with _on(scores):
        dev = scores.device
        values = torch.empty((n, k), dtype=torch.float32, device=dev)
        index = torch.empty((n, k), dtype=torch.int32, device=dev)
        lse = torch.empty(n, dtype=torch.float32, device=dev)
        size = _state["top_ws"](n, m, k)
        ws = _workspace(torch, size, scores)
        _state["check"](_state["top"](scores.data_ptr(), t, n, m, rs, cs, k, float(temperature), values.data_ptr(),
                                      index.data_ptr(), lse.data_ptr(), _addr(ws), size, _stream(scores)))
    return values, index, lse


def distill_gradients(scores, top_scores, top_index, *, top_lse=None, temperature=1.0, weight=None):
    """Loss [rows] f32 of a student's ``scores`` against a teacher's top classes, and its gradient, in the
    scores' type (``cbh_distill_gradients``: the formulas are there).  ``top_scores`` [rows][k] f32 and
    ``top_index`` [rows][k] i32 are the teacher's (an index outside the classes is no entry);
    ``top_lse`` [rows] f32 its log-sum-exp at this temperature, so that the classes it did not list
    share what is left of its mass, or None: the listed classes hold all of it.  ``weight`` [rows] f32
    scales a row's loss and gradient; 0 leaves the row out whatever it holds.  The loss carries no graph:
    a model's scores pass the gradient on with ``scores.backward(grad)``."""
    torch = _state.get("torch") or _bind()
    t, n, m, rs, cs = _scores(torch, scores)
    if not isinstance(top_scores, torch.Tensor) or top_scores.dim() != 2:
        raise ValueError("top_scores must be a torch tensor [rows][k]")
    k = top_scores.shape[1]
    u = _vector(torch, top_scores, (n, k), torch.float32, scores, "top_scores")
    ix = _vector(torch, top_index, (n, k), torch.int32, scores, "top_index")
    base = None if top_lse is None else _vector(torch, top_lse, (n,), torch.float32, scores, "top_lse")
    w = None if weight is None else _vector(torch, weight, (n,), torch.float32, scores, "weight")
    with _on(scores):
        loss = torch.empty(n, dtype=torch.float32, device=scores.device)
        grad = torch.empty_like(scores)
        grs, gcs = grad.stride()
        size = _state["distill_ws"](n, m)
        ws = _workspace(torch, size, scores)
        _state["check"](_state["distill"](scores.data_ptr(), t, n, m, rs, cs, u.data_ptr(), ix.data_ptr(), k, _addr(base),
                                          float(temperature), _addr(w), loss.data_ptr(), grad.data_ptr(), grs, gcs,
                                          _addr(ws), size, _stream(scores)))
    return loss, grad


def sample_classes(scores, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, allowed=None):
    """One class of every row (``index`` [rows] i32) and its log probability before the cuts (``logprob``
    [rows] f32), drawn with the given ``uniform`` [rows] f64 in [0, 1) (``cbh_sample_classes``: the order
    of the cuts is there).  ``temperature`` (<= 0: the largest score), ``top_k`` (0: all), ``top_p`` and
    ``min_p`` are numbers, or tensors [rows] (f32, ``top_k`` i32).  ``allowed``: i32 words
    [rows or 1][ceil(classes / 32)], bit ``j & 31`` of word ``j >> 5`` allows class j.  A row that allows
    nothing has index -1 and logprob -inf."""
    torch = _state.get("torch") or _bind()
    t, n, m, rs, cs = _scores(torch, scores)
    uniform = _vector(torch, uniform, (n,), torch.float64, scores, "uniform")

    def setting(v, dtype, what):
        if isinstance(v, torch.Tensor):
            return 0, _vector(torch, v, (n,), dtype, scores, what)
        return v, None

    tv, tr = setting(temperature, torch.float32, "temperature")
    kv, kr = setting(top_k, torch.int32, "top_k")
    pv, pr = setting(top_p, torch.float32, "top_p")
    mv, mr = setting(min_p, torch.float32, "min_p")
    astride = 0
    if allowed is not None:
        words = (m + 31) // 32
        one = isinstance(allowed, torch.Tensor) and allowed.dim() == 2 and allowed.shape[0] == 1
        allowed = _vector(torch, allowed, (1 if one else n, words), torch.int32, scores, "allowed")
        astride = 0 if one else words
    with _on(scores):
        index = torch.empty(n, dtype=torch.int32, device=scores.device)
        logprob = torch.empty(n, dtype=torch.float32, device=scores.device)
        size = _state["sample_ws"](n, m)
        ws = _workspace(torch, size, scores)
        _state["check"](_state["sample"](scores.data_ptr(), t, n, m, rs, cs, uniform.data_ptr(), float(tv), _addr(tr),
                                         min(max(int(kv), 0), m), _addr(kr), float(pv), _addr(pr), float(mv), _addr(mr),
                                         _addr(allowed), astride, index.data_ptr(), logprob.data_ptr(), _addr(ws), size,
                                         _stream(scores)))
    return index, logprob


ClassLogprobs = namedtuple("ClassLogprobs", "logprob entropy stats top_logprob top_index")


def _given(torch, given, n, like, what="given"):
    """Classes [rows] or [rows][m] i32, and their shape."""
    if not isinstance(given, torch.Tensor) or given.dim() not in (1, 2) or given.shape[0] != n:
        raise ValueError(f"{what} must be a torch tensor [rows] or [rows][m]")
    return _vector(torch, given, given.shape, torch.int32, like, what), given.shape[1] if given.dim() == 2 else 1


def _allowed(torch, allowed, n, m, like):
    """Words of allowed classes and their stride (0: one list for all rows)."""
    if allowed is None:
        return None, 0
    words = (m + 31) // 32
    one = isinstance(allowed, torch.Tensor) and allowed.dim() == 2 and allowed.shape[0] == 1
    return _vector(torch, allowed, (1 if one else n, words), torch.int32, like, "allowed"), 0 if one else words


def class_logprobs(scores, given=None, *, temperature=1.0, k=0, allowed=None):
    """Log probabilities of given classes with the entropy and the ``k`` most probable classes of every row
    (``cbh_class_logprobs``: the formulas are there), over the allowed classes at a temperature.  ``given``: i32
    [rows] or [rows][m], or None; an index outside the classes is no entry and has 0.  ``allowed`` as in
    :func:`sample_classes`.  Gives ``logprob`` f32 of given's shape, ``entropy`` [rows] f32 in nats, ``stats`` [rows][3]
    f32 (what :func:`logprob_gradients` takes), ``top_logprob`` [rows][k] f32, largest first, and ``top_index``
    [rows][k] i32 (-1 where fewer classes have a probability); 0 <= k <= min(classes, 1024).  ``logprob`` is None without
    ``given``, the top ones are without ``k``."""
    torch = _state.get("torch") or _bind()
    t, n, m, rs, cs = _scores(torch, scores)
    given, count = (None, 0) if given is None else _given(torch, given, n, scores)
    allowed, astride = _allowed(torch, allowed, n, m, scores)
    k = int(k)
    k = k if 0 <= k <= 1024 else 1 << 30   # (refused below, before anything of that size is allocated)
    with _on(scores):
        dev, f32 = scores.device, torch.float32
        logprob = None if given is None else torch.empty(given.shape, dtype=f32, device=dev)
        entropy, stats = torch.empty(n, dtype=f32, device=dev), torch.empty((n, 3), dtype=f32, device=dev)
        top_logprob = top_index = None
        if 0 < k <= 1024:
            top_logprob, top_index = torch.empty((n, k), dtype=f32, device=dev), torch.empty((n, k), dtype=torch.int32, device=dev)
        size = _state["logprobs_ws"](n, m, k) if k <= 1024 else 0
        ws = _workspace(torch, size, scores)
        _state["check"](_state["logprobs"](scores.data_ptr(), t, n, m, rs, cs, _addr(given), count, float(temperature),
                                           _addr(allowed), astride, k, _addr(logprob), entropy.data_ptr(),
                                           stats.data_ptr(), _addr(top_logprob), _addr(top_index), _addr(ws),
                                           size, _stream(scores)))
    return ClassLogprobs(logprob, entropy, stats, top_logprob, top_index)


def logprob_gradients(scores, given, logprob_grad, stats, *, entropy_grad=None, temperature=1.0, allowed=None):
    """Gradient by the scores, in their type and layout, of a function of what :func:`class_logprobs` gave for
    them (``cbh_logprob_gradients``): ``logprob_grad`` f32 of given's shape and ``entropy_grad`` [rows] f32 are its
    derivatives by the log probabilities and the entropy, ``stats`` what the forward call returned;
    ``temperature`` and ``allowed`` are those of that call.  For the entropy's derivative alone, ``given`` and
    ``logprob_grad`` may be [rows][0].  A row of zeros in both gives 0 whatever its scores
    hold."""
    torch = _state.get("torch") or _bind()
    t, n, m, rs, cs = _scores(torch, scores)
    given, count = _given(torch, given, n, scores)
    g = _vector(torch, logprob_grad, given.shape, torch.float32, scores, "logprob_grad")
    h = None if entropy_grad is None else _vector(torch, entropy_grad, (n,), torch.float32, scores, "entropy_grad")
    stats = _vector(torch, stats, (n, 3), torch.float32, scores, "stats")
    allowed, astride = _allowed(torch, allowed, n, m, scores)
    with _on(scores):
        grad = torch.empty_like(scores)
        grs, gcs = grad.stride()
        _state["check"](_state["logprob_grad"](scores.data_ptr(), t, n, m, rs, cs, given.data_ptr(), count, g.data_ptr(),
                                               _addr(h), stats.data_ptr(), float(temperature), _addr(allowed), astride,
                                               grad.data_ptr(), grs, gcs, _stream(scores)))
    return grad
