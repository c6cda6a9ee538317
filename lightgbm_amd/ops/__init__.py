"""Operators over class scores and class probabilities, on the host or on a HIP device.

`top_logits` selects what a teacher has to say about a row, `distill_loss` and
`distill_gradients` are the objective that trains a student on it (the `distill` objective of
`train` runs the same code), and `verify_drafts` turns classes that a student drafted into
classes distributed as the target's probabilities say.

Arrays are numpy arrays or torch tensors. Tensors on a HIP device are used where they are: the
work goes to the current stream of their device, nothing is copied and nothing waits, and the
results are tensors of that device. Everything else is computed on the host. Any strides will
do. The functions record nothing for automatic differentiation: `distill_gradients` is the
backward pass of `distill_loss`. A tensor that requires a gradient is refused where gradients are
recorded (detach it, or call under `torch.no_grad()`), and so is one that carries a tangent.
"""
import ctypes
import operator
import struct
import sys
from typing import Any, NamedTuple, Optional

import numpy as np

from ..basic import _LIB, LightGBMError, _safe_call

__all__ = ["TopLogits", "DistillGradients", "VerifiedDrafts", "top_logits", "distill_loss",
           "distill_gradients", "verify_drafts"]


class TopLogits(NamedTuple):
    """The top logits of a teacher.

    classes: [rows, k] integers; an id outside 0..num_classes-1 (top_logits writes -1) is an
        empty slot, whose logit is not looked at. Of a class named twice in a row the first
        slot counts.
    logits: [rows, k].
    log_rest: [rows] or None, the log-sum-exp at the loss's temperature of the teacher's logits
        of all other classes. Without it the teacher's probabilities are normalised over the
        slots; a row of -inf, with empty slots, has no teacher.
    """
    classes: Any
    logits: Any
    log_rest: Optional[Any] = None


class DistillGradients(NamedTuple):
    gradient: Any
    hessian: Optional[Any] = None
    loss: Optional[Any] = None


class VerifiedDrafts(NamedTuple):
    """classes: [sequences, drafts + 1] int32, the accepted drafts, the class drawn after them,
    then -1. accepted: [sequences] int32, how many drafts were accepted."""
    classes: Any
    accepted: Any


_F32, _F64, _I32, _I64, _F16, _BF16 = range(6)
_NUMPY_TYPES = {"f4": _F32, "f8": _F64, "i4": _I32, "i8": _I64, "f2": _F16}
_NUMPY_OF = {_F32: np.float32, _F64: np.float64, _I32: np.int32, _F16: np.float16}
_TORCH_TYPES = {}
_TORCH_OF = {}

# LGBM_Array: data, three strides, type, reserved
_TOP = struct.Struct("@qiid" + "Pqqqii" * 4)
_DISTILL = struct.Struct("@qiidd" + "Pqqqii" * 9)
_VERIFY = struct.Struct("@qii" + "Pqqqii" * 8 + "Pq")
_NONE = (0, 0, 0, 0, 0, 0)


def _unpackable(e):
    return LightGBMError(f"an argument is not of its kind, or out of range: {e}")


for _f in (_LIB.LGBM_TopLogits, _LIB.LGBM_Distill, _LIB.LGBM_VerifyDrafts):
    _f.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p]
_LIB.LGBM_VerifyDraftsWorkspace.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]

_WORKSPACE = {}  # bytes, by a call's sizes

# torch is looked up when the first array that may be its is seen: the package works without
_torch = None
_Tensor = ()
_raw_stream = None
_forward = None  # torch.autograd.forward_ad; its level is -1 where no tangents are about


def _is_tensor(x):
    global _torch, _Tensor, _raw_stream, _forward
    if _torch is None:
        torch = sys.modules.get("torch")
        if torch is None:
            return False
        for code, name in ((_F32, "float32"), (_F64, "float64"), (_I32, "int32"),
                           (_I64, "int64"), (_F16, "float16"), (_BF16, "bfloat16")):
            _TORCH_TYPES[getattr(torch, name)] = code
            _TORCH_OF[code] = getattr(torch, name)
        # the current stream of a device as a pointer, where torch has it without an object
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _forward = torch.autograd.forward_ad
        _torch = torch
        _Tensor = torch.Tensor  # last, as another thread's call looks at it first
    return isinstance(x, _torch.Tensor)


class _Place:
    """Where a call runs, and how its results are made: as its first array is."""

    __slots__ = ("tensor", "device", "on", "made")

    def __init__(self, x):
        self.made = []  # arrays that stand for other objects, alive as long as the call
        self.device = -1
        self.on = None
        self.tensor = isinstance(x, _Tensor) or _is_tensor(x)
        if self.tensor:
            self.on = x.device
            if x.is_cuda:
                self.device = x.get_device()
            elif self.on.type != "cpu":
                raise LightGBMError(f"tensors on {self.on} are not supported")

    def stream(self):
        return _raw_stream(self.device) if self.device >= 0 else None

    def empty(self, shape, code):
        """A new array in row order, and the six fields of its LGBM_Array."""
        step = shape[1] if len(shape) == 2 else 1
        if self.tensor:
            made = _torch.empty(shape, dtype=_TORCH_OF[code], device=self.on)
            at = made.data_ptr()
        else:
            made = np.empty(shape, dtype=_NUMPY_OF[code])
            at = made.__array_interface__["data"][0]
        return made, (at, step, 1, 0, code, 0)

    def scores(self, rows, classes, code, class_major):
        """The same, in the order of scores [rows, classes]."""
        if not class_major:
            return self.empty((rows, classes), code)
        made, (at, *_) = self.empty((classes, rows), code)
        return made.T, (at, 1, rows, 0, code, 0)

    def array(self, x, name, shape):
        """The six fields of an LGBM_Array of x, which has to be of this place and shape."""
        if x is None:
            return _NONE
        if isinstance(x, _Tensor) or _is_tensor(x):
            # -1: the host
            if x.get_device() != self.device if self.device >= 0 else not x.is_cpu:
                raise LightGBMError(f"{name} is on {x.device}, the first array on "
                                    f"{self.on or 'the host'}")
            if x.requires_grad or x.is_neg() or _forward._current_level >= 0:
                x = _plain_tensor(x, name)
                self.made.append(x)
            if x.shape != shape:
                raise _shape_error(x, name, shape)
            return _tensor_fields(x, name)
        if self.device >= 0:
            raise LightGBMError(f"{name} must be a tensor on {self.on}, as the first array is")
        if not isinstance(x, np.ndarray):
            x = np.asarray(x)
            self.made.append(x)
        if x.shape != shape:
            raise _shape_error(x, name, shape)
        return _array_fields(x, name)


def _shape_error(x, name, shape):
    return LightGBMError(f"{name} must have the shape {list(shape)}, got {list(x.shape)}")


def _plain_tensor(x, name):
    """A tensor that is no more than its memory's values: a view that negates (the imaginary part
    of a conjugate) is written out, on its device's current stream; one whose gradient or tangent
    would be lost is refused."""
    if x.requires_grad and _torch.is_grad_enabled():
        raise LightGBMError(f"{name} requires a gradient, and this function records none: detach "
                            "it, or call under torch.no_grad()")
    if _forward.unpack_dual(x).tangent is not None:
        raise LightGBMError(f"{name} carries a tangent, which this function would lose")
    return x.resolve_neg() if x.is_neg() else x


def _fields(x, name):
    return _array_fields(x, name) if isinstance(x, np.ndarray) else _tensor_fields(x, name)


def _array_fields(x, name):
    dtype = x.dtype
    code = _NUMPY_TYPES.get(dtype.kind + str(dtype.itemsize)) if dtype.isnative else None
    if code is None:
        raise _type_error(x, name)
    size = dtype.itemsize
    if any(s % size for s in x.strides):
        raise LightGBMError(f"{name} has strides that are no multiple of its elements")
    steps = [s // size for s in x.strides] + [0, 0]
    return (x.__array_interface__["data"][0], *steps[:3], code, 0)


def _tensor_fields(x, name):
    code = _TORCH_TYPES.get(x.dtype)
    if code is None:
        raise _type_error(x, name)
    steps = x.stride()
    n = len(steps)
    if n == 2:
        return (x.data_ptr(), steps[0], steps[1], 0, code, 0)
    if n == 1:
        return (x.data_ptr(), steps[0], 0, 0, code, 0)
    return (x.data_ptr(), *steps, code, 0)


def _type_error(x, name):
    return LightGBMError(f"{name} has the type {x.dtype}, which is not supported")


def _shaped(x, name, dims=2):
    """x as an array, with its shape, which has to have so many dimensions."""
    if isinstance(x, _Tensor) or _is_tensor(x):
        if x.requires_grad or x.is_neg() or _forward._current_level >= 0:
            x = _plain_tensor(x, name)
    elif not isinstance(x, np.ndarray):
        x = np.asarray(x)
    shape = x.shape
    if len(shape) != dims:
        raise LightGBMError(f"{name} must have {dims} dimensions, got {list(shape)}")
    return x, shape


def top_logits(scores, k, temperature=1.0, rest=True):
    """The k largest scores of each row, largest first, with the log-sum-exp of the others.

    scores: [rows, classes] float64, float32, float16 or bfloat16, at most 1048576 classes.
    k: 1..min(classes, 256).
    temperature: what the scores are divided by in log_rest; the logits stay as they are.
    rest: whether log_rest is computed; it is float64 for float64 scores, else float32.

    Equal scores go to the lowest class first. NaN and -inf are never selected: a row with
    fewer than k other scores ends in class -1 with logit -inf. log_rest leaves NaN out.
    """
    scores, (rows, classes) = _shaped(scores, "scores")
    where = _Place(scores)
    x = _fields(scores, "scores")
    code = x[4]
    try:
        k = operator.index(k)
    except TypeError:
        raise LightGBMError(f"k must be a whole number, got {k!r}") from None
    if not 1 <= k <= min(classes, 256):
        raise LightGBMError(f"k must be 1..{min(classes, 256)} for {classes} classes, got {k}")
    out_class, to_class = where.empty((rows, k), _I32)
    out_logit, to_logit = where.empty((rows, k), code)
    log_rest, to_rest = (where.empty((rows,), _F64 if code == _F64 else _F32) if rest
                         else (None, _NONE))
    try:
        args = _TOP.pack(rows, classes, k, temperature, *x, *to_class, *to_logit, *to_rest)
    except struct.error as e:
        raise _unpackable(e) from None
    _safe_call(_LIB.LGBM_TopLogits(args, where.device, where.stream()))
    return TopLogits(out_class, out_logit, log_rest)


def _distill(scores, teacher, labels, weight, temperature, alpha, loss, gradient, hessian):
    scores, (rows, classes) = _shaped(scores, "scores")
    where = _Place(scores)
    if not 2 <= len(teacher) <= 3:
        raise LightGBMError("teacher must be (classes, logits) or (classes, logits, log_rest)")
    t_class, (_, k) = _shaped(teacher[0], "teacher classes")
    # every row of the results; what is not asked for, or not looked at, is absent
    row, slots = (rows,), (rows, k)
    x = _fields(scores, "scores")
    code = x[4]
    out = _F32 if code == _F64 else code
    class_major = x[1] == 1 and x[2] != 1
    fields = (rows, classes, k, temperature, alpha, *x,
              *where.array(t_class, "teacher classes", slots),
              *where.array(teacher[1], "teacher logits", slots),
              *where.array(teacher[2] if len(teacher) == 3 else None, "teacher log_rest", row),
              *where.array(None if alpha == 1.0 else labels, "labels", row),
              *where.array(weight, "weight", row))
    absent = (None, _NONE)
    made_loss, to_loss = where.empty(row, _F64 if code == _F64 else _F32) if loss else absent
    made_grad, to_grad = where.scores(rows, classes, out, class_major) if gradient else absent
    made_hess, to_hess = where.scores(rows, classes, out, class_major) if hessian else absent
    try:
        args = _DISTILL.pack(*fields, *to_loss, *to_grad, *to_hess)
    except struct.error as e:
        raise _unpackable(e) from None
    _safe_call(_LIB.LGBM_Distill(args, where.device, where.stream()))
    return made_loss, made_grad, made_hess


def distill_loss(scores, teacher, labels=None, weight=None, temperature=1.0, alpha=1.0):
    """The distillation loss of each row, [rows] (float64 for float64 scores, else float32).

    With Q = softmax(scores / T) and P the teacher's probabilities at the same temperature,

        weight * (alpha * T**2 * KL(P || Q) + (1 - alpha) * -log softmax(scores)[label])

    where the classes that the teacher does not name are one event: P of it comes from
    log_rest, Q of it is the sum of theirs.

    scores: [rows, classes], the student's.
    teacher: TopLogits, or a tuple of its two or three arrays; 1..256 slots a row.
    labels: [rows] integers or float32, needed where alpha < 1; a label outside
        0..classes-1 leaves its row without that term.
    weight: [rows]. A row of weight zero, and a row whose scores are all -inf, has no loss and
        no gradient, whatever else stands in it.
    """
    return _distill(scores, teacher, labels, weight, temperature, alpha, True, False, False)[0]


def distill_gradients(scores, teacher, labels=None, weight=None, temperature=1.0, alpha=1.0,
                      hessian=False, loss=False):
    """The gradient of the sum of distill_loss with respect to the scores, [rows, classes], and
    in the same pass, where asked for, the diagonal of the hessian as the multiclass objective
    has it (classes / (classes - 1) * q * (1 - q)) and the loss.

    The scores' type and order (float32 for float64 scores, as all gradients of the framework).
    """
    made = _distill(scores, teacher, labels, weight, temperature, alpha, loss, True, hessian)
    return DistillGradients(made[1], made[2], made[0])


def verify_drafts(target_prob, drafts, draft_prob, accept_uniform, sample_uniform, lengths=None):
    """Accept or replace drafted classes so that the results are distributed as the target's.

    target_prob: [sequences, drafts + 1, classes], the target's probabilities at each drafted
        place and at the one after; float64, float32, float16 or bfloat16.
    drafts: [sequences, drafts] int32 or int64, at most 1024 a sequence.
    draft_prob: [sequences, drafts, classes], the target's type: the probabilities that the
        drafts were drawn from, or None for drafts that were not drawn (probability one).
    accept_uniform: [sequences, drafts] and
    sample_uniform: [sequences], uniform numbers in [0, 1), float32 or float64.
    lengths: [sequences] int32 or int64, how many drafts a sequence has, all where None.

    A draft x stands while accept * q(x) < p(x), compared in 64 bits. After the last that
    stands one class is drawn: from max(p - q, 0) at the first refused place, from p after the
    last draft; the smallest class with mass whose running sum exceeds sample times the whole. NaN,
    infinite and negative entries weigh nothing, a draft outside 0..classes-1 is refused. Where
    the difference has no mass the draw is from p, where p has none the class is -1.
    """
    target_prob, (rows, places, classes) = _shaped(target_prob, "target_prob", 3)
    where = _Place(target_prob)
    t = places - 1
    fields = (rows, classes, t, *_fields(target_prob, "target_prob"),
              *where.array(draft_prob, "draft_prob", (rows, t, classes)),
              *where.array(drafts, "drafts", (rows, t)),
              *where.array(accept_uniform, "accept_uniform", (rows, t)),
              *where.array(sample_uniform, "sample_uniform", (rows,)),
              *where.array(lengths, "lengths", (rows,)))
    out_class, to_class = where.empty((rows, places), _I32)
    out_accepted, to_accepted = where.empty((rows,), _I32)
    fields += (*to_class, *to_accepted)
    scratch = size = 0
    if where.device >= 0:
        # what the call needs goes by its sizes, types and strides alone
        plan = (rows, classes, t, fields[3 + 4], fields[3 + 3], draft_prob is None or fields[9 + 3])
        size = _WORKSPACE.get(plan)
        if size is None:
            need = ctypes.c_int64(0)
            _safe_call(_LIB.LGBM_VerifyDraftsWorkspace(_VERIFY.pack(*fields, 0, 0),
                                                       ctypes.byref(need)))
            if len(_WORKSPACE) >= 1024:
                _WORKSPACE.clear()
            size = _WORKSPACE[plan] = need.value
        if size:
            # freed to the caching allocator, which gives it out again in the stream's order
            space = _torch.empty((size,), dtype=_torch.uint8, device=where.on)
            scratch = space.data_ptr()
    _safe_call(_LIB.LGBM_VerifyDrafts(_VERIFY.pack(*fields, scratch, size), where.device,
                                      where.stream()))
    return VerifiedDrafts(out_class, out_accepted)
