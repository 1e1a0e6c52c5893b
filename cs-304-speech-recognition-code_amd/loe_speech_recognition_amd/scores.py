"""Operators on rows of log scores: what a model answers with, one row per frame, clip or token and one column per class.

The framework's own rows are the emission scores of a batch (``Engine.emission``, frames x states) and the scores of an
isolated-word collection (``ModelCollection.scores_device``, clips x models); a student network trained on them, or any
other classifier, has rows of the same kind.  The reference takes the arg-max of such rows
(model_collection.py:26-28); here are

* ``top_scores``     - the k best classes of every row and the log weight of the rest,
* ``sample_scores``  - a class per row, drawn with temperature, top-k, top-p and min-p from given uniform numbers,
* ``distill_scores`` - loss and gradient of a student's rows against a teacher's top scores.

Scores are CUDA tensors [rows, classes] of float32, float16 or bfloat16 on the device of the process's engine; the classes
of a row have to be adjacent, rows may have any stride (a slice of the emission matrix is taken as it is).  The kernels run
on torch's current stream, after what the engine has queued on its own; nothing is allocated besides the results, so
calls can be captured into a graph.  Results are the same bits whatever the launch.  Threads may call the three at once,
each on its own stream, also while another thread decodes with the engine.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

from . import _native

_DTYPES = {}                 # torch dtype -> LSR_F32 / LSR_F16 / LSR_BF16, filled on first use


def _dtype_code(scores) -> int:
    if not _DTYPES:
        import torch

        _DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    code = _DTYPES.get(scores.dtype)
    if code is None:
        raise TypeError(f"scores must be float32, float16 or bfloat16, got {scores.dtype}")
    return code


def _check_scores(scores) -> Tuple[int, int, int]:
    """(rows, classes, element type code) of a score matrix, or the error that says what is wrong with it."""
    import torch

    if not isinstance(scores, torch.Tensor):
        raise TypeError("scores must be a torch tensor")
    code = _dtype_code(scores)
    if scores.dim() != 2:
        raise ValueError(f"scores must have shape [rows, classes], got {tuple(scores.shape)}")
    rows, classes = scores.shape
    if not 1 <= classes <= _native.MAX_CLASSES:
        raise ValueError(f"scores must have 1..{_native.MAX_CLASSES} classes, got {classes}")
    if classes > 1 and rows > 0 and scores.stride(1) != 1:
        raise ValueError("the classes of a row must be adjacent in memory (stride 1 in the last dimension)")
    return rows, classes, code


def _check_like(name: str, t, shape: Tuple[int, ...], dtype: str, device) -> None:
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype != getattr(torch, dtype):
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the scores on {device}")


def _check_temperature(temperature) -> float:
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be in 1e-30..1e30, got {temperature}")
    return temperature


def _engine(scores) -> "_native.Engine":
    if not scores.is_cuda:
        raise ValueError(f"scores must be on the GPU, they are on {scores.device}")
    eng = _native.get_engine()
    if scores.device != eng.device:
        raise ValueError(f"scores are on {scores.device}, the engine of this process on {eng.device}")
    return eng


def top_scores(scores, k: int, temperature: float = 1.0, want_rest: bool = False):
    """(values float32 [rows, k], index int32 [rows, k], rest float32 [rows] or None): the ``k`` best classes of every
    row, best first, equal scores by ascending class.  Scores of -inf and NaN are absent; rows with fewer than ``k``
    others are filled with -inf / -1.  ``rest`` is the log of the sum of ``exp((x - best) / temperature)`` over all other
    classes, -inf where there are none; ``temperature`` has no other effect."""
    rows, classes, code = _check_scores(scores)
    if isinstance(k, bool) or int(k) != k or not 1 <= k <= min(classes, _native.MAX_TOP):
        raise ValueError(f"k must be an integer in 1..{min(classes, _native.MAX_TOP)}, got {k}")
    temperature = _check_temperature(temperature)
    eng = _engine(scores)
    t = eng.torch
    values = eng.empty((rows, int(k)), t.float32)
    index = eng.empty((rows, int(k)), t.int32)
    rest = eng.empty((rows,), t.float32) if want_rest else None
    eng.on_current_stream(eng.lib.lsr_top_scores, eng._ptr(scores), code, rows, classes, scores.stride(0), int(k), temperature,
                          eng._ptr(values), eng._ptr(index), eng._ptr(rest))
    return values, index, rest


def sample_scores(scores, uniform, temperature: Union[float, "torch.Tensor"] = 1.0, top_k: Union[int, "torch.Tensor"] = 0,
                  top_p: Union[float, "torch.Tensor"] = 1.0, min_p: Union[float, "torch.Tensor"] = 0.0):
    """(index int32 [rows], logprob float32 [rows]): a class per row drawn with ``uniform`` (float32 [rows], numbers in
    [0, 1), for instance ``torch.rand``).

    With weights ``w = exp((x - best) / temperature)`` a row keeps, of its classes ordered by score, the first ``top_k``
    (0: all), of those the shortest head that holds ``top_p`` of their weight (1: all), and the ones with
    ``w >= min_p`` (0: all); at least its best.  The result is the first class in ascending order at which the running
    weight of the kept classes exceeds ``uniform`` times their total, and the log of its share of that total.
    ``temperature`` 0 takes the best class.  Every setting is a number or a tensor [rows] (float32; int32 for ``top_k``)
    with a number for each row.  Scores of -inf and NaN are never drawn, nor are scores masked with a type's lowest number (or
    others without weight in 64 bits, beyond 745 temperatures below the best); a row without others gives -1 and -inf."""
    import torch

    rows, classes, code = _check_scores(scores)
    _check_like("uniform", uniform, (rows,), "float32", scores.device)
    numbers, tensors = [], []
    for name, v, dtype in (("temperature", temperature, "float32"), ("top_k", top_k, "int32"), ("top_p", top_p, "float32"),
                           ("min_p", min_p, "float32")):
        if isinstance(v, torch.Tensor):
            _check_like(name, v, (rows,), dtype, scores.device)
            numbers.append(0)
            tensors.append(v.contiguous())
            continue
        if name == "top_k":
            if isinstance(v, bool) or int(v) != v or v < 0:
                raise ValueError(f"top_k must be an integer >= 0, got {v}")
            v = min(int(v), classes)
        elif not 0.0 <= float(v) <= (1e38 if name == "temperature" else 1.0) or (name == "temperature" and 0 < float(v) < 1e-45):
            raise ValueError(f"{name} must be {'0 or in 1e-45..1e38' if name == 'temperature' else 'in [0, 1]'}, got {v}")
        numbers.append(v if name == "top_k" else float(v))
        tensors.append(None)
    eng = _engine(scores)
    uniform = uniform.contiguous()
    index = eng.empty((rows,), torch.int32)
    logprob = eng.empty((rows,), torch.float32)
    eng.on_current_stream(eng.lib.lsr_sample_scores, eng._ptr(scores), code, rows, classes, scores.stride(0),
                          eng._ptr(uniform), *numbers, *(eng._ptr(v) for v in tensors), eng._ptr(index), eng._ptr(logprob))
    return index, logprob


def distill_scores(scores, top_values, top_index, rest=None, temperature: float = 1.0, row_weight=None,
                   want_grad: bool = True):
    """(loss float32 [rows], gradient like ``scores`` or None) of a student's scores against a teacher's top scores as
    ``top_scores`` gives them: ``top_values`` float32 and ``top_index`` int32 [rows, k], ``rest`` float32 [rows] or None.

    ``loss = row_weight * temperature**2 * KL(p || q)``: p the softmax of the teacher's entries / temperature, with ``rest``
    as one more outcome if it is given (without it the listed classes share all weight); q the softmax of ``scores`` /
    temperature, its weight outside the listed classes taken together for that outcome.  The gradient is that of
    ``loss.sum()``: ``scores.backward(gradient)`` continues into the student, with ``row_weight`` (float32 [rows], None: 1)
    carrying the reduction, e.g. ``1 / rows`` for the mean, and 0 for rows that do not count.

    An entry of the teacher with a class outside the row or a value of -inf or NaN is absent; a class that is given twice
    counts with both.  Loss and gradient are 0 for rows of weight 0, without an entry of the teacher or without a score of
    the student above -inf, and NaN for other rows with a NaN or +inf among the student's scores.  With one entry per row,
    temperature 1 and no ``rest`` this is the cross entropy with a label."""
    import torch

    rows, classes, code = _check_scores(scores)
    if not isinstance(top_values, torch.Tensor) or top_values.dim() != 2:
        raise ValueError("top_values must be a tensor [rows, k]")
    k = top_values.shape[1]
    if not 1 <= k <= _native.MAX_TOP:
        raise ValueError(f"the teacher must have 1..{_native.MAX_TOP} entries per row, got {k}")
    _check_like("top_values", top_values, (rows, k), "float32", scores.device)
    _check_like("top_index", top_index, (rows, k), "int32", scores.device)
    if rest is not None:
        _check_like("rest", rest, (rows,), "float32", scores.device)
    if row_weight is not None:
        _check_like("row_weight", row_weight, (rows,), "float32", scores.device)
    temperature = _check_temperature(temperature)
    eng = _engine(scores)
    inputs = [top_values.contiguous(), top_index.contiguous(), None if rest is None else rest.contiguous(),
              None if row_weight is None else row_weight.contiguous()]
    loss = eng.empty((rows,), torch.float32)
    grad = eng.empty((rows, classes), scores.dtype) if want_grad else None
    eng.on_current_stream(eng.lib.lsr_distill_scores, eng._ptr(scores), code, rows, classes, scores.stride(0),
                          eng._ptr(inputs[0]), eng._ptr(inputs[1]), k, eng._ptr(inputs[2]), temperature, eng._ptr(inputs[3]),
                          eng._ptr(loss), eng._ptr(grad))
    return loss, grad
