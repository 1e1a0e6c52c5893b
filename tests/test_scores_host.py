"""Score-row operators without a GPU: what they refuse, and the reference forms against differences and enumeration."""
import numpy as np
import pytest
import torch

import scores_reference as R
from loe_speech_recognition_amd import _native, distill_scores, sample_scores, top_scores


def _rows(n=4, v=9, dtype=torch.float32):
    return torch.zeros((n, v), dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: top_scores(np.zeros((2, 3), np.float32), 1), TypeError),
    (lambda: top_scores(_rows(dtype=torch.float64), 1), TypeError),
    (lambda: top_scores(_rows()[0], 1), ValueError),
    (lambda: top_scores(_rows(4, 0), 1), ValueError),
    (lambda: top_scores(_rows().t(), 1), ValueError),
    (lambda: top_scores(torch.zeros(1).expand(2, _native.MAX_CLASSES + 1), 1), ValueError),
    (lambda: top_scores(_rows(), 0), ValueError),
    (lambda: top_scores(_rows(), 10), ValueError),
    (lambda: top_scores(_rows(), 2.5), ValueError),
    (lambda: top_scores(_rows(2, 1000), _native.MAX_TOP + 1), ValueError),
    (lambda: top_scores(_rows(), 2, temperature=0.0), ValueError),
    (lambda: top_scores(_rows(), 2, temperature=float("inf")), ValueError),
    (lambda: top_scores(_rows(), 2, temperature=1e-39), ValueError),
    (lambda: top_scores(_rows(), 2, temperature=1e39), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=1e-310), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(), temperature=1e-39), ValueError),
    (lambda: top_scores(_rows(), 2), ValueError),                                     # not on the GPU
])
def test_top_scores_refuses(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("call,error", [
    (lambda: sample_scores(_rows(), np.zeros(4, np.float32)), TypeError),
    (lambda: sample_scores(_rows(), torch.zeros(4, dtype=torch.float64)), TypeError),
    (lambda: sample_scores(_rows(), torch.zeros(3)), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=-1.0), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=float("nan")), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=float("inf")), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=torch.ones(4, dtype=torch.float64)), TypeError),
    (lambda: sample_scores(_rows(), torch.zeros(4), temperature=torch.ones(4, 1)), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), top_k=-1), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), top_k=1.5), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), top_k=torch.ones(4, dtype=torch.int64)), TypeError),
    (lambda: sample_scores(_rows(), torch.zeros(4), top_p=1.1), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), top_p=float("nan")), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4), min_p=-0.1), ValueError),
    (lambda: sample_scores(_rows(), torch.zeros(4)), ValueError),                     # not on the GPU
])
def test_sample_scores_refuses(call, error):
    with pytest.raises(error):
        call()


def _teacher(n=4, k=3):
    return torch.zeros((n, k)), torch.zeros((n, k), dtype=torch.int32)


@pytest.mark.parametrize("call,error", [
    (lambda: distill_scores(_rows(), torch.zeros(4), torch.zeros(4, dtype=torch.int32)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(3)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(4, 0)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(4, _native.MAX_TOP + 1)), ValueError),
    (lambda: distill_scores(_rows(), torch.zeros((4, 3)), torch.zeros((4, 3), dtype=torch.int64)), TypeError),
    (lambda: distill_scores(_rows(), torch.zeros((4, 3), dtype=torch.bfloat16), _teacher()[1]), TypeError),
    (lambda: distill_scores(_rows(), torch.zeros((4, 3)), torch.zeros((4, 2), dtype=torch.int32)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(), rest=torch.zeros(3)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(), row_weight=torch.zeros(4, 1)), ValueError),
    (lambda: distill_scores(_rows(), *_teacher(), temperature=-2.0), ValueError),
    (lambda: distill_scores(_rows(), *_teacher()), ValueError),                       # not on the GPU
])
def test_distill_scores_refuses(call, error):
    with pytest.raises(error):
        call()


def test_entry_points_refuse_a_missing_context():
    lib = _native.load_library()
    assert lib.lsr_top_scores(None, None, 0, 1, 1, 1, 1, 1.0, None, None, None) == -1
    assert lib.lsr_sample_scores(None, None, 0, 1, 1, 1, None, 1.0, 0, 1.0, 0.0, None, None, None, None, None, None) == -1
    assert lib.lsr_distill_scores(None, None, 0, 1, 1, 1, None, None, 1, None, 1.0, None, None, None) == -1


def test_reference_gradient_matches_differences():
    """The formula's gradient against central differences of the formula's loss: with a listed class twice, an absent entry,
    with and without the outcome of the rest.  Truncation h^2 / 6 times a third derivative of order t^-1, rounding
    2^-53 loss / h: both below 1e-9 at h = 1e-5."""
    rng = np.random.default_rng(3)
    for rest in (None, -0.7):
        for t in (1.0, 2.5):
            s = rng.normal(size=12) * 3
            values, index = rng.normal(size=5) * 2, np.array([4, 1, 4, -1, 9])
            _, grad = R.distill(s, values, index, rest, t, 0.3)
            for i in range(12):
                h = np.zeros(12)
                h[i] = 1e-5
                d = (R.distill(s + h, values, index, rest, t, 0.3)[0] - R.distill(s - h, values, index, rest, t, 0.3)[0]) / 2e-5
                assert abs(d - grad[i]) < 1e-8


def test_reference_draws_every_kept_class_in_proportion():
    x = np.array([1.0, 3.0, -np.inf, 3.0, 0.5, np.nan, 2.0])
    u = (np.arange(4000) + 0.5) / 4000
    drawn = np.bincount([R.sample(x, v, 1.5, 4, 0.97, 0.05)[0] for v in u], minlength=7)
    w = np.exp((np.array([1.0, 3.0, 0, 3.0, 0, 0, 2.0]) - 3) / 1.5) * np.array([1, 1, 0, 1, 0, 0, 1])
    assert np.abs(drawn - 4000 * w / w.sum()).max() <= 1      # one boundary per class, each between two of the numbers
