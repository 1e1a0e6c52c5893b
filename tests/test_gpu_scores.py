"""Score-row operators on the GPU against plain 64-bit forms (scores_reference.py), row by row."""
import ctypes

import numpy as np
import pytest
import torch

import scores_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# smallest positive number of the type; in the 32-bit exponent range 2^-120, as exponentials below 2^-126 may come out as 0
# and are multiplied by at most weight * temperature / smallest share of the tests
TINY = {"f32": 2.0 ** -120, "f16": 2.0 ** -24, "bf16": 2.0 ** -120}
WIDTHS = [1, 2, 3, 11, 17, 58, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2048, 4099, 8200, 33000]


def _device(x, dtype="f32", pad=0, fill=float("nan")):
    """The matrix on the GPU with ``pad`` elements of ``fill`` between its rows, and its values as float64."""
    x = torch.tensor(np.asarray(x, np.float64)).to(TYPES[dtype])
    buf = torch.full((x.shape[0], x.shape[1] + pad), fill, dtype=x.dtype, device="cuda")
    view = buf[:, :x.shape[1]]
    view.copy_(x)
    return view, x.double().numpy()


def _matrix(rng, rows, classes, hard=True):
    """Rows of log scores; with ``hard`` the last ones hold what goes wrong first: ties, masks, one score, none, infinities,
    signed zeros, NaN, numbers near the ends of the types."""
    x = rng.normal(size=(rows, classes)) * 3
    if not hard:
        return x
    special = []
    special.append(np.zeros(classes))
    special.append(np.full(classes, -np.inf))
    special.append(np.full(classes, np.nan))
    special.append(np.round(rng.normal(size=classes)))
    one = np.full(classes, -np.inf)
    one[classes // 2] = -3.0
    special.append(one)
    m = rng.normal(size=classes)
    m[rng.random(classes) < 0.7] = -np.inf
    special.append(m)
    z = np.where(np.arange(classes) % 2 == 0, -0.0, 0.0)
    special.append(z)
    m = rng.normal(size=classes)
    m[::3] = np.nan
    special.append(m)
    special.append(-60000.0 + 100 * rng.normal(size=classes))
    special.append(np.where(rng.random(classes) < 0.5, 60000.0, -60000.0))
    special.append(rng.normal(size=classes) * 1e-6)
    m = rng.normal(size=classes)
    m[rng.integers(0, classes)] = np.inf
    special.append(m)
    return np.concatenate([x, np.stack(special)])


def _span(x, t):
    """Largest |z| = |x - best| / t that still has weight in 32 bits (e^-104 has none)."""
    x = x[np.isfinite(x)]
    return min(104.0, (x.max() - x.min()) / t) if len(x) else 0.0


def _sum_error(classes, span):
    """Relative error of a sum of e^z in 32 bits: an argument off by 4 roundings of |z| (difference, reciprocal of t,
    product, change of base), an exponential and its scaling off by 4 half steps, additions in at most classes / 64 + 128
    steps (a lane adds every 64th element or, in short rows, all 128)."""
    return 2.0 ** -24 * (4 * span + 4 + classes / 64 + 128)


# ---- top ----------------------------------------------------------------------------------------------------------------
def _check_top(view, x, k, t):
    from loe_speech_recognition_amd import top_scores

    values, index, rest = (v.cpu().numpy().astype(np.float64) for v in top_scores(view, k, temperature=t, want_rest=True))
    for r in range(x.shape[0]):
        v, i, q = R.top(x[r], k, t)
        assert np.array_equal(index[r], i), (r, index[r], i)
        assert np.array_equal(values[r], v), r
        # the logarithm's own roundings and those of the distance to the best: four of |rest|
        tol = _sum_error(x.shape[1], _span(x[r], t)) + 2.0 ** -22 * abs(q)
        assert rest[r] == q or abs(rest[r] - q) <= tol, (r, rest[r], q, tol)
    plain = top_scores(view, k, temperature=t)
    assert plain[2] is None and np.array_equal(plain[1].cpu().numpy(), index)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("classes", WIDTHS)
def test_top_scores(classes, dtype):
    rng = np.random.default_rng(classes)
    view, x = _device(_matrix(rng, 5, classes), dtype, pad=[0, 1, 6][classes % 3])
    for k in sorted({1, min(classes, 2), min(classes, 8), min(classes, 17), min(classes, 64), min(classes, 256)}):
        _check_top(view, x, k, 1.0 if k % 2 else 3.0)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 200, 1000])
def test_top_scores_row_counts(rows):
    rng = np.random.default_rng(rows)
    view, x = _device(_matrix(rng, rows, 58, hard=False), "f32", pad=6, fill=float("-inf"))
    _check_top(view, x, 8, 8.0)


# ---- sample --------------------------------------------------------------------------------------------------------------
def _check_sample(view, x, u, t, top_k, top_p, min_p, as_tensor=False):
    from loe_speech_recognition_amd import sample_scores

    n = x.shape[0]
    per_row = [np.broadcast_to(np.asarray(s), (n,)) for s in (t, top_k, top_p, min_p)]
    if as_tensor:
        given = [torch.tensor(np.ascontiguousarray(s), dtype=torch.int32 if j == 1 else torch.float32, device="cuda")
                 for j, s in enumerate(per_row)]
        per_row = [g.cpu().numpy() for g in given]
    else:
        given = [t, top_k, top_p, min_p]
    d_u = torch.tensor(u, dtype=torch.float32, device="cuda")
    index, logprob = sample_scores(view, d_u, *given)
    index, logprob, u = index.cpu().numpy(), logprob.cpu().numpy().astype(np.float64), d_u.cpu().numpy().astype(np.float64)
    for r in range(n):
        i, lp = R.sample(x[r], float(u[r]), *(float(s[r]) if j != 1 else int(s[r]) for j, s in enumerate(per_row)))
        assert index[r] == i, (r, index[r], i, u[r], [s[r] for s in per_row])
        # 64-bit weights in multiples of 2^-38 at worst, then one rounding to 32 bits
        assert logprob[r] == lp or abs(logprob[r] - lp) <= 2.0 ** -24 * abs(lp) + 1e-10, (r, logprob[r], lp)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 1, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (2.0, 0, 0.5, 0.0), (1.0, 0, 0.95, 0.0),
            (1.0, 0, 0.0, 0.0), (1.5, 0, 1.0, 0.1), (1.0, 0, 1.0, 1.0), (0.8, 50, 0.9, 0.02), (3.0, 40, 0.99, 0.0),
            (0.0, 3, 0.9, 0.1), (1e-3, 0, 0.9, 0.0), (50.0, 300, 0.999, 0.0)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("classes", WIDTHS)
def test_sample_scores(classes, dtype):
    rng = np.random.default_rng(100 + classes)
    view, x = _device(_matrix(rng, 5, classes), dtype, pad=[0, 3, 8][classes % 3])
    for j, (t, top_k, top_p, min_p) in enumerate(SETTINGS):
        u = rng.random(x.shape[0])
        u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
        _check_sample(view, x, u, t, top_k, top_p, min_p)


@pytest.mark.parametrize("classes,dtype", [(11, "f32"), (58, "f32"), (100, "f16"), (1000, "bf16"), (20011, "bf16")])
def test_sample_scores_settings_per_row(classes, dtype):
    rng = np.random.default_rng(classes)
    n = 70
    view, x = _device(_matrix(rng, n, classes), dtype)
    n = x.shape[0]
    _check_sample(view, x, rng.random(n), rng.uniform(-0.2, 2.0, n), rng.integers(-2, 2 * min(classes, 100), n),
                  rng.uniform(-0.1, 1.2, n), np.where(rng.random(n) < 0.5, 0.0, rng.uniform(-0.1, 1.1, n)), as_tensor=True)


@pytest.mark.parametrize("classes", [4, 58, 128, 1000, 5000])
def test_sample_scores_on_the_borders(classes):
    """Equal weights: u = i / classes (exact for powers of two and otherwise on one side of the border in 64 bits as well)
    and cuts that fall between equal scores."""
    x = np.zeros((classes, classes)) - 7.0
    view, x = _device(x)
    u = np.arange(classes) / classes
    for top_k, top_p in ((0, 1.0), (classes // 2, 1.0), (0, 0.5), (3, 0.75)):
        _check_sample(view, x, u, 1.0, top_k, top_p, 0.0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("classes", [11, 58, 100, 1000, 8200, 20011, 70001])
def test_rows_masked_with_the_lowest_number(classes, dtype):
    """Nearly all scores are the type's lowest number: it has no weight, so that not even a uniform number of 0 draws it,
    but it is an entry of the row for top_scores."""
    rng = np.random.default_rng(classes)
    x = rng.normal(size=(8, classes))
    lowest = torch.finfo(TYPES[dtype]).min
    for r, allowed in enumerate([1, 2, 3, 5, 8, 10, 10, 0]):
        masked = np.ones(classes, bool)
        masked[rng.permutation(classes)[:allowed]] = False
        masked[0] = True
        x[r, masked] = lowest
    x[6, classes // 2:] = -np.inf                         # and some are not there at all
    x[6, -1] = 0.5
    view, x = _device(x, dtype, pad=3)
    u = np.array([0.0, 1.0, 0.0, 0.3, 0.0, 0.9, 0.0, 0.0])
    for t, top_k, top_p, min_p in [(1.0, 0, 1.0, 0.0), (1.0, 6, 1.0, 0.0), (0.7, 9, 0.9, 0.0), (1.0, 300, 1.0, 0.0),
                                   (2.0, 400, 0.95, 0.0), (1.0, 0, 0.95, 0.0), (1.0, 0, 0.95, 0.01), (1.5, 0, 1.0, 0.05)]:
        _check_sample(view, x, u, t, top_k, top_p, min_p)
    for k in sorted({1, 4, 9, min(classes, 64), min(classes, 256)}):
        _check_top(view, x, k, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [1000, 8200, 70001])
def test_top_scores_of_many_equal_ones(classes, dtype):
    """More equal scores at the last places than a list has room for: the first classes of them are taken."""
    rng = np.random.default_rng(classes)
    x = np.full((6, classes), 1.0)
    x[1, rng.permutation(classes)[:30]] = 2.0
    x[2, rng.permutation(classes)[:classes // 4]] = 0.5
    x[3, rng.permutation(classes)[:classes // 3]] = np.nan
    x[3, 7] = 3.0
    x[4] = np.where(rng.random(classes) < 0.1, 4.0, 5.0)
    x[5, ::2] = 1.5
    x[5, :3 * classes // 4] = -np.inf
    view, x = _device(x, dtype, pad=1)
    for k in [1, 5, 29, 30, 31, 64, 255, 256]:
        _check_top(view, x, k, 1.0)


@pytest.mark.parametrize("classes,dtype", [(58, "f32"), (1000, "f16"), (20011, "f32"), (70001, "bf16")])
def test_extreme_temperatures(classes, dtype):
    rng = np.random.default_rng(classes + 9)
    n = 12
    x = rng.normal(size=(n, classes))
    x[:, 3] = -np.inf
    x[1::2, 5] = x[1::2].max(axis=1)                      # two best ones
    view, x = _device(x, dtype)
    t = np.array([1e-45, 1e-45, 1e-38, 1e-38, 1e-30, 1e-20, 1e20, 1e30, 1e38, 3e38, 1e-3, 1e3])
    for top_k, top_p, min_p in [(0, 1.0, 0.0), (7, 1.0, 0.0), (400, 0.9, 0.0), (0, 0.8, 0.0), (0, 0.8, 0.5)]:
        _check_sample(view, x, rng.random(n), t, np.full(n, top_k), np.full(n, top_p), np.full(n, min_p), as_tensor=True)
    for one in (1e-30, 1e30):
        _check_top(view, x, 6, one)


def test_sample_scores_distribution():
    """The share of each class over evenly spread uniform numbers is its probability to within one number per border."""
    from loe_speech_recognition_amd import sample_scores

    rng = np.random.default_rng(8)
    for classes in (58, 700):
        row = torch.tensor(rng.normal(size=classes) * 2, dtype=torch.float32, device="cuda")
        n = 1 << 16
        u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().cuda()
        index, _ = sample_scores(row[None].expand(n, classes), u)              # row stride 0
        got = torch.bincount(index.long(), minlength=classes).double()
        want = torch.softmax(row.double(), 0) * n
        assert (got - want).abs().max().item() <= 1.0


# ---- distill -------------------------------------------------------------------------------------------------------------
def _check_distill(view, x, dtype, values, index, rest, t, weight):
    from loe_speech_recognition_amd import distill_scores

    n, classes = x.shape
    dev = lambda a, d: None if a is None else torch.tensor(a, dtype=d, device="cuda")
    values, rest, weight = (None if a is None else np.asarray(a, np.float32).astype(np.float64) for a in (values, rest, weight))
    d = (dev(values, torch.float32), dev(index, torch.int32))
    kw = dict(rest=dev(rest, torch.float32), temperature=t, row_weight=dev(weight, torch.float32))
    loss, grad = distill_scores(view, *d, **kw)
    only, none = distill_scores(view, *d, **kw, want_grad=False)
    assert none is None and torch.equal(only.view(torch.int32), loss.view(torch.int32)) and grad.dtype == view.dtype
    loss, grad = loss.cpu().numpy().astype(np.float64), grad.double().cpu().numpy()
    for r in range(n):
        w = 1.0 if weight is None else weight[r]
        want, g = R.distill(x[r], values[r], index[r], None if rest is None else rest[r], t, w)
        if w == 0:
            assert loss[r] == 0 and not grad[r].any()
            continue
        if not np.isfinite(want):
            assert (np.isnan(loss[r]) and np.isnan(want)) or loss[r] == want, (r, loss[r], want)
            assert np.array_equal(np.isnan(grad[r]), np.isnan(g)), r
            if np.isnan(want):
                continue
        span = _span(x[r], t)
        e = _sum_error(classes, span)
        # every p and q is off by e relative; the logarithms' errors come with the weights p, which sum to 1
        if np.isfinite(want):
            logs = abs(want) / (abs(w) * t * t) + 2
            tol = abs(w) * t * t * (4 * e + 2.0 ** -22 * logs * (1 + span)) + 2.0 ** -24 * abs(want)
            assert abs(loss[r] - want) <= tol, (r, loss[r], want, tol)
        q = np.zeros(classes)
        fine = x[r] > -np.inf
        if fine.any():
            z = (x[r] - x[r][fine].max()) / t
            q[fine] = np.exp(z[fine])
            q /= q.sum()
        # terms of the gradient before they cancel: q_i, what the teacher asks for (q_i - g_i / (w t)), each off by 3 e
        terms = abs(w) * t * (2 * q + np.abs(g / (w * t)))
        tol = 3 * e * terms + HALF_STEP[dtype] * np.abs(g) * (1 + 2.0 ** -8) + TINY[dtype]
        assert np.all(np.abs(grad[r] - g) <= tol), (r, np.max(np.abs(grad[r] - g) - tol), int(np.argmax(np.abs(grad[r] - g) - tol)))


def _teacher(rng, rows, classes, k, absent=True):
    values = -np.sort(-rng.normal(size=(rows, k)) * 2, axis=1)
    index = np.stack([rng.permutation(classes)[:k] if classes >= k else rng.integers(0, classes, k) for _ in range(rows)])
    if absent and rows > 4:
        index[0] = -1                                     # no entry at all
        values[1] = -np.inf
        index[2, k // 2] = classes                        # outside the row
        values[3, -1] = np.nan
        index[4] = index[4, 0]                            # the same class k times
    return values, index


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("classes", WIDTHS)
def test_distill_scores(classes, dtype):
    rng = np.random.default_rng(200 + classes)
    view, x = _device(_matrix(rng, 8, classes), dtype, pad=[0, 5, 2][classes % 3])
    n = x.shape[0]
    for j, k in enumerate(sorted({1, min(classes, 3), min(classes, 20), min(classes, 256)})):
        values, index = _teacher(rng, n, classes, k)
        rest = rng.normal(size=n)
        rest[5] = -np.inf
        weight = rng.uniform(0.1, 2.0, n)
        weight[6], weight[-1] = 0.0, 0.0
        _check_distill(view, x, dtype, values, index, rest, 1.0, weight)
        _check_distill(view, x, dtype, values, index, None, 2.5, None if j % 2 else weight)


def test_distill_scores_more_entries_than_classes():
    rng = np.random.default_rng(4)
    view, x = _device(_matrix(rng, 8, 5))
    values, index = _teacher(rng, x.shape[0], 5, 40)
    _check_distill(view, x, "f32", values, index, rng.normal(size=x.shape[0]), 1.0, None)


@pytest.mark.parametrize("classes", [58, 300, 5000])
def test_distill_scores_of_a_student_that_is_sure(classes):
    """Scores so far apart that the weight outside the listed classes is below e^-100: its logarithm is still there."""
    rng = np.random.default_rng(6)
    x = np.full((6, classes), -400.0) + rng.normal(size=(6, classes))
    index = np.stack([rng.permutation(classes)[:4] for _ in range(6)])
    for r in range(6):
        x[r, index[r]] = rng.normal(size=4)
    view, x = _device(x)
    _check_distill(view, x, "f32", rng.normal(size=(6, 4)), index, np.full(6, -2.0), 1.0, None)


def test_distill_scores_is_cross_entropy_for_one_entry():
    from loe_speech_recognition_amd import distill_scores

    rng = np.random.default_rng(5)
    x = torch.tensor(rng.normal(size=(300, 58)) * 4, dtype=torch.float32, device="cuda", requires_grad=True)
    label = torch.tensor(rng.integers(0, 58, 300), dtype=torch.int32, device="cuda")
    loss, grad = distill_scores(x, torch.zeros((300, 1), device="cuda"), label[:, None])
    want = torch.nn.functional.cross_entropy(x.double().cpu(), label.long().cpu(), reduction="none")
    g, = torch.autograd.grad(want.sum(), x)
    e = _sum_error(58, 40.0)
    assert (loss.cpu().double() - want).abs().max().item() <= 8 * e * 2 + 2.0 ** -24 * want.max().item()
    assert (grad - g).abs().max().item() <= 6 * e


# ---- long rows, many rows, 64-bit offsets ----------------------------------------------------------------------------------
@pytest.mark.parametrize("classes,dtype", [(70001, "f32"), (131072, "bf16"), (262144, "f32"), (300007, "f16"), (1500000, "bf16")])
def test_long_rows(classes, dtype):
    rng = np.random.default_rng(classes)
    x = rng.normal(size=(3, classes)) * 2
    x[1] = np.round(x[1])                                 # a few values, tens of thousands of ties
    x[2, rng.random(classes) < 0.9] = -np.inf
    view, x = _device(x, dtype)
    _check_top(view, x, 100, 1.0)
    for t, top_k, top_p, min_p in ((1.0, 0, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (2.0, 5000, 0.99, 1e-3)):
        _check_sample(view, x, rng.random(3), t, top_k, top_p, min_p)
    values, index = _teacher(rng, 3, classes, 64, absent=False)
    for r in range(3):                                    # classes the student has
        index[r] = rng.choice(np.nonzero(x[r] > -np.inf)[0], 64, replace=False)
    _check_distill(view, x, dtype, values, index, rng.normal(size=3), 1.0, None)
    _check_distill(view, x, dtype, values, index, None, 2.0, rng.uniform(0.5, 1.0, 3))


def test_offsets_beyond_32_bits():
    """Rows that start more than 2^32 elements behind the first one: a matrix of two rows with a large stride."""
    from loe_speech_recognition_amd import distill_scores, sample_scores, top_scores

    stride = (1 << 32) + 5
    buf = torch.zeros(stride + 4096, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(1)
    x = torch.tensor(rng.normal(size=(2, 4096)) * 3, dtype=torch.bfloat16)
    view = buf.as_strided((2, 4096), (stride, 1))
    view.copy_(x)
    near = x.cuda()
    u = torch.tensor([0.3, 0.8], device="cuda")
    teacher = top_scores(near, 20, want_rest=True)
    for a, b in zip(top_scores(view, 20, want_rest=True), teacher):
        assert torch.equal(a, b)
    for a, b in zip(sample_scores(view, u, top_p=0.9), sample_scores(near, u, top_p=0.9)):
        assert torch.equal(a, b)
    for a, b in zip(distill_scores(view, *teacher[:2], rest=teacher[2]), distill_scores(near, *teacher[:2], rest=teacher[2])):
        assert torch.equal(a, b)


def test_more_rows_than_one_launch_takes():
    """2^21 rows of more than 128 classes are a launch; what lies beyond is read and written at its own place."""
    from loe_speech_recognition_amd import distill_scores, sample_scores, top_scores

    rng = np.random.default_rng(21)
    n = 2 ** 21 + 3
    view, x = _device(_matrix(rng, 1, 130, hard=False), "f32")
    rows = view.expand(n, -1)
    u = torch.zeros(n, device="cuda")
    u[-2:] = torch.tensor([0.4, 0.999], device="cuda")
    values, index, rest = top_scores(rows, 2, want_rest=True)
    v, i, q = R.top(x[0], 2, 1.0)
    assert (index == torch.tensor(i, device="cuda")).all() and (values[-3:].cpu().numpy() == v).all()
    assert (rest == rest[0]).all() and abs(rest[0].item() - q) <= _sum_error(130, _span(x[0], 1.0)) + 2.0 ** -22 * abs(q)
    drawn, logprob = sample_scores(rows, u)
    want = [R.sample(x[0], float(a), 1.0, 0, 1.0, 0.0)[0] for a in u[-3:].tolist()]
    assert drawn[-3:].tolist() == want and (drawn[:-2] == want[0]).all() and (logprob[:-2] == logprob[0]).all()
    loss, grad = distill_scores(rows, values, index, rest=rest)
    assert (loss == loss[0]).all() and (grad[-4:] == grad[0]).all()
    del loss, grad


def test_rows_masked_in_a_long_batch():
    """Workgroups that go on from row to row meet rows whose equal scores overflow the list between ordinary ones."""
    rng = np.random.default_rng(8)
    x = torch.tensor(rng.normal(size=(700, 66000)), dtype=torch.bfloat16)
    for r in range(0, 700, 3):
        x[r, rng.random(66000) > 1e-3] = torch.finfo(x.dtype).min
    from loe_speech_recognition_amd import top_scores

    for want_rest in (False, True):
        values, index, rest = top_scores(x.cuda(), 200, want_rest=want_rest)
        for r in [*range(0, 12), *range(253, 262), *range(508, 520), *range(690, 700)]:
            v, i, q = R.top(x[r].double().numpy(), 200, 1.0)
            assert np.array_equal(index[r].cpu().numpy(), i) and np.array_equal(values[r].double().cpu().numpy(), v), r
            if want_rest:
                tol = _sum_error(66000, _span(x[r].double().numpy(), 1.0)) + 2.0 ** -22 * abs(q)
                assert abs(rest[r].item() - q) <= tol, (r, rest[r].item(), q)


def test_no_rows():
    from loe_speech_recognition_amd import distill_scores, sample_scores, top_scores

    x = torch.empty((0, 58), device="cuda")
    values, index, rest = top_scores(x, 4, want_rest=True)
    assert values.shape == (0, 4) and index.shape == (0, 4) and rest.shape == (0,)
    assert sample_scores(x, torch.empty(0, device="cuda"))[0].shape == (0,)
    loss, grad = distill_scores(x, values, index, rest=rest)
    assert loss.shape == (0,) and grad.shape == (0, 58)


def test_outputs_stop_at_their_ends():
    """Nothing is written outside the results, and the gaps between the rows of the scores stay as they are."""
    from loe_speech_recognition_amd import _native

    eng = _native.get_engine()
    rng = np.random.default_rng(2)
    for rows, classes, k, dtype in ((67, 58, 8, "f32"), (5, 1001, 33, "f16"), (3, 40003, 64, "bf16")):
        view, x = _device(rng.normal(size=(rows, classes)), dtype, pad=3, fill=7.0)
        whole = view.as_strided((rows, classes + 3), (classes + 3, 1))
        code = {"f32": 0, "f16": 1, "bf16": 2}[dtype]
        guard = lambda n, t: torch.full((n + 64,), 77, dtype=t, device="cuda")
        values, index, rest, drawn, share = (guard(n, t) for n, t in (
            (rows * k, torch.float32), (rows * k, torch.int32), (rows, torch.float32), (rows, torch.int32), (rows, torch.float32)))
        loss, grad = guard(rows, torch.float32), guard(rows * classes, TYPES[dtype])
        u = torch.rand(rows, device="cuda")
        p = eng._ptr
        common = (p(view), code, rows, classes, classes + 3)
        eng.on_current_stream(eng.lib.lsr_top_scores, *common, k, 1.0, p(values), p(index), p(rest))
        eng.on_current_stream(eng.lib.lsr_sample_scores, *common, p(u), 1.0, 0, 0.9, 0.0, None, None, None, None, p(drawn), p(share))
        eng.on_current_stream(eng.lib.lsr_distill_scores, *common, p(values), p(index), k, p(rest), 1.0, None, p(loss), p(grad))
        torch.cuda.synchronize()
        for t, n in ((values, rows * k), (index, rows * k), (rest, rows), (drawn, rows), (share, rows), (loss, rows),
                     (grad, rows * classes)):
            assert (t[n:] == 77).all() and not (t[:n] == 77).all()
        assert (whole[:, classes:] == 7.0).all()


def test_c_entry_points_refuse():
    """Errors of the C entry points with a valid context: the code, the name in the message, and no launch."""
    from loe_speech_recognition_amd import _native

    eng = _native.get_engine()
    x = torch.zeros((4, 9), device="cuda")
    out = torch.full((64,), 5.0, device="cuda")
    p = eng._ptr

    def code(fn, *args):
        rc = fn(eng.ctx, *args)
        return rc, eng.lib.lsr_last_error(eng.ctx).decode()

    top = lambda s=p(x), d=0, n=4, v=9, st=9, k=2, t=1.0, o=p(out): code(eng.lib.lsr_top_scores, s, d, n, v, st, k, t, o, o, None)
    for kw, want in (({"d": 3}, -1), ({"n": -1}, -1), ({"v": 0}, -1), ({"st": -1}, -1), ({"k": 0}, -1), ({"k": 10}, -1),
                     ({"t": 0.0}, -1), ({"t": float("nan")}, -1), ({"s": None}, -1), ({"o": None}, -1),
                     ({"s": ctypes.c_void_p(x.data_ptr() + 2)}, -1), ({"v": (1 << 24) + 1}, -3), ({"v": 1000, "k": 257}, -3),
                     ({"t": 1e-31}, -3), ({"t": 1e31}, -3)):
        rc, text = top(**kw)
        assert rc == want and "lsr_top_scores" in text, (kw, rc, text)
    for args in ((None, 1.0, 0, 1.0, 0.0), (p(out), float("nan"), 0, 1.0, 0.0), (p(out), 1.0, 0, float("nan"), 0.0)):
        rc, text = code(eng.lib.lsr_sample_scores, p(x), 0, 4, 9, 9, *args, None, None, None, None, p(out), p(out))
        assert rc == -1 and "lsr_sample_scores" in text
    for k, t, v, want in ((0, 1.0, p(out), -1), (257, 1.0, p(out), -3), (2, -1.0, p(out), -1), (2, 1.0, None, -1)):
        rc, text = code(eng.lib.lsr_distill_scores, p(x), 0, 4, 9, 9, v, p(out), k, None, t, None, p(out), None)
        assert rc == want and "lsr_distill_scores" in text
    torch.cuda.synchronize()
    assert (out == 5.0).all()


# ---- streams and graphs ----------------------------------------------------------------------------------------------------
def _all_three(x, u):
    from loe_speech_recognition_amd import distill_scores, sample_scores, top_scores

    teacher = top_scores(x, min(20, x.shape[1]), want_rest=True)
    drawn = sample_scores(x, u, temperature=0.9, top_k=100, top_p=0.9, min_p=0.01)
    return (*teacher, *drawn, *distill_scores((x.float() * 0.5).to(x.dtype), *teacher[:2], rest=teacher[2], temperature=2.0))


@pytest.mark.parametrize("rows,classes,dtype", [(300, 58, "f32"), (9, 20011, "bf16"), (1, 131072, "bf16")])
def test_on_another_stream(rows, classes, dtype):
    x = (torch.randn((rows, classes), device="cuda") * 3).to(TYPES[dtype])
    u = torch.rand(rows, device="cuda")
    want = _all_three(x, u)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 1.0                                       # made on the stream, used right behind it
        got = _all_three(y, u)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,classes,dtype", [(300, 58, "f32"), (9, 20011, "bf16"), (2, 131072, "bf16")])
def test_two_captured_graphs(rows, classes, dtype):
    """Two graphs of the same calls, replayed in turn and side by side with eager calls in between, equal the eager results."""
    inputs = [((torch.randn((rows, classes), device="cuda") * 3).to(TYPES[dtype]), torch.rand(rows, device="cuda")) for _ in range(2)]
    for x, u in inputs:
        _all_three(x, u)
    graphs, results = [], []
    for x, u in inputs:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(_all_three(x, u))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for x, u in inputs:
            x.copy_((torch.randn((rows, classes), device="cuda") * (2 + turn)).to(TYPES[dtype]))
            u.copy_(torch.rand(rows, device="cuda"))
        want = [_all_three(x, u) for x, u in inputs]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, w in zip(results, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b), turn


def test_threads_on_streams_of_their_own():
    import threading

    from loe_speech_recognition_amd import sample_scores, top_scores

    rng = np.random.default_rng(31)
    views = [_device(_matrix(rng, 40, 1000 + 100 * i, hard=False), "f32")[0] for i in range(4)]
    u = torch.tensor(rng.random(40), dtype=torch.float32, device="cuda")
    want = [(top_scores(v, 9)[1], sample_scores(v, u, 0.9, 50, 0.95)[0]) for v in views]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                x = views[i] + 0.0                        # on this thread's stream: a call on another one could overtake it
                got = top_scores(x, 9)[1], sample_scores(x, u, 0.9, 50, 0.95)[0]
                if not all(bool(torch.equal(a, b)) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_same_bits_in_any_batch():
    """A row's results do not depend on the rows around it nor on how often it is run."""
    from loe_speech_recognition_amd import distill_scores

    for classes, dtype in ((58, "f32"), (3001, "f16"), (70001, "bf16")):
        x = (torch.randn((130, classes), device="cuda") * 3).to(TYPES[dtype])
        u = torch.rand(130, device="cuda")
        want = _all_three(x, u)
        for a, b in zip(_all_three(x, u), want):
            assert torch.equal(a, b)
        for lo, hi in ((0, 1), (7, 9), (64, 130)):
            for a, b in zip(_all_three(x[lo:hi], u[lo:hi]), want):
                assert torch.equal(a, b[lo:hi]), (classes, lo, hi)
    index = torch.zeros((5, 30), dtype=torch.int32, device="cuda")          # one class thirty times
    x = torch.randn((5, 2000), device="cuda")
    v = torch.randn((5, 30), device="cuda")
    first = distill_scores(x, v, index)
    for _ in range(5):
        for a, b in zip(distill_scores(x, v, index), first):
            assert torch.equal(a, b)


# ---- the framework's own rows ------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def digits():
    from loe_speech_recognition_amd import MFCC, HiddenMarkovModelInference, ModelCollection, synthetic

    models = synthetic.load_word_models()
    inf = HiddenMarkovModelInference.from_models([models[lab] for lab in synthetic.LOOP_ORDER])
    mc = ModelCollection()
    mc._models = [models[lab] for lab in synthetic.LOOP_ORDER if lab != "S"]
    signals, truth = synthetic.batch(31, 12, 1)
    return inf, mc, MFCC.batch(signals, 16000), truth


def test_collection_nbest_and_draws(digits):
    _, mc, feats, _ = digits
    scores = mc.scores_batch(feats).astype(np.float64)
    names = [str(m) for m in mc._models]
    best = mc.predict_batch(feats)
    for n in (1, 3, len(names)):
        out = mc.nbest_batch(feats, n)
        assert [row[0][0] for row in out] == best
        for r, row in enumerate(out):
            assert [names.index(a) for a, _ in row] == R.order(scores[r])[:n].tolist()
            assert [float(v) for _, v in row] == scores[r][R.order(scores[r])[:n]].tolist()
    u = np.linspace(0, 0.999, len(feats)).astype(np.float32)
    for settings in ((50.0, 0, 1.0, 0.0), (200.0, 4, 0.9, 0.01), (0.0, 0, 1.0, 0.0)):
        want = [names[R.sample(scores[r], float(u[r]), *settings)[0]] for r in range(len(feats))]
        assert mc.sample_batch(feats, u, *settings) == want
    assert mc.sample_batch(feats, u, 0.0) == best


def test_a_student_of_the_word_models(digits):
    """Audio -> features -> state scores -> targets -> a student's loss and gradient -> its weights -> draws from the
    student: every step against the plain form on the values the step before gave."""
    from loe_speech_recognition_amd import distill_scores, sample_scores

    inf, _, feats, _ = digits
    t = 6.0
    fb, state_scores = inf.state_scores_device(feats)
    x = state_scores.cpu().numpy().astype(np.float64)
    assert x.shape == (fb.total_frames, len(inf._multivariate_normals)) and state_scores.stride(0) == 64
    fb, values, index, rest = inf.state_targets(fb, 8, temperature=t)
    v, i, q = values.cpu().numpy(), index.cpu().numpy(), rest.cpu().numpy().astype(np.float64)
    for r in range(0, fb.total_frames, 7):
        rv, ri, rq = R.top(x[r], 8, t)
        assert np.array_equal(v[r], rv) and np.array_equal(i[r], ri)
        assert abs(q[r] - rq) <= _sum_error(58, _span(x[r], t)) + 2.0 ** -22 * abs(rq)
    gen = torch.Generator(device="cuda").manual_seed(0)
    weight = (torch.randn((39, x.shape[1]), generator=gen, device="cuda") * 0.1).requires_grad_()
    share = torch.full((fb.total_frames,), 1.0 / fb.total_frames, device="cuda")
    for step in range(3):
        logits = fb.feats @ weight
        loss, grad = distill_scores(logits, values, index, rest=rest, temperature=t, row_weight=share)
        weight.grad = None
        logits.backward(grad)
        s = logits.detach().cpu().numpy().astype(np.float64)
        want = np.zeros((39, x.shape[1]))
        total, f = 0.0, fb.feats.cpu().numpy().astype(np.float64)
        for r in range(fb.total_frames):
            l, g = R.distill(s[r], v[r], i[r], q[r], t, 1.0 / fb.total_frames)
            total += l
            want += f[r][:, None] * g[None, :]
        assert abs(loss.double().sum().item() - total) <= 1e-4 * total
        got = weight.grad.double().cpu().numpy()
        assert np.linalg.norm(got - want) <= 1e-4 * np.linalg.norm(want)
        with torch.no_grad():
            weight -= 0.05 * weight.grad
    u = torch.rand((fb.total_frames,), generator=gen, device="cuda")
    _check_sample(logits.detach(), s, u.cpu().numpy(), 1.0, 20, 0.95, 0.0)
    _, drawn, _ = inf.sample_states(fb, u, temperature=t, top_p=0.9)
    for r in range(0, fb.total_frames, 11):
        assert drawn[r].item() == R.sample(x[r], float(u[r].item()), t, 0, 0.9, 0.0)[0]
    assert torch.equal(sample_scores(state_scores, u, t, 0, 0.9)[0], drawn)


@pytest.mark.parametrize("classes,dtype", [(1000, "f32"), (9001, "f16"), (131072, "bf16"), (50001, "f32")])
def test_sample_scores_of_hundreds_of_entries(classes, dtype):
    """min_p that hundreds or thousands of entries reach, with and without a cut by top_p among them."""
    rng = np.random.default_rng(classes + 5)
    view, x = _device(rng.normal(size=(24, classes)) * 2.0, dtype)
    best = x.max(axis=1)
    order = np.sort(x, axis=1)[:, ::-1]
    reach = np.array([260, 300, 400, 480, 511, 513, 900, 2000, 2049, 4000, 4100, 5000] * 2) % classes
    min_p = np.exp(order[np.arange(24), reach] - best)
    top_p = np.where(np.arange(24) < 12, 1.0, rng.uniform(0.02, 0.9, 24))
    u = rng.random(24)
    u[3], u[20] = 0.0, 1.0 - 2.0 ** -24
    _check_sample(view, x, u, np.ones(24), np.zeros(24, int), top_p, min_p, as_tensor=True)
