"""Score-row operators on the GPU: the paths that only rows of particular sizes, counts or contents take, against plain
64-bit forms (scores_reference.py) and against the same rows in calls that take another path."""
import numpy as np
import pytest
import torch

import scores_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _chain(classes, dtype):
    """Most additions in 32 bits that a term of a long row's sum goes through: the classes of one thread of its team, the
    entries of a list that a thread adds, six steps over the lanes, one per wavefront and the last ones."""
    run, four = (4, 8192) if dtype == "f32" else (8, 16384)
    least = 64 * (1 if classes <= 1024 else 4 if classes <= four else 8 if classes <= 4 * four else 16)
    return -(-classes // (least * run)) * run + 8 + 6 + 16 + 4


def _rest_error(x, dtype, t, q):
    """Bound of the error of ``rest``: arguments of the exponentials off by five roundings (difference, reciprocal of t, its
    product with log2 e, that constant, product) of at most the row's range, two exponentials of one step each and their
    product, the additions; the logarithm, the distance to the best and their sum four roundings of what they add up to."""
    there = x[np.isfinite(x)]
    span = min(104.0, (there.max() - there.min()) / t) if len(there) else 0.0
    gap = (there.max() - there.min()) / t if len(there) > 1 else 0.0
    return 2.0 ** -24 * (5 * span + 8 + _chain(len(x), dtype)) + 2.0 ** -24 * 4 * (abs(q) + min(gap, abs(q) + 17))


def _check_rows_of_top(got, x, rows, k, t, dtype):
    values, index, rest = got
    for r in rows:
        row = x[r].double().cpu().numpy()
        v, i, q = R.top(row, k, t)
        assert np.array_equal(index[r].cpu().numpy(), i) and np.array_equal(values[r].double().cpu().numpy(), v), r
        if rest is not None:
            assert rest[r].item() == q or abs(rest[r].item() - q) <= _rest_error(row, dtype, t, q), (r, rest[r].item(), q)


def _all_kinds(rng, rows, classes, dtype):
    """Ordinary rows with, every few rows, one that a list of the first entries cannot answer at once: nearly all classes masked
    with the type's lowest number; half of them equal to the best; high scores in a few places that lie 8192 classes apart, so
    that thousands of them are above what a bound from groups of classes finds; NaN among the scores; no score; a few."""
    x = torch.tensor(rng.normal(size=(rows, classes)).astype(np.float32)).to(TYPES[dtype])
    place = np.arange(classes) % 8192 // 32
    for r in range(0, rows):
        kind = r % 13
        if kind == 1:
            x[r, rng.random(classes) > 1e-3] = torch.finfo(x.dtype).min
        elif kind == 3:
            x[r, rng.random(classes) < 0.5] = 9.0
        elif kind == 5:
            x[r] -= 100.0
            x[r, place < 20] += 100.0
        elif kind == 7:
            x[r, rng.integers(0, classes, 50)] = float("nan")
        elif kind == 9:
            x[r] = float("-inf")
        elif kind == 10:
            x[r] = float("-inf")
            x[r, rng.integers(0, classes, 5)] = 1.0
        elif kind == 12:
            x[r, -3:] = torch.tensor([30.0, 31.0, 32.0])  # in the run that is cut short, where the width has one
    return x


@pytest.mark.parametrize("k", [1, 31, 64, 65])
@pytest.mark.parametrize("classes,dtype", [(65537, "bf16"), (66000, "f16"), (70003, "bf16"), (131072, "bf16"), (131071, "f16")])
def test_top_scores_of_workgroups_that_go_on(classes, dtype, k):
    """More rows of 16 wavefronts than compute units: for k of at most 64 a workgroup goes on to its next rows.  The results are
    those of calls of a few rows, which have a workgroup for each row, and those of the plain form."""
    from loe_speech_recognition_amd import top_scores

    rng = np.random.default_rng(classes + k)
    units = torch.cuda.get_device_properties(0).multi_processor_count
    rows = 2 * units + 77
    base = _all_kinds(rng, 130, classes, dtype)
    buf = torch.full((rows, classes + 3), 7.0, dtype=base.dtype, device="cuda")
    x = buf[:, :classes]
    pick = torch.arange(rows) * 37 % 130                  # a row's predecessors in its workgroup are of other kinds
    x.copy_(base.cuda()[pick.cuda()])
    for t in (1.0, 3.0):
        got = top_scores(x, k, temperature=t, want_rest=True)
        for lo in range(0, 130, 65):
            few = top_scores(base[lo:lo + 65].cuda(), k, temperature=t, want_rest=True)
            for a, b in zip(got, few):
                for r in range(rows):
                    if lo <= pick[r] < lo + 65:
                        assert torch.equal(a[r], b[pick[r] - lo]), (t, r, int(pick[r]) % 13)
        _check_rows_of_top(got, x, range(rows - 26, rows), k, t, dtype)
        only = top_scores(x, k, temperature=t)
        assert only[2] is None and torch.equal(only[0], got[0]) and torch.equal(only[1], got[1])


@pytest.mark.parametrize("classes,dtype", [(600, "bf16"), (1000, "f16"), (3000, "f32"), (9000, "f32"), (9000, "bf16"), (40000, "f32"),
                                           (40000, "f16"), (200000, "f32")])
def test_top_scores_when_the_list_overflows(classes, dtype):
    """Teams of 1, 4, 8 and 16 wavefronts: rows whose list is cleared and filled again, eight times over the same rows."""
    from loe_speech_recognition_amd import top_scores

    rng = np.random.default_rng(classes)
    x = _all_kinds(rng, 39, classes, dtype).cuda()
    for k in (7, 64, 200, 256):
        first = top_scores(x, k, want_rest=True)
        _check_rows_of_top(first, x, range(39), k, 1.0, dtype)
        for _ in range(7):
            for a, b in zip(top_scores(x, k, want_rest=True), first):
                assert torch.equal(a, b)


@pytest.mark.parametrize("classes,dtype", [(129, "f32"), (600, "bf16"), (1000, "f32"), (1024, "f16")])
def test_distill_scores_of_one_wavefront(classes, dtype):
    """A wavefront hands what its list adds up to from one lane to all: entries given several times and lists that end in every
    lane, the same bits as for the row alone, and the loss of the formula."""
    from loe_speech_recognition_amd import distill_scores

    rng = np.random.default_rng(classes)
    rows = 300
    x = torch.tensor(rng.normal(size=(rows, classes)) * 2).to(TYPES[dtype]).cuda()
    for k in (1, 63, 64, 65, 128, 200):
        k = min(k, classes)
        values = torch.tensor(rng.normal(size=(rows, k)), dtype=torch.float32, device="cuda")
        index = torch.tensor(rng.integers(-1, classes, (rows, k)), dtype=torch.int32, device="cuda")
        rest = torch.tensor(rng.normal(size=rows), dtype=torch.float32, device="cuda")
        loss, grad = distill_scores(x, values, index, rest=rest)
        for r in range(0, rows, 23):
            one = distill_scores(x[r:r + 1], values[r:r + 1], index[r:r + 1], rest=rest[r:r + 1])
            assert torch.equal(one[0][0], loss[r]) and torch.equal(one[1][0], grad[r])
            row = x[r].double().cpu().numpy()
            want, _ = R.distill(row, values[r].cpu().numpy(), index[r].cpu().numpy(), rest[r].item(), 1.0)
            # the sum over the others in 32 bits, with the weight of the rest; all else in 64 bits; one rounding at the end
            span = row.max() - row.min()
            assert abs(loss[r].item() - want) <= 2.0 ** -24 * (5 * span + 4 + _chain(classes, dtype) + abs(want)), (r, k)


@pytest.mark.parametrize("classes,dtype", [(600, "f32"), (1000, "bf16"), (9000, "f16"), (50001, "f32"), (131072, "bf16"), (300001, "f32")])
def test_sample_scores_of_rows_with_nan(classes, dtype):
    """A NaN is an absent score, like -infinity: the same draws with one as with the other, for every way in which a row is cut,
    and the draws of the plain form."""
    from loe_speech_recognition_amd import sample_scores

    rng = np.random.default_rng(classes)
    rows = 12
    x = torch.tensor(rng.normal(size=(rows, classes)) * np.where(np.arange(rows) % 2, 0.05, 3.0)[:, None]).to(TYPES[dtype])
    for r in range(rows):
        x[r, rng.integers(0, classes, 1 + r * r)] = float("nan")
    x[0, -1] = x[1, 0] = float("nan")
    clean = torch.where(torch.isnan(x), float("-inf"), x).to(x.dtype)
    u = torch.tensor(rng.random(rows), dtype=torch.float32)
    for t, top_k, top_p, min_p in [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (2.0, 0, 0.3, 0.0), (1.0, 40, 0.9, 0.0), (1.0, 400, 0.9, 0.0),
                                   (1.0, 0, 0.9, 0.5), (1.0, 0, 0.2, 0.001), (50.0, 0, 0.7, 0.0)]:
        index, share = sample_scores(x.cuda(), u.cuda(), t, top_k, top_p, min_p)
        same = sample_scores(clean.cuda(), u.cuda(), t, top_k, top_p, min_p)
        assert torch.equal(index, same[0]) and torch.equal(share, same[1]), (t, top_k, top_p, min_p)
        for r in range(rows):
            i, lp = R.sample(x[r].double().numpy(), float(u[r]), t, top_k, top_p, min_p)
            assert index[r].item() == i and abs(share[r].item() - lp) <= 2.0 ** -24 * abs(lp) + 1e-10, (r, t, top_k, top_p, min_p)


def test_sample_scores_next_to_zero_at_the_lowest_temperatures():
    """Scores and temperatures at the small end of 32 bits, whose quotients are ordinary numbers: what is listed by min_p is cut
    by top_p all the same."""
    rng = np.random.default_rng(2)
    from loe_speech_recognition_amd import sample_scores

    rows, classes = 40, 900
    t = torch.full((rows,), 2e-42, device="cuda")
    x = -torch.tensor(rng.uniform(0.0, 300.0, (rows, classes)) * 2e-42, dtype=torch.float32)
    x[:, 7] = 0.0
    u = torch.tensor(rng.random(rows), dtype=torch.float32)
    for top_p, min_p in ((0.5, 1e-30), (0.9, 0.0), (0.99, 1e-3)):
        index, share = sample_scores(x.cuda(), u.cuda(), t, 0, top_p, min_p)
        for r in range(rows):
            i, lp = R.sample(x[r].double().numpy(), float(u[r]), float(t[r]), 0, top_p, min_p)
            assert index[r].item() == i and abs(share[r].item() - lp) <= 2.0 ** -24 * abs(lp) + 1e-10, (r, top_p, min_p)


@pytest.mark.parametrize("classes,dtype", [(1 << 21, "f32"), (1 << 24, "bf16"), ((1 << 24) - 5, "f16")])
def test_sums_over_rows_that_are_not_kept(classes, dtype):
    """Millions of equal scores, the widest rows: adding them one after the other in 32 bits is off by 2^-12 to one side.  Bounds:
    five roundings of the arguments, the exponentials and their products, eight additions of a run, the list's and the
    team's."""
    from loe_speech_recognition_amd import distill_scores, top_scores

    rng = np.random.default_rng(classes)
    for gap in (2.9, 3.6):
        row = np.full((1, classes), -gap)
        row[0, rng.integers(0, classes, 3000)] = rng.uniform(0.0, 1.0, 3000)
        row[0, -2:] = -gap / 2
        x = torch.tensor(row).to(TYPES[dtype])
        exact = x[0].double().numpy()
        view = x.cuda()
        v, i, q = R.top(exact, 50, 1.0)
        values, index, rest = top_scores(view, 50, want_rest=True)
        assert np.array_equal(index[0].cpu().numpy(), i) and np.array_equal(values[0].double().cpu().numpy(), v)
        error = 2.0 ** -24 * (5 * (gap + 1) + 8 + 8 + 8 + 6 + 16 + 4)
        assert abs(rest[0].item() - q) <= error + 2.0 ** -24 * 4 * (2 * abs(q) + 1), (gap, rest[0].item(), q)
        teacher = values.flip(1).contiguous(), index
        for r in (rest, None):
            loss, grad = distill_scores(view, *teacher, rest=r)
            want, g = R.distill(exact, teacher[0][0].cpu().numpy(), i, None if r is None else r[0].item(), 1.0)
            assert abs(loss[0].item() - want) <= error + 2.0 ** -24 * abs(want), (gap, loss[0].item(), want)
            # a term of the gradient is off by the sum's error, its own exponential's and its rounding, and is no larger than this
            size = np.abs(g) + np.exp(exact - exact.max()) * (1 if r is None else 2) / np.exp(exact - exact.max()).sum()
            step = torch.finfo(TYPES[dtype]).eps / 2
            tiny = 2.0 ** -25 if dtype == "f16" else 0.0
            assert np.all(np.abs(grad[0].double().cpu().numpy() - g) <= (3 * error + step * (1 + 2.0 ** -8)) * size + tiny + 2.0 ** -120)


@pytest.mark.parametrize("classes,dtype", [(300007, "f32"), (300007, "bf16"), (70001, "f16"), (50001, "f32"), (1001, "f16"), (4099, "f32")])
def test_the_last_classes_carry_the_rest(classes, dtype):
    """The run of a row that is cut short holds nearly all of the weight that is not listed: leaving any of it out shows."""
    from loe_speech_recognition_amd import distill_scores, sample_scores, top_scores

    rng = np.random.default_rng(classes)
    x = rng.normal(size=(4, classes)) - 30.0
    x[:, :7] = 20.0 + np.arange(7)
    last = classes % (4 if dtype == "f32" else 8)
    x[:, -last:] = rng.uniform(5.0, 8.0, (4, last))
    x = torch.tensor(x).to(TYPES[dtype])
    values, index, rest = top_scores(x.cuda(), 7, want_rest=True)
    loss, grad = distill_scores(x.cuda(), values - 1.0, index, rest=rest + 3.0)
    index2, share = sample_scores(x.cuda(), torch.full((4,), 1.0 - 2.0 ** -24, device="cuda"), temperature=40.0)
    for r in range(4):
        row = x[r].double().numpy()
        v, i, q = R.top(row, 7, 1.0)
        assert np.array_equal(index[r].cpu().numpy(), i) and abs(rest[r].item() - q) <= 2.0 ** -24 * (5 * 60 + 100) + 2.0 ** -22 * 40
        want, g = R.distill(row, v - 1.0, i, rest[r].item() + 3.0, 1.0)
        assert abs(loss[r].item() - want) <= 2.0 ** -24 * (5 * 60 + 100 + abs(want) + 8 * 40)
        assert index2[r].item() == R.sample(row, 1.0 - 2.0 ** -24, 40.0, 0, 1.0, 0.0)[0]


@pytest.mark.parametrize("classes,dtype", [(11, "f32"), (58, "f32"), (100, "f16"), (300, "f32"), (5000, "bf16"), (20011, "f32"), (150001, "bf16")])
def test_distill_scores_with_a_rest_that_outweighs_the_list(classes, dtype):
    """Entries of the teacher that are far below its best classes, which are in the rest: weights e^rest that 64 bits do not
    hold, next to ordinary rows."""
    from loe_speech_recognition_amd import distill_scores

    rng = np.random.default_rng(classes)
    heavy = np.array([0.5, 16.0, 499.0, 501.0, 709.0, 710.0, 800.0, 1e4, 1e30, 3e38, -np.inf, np.nan, 3.0], np.float32)
    rows, k = len(heavy), 3
    x = torch.tensor(rng.normal(size=(rows, classes)) * 2).to(TYPES[dtype])
    values = torch.tensor(rng.normal(size=(rows, k)), dtype=torch.float32)
    index = torch.tensor(np.stack([rng.permutation(classes)[:k] for _ in range(rows)]), dtype=torch.int32)
    loss, grad = distill_scores(x.cuda(), values.cuda(), index.cuda(), rest=torch.tensor(heavy).cuda(), temperature=2.0)
    for r in range(rows):
        row = x[r].double().numpy()
        rest = -np.inf if np.isnan(heavy[r]) else float(heavy[r])          # a rest that is no number has no weight
        want, g = R.distill(row, values[r].numpy(), index[r].numpy(), rest, 2.0)
        span = (row.max() - row.min()) / 2
        # sum over the others and its exponentials in 32 bits, their errors in units of the loss (temperature^2) and of the
        # gradient's terms (temperature), which are at most 2
        error = 2.0 ** -24 * (5 * span + 8 + 8 + _chain(classes, dtype))
        assert abs(loss[r].item() - want) <= 4 * error + 2.0 ** -24 * abs(want), (heavy[r], loss[r].item(), want)
        step = torch.finfo(TYPES[dtype]).eps / 2
        tiny = 2.0 ** -25 if dtype == "f16" else 0.0
        assert np.all(np.abs(grad[r].double().numpy(force=True) - g) <= 4 * error + step * (1 + 2.0 ** -8) * np.abs(g) + tiny), heavy[r]
