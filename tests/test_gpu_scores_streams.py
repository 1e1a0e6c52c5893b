"""Score-row operators and the engine's own calls on different streams and in different threads."""
import ctypes
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

A_WHILE = 200_000_000              # clock cycles that a stream is kept busy for: tenths of a second


@pytest.fixture(scope="module")
def digits():
    from loe_speech_recognition_amd import MFCC, HiddenMarkovModelInference, ModelCollection, synthetic

    models = synthetic.load_word_models()
    inf = HiddenMarkovModelInference.from_models([models[lab] for lab in synthetic.LOOP_ORDER])
    mc = ModelCollection()
    mc._models = [models[lab] for lab in synthetic.LOOP_ORDER if lab != "S"]
    feats = [MFCC.batch(synthetic.batch(seed, 12, 1)[0], 16000) for seed in (31, 32)]
    return inf, mc, feats


def test_a_call_on_a_side_stream_leaves_the_engines_stream_alone(digits):
    """While one thread is inside an operator's call on a busy side stream, another thread's emission scores are computed on the
    engine's stream, not behind what the side stream does."""
    from loe_speech_recognition_amd import _native

    inf, _, feats = digits
    eng = inf._bind()
    fb = eng.feature_batch(feats[0])
    want = eng.emission(fb)[:fb.total_frames].clone()
    torch.cuda.synchronize()
    side, out = torch.cuda.Stream(), []

    def decode():
        got = eng.emission(fb)[:fb.total_frames]
        eng._stream.synchronize()
        out.append((bool(torch.equal(got, want)), side.query()))

    def inside(ctx, *args):
        thread = threading.Thread(target=decode)
        thread.start()
        thread.join()
        return 0

    with torch.cuda.stream(side):
        torch.cuda._sleep(5 * A_WHILE)                    # well beyond what the other thread needs
        eng.on_current_stream(inside)
    torch.cuda.synchronize()
    assert out == [(True, False)]                         # the scores were there while the side stream was still busy
    assert _native.get_engine() is eng


def test_errors_of_the_two_contexts_are_their_own():
    from loe_speech_recognition_amd import _native

    eng = _native.get_engine()
    p = ctypes.c_void_p(0)
    with pytest.raises(_native.NativeError, match="lsr_emission_batch: null"):
        eng._check(eng.lib.lsr_emission_batch(eng.ctx, p, 1, p))
    with pytest.raises(_native.NativeError, match="lsr_top_scores: unknown element type 9"):
        eng.on_current_stream(eng.lib.lsr_top_scores, p, 9, 1, 1, 1, 1, 1.0, p, p, p)
    assert "lsr_emission_batch" in eng.lib.lsr_last_error(eng.ctx).decode()


def test_times_of_the_operators_kernels():
    from loe_speech_recognition_amd import _native, sample_scores, top_scores

    eng = _native.get_engine()
    x, u = torch.randn((200, 58), device="cuda"), torch.rand(200, device="cuda")
    try:
        eng.profile_reset()
        eng.profile_enable(True, only=("top",))
        for _ in range(3):
            top_scores(x, 4)
        sample_scores(x, u)
        ms, n = eng.profile_get("top")
        assert n == 3 and ms > 0 and eng.profile_get("sample") == (0.0, 0)
    finally:
        eng.profile_enable(False)
        eng.profile_reset()
    assert eng.profile_get("top") == (0.0, 0)


def test_threads_while_another_one_decodes(digits):
    """Four threads with rows on streams of their own, and one that decodes batch after batch: everybody's results are right."""
    from loe_speech_recognition_amd import sample_scores, top_scores

    inf, mc, feats = digits
    want_scores = [mc.scores_batch(f) for f in feats]
    want_words = [inf.predict_batch(f) for f in feats]
    rng = np.random.default_rng(4)
    views = [torch.tensor(rng.normal(size=(50, 700 + 300 * i)), dtype=torch.float32, device="cuda") for i in range(4)]
    u = torch.tensor(rng.random(50), dtype=torch.float32, device="cuda")
    want = [(top_scores(v, 9)[1], sample_scores(v, u, 0.9, 50, 0.95)[0]) for v in views]
    torch.cuda.synchronize()
    wrong, done = [], threading.Event()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            while not done.is_set():
                x = views[i] + 0.0
                got = top_scores(x, 9)[1], sample_scores(x, u, 0.9, 50, 0.95)[0]
                if not all(bool(torch.equal(a, b)) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    try:
        for turn in range(40):
            if not np.array_equal(mc.scores_batch(feats[turn % 2]), want_scores[turn % 2]):
                wrong.append("scores")
            if inf.predict_batch(feats[turn % 2]) != want_words[turn % 2]:
                wrong.append("words")
    finally:
        done.set()
        for t in threads:
            t.join()
    assert not wrong


def test_times_of_calls_on_another_stream():
    """A kernel that is still waiting on a busy side stream when its time is asked for is waited for, and counted."""
    from loe_speech_recognition_amd import _native, top_scores

    eng = _native.get_engine()
    x = torch.randn((200, 58), device="cuda")
    want = top_scores(x, 4)[1].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        eng.profile_reset()
        eng.profile_enable(True)
        with torch.cuda.stream(side):
            torch.cuda._sleep(A_WHILE)
            index = top_scores(x, 4)[1]
        ms, n = eng.profile_get("top")
        assert n == 1 and ms > 0
        side.synchronize()
        assert torch.equal(index, want) and torch.equal(top_scores(x, 4)[1], want)
    finally:
        eng.profile_enable(False)
        eng.profile_reset()


def test_captured_calls_are_not_timed():
    """With timing on, a captured call records no event into its graph: replays leave the times of eager calls alone, and what
    follows works."""
    from loe_speech_recognition_amd import _native, top_scores

    eng = _native.get_engine()
    x = torch.randn((200, 58), device="cuda")
    want = top_scores(x, 4)[1].clone()
    torch.cuda.synchronize()
    try:
        eng.profile_reset()
        eng.profile_enable(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            index = top_scores(x, 4)[1]
        for turn in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(index, want)
            assert torch.equal(top_scores(x, 4)[1], want) and eng.profile_get("top")[1] == turn + 1
    finally:
        eng.profile_enable(False)
        eng.profile_reset()


def test_the_frameworks_rows_on_a_side_stream(digits):
    """The models' own entry points under another stream than the engine's, while the engine's is busy: they wait for what the
    engine computes, and give what they give without all that."""
    inf, mc, feats = digits
    rng = np.random.default_rng(7)
    u = rng.random(len(feats[0])).astype(np.float32)
    fb = inf._bind().feature_batch(feats[0])
    frames = torch.tensor(rng.random(fb.total_frames), dtype=torch.float32, device="cuda")

    def results():
        _, *targets = inf.state_targets(fb, 8, temperature=6.0)
        _, *drawn = inf.sample_states(fb, frames, temperature=6.0, top_p=0.9)
        return mc.nbest_batch(feats[0], 3), mc.sample_batch(feats[0], u, 100.0, top_p=0.9), [*targets, *drawn]

    want = results()
    torch.cuda.synchronize()
    for turn in range(3):
        torch.cuda._sleep(A_WHILE)                        # on the engine's stream
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = results()
            side.synchronize()
        assert got[0] == want[0] and got[1] == want[1]
        assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


def test_rows_are_not_overwritten_under_a_side_stream(digits):
    """Emission scores that an operator on a busy side stream has still to read: the next batch's do not take their place."""
    from loe_speech_recognition_amd import top_scores

    inf, _, feats = digits
    eng = inf._bind()
    batches = [eng.feature_batch(feats[0]), eng.feature_batch(feats[0][::-1])]
    want = [[v.clone() for v in inf.state_targets(fb, 5)[1:]] for fb in batches]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = []
        for turn in range(6):
            scores = eng.emission(batches[turn % 2])
            torch.cuda._sleep(A_WHILE // 10)
            got.append(top_scores(scores[:batches[0].total_frames, :len(inf._multivariate_normals)], 5, want_rest=True))
            del scores
        side.synchronize()
    for turn, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 2])), turn
    torch.cuda.synchronize()


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capturing_the_engines_calls(digits):
    """On the engine's own stream state scores and their targets can be captured together; under another one the capture is
    refused, not left without them."""
    from loe_speech_recognition_amd import _native

    inf, _, feats = digits
    eng = inf._bind()
    fb, other = eng.feature_batch(feats[0]), eng.feature_batch(feats[0][::-1])
    want = [[v.clone() for v in inf.state_targets(b, 5)[1:]] for b in (fb, other)]
    torch.cuda.synchronize()
    before, stream = eng._stream, torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_native.NativeError, match="own stream"):
        with torch.cuda.graph(graph, stream=stream):
            inf.state_targets(fb, 5)
    torch.cuda.synchronize()
    eng.use_stream(stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _, *out = inf.state_targets(fb, 5)
        first = fb.feats.clone()
        for turn in range(4):
            fb.feats.copy_(other.feats if turn % 2 else first)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 2])), turn
    finally:
        eng.use_stream(before)
