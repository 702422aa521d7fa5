"""Beam search's selection against NumPy in float64.

The chosen places have to be equal.  A score is s + (x - lse): its float64 value is off by the float32 sum of exponentials
(each off by 2 units in the last place of its value, rounded differences and the logarithm's own rounding: below 2^-20 of the
sum, so 2^-20 absolute in the logarithm), then rounded to float32."""
import numpy as np
import pytest

import orthon_b200 as ob
from orthon_b200 import _C

DEVICES = [pytest.param("cpu", "float32"), pytest.param("cpu", "float64")] + [
    pytest.param("cuda:0", t, marks=pytest.mark.gpu) for t in ("float32", "float16", "bfloat16")]


def give(a, dtype, device):
    t = _C.from_numpy(np.ascontiguousarray(a), dtype)
    return t if device == "cpu" else t.to(device)


def seen(t):
    t = t.to("cpu")
    return t.numpy() if t.dtype not in ("float16", "bfloat16") else t.cast("float32").numpy()


def select(x, s, done, eos):
    """(scores, parents, tokens, finished) in float64."""
    B, W, V = x.shape
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        lse = top + np.log(np.sort(np.exp(x - top), -1).sum(-1, keepdims=True))  # sorted: beams of the same values tie exactly
        cand = s[..., None] + (x - lse)
        cand[~np.isfinite(lse[..., 0])] = -np.inf
    if done is not None:
        cand[done] = -np.inf
        cand[..., eos] = np.where(done, s, cand[..., eos])
    cand[~np.isfinite(s)] = -np.inf
    cand = cand.reshape(B, W * V)
    at = np.lexsort((np.broadcast_to(np.arange(W * V), cand.shape), -cand), axis=-1)[:, :W]
    parents, tokens = at // V, at % V
    ended = np.zeros((B, W), bool) if done is None else np.take_along_axis(done, parents, 1)
    return np.take_along_axis(cand, at, 1), parents, tokens, ended | (tokens == (-1 if eos is None else eos))


def check(logits, scores, done, eos, dtype, device):
    x = give(logits, dtype, device)
    got = ob.beam_search_step(x, give(scores, "float32", device), None if done is None else give(done, "bool", device), eos_token=eos)
    want = select(seen(x).astype(np.float64), scores.astype(np.float32).astype(np.float64), done, eos)
    assert [t.dtype for t in got] == ["float32", "int64", "int64", "bool"]
    for g, w, name in zip(got[1:], want[1:], ("parents", "tokens", "finished")):
        assert np.array_equal(seen(g), w), name
    finite = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(seen(got[0])), finite)
    assert (abs(seen(got[0])[finite] - want[0][finite]) <= 2.0 ** -20 + abs(want[0][finite]) * 2.0 ** -24).all()


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 4, 2), (3, 4, 257), (2, 1, 1000), (2, 16, 33), (5, 5, 8192), (1, 64, 100), (2, 7, 50021), (1, 3, 70001), (1, 64, 4097)])
def test_selection_matches_the_definition(device, dtype, B, W, V):
    rng = np.random.default_rng(B + W + V)
    logits, scores = rng.standard_normal((B, W, V)) * 3, -rng.random((B, W)) * 5
    check(logits, scores, None, None, dtype, device)
    check(logits, scores, None, V - 1, dtype, device)
    check(logits, scores, rng.random((B, W)) < 0.4, V // 2, dtype, device)
    check(logits, scores, np.ones((B, W), bool), 0, dtype, device)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("V", [3, 300, 9000, 20001])
def test_ties_go_to_the_lowest_place(device, dtype, V):
    rng = np.random.default_rng(V)
    few = rng.integers(0, 3, (2, 6, V)).astype(float)       # hardly any different values
    check(few, np.zeros((2, 6)) - 1.5, None, None, dtype, device)
    same = np.broadcast_to(rng.standard_normal((2, 1, V)), (2, 6, V))  # beams that are alike, rows at every alignment
    check(same, np.zeros((2, 6)), None, None, dtype, device)
    check(np.zeros((2, 6, V)), np.zeros((2, 6)), None, None, dtype, device)


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("V", [5, 1000, 20001])
def test_nothing_to_choose_from(device, dtype, V):
    """-inf, NaN and +inf among logits and scores; fewer candidates than beams."""
    rng = np.random.default_rng(V + 1)
    logits = rng.standard_normal((6, 4, V))
    scores = np.tile([0.0, -np.inf, -np.inf, -np.inf], (6, 1))  # the first step: one beam is alive
    logits[1, 0, 1:] = -np.inf                               # one candidate in all
    logits[2, 0, :] = -np.inf                                # none
    logits[3, 0, V // 2] = np.nan
    logits[4, 0, V - 1] = np.inf
    scores[5] = [np.nan, np.inf, -1.0, -np.inf]
    check(logits, scores, None, 2, dtype, device)
    check(logits, scores, np.tile([False, True, False, True], (6, 1)), 2, dtype, device)
    lowest = np.full((1, 2, V), {"float16": -65504.0}.get(dtype, -3e38))
    lowest[0, 1, V - 1] = 0.0
    check(lowest, np.zeros((1, 2)), None, None, dtype, device)


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_all_of_the_best_in_one_place(device, dtype):
    """The whole selection inside a few neighbouring tokens, and far apart."""
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 8, 30000))
    logits[0, 3, 777:785] += 30
    logits[1, :, 12345] += 20
    logits[2, 7, ::3750] += 25
    logits[3, 0, -40:] += np.arange(40)
    check(logits, np.zeros((4, 8)), None, None, dtype, device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_strided_logits_and_refusals(device):
    rng = np.random.default_rng(3)
    a = rng.standard_normal((3, 2, 50)).astype(np.float32)
    x, s = give(a, "float32", device), give(np.zeros((2, 3)), "float32", device)
    got = ob.beam_search_step(x.transpose(0, 1), s)
    assert np.array_equal(seen(got[2]), select(a.transpose(1, 0, 2).astype(np.float64), np.zeros((2, 3)), None, None)[2])
    z = lambda *n, d="float32": ob.zeros(list(n), d).to(device)  # noqa: E731
    for bad in ((z(2, 50), z(2, 1)), (z(2, 3, 50), z(2, 2)), (z(2, 3, 50), z(6)), (z(2, 3, 50), z(2, 3, d="int32")), (z(1, 65, 4), z(1, 65)), (z(0, 3, 4), z(0, 3))):
        with pytest.raises(ValueError):
            ob.beam_search_step(*bad)
    with pytest.raises(ValueError):
        ob.beam_search_step(z(2, 3, 50), z(2, 3), z(2, 3, d="bool"))
    with pytest.raises(ValueError):
        ob.beam_search_step(z(2, 3, 50), z(2, 3), z(2, 3), eos_token=1)
    for token in (-2, 50):
        with pytest.raises(IndexError):
            ob.beam_search_step(z(2, 3, 50), z(2, 3), eos_token=token)
    with pytest.raises(RuntimeError, match="no_grad"):
        ob.beam_search_step(z(2, 3, 50).requires_grad_(), z(2, 3))
    with pytest.raises(ob.UnsupportedOperation):
        ob.beam_search_step(z(2, 3, 50, d="int32"), z(2, 3))


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("V", [300, 9000, 50021])
def test_the_same_logits_in_another_order(device, dtype, V):
    """Beams whose logits are those of another one in another order, the largest first, last, or anywhere.  The CPU, whose sums
    hardly depend on the order, ties them; CUDA tells them apart by no more than twice the error of a log-sum (2^-20 each)."""
    rng = np.random.default_rng(V)
    rows = np.sort(rng.standard_normal((3, 1, V)) * 3, -1) * np.ones((1, 6, 1))
    rows[:, 1] = rows[:, 1, ::-1]
    for b in range(3):
        for w in (2, 3, 4):
            rows[b, w] = rng.permutation(rows[b, w])
    rows[:, 5] = rows[:, 4]                                       # and one in the same order
    scores = np.zeros((3, 6)) - 1.0
    if device == "cpu":
        check(rows, scores, None, None, dtype, device)
    x = give(rows, dtype, device)
    got = [seen(t) for t in ob.beam_search_step(x, give(scores, "float32", device))]
    values = seen(x).astype(np.float64)
    lse = np.log(np.sort(np.exp(values - values.max(-1, keepdims=True)), -1).sum(-1, keepdims=True)) + values.max(-1, keepdims=True)
    cand = scores[..., None] + (values - lse)
    best = -np.sort(-cand.reshape(3, -1), -1)[:, :6]
    off = 2.0 ** -20 + abs(best) * 2.0 ** -24
    assert (abs(got[0] - best) <= 2 * off).all()
    for b in range(3):
        places = list(zip(got[1][b], got[2][b]))
        assert len(set(places)) == 6
        assert (abs(np.array([cand[b, w, v] for w, v in places]) - got[0][b]) <= off[b]).all()
        tokens = {w: [v for u, v in places if u == w] for w in (4, 5)}
        assert tokens[5] == tokens[4][: len(tokens[5])]           # beam 5 offers what beam 4 does, behind it


@pytest.mark.parametrize("device,dtype", DEVICES)
def test_many_sentences_and_calls_of_different_sizes(device, dtype):
    """Few and many sentences in turn, more than a first call makes room for."""
    rng = np.random.default_rng(11)
    for B, W, V in ((3, 2, 40), (5000, 2, 9), (1, 8, 5000), (4097, 1, 33), (9000, 3, 8), (2, 3, 30001), (5000, 2, 9)):
        check(rng.standard_normal((B, W, V)) * 3, -rng.random((B, W)), rng.random((B, W)) < 0.2, V - 1, dtype, device)


@pytest.mark.gpu
def test_two_threads_at_once():
    import threading

    rng, failed = np.random.default_rng(12), []
    work = [(rng.standard_normal(s) * 3, -rng.random(s[:2])) for s in ((6000, 2, 17), (3, 8, 20001), (64, 4, 999), (12000, 1, 50))]

    def run(logits, scores):
        try:
            for _ in range(5):
                check(logits, scores, None, 3, "float32", "cuda:0")
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=w) for w in work]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_a_negative_end_token_is_refused(device):
    """-1, by which the kernels know that there is none, is no exception."""
    with pytest.raises(IndexError):
        ob.beam_search_step(give(np.zeros((1, 2, 5)), "float32", device), give(np.zeros((1, 2)), "float32", device), eos_token=-1)
