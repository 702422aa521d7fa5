"""Generation: the page bookkeeping of PagedKVCache, and CausalLM's prompts, decoding steps, greedy and beam search against
the full forward pass over the whole sequence.

Tolerance of logits in float32: two ways of computing the same sums, each within the usual sqrt(n) 2^-24 of its size; over two
blocks of width 64 the logits (size 1) agree to 2^-24 * 64 * 4 * 4 < 1e-4.  In bfloat16 every one of about 12 stored
intermediates is rounded by 2^-8 of its size on either side: 2 * sqrt(12) * 2^-8 < 3e-2 of the logits' size, 4 times that for
the largest of thousands."""
import numpy as np
import pytest

import orthon_b200 as ob
from orthon_b200 import _C, nn
from orthon_b200.models import CausalLM, CausalLMConfig

DEVICES = [pytest.param("cpu", "float32"), pytest.param("cuda:0", "float32", marks=pytest.mark.gpu)]
ROTARY = dict(positions="rotary", rotary_dim=12, rotary_interleaved=True, rotary_scaling={"type": "yarn", "factor": 4.0, "original_length": 16})


def build(device="cpu", dtype="float32", seed=0, **more):
    cfg = CausalLMConfig(vocab_size=97, d_model=64, n_layers=2, n_heads=4, d_ff=128, max_seq=64, init_std=0.3, **more)
    ob.manual_seed(seed)
    model = CausalLM(cfg)
    if dtype != "float32":
        model.cast(dtype)
    return model if device == "cpu" else model.to(device)


def whole(a, device):
    t = _C.from_numpy(np.asarray(a, dtype=np.int64))
    return t if device == "cpu" else t.to(device)


def full_logits(model, sequence, device):
    """Logits behind every token of one sequence, by the training forward pass."""
    with ob.no_grad():
        return model(whole([sequence], device)).to("cpu").cast("float32").numpy().astype(np.float64)


# ------------------------------------------------------------------ bookkeeping
def check_cache(cache):
    count = [0] * cache.num_pages
    for pages in cache._pages.values():
        assert len(set(pages)) == len(pages)
        for p in pages:
            count[p] += 1
    assert count == cache._owners
    assert sorted(cache._free) == [p for p, n in enumerate(count) if n == 0]
    for s, pages in cache._pages.items():
        assert len(pages) * cache.page_size >= cache._lengths[s]


class Mirror:
    """What a cache holds, as plain lists of rows; every token writes its own number."""

    def __init__(self, device, dtype="float32", pages=40, page_size=4):
        self.cache = nn.PagedKVCache(2, 3, 8, pages, page_size, dtype=dtype, device=device)
        self.rows, self.device, self.dtype, self.number = {}, device, dtype, 0

    def grow(self, sequences, counts):
        starts = self.cache.extend(sequences, counts)
        T = max(counts)
        values = np.zeros((len(sequences), T, 3, 8), dtype=np.float32)
        for b, (s, n) in enumerate(zip(sequences, counts)):
            for t in range(n):
                self.number += 1
                values[b, t] = self.number % 200 + np.arange(3)[:, None] * 0.25
                self.rows[s].append(values[b, t].copy())
        k = _C.from_numpy(values, self.dtype).to(self.device)
        v = _C.from_numpy(-values, self.dtype).to(self.device)
        for layer in range(2):
            self.cache.append(layer, k, v, self.cache.table(sequences), self.cache._whole(starts), self.cache._whole(counts))

    def check(self):
        check_cache(self.cache)
        pool = self.cache.pool.to("cpu").cast("float32").numpy()
        for s, rows in self.rows.items():
            assert self.cache.length(s) == len(rows)
            for j, row in enumerate(rows):
                page, slot = self.cache.pages(s)[j // self.cache.page_size], j % self.cache.page_size
                for layer in range(2):
                    assert np.array_equal(pool[2 * layer, page, :, slot], row) and np.array_equal(pool[2 * layer + 1, page, :, slot], -row)


@pytest.mark.parametrize("device,dtype", DEVICES + [pytest.param("cuda:0", "bfloat16", marks=pytest.mark.gpu)])
def test_cache_operations_keep_every_sequence(device, dtype):
    m = Mirror(device, dtype)
    c, rng = m.cache, np.random.default_rng(0)
    for _ in range(3):
        m.rows[c.add()] = []
    m.grow([0, 1, 2], [5, 0, 8])
    m.check()
    m.rows[c.fork(0)] = list(m.rows[0])       # sequence 3 shares a page that is not full
    assert c.pages(3) == c.pages(0)
    m.grow([0, 3], [1, 2])                      # both grow: one of them has to copy it
    assert c.pages(3)[0] == c.pages(0)[0] and c.pages(3)[1] != c.pages(0)[1]
    m.check()
    m.rows[c.fork(2)] = list(m.rows[2])       # full pages only: nothing to copy
    free = c.free_pages
    m.grow([2, 4], [1, 1])
    assert free - c.free_pages == 2
    m.check()
    for step in range(30):
        alive = sorted(m.rows)
        kind = rng.integers(0, 4)
        if kind == 0 and len(alive) < 7:
            s = int(rng.choice(alive))
            m.rows[c.fork(s)] = list(m.rows[s])
        elif kind == 1 and len(alive) > 2:
            s = int(rng.choice(alive))
            c.free(s)
            del m.rows[s]
        elif kind == 2:
            c.compact()
            used = {p for s in m.rows for p in c.pages(s)}
            assert used == set(range(len(used)))
        else:
            some = [int(s) for s in rng.permutation(alive)[:3]]
            try:
                m.grow(some, [int(n) for n in rng.integers(0, 4, len(some))] if step % 2 else [1] * len(some))
            except ValueError:
                pass
        m.check()
    some = sorted(m.rows)[:3]
    parents = [1, 1, 0]
    old = [list(m.rows[s]) for s in some]
    new = c.reorder(some, parents)
    for s in some:
        del m.rows[s]
    for s, p in zip(new, parents):
        m.rows[s] = list(old[p])
    m.check()
    m.grow(new, [1, 1, 1])
    m.check()
    for s in list(m.rows):
        c.free(s)
        del m.rows[s]
    assert c.free_pages == c.num_pages and c.compact() == 0


def test_a_full_cache_refuses_and_stays_as_it_was():
    c = nn.PagedKVCache(1, 1, 4, 4, page_size=2)
    a, b = c.add(), c.add()
    c.extend([a, b], [3, 2])
    f = c.fork(a)
    before = c.pages(a), c.pages(b), c.pages(f), c.free_pages
    with pytest.raises(RuntimeError, match="out of pages"):
        c.extend([a, b], [1, 1])                    # a's shared page is copied, b needs a new one: one is free
    assert before == (c.pages(a), c.pages(b), c.pages(f), c.free_pages) and c.length(a) == 3 and c.length(b) == 2
    c.extend([a, f], 1)                             # one of the two takes a copy, the other keeps the page
    assert c.free_pages == 0 and c.pages(a)[1] != c.pages(f)[1]
    for bad in (lambda: c.extend([a, a], 1), lambda: c.extend([a], [1, 2]), lambda: c.extend([a], [-1]), lambda: c.reorder([a, a], [0, 1]),
                lambda: nn.PagedKVCache(1, 1, 4, 0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.length(99), lambda: c.fork(99), lambda: c.free(99), lambda: c.extend([99], 1), lambda: c.table([99])):
        with pytest.raises(KeyError):
            bad()
    c.free(a)
    with pytest.raises(KeyError):
        c.free(a)


# ------------------------------------------------------------------------ model
@pytest.mark.parametrize("device,dtype", DEVICES + [pytest.param("cuda:0", "bfloat16", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("more", [{}, ROTARY, dict(positions="rotary", rotary_base=500.0)])
def test_prompts_and_steps_give_the_full_pass_logits(device, dtype, more):
    model = build(device, dtype, **more)
    rng = np.random.default_rng(1)
    texts = [list(rng.integers(0, 97, n)) for n in (19, 1, 8)]
    tol = 1e-4 if dtype == "float32" else 4 * 3e-2
    cache = model.new_cache(40, page_size=4)
    sequences = [cache.add() for _ in texts]
    starts = [11, 1, 4]
    ids = np.zeros((3, 12), dtype=np.int64)
    for row, text, n in zip(ids, texts, starts):
        row[:n] = text[:n]
    got = model.prefill(whole(ids, device), cache, sequences, starts)
    want = [full_logits(model, t, device) for t in texts]
    size = max(abs(w).max() for w in want)

    def check(got, places):
        got = got.to("cpu").cast("float32").numpy()
        for row, w, n in zip(got, want, places):
            assert abs(row - w[n - 1]).max() <= tol * size

    check(got, starts)
    # The sequences go on one by one and together; in between one is forked and pages move.
    got = model.decode(whole([texts[0][11]], device), cache, sequences[:1])
    assert abs(got.to("cpu").cast("float32").numpy()[0] - want[0][11]).max() <= tol * size
    other = cache.fork(sequences[0])
    cache.compact()
    model.decode(whole([5], device), cache, [other])  # the fork goes its own way
    for i in range(4):
        got = model.decode(whole([texts[0][12 + i], texts[2][4 + i]], device), cache, [sequences[0], sequences[2]])
        check_pair = got.to("cpu").cast("float32").numpy()
        assert abs(check_pair[0] - want[0][12 + i]).max() <= tol * size and abs(check_pair[1] - want[2][4 + i]).max() <= tol * size
        if i == 1:
            cache.free(other)
            cache.compact()
    check_cache(cache)


def greedy_by_full_passes(model, text, steps, eos, device):
    out = []
    for _ in range(steps):
        out.append(int(full_logits(model, text + out, device)[-1].argmax()))
        if out[-1] == eos:
            break
    return out


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("more", [{}, ROTARY])
def test_greedy_generation(device, dtype, more):
    model = build(device, dtype, seed=3, **more)
    rng = np.random.default_rng(2)
    texts = [list(rng.integers(0, 97, n)) for n in (9, 3, 16)]
    ids = np.zeros((3, 16), dtype=np.int64)
    for row, text in zip(ids, texts):
        row[: len(text)] = text
    plain = [greedy_by_full_passes(model, t, 12, None, device) for t in texts]
    assert model.generate(whole(ids, device), 12, lengths=[9, 3, 16], page_size=4) == plain
    eos = plain[0][5]
    want = [greedy_by_full_passes(model, t, 12, eos, device) for t in texts]
    assert model.generate(whole(ids, device), 12, lengths=[9, 3, 16], eos_token=eos) == want
    assert model.generate(whole(ids[2:], device), 1) == [plain[2][:1]]
    assert model.generate(whole(ids, device), 0) == [[], [], []]
    assert all(p.requires_grad and p.grad is None for p in model.parameters())


def beams_by_full_passes(model, text, steps, eos, W, penalty, device):
    """The textbook search over lists, in float64."""
    beams = [(0.0, [], False)]
    for _ in range(steps):
        options = []
        for w, (score, tokens, done) in enumerate(beams):
            if done:
                options.append((score, w, eos, tokens + [eos], True))
                continue
            x = full_logits(model, text + tokens, device)[-1]
            logp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            options += [(score + logp[v], w, v, tokens + [v], v == eos) for v in range(len(x))]
        options.sort(key=lambda o: (-o[0], o[1], o[2]))
        beams = [(o[0], o[3], o[4]) for o in options[:W]]
        if eos is not None and all(b[2] for b in beams):
            break
    cut = [b[1][: b[1].index(eos) + 1] if eos in b[1] else b[1] for b in beams]
    ranks = [b[0] / len(c) ** penalty for b, c in zip(beams, cut)]
    return cut[int(np.argmax(ranks))]


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("W,penalty", [(2, 1.0), (4, 0.0), (5, 2.0)])
def test_beam_search(device, dtype, W, penalty):
    model = build(device, dtype, seed=5, **ROTARY)
    rng = np.random.default_rng(3)
    texts = [list(rng.integers(0, 97, n)) for n in (7, 2)]
    ids = np.zeros((2, 7), dtype=np.int64)
    for row, text in zip(ids, texts):
        row[: len(text)] = text
    plain = [beams_by_full_passes(model, t, 6, None, W, penalty, device) for t in texts]
    assert model.generate(whole(ids, device), 6, lengths=[7, 2], num_beams=W, length_penalty=penalty, page_size=2) == plain
    eos = plain[0][2]
    want = [beams_by_full_passes(model, t, 6, eos, W, penalty, device) for t in texts]
    assert model.generate(whole(ids, device), 6, lengths=[7, 2], num_beams=W, length_penalty=penalty, eos_token=eos, page_size=2) == want


def test_refusals():
    model = build()
    ids = whole(np.zeros((2, 5)), "cpu")
    for bad in (dict(max_new_tokens=-1), dict(max_new_tokens=1, lengths=[5]), dict(max_new_tokens=1, lengths=[5, 0]), dict(max_new_tokens=1, lengths=[6, 1]),
                dict(max_new_tokens=1, num_beams=0), dict(max_new_tokens=1, eos_token=97), dict(max_new_tokens=60)):
        with pytest.raises(ValueError):
            model.generate(ids, **bad)
    cache = model.new_cache(8, page_size=8)
    s = cache.add()
    with pytest.raises(ValueError):
        model.prefill(ids, cache, [s])
    model.prefill(ids.slice(0, 0, 1).contiguous(), cache, [s])
    with pytest.raises(ValueError):
        model.prefill(ids.slice(0, 0, 1).contiguous(), cache, [s])
    cache.extend([s], 59)
    with pytest.raises(ValueError):
        model.decode(whole([1], "cpu"), cache, [s])
    with pytest.raises(ValueError):
        build(positions="other")
    with pytest.raises(ValueError):
        nn.MultiHeadSelfAttention(16, 4, rotary=nn.RotaryEmbedding(8))
    with pytest.raises(TypeError):
        nn.MultiHeadSelfAttention(16, 4, rotary=True)


def test_rotary_model_trains_and_saves_like_any_other(tmp_path):
    model = build(seed=1, **ROTARY)
    assert not any("pos" in k for k in model.state_dict())
    ids, tgt = whole(np.arange(12).reshape(2, 6), "cpu"), whole(np.arange(1, 13).reshape(2, 6), "cpu")
    opt = ob.optim.SGD(model.parameters(), lr=0.01)
    first = model.loss(ids, tgt)
    first.backward()
    grads = {k: p.grad for k, p in model.named_parameters()}
    assert all(g is not None and np.isfinite(g.numpy()).all() for g in grads.values())
    # The gradient against differences of the loss along a direction through the projections.
    w = model.blocks[0].qkv_weight
    d = np.random.default_rng(0).standard_normal(w.shape).astype(np.float32)
    slope = float((grads["blocks.0.qkv_weight"].numpy().astype(np.float64) * d).sum())
    keep, losses = w.numpy().copy(), []
    for sign in (1, -1):
        with ob.no_grad():
            w._copy_data_(_C.from_numpy(keep + sign * 1e-3 * d))
        losses.append(model.loss(ids, tgt).item())
        with ob.no_grad():
            w._copy_data_(_C.from_numpy(keep))
    # Each loss (size 5) is rounded by about 5 * 2^-22; the quotient's own error is of second order in a step of 1e-3.
    assert abs((losses[0] - losses[1]) / 2e-3 - slope) <= 5 * 2.0 ** -22 / 1e-3 + 2e-2 * abs(slope) + 1e-3
    opt.step()
    ob.save_state_dict(model, tmp_path / "m.ckpt")
    again = build(seed=2, **ROTARY)
    ob.load_state_dict(again, tmp_path / "m.ckpt")
    assert again.generate(ids, 3) == model.generate(ids, 3)


def test_attention_module_turns_queries_and_keys():
    ob.manual_seed(0)
    rope = nn.RotaryEmbedding(4, base=50.0)
    m = nn.MultiHeadSelfAttention(16, 2, rotary=rope)
    x = _C.from_numpy(np.random.default_rng(0).standard_normal((2, 5, 16)).astype(np.float32))
    split = lambda t: rope(t.reshape([2, 5, 2, 8])).transpose(1, 2)  # noqa: E731
    y = ob.scaled_dot_product_attention(split(m.q_proj(x)), split(m.k_proj(x)), m.v_proj(x).reshape([2, 5, 2, 8]).transpose(1, 2), is_causal=True)
    want = m.out_proj(y.transpose(1, 2).contiguous().reshape([2, 5, 16]))
    assert np.array_equal(m(x, is_causal=True).numpy(), want.numpy())
    assert sorted(m.state_dict()) == sorted(nn.MultiHeadSelfAttention(16, 2).state_dict())


# ------------------------------------------------------------- calls that are refused
def everything(cache):
    return (dict(cache._lengths), {s: list(p) for s, p in cache._pages.items()}, list(cache._owners), sorted(cache._free))


def raises_and_keeps(cache, call, errors):
    before = everything(cache)
    with pytest.raises(errors):
        call()
    assert everything(cache) == before
    check_cache(cache)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("more", [{}, ROTARY])
def test_a_refused_step_leaves_the_cache_as_it_was(device, more):
    """The next step gives the logits that it gives without the refused ones, bit for bit."""
    model = build(device, **more)
    rng = np.random.default_rng(4)
    ids = rng.integers(0, 97, (2, 8))

    def start():
        cache = model.new_cache(20, page_size=4)
        sequences = [cache.add(), cache.add()]
        model.prefill(whole(ids, device), cache, sequences, [6, 8])
        sequences.append(cache.fork(sequences[0]))  # a shared page that is not full: the step copies it
        return cache, sequences

    cache, sequences = start()
    narrow = nn.PagedKVCache(2, 2, 16, 20, page_size=4, device=device)  # does not fit the model
    few = nn.PagedKVCache(1, 4, 16, 20, page_size=4, device=device)     # its first layer does
    for bad in (whole([1], device), whole([1, 2], device), whole([1, 2, 3, 4], device), whole([[1], [2], [3]], device), whole([[1, 2, 3]], device),
                _C.from_numpy(np.ones(3, np.float32)).to(device), [1, 2, 3], np.array([1, 2, 3])):
        raises_and_keeps(cache, lambda: model.decode(bad, cache, sequences), ValueError)
    raises_and_keeps(cache, lambda: model.decode(whole([1, 200, 3], "cpu"), cache, sequences), IndexError)  # host tokens are checked
    for other, errors in ((narrow, ValueError), (few, IndexError)):
        fresh = [other.add() for _ in range(2)]
        raises_and_keeps(other, lambda: model.prefill(whole(ids, device), other, fresh), errors)
        other.extend(fresh, 3)
        both = fresh + [other.fork(fresh[0])]
        raises_and_keeps(other, lambda: model.decode(whole([1, 2, 3], device), other, both), errors)
    got = model.decode(whole([5, 6, 7], device), cache, sequences).to("cpu").numpy()
    cache, sequences = start()
    assert np.array_equal(got, model.decode(whole([5, 6, 7], device), cache, sequences).to("cpu").numpy())


def test_a_refused_prompt_leaves_its_sequences_empty():
    model = build()
    cache = model.new_cache(6, page_size=4)
    a, b = cache.add(), cache.add()
    outside = np.array([[1, 2, 3], [4, 97, 6]])
    raises_and_keeps(cache, lambda: model.prefill(whole(outside, "cpu"), cache, [a, b]), IndexError)
    raises_and_keeps(cache, lambda: model.prefill(whole([1, 2, 3], "cpu"), cache, [a]), ValueError)
    raises_and_keeps(cache, lambda: model.prefill(_C.from_numpy(np.ones((1, 3), np.float32)), cache, [a]), ValueError)
    raises_and_keeps(cache, lambda: model.prefill(whole(np.ones((2, 16)), "cpu"), cache, [a, b]), RuntimeError)  # out of pages
    assert cache.free_pages == 6
    got = model.prefill(whole(outside % 97, "cpu"), cache, [a, b]).numpy()
    cache = model.new_cache(6, page_size=4)
    assert np.array_equal(got, model.prefill(whole(outside % 97, "cpu"), cache, [cache.add(), cache.add()]).numpy())


def test_an_interrupted_copy_leaves_the_cache_as_it_was(monkeypatch):
    from orthon_b200.nn import kv_cache

    cache = nn.PagedKVCache(1, 1, 4, 8, page_size=4)
    a = cache.add()
    cache.extend([a], 6)
    b = cache.fork(a)

    def fails(*args, **kw):
        raise RuntimeError("no copy")

    monkeypatch.setattr(kv_cache, "copy_pages_", fails)
    raises_and_keeps(cache, lambda: cache.extend([a, b], [5, 1]), RuntimeError)


@pytest.mark.parametrize("bad", [dict(rotary_dim=18), dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_base=1.0), dict(rotary_base=float("nan")),
                                 dict(rotary_scaling={"type": "other", "factor": 2.0}), dict(rotary_scaling={"type": "yarn", "factor": 2.0}),
                                 dict(rotary_dim=2, rotary_scaling={"type": "ntk", "factor": 2.0})])
def test_rotary_settings_are_refused_when_the_model_is_built(bad):
    with pytest.raises(ValueError):
        build(positions="rotary", **bad)
    settings = {k.replace("rotary_", ""): v for k, v in bad.items() if k != "rotary_dim"}
    if bad.get("rotary_dim") != 18:
        with pytest.raises(ValueError):
            nn.RotaryEmbedding(bad.get("rotary_dim", 16), **settings)


def test_a_module_takes_the_sizes_that_the_operator_takes():
    nn.RotaryEmbedding(512)
    with pytest.raises(ValueError):
        nn.RotaryEmbedding(514)


@pytest.mark.parametrize("more", [{}, dict(num_beams=2)])
@pytest.mark.parametrize("page_size", [0, -4])
def test_generation_refuses_pages_without_room(more, page_size):
    with pytest.raises(ValueError, match="page_size"):
        build().generate(whole(np.zeros((2, 3)), "cpu"), 3, page_size=page_size, **more)


@pytest.mark.parametrize("parents", [[0, -1], [2, 0]])
def test_parents_are_places_in_the_list(parents):
    cache = nn.PagedKVCache(1, 1, 4, 4, page_size=2)
    sequences = [cache.add(), cache.add()]
    cache.extend(sequences, [3, 1])
    raises_and_keeps(cache, lambda: cache.reorder(sequences, parents), IndexError)
