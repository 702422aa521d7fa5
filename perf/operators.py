"""Operators of text generation, measured: rotary positions, the paged key-value cache (writing new rows, copying pages),
attention of one new token over it, and beam search's selection.

With `own` false, `run` computes the plain form in elementary torch operations; with `own` true it calls the framework."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One decoding step of 8 sequences: the packed projection of 16 heads, queries and keys are turned, values pass through.
        dict(name="rotary_decode", op="rotary", batch=8, tokens=1, heads=48, rotary_heads=32, head_dim=128, rotary_dim=128,
             interleaved=False, scaling="none", factor=1.0, far=1024, gradient=False, dtype="bfloat16"),
        # A training step's forward and backward pass over 8 sequences of 1024 tokens.
        dict(name="rotary_train", op="rotary", batch=8, tokens=1024, heads=48, rotary_heads=32, head_dim=128, rotary_dim=128,
             interleaved=False, scaling="none", factor=1.0, far=0, gradient=True, dtype="bfloat16"),
        # A long prompt far behind its start: part of the head, neighbouring pairs, frequencies stretched by ramps, 32 bits.
        dict(name="rotary_far", op="rotary", batch=1, tokens=8191, heads=8, rotary_heads=8, head_dim=64, rotary_dim=48,
             interleaved=True, scaling="yarn", factor=16.0, far=1000000, gradient=False, dtype="float32"),
        # One decoding step of 64 sequences: a row of keys and of values for each head into its page.
        dict(name="append_decode", op="append", batch=64, tokens=1, heads=16, head_dim=128, page=16, history=4000, dtype="bfloat16"),
        # Prompts of different lengths, padded to one batch, into fresh pages.
        dict(name="append_prompts", op="append", batch=8, tokens=1024, heads=16, head_dim=128, page=16, history=0, dtype="bfloat16"),
        # Beams that part: the unfinished page of each is copied, through all layers of a small model.
        dict(name="copy_fork", op="copy", layers=8, pages=160, moves=8, heads=8, head_dim=64, page=16, dtype="float16"),
        # Compaction of a half empty cache of a model of 24 layers.
        dict(name="copy_compact", op="copy", layers=24, pages=512, moves=192, heads=16, head_dim=128, page=16, dtype="bfloat16"),
        # One short chat: latency is all there is.
        dict(name="attention_one", op="attention", batch=1, heads=16, kv_heads=16, head_dim=128, page=16, length=333, ragged=False,
             dtype="bfloat16"),
        # A served batch of sequences of every length, four query heads to a key head.
        dict(name="attention_batch", op="attention", batch=32, heads=32, kv_heads=8, head_dim=128, page=16, length=4096, ragged=True,
             dtype="bfloat16"),
        # One long document.
        dict(name="attention_long", op="attention", batch=1, heads=32, kv_heads=8, head_dim=128, page=64, length=131072, ragged=False,
             dtype="bfloat16"),
        # One translated sentence.
        dict(name="beam_one", op="beam", batch=1, beams=4, vocab=8192, done=0, dtype="float32"),
        # A batch of sentences, a large odd vocabulary, every fifth beam at its end.
        dict(name="beam_batch", op="beam", batch=64, beams=8, vocab=100003, done=5, dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "append", "copy", "attention", "attention", "attention", "beam", "beam"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "rotary":
        dim = rng.choice([32, 40, 64, 80, 96, 128, 256])
        heads = rng.randint(1, 40)
        rows = _log(rng, 1, max(1, 8192 * 48 * 128 // (heads * dim * BYTES[dtype] // 2)))
        batch = min(rows, _log(rng, 1, 64))
        part = rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 2 * (dim // 16)])
        return dict(op="rotary", batch=batch, tokens=max(1, rows // batch), heads=heads, rotary_heads=rng.choice([heads, heads, -(-2 * heads // 3)]),
                    head_dim=dim, rotary_dim=part, interleaved=rng.random() < 0.4, scaling=rng.choice(["none", "none", "linear", "ntk", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 8.0, 32.0]), far=rng.choice([0, 0, 5000, 300000]), gradient=rng.random() < 0.4, dtype=dtype)
    if kind == "append":
        dim, heads = rng.choice([64, 80, 128]), rng.randint(1, 16)
        rows = _log(rng, 1, 8192 * 2 // BYTES[dtype])
        batch = min(rows, _log(rng, 1, 128))
        return dict(op="append", batch=batch, tokens=max(1, rows // batch), heads=heads, head_dim=dim, page=rng.choice([8, 16, 32, 64]),
                    history=rng.choice([0, 100, 1000]), dtype=dtype)
    if kind == "copy":
        layers, heads, dim, page = rng.randint(1, 24), rng.randint(1, 16), rng.choice([64, 80, 128]), rng.choice([8, 16, 32])
        moves = _log(rng, 1, min(2000, max(1, 24 * 192 * 16 * 128 * 16 * 2 // (layers * heads * dim * page * BYTES[dtype]))))
        return dict(op="copy", layers=layers, pages=2 * moves + rng.randint(0, moves), moves=moves, heads=heads, head_dim=dim, page=page, dtype=dtype)
    if kind == "attention":
        dim, kv, group = rng.choice([64, 64, 80, 128, 128]), rng.randint(1, 16), rng.choice([1, 1, 2, 4, 5, 8])
        most = 130000 * 8 * 128 // (kv * dim * BYTES[dtype] // 2)
        length = _log(rng, 1, min(most, 131072))
        batch = _log(rng, 1, max(1, min(128, most // length)))
        return dict(op="attention", batch=batch, heads=kv * group, kv_heads=kv, head_dim=dim, page=rng.choice([8, 16, 32, 64]), length=length,
                    ragged=rng.random() < 0.7, dtype=dtype)
    beams, vocab = rng.randint(1, 16), _log(rng, 257, 150000)
    return dict(op="beam", batch=_log(rng, 1, max(1, min(256, 64 * 8 * 100003 // (beams * vocab * BYTES[dtype] // 2)))), beams=beams, vocab=vocab,
                done=rng.choice([0, 0, 2, 5]), dtype=dtype)


# --------------------------------------------------------- sizes that a case settles
def _lengths(batch, most, ragged):
    """Between 1 and `most` tokens, the first sequence the longest; without `ragged` all are."""
    return [most if i == 0 or not ragged else 1 + int((i * GOLDEN) % 1.0 * most) for i in range(batch)]


def _append_sizes(c):
    starts = [0 if c["history"] == 0 else int(((i + 1) * GOLDEN) % 1.0 * c["history"]) for i in range(c["batch"])]
    return starts, _lengths(c["batch"], c["tokens"], c["tokens"] > 1)


def work(case):
    c, size = case, BYTES[case["dtype"]]
    if c["op"] == "rotary":
        values = c["batch"] * c["tokens"] * c["heads"] * c["head_dim"]
        ways = 2 if c["gradient"] else 1
        turned = c["batch"] * c["tokens"] * c["rotary_heads"] * c["rotary_dim"]
        return {"bytes": ways * 2 * values * size + c["batch"] * c["tokens"] * 4, "flops": ways * 3 * turned}
    if c["op"] == "append":
        rows = sum(_append_sizes(c)[1])
        return {"bytes": 2 * 2 * rows * c["heads"] * c["head_dim"] * size, "flops": 0}
    if c["op"] == "copy":
        return {"bytes": 2 * 2 * c["layers"] * c["moves"] * c["heads"] * c["page"] * c["head_dim"] * size, "flops": 0}
    if c["op"] == "attention":
        tokens = sum(_lengths(c["batch"], c["length"], c["ragged"]))
        return {"bytes": (2 * tokens * c["kv_heads"] + 2 * c["batch"] * c["heads"]) * c["head_dim"] * size + 4 * (-(-tokens // c["page"]) + c["batch"]),
                "flops": 4 * tokens * c["heads"] * c["head_dim"]}
    rows = c["batch"] * c["beams"]
    alive = rows - (-(-rows // c["done"]) if c["done"] else 0)
    return {"bytes": alive * c["vocab"] * size + rows * (4 + 1 + 4 + 8 + 8 + 1), "flops": 4 * alive * c["vocab"]}


# ------------------------------------------------------------------- the inputs
def _table(lengths, page, gen):
    """Pages in random order: (table [batch, most pages], how many pages there are)."""
    need = torch.tensor([-(-n // page) for n in lengths])
    most, total = int(need.max()), int(need.sum())
    order = torch.randperm(total + 3, generator=gen, device="cuda")[:total].int()
    cell = torch.arange(most)[None, :]
    slot = torch.where(cell < need[:, None], (need.cumsum(0) - need)[:, None] + cell, 0)
    return order[slot.cuda()].contiguous(), total + 3


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = {"case": c}
    if c["op"] == "rotary":
        s["x"] = normal(c["batch"], c["tokens"], c["heads"], c["head_dim"])
        first = torch.randint(0, c["far"] + 1, (c["batch"], 1), generator=gen, device="cuda")
        s["positions"] = (first + torch.arange(c["tokens"], device="cuda")).int()
        if c["gradient"]:
            s["dy"] = normal(c["batch"], c["tokens"], c["heads"], c["head_dim"])
    elif c["op"] == "append":
        starts, counts = _append_sizes(c)
        s["table"], pages = _table([a + b for a, b in zip(starts, counts)], c["page"], gen)
        s["qkv"] = normal(c["batch"], c["tokens"], 3 * c["heads"], c["head_dim"])
        s["k_pages"], s["v_pages"] = (normal(pages, c["heads"], c["page"], c["head_dim"]) for _ in range(2))
        s["starts"], s["counts"] = whole(starts), whole(counts)
    elif c["op"] == "copy":
        s["pages"] = normal(2 * c["layers"], c["pages"], c["heads"], c["page"], c["head_dim"])
        order = torch.randperm(c["pages"], generator=gen, device="cuda")
        # The lists live on the host, as the cache's own bookkeeping has them.
        s["sources"], s["destinations"] = order[: c["moves"]].tolist(), order[c["moves"]: 2 * c["moves"]].tolist()
    elif c["op"] == "attention":
        lengths = _lengths(c["batch"], c["length"], c["ragged"])
        lengths = [lengths[i] for i in torch.randperm(c["batch"], generator=gen, device="cuda").tolist()]
        s["table"], pages = _table(lengths, c["page"], gen)
        s["lengths"] = whole(lengths)
        s["q"] = normal(c["batch"], c["heads"], c["head_dim"])
        s["k_pages"], s["v_pages"] = (normal(pages, c["kv_heads"], c["page"], c["head_dim"]) for _ in range(2))
    else:
        rows = torch.arange(c["batch"] * c["beams"], device="cuda").view(c["batch"], c["beams"])
        # A language model's scores: a wide spread, a few tokens far ahead.
        x = torch.randn(c["batch"], c["beams"], c["vocab"], generator=gen, device="cuda") * 2.5
        x += torch.rand(c["batch"], c["beams"], c["vocab"], generator=gen, device="cuda").pow(40) * 9
        s["logits"] = x.to(dtype)
        s["scores"] = -torch.rand(c["batch"], c["beams"], generator=gen, device="cuda") * 6 - 2
        s["done"] = rows % c["done"] == 0 if c["done"] else torch.zeros_like(rows, dtype=torch.bool)
    if own:
        _hand_over(s)
    return s


def _torch(t):
    """The framework's tensor, seen by torch without a copy."""
    kind = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4", "int64": "<i8", "bool": "|b1"}[t.dtype]
    v = torch.as_tensor(_Seen(t, kind), device="cuda")
    return v.view(torch.bfloat16) if t.dtype == "bfloat16" else v


class _Seen:
    def __init__(self, t, kind):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": kind, "data": (t._data_ptr, False), "version": 3, "strides": None}


def _hand_over(s):
    """A program on the framework has the same values in the framework's own tensors."""
    from orthon_b200 import _C

    for name, t in list(s.items()):
        if isinstance(t, torch.Tensor):
            o = _C._empty_on(list(t.shape), str(t.dtype).replace("torch.", ""), "cuda:0")
            s["torch_" + name] = _torch(o)
            s["torch_" + name].copy_(t)
            s[name] = o
    torch.cuda.synchronize()  # torch wrote on its stream, the framework reads on its own


# ------------------------------------------------------------------ the passes
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _frequencies(c, device):
    """Turns per position of each pair, in 64 bits, and the factor on the turned values."""
    dim, base, factor = c["rotary_dim"], 10000.0, c["factor"]
    if c["scaling"] == "ntk":
        base = base * factor ** (dim / (dim - 2))
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    f = base ** (-2 * i / dim)
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] != "yarn":
        return f, 1.0
    low, high = (dim * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1


def _scaling(c):
    if c["scaling"] == "none":
        return None
    return {"type": c["scaling"], "factor": c["factor"], **({"original_length": 4096} if c["scaling"] == "yarn" else {})}


def _turn(c, x, positions, sign):
    f, factor = _frequencies(c, x.device)
    angle = positions.double()[..., None] * f
    cos, sin = ((t * factor).float()[:, :, None, :] for t in (angle.cos(), angle.sin() * sign))
    y = x.float()
    part = y[:, :, : c["rotary_heads"], : c["rotary_dim"]]
    a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else part.chunk(2, -1)
    p, q = a * cos - b * sin, b * cos + a * sin
    new = torch.stack((p, q), -1).flatten(-2) if c["interleaved"] else torch.cat((p, q), -1)
    y = y.clone()
    y[:, :, : c["rotary_heads"], : c["rotary_dim"]] = new
    return y.to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    y = _turn(c, s["x"], s["positions"], 1.0)
    return {"y": y, "dx": _turn(c, s["dy"], s["positions"], -1.0)} if c["gradient"] else {"y": y}


def _plain_append(s):
    c = s["case"]
    step = torch.arange(c["tokens"], device="cuda")
    b, t = (step[None, :] < s["counts"][:, None]).nonzero(as_tuple=True)
    at = (s["starts"][b] + t).long()
    page = s["table"][b, at // c["page"]].long()
    for pages, first in ((s["k_pages"], c["heads"]), (s["v_pages"], 2 * c["heads"])):
        pages[page, :, at % c["page"]] = s["qkv"][b, t, first: first + c["heads"]]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_copy(s):
    source, destination = (torch.tensor(s[n], device="cuda") for n in ("sources", "destinations"))
    s["pages"][:, destination] = s["pages"][:, source]
    return s["pages"]


def _plain_attention(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]

    def dense(pages):  # [batch, kv heads, tokens, head_dim]
        return pages[s["table"].long()].transpose(1, 2).flatten(2, 3).float()

    q = s["q"].float().view(c["batch"], c["kv_heads"], group, c["head_dim"])
    k, v = dense(s["k_pages"]), dense(s["v_pages"])
    scores = q @ k.transpose(-1, -2) / math.sqrt(c["head_dim"])
    hidden = torch.arange(k.shape[2], device="cuda") >= s["lengths"][:, None]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (p / p.sum(-1, keepdim=True)) @ v
    return out.view(c["batch"], c["heads"], c["head_dim"]).to(s["q"].dtype)


def _candidates(c, logits, scores, done):
    """All candidates' scores, in 64 bits: they decide what is chosen."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    x = scores.double()[..., None] + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    ended = torch.full((c["vocab"],), -math.inf, dtype=torch.float64, device=x.device)
    ended = torch.where(torch.arange(c["vocab"], device=x.device) == c["vocab"] - 1, scores.double()[..., None], ended)
    return torch.where(done[..., None], ended, x).flatten(1)


def _plain_beam(s):
    c = s["case"]
    x = _candidates(c, s["logits"], s["scores"], s["done"])
    last = x.topk(c["beams"]).values[:, -1:]
    above, even = x > last, x == last
    take = above | (even & (even.cumsum(1) <= c["beams"] - above.sum(1, keepdim=True)))
    n = x.shape[1]
    at = n - torch.where(take, n - torch.arange(n, device=x.device), 0).topk(c["beams"]).values  # lowest first
    best, order = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    parents, tokens = at // c["vocab"], at % c["vocab"]
    return {"scores": best.float(), "parents": parents, "tokens": tokens, "done": s["done"].gather(1, parents) | (tokens == c["vocab"] - 1)}


def _own_rotary(s):
    import orthon_b200 as ob

    c = s["case"]

    def turn(x, back):
        return _torch(ob.rotary_embedding(x, s["positions"], rotary_dim=c["rotary_dim"], rotary_heads=c["rotary_heads"],
                                          interleaved=c["interleaved"], scaling=_scaling(c), transposed=back))

    return {"y": turn(s["x"], False), "dx": turn(s["dy"], True)} if c["gradient"] else {"y": turn(s["x"], False)}


def _own_append(s):
    import orthon_b200 as ob

    h = s["case"]["heads"]
    ob.paged_append_(s["k_pages"], s["v_pages"], s["qkv"].slice(2, h, 2 * h), s["qkv"].slice(2, 2 * h, 3 * h), s["table"], s["starts"], s["counts"])
    return {"k": s["torch_k_pages"], "v": s["torch_v_pages"]}


def _own_copy(s):
    import orthon_b200 as ob

    ob.copy_pages_(s["pages"], s["sources"], s["destinations"], dim=1)
    return s["torch_pages"]


def _own_attention(s):
    import orthon_b200 as ob

    return _torch(ob.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"]))


def _own_beam(s):
    import orthon_b200 as ob

    scores, parents, tokens, done = ob.beam_search_step(s["logits"], s["scores"], s["done"], eos_token=s["case"]["vocab"] - 1)
    return {"scores": _torch(scores), "parents": _torch(parents), "tokens": _torch(tokens), "done": _torch(done)}


_plain = {"rotary": _plain_rotary, "append": _plain_append, "copy": _plain_copy, "attention": _plain_attention, "beam": _plain_beam}
_own = {"rotary": _own_rotary, "append": _own_append, "copy": _own_copy, "attention": _own_attention, "beam": _own_beam}


# ------------------------------------------------------- the definitions in 64 bits
def _exact_frequencies(c):
    """Pair by pair, from its wavelength."""
    dim, stretch = c["rotary_dim"], c["factor"]
    base = 10000.0 * (stretch ** (dim / (dim - 2)) if c["scaling"] == "ntk" else 1.0)
    waves = [2 * math.pi * math.exp(math.log(base) * 2 * i / dim) for i in range(dim // 2)]
    if c["scaling"] == "linear":
        waves = [w * stretch for w in waves]
    if c["scaling"] != "yarn":
        return [2 * math.pi / w for w in waves], 1.0
    # The pair that turns 32 times over the original 4096 positions, and the one that turns once: between them the stretch sets in.
    first, last = (dim / 2 * math.log(4096 / turns / (2 * math.pi), base) for turns in (32, 1))
    first, last = max(0, math.floor(first)), min(dim - 1, math.ceil(last))
    share = [min(1.0, max(0.0, (i - first) / max(0.001, last - first))) for i in range(dim // 2)]
    return [2 * math.pi * ((1 - r) / w + r / (w * stretch)) for r, w in zip(share, waves)], 1 + math.log(stretch) / 10


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":  # a pair is a complex number, a turn the product with another
        f, factor = _exact_frequencies(c)
        angle = s["positions"].double()[:, :, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda")

        def turned(x, sign):
            x = x.double()
            h, d = c["rotary_heads"], c["rotary_dim"]
            part = x[:, :, :h, :d].unflatten(-1, (d // 2, 2) if c["interleaved"] else (2, d // 2))
            part = part if c["interleaved"] else part.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * torch.polar(torch.full_like(angle, factor), sign * angle))
            z = z if c["interleaved"] else z.transpose(-1, -2)
            return torch.cat((torch.cat((z.flatten(-2), x[:, :, :h, d:]), -1), x[:, :, h:]), 2)

        return {"y": turned(s["x"], 1), "dx": turned(s["dy"], -1)} if c["gradient"] else {"y": turned(s["x"], 1)}
    if c["op"] == "append":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        h, rows, table = c["heads"], s["qkv"].double(), s["table"].tolist()
        for b, (start, count) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
            t = 0
            while t < count:  # as far as the page goes
                slot = (start + t) % c["page"]
                n, page = min(c["page"] - slot, count - t), table[b][(start + t) // c["page"]]
                k[page, :, slot: slot + n] = rows[b, t: t + n, h: 2 * h].transpose(0, 1)
                v[page, :, slot: slot + n] = rows[b, t: t + n, 2 * h:].transpose(0, 1)
                t += n
        return {"k": k, "v": v}
    if c["op"] == "copy":
        pages = s["pages"].double()
        for a, b in zip(s["sources"], s["destinations"]):
            pages[:, b] = pages[:, a]
        return pages
    if c["op"] == "attention":
        out = torch.empty(c["batch"], c["heads"], c["head_dim"], dtype=torch.float64, device="cuda")
        group = c["heads"] // c["kv_heads"]
        for b, n in enumerate(s["lengths"].tolist()):
            pages = s["table"][b, : -(-n // c["page"])].long()
            for h in range(c["kv_heads"]):
                k, v = (s[name][pages, h].double().flatten(0, 1)[:n] for name in ("k_pages", "v_pages"))
                w = torch.softmax(s["q"][b, h * group: (h + 1) * group].double() @ k.T * c["head_dim"] ** -0.5, -1)
                out[b, h * group: (h + 1) * group] = w @ v
        return out
    logp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    logp[s["done"]] = -math.inf
    logp[..., -1] = torch.where(s["done"], s["scores"].double(), logp[..., -1])
    best, at = logp.flatten(1).sort(dim=1, descending=True, stable=True)
    best, at = best[:, : c["beams"]], at[:, : c["beams"]]
    parents, tokens = at // c["vocab"], at % c["vocab"]
    return {"scores": best, "parents": parents, "tokens": tokens, "done": s["done"].gather(1, parents) | (tokens == c["vocab"] - 1)}
