"""Decoder-only causal language model: token embeddings, learned or rotary positions, N pre-LayerNorm
blocks (multi-head causal self-attention, GELU MLP), final LayerNorm, linear head.

Each block is six kernel families: LayerNorm, one QKV GEMM (bias in the epilogue), packed-QKV
attention (heads read in place, causal mask applied in the softmax kernel), output projection
with the residual add in the epilogue, LayerNorm, and the MLP as two GEMMs with GELU and the
second residual add in their epilogues.  Weights are N(0, init_std).

Generation keeps the keys and values of all tokens in a `nn.PagedKVCache`: a prompt goes through the training
attention once and leaves its keys and values there, each further token is one pass with attention over the pages.
(reference project: examples/tiny_causal_lm.py:59-112)"""
import math
from dataclasses import dataclass
from typing import Optional

import numpy as np

from .. import _C, nn
from .._random import normal_array
from ..functional import beam_search_step


@dataclass(frozen=True)
class CausalLMConfig:
    vocab_size: int
    d_model: int
    n_layers: int
    n_heads: int
    d_ff: int
    max_seq: int
    init_std: float = 0.02
    eps: float = 1e-5
    positions: str = "learned"          # or "rotary": no position table, no limit by max_seq
    rotary_dim: Optional[int] = None    # values of a head that are turned (default: all)
    rotary_base: float = 10000.0
    rotary_interleaved: bool = False
    rotary_scaling: Optional[dict] = None


TINY_LM = CausalLMConfig(vocab_size=8192, d_model=512, n_layers=8, n_heads=8, d_ff=2048, max_seq=512)
LM_1P3B = CausalLMConfig(vocab_size=32000, d_model=2048, n_layers=24, n_heads=16, d_ff=8192, max_seq=1024)


def _no_grad():
    import orthon_b200 as ob
    return ob.no_grad()


def _whole(values, device):
    t = _C.from_numpy(np.ascontiguousarray(values, dtype=np.int32))
    return t if device == "cpu" else t.to(device)


def _until(tokens, end):
    """The tokens up to the first `end`, which is the last one kept."""
    return tokens[: tokens.index(end) + 1] if end is not None and end in tokens else tokens


def _normal(shape, std):
    return nn.Parameter(_C.from_numpy(normal_array(tuple(shape), std)))


class Block(nn.Module):
    def __init__(self, cfg: CausalLMConfig):
        super().__init__()
        E, F = cfg.d_model, cfg.d_ff
        self.n_heads, self.head_dim = cfg.n_heads, E // cfg.n_heads
        self.rotary = None
        if cfg.positions == "rotary":
            self.rotary = nn.RotaryEmbedding(self.head_dim if cfg.rotary_dim is None else cfg.rotary_dim, base=cfg.rotary_base,
                                             interleaved=cfg.rotary_interleaved, scaling=cfg.rotary_scaling)
            if self.rotary.rotary_dim > self.head_dim:
                raise ValueError(f"rotary_dim {self.rotary.rotary_dim} exceeds the head size {self.head_dim}")
        self.scale = 1.0 / math.sqrt(E // cfg.n_heads)
        self.ln1 = nn.LayerNorm(E, eps=cfg.eps)
        self.qkv_weight, self.qkv_bias = _normal((E, 3 * E), cfg.init_std), nn.Parameter(_C.zeros([3 * E]))
        self.proj_weight, self.proj_bias = _normal((E, E), cfg.init_std), nn.Parameter(_C.zeros([E]))
        self.ln2 = nn.LayerNorm(E, eps=cfg.eps)
        self.fc1_weight, self.fc1_bias = _normal((E, F), cfg.init_std), nn.Parameter(_C.zeros([F]))
        self.fc2_weight, self.fc2_bias = _normal((F, E), cfg.init_std), nn.Parameter(_C.zeros([E]))

    def forward(self, x):
        qkv = _C.linear(self.ln1(x), self.qkv_weight, self.qkv_bias)
        if self.rotary is not None:
            B, T, width = qkv.shape
            qkv = self.rotary(self._heads(qkv), rotary_heads=2 * self.n_heads).reshape([B, T, width])
        a = _C._attention_qkv(qkv, self.n_heads, None, True, self.scale)
        return self._rest(x, a)

    def _heads(self, qkv):
        """[B, T, 3H, D] view of a packed projection: queries, keys, values."""
        return qkv.reshape([qkv.shape[0], qkv.shape[1], 3 * self.n_heads, self.head_dim])

    def _rest(self, x, a):
        x = _C.linear(a, self.proj_weight, self.proj_bias, "none", x)
        h = self.ln2(x)
        return _C._mlp_gelu(h, self.fc1_weight, self.fc1_bias, self.fc2_weight, self.fc2_bias, x)

    def prefill(self, x, cache, layer, table, starts, counts):
        """forward() of prompts [B, T, E] whose keys and values go to the cache; no graph."""
        H = self.n_heads
        qkv = _C.linear(self.ln1(x), self.qkv_weight, self.qkv_bias)
        heads = self._heads(qkv)
        if self.rotary is not None:
            self.rotary.forward_(heads, rotary_heads=2 * H)
        cache.append(layer, heads.slice(2, H, 2 * H), heads.slice(2, 2 * H, 3 * H), table, starts, counts)
        return self._rest(x, _C._attention_qkv(qkv, H, None, True, self.scale))

    def decode(self, x, cache, layer, table, places, lengths):
        """One more token of every sequence, x [B, E], at `places` ([B], int32); `lengths` are places + 1; no graph."""
        B, E = x.shape
        H, D = self.n_heads, self.head_dim
        heads = _C.linear(self.ln1(x), self.qkv_weight, self.qkv_bias).reshape([B, 1, 3 * H, D])
        if self.rotary is not None:
            self.rotary.forward_(heads, places.reshape([B, 1]), rotary_heads=2 * H)
        cache.append(layer, heads.slice(2, H, 2 * H), heads.slice(2, 2 * H, 3 * H), table, places)
        a = cache.attend(layer, heads.reshape([B, 3 * H, D]).slice(1, 0, H), table, lengths, self.scale)
        return self._rest(x, a.reshape([B, E]))


class CausalLM(nn.Module):
    def __init__(self, cfg: CausalLMConfig):
        super().__init__()
        if cfg.positions not in ("learned", "rotary"):
            raise ValueError("positions must be 'learned' or 'rotary'")
        self.cfg = cfg
        self.tok_emb = _normal((cfg.vocab_size, cfg.d_model), cfg.init_std)
        if cfg.positions == "learned":
            self.pos_emb = _normal((cfg.max_seq, cfg.d_model), cfg.init_std)
        self.blocks = nn.Sequential(*[Block(cfg) for _ in range(cfg.n_layers)])
        self.ln_f = nn.LayerNorm(cfg.d_model, eps=cfg.eps)
        self.head_weight = _normal((cfg.d_model, cfg.vocab_size), cfg.init_std)
        if cfg.positions == "learned":
            self.register_buffer("positions", _C.from_numpy(np.arange(cfg.max_seq, dtype=np.int64)), persistent=False)

    def _check_length(self, T):
        if self.cfg.positions == "learned" and T > self.cfg.max_seq:
            raise ValueError(f"sequence length {T} exceeds max_seq {self.cfg.max_seq}")

    @staticmethod
    def _check_tokens(tokens, rank, message):
        if not isinstance(tokens, _C.Tensor) or tokens.ndim != rank or tokens.dtype not in ("int32", "int64"):
            raise ValueError(message)

    def _embed(self, ids):
        x = _C.embedding(ids, self.tok_emb)
        if self.cfg.positions == "rotary":
            return x
        T = ids.shape[1]
        pos = self.positions if T == self.cfg.max_seq else self.positions.slice(0, 0, T).contiguous()
        return x + _C.embedding(pos, self.pos_emb)

    def forward(self, ids):
        """ids: int tensor [B, T] -> logits [B*T, vocab]."""
        B, T = ids.shape
        self._check_length(T)
        x = self._embed(ids)
        x = self.blocks(x)
        x = self.ln_f(x)
        return _C.linear(x.reshape([B * T, self.cfg.d_model]), self.head_weight)

    def loss(self, ids, targets):
        """Mean next-token cross-entropy; `targets` is an int tensor [B, T] (or [B*T])."""
        logits = self.forward(ids)
        flat = targets if targets.ndim == 1 else targets.reshape([-1])
        return _C.cross_entropy(logits, flat)

    # ------------------------------------------------------------ generation
    def new_cache(self, num_pages, page_size=16):
        """An empty `nn.PagedKVCache` that fits this model, on its device and in its type."""
        cfg = self.cfg
        return nn.PagedKVCache(cfg.n_layers, cfg.n_heads, cfg.d_model // cfg.n_heads, num_pages, page_size, dtype=self.tok_emb.dtype,
                               device=str(self.tok_emb.device))

    def prefill(self, ids, cache, sequences, lengths=None):
        """Runs prompts ids [B, T] into empty cache sequences; row b has lengths[b] tokens (default T), padding behind them is
        ignored.  Returns the logits [B, vocab] of each prompt's last token.  A call that raises leaves the sequences empty."""
        self._check_tokens(ids, 2, "prefill: ids must be an int32 or int64 tensor [B, T]")
        B, T = ids.shape
        self._check_length(T)
        lengths = [T] * B if lengths is None else [int(n) for n in lengths]
        if len(lengths) != B or len(sequences) != B or any(not 1 <= n <= T for n in lengths):
            raise ValueError("prefill: one sequence and one length in [1, T] for each prompt")
        if any(cache.length(s) for s in sequences):
            raise ValueError("prefill: the sequences must be empty")
        with _no_grad():
            device = str(self.tok_emb.device)
            _, before = cache._extend(sequences, lengths)
            try:
                return self._prefill(ids, cache, cache.table(sequences), _whole([0] * B, device), _whole(lengths, device), lengths)
            except BaseException:  # rows that were written already lie behind the sequences' ends
                cache._take_back(before)
                raise

    def _prefill(self, ids, cache, table, starts, counts, lengths):
        T, E = ids.shape[1], self.cfg.d_model
        x = self._embed(ids)
        for layer, block in enumerate(self.blocks):
            x = block.prefill(x, cache, layer, table, starts, counts)
        last = _whole([b * T + n - 1 for b, n in enumerate(lengths)], str(x.device))
        return self._logits(_C.embedding(last, x.reshape([-1, E])))

    def _logits(self, x):
        return _C.linear(self.ln_f(x), self.head_weight)

    def decode(self, tokens, cache, sequences):
        """One more token of each sequence (int tensor [B]) into the cache.  Returns the logits [B, vocab] behind it.  A call
        that raises leaves the sequences as they were."""
        self._check_tokens(tokens, 1, "decode: tokens must be an int32 or int64 tensor [B]")
        if tokens.shape[0] != len(sequences):
            raise ValueError(f"decode: {tokens.shape[0]} tokens for {len(sequences)} sequences")
        self._check_length(max([cache.length(s) for s in sequences] + [0]) + 1)
        with _no_grad():
            starts, before = cache._extend(sequences, 1)
            try:
                places = _whole(starts, str(self.tok_emb.device))
                return self._decode(tokens, cache, cache.table(sequences), places, cache.lengths(sequences))
            except BaseException:  # rows that were written already lie behind the sequences' ends
                cache._take_back(before)
                raise

    def _decode(self, tokens, cache, table, places, lengths):
        x = _C.embedding(tokens, self.tok_emb)
        if self.cfg.positions == "learned":
            x = x + _C.embedding(places, self.pos_emb)
        for layer, block in enumerate(self.blocks):
            x = block.decode(x, cache, layer, table, places, lengths)
        return self._logits(x)

    def generate(self, ids, max_new_tokens, lengths=None, eos_token=None, num_beams=1, length_penalty=1.0, page_size=16):
        """Continues prompts ids [B, T] (rows padded behind lengths[b] tokens) by up to `max_new_tokens` tokens each: the most
        likely token at a time, or with ``num_beams`` > 1 the best of a beam search (score / length ** length_penalty).  A
        continuation ends with ``eos_token``.  Returns a list of token lists."""
        B, T = ids.shape
        lengths = [T] * B if lengths is None else [int(n) for n in lengths]
        steps, W = int(max_new_tokens), int(num_beams)
        if len(lengths) != B or any(not 1 <= n <= T for n in lengths):
            raise ValueError("generate: one length in [1, T] for each prompt")
        if steps < 0 or W < 1 or int(page_size) < 1:
            raise ValueError("generate: max_new_tokens must not be negative, num_beams and page_size at least 1")
        if eos_token is not None and not 0 <= int(eos_token) < self.cfg.vocab_size:
            raise ValueError("generate: eos_token is not in the vocabulary")
        self._check_length(max([T] + [n + steps for n in lengths]))
        if steps == 0 or B == 0:
            return [[] for _ in range(B)]
        with _no_grad():
            if W == 1:
                return self._greedy(ids, steps, lengths, eos_token, page_size)
            return self._beams(ids, steps, lengths, eos_token, W, float(length_penalty), page_size)

    def _greedy(self, ids, steps, lengths, eos_token, page_size):
        B, device = len(lengths), str(self.tok_emb.device)
        # All pages are taken at once, so that table and places are on the device before the first step.
        cache = self.new_cache(sum(-(-(n + steps) // page_size) for n in lengths), page_size)
        sequences = [cache.add() for _ in range(B)]
        cache.extend(sequences, [n + steps for n in lengths])
        table = cache.table(sequences)
        places = _whole(np.add.outer(np.arange(steps + 1), np.asarray(lengths)), device)
        logits = self._prefill(ids, cache, table, _whole([0] * B, device), places[0], lengths)
        found = _C._empty_on([steps, B], "int64", device)
        ended, done = np.zeros(B, dtype=bool), 0
        for i in range(steps):
            tokens = logits.argmax(1)
            found._copy_flat_range_from(i * B, tokens, 0, B)
            done = i + 1
            if eos_token is not None:
                ended |= tokens.numpy() == int(eos_token)
                if ended.all():
                    break
            if done < steps:
                logits = self._decode(tokens, cache, table, places[i], places[i + 1])
        columns = found.numpy()[:done].T.tolist()
        return [_until(row, eos_token) for row in columns]

    def _beams(self, ids, steps, lengths, eos_token, W, length_penalty, page_size):
        B, V, device = len(lengths), self.cfg.vocab_size, str(self.tok_emb.device)
        # Beams share their prompt's full pages; in the worst case each has its own from the first unfinished page on,
        # and while a step parts them the old and the new one are both held.
        own = [-(-(n + steps) // page_size) - n // page_size for n in lengths]
        cache = self.new_cache(sum(n // page_size + W * more for n, more in zip(lengths, own)) + B * W + B, page_size)
        prompts = [cache.add() for _ in range(B)]
        logits = self.prefill(ids, cache, prompts, lengths)
        sequences = [cache.fork(s) for s in prompts for _ in range(W)]
        for s in prompts:
            cache.free(s)
        logits = _C.embedding(_whole(np.repeat(np.arange(B), W), device), logits)
        first = np.full((B, W), -np.inf, dtype=np.float32)
        first[:, 0] = 0.0
        scores = _C.from_numpy(first).to(device)
        finished = None if eos_token is None else _C.from_numpy(np.zeros((B, W), dtype=bool)).to(device)
        history = np.zeros((B, W, 0), dtype=np.int64)
        rows = np.arange(B)[:, None]
        for i in range(steps):
            scores, parents, tokens, ended = beam_search_step(logits.reshape([B, W, V]), scores, finished, eos_token)
            if eos_token is not None:
                finished = ended
            chosen = parents.numpy()
            history = np.concatenate([history[rows, chosen], tokens.numpy()[:, :, None]], axis=2)
            if i + 1 == steps or (eos_token is not None and bool(ended.numpy().all())):
                break
            sequences = cache.reorder(sequences, (rows * W + chosen).reshape(-1))
            logits = self.decode(tokens.reshape([B * W]), cache, sequences)
        final, out = scores.numpy(), []
        for b in range(B):
            beams = [_until(history[b, w].tolist(), eos_token) for w in range(W)]
            ranks = [float(final[b, w]) / len(beam) ** length_penalty for w, beam in enumerate(beams)]
            out.append(beams[int(np.argmax(ranks))])
        return out

    def parameter_count(self):
        return sum(int(p.numel) for p in self.parameters())
