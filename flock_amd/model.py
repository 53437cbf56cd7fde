"""Decoding of a whole Qwen3 model on libflock_attn (kernels/model.ts).

``Model`` follows model.ts's engine: token ids -> embedding gather (embed.wgsl,
over the tied token_embd) -> the decoder layers -> output norm -> LM head ->
argmax (model.ts:227-346). ``step(ids)`` feeds ids (a prompt, or one token)
and returns the next id; ``generate(prompt, maxTokens, eos)`` is the greedy
loop of model.ts:572-590.

Where the reference records each step into a WebGPU command buffer, here the
one-token step is captured once into a HIP graph and replayed: the position,
the token the embedding reads (the previous step's argmax) and the log of
generated ids all live in device memory, so a token costs one graph launch
and no host round trip; the host reads the whole log at the end.

Extensions (the reference decodes one sequence, greedily): ``answers`` draws several
answers to one prompt together, the prompt's keys stored and read once for all of
them, and ``score`` gives the log probabilities of given ids.
"""
from __future__ import annotations

import numpy as np

from ._lib import CacheFullError
from . import ops
from .decoder import DecoderConfig, DecoderLayer


SCORE_ROWS = 128  # of logits at a time


class _Answers:
    """n answers of up to T ids: what a step of them reads and writes on the device, and
    the captured step. Sequence b's own keys are the T rows behind the prompt's and those of
    the b sequences before it, in every layer's cache."""

    def __init__(self, model: "Model", n: int, T: int, n_stops: int):
        cfg, V = model.cfg, model.vocab
        B, f = ops.DeviceBuffer, 4
        self.key, self.max_top_k = (n, T, n_stops), min(64, V)
        self.n_groups, self.n_seqs, self.max_prefix, self.max_n_keys = 1, n, cfg.maxKeys, T
        self.prefix_row = B.from_array(np.zeros(1, np.uint64))
        self.n_prefix = B(4)
        self.seq_off = B.from_array(np.array([0, n], np.uint32))
        self.seq_row_off, self.n_keys = B(8 * n), B(4 * n)
        self.ws = B(ops.decode_shared_ws_bytes(1, n, cfg.maxKeys, T, cfg.nHeads, cfg.nKvHeads,
                                               cfg.headDim))
        self.x, self.logits = B(n * cfg.hidden * f), B(n * V * f)
        self.token, self.logprob, self.uniform = B(4 * n), B(4 * n), B(4 * n)
        self.temperature, self.top_k = B(4 * n), B(4 * n)
        self.top_p, self.min_p = B(4 * n), B(4 * n)
        self.token_ws = B(max(256, ops.tokens_ws_bytes(n, V, self.max_top_k)))
        self.stops = B(4 * n_stops) if n_stops else None
        self.cursor = B(4)
        self.token_log, self.logprob_log, self.uniform_log = (B(4 * T * n) for _ in range(3))
        self.stream = ops.Stream()
        ops.set_stream(self.stream)
        try:
            with ops.Graph() as g:
                ops.embed(model.embd, self.token, n, self.x)
                for layer in model.layers:
                    layer.encode_shared(self.x, self, self.x)
                ops.q8_matvec_ex(model.embd, self.x, self.logits, n, norm_gain=model.g_out,
                                 eps=cfg.eps)
                ops.sample(self.logits, self.uniform, self.token, n, V, self.max_top_k,
                           self.token_ws, temperature=self.temperature, top_k=self.top_k,
                           top_p=self.top_p, min_p=self.min_p, logprob=self.logprob)
                ops.advance_seqs(self.n_keys, self.cursor, self.token, self.token_log, n, T,
                                 logprob=self.logprob, logprob_log=self.logprob_log,
                                 stops=self.stops, n_stops=n_stops,
                                 uniform_log=self.uniform_log, uniform=self.uniform)
        finally:
            ops.set_stream(None)
        self.graph = g

    def free(self) -> None:
        self.graph.free()
        self.stream.free()
        for x in vars(self).values():
            if isinstance(x, ops.DeviceBuffer):
                x.free()


class Model:
    def __init__(self, cfg: DecoderConfig, layer_weights: list, token_embd, output_norm,
                 vocab: int, max_generate: int = 4096):
        self.cfg, self.vocab = cfg, vocab
        hid = cfg.hidden
        self.layers = [DecoderLayer.create(cfg, w) for w in layer_weights]
        self.embd = ops.Q8Matrix.from_packed(token_embd, vocab, hid)  # tied: embed + LM head
        self.g_out = ops.DeviceBuffer.from_array(np.ascontiguousarray(output_norm, np.float32))
        B = ops.DeviceBuffer
        P = max(1, cfg.maxPrefill)
        self.ids = B(4 * P)
        self.x = B(4 * P * hid)               # embedding output (layer 0's input)
        self.normed = B(4 * hid)
        self.tok_val, self.tok_idx = B(4), B(4)
        self.head_ws = B(ops.lm_head_ws_bytes(vocab, hid))
        self.state = B(8)                     # {position + 1, log cursor} of the captured step
        self.max_generate = max_generate
        self.log = B(4 * max_generate)
        self.nKeys = 0
        self.graph = None
        self._stream = None
        self._answers = None
        self._score = None

    # ------------------------------------------------------------- host steps
    def reset(self) -> None:
        self.nKeys = 0
        for layer in self.layers:
            layer.reset()

    def _head(self, src_row) -> None:
        ops.lm_head(src_row, self.g_out, self.cfg.eps, self.embd, self.normed, None,
                    self.tok_val, self.tok_idx, self.head_ws)

    def step(self, ids) -> int:
        """Feed ``ids`` at positions nKeys.. and return the greedy next id
        (model.ts:387-393), prefilling in chunks of maxPrefill."""
        ids = np.ascontiguousarray(ids, np.uint32).ravel()
        if ids.size == 0:
            raise ValueError("step needs at least one token id")
        if self.nKeys + ids.size > self.cfg.maxKeys:
            raise CacheFullError(-2, f"KV cache would exceed {self.cfg.maxKeys} keys "
                                     f"({self.nKeys} + {ids.size})")
        for n, src in self._feed(ids):
            pass
        self._head(ops.ptr(src) + (n - 1) * self.cfg.hidden * 4)
        ops.sync()
        return int(self.tok_idx.download(1, np.uint32)[0])

    def _feed(self, ids):
        """Feed ids in chunks of maxPrefill; yields each chunk's size and output rows."""
        P = max(1, self.cfg.maxPrefill)
        for off in range(0, ids.size, P):
            chunk = ids[off:off + P]
            n = chunk.size
            self.ids.upload(chunk)
            ops.embed(self.embd, self.ids, n, self.x)
            src = self.x
            for layer in self.layers:
                if n == 1:
                    layer.encode(src=src)
                else:
                    layer.encodePrefill(n, src=src)
                src = layer.outputBuffer()
            self.nKeys += n
            yield n, src

    def score(self, ids) -> np.ndarray:
        """Feed ``ids`` at positions nKeys.. as step does; the log probability of
        each but the first, given all before it."""
        ids = np.ascontiguousarray(ids, np.uint32).ravel()
        if ids.size < 2:
            raise ValueError("score needs two token ids or more")
        if ids.max() >= self.vocab:
            raise ValueError(f"id {ids.max()} of a vocabulary of {self.vocab}")
        if self.nKeys + ids.size > self.cfg.maxKeys:
            raise CacheFullError(-2, f"KV cache would exceed {self.cfg.maxKeys} keys "
                                     f"({self.nKeys} + {ids.size})")
        B, hid, V = ops.DeviceBuffer, self.cfg.hidden, self.vocab
        if self._score is None:
            P = max(1, self.cfg.maxPrefill)
            R = min(P, SCORE_ROWS)
            self._score = (B(R * V * 4), B(4 * P), B(4 * P),
                           B(max(256, ops.tokens_ws_bytes(R, V, 0))))
        logits, tokens, logprob, ws = self._score
        out, off = [], 0
        for n, src in self._feed(ids):
            m = min(n, ids.size - 1 - off)  # rows with an id to score
            if m == 0:
                break
            tokens.upload(ids[off + 1:off + 1 + m])
            for r in range(0, m, SCORE_ROWS):
                rows = min(SCORE_ROWS, m - r)
                ops.q8_matvec_ex(self.embd, ops.ptr(src) + r * hid * 4, logits, rows,
                                 norm_gain=self.g_out, eps=self.cfg.eps)
                ops.token_logprobs(logits, tokens.ptr + 4 * r, logprob.ptr + 4 * r, rows, V, ws)
            ops.sync()
            out.append(logprob.download(m))
            off += n
        return np.concatenate(out)

    # --------------------------------------------------------- captured steps
    def _capture(self) -> None:
        """Record the one-token step: embed(tok_idx) -> layers (position from
        n_keys_dev) -> head -> log the token, n_keys_dev += 1."""
        self._stream = ops.Stream()
        ops.set_stream(self._stream)
        with ops.Graph() as g:
            ops.embed(self.embd, self.tok_idx, 1, self.x)
            src = self.x
            for layer in self.layers:
                layer.encode_dev(src, self.state)  # state[0] = position + 1
                src = layer.outputBufferDev()
            self._head(src)
            ops.advance(self.state, 1, self.tok_idx, self.log, self.max_generate)
        self.graph = g

    def generate(self, prompt, maxTokens: int, eos=()) -> list:
        """Greedy decode (model.ts:572-590): the prompt is one host step, each
        further token one replay of the captured step."""
        if maxTokens < 1:
            return []
        if maxTokens > self.max_generate + 1:
            raise ValueError(f"maxTokens {maxTokens} exceeds max_generate {self.max_generate} + 1")
        first = self.step(prompt)
        rest = maxTokens - 1
        if self.nKeys + rest > self.cfg.maxKeys:
            raise CacheFullError(-2, f"KV cache full at {self.cfg.maxKeys} keys")
        out = [first] + (self.replay(first, rest) if rest > 0 else [])
        eos = set(int(e) for e in eos)
        for i, t in enumerate(out):
            if t in eos:
                return out[:i]
        return out

    def replay(self, first: int, n: int, read: bool = True) -> list:
        """Feed ``first`` at position nKeys and decode n tokens by replaying
        the captured step n times (the first n - 1 outputs are fed back on
        the device). Returns the n ids (read=False: leave them in the device
        log and return [])."""
        if self.nKeys + n > self.cfg.maxKeys:
            raise CacheFullError(-2, f"KV cache full at {self.cfg.maxKeys} keys")
        if n > self.max_generate:
            raise ValueError(f"{n} tokens exceed max_generate {self.max_generate}")
        if self.graph is None:
            self._capture()
        ops.set_stream(self._stream)
        self.state.upload(np.array([self.nKeys + 1, 0], np.uint32))
        self.tok_idx.upload(np.array([first], np.uint32))
        for _ in range(n):
            self.graph.launch()
        ops.sync()
        out = [int(t) for t in self.log.download(n, np.uint32)] if read else []
        self.nKeys += n
        for layer in self.layers:
            layer.nKeys = self.nKeys
        ops.set_stream(None)
        return out

    def _answers_step(self, *key) -> "_Answers":
        """The captured step of ``key`` (answers, ids, stops), kept from call to call."""
        if self._answers is None or self._answers.key != key:
            ops.sync()  # (what has been launched, on whichever stream)
            if self._answers is not None:
                self._answers.free()
                self._answers = None
            self._answers = _Answers(self, *key)
        return self._answers

    def answers(self, prompt, n: int, maxTokens: int, eos=(), temperature: float = 1.0,
                top_k: int = 64, top_p: float = 1.0, min_p: float = 0.0, seed=None) -> list:
        """n answers to ``prompt`` (fed at positions nKeys..), drawn together: a list of
        (ids, their log probabilities), each up to maxTokens long and ending before an id in
        ``eos``. Tokens come from the top_k (up to 64) largest logits as ops.sample draws
        them (never from the whole vocabulary), temperature 0 takes the largest; log
        probabilities are the model's own, whatever the settings: not those of the draw, which is
        of the alternatives that stay. ``seed`` fixes the random numbers. RuntimeError where an answer's logits
        hold nothing to draw (all NaN or -infinity).

        A step is one replay of a captured step of all answers: their queries meet the
        prompt's keys together. The prompt's last id is each answer's first input, so
        the cache holds the prompt but for that id afterwards, and no answer."""
        prompt = np.ascontiguousarray(prompt, np.uint32).ravel()
        if prompt.size == 0:
            raise ValueError("answers need at least one token id")
        if prompt.max() >= self.vocab:
            raise ValueError(f"id {prompt.max()} of a vocabulary of {self.vocab}")
        if n < 1 or n > max(1, self.cfg.maxPrefill):
            raise ValueError(f"{n} answers: 1 .. maxPrefill ({self.cfg.maxPrefill}) at a time")
        if not 1 <= top_k <= 64:
            raise ValueError(f"top_k must be 1 .. 64, got {top_k}")
        with np.errstate(over="ignore"):  # (what the device gets)
            settings = np.float32(temperature), np.float32(top_p)
        if not temperature >= 0 or not settings[0] < np.inf:
            raise ValueError(f"temperature must be finite and >= 0 in f32, got {temperature}")
        if not settings[1] > 0 or not 0 <= min_p <= 1:
            raise ValueError(f"top_p must be > 0 in f32 and min_p 0 .. 1, got {top_p} and {min_p}")
        if maxTokens < 1:
            return [([], []) for _ in range(n)]
        held = self.nKeys + prompt.size - 1
        if held + n * maxTokens > self.cfg.maxKeys:
            raise CacheFullError(-2, f"KV cache would exceed {self.cfg.maxKeys} keys "
                                     f"({held} + {n} x {maxTokens})")
        eos = sorted(set(int(e) for e in eos if 0 <= e < self.vocab))
        u32, f32 = np.uint32, np.float32
        uniform = np.random.default_rng(seed).random((maxTokens, n), f32)
        # The prompt is fed when nothing is left that could fail.
        a = self._answers_step(n, maxTokens, len(eos))
        for _ in self._feed(prompt[:-1]):
            pass
        ops.sync()  # (the captured step is on a stream of its own)
        a.n_prefix.upload(np.array([held], u32))
        a.seq_row_off.upload(held + maxTokens * np.arange(n, dtype=np.uint64))
        a.n_keys.upload(np.ones(n, u32))
        a.cursor.upload(np.zeros(1, u32))
        a.token.upload(np.full(n, prompt[-1], u32))
        for buf, x, t in ((a.temperature, temperature, f32), (a.top_k, min(top_k, a.max_top_k), u32),
                          (a.top_p, top_p, f32), (a.min_p, min_p, f32)):
            buf.upload(np.full(n, x, t))
        if eos:
            a.stops.upload(np.array(eos, u32))
        a.uniform_log.upload(uniform)
        a.uniform.upload(uniform[0])
        done = 0
        ops.set_stream(a.stream)
        try:
            while done < maxTokens:
                for _ in range(min(32, maxTokens - done)):
                    a.graph.launch()
                    done += 1
                ops.sync()
                if not a.n_keys.download(n, u32).any():
                    break
        finally:
            ops.set_stream(None)
        ids = a.token_log.download(done * n, u32).reshape(done, n)
        logprob = a.logprob_log.download(done * n).reshape(done, n)
        out = []
        for b in range(n):
            stop = np.flatnonzero(np.isin(ids[:, b], eos + [0xffffffff]))
            end = stop[0] if stop.size else done
            if end < done and ids[end, b] == 0xffffffff:
                raise RuntimeError(f"answer {b} has no id {end}: none of its logits is above "
                                   "-infinity")
            out.append(([int(t) for t in ids[:end, b]], [float(x) for x in logprob[:end, b]]))
        return out

    def free(self) -> None:
        if self._answers is not None:
            self._answers.free()
        for x in self._score or ():
            x.free()
        if self.graph is not None:
            self.graph.free()
        if self._stream is not None:
            self._stream.free()
        for layer in self.layers:
            layer.free()
