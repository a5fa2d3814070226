"""Several sequences decoded together over one paged cache: the prefills of several requests, continuations that share their
prompts, follow-up questions. The reference decodes one sequence at a time (src/chunkkv/engine/torch_engine.py:180-198).

    session = engine.paged(n_pages=2048, n_sequences=32, max_tokens=16384)
    a = session.add(engine.prefill(tokens), tokens)
    b, c = session.fork(a, 2)                    # share a's whole pages
    session.feed({b: question, c: other})        # a chunk of new tokens each
    texts = session.generate([a, b, c], 256, repetition=1.1)
    session.free([b, c])
    session.compact()

The cache's book lives on the device (ops.extend_pages and the like), so a decode step takes its pages inside a captured
graph; the host keeps each sequence's tokens, which say how many rows and pages a call will need.
"""

from __future__ import annotations

from contextlib import contextmanager

import torch

from chunkkv_amd import _native, ops


class PagedSession:
    """Made by HipEngine.paged. Sequences are numbers in [0, n_sequences); calls go to torch's current stream, in order."""

    def __init__(self, engine, n_pages: int, n_sequences: int, max_tokens: int, page_tokens: int = 64):
        if not (engine._native_attention and engine.attention in ("fused", "sdpa")):
            raise ValueError("a paged cache needs the attention kernel: bf16, head_dim 64 or 128, attention 'fused' or 'sdpa'")
        self.engine = engine
        self.cache = ops.paged_cache(len(engine.layers), n_pages, engine.n_kv, engine.head_dim, n_sequences, max_tokens,
                                     engine.device, page_tokens)
        self.tokens: dict[int, list[int]] = {}  # of each sequence, one for each of its rows
        self._logits: dict[int, torch.Tensor] = {}  # (1, vocab) behind a sequence's last row
        self._err = torch.zeros(1, dtype=torch.int32, device=engine.device)

    # -- pages ----------------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return int((self.cache.refs == 0).sum().item())

    def _known(self, sequences) -> list[int]:
        sequences = [int(s) for s in sequences]
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is named twice")
        for s in sequences:
            if s not in self.tokens:
                raise ValueError(f"no sequence {s}")
        return sequences

    def _check_room(self, more: dict[int, int]) -> None:
        """Whether every sequence s can grow by more[s] rows."""
        T = self.cache.page_tokens
        room = self.cache.table.shape[1] * T
        need = 0
        for s, n in more.items():
            have = len(self.tokens.get(s, ()))
            if have + n > room:
                raise ValueError(f"sequence {s} would have {have + n} rows, a sequence of this cache has at most {room}")
            need += -(-(have + n) // T) - -(-have // T)
        if need > self.free_pages:
            raise ValueError(f"{need} more pages are needed, {self.free_pages} are free")

    def _check_err(self) -> None:
        bits = int(self._err.item())
        if bits:
            self._err.zero_()
            if bits & _native.DEVICE_ERR_NO_TOKEN:
                raise ValueError("a mask left no token to choose")
            raise RuntimeError(f"a paged cache kernel reported an error ({bits})")

    @contextmanager
    def _or_back(self, rows: dict[int, int]):
        """Where this block raises, an interrupt among it, sequences s go back to rows[s] rows, which the device may have left; else
        the next rows would come behind ones that were never written."""
        try:
            yield
        except BaseException:
            self._go_back(rows)
            self._err.zero_()  # what this call flagged is not the next one's
            raise

    def _go_back(self, rows: dict[int, int]) -> None:
        ops.free_pages(self.cache, self._ints(rows), self._ints(rows.values()), self._err)

    def _token_list(self, tokens) -> list[int]:
        tokens = [int(t) for t in tokens]
        vocab = self.engine.inner.embed_tokens.weight.shape[0]
        if any(not 0 <= t < vocab for t in tokens):
            raise ValueError(f"a token outside the vocabulary of {vocab}")
        return tokens

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32).to(self.engine.device)

    def _counts(self, more: dict[int, int]) -> torch.Tensor:
        return self._ints(more.get(s, 0) for s in range(self.cache.lengths.shape[0]))

    def _slots(self, n: int) -> list[int]:
        slots = [s for s in range(self.cache.lengths.shape[0]) if s not in self.tokens][:n]
        if len(slots) < n:
            raise ValueError(f"the cache has no room for {n} more sequences")
        return slots

    # -- sequences ------------------------------------------------------------------------

    @torch.inference_mode()
    def add(self, result, tokens) -> int:
        """A new sequence of a prefill's rows (PrefillResult, its logits' last row the last token's); its number."""
        tokens = self._token_list(tokens)
        c = self.cache
        if len(result.keys) != c.k.shape[0] or len(tokens) != result.keys[0].shape[2]:
            raise ValueError(f"{len(tokens)} tokens of {c.k.shape[0]} layers for {result.keys[0].shape[2]} rows of {len(result.keys)}")
        shape = (1, c.k.shape[2], len(tokens), c.k.shape[4])
        for layers in (result.keys, result.values):
            if len(layers) != c.k.shape[0] or any(t.shape != shape or t.dtype != c.k.dtype or t.device != c.k.device for t in layers):
                raise ValueError(f"a prefill's keys and values are {shape} {c.k.dtype} on {c.k.device} in each of {c.k.shape[0]} layers here")
        (s,) = self._slots(1)
        self._check_room({s: len(tokens)})
        with self._or_back({s: 0}):
            new = ops.extend_pages(c, self._counts({s: len(tokens)}), len(tokens), self._err)
            for li in range(c.k.shape[0]):
                ops.scatter_rows(c.k[li], c.v[li], result.keys[li], result.values[li], new.rows, self._err)
            logits = result.logits[-1:].clone()  # not the prefill's other rows
            self._check_err()
        self.tokens[s] = tokens
        if logits.shape[0]:
            self._logits[s] = logits
        return s

    @torch.inference_mode()
    def fork(self, sequence: int, n: int = 1) -> list[int]:
        """n new sequences that continue this one; its whole pages are shared."""
        (source,) = self._known([sequence])
        if n < 0:
            raise ValueError("a number of new sequences is 0 or more")
        targets = self._slots(n)
        if len(self.tokens[source]) % self.cache.page_tokens and n > self.free_pages:
            raise ValueError(f"{n} more pages are needed, {self.free_pages} are free")
        with self._or_back(dict.fromkeys(targets, 0)):
            ops.fork_pages(self.cache, self._ints([source] * n), self._ints(targets), self._err)
            self._check_err()
        for t in targets:
            self.tokens[t] = list(self.tokens[source])
            if source in self._logits:
                self._logits[t] = self._logits[source]
        return targets

    @torch.inference_mode()
    def free(self, sequences) -> None:
        """These sequences end; pages that no other shares are free again."""
        sequences = self._known(sequences)
        with self._or_back(dict.fromkeys(sequences, 0)):  # ended is what they are then, too
            for s in sequences:
                del self.tokens[s]
                self._logits.pop(s, None)
            ops.free_pages(self.cache, self._ints(sequences), err=self._err)
            self._check_err()

    @torch.inference_mode()
    def compact(self) -> int:
        """Move the used pages to the front of the pool; how many there are."""
        used = int(ops.compact_pages(self.cache, self._err).item())
        self._check_err()
        return used

    # -- the model ------------------------------------------------------------------------

    def _forward(self, tok: torch.Tensor, counts: torch.Tensor, most: int, rows: list[int]):
        """New tokens tok (n,), in the order of the sequences, counts[s] of each, most of one at most; rows: of each with them, or
        about. The new rows are taken and written, layer by layer. (h, pending, starts), for the engine's _final_logits."""
        e, c = self.engine, self.cache
        known = dict(most=most, longest=max(rows), total=sum(rows))
        H, D, n = e.n_kv, e.head_dim, tok.shape[0]
        new = ops.extend_pages(c, counts, n, self._err)
        h, pending = e.inner.embed_tokens(tok[None]), None
        for li, layer in enumerate(e.layers):
            h, x = e._norm(li, layer, h, pending)
            q_in, k_in, v_in = e._project(li, x)
            q, _ = ops.rope_qkv(q_in, k_in, v_in, new.positions, e.n_heads, H, D, e.theta, k_out=c.k[li], v_out=c.v[li], rows=new.rows,
                                err=self._err)
            o = ops.attention_paged(q.transpose(1, 2), c, li, new.starts, err=self._err, **known)
            h, pending = e._mlp(li, layer, h, layer.self_attn.o_proj(o.view(1, n, -1)))
        return h, pending, new.starts

    @torch.inference_mode()
    def feed(self, tokens: dict) -> dict[int, torch.Tensor]:
        """Append a chunk of tokens to each of these sequences, all in one pass; {sequence: (1, vocab) logits behind its last one}."""
        chunks = {s: self._token_list(tokens[s]) for s in sorted(self._known(tokens))}
        if any(not chunk for chunk in chunks.values()):
            raise ValueError("a chunk has a token at least")
        if not chunks:
            return {}
        more = {s: len(chunk) for s, chunk in chunks.items()}
        self._check_room(more)
        tok = torch.tensor([t for chunk in chunks.values() for t in chunk], dtype=torch.int64).to(self.engine.device)
        with self._or_back({s: len(self.tokens[s]) for s in chunks}):
            rows = [len(self.tokens[s]) + n for s, n in more.items()]
            h, pending, starts = self._forward(tok, self._counts(more), max(more.values()), rows)
            last = starts[1:].long()[torch.tensor(list(chunks)).to(starts.device)] - 1
            logits = self.engine._final_logits(h[:, last], None if pending is None else pending[:, last])[0]
            self._check_err()
        for i, (s, chunk) in enumerate(chunks.items()):
            self.tokens[s] += chunk
            self._logits[s] = logits[i:i + 1]
        return {s: self._logits[s] for s in chunks}

    @torch.inference_mode()
    def generate(self, sequences, max_tokens: int = 32, *, repetition=1.0, frequency=0.0, presence=0.0, bias=None,
                 allowed=None) -> list[list[int]]:
        """Greedy decode of these sequences together, each up to max_tokens tokens or its end-of-sequence token (not among those returned);
        the new tokens of each, in the order they were named. They stay in the cache, and a sequence that did not end can go on.

        repetition, frequency, presence, bias, allowed: as ops.next_tokens takes them, rows in the order of `sequences`; a
        sequence's tokens before this call are its prompt, those of this call its generated ones. allowed may be a function of the
        new tokens so far (a list for each sequence), called before each step, that returns the step's mask; what that leaves a sequence
        that ended is passed over. Where a mask leaves another nothing, the call raises at that step, and the sequences are what they were."""
        order = self._known(sequences)
        if not order or max_tokens <= 0:
            return [[] for _ in order]
        for s in order:
            if s not in self._logits:
                raise ValueError(f"sequence {s} has no logits to go on from: feed it tokens first")
        self._check_room({s: max_tokens for s in order})
        dev, B = self.engine.device, len(order)
        by_slot = sorted(range(B), key=lambda i: order[i])  # the batch is in the order of the cache's sequences
        slots = [order[i] for i in by_slot]
        place = torch.tensor(by_slot, dtype=torch.int64).to(dev)

        def rows_of(x):  # a value a sequence, in the batch's order
            return x.index_select(0, place) if isinstance(x, torch.Tensor) and x.dim() and x.shape[0] == B else x

        fixed = dict(repetition=rows_of(repetition), frequency=rows_of(frequency), presence=rows_of(presence),
                     bias=rows_of(bias) if isinstance(bias, torch.Tensor) and bias.dim() == 2 else bias)
        masks = None
        out = [[] for _ in range(B)]  # in the batch's order

        def mask():
            m = allowed([out[by_slot.index(i)] for i in range(B)]) if callable(allowed) else allowed
            m = rows_of(m) if m.dim() == 2 else m
            return m.expand(B, m.shape[-1]) if callable(allowed) else m  # one for all, or one each at another step

        if allowed is not None:
            masks = mask().clone()
        longest = max(len(self.tokens[s]) for s in slots)
        prompt = torch.tensor([self.tokens[s] + [-1] * (longest - len(self.tokens[s])) for s in slots], dtype=torch.int64).to(dev)
        generated = torch.full((B, max_tokens), -1, dtype=torch.int64, device=dev)
        at = torch.zeros((B, 1), dtype=torch.int64, device=dev)
        counts = self._counts({s: 1 for s in slots})
        logits = torch.cat([self._logits[s] for s in slots])
        read = torch.zeros(B + 1, dtype=torch.int64, device=dev)  # what the host reads of a step: its tokens, and what it flagged
        tok = read[:B]

        def step():
            ops.next_tokens(logits, prompt=prompt, generated=generated, allowed=masks, err=self._err, out=tok, **fixed)
            generated.scatter_(1, at, tok[:, None])
            at.add_(1)
            h, pending, _ = self._forward(tok, counts, 1, [len(self.tokens[s]) + (max_tokens + 1) // 2 for s in slots])
            logits.copy_(self.engine._final_logits(h, pending)[0])
            read[B:].copy_(self._err)

        before = {s: len(self.tokens[s]) for s in slots}
        live, graph, steps = set(range(B)), None, 0
        with self._or_back(before):
            while live and steps < max_tokens:
                if steps and callable(allowed):
                    masks.copy_(mask())
                    if len(live) < B:  # what a mask leaves an ended sequence is no matter
                        masks[[i for i in range(B) if i not in live]] = -1
                if graph is not None:
                    graph.replay()
                else:
                    step()  # also the warm-up of the capture
                    if max_tokens - steps >= 3 and self.engine.decode_graphs:
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph):
                            step()
                steps += 1
                *new, flagged = read.tolist()
                if flagged:
                    self._check_err()
                for i, t in enumerate(new):
                    if i in live:
                        if t in self.engine.eos:
                            live.discard(i)
                        else:
                            out[i].append(t)
            self._go_back({s: before[s] + len(out[i]) for i, s in enumerate(slots)})  # every one took a row a step
            self._check_err()
        for i, s in enumerate(slots):
            self.tokens[s] = self.tokens[s] + out[i]
            if i in live:
                self._logits[s] = logits[i:i + 1]
            else:
                del self._logits[s]
        return [out[by_slot.index(i)] for i in range(B)]
