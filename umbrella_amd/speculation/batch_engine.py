"""Autoregressive batch engine for the sequence-mixer models (models/seqmix.py).

Where the speculation engines run ONE conversation through a draft tree and a tree-masked verify, this engine serves
MANY requests with no draft at all -- a recurrent state cannot be rolled back the way a KV slot is recycled, so these models
are decoded token by token -- and gets its throughput from batching instead: every step is one ragged forward over all
running requests.

Scheduling is static batching: when nothing runs, queued requests are admitted first come first served while sequence
slots and cache pages last, and their prompts are prefilled together in one step; from then on every step decodes one token
for each of them; a request that finishes gives its pages and slot back at once; the queue is looked at again when the
batch has drained.  One function, ``run_step``, executes a step for both the scheduler and callers that bring their own
tokens (trace replay): it owns the page / slot bookkeeping and calls the model's ragged forward.

It keeps the engine surface (speculation/base.py) so the front-ends work unchanged: ``prefill`` / ``append`` /
``speculative_decoding`` drive one conversation (a tree of size one: ``build_tree`` has nothing to build, ``verify`` is a
plain decode step), ``generate`` / ``generate_stream`` answer one API request, ``generate_batch`` many.
Sampling uses the same device kernels as the speculation engines (arg-max, or penalty / top-k / temperature / top-p) for requests that go by
the engine's settings; a request may bring its own (``Sampling``: temperature, top-k, top-p, min-p, seed), ask for several continuations of
its prompt (prefilled once, then forked: they share its full cache pages) and name a low-rank adapter of the model.
"""
from __future__ import annotations

import random
import time
from collections import deque
from dataclasses import dataclass, field

import torch

from .. import _lib
from ..attn.cache import send
from ..logging_config import setup_logger
from ..models import AutoModelLM
from ..utils import TextColors
from .base import BaseEngine
from .sampling import MAX_VOCAB, sample_rows
from .speculation_utils import IdTokenizer, is_sentence_complete_regex

logger = setup_logger()


@dataclass
class Sampling:
    """a request's own settings; a temperature of 0 is greedy, top_k 0 keeps all (include/umbrella_seq.h, umb_sample_requests).  Requests of one
    seed draw from the same random numbers (continuation i of one from the i-th row of them); None: each has its own."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int | None = None

    def check(self):
        if not (0.0 <= self.temperature < float("inf") and 0.0 <= self.top_p <= 1.0 and 0.0 <= self.min_p <= 1.0 and 0 <= self.top_k < 1 << 31):
            raise ValueError(f"a temperature of 0 and more, top_p and min_p of 0 to 1 and a top_k of 0 (all) and more are wanted, got {self}")


class RequestError(RuntimeError):
    """some of a call's requests ended without what they were asked for; ``outputs``: what every one of the call has generated"""
    def __init__(self, failed, outputs):
        super().__init__("; ".join(f"request {r.id!r}: {r.error}" for r in failed))
        self.outputs = outputs


@dataclass
class Request:
    id: object
    prompt: list
    max_new_tokens: int
    generated: list = field(default_factory=list)
    done: bool = False
    error: str | None = None            # why it ended before its time
    pending: int | None = None          # sampled, not yet fed through the model
    recorded: int = 0                   # tokens written to the device-side history of its slot
    sampling: Sampling | None = None    # None: the engine's
    rng: random.Random | None = None
    nth: int = 0                        # which continuation of its prompt
    seed: torch.Tensor | None = field(default=None, compare=False)        # of a further continuation's draws where the engine's generator makes them row by row
    adapter: int | None = None          # one of the model's
    loaded: int = 0                     # the model's load_adapters that it counts by
    copies: list = field(default_factory=list)       # further continuations of the same prompt


class BatchEngine(BaseEngine):
    NEEDS_DRAFT = False
    CHAT = "__chat__"

    def __init__(self, draft_model_name=None, target_model_name=None, dtype=torch.bfloat16, device: str = "cuda:0", **kwargs):
        super().__init__()
        self.target_model_name, self.dtype, self.device = target_model_name, dtype, device
        self.max_length = kwargs.pop("max_length", 8192)
        self.max_batch = kwargs.pop("max_batch", 8)
        self.max_tokens = kwargs.pop("max_tokens", None)
        self.page_size = kwargs.pop("page_size", 64)
        self.stop_distance = kwargs.pop("stop_distance", 32)
        self.temperature = kwargs.pop("temperature", 0.0)
        self.topp = kwargs.pop("topp", 0.9)
        self.topk = kwargs.pop("topk", 32)
        self.repetition_penalty = kwargs.pop("repetition_penalty", 1.0)
        self.seed = kwargs.pop("seed", 0)
        self._target_model = kwargs.pop("target_model_obj", None)
        self._tokenizer = kwargs.pop("tokenizer", None)
        self.config = kwargs

    # ------------------------------------------------------------------ setup
    def initialize(self):
        if self._target_model is None:
            self.target_model = AutoModelLM.from_pretrained(
                model_name=self.target_model_name, batch_size=self.max_batch, max_length=self.max_length, device=self.device,
                dtype=self.dtype, max_tokens=self.max_tokens, page_size=self.page_size)
            self.target_model.alloc()
        else:
            self.target_model = self._target_model
        if not hasattr(self.target_model, "forward_batch"):
            raise ValueError("the batch engine serves sequence-mixer models (models/seqmix.py); tree-decoded models run on "
                             "the static / dynamic speculation engines")
        m = self.target_model
        self.max_length, self.max_batch = m.max_length, m.batch_size
        self.vocab_size = m.config.vocab_size
        self.eos_tokens = list(m.eos_tokens)
        if self._tokenizer is not None:
            self.tokenizer = self._tokenizer
        else:
            try:
                from transformers import AutoTokenizer
                self.tokenizer = AutoTokenizer.from_pretrained(self.target_model_name, local_files_only=True)
            except Exception as e:
                logger.warning(f"NO TOKENIZER for '{self.target_model_name}' ({type(e).__name__}): falling back to the "
                               "id tokenizer -- text is read and written as space-separated token ids")
                self.tokenizer = IdTokenizer()
        dev = self.device
        self.sampled = torch.zeros(self.max_batch, dtype=torch.int32, device=dev)
        self.rng_state = torch.tensor([self.seed], dtype=torch.int64, device=dev)
        self.step_count = torch.zeros(1, dtype=torch.int32, device=dev)
        self.history = torch.zeros(self.max_batch, self.max_length + 1, dtype=torch.int32, device=dev)   # per slot: its tokens
        self.hist_len = torch.zeros(self.max_batch, dtype=torch.int32, device=dev)
        self.queue, self.running, self.finished = deque(), [], {}
        self._next_id = 0
        self.num_nodes = 0

    # ------------------------------------------------------------------ the step function
    @torch.inference_mode()
    def run_step(self, entries, end=()):
        """One step.  entries: [(request id, next tokens, indices whose logits are wanted)]; a request seen for the first
        time gets a sequence slot, `end` lists the requests whose pages, state and slot are given back after the step.
        Returns fp32 logits [rows wanted, V] in the order of the entries (a workspace view, valid until the next step)."""
        m = self.target_model
        cache = m.kv_cache
        parts, want = [], []
        for rid, toks, w in entries:
            if rid not in cache.seqs:
                m.open(rid)
            if len(toks) == 0:                  # a request that brings nothing this step only keeps (or takes) its slot
                continue
            parts.append((rid, toks))
            want.append(list(w))
        logits = m.forward_batch(parts, want=want) if parts else None
        for rid in end:
            if rid in cache.seqs:
                m.close(rid)
        return logits

    def _greedy(self):
        return self.temperature < 0.05 and not (self.repetition_penalty > 1.01)

    def _draws(self):
        """whether the engine's kernels take the engine's settings"""
        return self._greedy() or (1 <= min(int(self.topk), self.vocab_size) <= 1024 and self.topp > 0)

    def _sample_own(self, logits, reqs):
        """each row by its request's settings, or by the engine's where it has none, from its own random numbers -> int32 tokens on the device"""
        R = len(reqs)
        mine = [r.sampling or Sampling(0.0 if self.temperature < 0.05 else self.temperature, int(self.topk), float(self.topp)) for r in reqs]
        for r in reqs:
            if r.rng is None:
                seeded = r.sampling is not None and r.sampling.seed is not None
                r.rng = random.Random(f"{r.sampling.seed}//{r.nth}" if seeded else f"{self.seed}/{r.id}")
        host = torch.tensor([[s.temperature for s in mine], [s.top_p for s in mine], [s.min_p for s in mine], [r.rng.random() for r in reqs]], dtype=torch.float32)
        both = send(torch.cat([host.view(torch.int32), torch.tensor([[s.top_k for s in mine]], dtype=torch.int32)]), self.device)
        f = both.view(torch.float32)
        return sample_rows(logits[:R], f[3], temperature=f[0], top_k=both[4], top_p=f[1], min_p=f[2])[0]

    def _seed(self, r):
        """What a request's row is drawn from by itself: that generator goes by seed, history length and row, and the continuations of a prompt have all three in
        common, so that the further ones bring seeds of their own."""
        if r.nth == 0:
            return self.rng_state
        if r.seed is None:
            r.seed = send(torch.tensor([random.Random(f"{self.seed}/{r.id}").getrandbits(63)], dtype=torch.int64), self.device)
        return r.seed

    def _sample(self, logits, reqs):
        """One token per logits row (row i belongs to reqs[i]) -> list of ints; -1 for a row with settings of its own that leaves no token.  Rows without settings are
        drawn as they would be if no row had any."""
        rows = [i for i, r in enumerate(reqs) if r.sampling is None]
        if len(rows) == len(reqs):
            return self._sample_engine(logits, reqs, rows).tolist()
        tokens = self._sample_own(logits, reqs)
        if rows and (self._draws() or self.repetition_penalty > 1.01):
            at = send(torch.tensor(rows, dtype=torch.long), tokens.device)
            tokens[at] = self._sample_engine(logits, reqs, rows)[at]
        return tokens.tolist()

    def _sample_engine(self, logits, reqs, rows):
        """`rows` of the logits by the engine's settings, kernels and generator, which goes by the place of a row -> int32 tokens on the device, others' as well"""
        R = logits.shape[0]
        out = self.sampled[:R]
        if self._greedy():
            _lib.seq_call("umb_argmax_rows", out, logits, R, self.vocab_size)
        else:
            k = min(int(self.topk), self.vocab_size)
            self.step_count += 1
            if self.repetition_penalty > 1.01:
                for i in rows:                        # every request is penalised over its own history
                    r = reqs[i]
                    slot = self.target_model.kv_cache.slot(r.id)
                    _lib.seq_call("umb_sample_rows", out[i:i + 1], logits[i:i + 1], 1, self.vocab_size, self.history[slot],
                                  self.hist_len[slot:slot + 1], float(self.repetition_penalty), float(self.temperature), k,
                                  float(self.topp), self._seed(r), 0, None, None)
            else:
                if len(rows) < R:                     # (the others' are not its business: a row of its own in their places)
                    logits = logits[send(torch.tensor([i if r.sampling is None else rows[0] for i, r in enumerate(reqs)], dtype=torch.long), logits.device)]
                _lib.seq_call("umb_sample_rows", out, logits, R, self.vocab_size, self.history[0], self.step_count, 1.0,
                              float(self.temperature), k, float(self.topp), self.rng_state, 0, None, None)
        return out

    def _record(self, req, tokens):
        """append tokens to the request's device-side history (read by the repetition penalty)"""
        if not (self.repetition_penalty > 1.01):
            return
        slot = self.target_model.kv_cache.slot(req.id)
        n = req.recorded
        t = torch.tensor(tokens, dtype=torch.int32, device=self.device)
        self.history[slot, n:n + len(tokens)] = t
        req.recorded = n + len(tokens)
        self.hist_len[slot] = req.recorded - 1             # the kernel reads indices 0 .. n inclusive

    # ------------------------------------------------------------------ scheduler
    def submit(self, input_ids, max_new_tokens: int = 128, request_id=None, sampling: Sampling | None = None, n: int = 1, adapter: int | None = None):
        """Queues a request.  n > 1: so many continuations of the prompt; the further ones are requests (request_id, 1) to (request_id, n - 1) of
        their own, each with random numbers of its own.  adapter: one of those that the model has now; if others are loaded before the request runs,
        it ends with an error."""
        ids = [int(t) for t in (input_ids.reshape(-1).tolist() if isinstance(input_ids, torch.Tensor) else input_ids)]
        if not ids:
            raise ValueError("a request needs at least one prompt token")
        if len(ids) + max_new_tokens > self.max_length:
            raise ValueError(f"prompt ({len(ids)}) + max_new_tokens ({max_new_tokens}) exceeds max_length {self.max_length}")
        if sampling is not None and self.repetition_penalty > 1.01:
            raise ValueError("a repetition penalty does not go with settings of a request's own")
        if sampling is not None:
            sampling.check()
            if self.vocab_size > MAX_VOCAB:
                raise ValueError(f"settings of a request's own go with up to {MAX_VOCAB} tokens, the model has {self.vocab_size}")
        if not 1 <= n <= self.max_batch:
            raise ValueError(f"1 to {self.max_batch} continuations (sequence slots) are possible, got {n}")
        if adapter is not None and not 0 <= adapter < getattr(self.target_model, "n_adapters", 0):
            raise ValueError(f"the model has {getattr(self.target_model, 'n_adapters', 0)} adapters, got number {adapter}")
        if request_id is None:
            request_id, self._next_id = self._next_id, self._next_id + 1
        r = Request(request_id, ids, int(max_new_tokens), sampling=sampling, adapter=adapter, loaded=getattr(self.target_model, "adapters_loaded", 0))
        r.copies = [Request((request_id, i), ids, int(max_new_tokens), sampling=sampling, adapter=adapter, nth=i) for i in range(1, n)]
        self.queue.append(r)
        return request_id

    def _pages_wanted(self, r) -> int:
        """pages that a request and its further continuations may come to hold"""
        page = self.target_model.kv_cache.page
        whole, shared = (len(r.prompt) + r.max_new_tokens + page - 1) // page, len(r.prompt) // page
        return whole + len(r.copies) * (whole - shared)

    def _admit(self):
        """static batching: called only when nothing runs; first come first served while slots and pages last.  RuntimeError for a request that does not fit
        though nothing runs: it ends there, and those behind it are admitted by the next step."""
        cache = self.target_model.kv_cache
        budget, room, slots = len(cache.free_pages), min(self.max_batch, len(cache.free_slots)), 0
        while self.queue:
            r = self.queue[0]
            if r.adapter is not None and r.loaded != self.target_model.adapters_loaded:
                self._fail(self.queue.popleft(), f"the model's adapters are others than those that number {r.adapter} was one of")
                continue
            need, seqs = self._pages_wanted(r), 1 + len(r.copies)
            if slots + seqs > room or need > budget:
                break
            budget -= need
            slots += seqs
            self.running.append(self.queue.popleft())
        if self.running or not self.queue or (seqs > room and seqs == 1):     # (no slot at all: others hold them, and it waits)
            return
        why = f"needs {seqs} sequence slots, {room} are free" if seqs > room else f"needs {need} cache pages, the cache has {budget} free"
        self._fail(self.queue.popleft(), why)
        raise RuntimeError(f"request {r.id!r} {why}")

    def _fail(self, r, why):
        for q in (r, *r.copies):
            q.error, q.done = why, True
            self.finished[q.id] = q
        r.copies = []

    def _retire(self, r):
        r.done = True
        self.finished[r.id] = r
        self.running.remove(r)

    @torch.inference_mode()
    def step(self) -> bool:
        """One scheduler step (prefill of a fresh batch, or one decoded token for every running request).  Returns
        whether anything is left to do."""
        fresh = not self.running
        if fresh:
            self._admit()
            if not self.running:
                return False
        if not self._draws() and any(r.sampling is None for r in self.running) and (self.repetition_penalty > 1.01 or all(r.sampling is None for r in self.running)):
            if fresh:                           # (before the model has seen anything: the step can be made again with other settings)
                self.queue.extendleft(reversed(self.running))
                self.running.clear()
            raise _lib.UmbError(f"the engine's settings cannot be drawn by: top-k {self.topk} (1 to 1024 is wanted), top-p {self.topp} (above 0)")
        if fresh:
            batch = list(self.running)
            entries = [(r.id, r.prompt, [len(r.prompt) - 1]) for r in batch]
            for r in batch:
                if r.adapter is None:
                    self.target_model.open(r.id)
                else:
                    self.target_model.open(r.id, adapter=r.adapter)
                self._record(r, r.prompt)
        else:
            batch = list(self.running)
            entries = [(r.id, [r.pending], [0]) for r in batch]
        logits = self.run_step(entries)
        if any(r.copies for r in batch):
            batch, logits = self._branch(batch, logits)
        new = self._sample(logits, batch)
        end = []
        for r, tok in zip(batch, new):
            if tok < 0:                         # (its neighbours' tokens hold, and the model has taken in what they were drawn behind)
                r.error = "its logits leave no token to draw"
                end.append(r)
                continue
            r.generated.append(tok)
            r.pending = tok
            self._record(r, [tok])
            if len(r.generated) >= r.max_new_tokens or tok in self.eos_tokens:
                end.append(r)
        for r in end:
            self.target_model.close(r.id)
            self._retire(r)
        return bool(self.running or self.queue)

    def _branch(self, batch, logits):
        """behind the prompts' step: the further continuations of each go on from its sequence, and from its logits"""
        row, out = [], []
        for i, r in enumerate(batch):
            self.target_model.kv_cache.fork(r.id, [c.id for c in r.copies])
            for c in r.copies:
                self._record(c, c.prompt)
            row += [i] * (1 + len(r.copies))
            out += [r, *r.copies]
            r.copies = []
        self.running = list(out)
        return out, logits[send(torch.tensor(row, dtype=torch.long), logits.device)]

    @torch.inference_mode()
    def generate_batch(self, prompts, max_new_tokens: int = 128, sampling=None, n: int = 1, adapters=None):
        """prompts: list of token-id lists -> list of generated token-id lists (greedy or sampled per the engine's knobs).  sampling: one
        ``Sampling`` for all, or one (or None) per prompt; adapters: a number (or None) per prompt; n > 1: a list of n continuations per prompt.
        RequestError, once all have ended, if some did so before their time."""
        each = list(sampling) if isinstance(sampling, (list, tuple)) else [sampling] * len(prompts)
        named = list(adapters) if adapters is not None else [None] * len(prompts)
        if len(each) != len(prompts) or len(named) != len(prompts):
            raise ValueError("settings and adapters: one per prompt")
        ids = [self.submit(p, max_new_tokens, sampling=s, n=n, adapter=a) for p, s, a in zip(prompts, each, named)]
        while self.step():
            pass
        done = [[self.finished.pop(i if k == 0 else (i, k)) for k in range(n)] for i in ids]
        out = [[r.generated for r in each] if n > 1 else each[0].generated for each in done]
        failed = [r for each in done for r in each if r.error]
        if failed:
            raise RequestError(failed, out)
        return out

    # ------------------------------------------------------------------ one conversation (engine surface)
    def prefill(self, text: str):
        return self._prefill(self.tokenizer.encode(text, return_tensors="pt"))

    def append(self, text: str):
        return self._append(self.tokenizer.encode(text, return_tensors="pt")[:, 1:])

    def _feed_chat(self, ids):
        cache = self.target_model.kv_cache
        held = cache.length(self.CHAT) if self.CHAT in cache.seqs else 0
        if held + len(ids) + self.stop_distance >= self.max_length or \
                (self.CHAT in cache.seqs and not cache.can_extend(self.CHAT, len(ids) + self.stop_distance)):
            return False
        logits = self.run_step([(self.CHAT, ids, [len(ids) - 1])])
        self._chat.prompt.extend(ids)
        self._record(self._chat, ids)
        self._chat.pending = self._sample(logits, [self._chat])[0]
        self.num_nodes = cache.length(self.CHAT)
        return True

    @torch.inference_mode()
    def _prefill(self, input_ids):
        if self.CHAT not in self.target_model.kv_cache.seqs:
            self._chat = Request(self.CHAT, [], 0)
        return self._feed_chat([int(t) for t in input_ids.reshape(-1).tolist()])

    @torch.inference_mode()
    def _append(self, input_ids):
        assert getattr(self, "_chat", None) is not None, "append() follows prefill()"
        ids = [int(t) for t in input_ids.reshape(-1).tolist()]
        return self._feed_chat([self._chat.pending] + ids)          # the pending token becomes context

    def build_tree(self):
        """nothing to draft: the 'tree' of an autoregressive step is its root"""

    @torch.inference_mode()
    def verify(self) -> bool:
        """feed the pending token, sample the next; returns continue_generation"""
        c = self._chat
        logits = self.run_step([(self.CHAT, [c.pending], [0])])
        c.generated.append(c.pending)
        self._record(c, [c.pending])
        c.pending = self._sample(logits, [c])[0]
        self.num_nodes = self.target_model.kv_cache.length(self.CHAT)
        return c.generated[-1] not in self.eos_tokens

    def validate_status(self):
        cache = self.target_model.kv_cache
        return self.num_nodes + self.stop_distance < self.max_length and \
            (self.CHAT not in cache.seqs or cache.can_extend(self.CHAT, 1))

    def _decode_words(self, ids):
        return (self.tokenizer.decode(ids, skip_special_tokens=True, clean_up_tokenization_spaces=False,
                                      spaces_between_special_tokens=False).strip().split(" "))

    @torch.inference_mode()
    def speculative_decoding(self, max_new_tokens=128):
        max_new_tokens = max(max_new_tokens, self.stop_distance)
        torch.cuda.synchronize()
        t1 = time.time()
        steps, decode, ids, pos, words = 0, True, [], 0, [""]
        while decode and self.validate_status():
            decode = self.verify()
            steps += 1
            ids.append(self._chat.generated[-1])
            words = self._decode_words(ids)
            now = len(words) - 1
            if now > pos:
                print(" ".join(words[pos:now]), end=" ", flush=True)
                pos = now
            if (is_sentence_complete_regex(words[-1]) and steps >= max_new_tokens - self.stop_distance) or steps >= max_new_tokens:
                decode = False
        print(" ".join(words[pos:]), flush=True)
        torch.cuda.synchronize()
        t2 = time.time()
        logger.info(TextColors.colorize("Avg Accept Tokens {:.2f} | TPOT {:.2f} ms ".format(1.0, 1000 * (t2 - t1) / max(steps, 1)),
                                        "magenta"))
        return steps + 1, (t2 - t1), steps

    # ------------------------------------------------------------------ API requests
    def update_generation_args(self, **generation_args):
        self.temperature = generation_args.pop("temperature", self.temperature)
        self.topp = generation_args.pop("topp", self.topp)
        self.repetition_penalty = generation_args.pop("repetition_penalty", self.repetition_penalty)
        self.topk = generation_args.pop("topk", self.topk)

    def manual_seed(self, seed: int):
        self.seed = seed
        self.rng_state.fill_(seed)

    def _api_sampling(self, api_args):
        """An API request that names min_p has settings of its own, made of the engine's; others run by the engine's.  So does one that names it where own settings are
        not possible (a repetition penalty, a vocabulary too large), as it would on the other engines, which do not know min_p."""
        min_p, seed = api_args.get("min_p"), api_args.get("seed")
        if min_p is None:
            return None
        if self.repetition_penalty > 1.01 or self.vocab_size > MAX_VOCAB:
            logger.warning("min_p is not taken: " + ("it does not go with a repetition penalty" if self.repetition_penalty > 1.01 else f"the vocabulary has more than {MAX_VOCAB} tokens"))
            return None
        seed = None if seed is None else int(seed)
        if self.temperature < 0.05:             # (greedy, whatever the rest says)
            return Sampling(0.0, min_p=float(min_p), seed=seed)
        return Sampling(float(self.temperature), int(self.topk), min(float(self.topp), 1.0), float(min_p), seed)

    def _request_ids(self, api_args):
        input_ids = api_args.get("input_ids", None)
        if input_ids is None:
            context = api_args.get("context", None)
            if not context:
                return None
            return self.tokenizer.encode(context, return_tensors="pt").reshape(-1).tolist()
        return list(input_ids)

    @torch.inference_mode()
    def generate(self, **api_args):
        self.update_generation_args(**api_args)
        ids, n = self._request_ids(api_args), api_args.get("max_new_tokens", 128)
        if not ids or n == 0 or len(ids) + n > self.max_length:
            api_args.update(generated_text="", generated_tokens=[], avg_accept_tokens=0, time_per_output_token=0)
            return api_args
        torch.cuda.synchronize()
        t1 = time.time()
        toks = self.generate_batch([ids], n, sampling=self._api_sampling(api_args))[0]
        torch.cuda.synchronize()
        t2 = time.time()
        api_args["generated_text"] = self.tokenizer.decode(toks, skip_special_tokens=True, clean_up_tokenization_spaces=False)
        api_args["generated_tokens"] = toks
        api_args["avg_accept_tokens"] = 1.0
        api_args["time_per_output_token"] = 1000 * (t2 - t1) / max(len(toks), 1)
        return api_args

    @torch.inference_mode()
    def generate_stream(self, **api_args):
        self.update_generation_args(**api_args)
        ids, n = self._request_ids(api_args), api_args.get("max_new_tokens", 128)
        if not ids or n == 0:
            return
        if len(ids) + n > self.max_length:
            yield "Exceeding reserved allowed context length", "Exceeding reserved allowed context length"
            return
        rid = self.submit(ids, n, sampling=self._api_sampling(api_args))
        t1, text = time.time(), ""
        while self.step():
            r = next((q for q in self.running if q.id == rid), None)
            if r is None:
                break
            text = " ".join(self._decode_words(r.generated))
            yield text, "Output Tokens {} | TPOT {:.2f} ms ".format(len(r.generated), 1000 * (time.time() - t1) / len(r.generated))
        r = self.finished.pop(rid)
        if r.error:
            raise RequestError([r], [r.generated])
        yield " ".join(self._decode_words(r.generated)), "Output Tokens {} | TPOT {:.2f} ms ".format(
            len(r.generated), 1000 * (time.time() - t1) / max(len(r.generated), 1))

    @torch.inference_mode()
    def reset(self):
        self.target_model.clear()
        self.queue.clear()
        self.running.clear()
        self.finished.clear()
        self._chat = None
        self.num_nodes = 0
        self.hist_len.zero_()
