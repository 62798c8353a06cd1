"""Serving engine of layer-list models: request queue, scheduler, cache / state manager, sampling.

One `Engine.step()` is one forward pass over a flat mixed batch: every running request contributes its one decoded token, and
prompts that are not yet in the cache contribute their next portion (chunked prefill under a token budget), as the reference's
batch engine does (src/engine/batch_engine.rs:172-272 chunked prefill, src/engine/batch_decode.rs:35-209 decode batches).
Requests take a state slot and KV pages from `CacheManager` (blazr_b200/cache.py) on admission / growth and give them back when
they finish; pages and slots are reused.

`Engine.run_entries()` is the same step with the batch given from outside (which request brings which tokens): trace replay and
the tests drive it; `step()` builds the same entries from its own queues.  Both go through `_forward`, the only place that
touches the model.

`fork()` lets a second request continue from where another is: KV pages are shared and copied when one of the two is about to write
into them, recurrent state is copied at once.  `SamplingParams.n` samples a prompt several times that way.  Penalties, biases and
masks of a request are applied to its logits on the GPU before its token is chosen (seqops.process_logits).
"""
from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field, replace
from typing import Callable, Deque, Dict, List, Optional, Sequence, Set, Tuple

import numpy as np
import torch

from . import seqops
from .batch import StepEntry, build_step
from .cache import CacheFull, CacheManager
from .layered import LayeredModel

F32_MAX, F32_TINY = float(np.finfo(np.float32).max), float(np.finfo(np.float32).tiny)


@dataclass
class SamplingParams:
    """temperature 0 = greedy (arg-max kernel); otherwise soft-max sampling, optionally among the top_k / top_p tokens.
    repetition_penalty: the logits of tokens of the prompt and the output are divided by it (multiplied where negative); frequency_penalty times how often, and
    presence_penalty once if, a token stands in the output is subtracted; logit_bias: added per token; mask_fn(output so far) -> int32 words, bit v % 32 of word
    v / 32 set where token v is allowed, or None (all).  n: samples of the prompt, which is run once (Request.siblings holds the others)"""
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    seed: Optional[int] = None
    max_new_tokens: int = 16
    stop_tokens: Tuple[int, ...] = ()
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    mask_fn: Optional[Callable[[List[int]], Optional[Sequence[int]]]] = None
    n: int = 1

    def ruled(self) -> bool:
        """whether the logits are changed before the token is chosen"""
        return bool(self.repetition_penalty != 1.0 or self.presence_penalty or self.frequency_penalty or self.logit_bias or self.mask_fn)


@dataclass
class Request:
    rid: str
    prompt: List[int]
    params: SamplingParams
    output: List[int] = field(default_factory=list)
    fed: int = 0                 # prompt tokens already in the cache
    finished: bool = False
    siblings: List["Request"] = field(default_factory=list)   # the other samples of params.n
    _gen: Optional[torch.Generator] = None


class Engine:
    def __init__(self, model: LayeredModel, max_tokens: int, max_seqs: int = 4, block_size: int = 16, max_step_tokens: int = 2048,
                 prefill_chunk: int = 512, kv_bits: int = 32):
        """max_tokens: tokens all live requests may hold together (the KV pool is made for this many, rounded up to pages);
        max_seqs: state slots = most requests live at a time; kv_bits: bits of a cached key or value, 32 or 4"""
        self.model = model
        self.cache = CacheManager(max_tokens, max_seqs, block_size, model.pooled_sizes() if hasattr(model, "pooled_sizes") else ())
        model.allocate(self.cache.pages.num_blocks, block_size, max_seqs, self.cache.pages.num_blocks * block_size, **({} if kv_bits == 32 else {"kv_bits": kv_bits}))
        self.max_step_tokens, self.prefill_chunk = max_step_tokens, prefill_chunk
        self.waiting: Deque[Request] = deque()
        self.running: List[Request] = []
        self.requests: Dict[str, Request] = {}
        self._sample_ids: Set[str] = set()       # of the samples that prompts which are not through will have
        self.steps = 0

    # ---- the one place that runs the model -----------------------------------------------------------------------------------
    def _forward(self, batch: Sequence[Tuple[str, Sequence[int], Sequence[int]]], sample: bool = False) -> torch.Tensor:
        """batch: (request id, next tokens, wanted places) per entry.  Admits unseen ids, reserves pages, runs the step, advances
        the token counts.  Returns the f32 logits [wanted, vocab] (device; valid until the next step).  Where it raises, the ids that it admitted are none again."""
        entries: List[StepEntry] = []
        copies: List[Tuple[int, int]] = []
        admitted: List[str] = []
        seen = set()
        for rid, _, _ in batch:
            if rid in seen:
                raise ValueError(f"request {rid} appears twice in one step")
            seen.add(rid)
        try:
            try:
                for rid, toks, want in batch:
                    seq = self.cache.live.get(rid)
                    if seq is None:
                        seq = self.cache.admit(rid)
                        admitted.append(rid)
                    copies += self.cache.reserve(seq, len(toks))
                    entries.append(StepEntry(tokens=toks, pos0=seq.n_tokens, slot=seq.slot, block_table=seq.blocks, want=want, prev=seq.last_token))
            finally:
                if copies:      # also when the pages ran out on the way: these requests hold their copies already
                    self.model.copy_pages(copies)
            sa = build_step(entries, self.cache.block_size)
            logits = self.model.forward(sa, sample=sample)
        except BaseException:
            for rid in admitted:
                self.cache.release(rid)
            raise
        for rid, toks, _ in batch:
            self.cache.live[rid].n_tokens += len(toks)
            self.cache.live[rid].last_token = int(toks[-1])
        self.steps += 1
        return logits

    def release(self, rid: str) -> None:
        """gives an externally scheduled request's pages and slot back; of an id that holds none nothing"""
        if self._scheduled(rid):
            raise ValueError(f"request {rid} belongs to the scheduler")
        if rid in self.cache.live:
            self.cache.release(rid)

    def fork(self, rid: str, new_rid: str, params: Optional[SamplingParams] = None) -> Optional[Request]:
        """a second request that continues from where the live request `rid` is.  Of a request of the engine's own scheduler a Request (with the prompt and the
        output so far, and params or the same ones) that runs from the next step on; of an externally scheduled one None.  A sampled one draws from the beginning of its
        seed's numbers, not from where `rid` is in them: params of another seed make another continuation"""
        rid, new_rid = str(rid), str(new_rid)
        if self._in_use(new_rid):
            raise ValueError(f"request id {new_rid} is in use")
        if rid not in self.cache.live:
            raise ValueError(f"request {rid} holds nothing in the cache")
        if self.cache.slots.free_slots <= self._promised():
            raise CacheFull(f"no state slot for request {new_rid}: {self.cache.slots.free_slots} free, {self._promised()} kept for samples of running prompts")
        r = self._scheduled(rid)
        if r is not None:
            self._check(replace(params or r.params, n=1))
        self._fork_cache(rid, new_rid)
        if r is None:
            return None
        q = self._request(new_rid, r.prompt, replace(params or r.params, n=1))
        q.output, q.fed = list(r.output), r.fed
        self.running.append(q)
        return q

    def _in_use(self, rid: str) -> bool:
        return rid in self.requests or rid in self.cache.live or rid in self._sample_ids

    def _scheduled(self, rid: str) -> Optional[Request]:
        """the scheduler's request of that id; an id whose request is through may be an external one's"""
        r = self.requests.get(rid)
        return None if r is None or r.finished else r

    def _promised(self) -> int:
        """slots that running requests take when their prompt is through, for its other samples"""
        return sum(r.params.n - 1 for r in self.running if r.params.n > 1 and not r.output and not r.siblings)

    def _fork_cache(self, rid: str, new_rid: str) -> None:
        src, new = self.cache.live[rid], self.cache.fork(rid, new_rid)
        if hasattr(self.model, "copy_slots"):
            self.model.copy_slots([(src.slot, new.slot)])

    def truncate(self, rid: str, n_tokens: int) -> None:
        """takes back the tokens of an externally scheduled request from position n_tokens on (rejected drafts); models whose layers carry state cannot"""
        rid = str(rid)
        if self._scheduled(rid):
            raise ValueError(f"request {rid} belongs to the scheduler")
        if rid not in self.cache.live:
            raise ValueError(f"request {rid} holds nothing in the cache")
        if hasattr(self.model, "has_state") and self.model.has_state():
            raise ValueError("layers of this model carry state that cannot be taken back")
        if getattr(self.model, "cfg", None) is not None and getattr(self.model.cfg, "bigram", None) is not None:
            raise ValueError("this model's embedding reads the token before the next one, which a truncated request has lost")
        self.cache.truncate(rid, n_tokens, -1)

    def compact(self) -> int:
        """moves the KV pages in use to the front of the pool; returns how many moved"""
        pairs = self.cache.compact()
        if pairs:
            self.model.copy_pages(pairs)
        return len(pairs)

    # ---- externally scheduled steps (trace replay) ----------------------------------------------------------------------------
    def run_entries(self, entries: Sequence[dict], end: Sequence[str] = ()) -> Optional[np.ndarray]:
        """entries: [{"id", "tokens", "want"}], of ids that are none of the scheduler's; end: requests whose pages and slot are given back after the step.
        Returns the logits of the wanted places as a host array, or None when nothing was wanted."""
        out = None
        entries = [e for e in entries if len(e.get("tokens", ()))]      # an entry that brings no token has nothing to run
        for rid in [str(e["id"]) for e in entries] + [str(i) for i in end]:
            if rid in self._sample_ids or self._scheduled(rid):
                raise ValueError(f"request {rid} belongs to the scheduler")
        new, free = len({str(e["id"]) for e in entries} - self.cache.live.keys()), self.cache.slots.free_slots
        if new and new > free - self._promised():
            raise CacheFull(f"{new} state slots wanted, {free} free, {self._promised()} of them kept for samples of running prompts")
        if entries:
            logits = self._forward([(str(e["id"]), list(e["tokens"]), list(e.get("want", ()))) for e in entries])
            if logits.shape[0]:
                out = logits.cpu().numpy()
        for rid in end:
            self.release(str(rid))
        return out

    # ---- own scheduler ---------------------------------------------------------------------------------------------------------
    def add_request(self, rid: str, prompt: Sequence[int], params: Optional[SamplingParams] = None) -> Request:
        rid = str(rid)
        if self._in_use(rid):
            raise ValueError(f"request id {rid} is in use")
        if not len(prompt):
            raise ValueError("empty prompt")
        params = params or SamplingParams()
        self._check(params)
        samples = [f"{rid}#{i}" for i in range(1, params.n)]
        if any(self._in_use(i) for i in samples):
            raise ValueError(f"request ids {rid}#1 and on are in use")
        r = self._request(rid, [int(t) for t in prompt], params)
        self._sample_ids.update(samples)
        self.waiting.append(r)
        return r

    def _check(self, p: SamplingParams) -> None:
        if not 1 <= p.n <= self.cache.slots.n:
            raise ValueError(f"{p.n} samples of a prompt, of {self.cache.slots.n} requests that may live at a time")
        # (numbers as the kernels have them: of 32 bits)
        if not F32_TINY <= p.repetition_penalty <= F32_MAX:
            raise ValueError(f"a repetition penalty of {p.repetition_penalty}")
        if not (abs(p.presence_penalty) <= F32_MAX and abs(p.frequency_penalty) <= F32_MAX):
            raise ValueError(f"presence and frequency penalties of {p.presence_penalty} and {p.frequency_penalty}")
        if p.temperature != p.temperature or 0 < p.temperature < F32_TINY or (p.temperature > F32_MAX and p.ruled()):
            raise ValueError(f"a temperature of {p.temperature}")
        if p.temperature > 0 and not p.top_p > 0:
            raise ValueError(f"a top_p of {p.top_p}")
        if p.temperature > 0 and p.top_k < 0:
            raise ValueError(f"a top_k of {p.top_k}")
        vocab = getattr(getattr(self.model, "cfg", None), "vocab", None)
        for t in p.logit_bias or ():
            if int(t) != t or t < 0 or (vocab is not None and t >= vocab):
                raise ValueError(f"a bias on token {t} of {vocab}")
        for t, v in (p.logit_bias or {}).items():
            if not v <= F32_MAX:
                raise ValueError(f"a bias of {v} on token {t}")
        if vocab is not None and len(self._forbidden(p)) == vocab:
            raise ValueError("biases that leave no token")

    @staticmethod
    def _forbidden(p: SamplingParams) -> List[int]:
        """tokens that a bias of minus infinity (in 32 bits) takes out"""
        return [int(t) for t, v in (p.logit_bias or {}).items() if v < -F32_MAX]

    def _request(self, rid: str, prompt: List[int], params: SamplingParams, place: int = 0) -> Request:
        r = Request(rid, prompt, params)
        if params.temperature > 0:
            r._gen = torch.Generator(device=self.model.dev)
            r._gen.manual_seed((params.seed if params.seed is not None else 0) + place)
        self.requests[r.rid] = r
        return r

    def has_work(self) -> bool:
        return bool(self.waiting or self.running)

    def _schedule(self) -> List[Tuple[Request, List[int], List[int]]]:
        """decoded tokens of running requests first, then prompt portions while the token budget, the slots and the pages last"""
        plan: List[Tuple[Request, List[int], List[int]]] = []
        budget = self.max_step_tokens
        free_pages = self.cache.pages.free_blocks
        free_slots = self.cache.slots.free_slots - self._promised()
        for r in self.running:
            if r.fed < len(r.prompt):
                continue
            seq = self.cache.live[r.rid]
            need = self.cache.pages_needed(seq, 1)
            if budget < 1 or need > free_pages:
                continue
            plan.append((r, [r.output[-1]], [0]))
            budget -= 1
            free_pages -= need
        prefilling = [r for r in self.running if r.fed < len(r.prompt)]
        for r in prefilling + list(self.waiting):
            if budget < 1:
                break
            seq = self.cache.live.get(r.rid)
            if seq is None:
                if free_slots < r.params.n:
                    break
                free_slots -= r.params.n
            n = min(len(r.prompt) - r.fed, self.prefill_chunk, budget)
            have = len(seq.blocks) if seq else 0
            held = seq.n_tokens if seq else 0
            own = self.cache.pages_to_copy(seq) if seq else 0       # shared pages that the portion would write into
            room = (have + free_pages - own) * self.cache.block_size - held if free_pages >= own else 0
            n = min(n, room)
            if n < 1:
                if seq is None:
                    free_slots += r.params.n
                break
            need = max(0, -(-(held + n) // self.cache.block_size) - have)
            free_pages -= need + own
            budget -= n
            last = r.fed + n == len(r.prompt)
            plan.append((r, r.prompt[r.fed:r.fed + n], [n - 1] if last else []))
        return plan

    def step(self) -> List[Request]:
        """one forward pass over what the scheduler picked; returns the requests that finished in it.  A request whose logits leave no choice (sampled, and the
        largest over its temperature is no number) finishes without a token; when all others have theirs, RuntimeError says so"""
        plan = self._schedule()
        if not plan:
            if self.has_work():
                raise CacheFull("no request can make progress: the KV pool is too small for the live requests")
            return []
        masks = {r.rid: self._mask(r) for r, _, w in plan if w and r.params.mask_fn is not None}
        greedy = all(r.params.temperature <= 0 and not r.params.ruled() and r.params.n == 1 for r, _, w in plan if w)
        logits = self._forward([(r.rid, toks, want) for r, toks, want in plan], sample=greedy)
        for r, _, _ in plan:        # (requests run from here on: a mask that was refused, or a pass that failed, leaves them waiting)
            if r in self.waiting:
                self.waiting.remove(r)
                self.running.append(r)
        sampled = [r for r, _, w in plan if w]
        ids = self.model.last_ids.cpu().tolist() if (greedy and sampled) else None
        for r, toks, _ in plan:
            if r.fed < len(r.prompt):
                r.fed += len(toks)
        done: List[Request] = []
        rows = list(range(len(sampled)))
        if any(r.params.n > 1 and not r.output and not r.siblings for r in sampled):
            rows, sampled = self._fan_out(sampled)      # the other samples of a prompt choose from the same logits
            logits = logits[torch.tensor(rows, device=logits.device)]
            rows = list(range(len(sampled)))
        if ids is None and any(r.params.ruled() for r in sampled):
            logits = self._apply_rules(logits[:len(sampled)], sampled, masks)
        # largest logits of rows that are sampled: where one is no number there is nothing to choose by (and a multinomial of it would end the process)
        tops = logits[:len(sampled)].max(1).values.tolist() if any(r.params.temperature > 0 for r in sampled) else None
        lost: List[str] = []
        for row, r in zip(rows, sampled):
            if r.params.temperature > 0 and not abs(tops[row] / r.params.temperature) <= F32_MAX:
                lost.append(f"{r.rid} (its largest logit is {tops[row]}, its temperature {r.params.temperature})")
                r.finished = True
                done.append(r)
                continue
            tok = ids[row] if ids is not None else self._sample(logits[row], r)
            r.output.append(int(tok))
            if len(r.output) >= r.params.max_new_tokens or int(tok) in r.params.stop_tokens:
                r.finished = True
                done.append(r)
        for r in done:
            self.running.remove(r)
            self.release(r.rid)
        if lost:
            raise RuntimeError("no token can be chosen for request " + ", ".join(lost))
        return done

    def _fan_out(self, sampled: List[Request]) -> Tuple[List[int], List[Request]]:
        """forks requests whose prompt is through into their params.n samples; (row of the step's logits, request) of every sample, in order"""
        rows, out = [], []
        for row, r in enumerate(sampled):
            rows.append(row)
            out.append(r)
            if r.params.n > 1 and not r.output and not r.siblings:
                for i in range(1, r.params.n):
                    rid = f"{r.rid}#{i}"
                    self._sample_ids.discard(rid)
                    self._fork_cache(r.rid, rid)
                    q = self._request(rid, r.prompt, r.params, i)
                    q.fed = r.fed
                    q.siblings = [r]
                    r.siblings.append(q)
                    self.running.append(q)
                    rows.append(row)
                    out.append(q)
        return rows, out

    def _mask(self, r: Request) -> Optional[np.ndarray]:
        """the words of the tokens that may come next, asked for before the step runs: a mask that is refused leaves the request as it was"""
        words = r.params.mask_fn(list(r.output))
        if words is None:
            return None
        m = np.asarray(words).reshape(-1).astype(np.int64).astype(np.uint32)
        vocab = getattr(getattr(self.model, "cfg", None), "vocab", 32 * m.size)
        if m.size != (vocab + 31) // 32:
            raise ValueError(f"the mask of request {r.rid} has {m.size} words, not {(vocab + 31) // 32}")
        forbidden = [t for t in self._forbidden(r.params) if t < 32 * m.size]
        if forbidden:
            bits = np.unpackbits(m.astype("<u4").view(np.uint8), bitorder="little")
            bits[forbidden] = 0
            m = np.packbits(bits, bitorder="little").view("<u4").astype(np.uint32)
        last = m[-1] if vocab % 32 == 0 else m[-1] & np.uint32((1 << vocab % 32) - 1)
        if not (m[:-1].any() or last):
            raise ValueError(f"the mask of request {r.rid} leaves no token")
        return m.view(np.int32)

    def _apply_rules(self, logits: torch.Tensor, requests: Sequence[Request], masks: Dict[str, Optional[np.ndarray]]) -> torch.Tensor:
        """the requests' penalties, biases and masks on their rows of logits (requests without any: the rows stay, bit by bit)"""
        V, dev = logits.shape[1], logits.device
        words = (V + 31) // 32
        rules = np.tile(np.array([1.0, 0.0, 0.0, 0.0], np.float32), (len(requests), 1))
        hist, start, prompt, bias, bstart, mask = [], [0], [], [], [0], None
        for i, r in enumerate(requests):
            p = r.params
            if p.ruled():
                rules[i, :3] = p.repetition_penalty, p.presence_penalty, p.frequency_penalty
                if p.repetition_penalty != 1.0:
                    hist += r.prompt
                    prompt.append(len(r.prompt))
                else:
                    prompt.append(0)
                hist += r.output
                bias += [(t, v if v >= -F32_MAX else -np.inf) for t, v in (p.logit_bias or {}).items()]
                m = masks.get(r.rid if r.rid in masks or not r.siblings else r.siblings[0].rid)      # (a sample's first token: the mask of its prompt's request)
                if m is not None:
                    if mask is None:
                        mask = np.full((len(requests), words), -1, np.int32)
                    mask[i] = m
            else:
                prompt.append(0)
            start.append(len(hist))
            bstart.append(len(bias))
        up = lambda x, dt: torch.from_numpy(np.asarray(x, dt)).to(dev)
        kw = {}
        if hist:
            kw.update(hist=up(hist, np.int32), hist_start=up(start, np.int32), hist_prompt=up(prompt, np.int32))
        if bias:
            kw.update(bias_start=up(bstart, np.int32), bias_ids=up([t for t, _ in bias], np.int32), bias_vals=up([v for _, v in bias], np.float32))
        if mask is not None:
            kw.update(mask=torch.from_numpy(mask).to(dev))
        return seqops.process_logits(logits, up(rules, np.float32), torch.empty_like(logits), **kw)

    def _sample(self, logits: torch.Tensor, r: Request) -> int:
        p = r.params
        if p.temperature <= 0:
            ids = torch.empty(1, dtype=torch.int32, device=logits.device)
            seqops.argmax(logits.reshape(1, -1).contiguous(), ids)
            return int(ids.item())
        z = logits.float() / p.temperature
        if p.top_k and p.top_k < z.numel():
            kth = torch.topk(z, p.top_k).values[-1]
            z = torch.where(z < kth, torch.full_like(z, float("-inf")), z)
        pr = torch.softmax(z, 0)
        if p.top_p < 1.0:
            sp, si = torch.sort(pr, descending=True)
            keep = torch.cumsum(sp, 0) - sp < p.top_p
            pr = torch.zeros_like(pr).scatter(0, si[keep], sp[keep])
            pr = pr / pr.sum()
        return int(torch.multinomial(pr, 1, generator=r._gen).item())

    def generate(self, prompts: Sequence[Sequence[int]], params: Optional[SamplingParams] = None) -> List[List[int]]:
        """runs the prompts to completion through the scheduler (more prompts than slots queue up); returns the new tokens of each (params.n > 1: a list of
        its n samples)"""
        reqs: List[Request] = []
        try:
            for i, p in enumerate(prompts):
                reqs.append(self.add_request(f"g{self.steps}_{i}", p, params))
            while any(not q.finished for r in reqs for q in [r] + r.siblings):
                self.step()
            flags = seqops.error_flags()
            if flags:
                raise RuntimeError(f"device error flags {flags:#x} (1: KV position outside its block table, 2: a bounded wait ran out, 4: expert table entry out of range, "
                                   "8: a key or value beyond what a 4-bit cache holds, 16: a token id outside the vocabulary)")
        finally:                    # also what is left of them where a step fails
            for r in reqs:
                self._sample_ids.difference_update(f"{r.rid}#{i}" for i in range(1, r.params.n))
                for q in [r] + r.siblings:
                    if not q.finished:
                        (self.running if q in self.running else self.waiting).remove(q)
                        q.finished = True
                        self.release(q.rid)
                    del self.requests[q.rid]
        return [[q.output for q in [r] + r.siblings] if r.params.n > 1 else r.output for r in reqs]
