"""Serving loop over a paged cache: requests of different lengths share the device step by step.

The reference generates for one batch at a time, every sequence in a row of the dense cache (model.py:313-396).  Here a
step holds one token of every request that generates and, in the rows that are left, the next piece of prompts that wait, one
request's rows behind another's.  Keys and values are in pages; a request has the pages of its prompt and its answer from the
moment it is admitted until it ends.

What a step works with lies in device tensors (tokens, q_offsets, kv_lens, page_table: see flash_attention_paged), written with
one copy from the host.  A step in which every request generates has one row for each and is replayed from a HIP graph, recorded
once per number of rows rounded up to a power of two; rows beyond the requests are no sequence's token.

Measured on the 1B architecture (python paged_serving.py), 64 requests of 16 .. 1000 prompt ids (five lengths, drawn) and 128
greedy tokens each: 26.4 k generated tokens/s with 512 rows to a step, 33.8 k with 2048, 36.4 k with 8192 (prompt passes included).
generate_graphed, which takes every prompt's tokens behind the shortest one's length one by one, gives 6.2 k on the same requests.
One request alone: 1.15 k, generate_graphed 1.9 k (up to four sequences its step is one launch; the steps here are operators one by
one).
"""

import gc
import random
import threading
import time
from collections import deque

import torch
import torch.nn.functional as F

from llama_arch import LlamaDecoder


class _Request:
    def __init__(self, index, prompt, limit):
        self.index, self.tokens, self.prompt_len, self.limit = index, list(prompt), len(prompt), limit
        self.cached = 0         # tokens whose keys and values are in the cache
        self.pages = []


class _Step:
    """Device tensors that describe a step of at most `rows` rows and `sequences` sequences: one buffer, one copy."""

    def __init__(self, rows, sequences, most_pages, device):
        self.rows, self.sequences, self.most_pages = rows, sequences, most_pages
        sizes = (rows, sequences + 1, sequences, sequences, sequences * most_pages)
        self.host = torch.zeros(sum(sizes), dtype=torch.int32, pin_memory=device.type == "cuda")
        self.device = torch.zeros(sum(sizes), dtype=torch.int32, device=device)
        self.tokens, self.q_offsets, self.kv_lens, self.last_rows, pages = self.device.split(sizes)
        self.page_table = pages.view(sequences, most_pages)
        self._host = tuple(t.numpy() for t in self.host.split(sizes))

    def fill(self, plan):
        """plan: (request, new tokens) one behind the other."""
        tokens, q_offsets, kv_lens, last_rows, pages = self._host
        for t in self._host:
            t[:] = 0
        at = 0
        for b, (r, n) in enumerate(plan):
            tokens[at:at + n] = r.tokens[r.cached:r.cached + n]
            at += n
            q_offsets[b + 1:] = at
            kv_lens[b] = r.cached + n
            last_rows[b] = at - 1
            pages[b * self.most_pages:b * self.most_pages + len(r.pages)] = r.pages
        self.device.copy_(self.host, non_blocking=True)


class PagedServer:
    """model: a LlamaDecoder whose operator module has the paged operators.  pages x page_size tokens of cache per layer;
    at most `max_sequences` requests at once and `max_rows` new tokens in a step.  The pages, the steps' tensors and the recorded
    steps are those of one generate() at a time: calls from several threads take turns."""

    def __init__(self, model: LlamaDecoder, pages: int, page_size: int = 64, max_sequences: int = 64, max_rows: int = 2048,
                 graphs: bool = True):
        if page_size < 8 or page_size & (page_size - 1):
            raise ValueError("page_size is a power of two from 8 on")
        if not 0 < max_sequences <= max_rows or pages < 1:
            raise ValueError("a step has rows for its sequences, a cache has pages")
        self.model, self.page_size, self.max_sequences, self.max_rows = model, page_size, max_sequences, max_rows
        c, dev = model.config, model.device
        self.most_pages = min(pages, -(-c.block_size // page_size))
        self.k_pages, self.v_pages = (
            [torch.zeros((pages, page_size, c.n_kv_head, model.hd), dtype=model.dtype, device=dev) for _ in range(c.n_layer)]
            for _ in range(2))
        self.free = deque(range(pages))
        self.graphs = {} if graphs and dev.type == "cuda" else None      # rows -> what _record returns
        self._recorded_of = None
        self._turn = threading.Lock()
        self.steps = {"mixed": 0, "generating": 0}

    # ------------------------------------------------------------------ one step on the device
    def _forward(self, step: _Step, max_new: int, every_row: bool):
        """The tokens that follow the sequences' last rows (or every row, where a sequence has no other)."""
        m, c, ops = self.model, self.model.config, self.model.ops
        where = (step.page_table, step.q_offsets, step.kv_lens)

        def attention(i, L, qkv):
            q = ops.rot_embed_append_paged(qkv, m.freqs_cis, self.k_pages[i], self.v_pages[i], *where, c.n_head, L.get("q_norm"),
                                           L.get("k_norm"), c.norm_eps)
            return ops.flash_attention_paged(q, self.k_pages[i], self.v_pages[i], *where, max_new)

        x = F.embedding(step.tokens, m.wte)
        if every_row and m.decode_linear_rows > 0 and m.FUSED_MAX_ROWS < step.rows <= m.QKV_FUSED_MAX_ROWS and self._streaming_linears():
            # the linears of a dense decode step of as many sequences
            x = x.unsqueeze(1)
            h = ops.rms_norm(x, m.layers[0]["ln_1"], c.norm_eps)
            for i, L in enumerate(m.layers):
                y = attention(i, L, ops.linear_decode(h, L["c_attn"])[:, 0]).reshape(-1, 1, c.n_embd)
                x, h = ops.add_rms_norm_partials(x, ops.linear_splitk(y, L["c_proj"]), L["ln_2"], c.norm_eps)
                t = m._swiglu(h, L["c_fc2"], L["c_fc"])
                next_norm = m.layers[i + 1]["ln_1"] if i + 1 < len(m.layers) else m.ln_f
                x, h = ops.add_rms_norm_partials(x, ops.linear_splitk(t, L["mlp_proj"]), next_norm, c.norm_eps)
            return ops.argmax(m._vocabulary(h[:, 0]))
        x = x.unsqueeze(0)
        h = ops.rms_norm(x, m.layers[0]["ln_1"], c.norm_eps)
        for i, L in enumerate(m.layers):
            y = attention(i, L, m._linear(h, L["c_attn"])[0]).reshape(1, -1, c.n_embd)
            x, h = m._add_norm(x, m._linear(y, L["c_proj"]), L["ln_2"])
            next_norm = m.layers[i + 1]["ln_1"] if i + 1 < len(m.layers) else m.ln_f
            x, h = m._add_norm(x, m._mlp(L, h), next_norm)
        h = h[0] if every_row else h[0].index_select(0, step.last_rows)
        logits = m._linear(h, m.wte)
        return ops.argmax(logits) if hasattr(ops, "argmax") else torch.argmax(logits, dim=-1)

    def _streaming_linears(self):
        """Whether the linears of 5 to 64 rows take the model's projections: whole chunks of 128 and dense 16-byte rows.  (The
        other steps' linears take more; LlamaDecoder._swiglu and _vocabulary see to theirs.)"""
        return hasattr(self.model.ops, "linear_splitk") and all(
            w.shape[1] % 128 == 0 and w.shape[0] % 8 == 0 and w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0
            for L in self.model.layers for w in (L["c_attn"], L["c_proj"], L["mlp_proj"]))

    def _drop_outdated(self):
        """Recorded steps hold the model's tensors by address and the choice of its linears: they go when either is another.
        (Looked at once per generate(): the model stays as it is during one.)"""
        m = self.model
        tensors = [m.wte, m.ln_f, m.freqs_cis, *(t for L in m.layers for name, t in L.items() if not name.startswith("cache_"))]
        now = m.ops, m.decode_linear_rows, [(t.data_ptr(), t.shape, t.stride()) for t in tensors]
        if now != self._recorded_of:
            if self.graphs:
                self.graphs.clear()
            self._recorded_of = now

    def _run(self, plan):
        rows = sum(n for _, n in plan)
        if rows == len(plan) and self.graphs is not None:
            self.steps["generating"] += 1
            rows = min(self.max_sequences, 1 << (rows - 1).bit_length())
            recorded = rows in self.graphs
            graph, step, out = self.graphs[rows] if recorded else (None, _Step(rows, rows, self.most_pages, self.model.device), None)
            step.fill(plan)
            if not recorded:
                graph, _, out = self.graphs[rows] = self._record(step)
            if graph is not None:
                graph.replay()
            else:
                out = self._forward(step, 1, True)
        else:
            self.steps["mixed"] += 1
            step = _Step(rows, len(plan), self.most_pages, self.model.device)
            step.fill(plan)
            out = self._forward(step, max(n for _, n in plan), False)
        return out.tolist()[:len(plan)]       # (waits for the step: its buffers are the host's again)

    def _record(self, step):
        """(graph, step, tokens that follow) of a generating step.  Run again a step writes what it wrote, so the recording is
        checked as GraphedDecodeLoop checks a prompt pass: it is used only after two replays gave the eager pass's tokens,
        with eager work in between (library products may record nodes that misbehave on later replays)."""
        dev = self.model.device
        ref = self._forward(step, 1, True).clone()      # eager: also the warm-up for the capture
        torch.cuda.synchronize(dev)
        gc.collect()      # (nothing may be collected while the stream is capturing)
        gc_was_enabled = gc.isenabled()
        gc.disable()
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = self._forward(step, 1, True)
        finally:
            if gc_was_enabled:
                gc.enable()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize(dev)
            if not torch.equal(out, ref) or not torch.equal(self._forward(step, 1, True), ref):
                return None, step, None
        return graph, step, out

    # ------------------------------------------------------------------------------- requests
    def _pages_for(self, request):
        # (the last token of an answer is never in the cache)
        return max(1, -(-(request.limit - 1) // self.page_size))

    def _plan(self, running):
        """One token of everyone who generates, then pieces of prompts in the order of their arrival."""
        left = self.max_rows - sum(len(r.tokens) - r.cached == 1 for r in running)
        plan = []
        for r in running:
            waiting = len(r.tokens) - r.cached
            n = 1 if waiting == 1 else min(waiting, left)
            left -= n if waiting > 1 else 0
            if n > 0:
                plan.append((r, n))
        return plan

    def generate(self, prompt_tokens, max_gen_len, echo=False, ignore_eos=False):
        """Greedy answers of LlamaDecoder.generate (each prompt a non-empty list of ids), requests admitted in order as pages
        become free."""
        with self._turn, torch.inference_mode():
            return self._generate(prompt_tokens, max_gen_len, echo, ignore_eos)

    def _generate(self, prompt_tokens, max_gen_len, echo, ignore_eos):
        self._drop_outdated()
        c, stop = self.model.config, set(self.model.tokenizer.stop_tokens)
        requests = [_Request(i, p, min(c.block_size, len(p) + max_gen_len)) for i, p in enumerate(prompt_tokens)]
        for r in requests:
            if not 0 < r.prompt_len <= c.block_size:
                raise ValueError(f"prompt {r.index} has {r.prompt_len} tokens, of 1 .. {c.block_size}")
            if min(r.tokens) < 0 or max(r.tokens) >= c.vocab_size:
                raise IndexError(f"token id outside the vocabulary of {c.vocab_size}")
            if self._pages_for(r) > len(self.free):
                raise ValueError(f"prompt {r.index} and its answer need {self._pages_for(r)} pages of {len(self.free)}")
        waiting, running = deque(r for r in requests if r.limit > r.prompt_len), []
        try:
            while waiting or running:
                while waiting and len(running) < self.max_sequences and self._pages_for(waiting[0]) <= len(self.free):
                    r = waiting.popleft()
                    r.pages = [self.free.popleft() for _ in range(self._pages_for(r))]
                    running.append(r)
                plan = self._plan(running)
                for (r, n), token in zip(plan, self._run(plan)):
                    r.cached += n
                    if r.cached == len(r.tokens):
                        r.tokens.append(token)
                        if len(r.tokens) == r.limit or (token in stop and not ignore_eos):
                            running.remove(r)
                            self._release(r)
        finally:
            for r in running:
                self._release(r)
        out = []
        for r in requests:
            toks = r.tokens if echo else r.tokens[r.prompt_len:]
            for s in self.model.tokenizer.stop_tokens:
                if s in toks and not ignore_eos:
                    toks = toks[:toks.index(s)]
            out.append(toks)
        return out

    def _release(self, request):
        self.free.extend(request.pages)
        request.pages = []


def timed_serving(generate, prompts, max_gen_len, repeats=3):
    """Generated tokens/s of a generate(prompts, max_gen_len, ignore_eos=True), prompt passes included: best of `repeats` behind
    one that records the steps."""
    best = 0.0
    for i in range(repeats + 1):
        torch.cuda.synchronize()
        begin = time.perf_counter()
        answers = generate(prompts, max_gen_len, ignore_eos=True)      # (ends with the last tokens on the host)
        if i > 0:
            best = max(best, sum(map(len, answers)) / (time.perf_counter() - begin))
    return best


if __name__ == "__main__":      # the figures above
    from custom_kernels import custom_kernels_extension
    from llama_arch import LlamaConfig, random_prompts

    draw = random.Random(0)
    every_prompt = [random_prompts(1, draw.choice((16, 64, 200, 500, 1000)), 128000, i)[0] for i in range(64)]
    model = LlamaDecoder(LlamaConfig(max_model_len=1300, max_gen_batch_size=64), custom_kernels_extension, "cuda")
    for prompts in every_prompt, every_prompt[:1]:
        loops = {f"{rows} rows to a step": PagedServer(model, len(prompts) * 20, max_rows=rows).generate for rows in (512, 2048, 8192)}
        for name, generate in {**loops, "generate_graphed": model.generate_graphed}.items():
            print(f"{len(prompts)} requests, {name}: {timed_serving(generate, prompts, 128):.0f} tokens/s", flush=True)
