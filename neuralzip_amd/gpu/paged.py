"""Greedy decoding of many requests with lengths of their own over a paged
key-value cache, on a Transformers decoder model, compressed or not.

PagedDecoder runs every new token of a step through the operators of
neuralzip_amd.gpu.serving: PageTables gives the tokens their pages, Rotary
norms, rotates and stores each layer's queries and keys, paged_attention
reads the pages and adjust_logits applies penalties and grammar masks. The
model's own Linears, norms and blocks do the rest, so a NeuralZipRuntime's
hooks decode the weights as in any forward. Prompts run through the model's
own forward, one at a time, and their keys and values are then stored into
the request's pages. A step never asks the device for anything, so that it
can be captured in a HIP graph (capture()) and replayed while requests grow.

Models are Llama-like, of the types in MODEL_TYPES:
model.model.{embed_tokens, layers, norm, rotary_emb} and model.lm_head, layers
with self_attn.{q,k,v,o}_proj and, optionally, RMS norms q_norm and k_norm over
a head, without a sliding window shorter than max_length. Others are refused.
The reference has no counterpart (its
forwards keep Transformers' cache, neuralzip/gpu/inference.py:476-509).
"""
import contextlib

import torch
from transformers import DynamicCache

from neuralzip_amd.gpu import serving
from neuralzip_amd.gpu.inference import RUNTIME_ATTRIBUTE

# Rotary tables that depend on the length they are asked for.
_GROWING_ROPES = ("dynamic", "longrope")
# Model types whose forward is what a step here computes: layers over the
# embeddings as they are, pairs (i, i + rotary_dim / 2) rotated in every layer,
# lm_head's products as logits. Each is compared with its own forward by
# tests/test_paged_decoder.py. Others may have the same modules and differ
# (neighbouring pairs, layers without rotation, scaled logits).
MODEL_TYPES = frozenset((
    "apertus", "arcee", "aria_text", "dots1", "exaone4", "gemma", "glm4_moe", "granite", "granitemoe",
    "granitemoeshared", "hy_v3", "hyperclovax", "jais2", "llama", "mistral", "mixtral", "nemotron", "olmo", "phimoe",
    "qwen2", "qwen2_moe", "qwen3", "qwen3_moe", "seed_oss", "solar_open", "stablelm", "starcoder2"))
# Settings of theirs that a step does not follow, with the values that change nothing.
_PLAIN_SETTINGS = {"embedding_multiplier": (None, 1), "logits_scaling": (None, 1), "clip_qkv": (None,),
                   "qk_layernorm": (None, False)}


def _check_model(config, max_length):
    """Refuses models that a step would compute otherwise than they do."""
    kind = getattr(config, "model_type", None)
    if kind not in MODEL_TYPES:
        raise ValueError(f"PagedDecoder runs models of the types {', '.join(sorted(MODEL_TYPES))}; this one is "
                         f"{kind!r}, whose forward may differ.")
    for name, plain in _PLAIN_SETTINGS.items():
        if getattr(config, name, None) not in plain:
            raise ValueError(f"PagedDecoder does not follow {name}={getattr(config, name)!r} of this {kind} model.")
    # (where layers differ, as layer_types says, their attention modules have the windows)
    window = getattr(config, "sliding_window", None)
    if window is not None and getattr(config, "use_sliding_window", True) and window < max_length \
            and getattr(config, "layer_types", None) is None:
        raise ValueError(f"PagedDecoder attends to whole contexts; this model has a sliding window of {window} tokens, "
                         f"less than max_length.")


class PagedDecoder:
    """`requests` places for requests of at most `max_length` tokens, prompt
    and answer together, on pages of `page_size` tokens: `num_pages` of them
    for all requests, or enough for all at full length.

    `repetition`, `frequency` and `presence` are adjust_logits' penalties,
    for all requests. With `grammar`, `masks` (int32, requests x ceil(vocab /
    32)) holds the tokens that each request may answer with next; it may be
    written between steps. All bits of a free place are set, at first and when
    its request ends."""

    def __init__(self, model, *, requests, max_length, page_size=16, num_pages=None, repetition=1.0, frequency=0.0,
                 presence=0.0, grammar=False):
        _check_model(model.config, max_length)
        body = model.model
        self.model, self.layers = model, list(body.layers)
        self._attentions = [layer.self_attn for layer in self.layers]
        first = self._attentions[0]
        for attention in self._attentions:
            for name in ("q_proj", "k_proj", "v_proj", "o_proj", "head_dim"):
                if not hasattr(attention, name):
                    raise ValueError(f"PagedDecoder needs Llama-like attention modules; {type(attention).__name__} "
                                     f"has no {name}.")
            if getattr(attention, "sliding_window", None) is not None:
                raise ValueError("PagedDecoder attends to whole contexts; this model's layers have a sliding window.")
        if getattr(body.rotary_emb, "rope_type", "default") in _GROWING_ROPES:
            raise ValueError("PagedDecoder needs rotary tables that do not depend on the length.")
        embedding = body.embed_tokens.weight
        self.device, dtype = embedding.device, embedding.dtype
        self.dim = first.head_dim
        self.kv_heads = model.config.num_key_value_heads
        self.heads = model.config.num_attention_heads
        self.requests, self.max_length, self.vocab = requests, max_length, model.config.vocab_size
        width = -(-max_length // page_size)
        self.tables = serving.PageTables(requests, width, page_size, requests * width if num_pages is None else num_pages,
                                         device=self.device)
        # one allocation for all layers: (layers, keys and values, pages, heads, places, elements)
        self.cache = torch.zeros((len(self.layers), 2, self.tables.num_pages, self.kv_heads, page_size, self.dim),
                                 dtype=dtype, device=self.device)
        positions = torch.arange(max_length, device=self.device)[None]
        cos, sin = body.rotary_emb(torch.zeros(1, dtype=torch.float32, device=self.device), positions)
        half = cos.shape[-1] // 2
        cos, sin = (t[0, :, :half].float().contiguous() for t in (cos, sin))
        self._rotaries = []
        for attention in self._attentions:
            q_norm, k_norm = getattr(attention, "q_norm", None), getattr(attention, "k_norm", None)
            weights = {} if q_norm is None else dict(q_weight=q_norm.weight.detach(), k_weight=k_norm.weight.detach(),
                                                     eps=q_norm.variance_epsilon)
            self._rotaries.append(serving.Rotary(cos, sin, **weights))
        # prompts' keys are rotated already: a rotation of no elements stores them
        self._store = serving.Rotary(cos[:, :0].contiguous(), sin[:, :0].contiguous())

        def filled(value, dtype=torch.float32):
            return torch.full((requests,), value, dtype=dtype, device=self.device)
        self._step = serving.Step(requests, requests, self.device)
        self._plan = serving.AttentionPlan(filled(0, torch.int32), heads=self.heads, kv_heads=self.kv_heads)
        self._live = filled(0, torch.int32)           # 1: the request gets a token in a step
        # row `requests` of what is written by request takes what a step's unused rows write
        self._last = torch.zeros(requests + 1, dtype=torch.int64, device=self.device)
        self._answers = torch.full((requests,), -1, dtype=torch.int64, device=self.device)   # of the last step
        self._history = torch.zeros((requests + 1, max_length + 1), dtype=torch.int32, device=self.device)
        self._prompts = filled(0, torch.int32)
        self._penalties = {}
        if (repetition, frequency, presence) != (1.0, 0.0, 0.0):
            self._penalties = dict(repetition=filled(repetition), frequency=filled(frequency),
                                   presence=filled(presence))
        self.masks = torch.full((requests, (self.vocab + 31) // 32), -1, dtype=torch.int32,
                                device=self.device) if grammar else None
        # of the last step, in token order, or of the prompt taken in since, as
        # adjusted; a step replayed from a graph writes the last one's anew
        self.logits = None
        self._graph = self._graph_logits = None
        self._taken = [False] * requests

    # --------------------------------------------------------------- requests

    @torch.no_grad()
    def add(self, ids, mask=None):
        """Takes in a prompt (1-D token ids), picks its first answer token
        and returns the request's place. `mask` (with `grammar`): the place's
        row of `masks` from the first answer token on."""
        ids = torch.as_tensor(ids, dtype=torch.int64)
        if ids.dim() != 1 or not 0 < ids.shape[0] <= self.max_length or int(ids.min()) < 0 \
                or int(ids.max()) >= self.vocab:
            raise ValueError(f"A prompt is a vector of 1 to {self.max_length} token ids below {self.vocab}.")
        if mask is not None:
            if self.masks is None:
                raise ValueError("A mask needs grammar=True.")
            if not torch.is_tensor(mask) or mask.dtype != torch.int32 or mask.shape != self.masks.shape[1:]:
                raise ValueError(f"A mask is an int32 vector of {self.masks.shape[1]} words.")
        ids, n = ids.to(self.device), ids.shape[0]
        if all(self._taken):
            raise RuntimeError("All requests' places are taken.")
        place = self._taken.index(False)
        new = torch.zeros(self.requests, dtype=torch.int32, device=self.device)
        new[place] = n
        step = self.tables.extend(new, n)
        if int(step.status[place]) != serving.PAGES_OK:
            raise RuntimeError("There are not enough free pages for the prompt.")
        try:
            # (a cache of its own: one that the model makes may keep a window only)
            out = self.model(input_ids=ids[None], past_key_values=DynamicCache(), use_cache=True)
            for layer, prompt in enumerate(out.past_key_values.layers):
                k, v = (t[0].transpose(0, 1) for t in (prompt.keys, prompt.values))
                self._store(k, k, v, step.positions, step.slots, *self.cache[layer])
            if mask is not None:
                self.masks[place] = mask.to(self.device)
            self._history[place, :n] = ids.int()
            self._prompts[place] = n
            rows = torch.full((1,), place, dtype=torch.int32, device=self.device)
            contexts = torch.full((1,), n, dtype=torch.int32, device=self.device)
            self._pick(out.logits[0, -1:], rows, contexts)
        except BaseException:
            self.tables.release(new > 0)   # a prompt that fails leaves no pages behind
            if mask is not None:
                self.masks[place] = -1
            raise
        self._live[place] = 1
        self._taken[place] = True
        return place

    def finish(self, *places):
        """Ends requests: their pages and places are free again."""
        for place in places:
            if not 0 <= place < self.requests or not self._taken[place]:
                raise ValueError(f"Place {place} holds no request.")
        if len(set(places)) < len(places):
            raise ValueError("A place is named twice.")
        done = torch.zeros(self.requests, dtype=torch.bool, device=self.device)
        for place in places:
            done[place] = True
        self.tables.release(done)
        self._live.masked_fill_(done, 0)
        if self.masks is not None:
            self.masks.masked_fill_(done[:, None], -1)
        for place in places:
            self._taken[place] = False

    @property
    def tokens(self):
        """The last token of every request's answer, the one that add()
        picked among them (a new int64 tensor, by place)."""
        return self._last[:self.requests].clone()

    # ------------------------------------------------------------------ steps

    def _attend(self, layer, attention, hidden, *args, **kwargs):
        """The attention module's forward during a step: hidden is (1, tokens, size)."""
        tokens = hidden.shape[1]
        q, k, v = (proj(hidden)[0].view(tokens, -1, self.dim) for proj in
                   (attention.q_proj, attention.k_proj, attention.v_proj))
        cache = self.cache[layer]
        q = self._rotaries[layer](q, k, v, self._step.positions, self._step.slots, *cache)
        scale = getattr(attention, "scaling", None)
        out = serving.paged_attention(q, *cache, self.tables.tables, self._plan, scale=scale)
        return attention.o_proj(out.view(1, tokens, -1)), None

    @contextlib.contextmanager
    def _paged(self):
        """Attention over the pages while a step runs."""
        def forward(layer, attention):
            return lambda hidden_states, *args, **kwargs: self._attend(layer, attention, hidden_states, *args, **kwargs)
        # (some modules may have a forward of their own already, as wrapped ones do)
        own = [attention.__dict__.get("forward") for attention in self._attentions]
        for layer, attention in enumerate(self._attentions):
            attention.forward = forward(layer, attention)
        try:
            yield
        finally:
            for attention, before in zip(self._attentions, own):
                if before is None:
                    del attention.forward
                else:
                    attention.forward = before

    def _run(self):
        """One step, all of it on the device."""
        # pages may reach past max_length; the rotary tables and the histories do not
        asked = torch.where(self.tables.lengths < self.max_length, self._live, 0)
        self.tables.extend(asked, self.requests, out=self._step)
        step = self._step
        self._plan.update(step.contexts, requests=step.requests)
        body, rows = self.model.model, self._rows(step.requests)
        hidden = body.embed_tokens(self._last[rows])[None]
        with self._paged():
            for layer in self.layers:
                hidden = layer(hidden)
                if isinstance(hidden, tuple):
                    hidden = hidden[0]
        logits = self.model.lm_head(body.norm(hidden))[0]
        self._pick(logits, step.requests, step.contexts)
        self._answers.copy_(torch.where(step.starts.diff() > 0, self._last[:self.requests], -1))

    def _rows(self, requests):
        return torch.where(requests < 0, self.requests, requests).long()

    def _pick(self, logits, requests, contexts):
        """Adjusts the logits of tokens that make their requests `contexts`
        long, and notes the likeliest next ones."""
        rows = self._rows(requests)
        adjust = {}
        if self._penalties:
            inside = rows.clamp(max=self.requests - 1)
            adjust.update({name: t[inside] for name, t in self._penalties.items()}, history=self._history[rows],
                          lengths=contexts, prompt_lengths=self._prompts[inside])
        if self.masks is not None:
            adjust.update(masks=self.masks, mask_rows=requests)
        if adjust:
            logits = serving.adjust_logits(logits, **adjust)
        self.logits = logits
        best = logits.argmax(-1)
        self._last.index_copy_(0, rows, best)
        place = rows * self._history.shape[1] + contexts.long()
        self._history.view(-1).index_copy_(0, place, best.int())

    @torch.no_grad()
    def step(self):
        """One new token for every request; returns the tokens (a new int64
        tensor, by place). Requests at max_length, or for which no page is free, stay as
        they are: -1, as in free places."""
        if self._graph is not None:
            self._graph.replay()
            self.logits = self._graph_logits
        else:
            self._run()
        return self._answers.clone()

    @torch.no_grad()
    def capture(self):
        """Captures the step in a HIP graph, which step() replays from then
        on. A step should have run eagerly before."""
        runtime = getattr(self.model, RUNTIME_ATTRIBUTE, None)
        graph, before = torch.cuda.CUDAGraph(), self.logits
        try:
            with runtime.graph_capture() if runtime is not None else contextlib.nullcontext(), torch.cuda.graph(graph):
                self._run()
            self._graph, self._graph_logits = graph, self.logits
        finally:
            self.logits = before   # nothing has run yet: the last step's still

    def generate(self, prompts, new_tokens, *, capture=False):
        """`new_tokens` greedy tokens for each prompt (as many prompts as
        there are free places); lists of token ids. `capture` replays the
        steps after the second from a HIP graph. Raises where the pages did
        not suffice for all."""
        if new_tokens < 1 or any(len(p) + new_tokens - 1 > self.max_length for p in prompts):
            raise ValueError("Prompts and answers must fit max_length.")
        if len(prompts) > self._taken.count(False):
            raise RuntimeError("There are more prompts than free places.")
        places = []
        try:
            for p in prompts:
                places.append(self.add(p))
            tokens = [self.tokens]
            for i in range(new_tokens - 1):
                if capture and i == 2 and self._graph is None:
                    self.capture()
                tokens.append(self.step())
            lengths = self.tables.lengths[places].tolist()
            answers = torch.stack(tokens, 1)[places].tolist()
        finally:
            self.finish(*places)
        if lengths != [len(p) + new_tokens - 1 for p in prompts]:
            raise RuntimeError("The pages ran out before all requests had their tokens.")
        return answers
