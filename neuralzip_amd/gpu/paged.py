"""Decoding of many requests with lengths of their own over a paged key-value
cache, on a Transformers decoder model, compressed or not: greedily, or sampled
at a temperature, with tokens drafted by the caller, behind shared prefixes.

PagedDecoder runs every new token of a step through the operators of
neuralzip_amd.gpu.serving: PageTables gives the tokens their pages, Rotary
norms, rotates and stores each layer's queries and keys, paged_attention
reads the pages and adjust_logits applies penalties and grammar masks. The
model's own Linears, norms and blocks do the rest, so a NeuralZipRuntime's
hooks decode the weights as in any forward. Prompts run through the model's
own forward, one at a time, and their keys and values are then stored into
the request's pages. A step never asks the device for anything, so that it
can be captured in a HIP graph (capture()) and replayed while requests grow.

Requests may begin with a prefix (add_prefix()), whose pages they share and
whose keys a step reads once for all of them. With `drafts`, a step takes that
many drafted tokens per request along, as certain ones (their drafter's
probabilities are not asked for), and verify_drafts keeps those that the model
would have answered; trim() takes the others' pages back. With `experts`, the
experts of a step's mixture-of-experts layers run through expert_mlp, which a
graph can hold, in place of the model's own.

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
from transformers.activations import ACT2FN

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


def _expert_modules(model, dtype):
    """The experts of a model's MoE layers, which expert_mlp computes: stacked
    weights gate_up_proj (experts, 2 * inter, hidden) and down_proj (experts,
    hidden, inter), SiLU and no bias."""
    found = [m for m in model.modules() if torch.is_tensor(getattr(m, "gate_up_proj", None))
             and torch.is_tensor(getattr(m, "down_proj", None))]
    if not found:
        raise ValueError("experts=True needs a model with mixture-of-experts layers.")
    for m in found:
        up, down = m.gate_up_proj, m.down_proj
        if up.dim() != 3 or down.dim() != 3 or up.shape != (down.shape[0], 2 * down.shape[2], down.shape[1]) \
                or up.dtype != dtype or down.dtype != dtype or up.shape[2] % 8 or down.shape[2] % 8 or up.shape[0] > 1024 \
                or not isinstance(getattr(m, "act_fn", None), (torch.nn.SiLU, type(ACT2FN["silu"]))) \
                or {name for name, _ in m.named_parameters()} != {"gate_up_proj", "down_proj"}:
            raise ValueError(f"expert_mlp does not compute {type(m).__name__}: it needs stacked weights of one type, sizes "
                             f"of a multiple of 8, SiLU and no bias.")
    return found


class PagedDecoder:
    """`requests` places for requests of at most `max_length` tokens, prompt
    and answer together, on pages of `page_size` tokens: `num_pages` of them
    for all requests and prefixes, or enough for all at full length.

    `repetition`, `frequency` and `presence` are adjust_logits' penalties,
    for all requests. With `grammar`, `masks` (int32, requests x ceil(vocab /
    32)) holds the tokens that each request may answer with next; it may be
    written between steps. All bits of a free place are set, at first and when
    its request ends.

    `temperature`: answers are sampled at it (0 or None: the likeliest token).
    `drafts`: drafted tokens that a request may bring to a step, at most;
    requests * (drafts + 1) is at most 2048. `prefixes`: places for prefixes of
    up to max_length tokens; requests and prefixes are then at most 2048 and
    1024. `experts`: steps run the experts of MoE layers by expert_mlp, the
    routers as the model has them. It is made for steps of few tokens: with more
    than some 64 of them, requests times drafts + 1, on wide experts, or some 1000
    on small ones, the model's own forward is faster."""

    def __init__(self, model, *, requests, max_length, page_size=16, num_pages=None, repetition=1.0, frequency=0.0,
                 presence=0.0, grammar=False, temperature=None, drafts=0, prefixes=0, experts=False):
        _check_model(model.config, max_length)
        if drafts < 0 or prefixes < 0:
            raise ValueError("drafts and prefixes must not be negative.")
        if drafts and grammar:
            raise ValueError("A mask holds for the next token only: drafts and a grammar do not go together.")
        if (drafts or prefixes) and (requests * (drafts + 1) > 2048 or prefixes > 1024):
            raise ValueError("requests * (drafts + 1) must be at most 2048 and prefixes at most 1024.")
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
        self._drafts_most, self.temperature = drafts, 0.0 if temperature is None else float(temperature)
        width, rows = -(-max_length // page_size), requests + prefixes
        # prefixes have the table rows behind the requests'
        self.tables = serving.PageTables(rows, width, page_size, rows * width if num_pages is None else num_pages,
                                         device=self.device)
        self._experts = _expert_modules(model, embedding.dtype) if experts else []
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
        tokens = requests * (drafts + 1)
        self._step = serving.Step(rows, tokens, self.device)
        none = torch.zeros(tokens, dtype=torch.int32, device=self.device)
        # the prefix that each request begins with (-1: none), and their lengths in whole pages
        self._prefix_of = [-1] * requests
        self._groups = {}
        if prefixes:
            self._groups = dict(groups=torch.full((rows,), -1, dtype=torch.int32, device=self.device),
                                shared=torch.zeros(prefixes, dtype=torch.int32, device=self.device))
        if drafts or prefixes:
            self._plan = serving.SharedPlan(none, heads=self.heads, kv_heads=self.kv_heads, requests=none, **self._groups)
        else:
            self._plan = serving.AttentionPlan(none, heads=self.heads, kv_heads=self.kv_heads)
        self._prefixes = [None] * prefixes            # their token ids
        self._live = torch.zeros(rows, dtype=torch.int32, device=self.device)   # 1: the request gets a token in a step
        # row `requests` of what is written by request takes what a step's unused rows write
        self._last = torch.zeros(requests + 1, dtype=torch.int64, device=self.device)
        # of the last step, and what it was given
        self._answers = torch.full((requests, drafts + 1) if drafts else (requests,), -1, dtype=torch.int64,
                                   device=self.device)
        self._drafted = torch.full((requests, drafts), -1, dtype=torch.int64, device=self.device)
        self._accept = torch.zeros(tokens, dtype=torch.float64, device=self.device)
        self._sample = torch.zeros(requests, dtype=torch.float64, device=self.device)
        self._temperatures = filled(self.temperature)
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

    def _checked(self, ids, before=0):
        """Token ids of a prompt or a prefix, behind `before` others, on the CPU."""
        ids = torch.as_tensor(ids, dtype=torch.int64)
        if ids.dim() != 1 or not 0 < ids.shape[0] <= self.max_length - before or int(ids.min()) < 0 \
                or int(ids.max()) >= self.vocab:
            raise ValueError(f"A prompt is a vector of 1 to {self.max_length - before} token ids below {self.vocab}.")
        return ids

    def _take_in(self, row, ids, cache, known):
        """Gives table row `row` pages for its tokens past the first ones it
        has, runs the model over `ids`, which follow the `known` tokens of
        `cache`, and stores all keys and values that the row has no page for
        yet; returns the logits. A row that fails is left as it was."""
        new = torch.zeros(self.tables.requests, dtype=torch.int32, device=self.device)
        held = int(self.tables.lengths[row])
        n = known + ids.shape[0] - held
        new[row] = n
        step = self.tables.extend(new, n)
        if int(step.status[row]) != serving.PAGES_OK:
            raise RuntimeError("There are not enough free pages for the prompt.")
        try:
            out = self.model(input_ids=ids[None], past_key_values=cache, use_cache=True)
            for layer, prompt in enumerate(out.past_key_values.layers):
                k, v = (t[0, :, held:].transpose(0, 1) for t in (prompt.keys, prompt.values))
                self._store(k, k, v, step.positions, step.slots, *self.cache[layer])
        except BaseException:
            self._give_back(row, held)   # a prompt that fails leaves no pages behind
            raise
        return out.logits

    def _give_back(self, row, held):
        """Takes a row's pages back, but for its first `held` tokens' (whole
        pages that it shares), and empties it."""
        if held:
            first = held // self.tables.page_size
            own = self.tables.tables[row, first:].clone()
            self.tables.tables[row, :own.shape[0]] = own
            self.tables.lengths[row] -= held
        done = torch.zeros(self.tables.requests, dtype=torch.bool, device=self.device)
        done[row] = True
        self.tables.release(done)

    @torch.no_grad()
    def add_prefix(self, ids):
        """Takes in a prefix (1-D token ids) that requests may begin with
        and returns its number."""
        ids = self._checked(ids)
        if None not in self._prefixes:
            raise RuntimeError("All prefixes' places are taken.")
        number = self._prefixes.index(None)
        self._take_in(self.requests + number, ids.to(self.device), DynamicCache(), 0)
        self._groups["shared"][number] = ids.shape[0] // self.tables.page_size * self.tables.page_size
        self._prefixes[number] = ids.to(self.device)
        return number

    def drop_prefix(self, number):
        """Ends a prefix that no request begins with any more."""
        if not 0 <= number < len(self._prefixes) or self._prefixes[number] is None:
            raise ValueError(f"There is no prefix {number}.")
        if number in self._prefix_of:
            raise ValueError(f"Requests begin with prefix {number}.")
        self._give_back(self.requests + number, 0)
        self._prefixes[number] = None

    def _prefix_cache(self, number):
        """A prefix's keys and values, out of its pages, as the model's cache."""
        cache, n, page = DynamicCache(), self._prefixes[number].shape[0], self.tables.page_size
        pages = self.tables.tables[self.requests + number, :-(-n // page)].long()
        for layer in range(len(self.layers)):
            keys, values = (t[pages].transpose(0, 1).reshape(self.kv_heads, -1, self.dim)[None, :, :n]
                            for t in self.cache[layer])
            cache.update(keys, values, layer)
        return cache

    @torch.no_grad()
    def add(self, ids, mask=None, prefix=None):
        """Takes in a prompt (1-D token ids), picks its first answer token
        and returns the request's place. `mask` (with `grammar`): the place's
        row of `masks` from the first answer token on. `prefix`: the number of
        a prefix that the prompt follows."""
        if prefix is not None and (not 0 <= prefix < len(self._prefixes) or self._prefixes[prefix] is None):
            raise ValueError(f"There is no prefix {prefix}.")
        before = 0 if prefix is None else self._prefixes[prefix].shape[0]
        ids = self._checked(ids, before)
        if mask is not None:
            if self.masks is None:
                raise ValueError("A mask needs grammar=True.")
            if not torch.is_tensor(mask) or mask.dtype != torch.int32 or mask.shape != self.masks.shape[1:]:
                raise ValueError(f"A mask is an int32 vector of {self.masks.shape[1]} words.")
        ids = ids.to(self.device)
        if all(self._taken):
            raise RuntimeError("All requests' places are taken.")
        place = self._taken.index(False)
        held = 0 if prefix is None else before // self.tables.page_size * self.tables.page_size
        if held:
            pages = held // self.tables.page_size
            self.tables.tables[place, :pages] = self.tables.tables[self.requests + prefix, :pages]
            self.tables.lengths[place] = held
        # (a cache of its own: one that the model makes may keep a window only)
        try:
            logits = self._take_in(place, ids, DynamicCache() if prefix is None else self._prefix_cache(prefix), before)
        except BaseException:
            self.tables.lengths[place] = 0
            raise
        try:
            if mask is not None:
                self.masks[place] = mask.to(self.device)
            n = before + ids.shape[0]
            if before:
                self._history[place, :before] = self._prefixes[prefix].int()
            self._history[place, before:n] = ids.int()
            self._prompts[place] = n
            rows = torch.full((1,), place, dtype=torch.int32, device=self.device)
            contexts = torch.full((1,), n, dtype=torch.int32, device=self.device)
            self._numbers(None)
            self._pick(logits[0, -1:], rows, contexts)
        except BaseException:
            self._give_back(place, held)   # a prompt that fails leaves no pages behind
            if mask is not None:
                self.masks[place] = -1
            raise
        if prefix is not None:
            self._groups["groups"][place] = prefix
            self._prefix_of[place] = prefix
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
        done = torch.zeros(self.tables.requests, dtype=torch.bool, device=self.device)
        for place in places:
            prefix = self._prefix_of[place]
            if prefix < 0:
                done[place] = True
            else:
                page = self.tables.page_size
                self._give_back(place, self._prefixes[prefix].shape[0] // page * page)
                self._groups["groups"][place] = -1
                self._prefix_of[place] = -1
            self._live[place] = 0
            if self.masks is not None:
                self.masks[place] = -1
        self.tables.release(done)
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
        """Attention over the pages while a step runs, and the experts' products."""
        def forward(layer, attention):
            return lambda hidden_states, *args, **kwargs: self._attend(layer, attention, hidden_states, *args, **kwargs)

        def mlp(experts):
            return lambda hidden, index, weights: serving.expert_mlp(
                hidden, index.contiguous(), weights.float().contiguous(), experts.gate_up_proj, experts.down_proj)
        modules = self._attentions + self._experts
        # (some modules may have a forward of their own already, as wrapped ones do)
        own = [module.__dict__.get("forward") for module in modules]
        for layer, attention in enumerate(self._attentions):
            attention.forward = forward(layer, attention)
        for experts in self._experts:
            experts.forward = mlp(experts)
        try:
            yield
        finally:
            for module, before in zip(modules, own):
                if before is None:
                    del module.forward
                else:
                    module.forward = before

    def _run(self):
        """One step, all of it on the device."""
        # pages may reach past max_length; the rotary tables and the histories do not
        room = self.max_length - self.tables.lengths
        wanted = self._live
        if self._drafts_most:
            given = (self._drafted >= 0).int().cumprod(1).sum(1, dtype=torch.int32)
            wanted = wanted * torch.nn.functional.pad(given + 1, (0, self.tables.requests - self.requests)).minimum(room)
        asked = torch.where(room > 0, wanted, 0)
        self.tables.extend(asked, self._step.max_tokens, out=self._step)
        step = self._step
        self._plan.update(step.contexts, requests=step.requests, **self._groups)
        body, rows = self.model.model, self._rows(step.requests)
        fed = self._last[rows]
        if self._drafts_most:
            drafted = torch.cat((self._last[:-1, None], self._drafted), 1)
            at = torch.arange(step.max_tokens, device=self.device) - step.starts[rows].long()
            fed = torch.where(step.requests < 0, 0, drafted[rows.clamp(max=self.requests - 1),
                                                            at.clamp(0, self._drafts_most)])
        # (a draft that is no token is fed as one, and refused)
        hidden = body.embed_tokens(fed.clamp(0, self.vocab - 1) if self._drafts_most else fed)[None]
        with self._paged():
            for layer in self.layers:
                hidden = layer(hidden)
                if isinstance(hidden, tuple):
                    hidden = hidden[0]
        logits = self.model.lm_head(body.norm(hidden))[0]
        if self._drafts_most:
            self._keep(logits, rows, fed)
            return
        self._pick(logits, step.requests, step.contexts)
        some = step.starts[:self.requests + 1].diff() > 0
        self._answers.copy_(torch.where(some, self._last[:self.requests], -1))

    def _keep(self, logits, rows, fed):
        """Verifies a step's drafts, takes back what was stored for those
        refused, and notes the answers."""
        step, n = self._step, self.requests
        # a row's history is what was fed up to it
        self._history[rows, torch.where(step.requests < 0, 0, step.positions).long()] = fed.int()
        logits = self._adjusted(logits, rows, step.requests, step.contexts)
        self.logits = logits
        starts = step.starts[:n + 1]
        accepted, following = serving.verify_drafts(logits, fed, starts, self._accept, self._sample,
                                                    temperature=self._temperatures)
        count, following = starts.diff(), following.clamp(min=0)
        kept = torch.where(count > 0, step.lengths[:n] - count + accepted + 1, step.lengths[:n])
        self.tables.trim(torch.cat((kept, step.lengths[n:])))
        some = count > 0
        self._last[:n] = torch.where(some, following, self._last[:n])
        owner = torch.where(some, torch.arange(n, device=self.device), n)   # (row n takes what is not to be written)
        self._history[owner, torch.where(some, kept, 0).long()] = following.int()
        place = torch.arange(self._drafts_most + 1, device=self.device)
        drafted = torch.cat((self._drafted, following[:, None]), 1)
        answers = torch.where(place < accepted[:, None], drafted, -1)
        answers = torch.where(place == accepted[:, None], following[:, None], answers)
        self._answers.copy_(torch.where(some[:, None], answers, -1))

    def _rows(self, requests):
        return torch.where(requests < 0, self.requests, requests).long()

    def _adjusted(self, logits, rows, requests, contexts):
        """The logits of rows of `requests` (-1: none) that make them `contexts` long."""
        adjust = {}
        if self._penalties:
            inside = rows.clamp(max=self.requests - 1)
            adjust.update({name: t[inside] for name, t in self._penalties.items()}, history=self._history[rows],
                          lengths=contexts, prompt_lengths=self._prompts[inside])
        if self.masks is not None:
            adjust.update(masks=self.masks, mask_rows=requests)
        return serving.adjust_logits(logits, **adjust) if adjust else logits

    def _pick(self, logits, requests, contexts):
        """Adjusts the logits of tokens that make their requests `contexts`
        long, one a request, and notes the likeliest next ones, or samples
        them."""
        rows = self._rows(requests)
        self.logits = logits = self._adjusted(logits, rows, requests, contexts)
        # (argmax of a row of 2^17 tokens or more clears counters by a memset; as a graph's last node it has given wrong
        # tokens from the second replay on. Of more rows than verify_drafts takes it needs none.)
        if self.temperature > 0 or (logits.is_cuda and logits.shape[0] <= 65535):
            # every row for itself, with its request's number
            one = torch.arange(rows.shape[0] + 1, dtype=torch.int32, device=self.device)
            at = rows.clamp(max=self.requests - 1)
            _, best = serving.verify_drafts(logits, rows, one, self._accept[:rows.shape[0]], self._sample[at],
                                            temperature=self._temperatures[at])
            best = best.clamp(min=0)
        else:
            best = logits.argmax(-1)
        self._last.index_copy_(0, rows, best)
        place = rows * self._history.shape[1] + contexts.long()
        self._history.view(-1).index_copy_(0, place, best.int())

    def _numbers(self, numbers):
        """Takes the step's random numbers, or draws them."""
        if numbers is None:
            if self.temperature > 0:
                self._accept.uniform_()
                self._sample.uniform_()
            return
        own, numbers = (self._accept, self._sample), tuple(numbers)
        if len(numbers) != 2 or any(not torch.is_tensor(given) or given.shape != t.shape or given.dtype != t.dtype
                                    for t, given in zip(own, numbers)):
            raise ValueError(f"numbers are float64 vectors of {self._accept.shape[0]} and {self.requests}.")
        for t, given in zip(own, numbers):
            t.copy_(given)

    @torch.no_grad()
    def step(self, drafts=None, *, numbers=None):
        """New tokens for every request; returns the tokens (a new int64
        tensor): one by place, or, with `drafts`, up to drafts + 1 by place,
        those accepted and the one after them, then -1. Requests at max_length,
        or without free pages for a token and their drafts, stay as they are:
        -1, as in free places.

        drafts (with the decoder's `drafts`): int64 (requests, drafts), by
        place, what a request's text is taken to go on with, -1 for none; the
        tokens after a -1 are not used. numbers: (accept, sample), float64 from
        [0, 1), requests * (drafts + 1) and requests of them, in place of
        torch's own. A step that raises leaves all requests as they were."""
        if drafts is not None:
            if not torch.is_tensor(drafts) or drafts.shape != self._drafted.shape or drafts.dtype != torch.int64 \
                    or not self._drafts_most:
                raise ValueError(f"drafts are int64 ({self.requests}, {self._drafts_most}).")
            self._drafted.copy_(drafts)
        else:
            self._drafted.fill_(-1)
        self._numbers(numbers)
        if self._graph is not None:
            self._graph.replay()
            self.logits = self._graph_logits
        else:
            pages = self.tables
            state = pages.lengths, pages.free, pages.n_free
            before = [t.clone() for t in state]
            try:
                self._run()
            except BaseException:
                # a step that fails changes no request (tables past the lengths mean nothing)
                for t, old in zip(state, before):
                    t.copy_(old)
                raise
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
        """`new_tokens` tokens for each prompt (as many prompts as
        there are free places); lists of token ids. `capture` replays the
        steps after the second from a HIP graph. Raises where the pages did
        not suffice for all."""
        if self._drafts_most:
            raise ValueError("generate() takes one token a step: it needs a decoder without drafts.")
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
