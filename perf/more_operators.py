"""More operators of a serving step and the cases they are measured on: what a
step needs whose requests share a long prefix, bring drafted tokens along or
run through experts.

  shared     attention over the paged key-value cache for requests that begin
             with the same pages, and for several rows of one request
  verify     drafted tokens against the model's probabilities, from given
             random numbers, and the token after the last one kept
  trim       pages past the tokens that a verification kept, back onto the
             stack of free ones
  experts    a mixture-of-experts layer for a few tokens: the router's choice
             and the chosen experts' products

Where `own` is false the operators run in plain torch, in 32 bits (the choices
of tokens and experts in 64, where sums lie next to a border); where it is
true, as neuralzip_amd.gpu.serving's calls. `exact` is the definition in 64
bits (whole numbers: in loops over requests).
"""
import math
import random

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One request of the Llama-3-8B shape, 2000 tokens in, with four
        # drafted tokens: five rows over the same keys, all latency.
        dict(name="shared-8b-one-drafts", kind="shared", dtype="bf16", requests=1, tokens=5, prefixes=0, prefix=0,
             loner=0, low=2005, high=2005, spread="linear", empty=0, heads=32, kv_heads=8, dim=128, page=16),
        # 32 chats of the same shape behind one system prompt, one of them
        # without it, one token each.
        dict(name="shared-8b-prefix-32", kind="shared", dtype="bf16", requests=32, tokens=1, prefixes=1, prefix=8190,
             loner=32, low=1, high=2000, spread="linear", empty=0, heads=32, kv_heads=8, dim=128, page=16),
        # 14 documents of the Qwen2-0.5B shape in fp32, three drafted tokens
        # each, idle places among them.
        dict(name="shared-qwen-drafts-fp32", kind="shared", dtype="fp32", requests=14, tokens=4, prefixes=0, prefix=0,
             loner=0, low=100, high=9001, spread="linear", empty=7, heads=14, kv_heads=2, dim=64, page=64),
        # The largest: 64 requests of the Llama-3-70B shape over three long
        # documents, one drafted token each.
        dict(name="shared-70b-prefix-64", kind="shared", dtype="fp16", requests=64, tokens=2, prefixes=3, prefix=16384,
             loner=0, low=2, high=2500, spread="linear", empty=0, heads=64, kv_heads=8, dim=128, page=32),
        # One request of the Qwen2-0.5B shape without drafts: plain sampling
        # from one row of logits. Latency.
        dict(name="verify-qwen-one", kind="verify", dtype="bf16", requests=1, low=0, high=0, vocab=151936, probs=False,
             greedy=0, empty=0),
        # 32 requests of the Llama-3-8B shape with up to five tokens drafted
        # from their own texts (certain drafts), a quarter of them greedy.
        dict(name="verify-8b-texts-32", kind="verify", dtype="bf16", requests=32, low=0, high=5, vocab=128256,
             probs=False, greedy=4, empty=11),
        # 48 requests with four tokens of a draft model and its probabilities,
        # logits in 32 bits.
        dict(name="verify-8b-model-48", kind="verify", dtype="fp32", requests=48, low=4, high=4, vocab=128256,
             probs=True, greedy=0, empty=0),
        # The refused drafts' pages of 32 requests, and of 1000.
        dict(name="trim-32", kind="trim", requests=32, page=16, low=1, high=4096, drop=5, empty=0),
        dict(name="trim-1000", kind="trim", requests=1000, page=32, low=1, high=32768, drop=3000, empty=7),
        # One token through a layer of many small experts. Latency, and
        # the chosen experts' weights.
        dict(name="experts-small-one", kind="experts", dtype="bf16", tokens=1, hidden=2048, inter=768, experts=128, top=8,
             scoring="softmax", normalize=True, bias=False),
        # 21 tokens in fp32 over sixteen experts of odd sizes, scored one by one.
        dict(name="experts-odd-21-fp32", kind="experts", dtype="fp32", tokens=21, hidden=1096, inter=520, experts=16,
             top=3, scoring="sigmoid", normalize=True, bias=True),
        # 32 requests' tokens through eight experts as wide as Llama-3-8B's MLP.
        dict(name="experts-8b-32", kind="experts", dtype="bf16", tokens=32, hidden=4096, inter=14336, experts=8, top=2,
             scoring="softmax", normalize=True, bias=False),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((32, 8, 128), (14, 2, 64), (64, 8, 128), (8, 8, 64), (12, 1, 96), (20, 4, 80), (9, 3, 256), (40, 2, 32))


def draw(rng):
    kind = rng.choice(("shared", "shared", "verify", "trim", "experts", "experts"))
    dtype = rng.choices(("bf16", "fp16", "fp32"), (4, 2, 2))[0]
    size = SIZE[dtype]
    if kind == "trim":
        return dict(kind=kind, requests=_log_uniform(rng, 1, 1500), page=rng.choice((16, 32, 64, 128)), low=1,
                    high=_log_uniform(rng, 16, 32768), drop=_log_uniform(rng, 1, 3000), empty=rng.choice((0, 3, 11)))
    if kind == "verify":
        vocab, high = _log_uniform(rng, 500, 152064), rng.choice((0, 1, 3, 5, 8))
        probs = rng.random() < 0.4
        most = 48 * 5 * 128256 * 8 // (vocab * (size + (4 if probs else 0)) * (high + 1))
        return dict(kind=kind, dtype=dtype, requests=_log_uniform(rng, 1, max(1, min(128, most))),
                    low=rng.choice((0, high // 2, high)), high=high, vocab=vocab, probs=probs,
                    greedy=rng.choice((0, 0, 1, 3)), empty=rng.choice((0, 0, 5)))
    if kind == "experts":
        experts = rng.choice((4, 8, 16, 60, 64, 128))
        hidden = 8 * _log_uniform(rng, 32, 512)
        most = 8 * 3 * 4096 * 14336 * 2 // (3 * hidden * experts * size)
        inter = 8 * _log_uniform(rng, 8, max(8, min(1792, most // 8)))
        scoring = rng.choice(("softmax", "softmax", "sigmoid"))
        return dict(kind=kind, dtype=dtype, tokens=_log_uniform(rng, 1, 100), hidden=hidden, inter=inter,
                    experts=experts, top=rng.randint(1, min(8, experts // 2)), scoring=scoring,
                    normalize=rng.random() < 0.7, bias=scoring == "sigmoid" and rng.random() < 0.7)
    heads, kv_heads, dim = rng.choice(HEADS)
    tokens = rng.choice((1, 1, 2, 5, 8))
    prefixes = rng.choice((0, 1, 1, 2, 5))
    requests = max(_log_uniform(rng, 1, 100), prefixes)
    page = rng.choice((16, 32, 64, 128))
    # at most as many keys and products as the largest listed case
    flops = 64 * 2 * (16384 + 1250) * 64 * 128 // (requests * tokens * heads * dim * (4 if dtype == "fp32" else 1))
    keys = min(32768, flops // 2)
    own_keys = max(tokens, min(keys, 400_000_000 // (requests * kv_heads * dim * size)))
    high = max(tokens, _log_uniform(rng, tokens, own_keys))
    return dict(kind=kind, dtype=dtype, requests=requests, tokens=tokens, prefixes=prefixes,
                prefix=_log_uniform(rng, 16, max(16, keys)) if prefixes else 0, loner=rng.choice((0, 0, 5)),
                low=rng.choice((tokens, max(tokens, high // 2), high)), high=high, spread=rng.choice(("linear", "log")),
                empty=rng.choice((0, 0, 6)), heads=heads, kv_heads=kv_heads, dim=dim, page=page)


def _spread(n, low, high, spread, empty):
    """n numbers between low and high, the same for every seed (which only
    orders them), so that a case's work is known; every `empty`-th is 0."""
    out = []
    for i in range(n):
        share = (i * 0.6180339887498949 + 0.5) % 1.0 if n > 1 else 1.0
        if spread == "log":
            value = int(round(math.exp(math.log(low) + share * (math.log(high) - math.log(low)))))
        else:
            value = int(round(low + share * (high - low)))
        out.append(0 if empty and i % empty == empty - 1 else min(max(value, low), high))
    return out


def _pages(tokens, page):
    return -(-tokens // page)


def _prefix(case, request):
    """The group whose prefix a request begins with (-1: none)."""
    if not case["prefixes"] or (case["loner"] and request % case["loner"] == case["loner"] - 1):
        return -1
    return request % case["prefixes"]


def _drafts(case):
    """Drafted tokens of every request, -1 for one that has no row at all."""
    out = []
    for i, k in enumerate(_spread(case["requests"], case["low"], case["high"], "linear", 0)):
        out.append(-1 if case["empty"] and i % case["empty"] == case["empty"] - 1 else k)
    return out


def _kept(case):
    """(length, tokens that stay) of every request, in the case's own order."""
    lengths = _spread(case["requests"], case["low"], case["high"], "log", case["empty"])
    return [(n, max(0, n - i * 7919 % (case["drop"] + 1))) for i, n in enumerate(lengths)]


# ----------------------------------------------------------------- their work

def work(case):
    kind = case["kind"]
    if kind == "trim":
        back = sum(_pages(n, case["page"]) - _pages(kept, case["page"]) for n, kept in _kept(case))
        return {"bytes": 12 * case["requests"] + 8 * back + 8, "flops": 0}
    size = SIZE[case["dtype"]]
    if kind == "shared":
        own_keys = _spread(case["requests"], case["low"], case["high"], case["spread"], case["empty"])
        first = case["prefix"] // case["page"] * case["page"]
        groups = [_prefix(case, i) for i in range(case["requests"])]
        live = [i for i, n in enumerate(own_keys) if n]
        used = len({groups[i] for i in live if groups[i] >= 0}) * first
        keys, rows, t = sum(own_keys) + used, len(live) * case["tokens"], case["tokens"]
        seen = sum(t * (own_keys[i] + (first if groups[i] >= 0 else 0)) - t * (t - 1) // 2 for i in live)
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + 2 * rows * case["heads"] * case["dim"] * size
                + 4 * keys // case["page"] + 8 * rows, "flops": 4 * seen * case["heads"] * case["dim"]}
    if kind == "verify":
        rows, requests, vocab = sum(k + 1 for k in _drafts(case)), case["requests"], case["vocab"]
        return {"bytes": rows * (vocab * size + 20) + requests * 24 + (requests * vocab * 4 if case["probs"] else 0),
                "flops": 4 * rows * vocab}
    t, h, i, e, k = (case[name] for name in ("tokens", "hidden", "inter", "experts", "top"))
    hit = e * (1.0 - (1.0 - k / e) ** t)      # of experts whose choice is even
    return {"bytes": int(hit * 3 * h * i * size) + e * h * size + 2 * t * h * size + 8 * t * k,
            "flops": 6 * t * k * h * i + 2 * t * e * h}


# ----------------------------------------------------------------- the inputs

def _host(case, seed):
    """The inputs as CPU or GPU tensors, the same for both forms and `exact`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    kind = case["kind"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def uniform(n):
        return torch.rand(n, generator=g, device="cuda", dtype=torch.float64)

    if kind == "trim":
        state = _kept(case)
        rng.shuffle(state)
        lengths = np.array([n for n, _ in state], dtype=np.int64)
        used = -(-lengths // case["page"])
        total, width = int(used.sum()) + 5, int(max(1, used.max()))
        order = np.random.default_rng(seed).permutation(total).astype(np.int32)
        tables = np.full((len(state), width), -1, dtype=np.int32)
        tables[np.arange(width)[None, :] < used[:, None]] = order[:used.sum()]
        free = np.full(total, -1, dtype=np.int32)
        free[:5] = order[used.sum():]
        return dict(lengths=torch.from_numpy(lengths.astype(np.int32)), tables=torch.from_numpy(tables),
                    free=torch.from_numpy(free), n_free=torch.tensor([5], dtype=torch.int32),
                    keep=torch.tensor([kept for _, kept in state], dtype=torch.int32))
    dtype = DTYPE[case["dtype"]]
    if kind == "shared":
        page, tokens, requests = case["page"], case["tokens"], case["requests"]
        own_keys = _spread(requests, case["low"], case["high"], case["spread"], case["empty"])
        groups = [_prefix(case, i) for i in range(requests)]
        both = list(zip(own_keys, groups))
        rng.shuffle(both)
        first = case["prefix"] // page          # whole pages are shared
        used = [_pages(n, page) + (first if group >= 0 and n else 0) for n, group in both]
        total = sum(_pages(n, page) for n, _ in both) + first * case["prefixes"] + 2
        order = torch.randperm(total, generator=g, device="cuda").int().cpu()
        tables = torch.full((requests, max(1, max(used))), -1, dtype=torch.int32)
        at = first * case["prefixes"]
        contexts, of = [], []
        for r, (n, group) in enumerate(both):
            if not n:
                continue
            shared = first if group >= 0 else 0
            if shared:
                tables[r, :first] = order[group * first:(group + 1) * first]
            tables[r, shared:used[r]] = order[at:at + _pages(n, page)]
            at += _pages(n, page)
            contexts += [shared * page + n - tokens + 1 + i for i in range(tokens)]
            of += [r] * tokens
        if case["empty"]:                       # a step's unused rows
            contexts, of = contexts + [0, 0], of + [-1, -1]
        shape = (total, case["kv_heads"], page, case["dim"])
        keys, values = normal(*shape, dtype=dtype), normal(*shape, dtype=dtype)
        # some heads attend evenly, some to few tokens
        sharp = torch.tensor([1.0, 1.0, 2.0, 4.0], device="cuda")[torch.arange(case["heads"], device="cuda") % 4]
        q = normal(len(of), case["heads"], case["dim"]) * sharp[None, :, None]
        return dict(q=q.to(dtype), key_cache=keys, value_cache=values, tables=tables.cuda(),
                    contexts=torch.tensor(contexts, dtype=torch.int32), requests=torch.tensor(of, dtype=torch.int32),
                    groups=torch.tensor([group for _, group in both], dtype=torch.int32),
                    shared=torch.full((case["prefixes"],), first * page, dtype=torch.int32),
                    host_rows=list(zip(of, contexts)))
    if kind == "verify":
        drafts, vocab = _drafts(case), case["vocab"]
        rng.shuffle(drafts)
        starts = [0]
        for k in drafts:
            starts.append(starts[-1] + k + 1)
        rows = max(1, starts[-1]) + (2 if case["empty"] else 0)     # a step's unused rows
        logits = 3.0 * normal(rows, vocab)
        # a draft model is off by a little; texts repeat what is likely
        guess = logits + 0.5 * normal(rows, vocab)
        noise = -torch.log(-torch.log(uniform(rows * vocab).float().clamp_(1e-12, 1 - 1e-7))).view(rows, vocab)
        out = dict(logits=logits.to(dtype))
        if case["probs"]:
            out["draft_probs"] = torch.softmax(guess, -1)
            drawn = (guess + noise).argmax(-1)
        else:
            drawn = torch.where(uniform(rows) < 0.7, logits.argmax(-1), (guess + noise).argmax(-1))
        temperature = 0.5 + uniform(case["requests"]).float()
        if case["greedy"]:
            temperature[::case["greedy"]] = 0.0
        out.update(tokens=drawn.roll(1), starts=torch.tensor(starts, dtype=torch.int32), accept=uniform(rows),
                   sample=uniform(case["requests"]), temperature=temperature, host_starts=starts)
        return out
    t, h, i, e = (case[name] for name in ("tokens", "hidden", "inter", "experts"))
    return dict(x=normal(t, h).to(dtype), router=(normal(e, h) * h ** -0.5).to(dtype),
                bias=0.1 * normal(e) if case["bias"] else None,
                gate_up=normal(e, 2 * i, h, dtype=dtype) * h ** -0.5, down=normal(e, h, i, dtype=dtype) * i ** -0.5)


def prepare(case, seed):
    state = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in _host(case, seed).items()}
    state["case"] = case
    kind = case["kind"]
    if kind == "experts":
        state["options"] = dict(scoring=case["scoring"], normalize=case["normalize"], bias=state["bias"])
    if own:
        from neuralzip_amd.gpu import serving
        state["serving"] = serving
        if kind == "trim":
            book = serving.PageTables(case["requests"], state["tables"].shape[1], case["page"],
                                      state["free"].numel(), device="cuda")
            book.lengths.copy_(state["lengths"])
            book.tables.copy_(state["tables"])
            book.free.copy_(state["free"])
            book.n_free.copy_(state["n_free"])
            state["book"] = book
        if kind == "shared":
            # one plan for all layers of a step
            groups = dict(groups=state["groups"], shared=state["shared"]) if case["prefixes"] else {}
            state["plan"] = serving.SharedPlan(state["contexts"], heads=case["heads"], kv_heads=case["kv_heads"],
                                               requests=state["requests"], **groups)
    return state


# ------------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        serving = state["serving"]
        if kind == "trim":
            after = state["book"].trim(state["keep"], advance=False)
            return after.lengths, after.n_free, state["book"].free
        if kind == "shared":
            return serving.paged_attention(state["q"], state["key_cache"], state["value_cache"], state["tables"],
                                           state["plan"])
        if kind == "verify":
            return serving.verify_drafts(state["logits"], state["tokens"], state["starts"], state["accept"],
                                         state["sample"], draft_probs=state.get("draft_probs"),
                                         temperature=state["temperature"])
        ids, weights = serving.route_experts(state["x"], state["router"], case["top"], **state["options"])
        return ids, weights, serving.expert_mlp(state["x"], ids, weights, state["gate_up"], state["down"])
    return {"trim": _plain_trim, "shared": _plain_shared, "verify": _plain_verify, "experts": _plain_experts}[kind](state)


def _plain_trim(s):
    page, tables, free = s["case"]["page"], s["tables"], s["free"]
    lengths = s["lengths"].long()
    kept = torch.minimum(s["keep"].long().clamp(min=0), lengths)
    stay = (kept + page - 1) // page
    back = (lengths + page - 1) // page - stay
    first = s["n_free"].long() + back.cumsum(0) - back
    j = torch.arange(tables.shape[1], device=tables.device) - stay[:, None]
    target = torch.where((j >= 0) & (j < back[:, None]), first[:, None] + j, free.numel())
    flat = torch.cat((free, free.new_zeros(1)))
    flat[target.view(-1)] = tables.view(-1)
    free.copy_(flat[:-1])
    return kept.int(), (s["n_free"] + back.sum()).int(), free


def _plain_shared(s):
    case, rows = s["case"], s["host_rows"]
    hk, d, t = case["kv_heads"], case["dim"], case["tokens"]
    group, out = case["heads"] // hk, torch.zeros_like(s["q"])
    for row in range(0, len(rows), t):
        request, n = rows[row][0], rows[min(row + t, len(rows)) - 1][1]
        if request < 0:
            continue
        pages = s["tables"][request, :_pages(n, case["page"])].long()
        k, v = (c[pages].transpose(0, 1).reshape(hk, -1, d)[:, :n].float()
                for c in (s["key_cache"], s["value_cache"]))
        q = s["q"][row:row + t].float().view(t, hk, group, d).transpose(0, 1).reshape(hk, t * group, d)
        scores = torch.matmul(q, k.transpose(1, 2)).view(hk, t, group, n) * d ** -0.5
        unseen = torch.arange(n, device=q.device) >= s["contexts"][row:row + t, None]
        scores = scores.masked_fill(unseen[None, :, None], -math.inf).view(hk, t * group, n)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[row:row + t] = o.view(hk, t, group, d).transpose(0, 1).reshape(t, -1, d).to(out.dtype)
    return out


def _plain_verify(s):
    x, starts, tokens = s["logits"].double(), s["starts"].long(), s["tokens"]
    rows, vocab = x.shape
    row = torch.arange(rows, device=x.device)
    request = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    live = request < len(starts) - 1
    request = request.clamp(max=len(starts) - 2)
    t = s["temperature"][request].double()[:, None]
    top = x.amax(-1, keepdim=True)
    p = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(t > 0, t, 1.0)))
    p = torch.where(t > 0, p, (torch.arange(vocab, device=x.device) == x.argmax(-1, keepdim=True)).double())
    p = p / p.sum(-1, keepdim=True)
    # rows whose token is followed by a draft
    more = live & (row + 1 < starts[request + 1])
    draft = tokens.roll(-1)
    known = (draft >= 0) & (draft < vocab)
    at = torch.where(known, draft, 0)[:, None]
    chance = torch.where(known, p.gather(1, at)[:, 0], 0.0)
    drawn = s["draft_probs"].gather(1, at)[:, 0].double() if "draft_probs" in s else 1.0
    stops = live & ~(more & (s["accept"] * drawn < chance))
    final = torch.full((len(starts) - 1,), rows, device=x.device)
    final = final.scatter_reduce(0, request, torch.where(stops, row, rows), "amin")
    has = starts[1:] > starts[:-1]
    final = torch.where(has, final, 0)
    accepted = torch.where(has, final - starts[:-1], 0)
    p, refused = p[final], more[final]
    if "draft_probs" in s:
        q = s["draft_probs"][final].double()
    else:
        q = (torch.arange(vocab, device=x.device) == draft[final][:, None]).double()
    rest = (p - torch.where(refused[:, None], q, 0.0)).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(-1)
    over = (upto > s["sample"][:, None] * upto[:, -1:]) & (rest > 0)
    last = vocab - 1 - (rest > 0).flip(-1).int().argmax(-1)
    token = torch.where(over.any(-1), over.int().argmax(-1), last)
    return accepted.int(), torch.where(has, token, -1)


def _plain_experts(s):
    case, x = s["case"], s["x"]
    # the router's choice, in 64 bits
    scores = torch.matmul(x.double(), s["router"].double().t())
    picked = scores.sigmoid() if case["scoring"] == "sigmoid" else scores
    if s["bias"] is not None:
        picked = picked + s["bias"].double()
    ids = torch.sort(picked, descending=True, stable=True)[1][:, :case["top"]]
    chances = scores.sigmoid() if case["scoring"] == "sigmoid" else scores.softmax(-1)
    weights = chances.gather(1, ids)
    if case["normalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    weights = weights.float()
    # the experts' products, in 32
    out = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    chosen = ids.tolist()
    for e in sorted({e for row in chosen for e in row}):
        token, slot = zip(*((t, k) for t, row in enumerate(chosen) for k, one in enumerate(row) if one == e))
        token, slot = torch.tensor(token, device=x.device), torch.tensor(slot, device=x.device)
        gate, up = torch.matmul(x[token].float(), s["gate_up"][e].float().t()).chunk(2, -1)
        y = torch.matmul(gate * torch.sigmoid(gate) * up, s["down"][e].float().t())
        out.index_add_(0, token, y * weights[token, slot][:, None])
    return ids.int(), weights, out.to(x.dtype)


# ------------------------------------------------------- the definition itself

def exact(case, seed):
    s = _host(case, seed)
    return {"trim": _exact_trim, "shared": _exact_shared, "verify": _exact_verify,
            "experts": _exact_experts}[case["kind"]](case, s)


def _exact_trim(case, s):
    lengths, tables, stack = s["lengths"].numpy().copy(), s["tables"].numpy(), s["free"].numpy().copy()
    top = int(s["n_free"])
    for r, keep in enumerate(s["keep"].tolist()):
        keep = min(max(keep, 0), int(lengths[r]))
        for j in range(_pages(keep, case["page"]), _pages(int(lengths[r]), case["page"])):
            stack[top] = tables[r, j]
            top += 1
        lengths[r] = keep
    return lengths, np.array([top], dtype=np.int32), stack


def _exact_shared(case, s):
    hk, d = case["kv_heads"], case["dim"]
    group, q = case["heads"] // hk, s["q"].double()
    out = torch.zeros_like(q)
    for row, (request, n) in enumerate(s["host_rows"]):
        if not n:
            continue
        slot = torch.arange(n, device="cuda")
        page, offset = s["tables"][request].long()[slot // case["page"]], slot % case["page"]
        for h in range(hk):
            k, v = s["key_cache"][page, h, offset].double(), s["value_cache"][page, h, offset].double()
            score = k @ q[row, h * group:(h + 1) * group].T / math.sqrt(d)
            out[row, h * group:(h + 1) * group] = (score - score.logsumexp(0)).exp().T @ v
    return out


def _exact_verify(case, s):
    starts, tokens = s["host_starts"], s["tokens"].tolist()
    accept, sample, temperature = (s[k].tolist() for k in ("accept", "sample", "temperature"))
    accepted, final = [], []

    def chances(row, t):
        x = s["logits"][row].double().cpu().numpy()
        if t <= 0:
            p = np.zeros_like(x)
            p[x.argmax()] = 1.0
            return p
        p = np.exp((x - x.max()) / t)
        return p / p.sum()

    for r in range(len(starts) - 1):
        first, last = starts[r], starts[r + 1] - 1
        if last < first:
            accepted.append(0)
            final.append(-1)
            continue
        for row in range(first, last + 1):
            p = chances(row, temperature[r])
            if row == last:
                weights = p
                break
            d = tokens[row + 1]
            q = np.zeros_like(p)
            if case["probs"]:
                q = s["draft_probs"][row].double().cpu().numpy()
            else:
                q[d] = 1.0
            if not accept[row] * q[d] < p[d]:
                weights = np.maximum(p - q, 0.0)
                weights = weights if weights.sum() > 0 else p
                break
        sums = np.cumsum(weights)
        over = np.flatnonzero((sums > sample[r] * sums[-1]) & (weights > 0))
        accepted.append(row - first)
        final.append(int(over[0]) if len(over) else int(np.flatnonzero(weights)[-1]))
    return np.array(accepted, dtype=np.int32), np.array(final, dtype=np.int64)


def _exact_experts(case, s):
    x = s["x"].double()
    ids, weights, out = [], [], torch.zeros_like(x)
    logits = (x @ s["router"].double().T).cpu().numpy()
    bias = s["bias"].double().cpu().numpy() if case["bias"] else 0.0
    for row in logits:
        if case["scoring"] == "sigmoid":
            chance = 1.0 / (1.0 + np.exp(-row))
        else:
            chance = np.exp(row - row.max())
            chance /= chance.sum()
        rank = chance + bias if case["scoring"] == "sigmoid" else row
        best = np.argsort(-rank, kind="stable")[:case["top"]]
        w = chance[best]
        ids.append(best)
        weights.append(w / w.sum() if case["normalize"] else w)
    ids, weights = np.array(ids, dtype=np.int32), torch.tensor(np.array(weights), device="cuda")
    for e in range(case["experts"]):
        token, slot = np.nonzero(ids == e)
        if len(token):
            y = x[token] @ s["gate_up"][e].double().T
            half = y.shape[1] // 2
            y = y[:, :half] / (1.0 + torch.exp(-y[:, :half])) * y[:, half:]
            out.index_add_(0, torch.tensor(token, device="cuda"),
                           y @ s["down"][e].double().T * weights[token, slot][:, None])
    return ids, weights, out
