"""The operators of a serving step and the cases they are measured on.

Four kinds, in the order in which a step of many requests with lengths of
their own runs them:

  tables     pages for the step's new tokens: block tables, slots, positions
             and contexts from the requests' lengths (extend), and finished
             requests' pages back onto the free stack (release)
  rotary     the heads' optional RMS norm and the position rotation of queries
             and keys, with keys and values stored into their pages
  attention  new tokens over the paged key-value cache
  logits     repetition, frequency and presence penalties, biases and
             grammar masks on the step's logits

Where `own` is false the operators run in plain torch, in 32 bits; where it
is true, as neuralzip_amd.gpu.serving's calls. `exact` is the definition in
64 bits (whole numbers: in loops over requests).
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
        # 32 requests in the middle of their answers, one token each: the
        # bookkeeping in front of every decode step. The smallest call.
        dict(name="tables-decode-32", kind="tables", op="extend", requests=32, page=16, low=1, high=4096, spread="log",
             new_low=1, new_high=1, empty=0, free_share=2.0),
        # 256 requests, most of them with a prompt still to be taken in, more
        # than the free pages hold: the last ones are refused.
        dict(name="tables-prompts-256", kind="tables", op="extend", requests=256, page=16, low=1, high=8192,
             spread="log", new_low=1, new_high=777, empty=5, free_share=0.9),
        # 1000 requests with long contexts, a quarter of them finished: their
        # pages go back.
        dict(name="tables-release-1000", kind="tables", op="release", requests=1000, page=32, low=1, high=32768,
             spread="log", done=4, empty=7),
        # One token of one request, Llama-3-8B's heads, q, k and v as views
        # of one product: pure latency.
        dict(name="rotary-8b-one-token", kind="rotary", dtype="bf16", tokens=1, heads=32, kv_heads=8, dim=128,
             rotary=128, interleaved=False, norm=False, packed=True, page=16, positions=8192),
        # 32 requests' tokens with norms of the heads, half of each head
        # rotated in neighbouring pairs, in fp16.
        dict(name="rotary-norm-32-fp16", kind="rotary", dtype="fp16", tokens=32, heads=16, kv_heads=4, dim=128,
             rotary=64, interleaved=True, norm=True, packed=False, page=32, positions=4096),
        # Prompts of several requests, Llama-3-70B's heads with norms.
        dict(name="rotary-70b-prompts", kind="rotary", dtype="bf16", tokens=8191, heads=64, kv_heads=8, dim=128,
             rotary=128, interleaved=False, norm=True, packed=True, page=16, positions=8192),
        # One request of the Llama-3-8B shape, 2000 tokens in: the step whose
        # attention is all latency.
        dict(name="attention-8b-one", kind="attention", dtype="bf16", rows=1, low=2001, high=2001, spread="linear",
             empty=0, heads=32, kv_heads=8, dim=128, page=16),
        # A ragged batch of the same shape, idle slots among the requests.
        dict(name="attention-8b-batch-32", kind="attention", dtype="bf16", rows=32, low=1, high=8191, spread="linear",
             empty=9, heads=32, kv_heads=8, dim=128, page=16),
        # Two long documents of the Qwen2-0.5B shape in fp32.
        dict(name="attention-qwen-long-fp32", kind="attention", dtype="fp32", rows=2, low=20011, high=32001,
             spread="linear", empty=0, heads=14, kv_heads=2, dim=64, page=64),
        # The largest: 64 requests of the Llama-3-70B shape, up to 16k tokens.
        dict(name="attention-70b-batch-64", kind="attention", dtype="fp16", rows=64, low=100, high=16384,
             spread="linear", empty=0, heads=64, kv_heads=8, dim=128, page=32),
        # One answer of the Qwen2-0.5B shape, penalties alone, on the logits
        # as the model's last product leaves them.
        dict(name="logits-qwen-one", kind="logits", dtype="bf16", rows=1, vocab=151936, history=700, prompt=0.3,
             penalties=True, bias=0, masks=False),
        # 32 answers of the Llama-3-8B shape with everything switched on,
        # in 32 bits, as a sampler takes them.
        dict(name="logits-8b-32", kind="logits", dtype="fp32", rows=32, vocab=128256, history=2048, prompt=0.6,
             penalties=True, bias=40, masks=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((32, 8, 128), (14, 2, 64), (64, 8, 128), (8, 8, 64), (12, 1, 96), (20, 4, 80), (9, 3, 256), (40, 2, 32))


def draw(rng):
    kind = rng.choice(("tables", "rotary", "attention", "attention", "logits"))
    dtype = rng.choices(("bf16", "fp16", "fp32"), (4, 2, 2))[0]
    if kind == "tables":
        case = dict(kind=kind, op=rng.choice(("extend", "extend", "release")), requests=_log_uniform(rng, 1, 1500),
                    page=rng.choice((16, 32, 64, 128)), low=1, high=_log_uniform(rng, 16, 32768), spread="log",
                    empty=rng.choice((0, 3, 11)))
        if case["op"] == "release":
            return dict(case, done=rng.choice((1, 2, 5, 50)))
        most = rng.choice((1, 1, _log_uniform(rng, 2, 1000)))
        return dict(case, new_low=rng.choice((0, 1)), new_high=min(most, 200_000 // case["requests"] + 1),
                    free_share=rng.choice((2.0, 1.0, 0.7)))
    if kind == "logits":
        return dict(kind=kind, dtype=dtype, rows=_log_uniform(rng, 1, 48), vocab=_log_uniform(rng, 500, 152064),
                    history=_log_uniform(rng, 1, 8000), prompt=rng.uniform(0.0, 1.0), penalties=rng.random() < 0.8,
                    bias=rng.choice((0, 0, _log_uniform(rng, 1, 300))), masks=rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice(HEADS)
    if kind == "rotary":
        tokens = _log_uniform(rng, 1, 8190 if heads * dim <= 4096 else 4000)
        if dtype == "fp32":
            tokens = max(1, tokens // 2)
        return dict(kind=kind, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice((dim, dim, dim // 32 * 16)), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5, packed=rng.random() < 0.5, page=rng.choice((16, 32, 64)),
                    positions=_log_uniform(rng, 100, 32768))
    rows = _log_uniform(rng, 1, 200)
    # at most as many bytes of keys and values as the largest listed case
    most = min(32768, 1_000_000_000 // (rows * kv_heads * dim * SIZE[dtype]))
    high = _log_uniform(rng, 1, most)
    return dict(kind=kind, dtype=dtype, rows=rows, low=rng.choice((1, max(1, high // 2), high)), high=high,
                spread=rng.choice(("linear", "log")), empty=rng.choice((0, 0, 6)), heads=heads, kv_heads=kv_heads,
                dim=dim, page=rng.choice((16, 32, 64, 128)))


def _spread(n, low, high, spread, empty):
    """n lengths between low and high, the same for every seed (which only
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


def _requests(case):
    """(length, new tokens or finished) of every request, in the case's own order."""
    lengths = _spread(case["requests"], case["low"], case["high"], case["spread"], case["empty"])
    if case["op"] == "release":
        return [(n, i % case["done"] == 0) for i, n in enumerate(lengths)]
    low, high = case["new_low"], case["new_high"]
    return [(n, low + (i * 7919) % (high - low + 1)) for i, n in enumerate(lengths)]


def _pages(tokens, page):
    return -(-tokens // page)


def _want(case):
    return sum(_pages(n + new, case["page"]) - _pages(n, case["page"]) for n, new in _requests(case))


# ----------------------------------------------------------------- their work

def work(case):
    kind = case["kind"]
    if kind == "tables":
        n = case["requests"]
        if case["op"] == "release":
            back = sum(_pages(length, case["page"]) for length, done in _requests(case) if done)
            return {"bytes": 9 * n + 8 * back + 8, "flops": 0}
        tokens = sum(new for _, new in _requests(case))
        taken = min(_want(case), int(_want(case) * case["free_share"]) + 1)
        # lengths and new tokens in; lengths, status and starts out; a table
        # entry of each part-filled page in; pages from the stack into the
        # tables; slot, position, request and context of every token out
        return {"bytes": 24 * n + 8 * taken + 20 * tokens, "flops": 0}
    size = SIZE[case["dtype"]]
    if kind == "rotary":
        t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        angles = min(t, case["positions"]) * case["rotary"] * 4
        return {"bytes": t * (2 * hq + 4 * hk) * d * size + angles + 12 * t + (2 * d * size if case["norm"] else 0),
                "flops": t * (hq + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    if kind == "attention":
        lengths = _spread(case["rows"], case["low"], case["high"], case["spread"], case["empty"])
        keys = sum(lengths)
        pages = sum(_pages(n, case["page"]) for n in lengths)
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size
                + 2 * case["rows"] * case["heads"] * case["dim"] * size + 4 * pages + 8 * case["rows"],
                "flops": 4 * keys * case["heads"] * case["dim"]}
    rows, vocab = case["rows"], case["vocab"]
    total = 2 * rows * vocab * size
    if case["penalties"]:
        total += 4 * sum(_spread(rows, 1, case["history"], "linear", 0)) + 20 * rows
    total += 8 * rows * case["bias"] + (rows * vocab // 8 if case["masks"] else 0)
    return {"bytes": total, "flops": 5 * rows * vocab}


# ----------------------------------------------------------------- the inputs

def _host(case, seed):
    """The inputs as CPU or GPU tensors, the same for both forms and `exact`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    kind = case["kind"]
    if kind == "tables":
        state = _requests(case)
        rng.shuffle(state)
        lengths = np.array([n for n, _ in state], dtype=np.int64)
        page = case["page"]
        grown = lengths + np.array([new for _, new in state]) if case["op"] == "extend" else lengths
        used = -(-lengths // page)
        width = int(max(1, (-(-grown // page)).max()))
        spare = int(_want(case) * case["free_share"]) + 1 if case["op"] == "extend" else 5
        total = int(used.sum()) + spare
        order = np.random.default_rng(seed).permutation(total).astype(np.int32)
        tables = np.full((len(state), width), -1, dtype=np.int32)
        tables[np.arange(width)[None, :] < used[:, None]] = order[:used.sum()]
        free = np.full(total, -1, dtype=np.int32)
        free[:spare] = order[used.sum():]
        out = dict(lengths=torch.from_numpy(lengths.astype(np.int32)), tables=torch.from_numpy(tables),
                   free=torch.from_numpy(free), n_free=torch.tensor([spare], dtype=torch.int32))
        if case["op"] == "extend":
            out["new"] = torch.tensor([new for _, new in state], dtype=torch.int32)
        else:
            out["done"] = torch.tensor([done for _, done in state])
        return out
    dtype = DTYPE[case["dtype"]]
    if kind == "rotary":
        t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:
            rows = torch.randn(t, (hq + 2 * hk) * d, generator=g, device="cuda").to(dtype)
            q, k, v = (x.view(t, -1, d) for x in rows.split((hq * d, hk * d, hk * d), dim=1))
        else:
            q, k, v = (torch.randn(t, h, d, generator=g, device="cuda").to(dtype) for h in (hq, hk, hk))
        half = case["rotary"] // 2
        rates = 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
        angles = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * rates
        pages = _pages(t, case["page"]) + 3
        # the tokens of one prompt in a row, or of requests at any position
        start = rng.randrange(case["positions"])
        positions = ((torch.arange(t, device="cuda") + start) % case["positions"]).int()
        if t <= 64:
            positions = positions[torch.randperm(t, generator=g, device="cuda")]
        order = torch.randperm(pages, generator=g, device="cuda")
        token = torch.arange(t, device="cuda")
        slots = order[token // case["page"]] * case["page"] + token % case["page"]
        if t > 8:
            slots[::t // 2] = -1        # tokens of a padded step are stored nowhere
        caches = [torch.randn(pages, hk, case["page"], d, generator=g, device="cuda").to(dtype) for _ in range(2)]
        weights = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) if case["norm"] else None
                   for _ in range(2)]
        return dict(q=q, k=k, v=v, cos=angles.cos().float(), sin=angles.sin().float(), positions=positions,
                    slots=slots, key_cache=caches[0], value_cache=caches[1], q_weight=weights[0],
                    k_weight=weights[1])
    if kind == "attention":
        contexts = _spread(case["rows"], case["low"], case["high"], case["spread"], case["empty"])
        rng.shuffle(contexts)
        used = [_pages(n, case["page"]) for n in contexts]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g, device="cuda").int()
        tables = torch.full((case["rows"], max(1, max(used))), -1, dtype=torch.int32, device="cuda")
        live = torch.arange(tables.shape[1], device="cuda")[None, :] < torch.tensor(used, device="cuda")[:, None]
        tables[live] = order[:sum(used)]
        shape = (pages, case["kv_heads"], case["page"], case["dim"])
        keys, values = (torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(2))
        q = torch.randn(case["rows"], case["heads"], case["dim"], generator=g, device="cuda")
        # some heads attend evenly, some to few tokens
        sharp = torch.tensor([1.0, 1.0, 2.0, 4.0], device="cuda")[torch.arange(case["heads"], device="cuda") % 4]
        return dict(q=(q * sharp[None, :, None]).to(dtype), key_cache=keys, value_cache=values, tables=tables,
                    contexts=torch.tensor(contexts, dtype=torch.int32, device="cuda"), host_contexts=contexts)
    rows, vocab = case["rows"], case["vocab"]
    out = dict(logits=(3.0 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype))
    if case["penalties"]:
        lengths = _spread(rows, 1, case["history"], "linear", 0)
        rng.shuffle(lengths)
        # texts repeat few tokens often: squared uniform numbers
        ids = torch.rand(rows, case["history"], generator=g, device="cuda").square() * vocab
        out.update(history=ids.int().clamp_(max=vocab - 1),
                   lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                   prompt_lengths=torch.tensor([int(n * case["prompt"]) for n in lengths], dtype=torch.int32,
                                               device="cuda"))
        for name, low, high in (("repetition", 1.0, 1.5), ("frequency", -0.2, 0.6), ("presence", -0.5, 1.0)):
            out[name] = low + (high - low) * torch.rand(rows, generator=g, device="cuda")
    if case["bias"]:
        n = case["bias"]
        out["bias"] = ((torch.arange(rows + 1, device="cuda") * n).int(),
                       torch.randint(0, vocab, (rows * n,), generator=g, device="cuda").int(),
                       4.0 * torch.randn(rows * n, generator=g, device="cuda"))
    if case["masks"]:
        words = (vocab + 31) // 32
        low, high = (torch.randint(0, 1 << 16, (rows, words), generator=g, device="cuda") for _ in range(2))
        out["masks"] = (low | high << 16).to(torch.int32)
        # every third request answers without a grammar
        out["mask_rows"] = torch.tensor([-1 if i % 3 == 2 else i for i in range(rows)], dtype=torch.int32,
                                        device="cuda")
    return out


def prepare(case, seed):
    state = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in _host(case, seed).items()}
    state["case"] = case
    kind = case["kind"]
    if kind == "tables":
        state["max_tokens"] = max(1, sum(new for _, new in _requests(case))) if case["op"] == "extend" else 0
    if own:
        from neuralzip_amd.gpu import serving
        state["serving"] = serving
        if kind == "tables":
            book = serving.PageTables(case["requests"], state["tables"].shape[1], case["page"],
                                      state["free"].numel(), device="cuda")
            book.lengths.copy_(state["lengths"])
            book.tables.copy_(state["tables"])
            book.free.copy_(state["free"])
            book.n_free.copy_(state["n_free"])
            state["book"] = book
        if kind == "rotary":
            state["rotary"] = serving.Rotary(state["cos"], state["sin"], interleaved=case["interleaved"],
                                             q_weight=state["q_weight"], k_weight=state["k_weight"], eps=1e-6)
        if kind == "attention":
            state["plan"] = serving.AttentionPlan(state["contexts"], heads=case["heads"], kv_heads=case["kv_heads"])
    return state


# ------------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if own:
        serving = state["serving"]
        if case["kind"] == "tables":
            if case["op"] == "release":
                after = state["book"].release(state["done"], advance=False)
                return after.lengths, after.n_free, state["book"].free
            step = state["book"].extend(state["new"], state["max_tokens"], advance=False)
            return (step.slots, step.positions, step.requests, step.contexts, step.starts, step.status, step.lengths,
                    step.n_free, state["book"].tables)
        if case["kind"] == "rotary":
            q = state["rotary"](state["q"], state["k"], state["v"], state["positions"], state["slots"],
                                state["key_cache"], state["value_cache"])
            return q, state["key_cache"], state["value_cache"]
        if case["kind"] == "attention":
            return serving.paged_attention(state["q"], state["key_cache"], state["value_cache"], state["tables"],
                                           state["plan"])
        return serving.adjust_logits(state["logits"], **{k: state[k] for k in LOGITS if k in state})
    return {"tables": _plain_release if case.get("op") == "release" else _plain_extend, "rotary": _plain_rotary,
            "attention": _plain_attention, "logits": _plain_logits}[case["kind"]](state)


LOGITS = ("history", "lengths", "prompt_lengths", "repetition", "frequency", "presence", "bias", "masks", "mask_rows")


def _plain_extend(s):
    page, capacity = s["case"]["page"], s["max_tokens"]
    lengths, new, tables, free = s["lengths"].long(), s["new"].long(), s["tables"], s["free"]
    width, n_free = tables.shape[1], s["n_free"].long()
    fits = (new >= 0) & (lengths + new <= width * page)
    asked = torch.where(fits, new, 0)
    room = fits & ((asked.cumsum(0) <= capacity) | (asked == 0))
    asked = torch.where(room, asked, 0)
    old = (lengths + page - 1) // page
    want = (lengths + asked + page - 1) // page - old
    have = (want.cumsum(0) <= n_free) | (want == 0)
    status = torch.where(fits, torch.where(room, torch.where(have, 0, 3), 2), 1).int()
    granted, want = torch.where(have, asked, 0), torch.where(have, want, 0)
    last = want.cumsum(0)
    starts = torch.cat((granted.new_zeros(1), granted.cumsum(0)))
    # the new pages' table entries (pages past the last one land behind the tables' end)
    j = torch.arange(free.numel(), device=free.device)
    owner = torch.searchsorted(last, j, right=True).clamp_(max=len(lengths) - 1)
    entry = owner * width + old[owner] + j - (last - want)[owner]
    flat = torch.cat((tables.view(-1), tables.new_zeros(1)))
    flat[torch.where(j < last[-1], entry, tables.numel())] = free[(n_free - 1 - j).clamp_(min=0)]
    tables.copy_(flat[:-1].view_as(tables))
    # the new tokens
    t = torch.arange(capacity, device=free.device)
    live = t < starts[-1]
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp_(max=len(lengths) - 1)
    position = torch.where(live, lengths[r] + t - starts[r], 0)
    slot = tables[r, position // page].long() * page + position % page
    return (torch.where(live, slot, -1), position.int(), torch.where(live, r, -1).int(),
            torch.where(live, position + 1, 0).int(), starts.int(), status, (lengths + granted).int(),
            (n_free - last[-1]).int(), tables)


def _plain_release(s):
    page, tables, free = s["case"]["page"], s["tables"], s["free"]
    lengths = s["lengths"].long()
    back = torch.where(s["done"], (lengths + page - 1) // page, 0)
    first = s["n_free"].long() + back.cumsum(0) - back
    j = torch.arange(tables.shape[1], device=tables.device)
    target = torch.where(j < back[:, None], first[:, None] + j, free.numel())
    flat = torch.cat((free, free.new_zeros(1)))
    flat[target.view(-1)] = tables.view(-1)
    free.copy_(flat[:-1])
    return torch.where(s["done"], 0, lengths).int(), (s["n_free"] + back.sum()).int(), free


def _plain_rotary(s):
    case = s["case"]
    rotary, half = case["rotary"], case["rotary"] // 2
    position = s["positions"].long()
    cos, sin = s["cos"][position][:, None, :], s["sin"][position][:, None, :]

    def turn(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        if case["interleaved"]:
            a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:rotary]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, x[..., rotary:]), -1)

    dtype = s["q"].dtype
    live = s["slots"] >= 0
    slots = s["slots"][live]
    block, offset = slots // case["page"], slots % case["page"]
    s["key_cache"][block, :, offset] = turn(s["k"], s["k_weight"]).to(dtype)[live]
    s["value_cache"][block, :, offset] = s["v"][live]
    return turn(s["q"], s["q_weight"]).to(dtype), s["key_cache"], s["value_cache"]


def _plain_attention(s):
    case = s["case"]
    hk, d = case["kv_heads"], case["dim"]
    group, out = case["heads"] // hk, torch.zeros_like(s["q"])
    for row, n in enumerate(s["host_contexts"]):
        if n == 0:
            continue
        pages = s["tables"][row, :_pages(n, case["page"])].long()
        k, v = (c[pages].transpose(0, 1).reshape(hk, -1, d)[:, :n].float()
                for c in (s["key_cache"], s["value_cache"]))
        scores = torch.matmul(s["q"][row].float().view(hk, group, d), k.transpose(1, 2)) * d ** -0.5
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        out[row] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(-1, d).to(out.dtype)
    return out


def _plain_logits(s):
    rows, vocab = s["logits"].shape
    x = s["logits"].float()
    if "history" in s:
        ids = s["history"].long()
        at = torch.arange(ids.shape[1], device=ids.device)
        live = at < s["lengths"][:, None]
        answer = live & (at >= s["prompt_lengths"][:, None])
        seen = torch.zeros(rows, vocab, dtype=torch.int32, device=ids.device).scatter_add_(1, ids, live.int())
        count = torch.zeros(rows, vocab, dtype=torch.int32, device=ids.device).scatter_add_(1, ids, answer.int())
        rep = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if "bias" in s:
        starts, tokens, values = s["bias"]
        entry = torch.arange(tokens.numel(), device=tokens.device)
        row = torch.searchsorted(starts[1:].contiguous(), entry.int(), right=True)
        last = torch.full((rows * vocab,), -1, dtype=torch.int64, device=tokens.device)
        last.scatter_reduce_(0, row * vocab + tokens, entry, "amax")
        last = last.view(rows, vocab)
        x = x + torch.where(last >= 0, values[last.clamp(min=0)], 0.0)
    if "masks" in s:
        v = torch.arange(vocab, device=x.device)
        bits = s["masks"][s["mask_rows"].clamp(min=0).long()][:, v // 32] >> (v % 32) & 1
        x = x.masked_fill((bits == 0) & (s["mask_rows"] >= 0)[:, None], -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------- the definition itself

def exact(case, seed):
    s = _host(case, seed)
    if case["kind"] == "tables":
        return _exact_release(case, s) if case["op"] == "release" else _exact_extend(case, s)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "logits": _exact_logits}[case["kind"]](case, s)


def _exact_extend(case, s):
    page, lengths, new = case["page"], s["lengths"].tolist(), s["new"].tolist()
    tables, stack = s["tables"].numpy().copy(), s["free"].numpy()
    top = int(s["n_free"])
    capacity = max(1, sum(n for _, n in _requests(case)))
    limit = tables.shape[1] * page
    slots, positions, requests, contexts = [], [], [], []
    starts, status, after = [0], [], []
    asked_tokens = asked_pages = 0
    left = top
    for r, (length, n) in enumerate(zip(lengths, new)):
        state = 0
        if n < 0 or length + n > limit:
            state = 1
        elif n > 0:
            asked_tokens += n
            if asked_tokens > capacity:
                state = 2
        if state == 0:
            pages = _pages(length + n, page) - _pages(length, page)
            asked_pages += pages
            if pages and asked_pages > top:
                state = 3
            else:
                for j in range(pages):
                    left -= 1
                    tables[r, _pages(length, page) + j] = stack[left]
        granted = n if state == 0 else 0
        for position in range(length, length + granted):
            slots.append(int(tables[r, position // page]) * page + position % page)
            positions.append(position)
            requests.append(r)
            contexts.append(position + 1)
        starts.append(starts[-1] + granted)
        status.append(state)
        after.append(length + granted)
    pad = capacity - len(slots)
    return (np.array(slots + [-1] * pad, dtype=np.int64), np.array(positions + [0] * pad, dtype=np.int32),
            np.array(requests + [-1] * pad, dtype=np.int32), np.array(contexts + [0] * pad, dtype=np.int32),
            np.array(starts, dtype=np.int32), np.array(status, dtype=np.int32), np.array(after, dtype=np.int32),
            np.array([left], dtype=np.int32), tables)


def _exact_release(case, s):
    lengths, tables, stack = s["lengths"].numpy().copy(), s["tables"].numpy(), s["free"].numpy().copy()
    top = int(s["n_free"])
    for r, done in enumerate(s["done"].tolist()):
        if done:
            n = _pages(int(lengths[r]), case["page"])
            stack[top:top + n] = tables[r, :n]
            top += n
            lengths[r] = 0
    return lengths, np.array([top], dtype=np.int32), stack


def _exact_rotary(case, s):
    rotary = case["rotary"]
    if case["interleaved"]:
        a, b = torch.arange(0, rotary, 2), torch.arange(1, rotary, 2)
    else:
        a, b = torch.arange(rotary // 2), torch.arange(rotary // 2, rotary)

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            rms = (x.pow(2).sum(-1) / x.shape[-1] + 1e-6).sqrt()
            x = x / rms[..., None] * weight.double()
        angle = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()]
        z = torch.complex(x[..., a], x[..., b]) * angle[:, None, :]
        y = x.clone()
        y[..., a], y[..., b] = z.real, z.imag
        return y

    keys, values = s["key_cache"].double(), s["value_cache"].double()
    at = s["slots"]
    token = torch.nonzero(at >= 0).flatten()
    at = at[token]
    keys = keys.transpose(1, 2).reshape(-1, *s["k"].shape[1:])
    values = values.transpose(1, 2).reshape(-1, *s["v"].shape[1:])
    keys[at], values[at] = turned(s["k"], s["k_weight"])[token], s["v"].double()[token]
    shape = (s["key_cache"].shape[0], case["page"], case["kv_heads"], case["dim"])
    return turned(s["q"], s["q_weight"]), keys.view(shape).transpose(1, 2), values.view(shape).transpose(1, 2)


def _exact_attention(case, s):
    hk, d = case["kv_heads"], case["dim"]
    group, q = case["heads"] // hk, s["q"].double()
    out = torch.zeros_like(q)
    for row, n in enumerate(s["host_contexts"]):
        if not n:
            continue
        slot = torch.arange(n, device="cuda")
        page, offset = s["tables"][row].long()[slot // case["page"]], slot % case["page"]
        for h in range(hk):
            k, v = s["key_cache"][page, h, offset].double(), s["value_cache"][page, h, offset].double()
            score = k @ q[row, h * group:(h + 1) * group].T / math.sqrt(d)
            out[row, h * group:(h + 1) * group] = (score - score.logsumexp(0)).exp().T @ v
    return out


def _exact_logits(case, s):
    logits = s["logits"].double().cpu().numpy()
    rows, vocab = logits.shape
    out = np.empty_like(logits)
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "logits"}
    for r in range(rows):
        x = logits[r].copy()
        if case["penalties"]:
            n, prompt = int(host["lengths"][r]), int(host["prompt_lengths"][r])
            ids = host["history"][r, :n].astype(np.int64)
            rep, frequency, presence = (float(host[k][r]) for k in ("repetition", "frequency", "presence"))
            seen = np.unique(ids)
            x[seen] = np.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
            token, count = np.unique(ids[prompt:], return_counts=True)
            x[token] -= frequency * count + presence
        if case["bias"]:
            starts, tokens, values = (v.cpu().numpy() for v in s["bias"])
            biases = {}
            for e in range(starts[r], starts[r + 1]):
                biases[int(tokens[e])] = float(values[e])
            for token, value in biases.items():
                x[token] += value
        if case["masks"] and host["mask_rows"][r] >= 0:
            words = host["masks"][host["mask_rows"][r]].view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]
            x[bits == 0] = -np.inf
        out[r] = x
    return torch.from_numpy(out)
