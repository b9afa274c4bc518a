"""Shared plans, trims, verification and experts in plain torch, for tests of
PagedDecoder on hosts without a GPU: those of neuralzip_amd.gpu.serving, whose
rules and results they follow, on the CPU."""
import torch

import plain_serving
from neuralzip_amd.gpu import serving


class PageTables(plain_serving.PageTables):
    def trim(self, keep, *, advance=True, stream=None):
        assert keep.dtype == torch.int32 and keep.shape == (self.requests,) and advance and stream is None
        out, left = serving.Released(self.requests, self.device), int(self.n_free)
        for r, (length, kept) in enumerate(zip(self.lengths.tolist(), keep.tolist())):
            kept = min(max(kept, 0), length)
            for j in range(-(-kept // self.page_size), -(-length // self.page_size)):
                self.free[left] = self.tables[r, j]
                left += 1
            out.lengths[r] = kept
        out.n_free[0] = left
        self.lengths.copy_(out.lengths)
        self.n_free.copy_(out.n_free)
        return out


class SharedPlan(plain_serving.AttentionPlan):
    """Groups change what is read, not what comes out; they are checked
    against the tables when they are used."""
    def __init__(self, contexts, *, heads, kv_heads, requests=None, groups=None, shared=None, stream=None):
        self.heads, self.kv_heads, self.rows = heads, kv_heads, contexts.shape[0]
        self.update(contexts, requests=requests, groups=groups, shared=shared)

    def update(self, contexts, *, requests=None, groups=None, shared=None, stream=None):
        super().update(contexts, requests=requests)
        self.groups = [] if groups is None else groups.tolist()
        self.shared = [] if shared is None else shared.tolist()
        return self


def paged_attention(q, key_cache, value_cache, tables, plan, **more):
    for g, n in enumerate(getattr(plan, "shared", ())):
        pages = {tuple(tables[r, :-(-n // key_cache.shape[2])].tolist()) for r, group in enumerate(plan.groups) if group == g}
        assert len(pages) <= 1
    return plain_serving.paged_attention(q, key_cache, value_cache, tables, plan, **more)


def verify_drafts(logits, tokens, starts, accept, sample, *, draft_probs=None, temperature=None, stream=None):
    assert draft_probs is None and tokens.dtype == torch.int64 and starts.dtype == torch.int32
    assert accept.dtype == sample.dtype == torch.float64 and accept.shape == tokens.shape == logits.shape[:1]
    n = starts.shape[0] - 1
    accepted, following = torch.zeros(n, dtype=torch.int32), torch.full((n,), -1, dtype=torch.int64)
    for r, (first, end) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
        for row in range(first, end):
            x, t = logits[row].double(), 1.0 if temperature is None else float(temperature[r])
            p = (x / t).softmax(-1) if t > 0 else torch.nn.functional.one_hot(x.argmax(), x.shape[0]).double()
            d = int(tokens[row + 1]) if row + 1 < end else -1
            accepted[r] = row - first
            if 0 <= d < x.shape[0]:
                if float(accept[row]) < float(p[d]):
                    continue
                rest = p.clone()
                rest[d] = 0.0
                p = rest if rest.sum() > 0 else p
            following[r] = int((p.cumsum(0) > float(sample[r]) * p.sum()).int().argmax())
            break
    return accepted, following


def expert_mlp(x, ids, weights, gate_up, down, *, activation="silu", out=None, stream=None):
    assert weights.dtype == torch.float32 and ids.shape == weights.shape and activation == "silu"
    out = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for e, w in zip(ids[t].tolist(), weights[t].tolist()):
            gate, up = (gate_up[e].detach() @ x[t]).chunk(2)
            out[t] += w * (down[e].detach() @ (torch.nn.functional.silu(gate) * up))
    return out


def install(monkeypatch):
    plain_serving.install(monkeypatch)
    for name in ("PageTables", "SharedPlan", "paged_attention", "verify_drafts", "expert_mlp"):
        monkeypatch.setattr(serving, name, globals()[name])
