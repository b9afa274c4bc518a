"""The serving operators in plain torch, for tests of PagedDecoder on hosts
without a GPU: the same classes and functions as neuralzip_amd.gpu.serving,
whose rules and results they follow, on the CPU."""
import math

import torch

from neuralzip_amd.gpu import serving


class PageTables(serving.PageTables):
    def extend(self, new_tokens, max_tokens, *, advance=True, out=None, stream=None):
        assert new_tokens.dtype == torch.int32 and new_tokens.shape == (self.requests,) and stream is None
        out = serving.Step(self.requests, max_tokens, self.device) if out is None else out
        assert out._sizes == (self.requests, max_tokens, self._index)
        page, left, at, asked, wanted = self.page_size, int(self.n_free), 0, 0, 0
        out.slots.fill_(-1), out.positions.zero_(), out.requests.fill_(-1), out.contexts.zero_()
        for r, (length, n) in enumerate(zip(self.lengths.tolist(), new_tokens.tolist())):
            state, old, pages = serving.PAGES_OK, -(-length // page), 0
            if n < 0 or length + n > self.max_pages * page:
                state = serving.PAGES_TOO_LONG
            elif n:
                asked += n
                if asked > max_tokens:
                    state = serving.PAGES_NO_ROOM
            if state == serving.PAGES_OK:
                pages = -(-(length + n) // page) - old
                wanted += pages
                if pages and wanted > int(self.n_free):
                    state = serving.PAGES_NO_PAGE
            n = n if state == serving.PAGES_OK else 0
            out.starts[r], out.status[r], out.lengths[r] = at, state, length + n
            for j in range(pages if n else 0):
                left -= 1
                self.tables[r, old + j] = self.free[left]
            for position in range(length, length + n):
                out.slots[at] = int(self.tables[r, position // page]) * page + position % page
                out.positions[at], out.requests[at], out.contexts[at] = position, r, position + 1
                at += 1
        out.starts[self.requests], out.n_free[0] = at, left
        if advance:
            self.lengths.copy_(out.lengths)
            self.n_free.copy_(out.n_free)
        return out

    def release(self, done, *, advance=True, stream=None):
        assert done.dtype == torch.bool and done.shape == (self.requests,) and advance and stream is None
        out, left = serving.Released(self.requests, self.device), int(self.n_free)
        for r, length in enumerate(self.lengths.tolist()):
            for j in range(-(-length // self.page_size) if done[r] else 0):
                self.free[left] = self.tables[r, j]
                left += 1
            out.lengths[r] = 0 if done[r] else length
        out.n_free[0] = left
        self.lengths.copy_(out.lengths)
        self.n_free.copy_(out.n_free)
        return out


class Rotary(serving.Rotary):
    def __call__(self, q, k, v, positions, slots=None, key_cache=None, value_cache=None, *, out=None, stream=None):
        known = (positions >= 0) & (positions < self.cos.shape[0])
        at = torch.where(known, positions, 0).long()
        c, s = (torch.where(known[:, None], t[at], math.nan)[:, None] for t in (self.cos, self.sin))
        half = self.rotary_dim // 2
        assert not self.interleaved and 2 * half <= q.shape[-1]

        def turned(x, weight):
            y = x.float()
            if weight is not None:
                assert weight.shape == y.shape[-1:]
                y = y * (y.square().mean(-1, keepdim=True) + self.eps).rsqrt() * weight.float()
            a, b, rest = y.split((half, half, y.shape[-1] - 2 * half), -1)
            return torch.cat((a * c - b * s, b * c + a * s, rest), -1).to(x.dtype)
        if slots is not None:
            page, most = key_cache.shape[2], key_cache.shape[0] * key_cache.shape[2]
            keys = turned(k, self.k_weight)
            for t, slot in enumerate(slots.tolist()):
                if 0 <= slot < most:
                    key_cache[slot // page, :, slot % page] = keys[t]
                    value_cache[slot // page, :, slot % page] = v[t]
        return turned(q, self.q_weight)


class AttentionPlan:
    def __init__(self, contexts, *, heads, kv_heads, requests=None, stream=None):
        self.heads, self.kv_heads, self.rows = heads, kv_heads, contexts.shape[0]
        self.update(contexts, requests=requests)

    def update(self, contexts, *, requests=None, stream=None):
        assert contexts.shape == (self.rows,)
        self.contexts = contexts.tolist()
        self.requests = list(range(self.rows)) if requests is None else requests.tolist()
        return self


def paged_attention(q, key_cache, value_cache, tables, plan, *, scale=None, out=None, stream=None):
    assert q.shape[:2] == (plan.rows, plan.heads) and key_cache.shape[1] == plan.kv_heads
    out, page, group = torch.zeros_like(q), key_cache.shape[2], plan.heads // plan.kv_heads
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for row, (n, request) in enumerate(zip(plan.contexts, plan.requests)):
        if n <= 0 or not 0 <= request < tables.shape[0]:
            continue
        pages = tables[request, :-(-n // page)].long()
        k, v = (c[pages].transpose(1, 2).reshape(-1, plan.kv_heads, q.shape[-1])[:n].float().repeat_interleave(group, 1)
                for c in (key_cache, value_cache))
        weights = ((k * q[row].float()).sum(-1) * scale).softmax(0)
        out[row] = (weights[..., None] * v).sum(0)
    return out


def adjust_logits(logits, *, history=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None,
                  presence=None, masks=None, mask_rows=None, out=None, stream=None):
    x, vocab = logits.float(), logits.shape[1]
    for row in range(x.shape[0]):
        ids = history[row, :int(lengths[row])].long() if history is not None else torch.zeros(0, dtype=torch.int64)
        answer = ids[int(prompt_lengths[row]) if prompt_lengths is not None else 0:]
        seen, counts = (torch.bincount(i, minlength=vocab) for i in (ids, answer))
        if history is not None:
            x[row] = torch.where(seen > 0, torch.where(x[row] > 0, x[row] / repetition[row], x[row] * repetition[row]),
                                 x[row])
            x[row] -= counts * frequency[row] + (counts > 0) * presence[row]
        m = row if mask_rows is None else int(mask_rows[row])
        if masks is not None and 0 <= m < masks.shape[0]:
            bits = (masks[m].long()[:, None] >> torch.arange(32)) & 1
            x[row] = x[row].masked_fill(bits.flatten()[:vocab] == 0, -math.inf)
    return x.to(logits.dtype)


def install(monkeypatch):
    """PagedDecoder and its caller get these instead of the kernels."""
    for name in ("PageTables", "Rotary", "AttentionPlan", "paged_attention", "adjust_logits"):
        monkeypatch.setattr(serving, name, globals()[name])
