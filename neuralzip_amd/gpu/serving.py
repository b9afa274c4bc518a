"""Operators of a serving step: many requests with lengths of their own in
one forward, around the weights that the runtime decodes.

  PageTables       block tables and a stack of free pages on the GPU; extend()
                   gives a step's tokens their pages, slots and positions and
                   release() takes finished requests' pages back
  Rotary           the heads' optional RMS norm and the position rotation of
                   queries and keys, with keys and values stored into their
                   pages, in one pass
  AttentionPlan    cuts a step's contexts into items of equal work, once for
  paged_attention  all layers; attention of single tokens over the pages
  adjust_logits    repetition, frequency and presence penalties, biases and
                   grammar masks, in one pass

Every call launches gfx950 kernels through the C ABI (nz_pages_*,
nz_rotary_store, nz_attention_*, nz_adjust_logits) on the current stream, or
on `stream`, where its tensors must be ready. They may be let go after the
call: they are recorded for `stream`. Results are that stream's, and who uses
them on another one waits for it and records them there. Nothing synchronises,
and lengths, tables and plans never leave the device, so that a step can be
captured in a HIP graph and replayed while the requests grow. The operators
serve: tensors that need a gradient are refused while gradients are on.

The reference has no counterpart; its forwards keep Transformers' own cache
and attention (neuralzip/gpu/inference.py:476-509).
"""
import torch

from neuralzip_amd import _native
from neuralzip_amd.gpu.decoder import _CURRENT, _stream_handle

_TYPES = {torch.bfloat16: _native.VALUE_BF16, torch.float16: _native.VALUE_FP16, torch.float32: _native.VALUE_FP32}
# Workgroups that an attention's items are cut into, over all key-value heads,
# if there are not more rows.
ATTENTION_WORKGROUPS = 256
# Query heads of one workgroup (the columns of a matrix instruction).
_HEADS = 16
# PageTables.extend's status of a request (enum nz_pages_status).
PAGES_OK, PAGES_TOO_LONG, PAGES_NO_ROOM, PAGES_NO_PAGE = range(4)


def _on(stream):
    return torch.cuda.stream(stream) if stream is not None else _CURRENT


def _like(t, stream):
    """A dense new tensor like t, allocated on `stream`."""
    if stream is None:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, memory_format=torch.contiguous_format)


def _call(function, device, args, stream):
    if device.type != "cuda":
        raise ValueError("The serving operators run on the GPU.")
    rc = function(args, _stream_handle(device, stream))
    if rc:
        _native.check(rc)


def _keep(stream, *tensors):
    """The tensors' memory is not given away before `stream` is done with them."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _refuse_gradients(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("The serving operators have no backward: call them under torch.no_grad().")


def _pointer(name, t, dtype, n, index):
    """The address of an optional vector, checked; 0 without one."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        _check_vector(name, t, dtype, n, index)
    return t.data_ptr()


# (Devices are compared by their index, -1 for the CPU: a call makes a dozen
# comparisons, and those of torch.device take twice as long.)
def _check_vector(name, t, dtype, n, index):
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {n} on device {index}; "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}.")


# Parts of one allocation. (The form that keeps no record of them as views of
# each other takes 0.7 us less for a step's eight arrays.)
_split = torch.unsafe_split_with_sizes


def _pool_layout(keys, values, kv_heads, head_dim, dtype, index):
    """Strides of a layer's two caches, (pages, kv_heads, page size, head_dim),
    their pages and page size."""
    shape = keys.shape
    if shape != values.shape or len(shape) != 4 or shape[1] != kv_heads or shape[3] != head_dim:
        raise ValueError(f"Caches must both be (pages, {kv_heads}, page size, {head_dim}); "
                         f"got {tuple(keys.shape)} and {tuple(values.shape)}.")
    if keys.dtype is not dtype or values.dtype is not dtype or keys.get_device() != index \
            or values.get_device() != index:
        raise ValueError("Caches must have the queries' dtype and device.")
    k0, k1, k2, k3 = keys.stride()
    v0, v1, v2, v3 = values.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("A head's elements must be contiguous in the caches.")
    return (k0, k1, k2, v0, v1, v2), shape[0], shape[2]


class Step:
    """What PageTables.extend found for a step's tokens, all on the device.

    Per token, `max_tokens` entries: `slots` (int64; page * page_size + place,
    -1 past the last token), `positions`, `requests` (-1 past the last) and
    `contexts` (position + 1; 0 past the last). Per request: `starts` (its
    first token; one more entry ends the last), `status` (PAGES_OK, or why it
    got no token) and `lengths` after the step; `n_free`, the free stack's
    height after it."""
    __slots__ = ("slots", "positions", "requests", "contexts", "starts", "status", "lengths", "n_free", "max_tokens",
                 "_sizes", "_pointers")

    def __init__(self, n_requests, max_tokens, device):
        self.max_tokens = max_tokens
        # one allocation: 8-byte slots first, then the 4-byte arrays
        words = torch.empty(5 * max_tokens + 3 * n_requests + 2, dtype=torch.int32, device=device)
        self._sizes = n_requests, max_tokens, words.get_device()
        at, starts = words.data_ptr(), words.data_ptr() + 20 * max_tokens
        self._pointers = (at, at + 8 * max_tokens, at + 12 * max_tokens, at + 16 * max_tokens, starts,
                          starts + 4 * (n_requests + 1), starts + 4 * (2 * n_requests + 1),
                          starts + 4 * (3 * n_requests + 1))
        (slots, self.positions, self.requests, self.contexts, self.starts, self.status, self.lengths,
         self.n_free) = _split(words, (2 * max_tokens, max_tokens, max_tokens, max_tokens, n_requests + 1, n_requests,
                                       n_requests, 1))
        self.slots = slots.view(torch.int64)


class Released:
    """Lengths and the free stack's height after PageTables.release."""
    __slots__ = ("lengths", "n_free")

    def __init__(self, n_requests, device):
        words = torch.empty(n_requests + 1, dtype=torch.int32, device=device)
        self.lengths, self.n_free = _split(words, (n_requests, 1))


class PageTables:
    """The pages of up to `requests` requests, of `page_size` tokens each (a
    power of two from 16 to 1024), out of `num_pages`.

    `lengths` (int32, one per request), `tables` (int32, requests x
    max_pages; entries past a request's pages mean nothing), `free` and
    `n_free` (the stack of unused pages and its height) are the state, on the
    device; they may be written by hand. All requests start empty and all pages
    free, the lowest on top. Calls that change one PageTables run one after
    another, on one stream or ordered by events."""

    def __init__(self, requests, max_pages, page_size, num_pages, device="cuda"):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024.")
        if requests < 1 or max_pages < 1 or num_pages < 1 or max_pages * page_size >= 1 << 31:
            raise ValueError("There must be requests and pages, and a request's tokens must be below 2**31.")
        self.requests, self.max_pages, self.page_size, self.num_pages = requests, max_pages, page_size, num_pages
        self._state = (torch.zeros(requests, dtype=torch.int32, device=device),
                       torch.full((requests, max_pages), -1, dtype=torch.int32, device=device),
                       torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device),
                       torch.full((1,), num_pages, dtype=torch.int32, device=device))
        self._pointers = tuple(t.data_ptr() for t in self._state)
        self.device, self._index = self.lengths.device, self.lengths.get_device()

    lengths = property(lambda self: self._state[0])
    tables = property(lambda self: self._state[1])
    free = property(lambda self: self._state[2])
    n_free = property(lambda self: self._state[3])

    def extend(self, new_tokens, max_tokens, *, advance=True, out=None, stream=None):
        """Gives every request its `new_tokens` (int32, one per request) new
        tokens, `max_tokens` in all at most, and returns the Step.

        In request order, a request gets nothing (and Step.status says why)
        if it would be negative or longer than its table row; else if it and
        those before it that fit their rows ask for more than max_tokens;
        else if it needs pages and it and those before it need more than are
        free. Without `advance` the state stays (but for table entries past
        the requests' pages): the step can be dropped, as after speculation.
        `out` is an earlier Step of the same sizes to write into."""
        _check_vector("new_tokens", new_tokens, torch.int32, self.requests, self._index)
        if max_tokens < 0:
            raise ValueError("max_tokens must not be negative.")
        if out is None:
            with _on(stream):
                out = Step(self.requests, max_tokens, self.device)
        elif out._sizes != (self.requests, max_tokens, self._index):
            raise ValueError("`out` is a Step of other sizes.")
        lengths, tables, free, n_free = self._pointers
        args = _native.PAGES_EXTEND.pack(lengths, new_tokens.data_ptr(), tables, free, n_free, *out._pointers,
                                         self.requests, self.max_pages, self.page_size, self.num_pages, max_tokens,
                                         bool(advance))
        _call(_native.lib().nz_pages_extend, self.device, args, stream)
        if stream is not None:
            _keep(stream, new_tokens, out.slots, *self._state)
        return out

    def release(self, done, *, advance=True, stream=None):
        """Puts the pages of the requests whose `done` (bool) is set back
        onto the free stack and sets their lengths to 0; returns the state
        after it. Without `advance` lengths and n_free stay."""
        _check_vector("done", done, torch.bool, self.requests, self._index)
        with _on(stream):
            out = Released(self.requests, self.device)
        lengths, tables, free, n_free = self._pointers
        args = _native.PAGES_RELEASE.pack(lengths, done.data_ptr(), tables, free, n_free, out.lengths.data_ptr(),
                                          out.n_free.data_ptr(), self.requests, self.max_pages, self.page_size,
                                          self.num_pages, bool(advance), 0)
        _call(_native.lib().nz_pages_release, self.device, args, stream)
        if stream is not None:
            _keep(stream, done, *self._state)
        return out


class Rotary:
    """Rotation by the angles whose cosines and sines are given, float32
    (positions, rotary_dim / 2): of the first rotary_dim elements of each
    head, in pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) when
    `interleaved`. With `q_weight` or `k_weight` (head_dim, in the values'
    dtype or float32) those heads are first divided by
    sqrt(mean(x^2) + eps) and multiplied by the weight."""

    def __init__(self, cos, sin, *, interleaved=False, q_weight=None, k_weight=None, eps=1e-6):
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise ValueError("cos and sin must both be float32 (positions, rotary_dim / 2).")
        if cos.shape[1] % 8 or cos.shape[1] > 128:
            raise ValueError("rotary_dim must be a multiple of 16 up to 256.")
        if sin.device != cos.device or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError("cos and sin must be contiguous on one device.")
        weights = [w for w in (q_weight, k_weight) if w is not None]
        if len({w.dtype for w in weights}) > 1 or len({w.shape for w in weights}) > 1:
            raise ValueError("The norm weights must have one dtype and size.")
        for w in weights:
            if w.dim() != 1 or not w.is_contiguous() or w.device != cos.device or w.dtype not in _TYPES:
                raise ValueError("Norm weights must be contiguous vectors on cos's device.")
        self.cos, self.sin, self.q_weight, self.k_weight = cos, sin, q_weight, k_weight
        self.rotary_dim, self.interleaved, self.eps = 2 * cos.shape[1], bool(interleaved), float(eps)
        self._device, self._index, self._positions = cos.device, cos.get_device(), cos.shape[0]
        self._weight_type = _TYPES[weights[0].dtype] if weights else None
        self._weight_dim = weights[0].shape[0] if weights else None
        self._tables = (cos.data_ptr(), sin.data_ptr(), q_weight.data_ptr() if q_weight is not None else 0,
                        k_weight.data_ptr() if k_weight is not None else 0)

    def __call__(self, q, k, v, positions, slots=None, key_cache=None, value_cache=None, *, out=None, stream=None):
        """Rotates q (tokens, heads, head_dim) and k (tokens, kv_heads,
        head_dim) to `positions` (int32, per token), stores k and v at
        `slots` (int64, per token; -1: nowhere) of the caches (pages,
        kv_heads, page size, head_dim) and returns the rotated q (`out`, which
        may be q, or a new tensor). head_dim is a multiple of 16 up to 256;
        any strides whose tokens and heads lie on 16-byte boundaries. Held in
        32 bits and rounded once. Tokens' slots must differ. A slot outside
        the caches stores nothing, a position outside the tables gives NaN."""
        if torch.is_grad_enabled():
            _refuse_gradients(q, k, v, self.q_weight, self.k_weight)
        dtype, index, shape, kv_shape = q.dtype, q.get_device(), q.shape, k.shape
        if len(shape) != 3 or len(kv_shape) != 3 or kv_shape != v.shape:
            raise ValueError("q, k and v must be (tokens, heads, head_dim), k and v alike.")
        tokens, heads, dim = shape
        kv_tokens, kv_heads, kv_dim = kv_shape
        kind = _TYPES.get(dtype)
        if kind is None or kv_tokens != tokens or kv_dim != dim or self.rotary_dim > dim:
            raise ValueError(f"q {tuple(shape)} {dtype} and k {tuple(kv_shape)} do not fit one another or the "
                             f"rotation of {self.rotary_dim} elements.")
        if k.dtype is not dtype or v.dtype is not dtype or k.get_device() != index or v.get_device() != index \
                or index != self._index:
            raise ValueError("q, k, v and the tables must match in dtype and device.")
        weight_type = self._weight_type
        if weight_type is None:
            weight_type = kind
        elif self._weight_dim != dim or weight_type not in (kind, _native.VALUE_FP32):
            raise ValueError("Norm weights must be head_dim values of q's dtype or float32.")
        _check_vector("positions", positions, torch.int32, tokens, index)
        q0, q1, q2 = q.stride()
        k0, k1, k2 = k.stride()
        v0, v1, v2 = v.stride()
        if q2 != 1 or k2 != 1 or v2 != 1:
            raise ValueError("A head's elements must be contiguous.")
        if key_cache is None and value_cache is None and slots is None:
            pool, key_ptr, value_ptr, slots_ptr, page_size, pages = (0, 0, 0, 0, 0, 0), 0, 0, 0, 0, 0
        elif key_cache is None or value_cache is None or slots is None:
            raise ValueError("The two caches and the slots go together.")
        else:
            _check_vector("slots", slots, torch.int64, tokens, index)
            pool, pages, page_size = _pool_layout(key_cache, value_cache, kv_heads, dim, dtype, index)
            key_ptr, value_ptr, slots_ptr = key_cache.data_ptr(), value_cache.data_ptr(), slots.data_ptr()
        if out is None:
            out = _like(q, stream)
            o0, o1 = heads * dim, dim
        else:
            o0, o1, o2 = out.stride() if out.dim() == 3 else (0, 0, 0)
            if out.shape != shape or out.dtype is not dtype or out.get_device() != index or o2 != 1:
                raise ValueError("`out` must be like q, with contiguous heads.")
        args = _native.ROTARY.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), key_ptr, value_ptr, *self._tables,
            positions.data_ptr(), slots_ptr, q0, q1, k0, k1, v0, v1, o0, o1, *pool, tokens, heads,
            kv_heads, dim, self.rotary_dim, self.interleaved, page_size, pages, self._positions, kind, weight_type,
            self.eps)
        _call(_native.lib().nz_rotary_store, self._device, args, stream)
        if stream is not None:
            _keep(stream, q, k, v, positions, slots, key_cache, value_cache, out, self.cos, self.sin, self.q_weight,
                  self.k_weight)
        return out


class AttentionPlan:
    """The work of a step's attention: `contexts` (int32, keys that each row
    of queries sees) cut into items of about equal length, for `heads` query
    heads over `kv_heads`. Row i belongs to request requests[i] (int32), or
    to request i. Made on the device, so it follows lengths that the host
    does not know; update() makes it anew in the same memory, also inside a
    captured graph. One plan serves all layers of the step, whose calls run
    one after another, on one stream or ordered by events."""

    def __init__(self, contexts, *, heads, kv_heads, requests=None, stream=None):
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a positive multiple of kv_heads.")
        if contexts.dim() != 1 or contexts.dtype != torch.int32 or not contexts.is_cuda:
            raise ValueError("contexts must be an int32 vector on the GPU.")
        self.rows, self.heads, self.kv_heads = contexts.shape[0], heads, kv_heads
        self.device, self._index = contexts.device, contexts.get_device()
        self._parts = kv_heads * -(-(heads // kv_heads) // _HEADS)
        self._target = max(1, ATTENTION_WORKGROUPS // self._parts)
        self.capacity = (max(1, -(-self.rows // self._target)) + 1) * self._target
        with _on(stream):
            words = torch.empty(self.capacity * (8 + self._parts), dtype=torch.int32, device=self.device)
        items, self._counters = words.split((8 * self.capacity, self.capacity * self._parts))
        self.items = items.view(self.capacity, 8)
        self._pointers = items.data_ptr(), self._counters.data_ptr()
        self._stream, self._scratch = _stream_handle(self.device, stream), {}
        self.update(contexts, requests=requests, stream=stream)

    def update(self, contexts, *, requests=None, stream=None):
        """Plans the same number of rows anew."""
        _check_vector("contexts", contexts, torch.int32, self.rows, self._index)
        if requests is not None:
            _check_vector("requests", requests, torch.int32, self.rows, self._index)
        rc = _native.lib().nz_attention_plan(contexts.data_ptr(), requests.data_ptr() if requests is not None else None,
                                             self.rows, self._target, self._parts, *self._pointers,
                                             _stream_handle(self.device, stream))
        if rc:
            _native.check(rc)
        if stream is not None:
            _keep(stream, contexts, requests, self.items)
        return self

    def _partials(self, head_dim, handle, stream):
        """Address of the scratch for calls of `head_dim` on one stream."""
        scratch = self._scratch.get((handle, head_dim))
        if scratch is None:
            words = _native.lib().nz_attention_partials(self.capacity, self.heads, head_dim)
            with _on(stream):
                scratch = torch.empty(words, dtype=torch.float32, device=self.device)
                if handle != self._stream:   # the plan's memory must outlive what runs there
                    self.items.record_stream(torch.cuda.current_stream(self.device))
            self._scratch[handle, head_dim] = scratch
        return scratch.data_ptr()


def paged_attention(q, key_cache, value_cache, tables, plan, *, scale=None, out=None, stream=None):
    """softmax(scale q.K) V for every row of q (rows, heads, head_dim), over
    the plan's context of its request: the keys and values at the request's
    pages (`tables`, int32 (requests, max_pages)) of the caches (pages,
    kv_heads, page size, head_dim). Query head h reads key-value head
    h // (heads / kv_heads). `scale` is head_dim ** -0.5 by default. A row
    without keys gives zeros; keys of pages outside the caches, and keys whose
    score is -infinity, count as masked. Sums and softmax in 32 bits, in an
    order that only the plan decides; values are summed before the division,
    so the largest one times the context must be below 3e38. head_dim is a multiple of 16 up to 256; strides may be any that
    keep heads, tokens and pages on 16-byte boundaries."""
    if torch.is_grad_enabled():
        _refuse_gradients(q, key_cache, value_cache)
    dtype, index, shape = q.dtype, q.get_device(), q.shape
    kind = _TYPES.get(dtype)
    if len(shape) != 3 or shape[0] != plan.rows or shape[1] != plan.heads or kind is None:
        raise ValueError(f"q must be ({plan.rows}, {plan.heads}, head_dim) in bfloat16, float16 or float32; "
                         f"got {tuple(shape)} {dtype}.")
    rows, heads, dim = shape
    if index != plan._index or tables.get_device() != index:
        raise ValueError("q, the tables and the plan must be on one device.")
    table_shape = tables.shape
    if len(table_shape) != 2 or tables.dtype is not torch.int32 or not tables.is_contiguous():
        raise ValueError("tables must be a contiguous int32 (requests, max_pages).")
    pool, pages, page_size = _pool_layout(key_cache, value_cache, plan.kv_heads, dim, dtype, index)
    q0, q1, q2 = q.stride()
    if out is None:
        out = _like(q, stream)
        o0, o1, o2 = heads * dim, dim, 1
    else:
        if out.shape != shape or out.dtype is not dtype or out.get_device() != index:
            raise ValueError("`out` must be like q.")
        o0, o1, o2 = out.stride()
    if q2 != 1 or o2 != 1:
        raise ValueError("A head's elements must be contiguous.")
    handle = _stream_handle(plan.device, stream)
    args = _native.ATTENTION.pack(
        q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), out.data_ptr(), tables.data_ptr(),
        *plan._pointers, plan._partials(dim, handle, stream), q0, q1, o0, o1, *pool, rows, plan.capacity, heads,
        plan.kv_heads, dim, *table_shape, page_size, pages, kind, dim ** -0.5 if scale is None else scale, 0)
    rc = _native.lib().nz_attention(args, handle)
    if rc:
        _native.check(rc)
    if stream is not None:
        _keep(stream, q, key_cache, value_cache, tables, out)
    return out


def adjust_logits(logits, *, history=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None,
                  presence=None, bias=None, masks=None, mask_rows=None, out=None, stream=None):
    """The logits (rows, vocab) that a sampler takes, in their own dtype:

      x / repetition, or x * repetition where x <= 0, for tokens in the row's
      history; minus frequency * count and presence for tokens in it after
      the prompt; plus the row's bias; -inf where the row's mask has no bit.

    history: int32 or int64 token ids (rows, capacity), the first lengths[row]
    (int32) of which count, the first prompt_lengths[row] (int32) of those as
    the prompt; ids outside the vocabulary are ignored. repetition, frequency,
    presence: float32 per row. bias: (starts, tokens, values), int32 (rows +
    1), int32 and float32: row r's entries are starts[r] .. starts[r + 1] - 1,
    and a token's last one counts. masks: int32 (any number, ceil(vocab /
    32)), token v's bit is bit v % 32 of word v // 32; mask_rows: int32 per
    row, the row's mask, -1 for none (row i has mask i by default). In 32
    bits, rounded once. At most 65535 rows. `out` may be logits itself."""
    if torch.is_grad_enabled():
        _refuse_gradients(logits)
    if logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda or logits.stride(1) != 1:
        raise ValueError("logits must be (rows, vocab) in bfloat16, float16 or float32 on the GPU, rows contiguous.")
    (rows, vocab), index = logits.shape, logits.get_device()
    history_ptr = lengths_ptr = prompt_ptr = history_row = capacity = id_bytes = 0
    if history is not None:
        if history.dim() != 2 or history.shape[0] != rows or history.dtype not in (torch.int32, torch.int64) \
                or history.get_device() != index or (history.stride(1) != 1 and history.shape[1] > 1):
            raise ValueError("history must be int32 or int64 (rows, capacity), rows contiguous, on the logits' device.")
        if lengths is None:
            raise ValueError("A history needs its lengths.")
        history_ptr = history.data_ptr()
        lengths_ptr = _pointer("lengths", lengths, torch.int32, rows, index)
        prompt_ptr = _pointer("prompt_lengths", prompt_lengths, torch.int32, rows, index)
        capacity, history_row, id_bytes = history.shape[1], history.stride(0), history.element_size()
    elif lengths is not None or prompt_lengths is not None or repetition is not None or frequency is not None \
            or presence is not None:
        raise ValueError("Penalties and lengths need the history.")
    starts_ptr = tokens_ptr = values_ptr = n_bias = 0
    if bias is not None:
        starts, tokens, values = bias
        n_bias = tokens.shape[0]
        starts_ptr = _pointer("bias starts", starts, torch.int32, rows + 1, index)
        tokens_ptr = _pointer("bias tokens", tokens, torch.int32, n_bias, index)
        values_ptr = _pointer("bias values", values, torch.float32, n_bias, index)
    masks_ptr = mask_rows_ptr = n_masks = 0
    if masks is not None:
        if masks.dim() != 2 or masks.dtype != torch.int32 or masks.shape[1] != (vocab + 31) // 32 \
                or masks.get_device() != index or not masks.is_contiguous():
            raise ValueError(f"masks must be contiguous int32 (masks, {(vocab + 31) // 32}) on the logits' device.")
        masks_ptr, n_masks = masks.data_ptr(), masks.shape[0]
        mask_rows_ptr = _pointer("mask_rows", mask_rows, torch.int32, rows, index)
        if mask_rows is None and n_masks != rows:
            raise ValueError("Without mask_rows there must be one mask per row.")
    elif mask_rows is not None:
        raise ValueError("mask_rows need masks.")
    if out is None:
        out = _like(logits, stream)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.get_device() != index or out.stride(1) != 1:
        raise ValueError("`out` must be like logits, rows contiguous.")
    args = _native.LOGITS.pack(
        logits.data_ptr(), out.data_ptr(), history_ptr, lengths_ptr, prompt_ptr,
        _pointer("repetition", repetition, torch.float32, rows, index),
        _pointer("frequency", frequency, torch.float32, rows, index),
        _pointer("presence", presence, torch.float32, rows, index), starts_ptr, tokens_ptr, values_ptr, masks_ptr,
        mask_rows_ptr, logits.stride(0), out.stride(0), history_row, rows, vocab, capacity, n_bias, n_masks,
        _TYPES[logits.dtype], id_bytes, 0)
    _call(_native.lib().nz_adjust_logits, logits.device, args, stream)
    if stream is not None:
        _keep(stream, logits, history, lengths, prompt_lengths, repetition, frequency, presence, *(bias or ()), masks,
              mask_rows, out)
    return out
