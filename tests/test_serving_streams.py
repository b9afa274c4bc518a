"""Memory of the serving operators' calls on a stream of their own: what a
call was given is kept until the stream is done with it, whatever the caller
does with it after the call. Without a GPU the records are watched; with one,
a busy stream reads what the caller has let go."""
import pytest
import torch

from neuralzip_amd.gpu import serving


class Watched(torch.Tensor):
    """A tensor that notes the streams it is recorded for."""
    records = []

    def record_stream(self, stream):
        Watched.records.append((self.data_ptr(), stream))


class Lane:
    """A stream's stand-in."""
    cuda_stream = 7


@pytest.fixture
def calls(monkeypatch):
    """The C entries' argument bytes; nothing is launched."""
    seen = []
    monkeypatch.setattr(serving, "_call", lambda function, device, args, stream: seen.append(args))
    monkeypatch.setattr(serving, "_on", lambda stream: serving._CURRENT)
    monkeypatch.setattr(serving, "_like", lambda t, stream: torch.zeros_like(t))
    monkeypatch.setattr(torch.Tensor, "record_stream", Watched.record_stream)
    Watched.records = []
    return seen


def addresses(*tensors):
    return {t.data_ptr() for t in tensors}


def test_pages_calls_keep_their_tensors(calls):
    book, lane = serving.PageTables(3, 4, 16, 8, device="cpu"), Lane()
    new, done = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.bool)
    state = addresses(book.lengths, book.tables, book.free, book.n_free)
    book.extend(new, 4)
    book.release(done)
    assert not Watched.records
    out = serving.Step(3, 4, "cpu")
    assert book.extend(new, 4, out=out, stream=lane) is out
    assert {a for a, s in Watched.records} >= state | addresses(new, out.slots) and \
        all(s is lane for _, s in Watched.records)
    Watched.records = []
    book.release(done, stream=lane)
    assert {a for a, s in Watched.records} >= state | addresses(done)


def test_rotary_keeps_its_tensors(calls):
    cos, sin, weight = torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(16)
    op, lane = serving.Rotary(cos, sin, q_weight=weight), Lane()
    q, k, v = torch.zeros(2, 4, 16), torch.zeros(2, 2, 16), torch.zeros(2, 2, 16)
    keys, values = torch.zeros(4, 2, 16, 16), torch.zeros(4, 2, 16, 16)
    at, slots, out = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(2, 4, 16)
    op(q, k, v, at, slots, keys, values)
    assert not Watched.records
    op(q, k, v, at, slots, keys, values, out=out, stream=lane)
    assert {a for a, _ in Watched.records} >= addresses(q, k, v, at, slots, keys, values, out, cos, sin, weight)
    op(q, k, v, at, stream=lane)


# ---------------------------------------------------------------- on the GPU

DEVICE = "cuda:0"


def kept(tensors, call):
    """`call` on a busy stream, then its tensors are let go and memory of
    their sizes is asked for and overwritten: whether the call had what was
    in them. `tensors` is a list, which is emptied."""
    want = call(*tensors, stream=None).clone()
    busy = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(busy):
        torch.cuda._sleep(20_000_000)      # some ten milliseconds
    got = call(*tensors, stream=busy)
    sizes = [t.untyped_storage().nbytes() for t in tensors]
    del tensors[:]
    taken = [torch.full((size,), 0x55, dtype=torch.uint8, device=DEVICE) for size in sizes for _ in range(2)]
    torch.cuda.synchronize()
    assert taken
    return torch.equal(got, want)


def random(*shape, seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEVICE).to(dtype)


@pytest.mark.gpu
def test_rotary_reads_what_the_caller_has_let_go():
    cos, sin = torch.rand(9, 32, device=DEVICE), torch.rand(9, 32, device=DEVICE)
    op = serving.Rotary(cos, sin)
    tensors = [random(64, 4, 64, seed=1), random(64, 2, 64, seed=2), random(64, 2, 64, seed=3),
               (torch.arange(64, device=DEVICE) % 9).int()]
    assert kept(tensors, lambda q, k, v, at, stream: op(q, k, v, at, stream=stream))


@pytest.mark.gpu
def test_attention_reads_what_the_caller_has_let_go():
    """The plan is let go too; it was made on the current stream."""
    contexts = torch.tensor([500, 3000], dtype=torch.int32, device=DEVICE)
    tables = torch.arange(2 * 200, dtype=torch.int32, device=DEVICE).view(2, 200)

    def call(q, keys, values, tables, contexts, stream):
        plan = serving.AttentionPlan(contexts, heads=4, kv_heads=2)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
            plan.update(contexts, stream=stream)
        return serving.paged_attention(q, keys, values, tables, plan, stream=stream)
    tensors = [random(2, 4, 64, seed=1), random(400, 2, 16, 64, seed=2), random(400, 2, 16, 64, seed=3), tables, contexts]
    del tables, contexts
    assert kept(tensors, call)


@pytest.mark.gpu
def test_logits_and_pages_read_what_the_caller_has_let_go():
    def logits(x, history, lengths, factor, starts, ids, values, masks, rows, stream):
        return serving.adjust_logits(x, history=history, lengths=lengths, prompt_lengths=lengths, repetition=factor,
                                     frequency=factor, presence=factor, bias=(starts, ids, values), masks=masks,
                                     mask_rows=rows, stream=stream)

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)
    tensors = [random(2, 5000, seed=1, dtype=torch.float32), ints(*range(600)).view(2, 300), ints(300, 200),
               torch.tensor([1.5, 2.0], device=DEVICE), ints(0, 1, 3), ints(7, 8, 9),
               torch.tensor([1.0, 2.0, 3.0], device=DEVICE), torch.full((2, 157), -5, dtype=torch.int32, device=DEVICE),
               ints(1, 0)]
    assert kept(tensors, logits)

    def pages(new, stream):
        book = serving.PageTables(3, 8, 16, 24, device=DEVICE)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        step = book.extend(new, 64, stream=stream)
        with serving._on(stream):
            return torch.cat([step.slots, step.lengths.long()])
    assert kept([ints(20, 0, 33)], pages)
