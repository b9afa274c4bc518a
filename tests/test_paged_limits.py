"""PagedDecoder with prefixes, drafts, sampling and experts: calls at the edges
of what it takes. On the CPU over the operators in plain torch, and on the GPU
over the kernels."""
import pytest
import torch

import plain_more_serving
from neuralzip_amd.gpu.paged import PagedDecoder
from test_paged_decoder import MOE, VOCAB, prompt, small_model


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        plain_more_serving.install(monkeypatch)
    return request.param


@pytest.mark.parametrize("count", [0, 1, 3])
def test_numbers_are_two(device, count):
    """One vector would leave the other's numbers of the step before, which
    must not be used twice."""
    decoder = PagedDecoder(small_model(device), requests=2, max_length=40, temperature=0.8, drafts=1)
    decoder.add(prompt(5))
    sizes = (4, 2, 2)
    given = tuple(torch.full((n,), 0.5, dtype=torch.float64, device=device) for n in sizes)
    lengths = decoder.tables.lengths.tolist()
    with pytest.raises(ValueError, match="float64 vectors of 4 and 2"):
        decoder.step(numbers=given[:count])
    with pytest.raises(ValueError, match="float64 vectors of 4 and 2"):
        decoder.step(numbers=([0.5] * 4, [0.5] * 2))
    assert decoder.tables.lengths.tolist() == lengths
    decoder.step(numbers=given[:2])
    decoder.step(numbers=list(given[:2]))
    assert decoder.tables.lengths.tolist() == [lengths[0] + 2, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind, more", [("llama", {}), ("qwen3_moe", dict(experts=True))])
def test_compressed_weights_behind_prefixes_and_drafts(kind, more):
    """bfloat16 weights decoded on the fly by the runtime: the same tokens as
    without it, since the decode is bit-exact, eagerly and from a graph, with
    prefixes, drafts, sampling and experts."""
    from neuralzip_amd.gpu.inference import NeuralZipRuntime, export_model_for_gpu
    from neuralzip_amd.setup import NeuralZipSetup
    device = "cuda:0"
    model = small_model(device, kind, **(dict(MOE, head_dim=32) if more else {})).bfloat16()

    def answers(capture):
        decoder = PagedDecoder(model, requests=3, max_length=100, drafts=2, prefixes=1, temperature=0.9, **more)
        prefix = decoder.add_prefix(prompt(40, 1))
        torch.manual_seed(2)
        for n, seed, behind in ((3, 2, prefix), (20, 3, prefix), (9, 4, None)):
            decoder.add(prompt(n, seed), prefix=behind)
        out = [decoder.tokens.tolist()]
        for turn in range(9):
            if turn == 3 and capture:
                decoder.capture()
            g = torch.Generator(device=device).manual_seed(turn)
            drafts = torch.randint(-1, VOCAB, (3, 2), generator=g, device=device)
            drafts[0] = decoder.tokens[0]
            # (by numbers of 0 every draft that has a chance is accepted)
            numbers = ((0.0 if turn % 2 else 0.3) * torch.rand(9, generator=g, device=device, dtype=torch.float64),
                       torch.rand(3, generator=g, device=device, dtype=torch.float64))
            out.append(decoder.step(drafts, numbers=numbers).tolist())
            if turn == 5:
                decoder.finish(1)
                torch.manual_seed(turn)
                assert decoder.add(prompt(30, 5), prefix=prefix) == 1
        return out
    want = answers(False)
    assert any(step[0][1] >= 0 for step in want[1:])      # some drafts were accepted
    runtime = NeuralZipRuntime.attach(model, export_model_for_gpu(model, NeuralZipSetup(chunk_size=16384).build(model)),
                                      device=device)
    assert answers(False) == want
    assert answers(True) == want
    assert runtime is not None


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 2, 5])
def test_replayed_steps_of_a_long_vocabulary(requests):
    """Replays give an eager decoder's tokens, with eager work between them."""
    vocab = 151936
    model = small_model("cuda:0", "llama", vocab_size=vocab)
    pair = [PagedDecoder(model, requests=requests, max_length=60) for _ in range(2)]
    for decoder in pair:
        for place in range(requests):
            decoder.add(torch.randint(3, vocab, (4 + place,), generator=torch.Generator().manual_seed(place)))
        decoder.step(), decoder.step()
    pair[1].capture()
    for _ in range(12):
        one, two = (decoder.step() for decoder in pair)
        assert torch.equal(one, two) and torch.equal(pair[0].tokens, pair[1].tokens)
        assert torch.equal(two, pair[1].logits.argmax(-1))
        torch.randn(1000, 1000, device="cuda:0").sum().item()


@pytest.mark.gpu
def test_a_replayed_choice_of_a_long_vocabulary():
    """The choice of a step alone, in a graph of few nodes."""
    vocab = 151936
    model = small_model("cuda:0", "llama", vocab_size=vocab)
    decoder = PagedDecoder(model, requests=1, max_length=60)
    decoder.add(prompt(5))
    logits = torch.randn(1, vocab, device="cuda:0")
    rows, contexts = torch.zeros(1, dtype=torch.int32, device="cuda:0"), torch.full((1,), 9, dtype=torch.int32, device="cuda:0")
    decoder._pick(logits, rows, contexts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder._pick(logits, rows, contexts)
    wrong = []
    for i in range(12):
        logits.copy_(torch.randn(1, vocab, device="cuda:0"))
        graph.replay()
        torch.cuda.synchronize()
        if int(decoder.tokens[0]) != int(logits.argmax(-1)):
            wrong.append(i)
    assert not wrong


@pytest.mark.parametrize("drafts", [0, 2])
@pytest.mark.parametrize("broken", ["layers", "lm_head"])
def test_a_step_that_fails_changes_no_request(device, drafts, broken):
    """Lengths and pages are those before it, and the next step's answers the
    ones that it would have given."""
    model = small_model(device)
    pair = [PagedDecoder(model, requests=3, max_length=60, drafts=drafts, prefixes=1) for _ in range(2)]
    texts = [prompt(15, 2), prompt(16, 3), prompt(5, 4)]
    for decoder in pair:
        prefix = decoder.add_prefix(prompt(20, 1))
        for text in texts:
            decoder.add(text, prefix=prefix)
        decoder.step()
    given = [] if not drafts else [torch.full((3, drafts), 7, device=device)]
    module = model.model.layers[1] if broken == "layers" else model.lm_head
    before = [t.clone() for t in pair[0].tables._state]

    def fails(*args, **kwargs):
        raise ArithmeticError("on purpose")
    module.forward = fails
    for _ in range(2):
        with pytest.raises(ArithmeticError):
            pair[0].step(*given)
    del module.forward
    state = pair[0].tables._state
    assert torch.equal(state[0], before[0]) and torch.equal(state[3], before[3])
    n = int(state[3])
    assert sorted(state[2][:n].tolist()) == sorted(before[2][:n].tolist())
    for _ in range(20):
        assert torch.equal(pair[0].step(*given), pair[1].step(*given))
        assert torch.equal(pair[0].tables.lengths, pair[1].tables.lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [65535, 65536, 70000])
def test_greedy_choices_of_more_requests_than_one_verification_takes(requests):
    device = "cuda:0"
    decoder = PagedDecoder(small_model(device), requests=requests, max_length=16)
    logits = torch.randn(requests, VOCAB, device=device)
    logits[:, 7] = logits.amax(-1)        # two largest, or one
    places = torch.arange(requests, dtype=torch.int32, device=device)
    decoder._pick(logits, places, torch.full_like(places, 3))
    assert torch.equal(decoder.tokens, (logits == logits.amax(-1, keepdim=True)).int().argmax(-1))
    assert torch.equal(decoder._history[:requests, 3].long(), decoder.tokens)
