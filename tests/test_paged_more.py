"""PagedDecoder behind shared prefixes, with drafted tokens, sampling and
experts, on small random models: on the CPU over the operators in plain torch
(plain_more_serving), and on the GPU over the kernels."""
import pytest
import torch

import plain_more_serving
from neuralzip_amd.gpu.paged import PagedDecoder
from test_paged_decoder import KINDS, MOE, VOCAB, agree, own_logits, prompt, small_model


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        plain_more_serving.install(monkeypatch)
    return request.param


def free_pages(decoder):
    return int(decoder.tables.n_free)


def check_free_pages(decoder):
    """Every page is in the stack once, or in one table row (a prefix's pages
    in its own row)."""
    page, n = decoder.tables.page_size, free_pages(decoder)
    used = decoder.tables.free[:n].tolist()
    for row, length in enumerate(decoder.tables.lengths.tolist()):
        first = 0
        if row < decoder.requests and decoder._prefix_of[row] >= 0:
            first = decoder._prefixes[decoder._prefix_of[row]].shape[0] // page
        used += decoder.tables.tables[row, first:-(-length // page)].tolist()
    assert sorted(used) == list(range(decoder.tables.num_pages))


# ------------------------------------------------------------------ prefixes

@pytest.mark.parametrize("length", [1, 15, 16, 17, 32, 45])
def test_requests_behind_a_prefix_compute_their_own_forward(device, length):
    model = small_model(device)
    decoder = PagedDecoder(model, requests=4, max_length=90, prefixes=2)
    prefix, other = prompt(length, 7), prompt(33, 8)
    numbers = [decoder.add_prefix(prefix), decoder.add_prefix(other)]
    assert numbers == [0, 1]
    before = free_pages(decoder)
    texts = []
    for i, (number, n) in enumerate(((0, 1), (0, 20), (1, 5), (None, 9))):
        ids = prompt(n, 10 + i)
        assert decoder.add(ids, prefix=number) == i
        texts.append((prefix if number == 0 else other if number == 1 else prompt(0)).tolist() + ids.tolist())
        assert agree(decoder.logits[0], own_logits(model, texts[-1]))
    # whole pages of the prefix are not taken again
    shared = [length // 16, length // 16, 2, 0]
    assert before - free_pages(decoder) == sum(-(-len(t) // 16) - s for t, s in zip(texts, shared))
    check_free_pages(decoder)
    for _ in range(18):
        for place, text in enumerate(texts):
            text.append(int(decoder.tokens[place]))
        decoder.step()
    for place, text in enumerate(texts):
        assert agree(decoder.logits[place], own_logits(model, text))
    check_free_pages(decoder)
    with pytest.raises(ValueError, match="begin with prefix 0"):
        decoder.drop_prefix(0)
    decoder.finish(0, 1)
    check_free_pages(decoder)
    decoder.drop_prefix(0)
    check_free_pages(decoder)
    # its pages serve others; the ones left are as they were
    assert decoder.add_prefix(prompt(50, 20)) == 0 and decoder.add(prompt(3, 21), prefix=0) == 0
    for place in (2, 3):
        texts[place].append(int(decoder.tokens[place]))
    decoder.step()
    for place, row in ((2, 1), (3, 2)):
        assert agree(decoder.logits[row], own_logits(model, texts[place]))
    decoder.finish(0, 2, 3)
    decoder.drop_prefix(0), decoder.drop_prefix(1)
    assert free_pages(decoder) == decoder.tables.num_pages and decoder.tables.lengths.sum() == 0


def test_prefix_refusals_leave_everything_as_it_was(device):
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=64, num_pages=5, prefixes=1)
    with pytest.raises(ValueError, match="no prefix"):
        decoder.add(prompt(3), prefix=0)
    with pytest.raises(ValueError, match="no prefix"):
        decoder.drop_prefix(0)
    number = decoder.add_prefix(prompt(40, 1))
    with pytest.raises(RuntimeError, match="places"):
        decoder.add_prefix(prompt(4, 2))
    with pytest.raises(ValueError, match="1 to 24"):
        decoder.add(prompt(25, 3), prefix=number)
    state = [t.clone() for t in decoder.tables._state]
    place = decoder.add(prompt(20, 4), prefix=number)        # 60 tokens: two pages shared, two of its own
    assert place == 0 and free_pages(decoder) == 0
    with pytest.raises(RuntimeError, match="free pages"):
        decoder.add(prompt(1, 5), prefix=number)
    assert decoder.tables.lengths.tolist() == [60, 0, 40]
    decoder.finish(place)
    for now, then in zip(decoder.tables._state[:1] + decoder.tables._state[3:], state[:1] + state[3:]):
        assert torch.equal(now, then)
    check_free_pages(decoder)

    def broken(*args, **kwargs):
        raise RuntimeError("on purpose")
    forward = model.model.layers[1].forward
    model.model.layers[1].forward = broken
    for n in (None, number):
        with pytest.raises(RuntimeError, match="on purpose"):
            decoder.add(prompt(4, 6), prefix=n)
        assert decoder.tables.lengths.tolist() == [0, 0, 40]
        check_free_pages(decoder)
    model.model.layers[1].forward = forward
    assert decoder.add(prompt(4, 6), prefix=number) == 0


# -------------------------------------------------------------------- drafts

def greedy(model, texts, n):
    """Answers of a decoder without drafts."""
    decoder = PagedDecoder(model, requests=len(texts), max_length=80)
    return decoder.generate(texts, n)


@pytest.mark.parametrize("most", [1, 3, 6])
def test_drafts_change_no_answer(device, most):
    """Right ones are accepted, wrong ones and those after them refused, none
    are none: the answers are those of one token at a time."""
    model = small_model(device)
    texts = [prompt(5, 1).tolist(), prompt(30, 2).tolist(), prompt(17, 3).tolist()]
    answers = greedy(model, texts, 30)
    decoder = PagedDecoder(model, requests=4, max_length=80, drafts=most)
    for text in texts:
        decoder.add(text)
    got = [[int(t)] for t in decoder.tokens[:3]]
    assert [g[0] for g in got] == [a[0] for a in answers]
    accepted = set()
    for turn in range(8):
        drafts = torch.full((4, most), -1)
        right = []
        for place in range(3):
            known = answers[place][len(got[place]):]
            good = (turn + place) % (most + 2)       # how many of the drafts are right
            ids = (known + [0] * most)[:most]
            if good < most:
                ids[good] = -1 if turn % 2 else (ids[good] + 1) % VOCAB
            drafts[place] = torch.tensor(ids)
            right.append(min(good, most))
        out = decoder.step(drafts.to(device))
        assert out.shape == (4, most + 1) and (out[3] == -1).all()
        for place in range(3):
            new = [t for t in out[place].tolist() if t >= 0]
            got[place] += new
            assert out[place, len(new):].eq(-1).all()
            if len(got[place]) <= 30:
                assert len(new) == right[place] + 1
            accepted.add(len(new) - 1)
        lengths = [len(text) + len(g) - 1 for text, g in zip(texts, got)]
        assert decoder.tables.lengths.tolist() == lengths + [0]
        assert decoder.tokens[:3].tolist() == [g[-1] for g in got]
        check_free_pages(decoder)
    assert accepted == set(range(most + 1))
    for g, a in zip(got, answers):
        assert g[:30] == a[:len(g)]


def test_drafts_up_to_max_length(device):
    """A request takes no more tokens than max_length leaves."""
    model = small_model(device)
    text = prompt(10, 1).tolist()
    answer = greedy(model, [text], 12)[0]
    decoder = PagedDecoder(model, requests=2, max_length=14, drafts=4, page_size=16)
    decoder.add(text)
    out = decoder.step(torch.tensor([answer[1:5], [-1] * 4], device=device))
    # four tokens fit: the last answer and three drafts
    assert out[0].tolist() == answer[1:5] + [-1] and decoder.tables.lengths.tolist() == [14, 0]
    keys = decoder.cache.clone()
    out = decoder.step(torch.tensor([answer[5:9], [-1] * 4], device=device))
    assert (out == -1).all() and decoder.tables.lengths.tolist() == [14, 0] and torch.equal(keys, decoder.cache)


def test_drafts_ask_for_the_pages_of_those_given(device):
    """A request asks for room for its drafts, not for as many as it might
    bring: without any it takes the last place of its last page."""
    model = small_model(device)
    text = prompt(10, 1).tolist()
    answer = greedy(model, [text], 12)[0]
    decoder = PagedDecoder(model, requests=2, max_length=80, drafts=4, page_size=16, num_pages=1)
    decoder.add(text)
    got = [int(decoder.tokens[0])]
    for n, fits in ((4, True), (4, False), (1, False), (0, True), (0, False)):   # 10 tokens, then 15, then 16
        drafts = torch.full((2, 4), -1)
        drafts[0, :n] = torch.tensor(answer[len(got):len(got) + n])
        lengths = decoder.tables.lengths.tolist()
        out = decoder.step(drafts.to(device))[0].tolist()
        new = answer[len(got):len(got) + n + 1] if fits else []
        assert out == new + [-1] * (5 - len(new))
        got += new
        assert decoder.tables.lengths.tolist() == [lengths[0] + len(new), 0]
        check_free_pages(decoder)
    assert got == answer[:7]


def test_drafts_with_penalties_see_the_drafts_before_them(device):
    model = small_model(device)
    texts = [prompt(6, 1).tolist()]
    plain = PagedDecoder(model, requests=1, max_length=60, repetition=1.4, frequency=0.3, presence=0.2)
    answer = plain.generate(texts, 12)[0]
    decoder = PagedDecoder(model, requests=1, max_length=60, repetition=1.4, frequency=0.3, presence=0.2, drafts=4)
    decoder.add(texts[0])
    got = [int(decoder.tokens[0])]
    while len(got) < 11:
        out = decoder.step(torch.tensor([(answer[len(got):] + [-1] * 4)[:4]], device=device))[0].tolist()
        got += [t for t in out if t >= 0]
    assert got[:12] == answer[:len(got)] and decoder._history[0, 6:6 + len(got)].tolist() == got


def test_draft_refusals(device):
    model = small_model(device)
    with pytest.raises(ValueError, match="grammar"):
        PagedDecoder(model, requests=2, max_length=20, drafts=1, grammar=True)
    with pytest.raises(ValueError, match="2048"):
        PagedDecoder(model, requests=1025, max_length=20, drafts=1)
    with pytest.raises(ValueError, match="1024"):
        PagedDecoder(model, requests=1, max_length=20, prefixes=1025)
    with pytest.raises(ValueError, match="negative"):
        PagedDecoder(model, requests=1, max_length=20, drafts=-1)
    decoder = PagedDecoder(model, requests=2, max_length=20, drafts=2)
    for bad in (torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 2), [[1, 2], [3, 4]]):
        with pytest.raises(ValueError, match="drafts are"):
            decoder.step(bad)
    with pytest.raises(ValueError, match="numbers"):
        decoder.step(numbers=(torch.zeros(6), torch.zeros(2)))
    with pytest.raises(ValueError, match="without drafts"):
        decoder.generate([[1, 2]], 3)
    plain = PagedDecoder(model, requests=2, max_length=20)
    with pytest.raises(ValueError, match="drafts are"):
        plain.step(torch.zeros(2, 0, dtype=torch.int64))


# ------------------------------------------------------------------ sampling

def picked(logits, t, u):
    p = (logits.double() / t).softmax(-1)
    return int((p.cumsum(0) > u * p.sum()).int().argmax())


@pytest.mark.parametrize("most", [0, 2])
def test_samples_follow_their_numbers(device, most):
    """From the model's own logits: sums of a few layers in 32 bits move a
    token's borders by some 1e-6, where the numbers here do not lie."""
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=50, temperature=0.8, drafts=most)
    texts = [prompt(5, 1).tolist(), prompt(12, 2).tolist()]
    for text in texts:
        decoder.add(text)
    tokens = decoder.tokens.tolist()
    for turn in range(5):
        for text, token in zip(texts, tokens):
            text.append(token)
        u = [0.13 + 0.17 * turn, 0.91 - 0.2 * turn]
        accept = torch.full((2 * (most + 1),), 0.999999, dtype=torch.float64, device=device)
        out = decoder.step(numbers=(accept, torch.tensor(u, dtype=torch.float64, device=device)))
        tokens = (out[:, 0] if most else out).tolist()
        assert tokens == [picked(own_logits(model, text).cpu(), 0.8, x) for text, x in zip(texts, u)]


def test_drafts_at_a_temperature_follow_their_numbers(device):
    model = small_model(device)
    decoder = PagedDecoder(model, requests=1, max_length=50, temperature=0.7, drafts=2)
    text = prompt(8, 4).tolist()
    decoder.add(text)
    text.append(int(decoder.tokens[0]))
    p = (own_logits(model, text).double() / 0.7).softmax(-1).cpu()
    first = int(p.topk(3)[1][2])
    chance = float(p[first])
    second = (own_logits(model, text + [first]).double() / 0.7).softmax(-1).cpu()
    likely = int(second.argmax())
    # the first accepted (its number below its chance), the second refused
    numbers = torch.tensor([chance * 0.9, 0.9999, 0.5], dtype=torch.float64, device=device)
    out = decoder.step(torch.tensor([[first, likely]], device=device),
                       numbers=(numbers, torch.tensor([0.4], dtype=torch.float64, device=device)))
    rest = second.clone()
    rest[likely] = 0.0
    following = int((rest.cumsum(0) > 0.4 * rest.sum()).int().argmax())
    assert out.tolist() == [[first, following, -1]]
    assert decoder.tables.lengths.tolist() == [len(text) + 1]


def test_sampling_draws_new_numbers(device):
    model = small_model(device)
    decoder = PagedDecoder(model, requests=16, max_length=40, temperature=5.0)
    torch.manual_seed(1)
    for _ in range(16):
        decoder.add(prompt(4, 3))
    first = decoder.tokens
    assert len(set(first.tolist())) > 4
    assert len(set(decoder.step().tolist())) > 4


# ------------------------------------------------------------------- experts

@pytest.mark.parametrize("kind", ["mixtral", "qwen2_moe", "qwen3_moe", "glm4_moe", "granitemoe", "granitemoeshared",
                                  "phimoe", "dots1", "hy_v3", "solar_open"])
def test_experts_compute_the_model_s_own_forward(device, kind):
    from transformers import CONFIG_MAPPING
    if kind not in CONFIG_MAPPING:
        pytest.skip(f"this Transformers has no {kind}")
    model = small_model(device, kind, **dict(MOE, head_dim=32, **KINDS.get(kind, {})))
    decoder = PagedDecoder(model, requests=2, max_length=40, experts=True)
    texts = [prompt(5, 1).tolist(), prompt(19, 2).tolist()]
    for text in texts:
        decoder.add(text)
    for _ in range(4):
        for place, text in enumerate(texts):
            text.append(int(decoder.tokens[place]))
        decoder.step()
        for place, text in enumerate(texts):
            assert agree(decoder.logits[place], own_logits(model, text))
    assert all("forward" not in m.__dict__ for m in decoder._experts + decoder._attentions)


def test_experts_refuse_what_they_do_not_compute(device):
    with pytest.raises(ValueError, match="mixture"):
        PagedDecoder(small_model(device), requests=1, max_length=20, experts=True)
    model = small_model(device, "mixtral", **dict(MOE, head_dim=32, hidden_act="relu"))
    with pytest.raises(ValueError, match="does not compute"):
        PagedDecoder(model, requests=1, max_length=20, experts=True)


# ----------------------------------------------------------------- all of it

@pytest.mark.gpu
@pytest.mark.parametrize("kind, more", [("llama", {}), ("qwen3_moe", dict(experts=True))])
def test_a_captured_step_with_prefixes_and_drafts(kind, more):
    """Replays beside an eager decoder on the same requests, drafts and
    numbers, while requests come and go."""
    device = "cuda:0"
    model = small_model(device, kind, **(dict(MOE, head_dim=32) if more else {}))
    pair = [PagedDecoder(model, requests=4, max_length=100, drafts=2, prefixes=1, temperature=0.9, num_pages=30, **more)
            for _ in range(2)]
    for decoder in pair:
        decoder.add_prefix(prompt(40, 1))

    def add(n, seed, prefix):
        places = []
        for decoder in pair:
            torch.manual_seed(seed)
            places.append(decoder.add(prompt(n, seed), prefix=prefix))
        assert places[0] == places[1]
    for n, seed, prefix in ((3, 2, 0), (20, 3, 0), (9, 4, None)):
        add(n, seed, prefix)

    def step(seed):
        g = torch.Generator(device=device).manual_seed(seed)
        drafts = torch.randint(-1, VOCAB, (4, 2), generator=g, device=device)
        drafts[0] = pair[0]._last[0]
        numbers = (0.3 * torch.rand(12, generator=g, device=device, dtype=torch.float64),
                   torch.rand(4, generator=g, device=device, dtype=torch.float64))
        outs = [decoder.step(drafts, numbers=numbers) for decoder in pair]
        assert torch.equal(outs[0], outs[1])
        for decoder in pair:
            assert torch.equal(decoder.tables.lengths, pair[0].tables.lengths)
            check_free_pages(decoder)
        assert torch.equal(pair[0].tokens, pair[1].tokens)
    step(1), step(2)
    pair[1].capture()
    torch.cuda.synchronize()
    for seed in range(3, 9):
        step(seed)
    for decoder in pair:
        decoder.finish(1)
    step(10)
    add(30, 5, 0)
    for seed in range(11, 16):
        step(seed)
