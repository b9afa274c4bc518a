"""PagedDecoder's bookkeeping, on small random models: on the CPU over the
operators in plain torch (plain_serving), and on the GPU over the kernels."""
import contextlib

import pytest
import torch

import plain_serving
from neuralzip_amd.gpu import paged
from neuralzip_amd.gpu.paged import PagedDecoder

VOCAB = 200
SIZES = dict(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, intermediate_size=96, num_hidden_layers=3,
             vocab_size=VOCAB, max_position_embeddings=256, tie_word_embeddings=False, pad_token_id=0, bos_token_id=1,
             eos_token_id=2)


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        plain_serving.install(monkeypatch)
    return request.param


def small_model(device, kind="llama", **config):
    from transformers import CONFIG_MAPPING, AutoModelForCausalLM
    torch.manual_seed(5)
    model = AutoModelForCausalLM.from_config(CONFIG_MAPPING[kind](**dict(SIZES, **config)))
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() > 1:
                p.copy_(torch.randn(p.shape) * 0.15)
            else:
                p.add_(torch.randn(p.shape) * 0.1)
    return model.float().to(device).eval()


def prompt(n, seed=1):
    return torch.randint(3, VOCAB, (n,), generator=torch.Generator().manual_seed(seed))


def own_logits(model, ids):
    """The model's own logits after `ids`."""
    with torch.no_grad():
        return model(input_ids=torch.as_tensor(ids, device=model.device)[None], use_cache=False).logits[0, -1]


def agree(got, want):
    """Logits of a few layers' float32 sums of at most some hundred terms, in
    two orders: they differ by far less than 1e-3 of the largest."""
    return bool((got - want).abs().max() <= 1e-3 * want.abs().max())


@pytest.mark.parametrize("most", [20, 32, 33])
def test_requests_at_max_length_stay_as_they_are(device, most):
    """Whether or not max_length fills its pages: a request that has reached
    it gets no more tokens, nothing of its keys changes and nothing of the
    next request's history is written."""
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=most, repetition=1.3)
    long, short = prompt(most - 2, 1), prompt(3, 2)
    first, second = decoder.add(long), decoder.add(short)
    decoder.step(), decoder.step()
    assert decoder.tables.lengths.tolist() == [most, 5]
    keys, history = decoder.cache.clone(), decoder._history[first].clone()
    pages = decoder.tables.tables[first, :-(-most // 16)].long()
    for i in range(4):
        decoder.step()
        assert decoder.tables.lengths.tolist() == [most, 6 + i]
    assert torch.equal(decoder.cache[:, :, pages], keys[:, :, pages]) and torch.isfinite(decoder.cache).all()
    assert torch.equal(decoder._history[first], history)
    assert decoder._history[second, :3].tolist() == short.tolist()


MOE = dict(num_experts=4, num_local_experts=4, n_routed_experts=4, num_experts_per_tok=2, moe_intermediate_size=48,
           shared_expert_intermediate_size=48, n_shared_experts=1, n_group=1, topk_group=1)
# What small models of a type need beside SIZES and MOE.
KINDS = {"stablelm": dict(hidden_size=256), "phimoe": dict(sliding_window=None), "mistral": dict(sliding_window=None),
         "exaone4": dict(sliding_window=None, layer_types=["full_attention"] * 3),
         "granite": dict(attention_multiplier=0.18), "granitemoe": dict(attention_multiplier=0.18),
         "granitemoeshared": dict(attention_multiplier=0.18)}
# Settings that a step follows, and that change what the model computes.
FOLLOWED = [("llama", dict(attention_bias=True, mlp_bias=True, head_dim=48)), ("mistral", dict(sliding_window=40)),
            ("starcoder2", dict(sliding_window=64)), ("qwen3", dict(head_dim=64, attention_bias=True)),
            ("stablelm", dict(hidden_size=256, use_parallel_residual=True, use_qkv_bias=True)),
            ("granite", dict(residual_multiplier=0.4, attention_multiplier=0.1)), ("qwen2", dict(sliding_window=8)),
            ("glm4_moe", dict(MOE, use_qk_norm=True)), ("nemotron", dict(hidden_size=256, partial_rotary_factor=0.25)),
            ("llama", dict(rope_parameters=dict(rope_type="yarn", factor=4.0, rope_theta=1e4,
                                                original_max_position_embeddings=16)))]


def check_against_own_forward(model, device):
    """Two requests of different lengths: every step's logits are the
    model's own after the same tokens."""
    decoder = PagedDecoder(model, requests=2, max_length=40)
    texts = [prompt(5, 1).tolist(), prompt(19, 2).tolist()]
    for place, text in enumerate(texts):
        assert decoder.add(text) == place
        assert agree(decoder.logits[0], own_logits(model, text))
    for _ in range(6):
        for place, text in enumerate(texts):
            text.append(int(decoder._last[place]))
        decoder.step()
        for place, text in enumerate(texts):
            assert agree(decoder.logits[place], own_logits(model, text))


def known(kind):
    from transformers import CONFIG_MAPPING
    if kind not in CONFIG_MAPPING:
        pytest.skip(f"this Transformers has no {kind}")


@pytest.mark.parametrize("kind", sorted(paged.MODEL_TYPES))
def test_accepted_models_compute_their_own_forward(kind, device):
    known(kind)
    model = small_model(device, kind, **dict(MOE, head_dim=None if kind == "stablelm" else 32, **KINDS.get(kind, {})))
    check_against_own_forward(model, device)


@pytest.mark.parametrize("kind, settings", FOLLOWED)
def test_settings_that_are_followed(kind, settings, device):
    known(kind)
    check_against_own_forward(small_model(device, kind, **settings), device)


@pytest.mark.parametrize("kind, settings, message", [
    ("mistral", dict(sliding_window=8), "sliding window of 8"), ("mixtral", dict(sliding_window=39), "window of 39"),
    ("starcoder2", dict(sliding_window=8), "sliding window"), ("phimoe", dict(sliding_window=8), "sliding window"),
    ("qwen3", dict(use_sliding_window=True, sliding_window=8, max_window_layers=1), "sliding window"),
    ("granite", dict(embedding_multiplier=12.0), "embedding_multiplier"),
    ("granite", dict(logits_scaling=8.0), "logits_scaling"), ("granitemoe", dict(logits_scaling=8.0), "logits_scaling"),
    ("hyperclovax", dict(embedding_multiplier=2.0), "embedding_multiplier"), ("olmo", dict(clip_qkv=0.5), "clip_qkv"),
    ("stablelm", dict(hidden_size=256, head_dim=None, qk_layernorm=True), "qk_layernorm"),
    ("cohere", {}, "cohere"), ("glm", {}, "glm"), ("glm4", {}, "glm4"), ("ernie4_5", {}, "ernie4_5"),
    ("helium", {}, "helium"), ("smollm3", {}, "smollm3"), ("bitnet", {}, "bitnet"), ("olmo2", {}, "olmo2"),
    ("diffllama", {}, "diffllama"), ("ministral3", {}, "ministral3"), ("hunyuan_v1_dense", {}, "hunyuan"),
    ("llama", dict(rope_parameters=dict(rope_type="dynamic", factor=2.0, rope_theta=1e4)), "do not depend"),
])
def test_models_computed_otherwise_are_refused(kind, settings, message, device):
    """Configurations as Transformers makes them, in models of their own."""
    known(kind)
    model = small_model(device, kind, **dict(dict(MOE, head_dim=32), **settings))
    with pytest.raises(ValueError, match=message):
        PagedDecoder(model, requests=1, max_length=40)


def state(decoder):
    return (decoder.tables.lengths.tolist(), decoder.tables.n_free.tolist(), decoder._live.tolist(),
            list(decoder._taken))


@pytest.mark.parametrize("places", [(0, 0), (0, 2), (2, 0), (0, -3), (0, 3), (0, 1, 0)])
def test_a_refused_finish_changes_nothing(device, places):
    """Places named twice, free ones and ones that do not exist."""
    decoder = PagedDecoder(small_model(device), requests=3, max_length=40)
    decoder.add(prompt(20)), decoder.add(prompt(5))
    before = state(decoder)
    with pytest.raises(ValueError, match="holds no request|named twice"):
        decoder.finish(*places)
    assert state(decoder) == before
    decoder.step()
    decoder.finish(0, 1)
    assert state(decoder) == ([0, 0, 0], [9], [0, 0, 0], [False] * 3)
    decoder.finish()


def only(*tokens):
    """Mask words that allow these tokens."""
    words = [0] * -(-VOCAB // 32)
    for t in tokens:
        words[t // 32] |= 1 << t % 32
    return torch.tensor([w - (1 << 32) if w >> 31 else w for w in words], dtype=torch.int32)


def test_a_place_used_again_has_no_grammar(device):
    """A request's mask ends with it, in a place used again as in a new one;
    a mask given to add() holds for the first answer token and after it."""
    model, text = small_model(device), prompt(9)
    free = int(own_logits(model, text).argmax())
    decoder = PagedDecoder(model, requests=2, max_length=40, grammar=True)
    other = (free + 31) % VOCAB
    place = decoder.add(text, mask=only(other, 7))
    assert int(decoder._last[place]) in (other, 7)
    decoder.masks[place] = only(5).to(device)
    decoder.step()
    assert int(decoder._last[place]) == 5
    decoder.finish(place)
    assert decoder.add(text) == place and int(decoder._last[place]) == free
    assert (decoder.masks == -1).all()
    # written before the place is taken: also for the first token
    decoder.masks[1] = only(other).to(device)
    assert decoder.add(text) == 1 and int(decoder._last[1]) == other
    decoder.finish(0, 1)
    # through generate()
    decoder.masks[0] = only(11).to(device)
    assert decoder.generate([text], 3) == [[11, 11, 11]]
    assert decoder.generate([text], 1) == [[free]]


def test_wrong_masks_are_refused(device):
    decoder = PagedDecoder(small_model(device), requests=1, max_length=40, grammar=True)
    before = state(decoder)
    for bad in (only(1)[:-1], only(1).long(), only(1)[None], [1] * 7):
        with pytest.raises(ValueError, match="mask"):
            decoder.add(prompt(4), mask=bad)
    assert state(decoder) == before
    plain = PagedDecoder(decoder.model, requests=1, max_length=40)
    with pytest.raises(ValueError, match="grammar"):
        plain.add(prompt(4), mask=only(1))


def failing(*args, **kwargs):
    raise ArithmeticError("on purpose")


def test_a_prompt_that_fails_late_leaves_nothing_behind(device, monkeypatch):
    """The first pick fails, after the prompt's keys are stored."""
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=40, repetition=1.2, grammar=True)
    decoder.add(prompt(5))
    before, masks = state(decoder), decoder.masks.clone()
    with monkeypatch.context() as patch:
        patch.setattr(decoder, "_pick", failing)
        with pytest.raises(ArithmeticError):
            decoder.add(prompt(20), mask=only(3))
    assert state(decoder) == before and torch.equal(decoder.masks, masks)
    assert decoder.add(prompt(20)) == 1


@pytest.mark.parametrize("where", ["second prompt", "step", "wrong id"])
def test_a_generate_that_fails_leaves_nothing_behind(device, monkeypatch, where):
    """Its requests end; one that was there before goes on."""
    model = small_model(device)
    decoder = PagedDecoder(model, requests=3, max_length=64, num_pages=6)
    held = decoder.add(prompt(20))
    before = state(decoder)
    texts = [prompt(33), prompt(17) if where == "second prompt" else prompt(3)]
    if where == "wrong id":
        texts[1] = torch.tensor([VOCAB])
    with monkeypatch.context() as patch:
        if where == "step":
            patch.setattr(decoder, "step", failing)
        with pytest.raises(ArithmeticError if where == "step" else ValueError if where == "wrong id" else RuntimeError):
            decoder.generate(texts, 2)
    assert state(decoder) == before
    assert len(decoder.generate([prompt(33)], 2)[0]) == 2 and decoder.tables.lengths[held] == 21


def test_steps_say_which_requests_got_no_token(device):
    """-1 at max_length, without a free page and in free places."""
    decoder = PagedDecoder(small_model(device), requests=4, max_length=24, num_pages=4)
    full, starved, fine = decoder.add(prompt(22, 1)), decoder.add(prompt(16, 2)), decoder.add(prompt(3, 3))
    for got_full in (True, True, False, False):
        tokens = decoder.step().tolist()
        assert (tokens[full] == -1) != got_full and tokens[starved] == -1 and tokens[3] == -1
        assert 0 <= tokens[fine] == int(decoder._last[fine])
    decoder.finish(full)      # its pages let the other go on
    tokens = decoder.step().tolist()
    assert tokens[full] == -1 and 0 <= tokens[starved] == int(decoder._last[starved])


def test_steps_return_tensors_of_their_own(device):
    """What step() returned stays; `tokens` has a prompt's first answer token too."""
    model, text = small_model(device), prompt(6)
    decoder = PagedDecoder(model, requests=2, max_length=40)
    place = decoder.add(text)
    answer = [int(decoder.tokens[place])]
    assert answer[0] == int(own_logits(model, text).argmax())
    kept, seen = [], []
    for _ in range(4):
        kept.append(decoder.step())
        seen.append(kept[-1].tolist())
        assert int(decoder.tokens[place]) == seen[-1][place]
    first = decoder.tokens
    decoder.add(prompt(7))
    decoder.step()
    assert [t.tolist() for t in kept] == seen and first[place] == seen[-1][place]


def captured(decoder, device, monkeypatch):
    """decoder.capture(); on the CPU a graph's stand-in: capturing runs
    nothing, and a replay writes the memory that was there at the capture
    and no attribute."""
    if device != "cpu":
        return decoder.capture()
    run, memory = decoder._run, torch.full((decoder.requests, VOCAB), float("nan"))

    class Graph:
        def replay(self):
            before = decoder.logits
            run()
            memory.copy_(decoder.logits)
            decoder.logits = before
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "CUDAGraph", Graph)
        patch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())
        patch.setattr(decoder, "_run", lambda: setattr(decoder, "logits", memory))
        decoder.capture()


def test_logits_are_the_last_steps_from_a_graph_too(device, monkeypatch):
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=40, repetition=1.3)
    plain = PagedDecoder(model, requests=2, max_length=40, repetition=1.3)
    for d in (decoder, plain):
        d.add(prompt(6)), d.step()
    before = decoder.logits.clone()
    captured(decoder, device, monkeypatch)
    assert torch.equal(decoder.logits, before)     # nothing has run yet
    for i in range(6):
        if i == 2:
            assert decoder.add(prompt(9)) == plain.add(prompt(9)) == 1
            assert decoder.logits.shape == (1, VOCAB)
        assert torch.equal(decoder.step(), plain.step())
        n = 1 if i < 2 else 2
        assert decoder.logits.shape == (2, VOCAB) and agree(decoder.logits[:n], plain.logits[:n])
        assert torch.equal(decoder.tokens, plain.tokens)


@pytest.mark.parametrize("adjusted", ["penalties", "grammar"])
def test_captured_steps_with_penalties_and_grammar(device, monkeypatch, adjusted):
    """Replays give the eager steps' tokens, with requests that come and go
    between them and masks written between them."""
    model = small_model(device)
    how = dict(repetition=1.4, frequency=0.3, presence=0.2) if adjusted == "penalties" else dict(grammar=True)
    decoder, plain = (PagedDecoder(model, requests=3, max_length=30, **how) for _ in range(2))
    for d in (decoder, plain):
        d.add(prompt(6, 1)), d.add(prompt(20, 2)), d.step()
    captured(decoder, device, monkeypatch)
    for i in range(14):
        for d in (decoder, plain):
            if i == 3:
                d.finish(0)
            if i == 5:
                assert d.add(prompt(4, 3)) == 0
            if i in (1, 6) and adjusted == "grammar":
                d.masks[i % 2] = only(*range(i, VOCAB, 7)).to(device)
        got = decoder.step()
        assert torch.equal(got, plain.step()) and torch.equal(decoder.tables.lengths, plain.tables.lengths)
        if adjusted == "grammar" and i >= 6 and got[0] >= 0:
            assert got[0] % 7 == 6


@pytest.mark.parametrize("fails", [False, True])
def test_forwards_of_the_attention_modules_own_are_put_back(device, monkeypatch, fails):
    """A forward that another library set on a module is there again after a
    step, also one that fails, and none is left where there was none."""
    model = small_model(device)
    calls = []
    attention = model.model.layers[1].self_attn
    original = attention.forward

    def wrapped(*args, **kwargs):
        calls.append(1)
        return original(*args, **kwargs)
    attention.forward = wrapped
    decoder = PagedDecoder(model, requests=1, max_length=40)
    decoder.add(prompt(5))
    if fails:
        monkeypatch.setattr(paged.serving, "paged_attention", failing)
        with pytest.raises(ArithmeticError):
            decoder.step()
    else:
        decoder.step()
    assert attention.forward is wrapped
    assert all("forward" not in layer.self_attn.__dict__ for layer in model.model.layers if layer.self_attn is not attention)
    del calls[:]
    own_logits(model, prompt(3))
    assert calls == [1]


def test_no_pages_are_refused(device):
    with pytest.raises(ValueError, match="pages"):
        PagedDecoder(small_model(device), requests=1, max_length=40, num_pages=0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["qwen3", "mixtral"])
def test_compressed_models_answer_as_they_are(kind):
    """Head norms, and experts whose weights are not the runtime's, beside
    Linears that are decoded on the fly: the same tokens, eagerly and, without
    experts, captured."""
    from neuralzip_amd.gpu.inference import NeuralZipRuntime, export_model_for_gpu
    from neuralzip_amd.setup import NeuralZipSetup
    model = small_model("cuda:0", kind, **dict(MOE, head_dim=32, **KINDS.get(kind, {}))).to(torch.bfloat16)
    texts, how = [prompt(3, 1), prompt(25, 2)], dict(requests=2, max_length=60, page_size=32)
    want = PagedDecoder(model, **how).generate(texts, 20)
    setup = NeuralZipSetup(chunk_size=16384).build(model)
    runtime = NeuralZipRuntime.attach(model, export_model_for_gpu(model, setup), device="cuda:0")
    decoder = PagedDecoder(model, **how)
    assert decoder.generate(texts, 20) == want
    if kind == "qwen3":       # (experts' forwards are not captured here)
        assert decoder.generate(texts, 20, capture=True) == want
    del decoder
    assert runtime is not None


@pytest.mark.parametrize("n", [39, 40])
def test_prompts_as_long_as_the_window(device, n):
    """A window of max_length tokens hides nothing, whatever the model's own
    cache keeps."""
    model = small_model(device, "mistral", sliding_window=40)
    decoder = PagedDecoder(model, requests=1, max_length=40)
    text = prompt(n)
    assert decoder.add(text) == 0 and agree(decoder.logits[0], own_logits(model, text))
    if n < 40:
        first = int(decoder.tokens[0])
        decoder.step()
        assert agree(decoder.logits[0], own_logits(model, text.tolist() + [first]))


def test_a_capture_that_fails_keeps_the_logits(device, monkeypatch):
    decoder = PagedDecoder(small_model(device), requests=1, max_length=40)
    decoder.add(prompt(4))
    before = decoder.logits

    def run():
        decoder.logits = None
        failing()
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "CUDAGraph", object)
        patch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())
        patch.setattr(decoder, "_run", run)
        with pytest.raises(ArithmeticError):
            decoder.capture()
    assert decoder.logits is before and decoder._graph is None
    decoder.step()
