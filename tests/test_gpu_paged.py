"""PagedDecoder on small random models: the tokens that Transformers' own
greedy generation gives, and its logits, with the weights compressed and not,
eagerly and from a HIP graph."""
import pytest
import torch

from neuralzip_amd.gpu import serving
from neuralzip_amd.gpu.paged import PagedDecoder

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
SHAPES = {
    "LlamaConfig": dict(hidden_size=256, num_attention_heads=8, num_key_value_heads=2),
    "Qwen2Config": dict(hidden_size=448, num_attention_heads=7, num_key_value_heads=1),
}


def small_model(config, dtype=torch.float32):
    import transformers
    torch.manual_seed(7)
    shape = dict(SHAPES[config], intermediate_size=512, num_hidden_layers=3, vocab_size=1000,
                 max_position_embeddings=512, tie_word_embeddings=False)
    model = transformers.AutoModelForCausalLM.from_config(getattr(transformers, config)(**shape))
    with torch.no_grad():
        for name, p in model.named_parameters():
            p.copy_(torch.randn(p.shape) * (0.08 if p.dim() > 1 else 0.1) + (1.0 if "norm" in name else 0.0))
    return model.to(dtype).to(DEVICE).eval()


def prompts(*lengths):
    g = torch.Generator().manual_seed(11)
    return [torch.randint(0, 1000, (n,), generator=g) for n in lengths]


def full_logits(model, prompt, answer):
    """The logits that chose each token of the answer, from one forward."""
    ids = torch.cat([prompt, torch.tensor(answer[:-1], dtype=torch.int64)])[None].to(DEVICE)
    with torch.no_grad():
        return model(ids).logits[0, len(prompt) - 1:].double()


def near(chosen, logits):
    """Whether each chosen token's logit is within `bound` of the best one:
    float32 sums of three layers of at most 512 terms each differ between
    two orders by far less than 1e-3 of the largest logit."""
    bound = 1e-3 * logits.abs().amax()
    return bool((logits.amax(-1) - logits[torch.arange(len(chosen)), torch.tensor(chosen)] <= bound).all())


@pytest.mark.parametrize("config", SHAPES)
@pytest.mark.parametrize("capture", [False, True])
def test_answers_are_the_models_own(config, capture):
    """Five prompts of different lengths together: every token is the
    model's own choice given the ones before."""
    model = small_model(config)
    decoder = PagedDecoder(model, requests=6, max_length=120)
    texts = prompts(1, 15, 16, 17, 70)
    answers = decoder.generate(texts, 40, capture=capture)
    for text, answer in zip(texts, answers):
        assert len(answer) == 40 and near(answer, full_logits(model, text, answer))
    assert decoder.tables.n_free.item() == decoder.tables.num_pages
    # the same places again, after others have been through them
    again = decoder.generate(texts[::-1], 12, capture=capture)
    assert [a[:12] for a in answers] == again[::-1]


class HeadNorm(torch.nn.Module):
    """x / rms(x) * weight over a head."""

    def __init__(self, dim, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.weight = torch.nn.Parameter(1 + 0.3 * torch.randn(dim, generator=g))
        self.variance_epsilon = 1e-5

    def forward(self, x):
        heads = x.view(*x.shape[:-1], -1, self.weight.shape[0])
        scale = (heads.square().mean(-1, keepdim=True) + self.variance_epsilon).rsqrt()
        return (heads * scale * self.weight).view(x.shape)


def test_norms_of_queries_and_keys():
    """q_norm and k_norm of the attention modules: the same as norms right
    after the projections, which the model's own forward then has."""
    model, plain = small_model("LlamaConfig"), small_model("LlamaConfig")
    for i, (a, b) in enumerate(zip(model.model.layers, plain.model.layers)):
        for name, seed in (("q", 2 * i), ("k", 2 * i + 1)):
            norm = HeadNorm(a.self_attn.head_dim, seed).to(DEVICE)
            setattr(a.self_attn, name + "_norm", norm)
            setattr(b.self_attn, name + "_proj",
                    torch.nn.Sequential(getattr(b.self_attn, name + "_proj"), norm))
    text = prompts(1)[0]     # a single token: the prompt's own forward has no norms of this kind
    decoder = PagedDecoder(model, requests=1, max_length=40)
    place = decoder.add(text)
    answer = [int(decoder._last[place])]
    decoder.tables.lengths.zero_()       # run the prompt's token through the pages instead
    decoder._last[place] = int(text[0])
    answer = [int(decoder.step()[place]) for _ in range(30)]
    assert near(answer, full_logits(plain, text, answer))


def test_compressed_weights_give_the_same_tokens():
    """bfloat16 weights decoded on the fly by the runtime: the same tokens,
    as the decode is bit-exact; eagerly and from a graph."""
    from neuralzip_amd.gpu.inference import NeuralZipRuntime, export_model_for_gpu
    from neuralzip_amd.setup import NeuralZipSetup
    model = small_model("LlamaConfig", torch.bfloat16)
    texts = prompts(3, 40, 21)
    want = PagedDecoder(model, requests=3, max_length=80).generate(texts, 25)
    setup = NeuralZipSetup(chunk_size=16384).build(model)
    runtime = NeuralZipRuntime.attach(model, export_model_for_gpu(model, setup), device=DEVICE)
    decoder = PagedDecoder(model, requests=3, max_length=80)
    assert decoder.generate(texts, 25) == want
    assert decoder.generate(texts, 25, capture=True) == want
    del decoder
    assert runtime is not None


def test_requests_come_and_go():
    """Requests of different ages in one step, places and pages reused."""
    model = small_model("LlamaConfig")
    decoder = PagedDecoder(model, requests=2, max_length=64, num_pages=6)
    a, b, c = prompts(20, 30, 5)
    got = {}
    first = decoder.add(a)
    got["a"] = [int(decoder._last[first])]
    for _ in range(5):
        got["a"].append(int(decoder.step()[first]))
    second = decoder.add(b)
    got["b"] = [int(decoder._last[second])]
    with pytest.raises(RuntimeError, match="places"):
        decoder.add(c)
    for _ in range(4):
        tokens = decoder.step().tolist()
        got["a"].append(tokens[first]), got["b"].append(tokens[second])
    decoder.finish(first)
    third = decoder.add(c)
    got["c"] = [int(decoder._last[third])]
    for _ in range(6):
        tokens = decoder.step().tolist()
        got["b"].append(tokens[second]), got["c"].append(tokens[third])
    for text, name in ((a, "a"), (b, "b"), (c, "c")):
        assert near(got[name], full_logits(model, text, got[name])), name
    decoder.finish(second, third)
    assert decoder.tables.n_free.item() == 6
    with pytest.raises(RuntimeError, match="pages"):
        PagedDecoder(model, requests=2, max_length=64, num_pages=1).add(prompts(17)[0])
    tight = PagedDecoder(model, requests=2, max_length=64, num_pages=3)
    with pytest.raises(RuntimeError, match="ran out"):
        tight.generate(prompts(16, 16), 20)
    assert tight.tables.n_free.item() == 3 and not any(tight._taken)
    with pytest.raises(RuntimeError, match="more prompts"):
        tight.generate(prompts(1, 1, 1), 2)
    for ids in ([], [3, 1000], [-1], 5, [[1, 2]]):
        with pytest.raises(ValueError, match="token ids"):
            tight.add(ids)
    model.lm_head, head = None, model.lm_head     # a forward that fails
    with pytest.raises(TypeError):
        tight.add(prompts(20)[0])
    model.lm_head = head
    assert tight.tables.n_free.item() == 3 and tight.tables.lengths.tolist() == [0, 0]
    assert len(tight.generate(prompts(20), 5)[0]) == 5
    with pytest.raises(ValueError, match="holds no request"):
        decoder.finish(0)
    with pytest.raises(ValueError, match="token ids"):
        decoder.add(prompts(65)[0])


def test_penalties_and_grammar_masks_choose_the_tokens():
    """Each token is the best one under the penalties and the masks."""
    model = small_model("LlamaConfig")
    text = prompts(12)[0]
    decoder = PagedDecoder(model, requests=2, max_length=64, repetition=1.4, frequency=0.3, presence=0.2, grammar=True)
    allowed = torch.arange(1000) % 3 == 0
    bits = torch.zeros(1024, dtype=torch.int64)
    bits[:1000] = allowed
    words = (bits.view(32, 32) << torch.arange(32)).sum(1)
    decoder.masks[0] = torch.where(words >= 1 << 31, words - (1 << 32), words).int().to(DEVICE)
    answer = decoder.generate([text], 20)[0]
    assert all(t % 3 == 0 for t in answer)
    logits = full_logits(model, text, answer).cpu()
    for i, token in enumerate(answer):
        x, seen = logits[i].clone(), text.tolist() + answer[:i]
        for t in set(seen):
            x[t] = x[t] / 1.4 if x[t] > 0 else x[t] * 1.4
        for t in set(answer[:i]):
            x[t] -= 0.3 * answer[:i].count(t) + 0.2
        x[~allowed] = -float("inf")
        assert x.max() - x[token] <= 1e-3 * logits.abs().amax()


def test_models_that_do_not_fit_are_refused():
    model = small_model("LlamaConfig")
    model.model.layers[1].self_attn.sliding_window = 128
    with pytest.raises(ValueError, match="sliding window"):
        PagedDecoder(model, requests=1, max_length=32)
    del model.model.layers[1].self_attn.sliding_window, model.model.layers[0].self_attn.o_proj
    with pytest.raises(ValueError, match="o_proj"):
        PagedDecoder(model, requests=1, max_length=32)
    assert serving.PAGES_OK == 0
