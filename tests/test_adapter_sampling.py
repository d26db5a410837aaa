"""ModelAdapterHF.process_tokens with `sampling`: the default stays greedy, drawn tokens are sample_tokens' own."""
import pytest
import torch

transformers = pytest.importorskip("transformers")


def _tiny_llama(seed=0):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=96, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=32, max_position_embeddings=1024)
    return LlamaForCausalLM(cfg).eval()


def _tokens(device):
    g = torch.Generator().manual_seed(1)
    context = torch.randint(0, 96, (1, 40), generator=g).to(device)
    return context, [torch.randint(0, 96, (1, n), generator=g).to(device) for n in (6, 3)]


def _adapter(model):
    from sparse_attention_hub_amd.adapters import ModelAdapterHF
    from sparse_attention_hub_amd.sparse_attention import LocalMaskerConfig, ResearchAttentionConfig, SinkMaskerConfig

    return ModelAdapterHF(model, ResearchAttentionConfig(masker_configs=[SinkMaskerConfig(sink_size=4), LocalMaskerConfig(window_size=8)]))


def test_an_unknown_setting_is_refused_before_anything_runs():
    from sparse_attention_hub_amd.adapters import ModelAdapterHF

    context, questions = _tokens("cpu")
    with pytest.raises(ValueError, match="beams"):
        ModelAdapterHF(torch.nn.Linear(1, 1), None).process_tokens(context, questions, 2, sampling=dict(beams=3))


def test_settings_reach_sample_tokens_with_one_number_per_token(monkeypatch):
    from sparse_attention_hub_amd.adapters import ModelAdapterHF, huggingface

    calls = []

    def stand_in(logits, uniforms, **settings):
        calls.append((logits.shape, uniforms.clone(), settings))
        return torch.tensor([len(calls) % 96 if len(calls) != 2 else -1]), torch.zeros(1)

    monkeypatch.setattr(huggingface, "sample_tokens", stand_in)
    context, questions = _tokens("cpu")
    adapter = ModelAdapterHF(_tiny_llama(), None)
    settings = dict(temperature=0.7, top_p=0.9)
    got = adapter.process_tokens(context, questions[:1], 4, sampling=settings, generator=torch.Generator().manual_seed(5))
    assert got[0].tolist() == [1, 0, 3, 4]  # -1, a row without a token, is the first one
    want = torch.Generator().manual_seed(5)
    for shape, uniforms, given in calls:
        assert shape == (1, 96) and given == settings and torch.equal(uniforms, torch.rand(1, generator=want))
    # without it nothing is drawn
    adapter.process_tokens(context, questions[:1], 3)
    assert len(calls) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0)])
def test_settings_that_leave_one_token_answer_greedily(cuda, settings):
    context, questions = _tokens(cuda)
    adapter = _adapter(_tiny_llama().to(cuda))
    try:
        greedy = adapter.process_tokens(context, questions, 6)
        drawn = adapter.process_tokens(context, questions, 6, sampling=settings)
    finally:
        adapter._cleanup_attention_registration()
    assert [a.tolist() for a in greedy] == [a.tolist() for a in drawn]


@pytest.mark.gpu
def test_drawn_answers_follow_the_generator(cuda):
    from sparse_attention_hub_amd.sparse_attention.utils.token_sampling import sample_tokens

    context, questions = _tokens(cuda)
    adapter = _adapter(_tiny_llama().to(cuda))
    seen = []
    hook = adapter.model.register_forward_hook(lambda module, args, out: seen.append(out.logits[0, -1].clone()))
    settings = dict(temperature=3.0, top_k=40, top_p=0.95, min_p=0.01)
    try:
        runs = []
        for seed in (3, 3, 4):
            seen.clear()
            answer = adapter.process_tokens(context, questions[:1], 8, sampling=settings, generator=torch.Generator(device=cuda).manual_seed(seed))[0]
            numbers = torch.Generator(device=cuda).manual_seed(seed)
            # (the first forward is the context's)
            want = [int(sample_tokens(x[None], torch.rand(1, device=cuda, generator=numbers), **settings)[0]) for x in seen[1:]]
            assert answer.tolist() == want
            runs.append(want)
    finally:
        hook.remove()
        adapter._cleanup_attention_registration()
    assert runs[0] == runs[1] != runs[2]
