"""Which Hugging Face models ``PagedDecoder`` computes: the ones it takes against their own forward, with plain stand-ins
for the operators on the CPU, and the ones it refuses."""

import pytest
import torch

import megabake_b200.hf as hf
from megabake_b200 import PagedBatch, PagedDecoder, paged
from megabake_b200.diagnostics import CompilerError
from tests import paged_reference as reference

transformers = pytest.importorskip("transformers")

PAGE, TOKENS = 8, 20
SIZES = dict(vocab_size=97, hidden_size=128, intermediate_size=160, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, max_position_embeddings=256, pad_token_id=0, bos_token_id=1, eos_token_id=2)
GRANITE = dict(embedding_multiplier=1.0, residual_multiplier=1.0, logits_scaling=1.0, attention_multiplier=0.1)


def _model(kind, **changes):
    config = transformers.AutoConfig.for_model(kind, **{**SIZES, **changes})
    g = torch.Generator().manual_seed(0)
    model = transformers.AutoModelForCausalLM.from_config(config, attn_implementation="eager").eval().float()
    with torch.no_grad():
        for parameter in model.parameters():
            parameter.add_(0.15 * torch.randn(parameter.shape, generator=g))
    return model


@pytest.fixture
def plain_operators(monkeypatch):
    def append(key, value, key_pages, value_pages, slots):
        key_pages[slots // PAGE, slots % PAGE], value_pages[slots // PAGE, slots % PAGE] = key, value

    def attend(query, key_pages, value_pages, table, lengths, offsets, *, scale, **_):
        new, cached = int(offsets[1]), int(lengths[0] - offsets[1])
        return torch.stack([reference.attend(query[t], key_pages, value_pages, table[0], cached + t + 1, scale)[0].float()
                            for t in range(new)])

    monkeypatch.setitem(paged._ELEMENTS, torch.float32, 2)
    monkeypatch.setattr(hf, "paged_append", append)
    monkeypatch.setattr(hf, "paged_prefill_attention", attend)


@pytest.mark.parametrize("kind,changes", [
    ("llama", {}), ("qwen2", {}), ("gemma", {}), ("mistral", dict(sliding_window=None)), ("mistral", dict(sliding_window=32)),
    ("granite", GRANITE), ("olmo", {}), ("llama", dict(rope_parameters=dict(
        rope_type="llama3", rope_theta=1e4, factor=2.0, low_freq_factor=1.0, high_freq_factor=4.0,
        original_max_position_embeddings=64)))])
def test_models_that_are_computed(plain_operators, kind, changes):
    """In 32 bits on both sides: some ten sums of up to 160 terms in a row, each off by 160 * 2^-24 at most, are 1e-4; what a
    part that is left out is worth is a thousand times that."""
    model = _model(kind, **changes)
    decoder = PagedDecoder(model).eval()
    state = decoder.make_paged_state(1, 32, page_size=PAGE, device="cpu")
    state.block_table[0] = torch.tensor([2, 0, 3, 1])
    state.lengths[0] = TOKENS
    places = torch.arange(TOKENS)
    slots = state.block_table[0, places // PAGE].long() * PAGE + places % PAGE
    batch = PagedBatch(torch.tensor([0, TOKENS], dtype=torch.int32), slots, places,
                       torch.zeros(TOKENS, dtype=torch.int32), torch.tensor([TOKENS], dtype=torch.int32))
    ids = torch.randint(3, 97, (TOKENS,), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        expected = model(input_ids=ids[None], use_cache=False).logits[0]
    assert float((decoder(ids, batch, state) - expected).norm() / expected.norm()) < 1e-4


@pytest.mark.parametrize("kind,changes,match", [
    ("qwen3", {}, "q_norm"), ("glm4", {}, "post_self_attn_layernorm"), ("cohere", {}, "post_attention_layernorm"),
    ("phi3", {}, "resid_attn_dropout"), ("olmo2", {}, "input_layernorm"), ("diffllama", {}, "lambda_q1"),
    ("smollm3", dict(num_hidden_layers=4), "rotates"), ("olmo", dict(clip_qkv=0.1), "clip_qkv"),
    ("granite", {**GRANITE, "embedding_multiplier": 3.0}, "embedding_multiplier"),
    ("granite", {**GRANITE, "residual_multiplier": 0.5}, "residual_multiplier"),
    ("granite", {**GRANITE, "logits_scaling": 4.0}, "logits_scaling"),
    ("llama", dict(rope_parameters=dict(rope_type="dynamic", rope_theta=1e4, factor=2.0)), "dynamic"),
])
def test_models_that_are_refused(kind, changes, match):
    with pytest.raises(NotImplementedError, match=match):
        PagedDecoder(_model(kind, **changes))


def test_soft_caps_are_refused():
    model = _model("llama")
    for name in ("attn_logit_softcapping", "final_logit_softcapping"):
        setattr(model.config, name, 30.0)
        with pytest.raises(NotImplementedError, match=name):
            PagedDecoder(model)
        setattr(model.config, name, None)
    PagedDecoder(model)


def test_rotary_positions_are_looked_at_in_every_kind_of_layer():
    model = _model("llama")
    for rope, match in (({"rope_type": "longrope"}, "longrope"), ({"llama_4_scaling_beta": 0.1}, "scaled by position")):
        model.config.rope_parameters = {"full_attention": {"rope_type": "default", **rope}}
        with pytest.raises(NotImplementedError, match=match):
            PagedDecoder(model)


@pytest.mark.parametrize("kind", ["mistral", "starcoder2", "mixtral"])
def test_a_window_shorter_than_the_capacity_is_refused(plain_operators, kind):
    """Rows hold whole pages, and requests may grow to all of them."""
    changes = dict(num_local_experts=2) if kind == "mixtral" else {}
    decoder = PagedDecoder(_model(kind, sliding_window=30, **changes))
    with pytest.raises(NotImplementedError, match="30-token"):
        decoder.make_paged_state(1, 30, page_size=PAGE, device="cpu")
    decoder.make_paged_state(1, 24, page_size=PAGE, device="cpu")
    state = paged.PagedState(2, 1, 32, 2, 64, page_size=PAGE, dtype=torch.float32, device="cpu")
    ids = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="30-token"):
        decoder(ids, PagedBatch(None, ids, ids, None, None), state)


@pytest.mark.parametrize("one_token", [False, True])
def test_the_state_has_the_status_word_of_every_layer(plain_operators, monkeypatch, one_token):
    given = []

    def attend(query, *_, status, **__):
        given.append(status)
        return torch.zeros_like(query)

    monkeypatch.setattr(hf, "paged_kv_attention", attend)
    monkeypatch.setattr(hf, "paged_prefill_attention", attend)
    decoder = PagedDecoder(_model("llama")).eval()
    state = decoder.make_paged_state(1, 32, page_size=PAGE, device="cpu")
    place = torch.zeros(1, dtype=torch.int64)
    batch = PagedBatch(torch.tensor([0, 1], dtype=torch.int32), place, place, place.int(), place.int())
    decoder(place, batch, state, one_token=one_token)
    assert len(given) == 2 and all(status is state.status for status in given)


def test_a_recorded_fault_is_raised_once():
    state = paged.PagedState(1, 1, 32, 2, 64, page_size=PAGE, device="cpu")
    state.check()
    state.status.fill_(2)   # what a kernel writes when a wait ran out
    with pytest.raises(CompilerError, match="status pipeline-timeout") as info:
        state.check()
    assert info.value.diagnostic.stage == "runtime"
    state.check()
    state.status.fill_(2)
    state.reset()
    state.check()
