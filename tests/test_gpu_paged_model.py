"""A model over a paged cache against the oracle, and generation of prompts of any lengths."""

import pytest
import torch

from megabake_b200 import PagedDecoder, PagedGenerator, models
from oracle import decoder_oracle as oracle
from oracle.adapters import oracle_config, oracle_weights
from tests.helpers import LOGIT_COSINE, cosine, greedy_pick_matches, logits_close

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

MODELS = ["tiny-llama", "tiny-llama3", "tiny-qwen2", "tiny-mha", "tiny-gemma", "tiny-gemma256"]


def _model(name):
    spec = models.get_spec(name)
    weights = models.init_weights(spec, 0)
    inv_freq = models.inv_freq_buffer(spec)
    model = models.build_hf_model(spec, 0, "cuda", {k: v.cuda() for k, v in weights.items()})
    return spec, model, oracle_config(spec), oracle_weights(weights, inv_freq)


def _check(logits, expected):
    ok, worst = logits_close(logits, expected)
    assert ok, worst
    assert cosine(logits, expected) > LOGIT_COSINE


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name", MODELS)
def test_prompts_chunks_and_steps_match_the_oracle(name):
    """Two requests of their own lengths: a whole prompt, one in two chunks, then single tokens for both; the logits of
    every position against the oracle's prefill of the whole sequence."""
    spec, model, cfg, weights = _model(name)
    decoder = PagedDecoder(model).eval()
    state = decoder.make_paged_state(3, 64, page_size=8, pages=12)
    g = torch.Generator().manual_seed(3)
    lengths = [19, 23]
    ids = [torch.randint(0, spec.vocab, (1, n), generator=g) for n in lengths]
    expected = [oracle.prefill(cfg, weights, x)[0] for x in ids]
    seen = [0, 0, 0]

    def step(counts, places, one_token=False):
        batch = state.reserve(_int32(counts), places)
        assert batch.granted.tolist() == counts
        packed = torch.cat([ids[r][0, seen[r]:seen[r] + counts[r]] for r in range(2)])
        packed = torch.cat([packed, packed.new_zeros(places - packed.numel())])
        logits = decoder(packed.cuda(), batch, state, one_token=one_token)
        at = 0
        for r in range(2):
            if counts[r]:
                _check(logits[at:at + counts[r]], expected[r][seen[r]:seen[r] + counts[r]])
            at += counts[r]
            seen[r] += counts[r]

    step([9, 13, 0], 22)
    step([1, 6, 0], 10)           # one decodes while the other's prompt goes on
    for _ in range(4):
        step([1, 1, 0], 3, one_token=True)
    step([1, 0, 0], 3, one_token=True)
    step([4, 0, 0], 4)
    assert state.lengths.tolist() == [19, 23, 0]


@pytest.mark.parametrize("name", ["tiny-llama", "tiny-qwen2"])
@pytest.mark.parametrize("pages", [None, 9])
def test_generation(name, pages):
    """Seven prompts over three rows: every id is the oracle's pick after what came before it."""
    spec, model, cfg, weights = _model(name)
    generator = PagedGenerator(model, 3, 64, page_size=8, pages=pages)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, spec.vocab, (n,), generator=g) for n in (5, 17, 1, 30, 8, 9, 16)]
    wanted = [6, 1, 9, 4, 12, 2, 7]
    out = generator(prompts, wanted)
    again = generator(prompts, wanted)
    for prompt, count, ids, repeated in zip(prompts, wanted, out, again):
        assert ids.shape == (count,) and torch.equal(ids, repeated)
        whole = torch.cat([prompt, ids.cpu()])[None]
        logits = oracle.prefill(cfg, weights, whole[:, :-1])[0, prompt.numel() - 1:]
        picks = torch.full_like(logits, -torch.inf).scatter_(1, ids.cpu()[:, None], 1.0)
        ok, _ = greedy_pick_matches(picks, logits)
        assert ok
    state = generator.state
    assert state.free_count.item() == generator.pages and state.block_table.eq(-1).all()
    assert sorted(state.free_pages.tolist()) == list(range(generator.pages))


def test_generation_refuses_what_does_not_fit():
    _, model, _, _ = _model("tiny-llama")
    generator = PagedGenerator(model, 2, 32, page_size=8, pages=3)
    for prompts, wanted in (([torch.zeros(0, dtype=torch.int64)], 1), ([torch.zeros(3, dtype=torch.int64)], 0),
                            ([torch.zeros(20, dtype=torch.int64)], 6), ([torch.zeros(3, dtype=torch.int64)], [1, 2])):
        with pytest.raises(ValueError):
            generator(prompts, wanted)
    assert generator([], 3) == []
    with pytest.raises(ValueError):
        generator.decoder(torch.zeros(3, dtype=torch.int64, device="cuda"), generator.state.reserve(_int32([1, 1]), 2),
                          generator.state)


def test_compiled_prefill_hands_over_to_pages():
    """A prompt through the compiled prefill, whose contiguous caches are appended to the pages, then single tokens."""
    from megabake_b200 import StatefulPrefill, make_backend, paged_append

    spec, model, cfg, weights = _model("tiny-llama")
    tokens, total = 24, 30
    ids = torch.randint(0, spec.vocab, (1, total), generator=torch.Generator().manual_seed(7))
    expected = oracle.prefill(cfg, weights, ids)[0]
    prefill = StatefulPrefill(model, 32).eval()
    contiguous = prefill.make_state(1, device="cuda")
    compiled = torch.compile(prefill, backend=make_backend(mode="prefill"), fullgraph=True, dynamic=False)
    with torch.no_grad():
        _check(compiled(ids[:, :tokens].cuda(), *contiguous)[0], expected[:tokens])
    decoder = PagedDecoder(model).eval()
    state = decoder.make_paged_state(2, 64, page_size=16)
    batch = state.reserve(_int32([0, tokens]), tokens)
    for layer in range(spec.layers):
        keys, values = (c[0, :tokens] for c in contiguous[3 * layer:3 * layer + 2])
        paged_append(keys, values, state.key_pages[layer], state.value_pages[layer], batch.slots)
    for position in range(tokens, total):
        batch = state.reserve(_int32([0, 1]), 1)
        logits = decoder(ids[0, position:position + 1].cuda(), batch, state, one_token=True)
        _check(logits, expected[position:position + 1])
