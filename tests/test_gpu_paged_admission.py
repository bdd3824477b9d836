"""How prompts are admitted to a paged cache."""

import pytest
import torch

from megabake_b200 import PagedGenerator, models

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("limit,passes", [(8192, [48]), (30, [22, 26]), (1, [5, 17, 20, 6])])
def test_prompts_of_one_pass_are_bounded(limit, passes):
    """The prompts of a pass have ``prompt_tokens`` tokens together, or are one; the ids stay what they are."""
    spec = models.get_spec("tiny-llama")
    weights = {k: v.cuda() for k, v in models.init_weights(spec, 0).items()}
    model = models.build_hf_model(spec, 0, "cuda", weights)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, spec.vocab, (n,), generator=g) for n in (5, 17, 20, 6)]
    alone = PagedGenerator(model, 1, 64, page_size=8)
    generator = PagedGenerator(model, 4, 64, page_size=8, prompt_tokens=limit)
    forward, seen = generator.decoder.forward, []

    def counted(ids, *args, **options):
        if not options.get("one_token"):
            seen.append(ids.numel())
        return forward(ids, *args, **options)

    generator.decoder.forward = counted
    out = generator(prompts, [3, 4, 1, 5])
    assert seen == passes
    assert [ids.numel() for ids in out] == [3, 4, 1, 5]
    # the first pick of a prompt, in whatever company
    for prompt, ids in zip(prompts, out):
        assert ids[0] == alone([prompt], 1)[0][0]
