"""Waits inside the paged kernels that run out."""

import pytest
import torch

import megabake_b200.hf as hf
from megabake_b200 import PagedGenerator, models
from megabake_b200.diagnostics import CompilerError

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("operator", ["paged_prefill_attention", "paged_kv_attention"])
def test_generation_tells_when_a_kernel_recorded_a_fault(monkeypatch, operator):
    spec = models.get_spec("tiny-llama")
    weights = {k: v.cuda() for k, v in models.init_weights(spec, 0).items()}
    generator = PagedGenerator(models.build_hf_model(spec, 0, "cuda", weights), 2, 64, page_size=8)
    prompts = [torch.arange(1, 12), torch.arange(5, 9)]
    real, calls = getattr(hf, operator), []

    def recorded(*args, status, **options):
        out = real(*args, status=status, **options)
        calls.append(status.fill_(2))
        return out

    monkeypatch.setattr(hf, operator, recorded)
    with pytest.raises(CompilerError, match="status pipeline-timeout") as info:
        generator(prompts, 2)
    assert info.value.diagnostic.stage == "runtime" and calls
    monkeypatch.undo()
    generator._graph = None        # the step that was captured with the other function
    assert [ids.numel() for ids in generator(prompts, 5)] == [5, 5]
