"""Waits inside the paged kernels that run out."""

import ctypes

import pytest
import torch

import megabake_b200.hf as hf
from megabake_b200 import PagedGenerator, PagedState, models, paged_kv_attention, paged_prefill_attention
from megabake_b200 import runtime as rt
from megabake_b200.diagnostics import CompilerError
from tests.test_gpu_paged import BF16, FP16, Cache, _int32, _normal

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


def _native(prefill, query, cache, index, status, limit):
    """The C entry, with a limit for its waits."""
    out = torch.zeros_like(query)
    kv_heads, pools = cache.pools[0].shape[2], cache.pools
    args = rt.PagedAttentionArgs(
        0 if query.dtype == BF16 else 1, query.shape[0], cache.table.shape[0], query.shape[1], kv_heads, query.shape[2],
        cache.table.shape[1], pools[0].shape[0], cache.page, 0, query.shape[2] ** -0.5, limit, *query.stride()[:2], 0, 0, 0, 0,
        *pools[0].stride()[:3], *pools[1].stride()[:3], query.data_ptr(), 0, 0, pools[0].data_ptr(), pools[1].data_ptr(),
        cache.table.data_ptr(), cache.lengths.data_ptr(), index.data_ptr(), out.data_ptr(), 0, status.data_ptr())
    name = "mb_paged_prefill" if prefill else "mb_paged_attention"
    size = getattr(rt.load_library(), name + "_workspace")(ctypes.byref(args))
    workspace = torch.zeros(size + 1, dtype=torch.uint8, device="cuda")
    args.workspace = workspace.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    assert getattr(rt.load_library(), name)(ctypes.byref(args), stream) == 0
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("width", [8, 400])
@pytest.mark.parametrize("heads,dtype", [((4, 2, 64), BF16), ((34, 2, 128), FP16), ((8, 1, 256), BF16)])
@pytest.mark.parametrize("prefill", [False, True])
def test_a_wait_that_runs_out_ends_the_launch(prefill, heads, dtype, width):
    """A nanosecond is less than keys take to come.  The launch ends, says so, and leaves the device usable."""
    count, kv_heads, dim = heads
    lengths = [min(n, 16 * width) for n in (100, 70, 5000)]
    cache = Cache(lengths, kv_heads, dim, 16, dtype, width)
    cache.table = torch.nn.functional.pad(cache.table[:, :width], (0, max(0, width - cache.table.shape[1])), value=-1).contiguous()
    query = _normal((3 if not prefill else 60, count, dim), cache.g, dtype)
    index = _int32([0, 1, 2]) if not prefill else _int32([0, 20, 21, 60])
    good, status = _int32([0]), _int32([0])
    expected = _native(prefill, query, cache, index, good, 0)
    for _ in range(2):
        _native(prefill, query, cache, index, status, 1)
        assert status.item() == 2          # MB_ST_PIPE_TIMEOUT
        status.zero_()
    assert torch.equal(_native(prefill, query, cache, index, good, 0), expected) and good.item() == 0
    same = (paged_prefill_attention(query, *cache.pools, cache.table, cache.lengths, index) if prefill else
            paged_kv_attention(query, None, None, *cache.pools, cache.table, cache.lengths, index))
    assert torch.equal(same, expected)


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


def test_a_fault_of_another_stream_is_seen():
    state = PagedState(1, 1, 16, 1, 64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)      # cycles: about ten milliseconds of a step
        state.status.fill_(2)
    with pytest.raises(CompilerError, match="pipeline-timeout"):
        state.check()
    state.check()
