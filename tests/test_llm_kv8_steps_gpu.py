"""Decode steps of the LLM engine on its 8-bit KV cache: refusals and buffers."""
import pytest
import torch

from test_llm_kv8_engine_gpu import dev, engine, prompt, tiny_gguf   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["decode", "decode_greedy", "decode_greedy_async"])
def test_a_refused_step_leaves_the_steps_buffers_alone(dev, tiny_gguf, call):   # noqa: F811
    eng = engine(tiny_gguf, dev, kv_type="int8")
    eng.prefill(prompt(20, 1), 0)
    eng.prefill(prompt(30, 2), 1)
    eng.decode([3, 4], [20, 30], [0, 1])
    torch.cuda.synchronize()
    b = eng._bufs[2]
    before = b.host.clone(), b.meta.clone(), b.runs.clone()
    with pytest.raises(ValueError, match="consecutive"):
        getattr(eng, call)([5, 6], [21, 21], [0, 0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((b.host, b.meta, b.runs), before))


def test_a_step_holds_no_partials_of_the_other_cache(dev, tiny_gguf):   # noqa: F811
    """The 8-bit cache's attention takes its scratch from the allocator: nothing of the size of the context."""
    for kind in ("f16", "int8"):
        eng = engine(tiny_gguf, dev, kv_type=kind, max_ctx=4096)
        eng.decode([3], [5], [0])
        b = eng._bufs[1]
        size = sum(t.numel() * t.element_size() for t in vars(b).values() if isinstance(t, torch.Tensor) and t.is_cuda)
        partials = eng.cfg.heads * (eng.max_ctx // eng.LK.attn_chunk()) * (eng.cfg.head_dim + 2) * 4
        assert (b.po is not None) == (b.pml is not None) == (b.qrot is not None) == (kind == "f16")
        if kind == "f16":
            with_partials = size
        else:
            assert size <= with_partials - partials + 2 * eng.kv_pages.shape[1] * 4 + 4 * eng.cfg.dim + 256
