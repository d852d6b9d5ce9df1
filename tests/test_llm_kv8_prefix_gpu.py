"""Prompt caching over the 8-bit KV cache: what a slot's page held behind the reused prefix (a dropped tail, a
step that ran past a sequence's end) leaves no trace in a later request."""
import pytest
import torch

from test_llm_kv8_engine_gpu import BOUND, cosine, dev, prompt, tiny_gguf   # noqa: F401

pytestmark = pytest.mark.gpu


def ask(sched, tok_ids, n=1):
    """One greedy request through the scheduler -> its job."""
    from k8s_nvidia_gpus_amd.models.llm.server import _job_from

    job = sched.submit(_job_from(dict(temperature=0, ignore_eos=True), tok_ids, n, sched.engine.cfg.vocab))
    while True:
        kind, val = job.out.get(timeout=60)
        assert kind != "error", val
        if kind == "done":
            return job


@pytest.mark.parametrize("kind", BOUND)
@pytest.mark.parametrize("keep", [70, 100, 127, 128, 129])
@pytest.mark.parametrize("dead", [float("nan"), 3000.0, 1.0])
def test_a_reused_prefix_does_not_keep_what_a_dropped_tail_left(dev, tiny_gguf, kind, keep, dead):   # noqa: F811
    from k8s_nvidia_gpus_amd.models.llm.server import Scheduler
    from k8s_nvidia_gpus_amd.models.llm.synthetic import load

    def serving():
        eng, tok = load(tiny_gguf, device=dev, max_ctx=512, slots=1, dense=True, kv_type=kind)
        return eng, Scheduler(eng, tok, parallel=1)

    eng, sched = serving()
    fresh, other = serving()
    try:
        first = prompt(130, 60)
        ask(sched, first)
        # the pages behind position `keep` got larger values (or a non-finite one) before the cut
        x = torch.full((1, eng.cfg.kv_heads, eng.cfg.head_dim), dead, device=dev)
        at = eng._kv8_runs([(0, keep, 1)])
        for layer in eng.kv8:
            eng.KV.kv8_append(layer, x, x, *at)
        second = first[:keep] + [(t + 1) % 512 for t in first[keep:keep + 1]] + prompt(20, 61)
        seen = []
        real = eng.prefill
        eng.prefill = lambda ids, slot, start=0: seen.append((start, real(ids, slot, start))) or seen[-1][1]
        job = ask(sched, second)
        assert 0 < job.n_cached <= keep and seen[0][0] == job.n_cached
        want = fresh.prefill(second, 0)
        assert torch.isfinite(seen[-1][1]).all() and cosine(seen[-1][1], want) > 0.9999
        for layer in range(len(eng.kv8)):                      # and the cache holds what a fresh one holds
            for a, b in zip(eng._kv_load(layer, 0, len(second)), fresh._kv_load(layer, 0, len(second))):
                assert cosine(a, b) > 0.9999
    finally:
        sched.close()
        other.close()
