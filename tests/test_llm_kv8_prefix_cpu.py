"""The server reuses a cached prefix in whole steps of the engine's ``prefix_step``."""
import pytest


@pytest.fixture(scope="module")
def tiny_model(tmp_path_factory):
    from k8s_nvidia_gpus_amd.models.llm import tiny
    from k8s_nvidia_gpus_amd.models.llm.synthetic import write_synthetic_gguf

    return write_synthetic_gguf(str(tmp_path_factory.mktemp("llm") / "tiny.gguf"), tiny())


@pytest.mark.parametrize("step,cached", [(None, (99, 80)), (1, (99, 80)), (64, (64, 64)), (16, (96, 80)), (128, (0, 0))])
def test_server_cuts_a_reused_prefix_to_whole_steps(tiny_model, step, cached):
    from k8s_nvidia_gpus_amd.models.llm.server import Scheduler, _job_from
    from k8s_nvidia_gpus_amd.models.llm.synthetic import load

    eng, tok = load(tiny_model, device="cpu", max_ctx=256, slots=1)
    if step is not None:
        eng.prefix_step = step
    sched = Scheduler(eng, tok, parallel=1)
    ids = [3 + i % 200 for i in range(100)]

    def ask(ids):
        job = sched.submit(_job_from(dict(temperature=0, ignore_eos=True), ids, 2, eng.cfg.vocab))
        while True:
            kind, val = job.out.get(timeout=60)
            assert kind != "error", val
            if kind == "done":
                return job

    try:
        a = ask(ids)
        b = ask(ids)                                           # all but the last token is cached
        c = ask(ids[:80] + [1, 2])
        assert (a.n_cached, b.n_cached, c.n_cached) == (0, *cached)
        assert a.gen == b.gen
    finally:
        sched.close()


def test_the_step_is_one_token_unless_the_cache_is_in_8_bits(tiny_model):
    from k8s_nvidia_gpus_amd.models.llm.synthetic import load

    assert load(tiny_model, device="cpu", max_ctx=256)[0].prefix_step == 1
