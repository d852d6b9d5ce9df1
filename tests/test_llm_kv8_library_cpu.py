"""The 8-bit cache's entry points and the kernel library agree on the page size, or no call is made; an
engine that cannot keep the cache in 8 bits says so."""
import warnings

import pytest

from k8s_nvidia_gpus_amd.ops import llm_kv8 as KV


def test_the_library_has_the_page_size_of_the_entry_points():
    assert KV._lib().amdk8s_llm_kv8_page() == KV.PAGE


def test_another_page_size_is_refused(monkeypatch):
    monkeypatch.setattr(KV, "_entries", None)
    monkeypatch.setattr(KV, "PAGE", 32)
    with pytest.raises(RuntimeError, match="64 positions"):
        KV._lib()
    assert KV._entries is None


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_an_engine_without_a_gpu_says_that_its_cache_is_not_rounded(tmp_path, kind):
    from k8s_nvidia_gpus_amd.models.llm import tiny
    from k8s_nvidia_gpus_amd.models.llm.synthetic import load, write_synthetic_gguf

    path = write_synthetic_gguf(str(tmp_path / "tiny.gguf"), tiny())
    with pytest.warns(UserWarning, match="not rounded"):
        load(path, device="cpu", max_ctx=256, kv_type=kind)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        load(path, device="cpu", max_ctx=256)
