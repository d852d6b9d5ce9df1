"""The 8-bit cache's entry points and the kernel library agree on the page size, or no call is made."""
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
