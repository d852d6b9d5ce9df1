"""What the 8-bit paged cache's entry points refuse: every check runs before anything is launched, so
none of this needs a GPU (a call that is right in all else ends at the check for one)."""
import pytest
import torch

from k8s_nvidia_gpus_amd.ops import llm_kv8 as KV

S, HKV, H, D, N, COLS = 2, 2, 4, 64, 5, 3


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def good(name):
    cache = KV.KV8Cache.empty(4, HKV, D, torch.int8, "cpu")
    pages = torch.zeros(S, COLS, dtype=torch.int32)
    start, cu = ints(0, 3), ints(0, 2, N)
    kv = torch.zeros(N, HKV, D, dtype=torch.float16)
    q = torch.zeros(N, H, D, dtype=torch.float16)
    table = torch.zeros(COLS * KV.PAGE, D // 2)
    if name == "append":
        return dict(cache=cache, k=kv, v=kv.clone(), pages=pages, start=start, cu=cu, cos_t=table,
                    sin_t=table.clone(), q=q, q_out=q.clone())
    if name == "read":
        return dict(cache=cache, pages=pages, start=start, cu=cu, k_out=kv, v_out=kv.clone())
    if name == "decode":
        return dict(q=q[:S], cache=cache, pages=pages, pos=ints(4, 70), out=q[:S].clone(), scale=0.1)
    return dict(q=q, cache=cache, pages=pages, start=start, cu=cu, out=q.clone(), scale=0.1)


CALLS = {"append": KV.kv8_append, "read": KV.kv8_read, "decode": KV.kv8_attn_decode, "prompt": KV.kv8_attn_prompt}


@pytest.mark.parametrize("name", CALLS)
def test_a_right_call_gets_as_far_as_the_device(name):
    with pytest.raises(ValueError, match="GPU"):
        CALLS[name](**good(name))


@pytest.mark.parametrize("layout", [
    lambda z: z(H, N, D).transpose(0, 1),                    # head-major
    lambda z: z(N, H + 3, 2 * D)[:, 1:-2, D:],
    lambda z: z(H, 2 * N, D)[:, ::2].transpose(0, 1),
])
def test_outputs_of_any_layout_whose_rows_are_their_own_are_taken(layout):
    out = layout(lambda *shape: torch.zeros(shape, dtype=torch.float16))
    with pytest.raises(ValueError, match="GPU"):
        KV.kv8_attn_prompt(**{**good("prompt"), "out": out})


def with_cache(i, t):
    def change(a):
        c = list(a["cache"])
        c[i] = t(c[i])
        a["cache"] = c
    return change


def with_arg(key, t):
    def change(a):
        a[key] = t(a[key]) if callable(t) else t
    return change


COMMON = [
    (with_cache(0, lambda t: t.float()), "codes"),
    (with_cache(0, lambda t: t[:, :, :32]), "codes"),
    (with_cache(0, lambda t: t.transpose(0, 1)), "codes"),
    (with_cache(1, lambda t: t.transpose(2, 3).contiguous()[:, :, :, :32]), "codes"),
    (with_cache(1, lambda t: t.view(torch.float8_e4m3fn)), "codes"),
    (with_cache(2, lambda t: t.double()), "scales"),
    (with_cache(3, lambda t: t[:2]), "scales"),
    (with_arg("pages", lambda t: t.long()), "page table"),
    (with_arg("pages", lambda t: t[0]), "page table"),
    (with_arg("pages", lambda t: t.t().contiguous().t()), "page table"),
    (with_arg("pages", lambda t: t[:0]), "page table"),
]
OWN = {
    "append": [
        (with_arg("k", lambda t: t.double()), "type"),
        (with_arg("k", lambda t: t[:, :1]), "k "),
        (with_arg("k", lambda t: t[:-1]), "v "),
        (with_arg("v", lambda t: t.bfloat16()), "type"),
        (with_arg("v", lambda t: torch.zeros(N, D, HKV, dtype=t.dtype).transpose(1, 2)), "v "),
        (with_arg("start", lambda t: t.long()), "start"),
        (with_arg("start", lambda t: t[:1]), "start"),
        (with_arg("cu", lambda t: t[:2]), "cu"),
        (with_arg("cos_t", None), "cos_t goes"),
        (with_arg("cos_t", lambda t: t[:-1]), "rotation tables"),
        (with_arg("sin_t", lambda t: t.half()), "rotation tables"),
        (with_arg("q_out", None), "q with q_out"),
        (with_arg("q_out", lambda t: t.bfloat16()), "q_out"),
        (with_arg("q_out", lambda t: t.float()), "q_out"),
        (with_arg("q", lambda t: t.float()), "type"),
        (with_arg("q", lambda t: t[:-1]), "q "),
        (with_arg("q", lambda t: t[0]), "q "),
        (with_arg("q", lambda t: t[:, :0]), "q "),
        (with_arg("k", lambda t: t[0, 0]), "k "),
        (with_arg("q_out", lambda t: t[:1].expand(N, H, D)), "overlap"),
        (with_arg("q_out", lambda t: t.view(-1).as_strided((N, H, D), (H * D // 2, D // 2, 1))), "overlap"),
    ],
    "read": [
        (with_arg("k_out", lambda t: t.double()), "type"),
        (with_arg("v_out", lambda t: t[:-1]), "v_out"),
        (with_arg("cu", lambda t: t.float()), "cu"),
        (with_arg("k_out", lambda t: t[0, 0, 0]), "k_out"),
        (with_arg("k_out", lambda t: t[:, :1].expand(N, HKV, D)), "overlap"),
        (with_arg("v_out", lambda t: t[:1].expand(N, HKV, D)), "overlap"),
    ],
    "decode": [
        (with_arg("q", lambda t: t[:, :3]), "multiple"),
        (with_arg("q", lambda t: t.float()), "fp16 or bf16"),
        (with_arg("q", lambda t: t[:1]), "out"),
        (with_arg("out", lambda t: t.bfloat16()), "out"),
        (with_arg("out", None), "neither"),
        (with_arg("out", lambda t: t[:1].expand(S, H, D)), "overlap"),
        (with_arg("pos", lambda t: t[:1]), "pos"),
        (with_arg("window", -1), "window"),
        (with_arg("sinks", 1 << 31), "sinks"),
        (with_arg("span", COLS * 64 + 1), "span"),
        (with_arg("span", -1), "span"),
        (with_arg("q8_out", lambda t: (torch.zeros(S, H * D, dtype=torch.int8), torch.zeros(S, 1),
                                       torch.zeros(S, H * D // 16))), "q8_out"),
    ],
    "prompt": [
        (with_arg("q", lambda t: t[:, :3]), "multiple"),
        (with_arg("q", lambda t: t.float()), "fp16 or bf16"),
        (with_arg("out", lambda t: t[:-1]), "out"),
        (with_arg("start", lambda t: t[:1]), "start"),
        (with_arg("cu", lambda t: t[:2]), "cu"),
        (with_arg("out", None), "out"),
        (with_arg("out", lambda t: t.view(-1).as_strided((N, H, D), (D, D, 1))), "overlap"),
        (with_arg("span", 1000), "span"),
    ],
}


@pytest.mark.parametrize("name,i", [(n, i) for n in CALLS for i in range(len(COMMON + OWN[n]))])
def test_wrong_arguments_are_refused(name, i):
    change, why = (COMMON + OWN[name])[i]
    a = {"q8_out": None, **good(name)} if name == "decode" else good(name)
    change(a)
    with pytest.raises(ValueError, match=why):
        CALLS[name](**a)


@pytest.mark.parametrize("bad", [dict(dtype=torch.float16), dict(head_dim=96), dict(pages=0), dict(kv_heads=0)])
def test_a_cache_that_no_kernel_reads_is_refused(bad):
    with pytest.raises(ValueError, match="KV8Cache"):
        KV.KV8Cache.empty(**{**dict(pages=2, kv_heads=1, head_dim=64, dtype=torch.int8, device="cpu"), **bad})


# ------------------------------------------------------------------------------------------- the engine
@pytest.fixture(scope="module")
def tiny_model(tmp_path_factory):
    from k8s_nvidia_gpus_amd.models.llm import tiny
    from k8s_nvidia_gpus_amd.models.llm.synthetic import write_synthetic_gguf

    return write_synthetic_gguf(str(tmp_path_factory.mktemp("llm") / "tiny.gguf"), tiny())


def test_engine_takes_the_cache_types_it_knows(tiny_model):
    from k8s_nvidia_gpus_amd.models.llm.synthetic import load

    with pytest.raises(ValueError, match="kv_type"):
        load(tiny_model, device="cpu", max_ctx=256, kv_type="q4_0")
    a, _ = load(tiny_model, device="cpu", max_ctx=256)
    b, _ = load(tiny_model, device="cpu", max_ctx=256, kv_type="int8")   # the CPU reference maths
    assert b.kv_type == "int8" and b.kv8 is None
    assert torch.equal(a.prefill([5, 6, 7], 1), b.prefill([5, 6, 7], 1))
    assert torch.equal(a.decode([9], [3], [1]), b.decode([9], [3], [1]))


def test_engine_runs_of_a_step():
    from k8s_nvidia_gpus_amd.models.llm.engine import Engine

    assert Engine._runs_of([4, 5, 6], [2, 2, 2]).tolist() == [[4, 0, 0, 0], [0, 3, 3, 3], [2, 0, 0, 0]]
    assert Engine._runs_of([9, 3, 4], [0, 1, 1]).tolist() == [[9, 3, 0, 0], [0, 1, 3, 3], [0, 1, 0, 0]]
    for positions, slots in (([4, 4], [0, 0]), ([5, 4], [0, 0]), ([1, 7, 2], [0, 1, 0])):
        with pytest.raises(ValueError, match="consecutive"):
            Engine._runs_of(positions, slots)


def test_server_passes_the_cache_type_on(tmp_path):
    from types import SimpleNamespace

    from k8s_nvidia_gpus_amd.models.llm import server

    eng, _, _ = server.build_engine(SimpleNamespace(model=None, synthetic="tiny", ctx_size=256, parallel=2,
                                                    cache_type="e4m3"))
    assert eng.kv_type == "e4m3"
    with pytest.raises(SystemExit):
        server.main(["--cache-type", "fp4"])
