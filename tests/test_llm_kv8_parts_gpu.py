"""Attention over the 8-bit cache where a lost page or a lost part would show: values of each page in dims of
its own, and very long rows whose last parts hold most of the weight.

Tolerance of an output element, A = sum_j p_j |v_j|: half a step of the output's type; a weight's fp16
rounding, 2^-11 A; scores, exponents and sums in fp32, 2^-11 A (a wave's chain of up to 64 pages of some 70
operations is 4500 steps of 2^-24, a join's of two rounds of 64 parts 200); and a weight below fp16's normal
range, 2^-32 of the largest weight times the largest value scale, for each key times its code in that dim (a
code of 0 adds nothing).  Each test also makes sure that the outputs it guards against lie outside."""
import math

import pytest
import torch

from test_llm_kv8_gpu import CODES, DEV, KV, PAGE, bits, dense, ints, random_cache, run_prompt, table_of   # noqa: F401

pytestmark = pytest.mark.gpu


def tolerance(want, a, top, vs, codes, dtype):
    """top: the largest softmax weight; vs: the largest value scale; codes: sum of |code| over the keys, by dim."""
    return (torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2 ** -8) + 2 ** -10 * a
            + 2.0 ** -32 * top * vs * codes + 1e-36)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("pages", [2, 5, 16])
@pytest.mark.parametrize("low", [0, 5, 12, 18, 24])
@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_every_page_counts_whatever_its_value_scale(KV, code, pages, low, form):   # noqa: F811
    """Page i has values in dims 8 i .. 8 i + 7 only; value scales fall to 2^-low of the largest, so that a
    weight keeps 2^-11 of itself down to 2^-20 and at worst 2^-8 at 2^-24."""
    g = torch.Generator(device=DEV).manual_seed(90)
    d, h, hkv = 128, 4, 2
    cache = random_cache(KV, pages, hkv, d, code, g)
    row = torch.randperm(pages, generator=torch.Generator().manual_seed(91)).tolist()
    cache.ks.fill_(2.0 ** (-6 if code == "int8" else -7))
    for i, at in enumerate(row):
        v = torch.randint(64, 120, (hkv, 8, PAGE), device=DEV, generator=g).float()   # (e4m3 rounds them)
        cache.v[at] = torch.zeros(hkv, d, PAGE, device=DEV).to(cache.v.dtype)
        cache.v[at, :, 8 * i:8 * i + 8] = v.to(cache.v.dtype)
        cache.vs[at] = 2.0 ** math.floor(4 - low * i / (pages - 1))
    n, scale = pages * PAGE, 1 / math.sqrt(d)
    q = torch.randn(1, h, d, device=DEV, generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    if form == "decode":
        KV.kv8_attn_decode(q, cache, ints([row]), ints([n - 1]), out, scale)
    else:
        KV.kv8_attn_prompt(q, cache, ints([row]), ints([n - 1]), ints([0, 1]), out, scale)
    for g_ in range(h):
        k, v, _ = dense(cache, row, g_ * hkv // h, n)
        p = torch.softmax(q[0, g_].double() @ k.t() * scale, -1)
        want = p @ v
        codes = bits(cache.v)[row, g_ * hkv // h].view(cache.v.dtype).double().sum((0, 2))
        tol = tolerance(want, want, p.max(), 16.0, codes, out.dtype)
        assert ((out[0, g_].double() - want).abs() <= tol).all()
        assert (want[:8 * pages] > 2 * tol[:8 * pages]).all()          # a page lost would show


@pytest.mark.parametrize("s,pages,part", [(1, 33000, 512), (130, 16500, 256)])
def test_decode_more_parts_than_a_join_takes_at_once(KV, s, pages, part):   # noqa: F811
    """65 parts: pages that only the last one has hold most of the weight and values of their own."""
    g = torch.Generator(device=DEV).manual_seed(92)
    d, h, scale = 64, 4, 0.125
    cache = KV.KV8Cache.empty(12, 1, d, torch.int8, DEV)
    cache.k.copy_(torch.randint(-20, 21, cache.k.shape, device=DEV, generator=g))
    cache.v.copy_(torch.randint(1, 30, cache.v.shape, device=DEV, generator=g))
    cache.ks.fill_(2.0 ** -10)
    cache.vs.fill_(2.0 ** -6)
    table = torch.randint(0, 8, (pages,), device=DEV, generator=g, dtype=torch.int32)
    late = 64 * part
    assert late + 4 <= pages
    where = [late, late + 1, late + 3, pages - 1]
    for i, at in enumerate(where):                             # pages 8 .. 11: once each, behind part 63
        table[at] = 8 + i
        cache.v[8 + i] = 0
        cache.v[8 + i, :, 8 * i:8 * i + 8] = torch.randint(60, 120, (1, 8, PAGE), device=DEV, generator=g).to(torch.int8)
    direction = torch.randint(0, 2, (d,), device=DEV, generator=g) * 2.0 - 1
    cache.k[8:] = (direction * 100).to(torch.int8)
    cache.ks[8:] = 2.0 ** -6
    q = (direction * (0.9 + 0.05 * torch.arange(h, device=DEV)[:, None]))[None].half()   # scores of 11 to 13
    q = q.expand(s, h, d)
    pos = pages * PAGE - 5
    out = torch.full((s, h, d), 7.0, device=DEV, dtype=torch.float16)
    KV.kv8_attn_decode(q, cache, table[None].expand(s, -1), ints([pos] * s), out, scale)
    count = torch.bincount(table.long(), minlength=12).double()[:, None].repeat(1, PAGE)
    count[11, PAGE - 4:] = 0
    first = torch.bincount(table[:late].long(), minlength=12).double()[:, None].repeat(1, PAGE)
    k, v, _ = dense(cache, list(range(12)), 0, 12 * PAGE)
    e = torch.exp(q[0].double() @ k.t() * scale)

    def of(times):
        w = e * times.reshape(-1)
        return w @ v / w.sum(-1, keepdim=True)

    want = of(count)
    top = e.amax(-1, keepdim=True) / (e @ count.reshape(-1))[:, None]
    codes = count.reshape(-1) @ (v * 2.0 ** 6)
    tol = tolerance(want, want, top, 2.0 ** -6, codes, out.dtype)
    for lost in (torch.zeros_like(want), of(first)):           # zeros, and all parts but the last
        assert ((lost - want).abs() > 2 * tol).any(-1).all()
    for i in range(4):
        one = count.clone()
        one[8 + i] = 0
        assert ((of(one) - want).abs() > 2 * tol).any(-1).all()
    assert ((out.double() - want).abs() <= tol).all()
    assert torch.equal(out, out[:1].expand_as(out))
