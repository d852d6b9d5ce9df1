"""The 8-bit cache's attentions and pages that a row does not see: their scales and poison stay without
effect on it, although other rows of the same call, or other keys of the same span, meet them.

Tolerance of an output element, A = sum_j p_j |v_j| over the row's n visible keys: half a step of the output's
type; a weight's fp16 rounding, 2^-11 A, and scores, exponents and sums in fp32, 2^-12 A (chains of up to 64
pages of some 70 operations); and a weight below fp16's normal range, 2^-32 of the largest weight times the
largest value scale that the row sees times the largest code."""
import math

import pytest
import torch

from test_llm_kv8_gpu import CODES, DEV, KV, PAGE, dense, ints, prompt_case, run_prompt   # noqa: F401

pytestmark = pytest.mark.gpu
TOP = {"int8": 127.0, "e4m3": 448.0}


def check_rows(cache, row, q, pos, scale, got, code, window=0, sinks=0, span=1 << 30):
    """Rows q [R, H, D] at positions pos .. against the definition in 64 bits."""
    hkv, group = cache.k.shape[1], q.shape[1] // cache.k.shape[1]
    n = min(pos + len(q), span, len(row) * PAGE)
    p, j = pos + torch.arange(len(q), device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    pages = torch.tensor(row, device=DEV)[torch.arange(n, device=DEV) // PAGE]
    for kh in range(hkv):
        k, v, mapped = dense(cache, row, kh, n)
        seen = (j <= p) & mapped
        if window:
            seen &= (j > p - window) | (j < sinks)
        k, v = torch.where(seen.any(0)[:, None], k, 0.0), torch.where(seen.any(0)[:, None], v, 0.0)
        vs = torch.where(seen, cache.vs[pages.clamp(min=0), kh].double().nan_to_num(), 0.0).amax(1)
        for g in range(kh * group, (kh + 1) * group):
            s = (q[:, g].double() @ k.t() * scale).masked_fill(~seen, -math.inf)
            w = torch.where(seen.any(1, keepdim=True), torch.softmax(s, 1), 0.0)
            want, a = w @ v, w @ v.abs()
            tol = (torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2 ** -8) + (2 ** -11 + 2 ** -12) * a
                   + (seen.sum(1) * vs)[:, None] * 2.0 ** -32 * TOP[code] + 1e-36)
            worst = ((got[:, g].double() - want).abs() / tol).max()
            assert worst <= 1.0, f"head {g}: {float(worst):.3f} of the tolerance"


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("h,hkv,d", [(2, 2, 128), (28, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("low", [-20, -40, -90])
@pytest.mark.parametrize("starts,lens", [([0, 200], [330, 100]), ([100], [900])])
def test_prompt_a_large_page_outside_of_a_rows_window(KV, code, h, hkv, d, low, starts, lens):   # noqa: F811
    """Pages of value scales 2^4 and 2^low in turn, a window of 10: rows next to each other see only the one
    or only the other."""
    cache, rows, q = prompt_case(KV, starts, lens, h, hkv, d, code, torch.bfloat16, seed=80)
    for row in rows:
        for j, i in enumerate(row):
            if i >= 0:
                cache.vs[i] = 2.0 ** (low if j % 2 else 4)
    for window, sinks in ((10, 0), (1, 0), (70, 3)):
        got, at = run_prompt(KV, cache, rows, q, starts, lens, window=window, sinks=sinks), 0
        for s, n in enumerate(lens):
            check_rows(cache, rows[s], q[at:at + n], starts[s], 1 / math.sqrt(d), got[at:at + n], code, window, sinks)
            at += n


@pytest.mark.parametrize("code", CODES)
def test_prompt_a_large_page_behind_a_row(KV, code):   # noqa: F811
    """Causal: rows of the first page do not see the second one's value scale, 2^160 of their own."""
    cache, rows, q = prompt_case(KV, [0], [100], 8, 2, 128, code, torch.bfloat16, seed=81)
    cache.vs[rows[0][0]], cache.vs[rows[0][1]] = 2.0 ** -100, 2.0 ** 60
    check_rows(cache, rows[0], q, 0, 1 / math.sqrt(128), run_prompt(KV, cache, rows, q, [0], [100]), code)


@pytest.mark.parametrize("poison", [float("nan"), 2.0 ** 60])
@pytest.mark.parametrize("span,window,sinks", [(100, 190, 0), (100, 190, 5), (70, 300, 60), (70, 240, 0), (65, 299, 0)])
def test_a_page_that_a_window_leaves_within_the_span(KV, poison, span, window, sinks):   # noqa: F811
    """Position 300, keys below `span` only: the window begins in page 1, at or behind the span, or not."""
    cache, rows, q = prompt_case(KV, [300], [1], 8, 2, 128, "int8", torch.bfloat16, seed=82)
    seen = max(0, 300 - window + 1) < span
    if not seen:
        cache.vs[rows[0][1]] = poison
    scale = 1 / math.sqrt(128)
    for name in ("decode", "prompt"):
        out = torch.full_like(q, 7.0)
        if name == "decode":
            KV.kv8_attn_decode(q, cache, ints(rows), ints([300]), out, scale, window=window, sinks=sinks, span=span)
        else:
            KV.kv8_attn_prompt(q, cache, ints(rows), ints([300]), ints([0, 1]), out, scale, window=window,
                               sinks=sinks, span=span)
        check_rows(cache, rows[0], q, 300, scale, out, "int8", window, sinks, span)
