"""What 8 bits cost the attention when a few key channels are large (a key bias): the format's own rounding and
no more.

With one scale for 64 positions of a head's keys an int8 key is off by step / sqrt(12) (rms) in every channel,
the step following the largest channel; with normal queries a score (over sqrt(D)) is off by as much, and a
softmax weight by that share.  Values are off by their own step / sqrt(12).  The output of random values then is
off by the root of both squares, as a share of its norm.  e4m3 is off by at most 2^-4 / sqrt(3) (rms over a
binade's worst place) of each key and value, whatever the largest channel is.  A quarter is allowed for the
second order and for the sample."""
import math

import pytest
import torch

from test_llm_kv8_gpu import CODES, DEV, KV, PAGE, ints, rotated, tables   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bias", [0, 10, 30, 100])
def test_large_key_channels_cost_what_the_format_rounds(KV, code, bias):   # noqa: F811
    n, h, hkv, d = 1024, 8, 2, 128
    g = torch.Generator(device=DEV).manual_seed(95)
    q, k, v = (torch.randn(n, x, d, device=DEV, generator=g) for x in (h, hkv, hkv))
    k[:, :, 60] += bias                                       # a pair that turns slowly; queries are small there
    k[:, :, 60 + d // 2] += bias / 2
    q[:, :, 60] *= 0.02
    q[:, :, 60 + d // 2] *= 0.02
    cos, sin = tables(n, d)
    pos, rows = torch.arange(n, device=DEV), ints([list(range(n // PAGE))])
    cache = KV.KV8Cache.empty(n // PAGE, hkv, d, CODES[code], DEV)
    q16, out = (torch.empty(n, h, d, device=DEV, dtype=torch.float16) for _ in range(2))
    KV.kv8_append(cache, k, v, rows, ints([0]), ints([0, n]), cos, sin, q=q, q_out=q16)
    KV.kv8_attn_prompt(q16, cache, rows, ints([0]), ints([0, n]), out, 1 / math.sqrt(d))
    qr, kr = rotated(q, pos, cos, sin).double(), rotated(k, pos, cos, sin).double()
    err = norm = 0.0
    hidden = torch.ones(n, n, device=DEV, dtype=torch.bool).triu(1)
    for i in range(h):
        w = torch.softmax((qr[:, i] @ kr[:, i * hkv // h].t() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
        want = w @ v[:, i * hkv // h].double()
        err += float((out[:, i].double() - want).square().sum())
        norm += float(want.square().sum())
    if code == "int8":
        share = math.sqrt(float(cache.ks.max()) ** 2 / 12 + float(cache.vs.max()) ** 2 / 12)
    else:
        share = math.sqrt(2) * 2 ** -4 / math.sqrt(3)
    assert math.sqrt(err / norm) <= 1.25 * share
