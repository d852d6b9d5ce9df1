"""MI355X numerics of the 8-bit paged KV cache (ops/csrc/llm_kv8.hip) against plain forms in 64 bits.

Tolerances of the attentions, for each output element with A = sum_j p_j |v_j| (p the softmax weights):
* the output's own rounding: half a step, finfo.eps / 2 of its value;
* a weight goes to the matrix instruction as fp16: 2^-11 of it, so 2^-11 A; scores, exp2 and sums in fp32
  add (n + 64) 2^-24 A at most (n keys); both sides together below 2^-10.9 A for the sizes here;
* weights below fp16's normal range (of the largest weight, or when their page's value scale lies far
  under the largest one): an absolute 2^-25 of the largest value magnitude vmax, for each key.
q enters exactly (bf16 is shifted into fp16's range), codes are exact in fp16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def KV():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from k8s_nvidia_gpus_amd.ops import kernels, llm_kv8

    kernels.library()            # must load the in-tree .so: no fallback
    return llm_kv8


DEV = "cuda:0"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def scale_of(amax, code):
    """The least power of two s with amax <= qmax s."""
    qmax = 127.0 if code == "int8" else 448.0
    e = torch.ceil(torch.log2(amax.double() / qmax))
    e = torch.where(torch.exp2(e - 1) * qmax >= amax.double(), e - 1, e)
    return torch.where(amax > 0, torch.exp2(e), 0.0)


def to_codes(x, s, code):
    y = torch.where(s > 0, x.double() / torch.where(s > 0, s.double(), 1.0), 0.0)
    return y.round().to(torch.int8) if code == "int8" else y.float().to(torch.float8_e4m3fn)


def bits(t):
    return t.view(torch.uint8)


def random_cache(KV, pool, hkv, d, code, gen, spread=1.0):
    """Codes of any values, scales over 2^-4 .. 2^4 times `spread`; dead rows hold them too."""
    c = KV.KV8Cache.empty(pool, hkv, d, CODES[code], DEV)
    for t, s in ((c.k, c.ks), (c.v, c.vs)):
        x = torch.randn(t.shape, device=DEV, generator=gen)
        t.copy_((x * 30).round().clamp(-127, 127)) if code == "int8" else t.copy_(x * 60)
        e = torch.randint(-4, 5, s.shape, device=DEV, generator=gen).double()
        s.copy_(torch.exp2(e - 6 if code == "int8" else e - 7))
    c.ks.mul_(spread)
    return c


def table_of(lens, cols, pool, seed=0):
    """A table of distinct pages in no order, -1 behind each sequence's end."""
    g = torch.Generator().manual_seed(seed)
    order, at, rows = torch.randperm(pool, generator=g).tolist(), 0, []
    for n in lens:
        need = -(-n // PAGE)
        rows.append(order[at:at + need] + [-1] * (cols - need))
        at += need
    return rows


def dense(cache, row, head, n):
    """Keys and values [n, D] of a sequence's first n positions in 64 bits, and which are mapped."""
    ids = [i for i in row[:-(-n // PAGE)]]
    good = torch.tensor([0 <= i < cache.k.shape[0] for i in ids], device=DEV)
    at = torch.tensor([i if 0 <= i < cache.k.shape[0] else 0 for i in ids], device=DEV, dtype=torch.long)
    k = bits(cache.k)[at, head].view(cache.k.dtype).double() * cache.ks[at, head].double()[:, None, None]
    v = bits(cache.v)[at, head].view(cache.v.dtype).double() * cache.vs[at, head].double()[:, None, None]
    return (k.reshape(-1, k.shape[-1])[:n], v.transpose(1, 2).reshape(-1, k.shape[-1])[:n],
            good.repeat_interleave(PAGE)[:n])


def reference(cache, row, q, pos, scale, window=0, sinks=0, span=1 << 30):
    """q [R, H, D] at positions pos.. of one sequence -> (output, A, n keys, vmax) in 64 bits."""
    r, h, d = q.shape
    hkv = cache.k.shape[1]
    n = max(0, min(pos + r, span, len(row) * PAGE))
    out = torch.zeros(r, h, d, dtype=torch.float64, device=DEV)
    a, vmax = torch.zeros_like(out), 0.0
    if n == 0:
        return out, a, 0, 0.0
    p = pos + torch.arange(r, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None]
    for kh in range(hkv):
        k, v, mapped = dense(cache, row, kh, n)
        seen = (j <= p) & mapped
        if window:
            seen &= (j > p - window) | (j < sinks)
        any_row = seen.any(0)
        k, v = torch.where(any_row[:, None], k, 0.0), torch.where(any_row[:, None], v, 0.0)
        vmax = max(vmax, float(v.nan_to_num().abs().max()))
        for g in range(kh * (h // hkv), (kh + 1) * (h // hkv)):
            s = (q[:, g].double() @ k.t()) * scale
            s = s.masked_fill(~seen, -math.inf)
            w = torch.softmax(s, -1)
            w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
            out[:, g], a[:, g] = w @ v, w @ v.abs()
    return out, a, n, vmax


def check(got, ref):
    want, a, n, vmax = ref
    tol = (torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2 ** -8)
           + (2 ** -11 + (n + 64) * 2 ** -24) * a + n * 2 ** -25 * vmax + 1e-30)
    worst = ((got.double() - want).abs() / tol).max() if got.numel() else torch.tensor(0.0)
    assert torch.isfinite(got).all()
    assert worst <= 1.0, f"{float(worst):.3f} of the tolerance"


# ------------------------------------------------------------------------------------------------ decode
LENS = [0, 1, 63, 64, 65, 200, 5, 1000]


def decode_case(KV, lens, h, hkv, d, code, dtype, seed=0, cols=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cols = cols or max(1, -(-max(lens) // PAGE))
    pool = sum(-(-n // PAGE) for n in lens) + 2
    cache = random_cache(KV, pool, hkv, d, code, g)
    rows = table_of(lens, cols, pool, seed)
    q = torch.randn(len(lens), h, d, device=DEV, generator=g).to(dtype)
    return cache, rows, q, ints([n - 1 for n in lens])


def run_decode(KV, cache, rows, q, pos, **kw):
    out = torch.full_like(q, float("nan"))
    KV.kv8_attn_decode(q, cache, ints(rows), pos, out, 1 / math.sqrt(q.shape[2]), **kw)
    return out


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hkv,d", [(28, 4, 128), (4, 4, 64), (3, 1, 128), (16, 1, 64), (34, 2, 128)])
def test_decode(KV, code, dtype, h, hkv, d):
    cache, rows, q, pos = decode_case(KV, LENS, h, hkv, d, code, dtype)
    got = run_decode(KV, cache, rows, q, pos)
    for s, n in enumerate(LENS):
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(d)))
    assert not got[0].any()                                # nothing to see: zeros


@pytest.mark.parametrize("n", [4095, 4097, 16384, 16385, 40000])
def test_decode_long(KV, n):
    cache, rows, q, pos = decode_case(KV, [n, 700], 14, 2, 128, "int8", torch.float16)
    got = run_decode(KV, cache, rows, q, pos)
    for s, m in enumerate([n, 700]):
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], m - 1, 1 / math.sqrt(128)))


@pytest.mark.parametrize("s,pages", [(1, 65), (3, 9), (64, 9), (64, 17), (64, 33), (129, 10), (70, 130)])
def test_decode_many_rows_share_pages(KV, s, pages):
    """Parts by the number of rows; the rows' tables name the same pages in other orders."""
    g = torch.Generator(device=DEV).manual_seed(60)
    cache = random_cache(KV, 40, 4, 128, "e4m3", g)
    table = torch.randint(0, 40, (s, pages), device=DEV, generator=g, dtype=torch.int32)
    pos = torch.randint(0, pages * PAGE, (s,), device=DEV, generator=g, dtype=torch.int32)
    pos[-1] = pages * PAGE - 1
    q = torch.randn(s, 8, 128, device=DEV, generator=g).half()
    out = torch.full_like(q, float("nan"))
    KV.kv8_attn_decode(q, cache, table, pos, out, 0.08)
    rows, at = table.tolist(), pos.tolist()
    for i in {0, s // 2, s - 1}:
        check(out[i:i + 1], reference(cache, rows[i], q[i:i + 1], at[i], 0.08))


def test_decode_more_than_a_million_positions(KV):
    """More pages than 64 parts of four waves hold table entries for; few distinct ones, so that the plain
    form is a sum over those: page u is seen n_u times and the last one up to the position."""
    g = torch.Generator(device=DEV).manual_seed(61)
    cache = random_cache(KV, 8, 1, 64, "int8", g, spread=0.01)
    pages, scale = 16500, 0.1
    table = torch.randint(0, 7, (1, pages), device=DEV, generator=g, dtype=torch.int32)
    table[0, -1] = 7                                        # the last page is its own
    pos = pages * PAGE - 10
    q = torch.randn(1, 4, 64, device=DEV, generator=g).half()
    out = torch.empty_like(q)
    KV.kv8_attn_decode(q, cache, table, ints([pos]), out, scale)
    count = torch.bincount(table[0].long(), minlength=8).double().repeat_interleave(PAGE)
    count[-9:] = 0
    k, v, _ = dense(cache, list(range(8)), 0, 8 * PAGE)
    w = torch.exp((q[0].double() @ k.t()) * scale) * count
    w /= w.sum(-1, keepdim=True)
    check(out, ((w @ v)[None], (w @ v.abs())[None], pages * PAGE, float(v.abs().max())))


WINDOWS = [(1, 0), (1, 1), (64, 0), (65, 4), (100, 64), (130, 70), (5000, 3), (7, 1000)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("code", CODES)
def test_decode_window_and_sinks(KV, code, window, sinks):
    lens = [0, 1, 64, 66, 129, 700, 2000]
    cache, rows, q, pos = decode_case(KV, lens, 8, 2, 128, code, torch.bfloat16, seed=3)
    got = run_decode(KV, cache, rows, q, pos, window=window, sinks=sinks)
    for s, n in enumerate(lens):
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(128), window, sinks))


def test_decode_unmapped_pages_and_bad_entries_are_not_attended(KV):
    lens = [640, 640, 64, 300]
    cache, rows, q, pos = decode_case(KV, lens, 8, 2, 128, "e4m3", torch.float16, seed=5)
    rows[0][3:7] = [-1] * 4
    rows[1][2], rows[1][5] = cache.k.shape[0], 2 ** 31 - 1   # past the pool
    rows[2][0] = -7                                          # all a sequence has
    got = run_decode(KV, cache, rows, q, pos)
    for s, n in enumerate(lens):
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(128)))
    assert not got[2].any()


def test_decode_ignores_what_lies_behind_a_sequence(KV):
    lens = [5, 64, 100, 333]
    cache, rows, q, pos = decode_case(KV, lens, 8, 2, 64, "e4m3", torch.bfloat16, seed=6)
    want = run_decode(KV, cache, rows, q, pos)
    for s, n in enumerate(lens):                             # NaN codes in the dead rows
        if n % PAGE:
            bits(cache.k)[rows[s][n // PAGE], :, n % PAGE:] = 0x7f
            bits(cache.v)[rows[s][n // PAGE], :, :, n % PAGE:] = 0xff
    assert torch.equal(run_decode(KV, cache, rows, q, pos), want)


def test_decode_span_bounds_the_keys(KV):
    lens = [1000, 200, 64]
    cache, rows, q, pos = decode_case(KV, lens, 8, 2, 128, "int8", torch.float16, seed=7)
    for span in (64, 129, 512, 1024):
        got = run_decode(KV, cache, rows, q, pos, span=min(span, len(rows[0]) * PAGE))
        for s, n in enumerate(lens):
            check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(128), span=span))


def test_decode_positions_behind_the_table(KV):
    cache, rows, q, _ = decode_case(KV, [128, 128], 4, 2, 64, "int8", torch.float16, seed=8)
    got = run_decode(KV, cache, rows, q, ints([2 ** 31 - 1, 500]))
    for s, p in enumerate((2 ** 31 - 1, 500)):               # all of the table is seen
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1], min(p, 127), 1 / math.sqrt(64)))


@pytest.mark.parametrize("code", CODES)
def test_decode_pages_of_unlike_scales(KV, code):
    """Value scales 2^-40 .. 2^40 from page to page, zero pages and zero keys among them."""
    cache, rows, q, pos = decode_case(KV, [900, 450], 8, 2, 128, code, torch.float16, seed=9)
    e = torch.randint(-40, 41, cache.vs.shape, device=DEV).double()
    cache.vs.copy_(torch.exp2(e))
    for i in (rows[0][0], rows[0][4], rows[1][1]):
        cache.vs[i], cache.ks[i] = 0.0, 0.0
        bits(cache.k)[i], bits(cache.v)[i] = 0, 0
    got = run_decode(KV, cache, rows, q.float().to(torch.bfloat16), pos)   # bf16 has the range
    for s, n in enumerate((900, 450)):
        check(got[s:s + 1], reference(cache, rows[s], q[s:s + 1].float().to(torch.bfloat16), n - 1, 1 / math.sqrt(128)))


def test_decode_large_and_small_queries(KV):
    """bf16 queries past fp16's range on both sides (scores stay moderate through `scale`)."""
    for size in (1e30, 1e6, 1e-6, 1e-30):
        cache, rows, q, pos = decode_case(KV, [300, 64], 8, 2, 128, "int8", torch.bfloat16, seed=10)
        q = (q.float() * size).to(torch.bfloat16)
        out = torch.empty_like(q)
        KV.kv8_attn_decode(q, cache, ints(rows), pos, out, 0.1 / size)
        for s, n in enumerate((300, 64)):
            check(out[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 0.1 / size))


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-20])
def test_scales_of_any_sign(KV, scale):
    cache, rows, q = prompt_case(KV, [0, 130], [100, 40], 8, 2, 128, "int8", torch.float16, seed=18)
    cache.ks[rows[0][0]] = 0.0
    bits(cache.k)[rows[0][0]] = 0
    out = torch.empty_like(q)
    KV.kv8_attn_prompt(q, cache, ints(rows), ints([0, 130]), ints([0, 100, 140]), out, scale)
    check(out[:100], reference(cache, rows[0], q[:100], 0, scale))
    check(out[100:], reference(cache, rows[1], q[100:], 130, scale))
    KV.kv8_attn_decode(q[:2], cache, ints(rows), ints([99, 169]), out[:2], scale)
    for s, p in enumerate((99, 169)):
        check(out[s:s + 1], reference(cache, rows[s], q[s:s + 1], p, scale))


def test_decode_a_poisoned_page_poisons_those_that_see_it(KV):
    cache, rows, q, pos = decode_case(KV, [300, 300, 300], 8, 2, 128, "int8", torch.float16, seed=11)
    cache.vs[rows[0][2], 1] = float("nan")
    cache.ks[rows[1][0], 0] = float("nan")
    got = run_decode(KV, cache, rows, q, pos, window=100)    # positions 200 .. 299: pages 3 and 4
    assert got.isfinite().all()
    got = run_decode(KV, cache, rows, q, pos)
    assert got[0, 4:].isnan().all() and got[0, :4].isfinite().all()
    assert got[1, :4].isnan().all() and got[1, 4:].isfinite().all() and got[2].isfinite().all()


def test_decode_strides_and_alignments(KV):
    lens = [70, 500]
    cache, rows, q, pos = decode_case(KV, lens, 8, 2, 128, "int8", torch.float16, seed=12)
    want = run_decode(KV, cache, rows, q, pos)
    wide = torch.zeros(2, 8, 131, device=DEV, dtype=q.dtype)
    wide[..., 1:129] = q
    out = torch.zeros(8, 2, 129, device=DEV, dtype=q.dtype)
    KV.kv8_attn_decode(wide[..., 1:129], cache, ints(rows), pos, out.transpose(0, 1)[..., :128], 1 / math.sqrt(128))
    assert torch.equal(out.transpose(0, 1)[..., :128], want) and not out[..., 128].any()
    table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)      # a table with a row stride
    table[:, :len(rows[0])] = ints(rows)
    out = torch.empty_like(q)
    KV.kv8_attn_decode(q, cache, table[:, :len(rows[0])], pos, out, 1 / math.sqrt(128))
    assert torch.equal(out, want)


def test_decode_the_same_row_in_any_batch(KV):
    """Alone, in a batch of others and many times over (the batch decides how the pages are cut)."""
    lens = [1, 500, 3000, 9000, 64]
    cache, rows, q, pos = decode_case(KV, lens, 28, 4, 128, "int8", torch.float16, seed=13)
    many = run_decode(KV, cache, rows * 60, q.repeat(60, 1, 1), pos.repeat(60))
    assert torch.equal(many, many[:5].repeat(60, 1, 1))
    for s, n in enumerate(lens):
        ref = reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(128))
        check(many[s:s + 1], ref)
        check(run_decode(KV, cache, rows[s:s + 1], q[s:s + 1], pos[s:s + 1], span=max(64, -(-n // 64) * 64)), ref)


def test_decode_q8_output(KV):
    lens = [0, 5, 3000, 700]
    cache, rows, q, pos = decode_case(KV, lens, 28, 4, 128, "int8", torch.float16, seed=14)
    k = 28 * 128
    x8 = torch.empty(4, k, dtype=torch.int8, device=DEV)
    dx, sx = torch.empty(4, k // 32, device=DEV), torch.empty(4, k // 16, device=DEV)
    out = torch.empty_like(q)
    KV.kv8_attn_decode(q, cache, ints(rows), pos, out, 1 / math.sqrt(128), q8_out=(x8, dx, sx))
    assert torch.equal(out, run_decode(KV, cache, rows, q, pos))
    y, d = out.view(4, -1, 32).float(), dx.view(4, -1, 1)
    assert torch.equal(x8.view(4, -1, 32).abs().amax(-1).int(), torch.where(dx > 0, 127, 0).int())
    # half a step of the codes, half one of the fp16 output and its share in the scale
    assert ((x8.view(4, -1, 32) * d - y).abs() <= d * 0.5 + y.abs().amax(-1, keepdim=True) * 2 ** -10 + 1e-6).all()
    torch.testing.assert_close(sx, (x8.view(4, -1, 16).float().sum(-1) * dx.repeat_interleave(2, 1)), rtol=1e-6, atol=0)
    only = torch.empty_like(x8)
    KV.kv8_attn_decode(q, cache, ints(rows), pos, None, 1 / math.sqrt(128), q8_out=(only, dx, sx))
    assert torch.equal(only, x8)


@pytest.mark.parametrize("d", [64, 128])
def test_decode_q8_of_a_short_context(KV, d):
    cache, rows, q, pos = decode_case(KV, [30, 64], 8, 2, d, "e4m3", torch.bfloat16, seed=15)
    x8 = torch.empty(2, 8 * d, dtype=torch.int8, device=DEV)
    dx, sx = torch.empty(2, 8 * d // 32, device=DEV), torch.empty(2, 8 * d // 16, device=DEV)
    out = torch.empty_like(q)
    KV.kv8_attn_decode(q, cache, ints(rows), pos, out, 1 / math.sqrt(d), q8_out=(x8, dx, sx))
    y, e = out.view(2, -1, 32).float(), dx.view(2, -1, 1)
    assert ((x8.view(2, -1, 32) * e - y).abs() <= e * 0.5 + y.abs().amax(-1, keepdim=True) * 2 ** -7 + 1e-6).all()
    for s, n in enumerate((30, 64)):
        check(out[s:s + 1], reference(cache, rows[s], q[s:s + 1], n - 1, 1 / math.sqrt(d)))


@pytest.mark.parametrize("n", [300, 3000])
def test_decode_q8_of_a_poisoned_page_is_not_silent(KV, n):
    cache, rows, q, pos = decode_case(KV, [n, n], 8, 2, 128, "int8", torch.float16, seed=17)
    cache.vs[rows[0][1], 1] = float("nan")
    x8 = torch.empty(2, 1024, dtype=torch.int8, device=DEV)
    dx, sx = torch.empty(2, 32, device=DEV), torch.empty(2, 64, device=DEV)
    KV.kv8_attn_decode(q, cache, ints(rows), pos, None, 1 / math.sqrt(128), q8_out=(x8, dx, sx))
    assert dx[0, 16:].isnan().all() and dx[0, :16].isfinite().all() and dx[1].isfinite().all()


def test_decode_offsets_pass_32_bits(KV):
    pool, hkv, d = 33100, 8, 128                            # 2.17 GB of key codes, as many of values
    cache = KV.KV8Cache.empty(pool, hkv, d, torch.int8, DEV)
    g = torch.Generator(device=DEV).manual_seed(16)
    small = random_cache(KV, 4, hkv, d, "int8", g)
    ids = [33099, 3, 32900, 33000]
    for i, at in enumerate(ids):
        cache.k[at], cache.v[at], cache.ks[at], cache.vs[at] = small.k[i], small.v[i], small.ks[i], small.vs[i]
    q = torch.randn(1, 16, d, device=DEV, generator=g).half()
    out, want = torch.empty_like(q), torch.empty_like(q)
    KV.kv8_attn_decode(q, cache, ints([ids]), ints([250]), out, 0.1)
    KV.kv8_attn_decode(q, small, ints([[0, 1, 2, 3]]), ints([250]), want, 0.1)
    assert torch.equal(out, want)
    KV.kv8_attn_prompt(q, cache, ints([ids]), ints([250]), ints([0, 1]), out, 0.1)
    check(out, reference(small, [0, 1, 2, 3], q, 250, 0.1))
    x = torch.randn(10, hkv, d, device=DEV, generator=g).half()
    KV.kv8_append(cache, x, x, ints([ids]), ints([186]), ints([0, 10]))
    KV.kv8_append(small, x, x, ints([[0, 1, 2, 3]]), ints([186]), ints([0, 10]))
    got, ref = torch.empty(250, hkv, d, device=DEV), torch.empty(250, hkv, d, device=DEV)
    got2, ref2 = torch.empty_like(got), torch.empty_like(ref)
    KV.kv8_read(cache, ints([ids]), ints([0]), ints([0, 250]), got, got2)
    KV.kv8_read(small, ints([[0, 1, 2, 3]]), ints([0]), ints([0, 250]), ref, ref2)
    assert torch.equal(got, ref) and torch.equal(got2, ref2)


# ------------------------------------------------------------------------------------------------ prompt
def prompt_case(KV, starts, lens, h, hkv, d, code, dtype, seed=0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ends = [a + b if b else 0 for a, b in zip(starts, lens)]
    cols = max(1, -(-max(ends) // PAGE))
    pool = sum(-(-n // PAGE) for n in ends) + 2
    cache = random_cache(KV, pool, hkv, d, code, g)
    rows = table_of(ends, cols, pool, seed)
    q = torch.randn(sum(lens) + pad, h, d, device=DEV, generator=g).to(dtype)
    return cache, rows, q


def run_prompt(KV, cache, rows, q, starts, lens, **kw):
    out = torch.full_like(q, 7.0)
    KV.kv8_attn_prompt(q, cache, ints(rows), ints(starts), ints(cumulative(lens)), out, 1 / math.sqrt(q.shape[2]), **kw)
    return out


def check_prompt(cache, rows, q, starts, lens, got, **kw):
    cu = cumulative(lens)
    for s, n in enumerate(lens):
        if n:
            check(got[cu[s]:cu[s + 1]],
                  reference(cache, rows[s], q[cu[s]:cu[s + 1]], starts[s], 1 / math.sqrt(q.shape[2]), **kw))
    assert (got[cu[-1]:] == 7.0).all()                       # rows in no sequence


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hkv,d", [(28, 4, 128), (4, 4, 64), (3, 1, 128), (16, 1, 64), (34, 2, 128)])
def test_prompt(KV, code, dtype, h, hkv, d):
    starts, lens = [0, 10, 0, 63, 64, 300, 1], [1, 7, 0, 65, 64, 150, 300]
    cache, rows, q = prompt_case(KV, starts, lens, h, hkv, d, code, dtype, pad=3)
    check_prompt(cache, rows, q, starts, lens, run_prompt(KV, cache, rows, q, starts, lens))


@pytest.mark.parametrize("starts,lens", [([0], [1500]), ([8000], [1]), ([20000], [9]), ([9001], [130]), ([5000, 3], [40, 900])])
@pytest.mark.parametrize("h,hkv", [(28, 4), (8, 8)])
def test_prompt_long(KV, starts, lens, h, hkv):
    cache, rows, q = prompt_case(KV, starts, lens, h, hkv, 128, "int8", torch.float16, seed=1)
    check_prompt(cache, rows, q, starts, lens, run_prompt(KV, cache, rows, q, starts, lens))


def test_prompt_of_more_rows_than_a_join_takes(KV):
    n, at = 66000, [0, 1, 4000, 65535, 65536, 65999]
    cache, rows, q = prompt_case(KV, [0], [n], 1, 1, 64, "int8", torch.float16, seed=9)
    got = run_prompt(KV, cache, rows, q, [0], [n])
    for i in at:
        check(got[i:i + 1], reference(cache, rows[0], q[i:i + 1], i, 1 / 8))


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("code", CODES)
def test_prompt_window_and_sinks(KV, code, window, sinks):
    starts, lens = [0, 500, 3000], [300, 1, 77]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, code, torch.bfloat16, seed=2)
    got = run_prompt(KV, cache, rows, q, starts, lens, window=window, sinks=sinks)
    check_prompt(cache, rows, q, starts, lens, got, window=window, sinks=sinks)


def test_prompt_unmapped_pages_and_empty_rows(KV):
    starts, lens = [0, 128, 700], [200, 64, 130]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 64, "e4m3", torch.float16, seed=3)
    rows[0][0] = -1                                          # rows 0..63 see nothing
    rows[1][:] = [cache.k.shape[0] + 5] * len(rows[1])
    rows[2][3:9] = [-1] * 6
    got = run_prompt(KV, cache, rows, q, starts, lens)
    check_prompt(cache, rows, q, starts, lens, got)
    assert not got[:64].any() and not got[200:264].any()


def test_prompt_ignores_what_lies_behind_a_chunk(KV):
    starts, lens = [0, 100], [70, 30]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, "e4m3", torch.float16, seed=4)
    want = run_prompt(KV, cache, rows, q, starts, lens)
    for s, n in enumerate((70, 130)):
        bits(cache.k)[rows[s][n // PAGE], :, n % PAGE:] = 0x7f
        bits(cache.v)[rows[s][n // PAGE], :, :, n % PAGE:] = 0xff
    assert torch.equal(run_prompt(KV, cache, rows, q, starts, lens), want)


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 70), (64, 0), (1, 1)])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("h,hkv,d,dtype", [(28, 4, 128, torch.float16), (8, 4, 64, torch.bfloat16)])
def test_prompt_of_middling_grids(KV, window, sinks, code, h, hkv, d, dtype):
    """Grids between a quarter and all of the chip, odd and even numbers of pages: unmapped pages, dead rows
    full of NaN codes, value scales from page to page, a sequence without rows and rows behind the last."""
    starts, lens = [480, 333, 0, 0, 1000], [500, 130, 0, 190, 65]
    cache, rows, q = prompt_case(KV, starts, lens, h, hkv, d, code, dtype, seed=70, pad=3)
    e = torch.randint(-12, 13, cache.vs.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(71))
    cache.vs.copy_(torch.exp2(e.double() - 6))
    for s, i in ((0, 3), (0, 10), (1, 0), (4, 15)):
        rows[s][i] = -1
    if code == "e4m3":
        for s in (0, 1, 3, 4):
            n = starts[s] + lens[s]
            if n % PAGE:
                bits(cache.k)[rows[s][n // PAGE], :, n % PAGE:] = 0x7f
                bits(cache.v)[rows[s][n // PAGE], :, :, n % PAGE:] = 0xff
    got = run_prompt(KV, cache, rows, q, starts, lens, window=window, sinks=sinks)
    if code == "e4m3":                                       # (the plain form would meet the NaNs)
        dead = bits(cache.v) & 0x7f == 0x7f
        bits(cache.v)[dead] = 0
        bits(cache.k)[bits(cache.k) & 0x7f == 0x7f] = 0
    check_prompt(cache, rows, q, starts, lens, got, window=window, sinks=sinks)


@pytest.mark.parametrize("n", [960, 1000])
def test_prompt_of_a_middling_grid_with_poisoned_pages(KV, n):
    cache, rows, q = prompt_case(KV, [0], [n], 28, 4, 128, "int8", torch.float16, seed=72)
    clean = run_prompt(KV, cache, rows, q, [0], [n])
    for i, t in ((6, cache.ks), (9, cache.vs)):
        old = t[rows[0][i]].clone()
        t[rows[0][i]] = float("nan")
        got = run_prompt(KV, cache, rows, q, [0], [n])
        assert torch.equal(got[:i * PAGE], clean[:i * PAGE]) and got[i * PAGE:].isnan().all()
        t[rows[0][i]] = old


def test_prompt_pages_of_unlike_scales(KV):
    starts, lens = [0, 400], [300, 100]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, "int8", torch.bfloat16, seed=5)
    cache.vs.copy_(torch.exp2(torch.randint(-40, 41, cache.vs.shape, device=DEV).double()))
    for i in (rows[0][0], rows[1][3]):
        cache.vs[i], cache.ks[i] = 0.0, 0.0
        bits(cache.k)[i], bits(cache.v)[i] = 0, 0
    check_prompt(cache, rows, q, starts, lens, run_prompt(KV, cache, rows, q, starts, lens))


def test_prompt_a_poisoned_page_reaches_only_rows_that_see_it(KV):
    starts, lens = [0], [300]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, "int8", torch.float16, seed=6)
    cache.vs[rows[0][2], 0] = float("nan")                   # positions 128..191
    got = run_prompt(KV, cache, rows, q, starts, lens)
    assert got[:128].isfinite().all() and got[128:, :4].isnan().all() and got[:, 4:].isfinite().all()


@pytest.mark.parametrize("cu", [[0, -2 ** 31, 70, 100], [2 ** 31 - 1, 0, 50, 100], [90, 20, 60, 2 ** 31 - 1]])
def test_segments_out_of_order(KV, cu):
    """Nothing out of range is touched, and what is in a segment that makes sense is right."""
    g = torch.Generator(device=DEV).manual_seed(19)
    cache, rows, q = prompt_case(KV, [0, 0, 0], [100, 100, 100], 8, 2, 64, "int8", torch.float16, seed=19)
    q, out = q[:100], torch.full_like(q[:100], 7.0)
    x = torch.randn(100, 2, 64, device=DEV, generator=g)
    k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    KV.kv8_attn_prompt(q, cache, ints(rows), ints([0, 0, 0]), ints(cu), out, 1 / 8)
    KV.kv8_read(cache, ints(rows), ints([0, 0, 0]), ints(cu), k, v)
    for s in range(3):
        a, b = max(cu[s], 0), min(cu[s + 1], 100)
        if a < b and sorted(cu)[2:] == cu[2:] and s == 2:
            check(out[a:b], reference(cache, rows[s], q[a:b], 0, 1 / 8))
    before = clone(KV, cache)
    KV.kv8_append(cache, x, x, ints(rows), ints([0, 0, 0]), ints(cu), q=q.float(), q_out=out)
    spare = [i for i in range(cache.k.shape[0]) if i not in {i for r in rows for i in r}]
    assert torch.equal(bits(cache.k)[spare], bits(before.k)[spare])


def test_prompt_bad_segments_are_left_alone(KV):
    starts, lens = [0, 64, 0], [50, 20, 30]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, "int8", torch.float16, seed=7)
    out = torch.full_like(q, 7.0)
    KV.kv8_attn_prompt(q, cache, ints(rows), ints([0, -3, 0]), ints([0, 50, 70, 5000]), out, 1 / math.sqrt(128))
    check(out[:50], reference(cache, rows[0], q[:50], 0, 1 / math.sqrt(128)))
    assert (out[50:70] == 7.0).all()                         # a negative start: no rows
    check(out[70:], reference(cache, rows[2], q[70:], 0, 1 / math.sqrt(128)))   # cut at the last row


def test_prompt_strides_and_alignments(KV):
    starts, lens = [5, 0], [60, 90]
    cache, rows, q = prompt_case(KV, starts, lens, 8, 2, 128, "int8", torch.float16, seed=8)
    want = run_prompt(KV, cache, rows, q, starts, lens)
    wide = torch.zeros(8, 150, 133, device=DEV, dtype=q.dtype)
    wide[..., 3:131] = q.transpose(0, 1)
    out = torch.zeros(150, 8, 130, device=DEV, dtype=q.dtype)
    KV.kv8_attn_prompt(wide.transpose(0, 1)[..., 3:131], cache, ints(rows), ints(starts), ints(cumulative(lens)),
                       out[..., 1:129], 1 / math.sqrt(128))
    assert torch.equal(out[..., 1:129], want) and not out[..., 0].any() and not out[..., 129].any()


# ------------------------------------------------------------------------------------------------ append
def rotated(x, pos, cos, sin):
    """fp32, each operation rounded: the definition."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].float(), x[..., h:].float()
    c, s = cos[pos][:, None], sin[pos][:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def tables(n, d):
    inv = 1.0 / (1.0e4 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


def plain_append(cache, code, kn, vn, rows, starts, lens):
    """The definition, page by page (kn / vn fp32, rotated)."""
    at = 0
    pool = cache.k.shape[0]
    for row, start, n in zip(rows, starts, lens):
        for j in range(start // PAGE, (start + n - 1) // PAGE + 1 if n else 0):
            low, high = max(start, j * PAGE), min(start + n, (j + 1) * PAGE)
            i = row[j] if j < len(row) else -1
            if not 0 <= i < pool:
                continue
            r0, r1 = low - j * PAGE, high - j * PAGE
            src = slice(at + low - start, at + high - start)
            for c, sc, x in ((cache.k, cache.ks, kn[src].transpose(0, 1)),
                             (cache.v, cache.vs, vn[src].permute(1, 2, 0))):
                page = c[i].float() if c is cache.k else c[i].float().transpose(1, 2)
                x = x if c is cache.k else x.transpose(1, 2)      # [Hkv, rows, D]
                own = scale_of(x.abs().amax((1, 2)), code)
                old = sc[i].double() if r0 else torch.zeros_like(own)
                new = torch.maximum(own, old)
                ratio = torch.where(new > 0, old / new, 0.0)[:, None, None]
                page = page.double() * ratio
                page = page.round() if code == "int8" else page.float().to(torch.float8_e4m3fn).double()
                if not r0:
                    page = (c[i].double() if c is cache.k else c[i].double().transpose(1, 2))
                page[:, r0:r1] = to_codes(x, new[:, None, None], code).double()
                page = page if c is cache.k else page.transpose(1, 2)
                c[i] = page.to(c.dtype)
                sc[i] = new.float()
        at += n


def clone(KV, c):
    return KV.KV8Cache(*(t.clone() for t in c))


def live_equal(a, b, rows, starts, lens):
    """Codes of all live positions and scales of all pages."""
    assert torch.equal(a.ks, b.ks) and torch.equal(a.vs, b.vs)
    for row, start, n in zip(rows, starts, lens):
        for j, i in enumerate(row):
            top = min(PAGE, start + n - j * PAGE)
            if 0 <= i < a.k.shape[0] and top > 0:
                assert torch.equal(bits(a.k)[i, :, :top], bits(b.k)[i, :, :top]), (j, i)
                assert torch.equal(bits(a.v)[i, :, :, :top], bits(b.v)[i, :, :, :top]), (j, i)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [0.02, 1.0, 300.0])
def test_append(KV, code, dtype, d, size):
    g = torch.Generator(device=DEV).manual_seed(20)
    starts, lens = [0, 5, 63, 64, 100, 127, 0, 130], [1, 1, 3, 64, 200, 1, 0, 62]
    ends = [a + b for a, b in zip(starts, lens)]
    hkv, h, n = 3, 6, sum(lens)
    pool = sum(-(-e // PAGE) for e in ends) + 1
    cache = random_cache(KV, pool, hkv, d, code, g)
    rows = table_of(ends, 6, pool, 1)
    x = (torch.randn(n + 2, h + 2 * hkv, d, device=DEV, generator=g) * size).to(dtype)
    q, k, v = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
    cos, sin = tables(6 * PAGE, d)
    want, before = clone(KV, cache), clone(KV, cache)
    pos = torch.cat([torch.arange(s, s + m) for s, m in zip(starts, lens)]).to(DEV)
    plain_append(want, code, rotated(k[:n], pos, cos, sin), v[:n].float(), rows, starts, lens)
    q_out = torch.full((n + 2, h, d), 7.0, device=DEV, dtype=torch.float16 if dtype == torch.float32 else dtype)
    KV.kv8_append(cache, k, v, ints(rows), ints(starts), ints(cumulative(lens)), cos, sin, q=q, q_out=q_out)
    live_equal(cache, want, rows, starts, lens)
    assert torch.equal(q_out[:n], rotated(q[:n], pos, cos, sin).to(q_out.dtype)) and (q_out[n:] == 7.0).all()
    spare = [i for i in range(pool) if i not in {x for r in rows for x in r}]
    for i in spare:
        assert all(torch.equal(bits(a[i:i + 1].contiguous()), bits(b[i:i + 1].contiguous())) for a, b in zip(cache, before))


@pytest.mark.parametrize("code", CODES)
def test_append_token_by_token_stays_near_the_whole(KV, code):
    """A page grown token by token (its scale grows with it) against the same rows at once: int8 is at
    most one step of the last scale off (1/2 + 1/4 + ... by growth, 1/2 for the last), e4m3 half a
    subnormal step for each growth."""
    g = torch.Generator(device=DEV).manual_seed(21)
    d, hkv, n = 128, 2, 100
    x = torch.randn(n, 2 * hkv, d, device=DEV, generator=g) * torch.logspace(-2, 2, n, device=DEV)[:, None, None]
    one, all_ = (KV.KV8Cache.empty(2, hkv, d, CODES[code], DEV) for _ in range(2))
    rows = ints([[1, 0]])
    for i in range(n):
        KV.kv8_append(one, x[i:i + 1, :hkv], x[i:i + 1, hkv:], rows, ints([i]), ints([0, 1]))
    KV.kv8_append(all_, x[:, :hkv], x[:, hkv:], rows, ints([0]), ints([0, n]))
    assert torch.equal(one.ks, all_.ks) and torch.equal(one.vs, all_.vs)
    out = [[torch.empty(n, hkv, d, device=DEV) for _ in range(2)] for _ in range(2)]
    for c, (ko, vo) in zip((one, all_), out):
        KV.kv8_read(c, rows, ints([0]), ints([0, n]), ko, vo)
    for a, b, s, y in ((out[0][0], out[1][0], one.ks, x[:, :hkv]), (out[0][1], out[1][1], one.vs, x[:, hkv:])):
        step = s[[1] * PAGE + [0] * (n - PAGE)][..., None]
        if code == "int8":
            assert ((a - y).abs() <= step * 1.001).all() and ((b - y).abs() <= step * 0.501).all()
        else:                                                # 2^-4 of the value, subnormal steps of 2^-9
            assert ((b - y).abs() <= y.abs() * 2 ** -4 + step * 2 ** -10).all()
            assert ((a - y).abs() <= y.abs() * 2 ** -4 + step * 2 ** -9).all()


def test_append_again_from_the_middle(KV):
    """A sequence cut back and continued: the page keeps its earlier rows, the dead ones are replaced."""
    g = torch.Generator(device=DEV).manual_seed(22)
    x, y = (torch.randn(150, 2, 64, device=DEV, generator=g) for _ in range(2))
    cache = KV.KV8Cache.empty(4, 2, 64, torch.int8, DEV)
    rows = [[2, 0, 3]]
    want = clone(KV, cache)
    KV.kv8_append(cache, x, x, ints(rows), ints([0]), ints([0, 150]))
    KV.kv8_append(cache, y[:9], y[:9], ints(rows), ints([70]), ints([0, 9]))
    plain_append(want, "int8", x, x, rows, [0], [150])
    plain_append(want, "int8", y[:9], y[:9], rows, [70], [9])
    live_equal(cache, want, rows, [70], [9])


def test_append_zeros_and_tiny_values(KV):
    cache = KV.KV8Cache.empty(2, 1, 64, torch.int8, DEV)
    z = torch.zeros(3, 1, 64, device=DEV)
    rows = ints([[1, 0]])
    KV.kv8_append(cache, z, z, rows, ints([0]), ints([0, 3]))
    assert cache.ks[1, 0] == 0 and cache.vs[1, 0] == 0 and not cache.k.any()
    tiny = torch.full((1, 1, 64), 1e-40, device=DEV)
    KV.kv8_append(cache, tiny, z[:1] + 5, rows, ints([3]), ints([0, 1]))
    assert cache.ks[1, 0] == 2.0 ** -100 and not cache.k.any()
    out = torch.empty(4, 1, 64, device=DEV), torch.empty(4, 1, 64, device=DEV)
    KV.kv8_read(cache, rows, ints([0]), ints([0, 4]), *out)
    assert not out[0].any() and not out[1][:3].any() and (out[1][3] == 5).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_a_non_finite_value_poisons_its_block(KV, code, bad):
    g = torch.Generator(device=DEV).manual_seed(23)
    x = torch.randn(70, 2, 64, device=DEV, generator=g)
    v = x.clone()
    v[10, 1, 5] = bad
    cache = KV.KV8Cache.empty(2, 2, 64, CODES[code], DEV)
    rows = ints([[0, 1]])
    KV.kv8_append(cache, x, v, rows, ints([0]), ints([0, 70]))
    assert cache.vs.isnan().tolist() == [[False, True], [False, False]] and cache.ks.isfinite().all()
    KV.kv8_append(cache, x[:1], x[:1], rows, ints([20]), ints([0, 1]))
    assert bool(cache.vs[0, 1].isnan())                     # still: its earlier rows are
    KV.kv8_append(cache, x[:5], x[:5], rows, ints([0]), ints([0, 5]))
    assert cache.vs.isfinite().all()                        # begun anew


def test_append_unmapped_pages_and_positions_behind_the_table_are_dropped(KV):
    g = torch.Generator(device=DEV).manual_seed(24)
    x = torch.randn(400, 2, 64, device=DEV, generator=g).half()
    cache = random_cache(KV, 4, 2, 64, "int8", g)
    want = clone(KV, cache)
    rows = [[1, -1, 2], [9, 3, 2 ** 31 - 1]]
    starts, lens = [10, 0], [200, 200]
    KV.kv8_append(cache, x, x, ints(rows), ints(starts), ints([0, 200, 400]))
    plain_append(want, "int8", x.float(), x.float(), rows, starts, lens)
    live_equal(cache, want, rows, starts, lens)
    assert torch.equal(cache.k[0], want.k[0])
    # all of it behind the table, at a negative start, or in segments that are out of order
    before = clone(KV, cache)
    KV.kv8_append(cache, x, x, ints(rows), ints([192, -1]), ints([0, 200, 400]))
    KV.kv8_append(cache, x, x, ints(rows), ints([0, 2 ** 31 - 1]), ints([300, 200, 400]))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(cache, before))


def test_append_strides_and_in_place_rotation(KV):
    g = torch.Generator(device=DEV).manual_seed(25)
    n, hkv, h, d = 70, 2, 4, 128
    x = torch.randn(n, h + 2 * hkv, d, device=DEV, generator=g).half()
    cos, sin = tables(2 * PAGE, d)
    a, b = (KV.KV8Cache.empty(3, hkv, d, torch.int8, DEV) for _ in range(2))
    q = x[:, :h].clone()
    args = ints([[2, 0]]), ints([3]), ints([0, n]), cos, sin
    KV.kv8_append(a, x[:, h:h + hkv], x[:, h + hkv:], *args, q=x[:, :h], q_out=q)
    odd = torch.zeros(h + 2 * hkv, n, d + 3, device=DEV, dtype=torch.float16)
    odd[..., 1:d + 1] = x.transpose(0, 1)
    view = odd.transpose(0, 1)[..., 1:d + 1]
    KV.kv8_append(b, view[:, h:h + hkv], view[:, h + hkv:], *args, q=view[:, :h], q_out=view[:, :h])
    assert all(torch.equal(bits(s), bits(t)) for s, t in zip(a, b))
    assert torch.equal(view[:, :h], q) and not odd[..., 0].any() and not odd[..., d + 1:].any()


# -------------------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("first", [0, 1, 6, 4099])
def test_append_rows_before_the_first_sequence_are_left_alone(KV, first):
    n, rest, d = 8300, 37, 64                               # enough rows that a wave takes several
    cos, sin = tables(200 * PAGE, d)
    cache = KV.KV8Cache.empty(140, 1, d, torch.int8, DEV)
    g = torch.Generator(device=DEV).manual_seed(50)
    x = torch.randn(n, 4, d, device=DEV, generator=g).half()
    table, out = ints([list(range(135))]), torch.full((n, 2, d), 7.0, device=DEV, dtype=torch.float16)
    KV.kv8_append(cache, x[:, 2:3], x[:, 3:], table, ints([2]), ints([first, n - rest]), cos, sin, q=x[:, :2], q_out=out)
    want, ref = KV.KV8Cache.empty(140, 1, d, torch.int8, DEV), torch.empty_like(out)
    y = x[first:n - rest]
    KV.kv8_append(want, y[:, 2:3], y[:, 3:], table, ints([2]), ints([0, len(y)]), cos, sin, q=y[:, :2], q_out=ref[:len(y)])
    assert torch.equal(out[first:n - rest], ref[:len(y)])
    assert (out[:first] == 7.0).all() and (out[n - rest:] == 7.0).all()
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_read(KV, code, dtype, d):
    g = torch.Generator(device=DEV).manual_seed(30)
    starts, lens = [0, 60, 64, 5, 100], [1, 10, 128, 0, 161]
    ends = [a + b for a, b in zip(starts, lens)]
    pool = sum(-(-e // PAGE) for e in ends) + 1
    cache = random_cache(KV, pool, 3, d, code, g)
    rows = table_of(ends, 5, pool, 2)
    rows[4][2] = -1
    n = sum(lens)
    k, v = (torch.full((n + 1, 3, d), 7.0, device=DEV, dtype=dtype) for _ in range(2))
    KV.kv8_read(cache, ints(rows), ints(starts), ints(cumulative(lens)), k, v)
    cu = cumulative(lens)
    for s in range(5):
        for h in range(3):
            if lens[s]:
                kk, vv, good = dense(cache, rows[s], h, ends[s])
                kk, vv = (torch.where(good[:, None], t, 0.0)[starts[s]:].to(dtype) for t in (kk, vv))
                assert torch.equal(k[cu[s]:cu[s + 1], h], kk) and torch.equal(v[cu[s]:cu[s + 1], h], vv)
    assert (k[n:] == 7.0).all() and (v[n:] == 7.0).all()


def test_read_strides(KV):
    g = torch.Generator(device=DEV).manual_seed(31)
    cache = random_cache(KV, 2, 2, 64, "int8", g)
    want = torch.empty(2, 100, 2, 64, device=DEV)
    KV.kv8_read(cache, ints([[1, 0]]), ints([7]), ints([0, 100]), *want)
    odd = torch.zeros(2, 2, 100, 65, device=DEV)
    view = odd.transpose(1, 2)[..., 1:]
    KV.kv8_read(cache, ints([[1, 0]]), ints([7]), ints([0, 100]), view[0], view[1])
    assert torch.equal(view, want) and not odd[..., 0].any()


# ---------------------------------------------------------------------------------------------- together
def serve(KV, cache, rows, x, h, hkv, prompts, steps, d, window=0, sinks=0):
    """Prompts appended and attended, then `steps` tokens each: outputs of all rows, by sequence."""
    cols = len(rows[0])
    cos, sin = tables(cols * PAGE, d)
    table, outs = ints(rows), [[] for _ in prompts]
    q = torch.empty(sum(prompts), h, d, device=DEV, dtype=torch.float16)
    y = torch.empty_like(q)
    flat = torch.cat([x[s][:p] for s, p in enumerate(prompts)])
    start, cu = ints([0] * len(prompts)), ints(cumulative(prompts))
    KV.kv8_append(cache, flat[:, h:h + hkv], flat[:, h + hkv:], table, start, cu, cos, sin, q=flat[:, :h], q_out=q)
    KV.kv8_attn_prompt(q, cache, table, start, cu, y, 1 / math.sqrt(d), window=window, sinks=sinks)
    for s, part in enumerate(y.split(prompts)):
        outs[s].append(part.clone())
    each = ints(list(range(len(prompts) + 1)))
    for t in range(steps):
        pos = ints([p + t for p in prompts])
        row = torch.stack([x[s][p + t] for s, p in enumerate(prompts)])
        q = torch.empty(len(prompts), h, d, device=DEV, dtype=torch.float16)
        o = torch.empty_like(q)
        KV.kv8_append(cache, row[:, h:h + hkv], row[:, h + hkv:], table, pos, each, cos, sin, q=row[:, :h], q_out=q)
        KV.kv8_attn_decode(q, cache, table, pos, o, 1 / math.sqrt(d), window=window, sinks=sinks)
        for s in range(len(prompts)):
            outs[s].append(o[s:s + 1])
    return [torch.cat(o) for o in outs]


@pytest.mark.parametrize("code,bound", [("int8", 0.02), ("e4m3", 0.06)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 4)])
def test_a_run_of_them_together_against_attention_in_64_bits(KV, code, bound, window, sinks):
    """Prompts, then single tokens, against attention over the unrounded keys and values.  What 8 bits
    cost: a code is off by half a step of at most 2 amax / 127 (int8; about 4.5 sigma of normal values
    is 127 to 64 steps, so 0.5 / sqrt(3) / 64 x 4.5 = 2 % of sigma at the worst, 1 % in the middle) or
    2^-4 / sqrt(3) of the value's own binade (e4m3: below 3.6 % of each).  Keys enter through scores of
    size |q| |k| / sqrt(D) ~ 1, so outputs are off by about that share of the values' spread twice
    over, in the root mean square."""
    g = torch.Generator(device=DEV).manual_seed(40)
    h, hkv, d, steps = 8, 2, 128, 40
    prompts = [1, 130, 50, 200]
    x = [torch.randn(p + steps, h + 2 * hkv, d, device=DEV, generator=g) for p in prompts]
    ends = [p + steps for p in prompts]
    pool = sum(-(-e // PAGE) for e in ends)
    cache = KV.KV8Cache.empty(pool, hkv, d, CODES[code], DEV)
    rows = table_of(ends, 4, pool, 4)
    got = serve(KV, cache, rows, x, h, hkv, prompts, steps, d, window, sinks)
    cos, sin = tables(4 * PAGE, d)
    err = norm = 0.0
    for s, e in enumerate(ends):
        p = torch.arange(e, device=DEV)
        q, k, v = rotated(x[s][:, :h], p, cos, sin).double(), rotated(x[s][:, h:h + hkv], p, cos, sin).double(), x[s][:, h + hkv:].double()
        seen = p[None] <= p[:, None]
        if window:
            seen &= (p[None] > p[:, None] - window) | (p[None] < sinks)
        for i in range(h):
            w = torch.softmax((q[:, i] @ k[:, i * hkv // h].t() / math.sqrt(d)).masked_fill(~seen, -math.inf), -1)
            err += float((got[s][:, i].double() - w @ v[:, i * hkv // h]).square().sum())
            norm += float((w @ v[:, i * hkv // h].abs()).square().sum())
    assert math.sqrt(err / norm) < bound


def test_captured_calls_replay_with_new_contents(KV):
    """Append and both attentions in two graphs over their own scratch, replayed between eager work with
    other positions, tables and rows; each replay equals the eager calls."""
    g = torch.Generator(device=DEV).manual_seed(41)
    h, hkv, d, s = 28, 4, 128, 4
    pool, cols = 60, 40
    cos, sin = tables(cols * PAGE, d)
    base = random_cache(KV, pool, hkv, d, "int8", g)
    cache = clone(KV, base)
    x = torch.randn(s, h + 2 * hkv, d, device=DEV, generator=g).half()
    table, pos = torch.zeros(s, cols, dtype=torch.int32, device=DEV), torch.zeros(s, dtype=torch.int32, device=DEV)
    each = ints(list(range(s + 1)))
    q, o, o2 = (torch.empty(s, h, d, device=DEV, dtype=torch.float16) for _ in range(3))

    def step():
        KV.kv8_append(cache, x[:, h:h + hkv], x[:, h + hkv:], table, pos, each, cos, sin, q=x[:, :h], q_out=q)
        KV.kv8_attn_decode(q, cache, table, pos, o, 0.08)

    def other():
        KV.kv8_attn_prompt(q, cache, table, pos, each, o2, 0.08)

    def fill(seed):
        r = torch.Generator().manual_seed(seed)
        order = torch.randperm(pool, generator=r).tolist()
        lens = [[1, 700, 1500, 64], [900, 30, 2, 2000], [2500, 5, 64, 65]][seed % 3]
        rows, at = [], 0
        for n in lens:
            need = -(-n // PAGE)
            rows.append(order[at:at + need] + [-1] * (cols - need))
            at += need
        table.copy_(ints(rows))
        pos.copy_(ints([n - 1 for n in lens]))
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        for a, b in zip(cache, base):
            bits(a).copy_(bits(b))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), other()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, f in zip(graphs, (step, other)):
        with torch.cuda.graph(graph):
            f()
    for seed in (1, 2, 3, 4):
        fill(seed)
        step(), other()
        want = [t.clone() for t in (q, o, o2, *cache)]
        torch.cuda.synchronize()
        fill(seed)
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(bits(a.contiguous()), bits(b.contiguous())) for a, b in zip((q, o, o2, *cache), want))


def test_calls_on_their_own_streams(KV):
    cache, rows, q, pos = decode_case(KV, [3000, 4000], 28, 4, 128, "int8", torch.float16, seed=42)
    want = run_decode(KV, cache, rows, q, pos)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], [torch.empty_like(q) for _ in range(3)]
    table = ints(rows)
    torch.cuda.synchronize()
    for _ in range(5):
        for st, out in zip(streams, outs):
            with torch.cuda.stream(st):
                KV.kv8_attn_decode(q, cache, table, pos, out, 1 / math.sqrt(128))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
