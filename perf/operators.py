"""Cases of the operators on the 8-bit paged KV cache (``k8s_nvidia_gpus_amd.ops.llm_kv8``).

The cache holds pages of 64 positions: key codes ``k`` [pages, Hkv, 64, D], value codes ``v``
[pages, Hkv, D, 64] (int8 or e4m3) and one scale for each page and head, ``ks`` / ``vs`` [pages, Hkv],
a power of two.  A sequence owns a row of the page table; an entry of -1 is a page that is not mapped.

* ``append``: rotated keys and values of new tokens go into the cache (and the queries are rotated);
  the pages that they touch are then read back as values, which is what the pass returns.
* ``read``: cached positions as bf16 keys and values.
* ``decode``: attention of one new token for each sequence.
* ``prompt``: attention of chunks of prompt tokens of several sequences.

The decoder's sizes are Qwen2.5-7B's (28 query heads, 4 key heads of 128, contexts of 4096 and 32768);
the others are generic.
"""
import math
import random

import torch

own = False

PAGE = 64
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------------------------------- cases
def listed():
    m = dict(heads=28, kv_heads=4, dim=128)
    return [
        # one decode step of four chat slots at contexts up to 4096: the smallest append
        dict(m, name="append step 4 int8", op="append", seqs=4, new=1, past=4000, code="int8", type="fp32"),
        # a large serving batch: 64 sequences, a token each
        dict(name="append step 64 e4m3", op="append", seqs=64, new=1, past=8000, heads=32, kv_heads=8,
             dim=128, code="e4m3", type="bf16"),
        # prompts of several slots in one batch, each continuing behind a cached prefix (odd lengths)
        dict(m, name="append prompt 8x2048 int8", op="append", seqs=8, new=2048, past=1500, code="int8",
             type="fp16"),
        # a slot's cached prefix read back, and a batch of long ones
        dict(m, name="read 1x2000 int8", op="read", seqs=1, past=2000, code="int8"),
        dict(m, name="read 8x16384 e4m3", op="read", seqs=8, past=16384, code="e4m3"),
        # single stream chat at a short context: latency counts
        dict(m, name="decode 1x500 int8", op="decode", seqs=1, past=500, code="int8", type="fp16",
             window=0, sinks=0),
        # eight slots of ragged lengths up to the server's default context
        dict(m, name="decode 8x4096 int8", op="decode", seqs=8, past=4096, code="int8", type="fp16",
             window=0, sinks=0),
        # full 32k contexts of eight slots: the largest cache read
        dict(m, name="decode 8x32768 e4m3", op="decode", seqs=8, past=32768, code="e4m3", type="bf16",
             window=0, sinks=0),
        # streaming generation: a window and four sink tokens, pages between them already freed
        dict(name="decode 32x16000 window", op="decode", seqs=32, past=16000, heads=32, kv_heads=8,
             dim=128, code="int8", type="bf16", window=4000, sinks=4),
        # ragged short prompts and continuations of several slots, rows of padding behind them
        dict(m, name="prompt 6x300 ragged", op="prompt", seqs=6, new=300, past=700, pad=37, code="int8",
             type="fp16", window=0, sinks=0),
        # one 512-token chunk at the end of a 32k prompt: few rows, many keys
        dict(m, name="prompt 512 at 31488", op="prompt", seqs=1, new=512, past=31488, pad=0, code="e4m3",
             type="fp16", window=0, sinks=0),
        # a whole prompt of 8192 tokens: the most work
        dict(m, name="prompt 8192 at 0", op="prompt", seqs=1, new=8192, past=0, pad=0, code="int8",
             type="bf16", window=0, sinks=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]),
                code=rng.choice(["int8", "e4m3"]))
    if op == "append":
        new = rng.choice([1, _log(rng, 1, 2048)])
        rows = 16384 * 28 // case["heads"]
        return dict(case, seqs=min(_log(rng, 1, 64), max(1, min(16384, rows) // new)), new=new,
                    past=_log(rng, 1, 4000), type=rng.choice(["fp32", "fp16", "bf16"]))
    if op == "read":
        past = _log(rng, 1, 16384)
        return dict(case, seqs=min(_log(rng, 1, 32), max(1, 8 * 16384 * 4 // (past * kv_heads))), past=past)
    case = dict(case, type=rng.choice(["fp16", "bf16"]), window=0, sinks=0)
    if rng.random() < 0.4:
        case = dict(case, window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 64, 100]))
    if op == "decode":
        past = _log(rng, 1, 32768)
        return dict(case, seqs=min(_log(rng, 1, 64), max(1, 8 * 32768 * 4 // (past * kv_heads))), past=past)
    new = _log(rng, 1, 4096)
    past = rng.choice([0, _log(rng, 1, 8192)])
    most = 28 * 8192 * 8192 // 4
    while new * (new + past) * case["heads"] > most:
        new, past = (new + 1) // 2, past // 2
    seqs = max(1, min(_log(rng, 1, 8), most // (new * (new + past) * case["heads"])))
    return dict(case, seqs=seqs, new=new, past=past, pad=rng.choice([0, 0, 1, 50]))


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Cached and new positions of each sequence (the case fixes them): the first has the case's own,
    the others down to half as many."""
    rng = random.Random("%(op)s %(seqs)d %(past)d" % case)
    past, new = [case["past"]], [case.get("new", 0)]
    for _ in range(case["seqs"] - 1):
        past.append(case["past"] - rng.randrange(case["past"] // 2 + 1))
        new.append(max(1, new[0] - rng.randrange(new[0] // 2 + 1)) if "new" in case else 0)
    return past, new


def _page_scale(amax, code):
    """The least power of two s with amax <= qmax s (0 for amax 0)."""
    mant, expo = torch.frexp(amax)
    top = QMAX[code] / 2.0 ** (7 if code == "int8" else 9)
    expo = expo - (7 if code == "int8" else 9) + (mant > top).int()
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), expo.clamp(-100, 120)), 0.0)


def _codes(x, scale, code):
    y = x * torch.where(scale > 0, 1 / scale, 0.0)
    return y.round().to(torch.int8) if code == "int8" else y.to(torch.float8_e4m3fn)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dim, kv_heads, heads = "cuda", case["dim"], case["kv_heads"], case["heads"]
    past, new = _lengths(case)
    seqs = len(past)
    ends = [p + n for p, n in zip(past, new)]
    width = max(1, -(-max(ends) // PAGE))
    need = [-(-e // PAGE) for e in ends]
    pool = sum(need) + 3

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    # keys with channels of unlike sizes and values with pages of unlike sizes, as projections give them
    channel = torch.exp(0.5 * randn(kv_heads, 1, dim))
    k = randn(pool, kv_heads, PAGE, dim) * channel
    ks = _page_scale(k.abs().amax((2, 3)), case["code"])
    k = _codes(k, ks[:, :, None, None], case["code"])
    v = randn(pool, kv_heads, dim, PAGE) * torch.exp(randn(pool, kv_heads, 1, 1))
    vs = _page_scale(v.abs().amax((2, 3)), case["code"])
    v = _codes(v, vs[:, :, None, None], case["code"])

    order, at = list(range(pool)), 0
    rng.shuffle(order)
    table = []
    for n, p in zip(need, past):
        row = order[at:at + n] + [-1] * (width - n)
        if case.get("window") and case["op"] == "decode":   # pages that no later token can see
            low, high = -(-case["sinks"] // PAGE), max(0, p - case["window"] - 1) // PAGE
            row[low:high] = [-1] * max(0, high - low)
        at += n
        table.append(row)
    cu = [0]
    for n in new if "new" in case else [0] * seqs:
        cu.append(cu[-1] + n)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    state = dict(case=case, cache=(k, v, ks, vs), pages=ints(table), span=width * PAGE,
                 scale=1.0 / math.sqrt(dim))
    if case["op"] == "append":
        t = TYPES[case["type"]]
        # q | k | v rows of one projection, as the decoder's product leaves them
        qkv = (randn(cu[-1], heads + 2 * kv_heads, dim)).to(t)
        state.update(q=qkv[:, :heads], k_new=qkv[:, heads:heads + kv_heads], v_new=qkv[:, heads + kv_heads:])
        state["q_out"] = torch.empty(cu[-1], heads, dim, device=dev,
                                     dtype=torch.float16 if t == torch.float32 else t)
        inv = 1.0 / (1.0e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim))
        angle = torch.arange(width * PAGE, dtype=torch.float64, device=dev)[:, None] * inv
        state.update(cos=angle.cos().float(), sin=angle.sin().float(), start=ints(past), cu=ints(cu))
        # the pages that the new tokens touch, and from where they are read back
        begin = [p // PAGE * PAGE for p in past]
        back = [0]
        for b, e in zip(begin, ends):
            back.append(back[-1] + e - b)
        state.update(read_start=ints(begin), read_cu=ints(back), read_rows=back[-1])
        state["touched"] = torch.tensor(sorted({table[s][j] for s in range(seqs)
                                                for j in range(past[s] // PAGE, need[s])}), device=dev)
    elif case["op"] == "read":
        back = [0]
        for p in past:
            back.append(back[-1] + p)
        state.update(read_start=ints([0] * seqs), read_cu=ints(back), read_rows=back[-1])
    elif case["op"] == "decode":
        state.update(q=(1.5 * randn(seqs, heads, dim)).to(TYPES[case["type"]]), pos=ints([p - 1 for p in past]))
        state["out"] = torch.empty_like(state["q"])
    else:
        rows = cu[-1] + case["pad"]
        state.update(q=(1.5 * randn(rows, heads, dim)).to(TYPES[case["type"]]), start=ints(past), cu=ints(cu),
                     most=max(new))
        state["out"] = torch.full_like(state["q"], 0.25)       # rows behind the last chunk stay as they are
    if "read_rows" in state:
        for name in ("k_out", "v_out"):
            state[name] = torch.empty(state["read_rows"], kv_heads, dim, device=dev, dtype=torch.bfloat16)
    return state


# -------------------------------------------------------------------------------------- plain forms
def _rows(start, cu, count):
    """Sequence and position of each of `count` rows (rows behind the last sequence: sequence S - 1)."""
    row = torch.arange(count, device=cu.device)
    seq = (torch.searchsorted(cu.long(), row, right=True) - 1).clamp(0, start.numel() - 1)
    return seq, start[seq] + row - cu[seq]


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _grow(codes, scale, values, at, seen, touched, code):
    """Scales of the touched pages once `values` [N, Hkv, D] came in at page indexes `at`; `seen`
    [pages] says which pages hold earlier positions.  Returns the new scales; the pages' earlier codes
    are put into them."""
    new = torch.zeros_like(scale).scatter_reduce(
        0, at[:, None].expand(-1, scale.shape[1]), values.abs().amax(-1), "amax")[touched]
    new = _page_scale(new, code)
    old = torch.where(seen[touched][:, None], scale[touched], 0.0)
    new = torch.maximum(old, new)
    ratio = torch.where(new > 0, old / new, 0.0)[:, :, None, None]
    again = codes.view(torch.uint8)[touched].view(codes.dtype).float() * ratio
    again = again.round().to(torch.int8) if code == "int8" else again.to(codes.dtype)
    codes.view(torch.uint8)[touched] = again.view(torch.uint8)
    scale[touched] = new


def _plain_append(s):
    k, v, ks, vs = s["cache"]
    code = s["case"]["code"]
    seq, pos = _rows(s["start"], s["cu"], s["k_new"].shape[0])
    page, slot = s["pages"][seq, pos // PAGE].long(), pos % PAGE
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["q_out"].copy_(_rotate(s["q"], cos, sin))
    kn, vn = _rotate(s["k_new"], cos, sin), s["v_new"].float()
    first = s["pages"].gather(1, (s["start"] // PAGE)[:, None].long())[:, 0].long()
    seen = torch.zeros(k.shape[0], dtype=torch.bool, device=k.device)
    seen[first] = s["start"] % PAGE > 0
    _grow(k, ks, kn, page, seen, s["touched"], code)
    _grow(v, vs, vn, page, seen, s["touched"], code)
    k.view(torch.uint8)[page, :, slot] = _codes(kn, ks[page][..., None], code).view(torch.uint8)
    v.view(torch.uint8)[page, :, :, slot] = _codes(vn, vs[page][..., None], code).view(torch.uint8)


def _plain_read(s):
    k, v, ks, vs = s["cache"]
    seq, pos = _rows(s["read_start"], s["read_cu"], s["read_rows"])
    page, slot = s["pages"][seq, pos // PAGE].long(), pos % PAGE
    kr = k.view(torch.uint8)[page, :, slot].view(k.dtype).float() * ks[page][..., None]
    vr = v.view(torch.uint8)[page, :, :, slot].view(v.dtype).float() * vs[page][..., None]
    s["k_out"].copy_(kr)
    s["v_out"].copy_(vr)


def _gathered(s):
    """The whole table's keys [S, Hkv, L, D] and values [S, Hkv, D, L] in 32 bits, and which are mapped."""
    k, v, ks, vs = s["cache"]
    table = s["pages"].long()
    at = table.clamp(min=0)
    seqs, width = table.shape
    kk = k.view(torch.uint8)[at].view(k.dtype).float() * ks[at][..., None, None]     # [S, W, Hkv, 64, D]
    vv = v.view(torch.uint8)[at].view(v.dtype).float() * vs[at][..., None, None]     # [S, W, Hkv, D, 64]
    kk = kk.transpose(1, 2).reshape(seqs, k.shape[1], width * PAGE, k.shape[3])
    vv = vv.permute(0, 2, 3, 1, 4).reshape(seqs, k.shape[1], k.shape[3], width * PAGE)
    return kk, vv, (table >= 0).repeat_interleave(PAGE, 1)


def _plain_attention(s, q, pos):
    """q [S, R, H, D] at positions pos [S, R] -> [S, R, H, D] in 32 bits."""
    kk, vv, mapped = _gathered(s)
    seqs, rows, heads, dim = q.shape
    kv_heads = kk.shape[1]
    q = q.float().view(seqs, rows, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(seqs, kv_heads, rows * (heads // kv_heads), dim)
    score = (q @ kk.transpose(2, 3)).mul_(s["scale"])
    j = torch.arange(kk.shape[2], device=q.device)
    seen = (j <= pos[..., None]) & mapped[:, None]
    if s["case"]["window"]:
        seen &= (j > pos[..., None] - s["case"]["window"]) | (j < s["case"]["sinks"])
    score = score.view(seqs, kv_heads, rows, heads // kv_heads, -1)
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = score.sum(-1, keepdim=True)
    o = score.view(seqs, kv_heads, -1, kk.shape[2]) @ vv.transpose(2, 3)
    o = o.view(seqs, kv_heads, rows, heads // kv_heads, dim) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 2, 1, 3, 4).reshape(seqs, rows, heads, dim)


def _plain_decode(s):
    s["out"].copy_(_plain_attention(s, s["q"][:, None], s["pos"][:, None])[:, 0])


def _plain_prompt(s):
    step = torch.arange(s["most"], device=s["q"].device)
    at = (s["cu"][:-1, None] + step).clamp(max=s["q"].shape[0] - 1)
    o = _plain_attention(s, s["q"][at], s["start"][:, None] + step)
    count = s["q"].shape[0]
    seq, pos = _rows(s["start"], s["cu"], count)
    o = o[seq, (pos - s["start"][seq]).clamp(max=s["most"] - 1)].to(s["out"].dtype)
    live = torch.arange(count, device=o.device) < s["cu"][-1]
    s["out"].copy_(torch.where(live[:, None, None], o, s["out"]))


# -------------------------------------------------------------------------------------------- passes
def run(s):
    op, window, sinks = s["case"]["op"], s["case"].get("window", 0), s["case"].get("sinks", 0)
    if own:
        from k8s_nvidia_gpus_amd.ops import llm_kv8 as KV

        if op == "append":
            KV.kv8_append(s["cache"], s["k_new"], s["v_new"], s["pages"], s["start"], s["cu"], s["cos"],
                          s["sin"], q=s["q"], q_out=s["q_out"])
        if op in ("append", "read"):
            KV.kv8_read(s["cache"], s["pages"], s["read_start"], s["read_cu"], s["k_out"], s["v_out"])
        elif op == "decode":
            KV.kv8_attn_decode(s["q"], s["cache"], s["pages"], s["pos"], s["out"], s["scale"],
                               window=window, sinks=sinks)
        else:
            KV.kv8_attn_prompt(s["q"], s["cache"], s["pages"], s["start"], s["cu"], s["out"], s["scale"],
                               window=window, sinks=sinks)
    elif op == "append":
        _plain_append(s)
        _plain_read(s)
    elif op == "read":
        _plain_read(s)
    elif op == "decode":
        _plain_decode(s)
    else:
        _plain_prompt(s)
    if op == "append":
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    return {"k": s["k_out"], "v": s["v_out"]} if op == "read" else s["out"]


# ---------------------------------------------------------------------------------------------- work
def _attended(case):
    """Visible (query, key) pairs and cached positions that any query sees, of all sequences."""
    pairs = seen = 0
    for past, new in zip(*_lengths(case)):
        if "new" not in case:
            past, new = past - 1, 1
        reach = case["window"] + case["sinks"] if case["window"] else past + new
        full = max(0, min(new, reach - past))           # rows that see everything before them
        pairs += full * past + full * (full + 1) // 2 + (new - full) * min(reach, past + new)
        seen += min(past + new, new + reach)
    return pairs, seen


def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    wide = 4 if case.get("type") == "fp32" else 2
    past, new = _lengths(case)
    rows = sum(new) if "new" in case else len(past)
    if case["op"] == "append":
        # in: q, k, v; out: q, codes; then the touched pages' codes in and their values out
        back = sum(p % PAGE + n for p, n in zip(past, new))
        return {"bytes": rows * dim * (wide * (heads + 2 * kv_heads) + 2 * heads + 2 * kv_heads)
                + back * kv_heads * dim * 2 * 3, "flops": 3 * rows * dim * (heads + kv_heads)}
    if case["op"] == "read":
        return {"bytes": sum(past) * kv_heads * dim * 2 * 3, "flops": 0}
    pairs, seen = _attended(case)
    return {"bytes": seen * kv_heads * dim * 2 + rows * heads * dim * 4, "flops": 4 * pairs * heads * dim}


# --------------------------------------------------------------------------------------------- exact
def _value(cache, page, head):
    """A page's keys [64, D] and values [64, D] of one head (or of a list of pages, joined) in 64 bits."""
    k, v, ks, vs = cache
    kk = k.view(torch.uint8)[page, head].view(k.dtype).double() * ks[page, head].double()[:, None, None]
    vv = v.view(torch.uint8)[page, head].view(v.dtype).double() * vs[page, head].double()[:, None, None]
    return kk.reshape(-1, kk.shape[-1]), vv.transpose(1, 2).reshape(-1, kk.shape[-1])


def _exact_attention(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    out = s["out"].double()
    table = s["pages"].tolist()
    if case["op"] == "decode":
        spans = [(i, 1, p) for i, p in enumerate(s["pos"].tolist())]
    else:
        cu = s["cu"].tolist()
        spans = [(cu[i], cu[i + 1] - cu[i], p) for i, p in enumerate(s["start"].tolist())]
    for i, (row, count, pos) in enumerate(spans):
        live = [j for j in range(min(len(table[i]), (pos + count + PAGE - 1) // PAGE)) if table[i][j] >= 0]
        where = torch.tensor(live, device=out.device, dtype=torch.long)
        key_pos = (where[:, None] * PAGE + torch.arange(PAGE, device=out.device)).reshape(-1)
        for h in range(case["kv_heads"]):
            if not live:
                out[row:row + count, h * group:(h + 1) * group] = 0
                continue
            kk, vv = _value(s["cache"], s["pages"][i].long()[where], h)
            for a in range(row, row + count, 2048):           # some rows at a time
                b = min(a + 2048, row + count)
                at = (pos + torch.arange(a - row, b - row, device=out.device))[:, None]
                hidden = key_pos > at
                if case["window"]:
                    hidden |= (key_pos <= at - case["window"]) & (key_pos >= case["sinks"])
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][a:b, g].double() @ kk.t() * s["scale"]
                    x = x.masked_fill(hidden, -math.inf)
                    y = torch.softmax(x, -1)
                    y = torch.where(hidden.all(-1, keepdim=True), 0.0, y)
                    out[a:b, g] = y @ vv
    return out


def _exact_read(s):
    table, cu = s["pages"].tolist(), s["read_cu"].tolist()
    kv_heads, dim = s["case"]["kv_heads"], s["case"]["dim"]
    ko = torch.empty(s["read_rows"], kv_heads, dim, dtype=torch.float64, device="cuda")
    vo = torch.empty_like(ko)
    for i, first in enumerate(s["read_start"].tolist()):
        count = cu[i + 1] - cu[i]
        if not count:
            continue
        ids = table[i][first // PAGE:(first + count - 1) // PAGE + 1]
        for h in range(kv_heads):
            kk, vv = _value(s["cache"], torch.tensor(ids, device="cuda"), h)
            lead = first % PAGE
            ko[cu[i]:cu[i + 1], h], vo[cu[i]:cu[i + 1], h] = kk[lead:lead + count], vv[lead:lead + count]
    return {"k": ko, "v": vo}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        return _exact_read(s)
    if case["op"] in ("decode", "prompt"):
        return _exact_attention(s)
    # append: the rotation in 64 bits; cached values as if nothing were rounded to 8 bits, but for what
    # was in a begun page before (that is in 8 bits already)
    old = _exact_read(s)
    start, cu, back = s["start"].tolist(), s["cu"].tolist(), s["read_cu"].tolist()
    half = case["dim"] // 2
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, first in enumerate(start):
        rows = slice(cu[i], cu[i + 1])
        n = cu[i + 1] - cu[i]
        lead = first % PAGE
        c, t = (s[x][first:first + n].double()[:, None] for x in ("cos", "sin"))
        turned = []
        for x in (s["q"][rows].double(), s["k_new"][rows].double()):
            turned.append(torch.cat([x[..., :half] * c - x[..., half:] * t,
                                     x[..., half:] * c + x[..., :half] * t], -1))
        q[rows] = turned[0]
        at = slice(back[i] + lead, back[i + 1])
        # in 8 bits by the page's scale, each page of the sequence for itself
        for name, x in (("k", turned[1]), ("v", s["v_new"][rows].double())):
            whole = old[name]
            whole[at] = x
            scales = s["cache"][2 if name == "k" else 3]
            page0 = first // PAGE
            for j in range(page0, (first + n - 1) // PAGE + 1):
                low = max(first, j * PAGE)
                high = min(first + n, (j + 1) * PAGE)
                base = back[i] - page0 * PAGE
                fresh = whole[base + low:base + high]
                need = fresh.abs().amax((0, 2)) / QMAX[case["code"]]
                e = torch.ceil(torch.log2(need))
                e = torch.where(torch.exp2(e - 1) >= need, e - 1, e)
                scale = torch.exp2(e)
                if low % PAGE:
                    scale = torch.maximum(scale, scales[s["pages"][i, j].long()].double())
                page = whole[base + j * PAGE:base + high]
                y = page / scale[:, None]
                y = y.round() if case["code"] == "int8" else y.float().to(torch.float8_e4m3fn).double()
                page.copy_(y * scale[:, None])
    return {"q": q, "k": old["k"], "v": old["v"]}
