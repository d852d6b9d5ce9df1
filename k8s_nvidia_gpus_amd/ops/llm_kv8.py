"""Paged KV cache in 8 bits and the attention that reads it (``csrc/llm_kv8.hip``).

The cache is a pool of pages of 64 positions (``PAGE``), every KV head in each; a page and head has one
key scale and one value scale (:class:`KV8Cache`).  A sequence is a row of a page table (int32
[S, columns]): column ``j`` holds the page of positions 64 j .. 64 j + 63, and an entry outside the pool
(-1) is an unmapped page: nothing is written there and its positions are not attended, so the pages that
a sliding window has left behind can be freed.

* :func:`kv8_append` — new keys (rotated on the way) and values of ragged sequences into the cache, and
  the rotated queries;
* :func:`kv8_read` — cached positions back as values;
* :func:`kv8_attn_decode` — attention of one token for each sequence;
* :func:`kv8_attn_prompt` — causal attention of ragged prompt chunks.

A decode step is fastest with a sequence's pages in no order: where they follow one another and sequences start
at multiples of 2 MB, all parts of the launch stream in step (8 sequences at 32000 positions 54 to 62 us
instead of 50).  How many sequences a step has, and its ``span``, decide how a row's pages are cut into sums:
outputs depend on them in the last bits.

An int8 key shares its step with its page and head: 1/127 to 2/127 of the largest channel.  Where a few key
channels are far larger than the others (a key bias), the others lose: attention over random keys is off by
2.1 % (rms) without such channels, 3.6 % with one of 10, 11 % of 30 and 26 % of 100 times the others' spread.
e4m3 keeps 3.6 % whatever their size.

Both attentions take a sliding window and a number of first positions that stay visible (sinks): the
query at position p sees key j when ``j <= p and (window == 0 or j > p - window or j < sinks)``.  A row
that sees nothing is zero.  Softmax weights are rounded to fp16 after the value scales have been put on
them: a weight times its page's value scale loses up to 2^-11 of itself, and where it is 2^-32 or less of the
largest weight times the largest value scale that the row sees, it adds nothing to the output.

Ragged sequences: ``cu`` (int32 [S + 1]) has the first row of each sequence, ``start`` (int32 [S]) its
first position; rows at or behind ``cu[S]`` belong to none and their outputs stay as they were.  Lengths,
positions and tables are read on the GPU: a captured graph replays with new ones.

Same conventions as ``llm_kernels.py``: raw device pointers, torch's current stream of the tensors'
device, and no fallback.  Scratch memory comes from torch's allocator at each call, so concurrent calls
and captured graphs never share it.
"""
from __future__ import annotations

import ctypes
import struct
import threading
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from .kernels import library

PAGE = 64

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_QTYPES = {torch.float16: 0, torch.bfloat16: 1}
_I32, _F32 = torch.int32, torch.float32

# The C entries take one record of 64-bit fields (the structs of csrc/llm_kv8.hip): the page pool, the
# segments, then the call's own.
_APPEND = struct.Struct("33q")
_READ = struct.Struct("22q")
_ATTN = struct.Struct("29q")
_NONE = (0, 0, 0)

_entries = None
_lock = threading.Lock()


def _lib():
    global _entries
    if _entries is None:
        with _lock:
            lib = library()
            vp, ci, cl, cf = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
            for name in ("append", "read"):
                f = getattr(lib, f"amdk8s_llm_kv8_{name}")
                f.argtypes, f.restype = [ctypes.c_char_p, vp], ci
            for name in ("decode", "prompt"):
                f = getattr(lib, f"amdk8s_llm_kv8_{name}")
                f.argtypes, f.restype = [ctypes.c_char_p, cf, vp, cl, vp], ci
                f = getattr(lib, f"amdk8s_llm_kv8_{name}_work")
                f.argtypes, f.restype = [ctypes.c_char_p], cl
            if lib.amdk8s_llm_kv8_page() != PAGE:
                raise RuntimeError(f"llm_kv8: the kernel library's pages have {lib.amdk8s_llm_kv8_page()} "
                                   f"positions, not {PAGE}: built from other sources")
            _entries = lib
    return _entries


class KV8Cache(NamedTuple):
    """A pool of pages.  Codes are int8 or e4m3; ``ks`` / ``vs`` are powers of two: the least that bring
    the block's largest magnitude to at most 127 (int8) or 448 (e4m3), 0 for an all-zero block and NaN
    for one that got a non-finite value (what reads it is NaN until the page is begun anew).  The codes of
    appended positions are finite; the attentions count on it."""
    k: torch.Tensor       # codes [pages, Hkv, 64, D]
    v: torch.Tensor       # codes [pages, Hkv, D, 64]
    ks: torch.Tensor      # fp32 [pages, Hkv]
    vs: torch.Tensor      # fp32 [pages, Hkv]

    @staticmethod
    def empty(pages: int, kv_heads: int, head_dim: int = 128, dtype: torch.dtype = torch.int8,
              device="cuda") -> "KV8Cache":
        if dtype not in _CODES or head_dim not in (64, 128) or pages < 1 or kv_heads < 1:
            raise ValueError(f"KV8Cache: {pages} pages x {kv_heads} heads x {head_dim} of {dtype}: codes "
                             f"are int8 or float8_e4m3fn, head_dim 64 or 128")
        z = torch.zeros(2, pages, kv_heads, PAGE * head_dim, dtype=torch.uint8, device=device)
        s = torch.zeros(2, pages, kv_heads, dtype=_F32, device=device)
        return KV8Cache(z[0].view(pages, kv_heads, PAGE, head_dim).view(dtype),
                        z[1].view(pages, kv_heads, head_dim, PAGE).view(dtype), s[0], s[1])


def _bad(what: str, why: str):
    raise ValueError(f"{what}: {why}")


def _pool(what: str, cache: Sequence[torch.Tensor], pages: torch.Tensor):
    """Checked cache and table -> (device index, Hkv, D, sequences, columns, the record's fields)."""
    k, v, ks, vs = cache
    shape, kind = k.shape, k.dtype
    code = _CODES.get(kind)
    if code is None or len(shape) != 4 or v.dtype is not kind or shape[2] != PAGE \
            or shape[3] not in (64, 128) or v.shape != (shape[0], shape[1], shape[3], PAGE) \
            or not k.is_contiguous() or not v.is_contiguous() or shape[0] < 1 or shape[1] < 1:
        _bad(what, f"cache codes k {tuple(shape)} {kind}, v {tuple(v.shape)} {v.dtype} are not "
                   f"contiguous [pages, Hkv, {PAGE}, D] and [pages, Hkv, D, {PAGE}] of int8 or "
                   f"float8_e4m3fn with D 64 or 128")
    n, hkv, _, d = shape
    dev, each = k.get_device(), (n, hkv)
    if ks.dtype is not _F32 or ks.shape != each or not ks.is_contiguous() or ks.get_device() != dev \
            or vs.dtype is not _F32 or vs.shape != each or not vs.is_contiguous() or vs.get_device() != dev:
        _bad(what, f"scales must be contiguous fp32 [{n}, {hkv}] on {k.device}")
    if v.get_device() != dev:
        _bad(what, f"the cache must lie on one device, not {k.device} / {v.device}")
    table, strides = pages.shape, pages.stride()
    if pages.dtype is not _I32 or len(table) != 2 or table[0] < 1 or table[1] < 1 or strides[1] != 1 \
            or pages.get_device() != dev:
        _bad(what, f"the page table must be int32 [S, columns] with a unit inner stride on {k.device}")
    return dev, hkv, d, table[0], table[1], (
        k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages.data_ptr(), n, hkv, d,
        code, table[1], strides[0])


def _ints(what: str, name: str, t: torch.Tensor, n: int, dev: int) -> int:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous() or t.get_device() != dev:
        _bad(what, f"{name} must be contiguous int32 [{n}] on the cache's device")
    return t.data_ptr()


def _rows(what: str, name: str, t: torch.Tensor, n: int, heads: int, d: int, dev: int) -> Tuple[int, int, int]:
    """A [n, heads, D] view with a unit inner stride -> (pointer, row stride, head stride)."""
    strides = t.stride()
    if t.shape != (n, heads, d) or strides[2] != 1 or t.get_device() != dev:
        _bad(what, f"{name} {tuple(t.shape)} / {strides} on {t.device} is not [{n}, {heads}, {d}] with a "
                   f"unit inner stride on the cache's device")
    return t.data_ptr(), strides[0], strides[1]


def _out_rows(what: str, name: str, t: torch.Tensor, n: int, heads: int, d: int, dev: int) -> Tuple[int, int, int]:
    """`_rows` of an output: its rows must not share memory (an expanded view would)."""
    rows = _rows(what, name, t, n, heads, d, dev)
    _, row, head = rows
    if head >= d and row >= heads * head:
        return rows
    if (heads > 1 and head < d) or (n > 1 and row < d) \
            or (n > 1 and heads > 1 and row < (heads - 1) * head + d and head < (n - 1) * row + d):
        _bad(what, f"{name} {tuple(t.shape)} / {t.stride()}: its rows overlap")
    return rows


def _gpu(what: str, dev: int) -> None:
    if dev < 0:
        _bad(what, "the tensors are not on a GPU, and the kernels run nowhere else")


def _launch(what: str, dev: int, fn, *args) -> None:
    if dev != torch._C._cuda_getDevice():                # (a tensor there: the runtime is up)
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        raise RuntimeError(f"{what} failed (rc={rc})")


def kv8_append(cache: Sequence[torch.Tensor], k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor,
               start: torch.Tensor, cu: torch.Tensor, cos_t: Optional[torch.Tensor] = None,
               sin_t: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> None:
    """Rows of ``k`` / ``v`` [N, Hkv, D] (fp16, bf16 or fp32; any row and head strides) into the cache:
    row ``cu[s] + i`` goes to position ``start[s] + i`` of sequence s (row s of ``pages``).

    ``cos_t`` / ``sin_t`` (fp32 [positions, D / 2]): the keys are rotated by their positions (NeoX pairs
    i, i + D / 2) in fp32, and so is ``q`` [N, H, D] into ``q_out`` (fp16 or bf16; of q's type unless q
    is fp32; may be q itself).  Without tables nothing is rotated.

    A page that is begun (its first position is among the rows) takes the rows' own scale; one that was
    begun before keeps the larger scale, its earlier codes shifted to it.  What lies behind the last
    appended position of a page is dead.  What lies behind the table is dropped.  A page must be appended
    to by one sequence of a call only (shared prefix pages are for reading), and a page that is entered
    behind its first position must have scales (zeros, if nothing was written: :meth:`KV8Cache.empty`)."""
    what = "kv8_append"
    dev, hkv, d, s, columns, pool = _pool(what, cache, pages)
    kind = k.dtype
    if kind not in _TYPES or v.dtype != kind:
        _bad(what, f"k is {kind}, v {v.dtype}: one type of fp16, bf16, fp32")
    n = k.shape[0] if k.dim() == 3 else -1
    kp, vp = _rows(what, "k", k, n, hkv, d, dev), _rows(what, "v", v, n, hkv, d, dev)
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    if (cos_t is None) != (sin_t is None) or (q is None) != (q_out is None):
        _bad(what, "cos_t goes with sin_t, and q with q_out")
    turn = _NONE
    if cos_t is not None:
        size = cos_t.shape
        if len(size) != 2 or size[0] < columns * PAGE or size[1] != d // 2 or sin_t.shape != size \
                or cos_t.dtype != _F32 or sin_t.dtype != _F32 or not cos_t.is_contiguous() \
                or not sin_t.is_contiguous() or cos_t.get_device() != dev or sin_t.get_device() != dev:
            _bad(what, f"rotation tables must be contiguous fp32 [>= {columns * PAGE}, {d // 2}] on the "
                       f"cache's device")
        turn = (cos_t.data_ptr(), sin_t.data_ptr(), size[0])
        if (turn[0] | turn[1]) & 15:
            _bad(what, "rotation tables must be 16-byte aligned")
    qp = op = _NONE
    heads, otype = 0, kind
    if q is not None:
        heads, otype = q.shape[1] if q.dim() == 3 and q.shape[1] else -1, q_out.dtype
        if q.dtype != kind or otype not in _QTYPES or (kind != _F32 and otype != kind):
            _bad(what, f"q is {q.dtype}, q_out {otype}: q of k's type ({kind}), q_out the same, or fp16 or "
                       f"bf16 for fp32")
        qp, op = _rows(what, "q", q, n, heads, d, dev), _out_rows(what, "q_out", q_out, n, heads, d, dev)
    _gpu(what, dev)
    if n:
        _launch(what, dev, _lib().amdk8s_llm_kv8_append,
                _APPEND.pack(*pool, starts, cus, s, n, *kp, *vp, *qp, *op, heads, *turn, _TYPES[kind],
                             _QTYPES.get(otype, 0)))


def kv8_read(cache: Sequence[torch.Tensor], pages: torch.Tensor, start: torch.Tensor, cu: torch.Tensor,
             k_out: torch.Tensor, v_out: torch.Tensor) -> None:
    """Cached positions as values: position ``start[s] + i`` of sequence s into row ``cu[s] + i`` of
    ``k_out`` / ``v_out`` [N, Hkv, D] (fp16, bf16 or fp32; bf16 and fp32 hold them exactly).  Positions of
    unmapped pages read as zeros."""
    what = "kv8_read"
    dev, hkv, d, s, _, pool = _pool(what, cache, pages)
    kind, n = k_out.dtype, k_out.shape[0] if k_out.dim() == 3 else -1
    if kind not in _TYPES or v_out.dtype != kind:
        _bad(what, f"k_out is {kind}, v_out {v_out.dtype}: one type of fp16, bf16, fp32")
    kp, vp = _out_rows(what, "k_out", k_out, n, hkv, d, dev), _out_rows(what, "v_out", v_out, n, hkv, d, dev)
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    _gpu(what, dev)
    if n:
        _launch(what, dev, _lib().amdk8s_llm_kv8_read,
                _READ.pack(*pool, starts, cus, s, n, *kp, *vp, _TYPES[kind]))


def _attention(what, q, out, hkv, d, dev, columns, span, window, sinks):
    """Checked query and output rows -> (rows, heads, span, the record's fields of q, of out, type)."""
    shape, kind = q.shape, q.dtype
    if len(shape) != 3 or shape[1] < 1 or shape[1] % hkv:
        _bad(what, f"q {tuple(shape)}: [rows, heads, D], heads a multiple of the cache's {hkv}")
    if kind not in _QTYPES:
        _bad(what, f"q is {kind}: fp16 or bf16")
    n, heads, _ = shape
    qp, op = _rows(what, "q", q, n, heads, d, dev), _NONE
    if out is not None:
        if out.dtype != kind:
            _bad(what, f"out is {out.dtype}, q {kind}")
        op = _out_rows(what, "out", out, n, heads, d, dev)
    most = columns * PAGE
    span = span or most
    if not 0 < span <= most:
        _bad(what, f"span {span} is not in 1 .. {most} (the table's positions)")
    if not 0 <= window <= 1 << 30 or not 0 <= sinks <= 1 << 30:
        _bad(what, f"window {window} and sinks {sinks} must be in 0 .. 2^30")
    return n, heads, span, qp, op, _QTYPES[kind]


def _attend(what, dev, size, run, record, scale) -> None:
    need = size(record)
    if need:
        if need < 0:
            raise RuntimeError(f"{what} failed (bad arguments)")
        work = torch.empty(need, dtype=_F32, device=torch.device("cuda", dev))
        _launch(what, dev, run, record, scale, work.data_ptr(), need)
    else:
        _launch(what, dev, run, record, scale, None, 0)


def kv8_attn_decode(q: torch.Tensor, cache: Sequence[torch.Tensor], pages: torch.Tensor, pos: torch.Tensor,
                    out: Optional[torch.Tensor], scale: float, window: int = 0, sinks: int = 0,
                    span: int = 0, q8_out: Optional[Sequence[torch.Tensor]] = None) -> None:
    """Attention of one token for each sequence: ``q`` / ``out`` [S, H, D] (fp16 or bf16, any row and head
    strides), the query of sequence s at position ``pos[s]`` (int32 [S]; its own key is in the cache
    already; -1: a padded row, zeros).

    ``span``: keys at or behind it are not attended (0: the table's end); a bound near the longest
    sequence saves empty workgroups.  ``q8_out`` = (x8, dx, sx): the output as Q8 rows as well (int8
    [S, H D], a scale for each 32 and the scaled sum of each 16: the quantised GEMV's input); ``out`` may
    then be None. """
    what = "kv8_attn_decode"
    dev, hkv, d, s, columns, pool = _pool(what, cache, pages)
    n, heads, span, qp, op, kind = _attention(what, q, out, hkv, d, dev, columns, span, window, sinks)
    if n != s or s > 65535:
        _bad(what, f"{n} rows of q, {s} of the page table: as many, and at most 65535")
    at = _ints(what, "pos", pos, s, dev)
    q8 = _NONE
    if q8_out is not None:
        x8, dx, sx = q8_out
        k = heads * d
        for t, dt, m in ((x8, torch.int8, k), (dx, _F32, k // 32), (sx, _F32, k // 16)):
            if t.dtype != dt or t.shape != (s, m) or not t.is_contiguous() or t.get_device() != dev:
                _bad(what, f"q8_out must be contiguous int8 [{s}, {k}], fp32 [{s}, {k // 32}] and fp32 "
                           f"[{s}, {k // 16}]")
        q8 = (x8.data_ptr(), dx.data_ptr(), sx.data_ptr())
    elif out is None:
        _bad(what, "neither out nor q8_out")
    _gpu(what, dev)
    lib = _lib()
    _attend(what, dev, lib.amdk8s_llm_kv8_decode_work, lib.amdk8s_llm_kv8_decode,
            _ATTN.pack(*pool, at, 0, s, s, *qp, *op, heads, span, window, sinks, kind, *q8), scale)


def kv8_attn_prompt(q: torch.Tensor, cache: Sequence[torch.Tensor], pages: torch.Tensor, start: torch.Tensor,
                    cu: torch.Tensor, out: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                    span: int = 0) -> None:
    """Causal attention of prompt chunks: row ``cu[s] + i`` of ``q`` / ``out`` [N, H, D] (fp16 or bf16, any
    row and head strides) is position ``start[s] + i`` of sequence s; its chunk's keys are in the cache
    already (:func:`kv8_append`).  ``span`` as for :func:`kv8_attn_decode`."""
    what = "kv8_attn_prompt"
    dev, hkv, d, s, columns, pool = _pool(what, cache, pages)
    n, heads, span, qp, op, kind = _attention(what, q, out, hkv, d, dev, columns, span, window, sinks)
    if out is None:
        _bad(what, "no out")
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    if n * heads > 1 << 30:
        _bad(what, f"{n} rows x {heads} heads: at most 2^30 in a call")
    _gpu(what, dev)
    if n:
        lib = _lib()
        _attend(what, dev, lib.amdk8s_llm_kv8_prompt_work, lib.amdk8s_llm_kv8_prompt,
                _ATTN.pack(*pool, starts, cus, s, n, *qp, *op, heads, span, window, sinks, kind, 0, 0, 0), scale)
