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

Both attentions take a sliding window and a number of first positions that stay visible (sinks): the
query at position p sees key j when ``j <= p and (window == 0 or j > p - window or j < sinks)``.  A row
that sees nothing is zero.

Ragged sequences: ``cu`` (int32 [S + 1]) has the first row of each sequence, ``start`` (int32 [S]) its
first position; rows at or behind ``cu[S]`` belong to none and their outputs stay as they were.  Lengths,
positions and tables are read on the GPU: a captured graph replays with new ones.

Same conventions as ``llm_kernels.py``: raw device pointers, torch's current stream of the tensors'
device, and no fallback.  Scratch memory comes from torch's allocator at each call, so concurrent calls
and captured graphs never share it.
"""
from __future__ import annotations

import ctypes
import threading
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from .kernels import library

PAGE = 64

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_I32, _F32 = torch.int32, torch.float32

_declared = False
_lock = threading.Lock()


def _lib():
    global _declared
    lib = library()
    if not _declared:
        with _lock:
            vp, ci, cl, cf = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
            pool = [vp] * 5 + [ci] * 6
            lib.amdk8s_llm_kv8_append.argtypes = pool + [vp, vp, ci, ci] + [vp, cl, cl] * 4 \
                + [ci, vp, vp, ci, ci, ci, vp]
            lib.amdk8s_llm_kv8_append.restype = ci
            lib.amdk8s_llm_kv8_read.argtypes = pool + [vp, vp, ci, ci] + [vp, cl, cl] * 2 + [ci, vp]
            lib.amdk8s_llm_kv8_read.restype = ci
            lib.amdk8s_llm_kv8_decode_work.argtypes = [ci] * 8
            lib.amdk8s_llm_kv8_decode_work.restype = cl
            lib.amdk8s_llm_kv8_decode.argtypes = pool + [vp, cl, cl, vp, ci, ci, ci, ci, ci, cf, vp, cl,
                                                         cl, ci, vp, vp, vp, vp, cl, vp]
            lib.amdk8s_llm_kv8_decode.restype = ci
            lib.amdk8s_llm_kv8_prompt_work.argtypes = [ci] * 8
            lib.amdk8s_llm_kv8_prompt_work.restype = cl
            lib.amdk8s_llm_kv8_prompt.argtypes = pool + [vp, vp, ci, ci, vp, cl, cl, ci, ci, ci, ci, cf,
                                                         vp, cl, cl, ci, vp, cl, vp]
            lib.amdk8s_llm_kv8_prompt.restype = ci
            _declared = True
    return lib


class KV8Cache(NamedTuple):
    """A pool of pages.  Codes are int8 or e4m3; ``ks`` / ``vs`` are powers of two: the least that bring
    the block's largest magnitude to at most 127 (int8) or 448 (e4m3), 0 for an all-zero block and NaN
    for one that got a non-finite value (what reads it is NaN until the page is begun anew)."""
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
    """Checked cache and table -> (device, Hkv, D, columns, the C arguments of both)."""
    k, v, ks, vs = cache
    dev = k.device
    if k.dim() != 4 or k.dtype not in _CODES or v.dtype != k.dtype or k.shape[2] != PAGE \
            or k.shape[3] not in (64, 128) or v.shape != (k.shape[0], k.shape[1], k.shape[3], PAGE) \
            or not k.is_contiguous() or not v.is_contiguous():
        _bad(what, f"cache codes k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype} are not "
                   f"contiguous [pages, Hkv, {PAGE}, D] and [pages, Hkv, D, {PAGE}] of int8 or "
                   f"float8_e4m3fn with D 64 or 128")
    n, hkv, _, d = k.shape
    if n < 1 or hkv < 1:
        _bad(what, f"an empty cache {tuple(k.shape)}")
    for s in (ks, vs):
        if s.dtype != _F32 or s.shape != (n, hkv) or not s.is_contiguous() or s.device != dev:
            _bad(what, f"scales must be contiguous fp32 [{n}, {hkv}] on {dev}")
    if v.device != dev:
        _bad(what, f"the cache must lie on one device, not {dev} / {v.device}")
    if pages.dtype != _I32 or pages.dim() != 2 or pages.shape[0] < 1 or pages.shape[1] < 1 \
            or pages.stride(1) != 1 or pages.stride(0) < 0 or pages.device != dev:
        _bad(what, f"the page table must be int32 [S, columns] with a unit inner stride on {dev}")
    return dev, hkv, d, pages.shape[1], (
        k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages.data_ptr(), n, hkv, d,
        _CODES[k.dtype], pages.shape[1], pages.stride(0))


def _ints(what: str, name: str, t: torch.Tensor, n: int, dev) -> int:
    if t.dtype != _I32 or t.shape != (n,) or t.device != dev or (n > 1 and t.stride(0) != 1):
        _bad(what, f"{name} must be contiguous int32 [{n}] on {dev}")
    return t.data_ptr()


def _rows(what: str, name: str, t: torch.Tensor, heads: int, d: int, dev) -> Tuple[int, int, int]:
    """A [rows, heads, D] view with a unit inner stride -> (pointer, row stride, head stride)."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != d or t.stride(2) != 1 or t.device != dev:
        _bad(what, f"{name} {tuple(t.shape)} / {t.stride()} on {t.device} is not [rows, {heads}, {d}] "
                   f"with a unit inner stride on {dev}")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _gpu(what: str, dev) -> None:
    if dev.type != "cuda":
        _bad(what, f"the tensors lie on {dev}: the kernels run on a GPU only")


def _launch(what: str, dev, fn, *args) -> None:
    if dev.index is not None and dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        raise RuntimeError(f"amdk8s_llm_{what} failed (rc={rc})")


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
    appended position of a page is dead.  A page must be appended to by one sequence of a call only
    (shared prefix pages are for reading)."""
    what = "kv8_append"
    dev, hkv, d, columns, pool = _pool(what, cache, pages)
    n, s = k.shape[0], pages.shape[0]
    kp = _rows(what, "k", k, hkv, d, dev)
    vp = _rows(what, "v", v, hkv, d, dev)
    if k.dtype not in _TYPES or v.dtype != k.dtype or v.shape[0] != n:
        _bad(what, f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} must have one shape and "
                   f"one type of fp16, bf16, fp32")
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    if (cos_t is None) != (sin_t is None) or (q is None) != (q_out is None):
        _bad(what, "cos_t goes with sin_t, and q with q_out")
    tables = (None, None, 0)
    if cos_t is not None:
        for t in (cos_t, sin_t):
            if t.dtype != _F32 or t.dim() != 2 or t.shape[1] != d // 2 or t.shape[0] < columns * PAGE \
                    or not t.is_contiguous() or t.device != dev or t.data_ptr() % 16:
                _bad(what, f"rotation tables must be contiguous fp32 [>= {columns * PAGE}, {d // 2}] on "
                           f"{dev}, 16-byte aligned")
        tables = (cos_t.data_ptr(), sin_t.data_ptr(), min(cos_t.shape[0], sin_t.shape[0]))
    qp = op = (None, 0, 0)
    heads, otype = 0, _TYPES[k.dtype] if k.dtype != _F32 else 0
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        qp, op = _rows(what, "q", q, heads, d, dev), _rows(what, "q_out", q_out, heads, d, dev)
        if q.dtype != k.dtype or q.shape[0] != n or q_out.shape[0] != n or heads < 1 \
                or q_out.dtype not in (torch.float16, torch.bfloat16) or (q.dtype != _F32 and q_out.dtype != q.dtype):
            _bad(what, f"q {tuple(q.shape)} {q.dtype} / q_out {tuple(q_out.shape)} {q_out.dtype} must have "
                       f"k's rows and type, q_out 16 bits")
        otype = _TYPES[q_out.dtype]
    _gpu(what, dev)
    if n == 0:
        return
    _launch(what, dev, _lib().amdk8s_llm_kv8_append, *pool, starts, cus, s, n, *kp, *vp, *qp, *op, heads,
            *tables, _TYPES[k.dtype], otype)


def kv8_read(cache: Sequence[torch.Tensor], pages: torch.Tensor, start: torch.Tensor, cu: torch.Tensor,
             k_out: torch.Tensor, v_out: torch.Tensor) -> None:
    """Cached positions as values: position ``start[s] + i`` of sequence s into row ``cu[s] + i`` of
    ``k_out`` / ``v_out`` [N, Hkv, D] (fp16, bf16 or fp32; bf16 and fp32 hold them exactly).  Positions of
    unmapped pages read as zeros."""
    what = "kv8_read"
    dev, hkv, d, _, pool = _pool(what, cache, pages)
    n, s = k_out.shape[0], pages.shape[0]
    kp, vp = _rows(what, "k_out", k_out, hkv, d, dev), _rows(what, "v_out", v_out, hkv, d, dev)
    if k_out.dtype not in _TYPES or v_out.dtype != k_out.dtype or v_out.shape[0] != n:
        _bad(what, f"k_out {tuple(k_out.shape)} {k_out.dtype} and v_out {tuple(v_out.shape)} {v_out.dtype} "
                   f"must have one shape and one type of fp16, bf16, fp32")
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    _gpu(what, dev)
    if n == 0:
        return
    _launch(what, dev, _lib().amdk8s_llm_kv8_read, *pool, starts, cus, s, n, *kp, *vp, _TYPES[k_out.dtype])


def _attention(what, q, out, hkv, d, dev, columns, span, window, sinks):
    heads = q.shape[1] if q.dim() == 3 else 0
    if heads < 1 or heads % hkv:
        _bad(what, f"q {tuple(q.shape)}: heads must be a multiple of the cache's {hkv}")
    qp = _rows(what, "q", q, heads, d, dev)
    if q.dtype not in (torch.float16, torch.bfloat16):
        _bad(what, f"q is {q.dtype}: fp16 or bf16")
    op = (None, 0, 0)
    if out is not None:
        op = _rows(what, "out", out, heads, d, dev)
        if out.dtype != q.dtype or out.shape[0] != q.shape[0]:
            _bad(what, f"out {tuple(out.shape)} {out.dtype} must have q's shape and type")
    most = columns * PAGE
    span = most if span == 0 else span
    if not 0 < span <= most:
        _bad(what, f"span {span} is not in 1 .. {most} (the table's positions)")
    if not 0 <= window <= 1 << 30 or not 0 <= sinks <= 1 << 30:
        _bad(what, f"window {window} and sinks {sinks} must be in 0 .. 2^30")
    return heads, qp, op, span


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
    dev, hkv, d, columns, pool = _pool(what, cache, pages)
    heads, qp, op, span = _attention(what, q, out, hkv, d, dev, columns, span, window, sinks)
    s = q.shape[0]
    if pages.shape[0] != s:
        _bad(what, f"{s} rows of q, {pages.shape[0]} of the page table")
    if s > 65535:
        _bad(what, f"{s} sequences: at most 65535 in a call")
    at = _ints(what, "pos", pos, s, dev)
    q8 = (None, None, None)
    if q8_out is not None:
        x8, dx, sx = q8_out
        k = heads * d
        for t, dt, m in ((x8, torch.int8, k), (dx, _F32, k // 32), (sx, _F32, k // 16)):
            if t.dtype != dt or t.shape != (s, m) or not t.is_contiguous() or t.device != dev:
                _bad(what, f"q8_out must be contiguous int8 [{s}, {k}], fp32 [{s}, {k // 32}] and fp32 "
                           f"[{s}, {k // 16}]")
        q8 = (x8.data_ptr(), dx.data_ptr(), sx.data_ptr())
    elif out is None:
        _bad(what, "neither out nor q8_out")
    _gpu(what, dev)
    if s == 0:
        return
    lib = _lib()
    need = lib.amdk8s_llm_kv8_decode_work(s, heads, hkv, d, span, window, sinks, q8_out is not None)
    work = torch.empty(need, dtype=_F32, device=dev) if need else None
    _launch(what, dev, lib.amdk8s_llm_kv8_decode, *pool, *qp, at, s, heads, span, window, sinks, float(scale),
            *op, _TYPES[q.dtype], *q8, work.data_ptr() if need else None, need)


def kv8_attn_prompt(q: torch.Tensor, cache: Sequence[torch.Tensor], pages: torch.Tensor, start: torch.Tensor,
                    cu: torch.Tensor, out: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                    span: int = 0) -> None:
    """Causal attention of prompt chunks: row ``cu[s] + i`` of ``q`` / ``out`` [N, H, D] (fp16 or bf16, any
    row and head strides) is position ``start[s] + i`` of sequence s; its chunk's keys are in the cache
    already (:func:`kv8_append`).  ``span`` as for :func:`kv8_attn_decode`."""
    what = "kv8_attn_prompt"
    dev, hkv, d, columns, pool = _pool(what, cache, pages)
    heads, qp, op, span = _attention(what, q, out, hkv, d, dev, columns, span, window, sinks)
    n, s = q.shape[0], pages.shape[0]
    starts, cus = _ints(what, "start", start, s, dev), _ints(what, "cu", cu, s + 1, dev)
    if n * heads > 1 << 30:
        _bad(what, f"{n} rows x {heads} heads: at most 2^30 in a call")
    _gpu(what, dev)
    if n == 0:
        return
    lib = _lib()
    need = lib.amdk8s_llm_kv8_prompt_work(n, s, heads, hkv, d, span, window, sinks)
    work = torch.empty(need, dtype=_F32, device=dev) if need else None
    _launch(what, dev, lib.amdk8s_llm_kv8_prompt, *pool, starts, cus, s, n, *qp, heads, span, window, sinks,
            float(scale), *op, _TYPES[q.dtype], work.data_ptr() if need else None, need)
