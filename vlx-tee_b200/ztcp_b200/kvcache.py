"""Operators on the hot side of the paged KV pool: what fills the pages that egress encrypts, reads the pages that
ingress restores, and chooses the pages that leave the pool.

* ``append_tokens``      norms of queries and keys per head, position rotation, K/V into their pool slots
* ``attend_pages``       attention of the sequences' newest tokens (one or a chunk each) over their pages
* ``page_mass``          attention weight of those tokens, accumulated per page
* ``select_cold_pages``  the pages with the least weight -- a block table for ``codec.encode_pages`` -- and the
                         compacted tables of the pages that stay

The pool is the codec's: [pool_pages, T, H, D] contiguous fp16 or bf16, addressed through int32 block tables, one
row per sequence; ``v_pool=None`` is a single-buffer (MLA) pool whose values are columns [rope_dim, D) of K.  Every
operator has a one-shot form and a ``prepare_*`` form that checks and packs the call once (``codec.PreparedCall``);
both enqueue on `stream` (default: the current stream).  Lengths, tables, slots and positions are read on the device at
every call and checked there before they address memory: the int32 status tensor that the calls return holds 0, or
``SEQ_BAD_LENGTH`` / ``SEQ_BAD_BLOCK`` for a sequence (or appended token) that had a bad one.  ``attend_pages``,
``page_mass`` and their ``prepare_*`` forms also check lengths and tables on the host, which waits for the stream;
``check_block_table=False`` leaves that out, and so does a stream that is being captured into a CUDA graph.  Nothing else
synchronizes.  A batch holds at least one sequence, query row or token: an empty one is refused.  The reference has no
operator of this kind (its research/baseline_codec encodes and decodes pages only).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import capi
from .codec import PreparedCall, _on_device, _ptr, _require_cuda, _stream_arg, _stream_handle

SEQ_OK = 0
SEQ_BAD_LENGTH = 5  # ZTCP_SEQ_BAD_LENGTH
SEQ_BAD_BLOCK = 6   # ZTCP_SEQ_BAD_BLOCK
SEQ_TIMEOUT = 7     # ZTCP_SEQ_TIMEOUT: a wait inside the attention kernel did not end; the outputs are not valid

# every symbol include/ztcp_kvcache.h declares
KVCACHE_SYMBOLS = ("ztcp_attend_workspace_bytes", "ztcp_attend_pages", "ztcp_page_mass_workspace_bytes",
                   "ztcp_page_mass", "ztcp_append_tokens", "ztcp_select_cold_pages")

_FLOATS = (torch.float16, torch.bfloat16)


class _Cache(C.Structure):
    _fields_ = [("k_pool", C.c_void_p), ("v_pool", C.c_void_p), ("dtype", C.c_int32), ("reserved", C.c_int32),
                ("geom", capi.Geometry), ("pool_pages", C.c_int64), ("block_tables", C.c_void_p),
                ("table_stride", C.c_int64), ("max_pages", C.c_int64), ("kv_lens", C.c_void_p), ("n_seqs", C.c_int64)]


class _Queries(C.Structure):
    _fields_ = [("q", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("q_starts", C.c_void_p),
                ("total_rows", C.c_int64), ("num_heads", C.c_int64), ("max_q_len", C.c_int64), ("scale", C.c_float),
                ("causal", C.c_int32)]


class _Append(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v")] + [
        (n, C.c_int64) for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride",
                                 "v_token_stride", "v_head_stride")] + [
        (n, C.c_void_p) for n in ("q_out", "k_pool", "v_pool", "slots", "positions", "rope_table", "q_weight",
                                  "k_weight")] + [
        (n, C.c_int64) for n in ("n_tokens", "num_q_heads", "pool_pages", "max_pos")] + [
        ("geom", capi.Geometry), ("dtype", C.c_int32), ("norm_from", C.c_int32), ("interleaved", C.c_int32),
        ("eps", C.c_float)]


class _Selection(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("mass", "block_tables", "kv_lens")] + [
        (n, C.c_int64) for n in ("n_seqs", "max_pages", "page_tokens", "keep", "sink", "recent")] + [
        (n, C.c_void_p) for n in ("cold_blocks", "cold_index", "cold_starts", "kept_tables", "kept_mass", "kept_lens",
                                  "status")]


_lib = None


def _load() -> C.CDLL:
    global _lib
    if _lib is None:
        lib = capi.load()
        vp, i64 = C.c_void_p, C.c_int64
        lib.ztcp_attend_workspace_bytes.restype = i64
        lib.ztcp_attend_workspace_bytes.argtypes = [C.POINTER(_Cache), C.POINTER(_Queries)]
        lib.ztcp_attend_pages.restype = C.c_int32
        lib.ztcp_attend_pages.argtypes = [C.POINTER(_Cache), C.POINTER(_Queries), vp, vp, vp, vp, i64, vp]
        lib.ztcp_page_mass.restype = C.c_int32
        lib.ztcp_page_mass_workspace_bytes.restype = i64
        lib.ztcp_page_mass_workspace_bytes.argtypes = [C.POINTER(_Cache), C.POINTER(_Queries)]
        lib.ztcp_page_mass.argtypes = [C.POINTER(_Cache), C.POINTER(_Queries), vp, vp, C.c_float, vp, vp, vp, i64, vp]
        lib.ztcp_append_tokens.restype = C.c_int32
        lib.ztcp_append_tokens.argtypes = [C.POINTER(_Append), vp, vp]
        lib.ztcp_select_cold_pages.restype = C.c_int32
        lib.ztcp_select_cold_pages.argtypes = [C.POINTER(_Selection), vp]
        _lib = lib
    return _lib


# ---- checks -----------------------------------------------------------------------------------------------------
def _overlap(a: torch.Tensor | None, b: torch.Tensor | None) -> bool:
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _check_disjoint(outputs, inputs) -> None:
    """Every output apart from every input and from the other outputs ((name, tensor or None) pairs)."""
    for i, (name, t) in enumerate(outputs):
        for other, u in (*outputs[i + 1:], *inputs):
            if _overlap(t, u):
                raise RuntimeError(f"{name} must not overlap {other}")


def _check_vector(name, t, n, dtypes, dev) -> None:
    _require_cuda(name, t, dtypes, dev)
    if t.dim() != 1 or t.numel() != n:
        raise RuntimeError(f"{name} must be 1D with {n} entries")


def _check_rows(name, t, dtype, dev, heads=None, dim=None) -> None:
    """[rows, heads, D] whose vectors are contiguous; rows and heads may be strided (a slice of a projection)."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda or (dev is not None and t.get_device() != dev.index):
        raise RuntimeError(f"{name} must be a CUDA tensor" if dev is None or not t.is_cuda else
                           f"{name} must be on {dev}, got {t.device}")
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise RuntimeError(f"{name} must have shape [rows, {heads or 'heads'}, {dim or 'head_dim'}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must have the pool's dtype {dtype}, got {t.dtype}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise RuntimeError(f"{name}'s vectors must be contiguous")
    if t.numel() and any(s % 8 for s in t.stride()[:2]) or t.data_ptr() % 16:
        raise RuntimeError(f"{name} must be 16-byte aligned with strides of multiples of 8 elements")


def _check_pool(k_pool, v_pool) -> torch.device:
    _require_cuda("k_pool", k_pool, _FLOATS)
    if k_pool.dim() != 4:
        raise RuntimeError("k_pool must have shape [pool_pages, num_tokens, num_heads, head_dim]")
    if v_pool is not None:
        _require_cuda("v_pool", v_pool, (k_pool.dtype,), k_pool.device)
        if v_pool.shape != k_pool.shape:
            raise RuntimeError("v_pool shape must match k_pool shape")
    return k_pool.device


def _check_tables(block_tables, kv_lens, pool_pages, page_tokens, check) -> None:
    """Host check of the entries that the lengths reach, at the cost of one synchronizing reduction.  The kernels
    check every entry on the device as well; this turns a bad table into an exception before launch.  A stream that is
    being captured cannot be waited for: there the device's check stands alone."""
    if not check or torch.cuda.is_current_stream_capturing():
        return
    used = (torch.arange(block_tables.shape[1], device=block_tables.device) * page_tokens)[None] < kv_lens[:, None]
    bad = (used & ((block_tables < 0) | (block_tables >= pool_pages))).any()
    bad_len = ((kv_lens < 0) | (kv_lens > block_tables.shape[1] * page_tokens)).any()
    bad, bad_len = torch.stack([bad, bad_len]).tolist()
    if bad_len:
        raise RuntimeError(f"kv_lens entries must lie in [0, {block_tables.shape[1] * page_tokens}]")
    if bad:
        raise RuntimeError(f"block_tables entries must lie in [0, {pool_pages})")


def _dtype(t: torch.Tensor) -> int:
    return capi.DTYPE_BF16 if t.dtype == torch.bfloat16 else capi.DTYPE_F16


def _pack_cache(q, k_pool, v_pool, block_tables, kv_lens, q_starts, max_q_len, rope_dim, scale, causal, check):
    """Checks what attend and page_mass share; returns (device, cache block, query block, kept tensors)."""
    dev = _check_pool(k_pool, v_pool)
    pages, T, H, D = k_pool.shape
    _check_rows("q", q, k_pool.dtype, dev, None, D)
    _require_cuda("block_tables", block_tables, (torch.int32,), dev)
    if block_tables.dim() != 2:
        raise RuntimeError("block_tables must be 2D int32 [sequences, pages]")
    n = block_tables.shape[0]
    _check_vector("kv_lens", kv_lens, n, (torch.int32,), dev)
    if q_starts is not None:
        _check_vector("q_starts", q_starts, n + 1, (torch.int32,), dev)
    elif q.shape[0] != n:
        raise RuntimeError("without q_starts, q must hold one row per sequence")
    _check_tables(block_tables, kv_lens, pages, T, check)
    if max_q_len is None:
        max_q_len = 1 if q_starts is None else max(int(q.shape[0]), 1)
    cache = _Cache(k_pool.data_ptr(), _ptr(v_pool), _dtype(k_pool), 0, capi.geometry(T, H, D, rope_dim, v_pool is None),
                   pages, block_tables.data_ptr(), block_tables.shape[1], block_tables.shape[1], kv_lens.data_ptr(), n)
    queries = _Queries(q.data_ptr(), q.stride(0), q.stride(1), _ptr(q_starts), q.shape[0], q.shape[1], int(max_q_len),
                       D ** -0.5 if scale is None else float(scale), int(bool(causal)))
    return dev, cache, queries, (q, k_pool, v_pool, block_tables, kv_lens, q_starts)


def _status(status, n, dev):
    if status is None:
        return torch.empty(n, dtype=torch.int32, device=dev)
    _check_vector("status", status, n, (torch.int32,), dev)
    return status


def _workspace(size_of, cache, queries, dev) -> torch.Tensor:
    with torch.cuda.device(dev):
        size = size_of(cache, queries)
    if size < 0:
        capi.check(capi.ZTCP_EINVAL)
    return torch.empty(size, dtype=torch.uint8, device=dev)


class _OwningCall(PreparedCall):
    """A prepared call with buffers of its own (workspace, status, new outputs).  They come from the stream that was
    current when it was prepared, where earlier work may still be using the memory, and may be dropped while another
    stream runs it.  So each further stream that it runs on waits for that point once, and the buffers are handed back only
    when all of these streams are done with them."""

    __slots__ = ("_own", "_made", "_streams")

    def __init__(self, fn, args, dev, keep, result, own):
        super().__init__(fn, args, dev, keep, result)
        with torch.cuda.device(dev):
            self._own = own
            self._streams = {_stream_handle(dev)}
            self._made = None
            if not torch.cuda.is_current_stream_capturing():
                self._made = torch.cuda.Event()
                self._made.record()

    def __call__(self, stream=None):
        handle = _stream_arg(self._dev, stream)
        if handle not in self._streams:
            self._meet(handle)
        rc = _on_device(self._dev, self._fn, *self._args, handle)
        if rc != capi.ZTCP_OK:
            capi.check(rc)
        return self._result

    def _meet(self, handle: int) -> None:
        other = torch.cuda.ExternalStream(handle, device=self._dev)
        with torch.cuda.stream(other):
            # (a capture begins behind a synchronization, and cannot wait for work outside itself)
            if self._made is not None and not torch.cuda.is_current_stream_capturing():
                other.wait_event(self._made)
        for t in self._own:
            t.record_stream(other)
        self._streams.add(handle)


def _run_once(prepare, first: torch.Tensor | None, stream, checks: bool = False):
    """Prepares and enqueues a call whose own buffers die with it, on `stream` (None: the current one) of the device of
    `first`, an argument.  On another stream than the current one, all of it happens in that stream's order: the host's
    check reads lengths and tables there, and the buffers are its own.  A call that the host checks also follows what the
    current stream has been given so far (``checks``; its host waits anyhow).  Whatever the call was given may be dropped at
    once, and what it returns is used on the current stream: both are handed back only when both streams are done."""
    if stream is None or not isinstance(first, torch.Tensor) or not first.is_cuda:
        return prepare()(stream)
    dev, handle = first.device, _stream_arg(first.device, stream)
    if handle == _stream_handle(dev):
        return prepare()(handle)
    here, other = torch.cuda.current_stream(dev), torch.cuda.ExternalStream(handle, device=dev)
    with torch.cuda.device(dev):
        if checks and not torch.cuda.is_current_stream_capturing():
            other.wait_stream(here)
    with torch.cuda.stream(other):
        call = prepare()
        result = call(handle)
    for t in call._keep:
        if isinstance(t, torch.Tensor):
            t.record_stream(other)
    for t in (result if isinstance(result, tuple) else (result,)):
        t.record_stream(here)
    return result


# ---- attention --------------------------------------------------------------------------------------------------
def prepare_attend(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor | None, block_tables: torch.Tensor,
                   kv_lens: torch.Tensor, out: torch.Tensor, *, lse: torch.Tensor | None = None,
                   q_starts: torch.Tensor | None = None, max_q_len: int | None = None, rope_dim: int = 0,
                   scale: float | None = None, causal: bool = True, status: torch.Tensor | None = None,
                   check_block_table: bool = True) -> PreparedCall:
    """Attention of packed query rows q [rows, Hq, D] over the sequences' pages, checked and packed once.

    Sequence b owns rows [q_starts[b], q_starts[b + 1]) (default: one row per sequence) and holds kv_lens[b] tokens,
    its query tokens the last of them; with ``causal`` row i sees tokens up to kv_len - q_len + i.  Query head h
    reads KV head h // (Hq // H).  out [rows, Hq, D] (``v_pool=None``: [rows, Hq, D - rope_dim]) gets the outputs,
    lse [rows, Hq] fp32 the natural logarithm of the softmax sums; a row that sees nothing gets 0 and -inf, rows
    behind the last sequence are left as they were.  ``max_q_len`` is the longest q_len to expect (it chooses the
    kernel; any q_len is computed).  K and V rows below kv_lens must be finite.

    Calling the result enqueues the kernels and returns status[n] int32.  The prepared call owns its workspace: run
    one at a time, as with any call that writes the same outputs.
    """
    dev, cache, queries, keep = _pack_cache(q, k_pool, v_pool, block_tables, kv_lens, q_starts, max_q_len, rope_dim,
                                            scale, causal, check_block_table)
    dv = k_pool.shape[3] - (rope_dim if v_pool is None else 0)
    _require_cuda("out", out, (q.dtype,), dev)
    if tuple(out.shape) != (q.shape[0], q.shape[1], dv):
        raise RuntimeError(f"out must have shape {(q.shape[0], q.shape[1], dv)}, got {tuple(out.shape)}")
    if lse is not None:
        _require_cuda("lse", lse, (torch.float32,), dev)
        if tuple(lse.shape) != tuple(q.shape[:2]):
            raise RuntimeError(f"lse must have shape {tuple(q.shape[:2])}, got {tuple(lse.shape)}")
    status = _status(status, kv_lens.numel(), dev)
    _check_disjoint([("out", out), ("lse", lse), ("status", status)],
                    [("q", q), ("k_pool", k_pool), ("v_pool", v_pool), ("block_tables", block_tables),
                     ("kv_lens", kv_lens), ("q_starts", q_starts)])
    lib = _load()
    workspace = _workspace(lib.ztcp_attend_workspace_bytes, cache, queries, dev)
    args = (cache, queries, out.data_ptr(), _ptr(lse), status.data_ptr(), workspace.data_ptr(), workspace.numel())
    return _OwningCall(lib.ztcp_attend_pages, args, dev, (*keep, out, lse, workspace, status), status, (workspace, status))


def attend_pages(q, k_pool, v_pool, block_tables, kv_lens, out, *, stream=None, **kw) -> torch.Tensor:
    """Attention of packed query rows over the sequences' pages, enqueued on `stream` (default: the current
    stream); arguments as for ``prepare_attend``.  Returns status[n] int32 (device)."""
    return _run_once(lambda: prepare_attend(q, k_pool, v_pool, block_tables, kv_lens, out, **kw), k_pool, stream,
                     kw.get("check_block_table", True))


# ---- attention weight per page ----------------------------------------------------------------------------------
def prepare_page_mass(q: torch.Tensor, k_pool: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor,
                      lse: torch.Tensor, mass: torch.Tensor | None, out_mass: torch.Tensor, *, decay: float = 1.0,
                      q_starts: torch.Tensor | None = None, max_q_len: int | None = None, scale: float | None = None,
                      causal: bool = True, status: torch.Tensor | None = None,
                      check_block_table: bool = True) -> PreparedCall:
    """Attention weight of packed query rows per page, checked and packed once:

    out_mass[b, p] = decay * mass[b, p] + sum over the sequence's rows, heads and the tokens of page p that the row
    sees, of exp(scale * q.k - lse); 0 past the last page.  mass and out_mass are [sequences, pages] fp32 like
    block_tables and may be one tensor; ``mass=None`` starts from nothing.  q, lse and the other arguments as
    ``prepare_attend`` takes and writes them; q may be the last rows of a chunk (an observation window) with their
    lse.  Calling the result enqueues the kernels and returns status[n] int32.  The prepared call owns its workspace, as
    ``prepare_attend``'s does."""
    dev, cache, queries, keep = _pack_cache(q, k_pool, None, block_tables, kv_lens, q_starts, max_q_len, 0, scale,
                                            causal, check_block_table)
    _require_cuda("lse", lse, (torch.float32,), dev)
    if tuple(lse.shape) != tuple(q.shape[:2]):
        raise RuntimeError(f"lse must have shape {tuple(q.shape[:2])}, got {tuple(lse.shape)}")
    for name, t in (("mass", mass), ("out_mass", out_mass)):
        if t is not None or name == "out_mass":
            _require_cuda(name, t, (torch.float32,), dev)
            if t.shape != block_tables.shape:
                raise RuntimeError(f"{name} must have block_tables' shape {tuple(block_tables.shape)}")
    status = _status(status, kv_lens.numel(), dev)
    same = mass is not None and mass.data_ptr() == out_mass.data_ptr()
    _check_disjoint([("out_mass", out_mass), ("status", status)],
                    [("q", q), ("k_pool", k_pool), ("block_tables", block_tables), ("kv_lens", kv_lens),
                     ("q_starts", q_starts), ("lse", lse), ("mass", None if same else mass)])
    lib = _load()
    workspace = _workspace(lib.ztcp_page_mass_workspace_bytes, cache, queries, dev)
    args = (cache, queries, lse.data_ptr(), _ptr(mass), float(decay), out_mass.data_ptr(), status.data_ptr(),
            workspace.data_ptr(), workspace.numel())
    return _OwningCall(lib.ztcp_page_mass, args, dev, (*keep, lse, mass, out_mass, workspace, status), status,
                       (workspace, status))


def page_mass(q, k_pool, block_tables, kv_lens, lse, mass, out_mass, *, stream=None, **kw) -> torch.Tensor:
    """Attention weight per page, enqueued on `stream` (default: the current stream); arguments as for
    ``prepare_page_mass``.  Returns status[n] int32 (device)."""
    return _run_once(lambda: prepare_page_mass(q, k_pool, block_tables, kv_lens, lse, mass, out_mass, **kw), k_pool, stream,
                     kw.get("check_block_table", True))


# ---- append -----------------------------------------------------------------------------------------------------
def rope_table(max_pos: int, rope_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """[max_pos, rope_dim] fp32 table of ``append_tokens``: cosines, then sines, of position * base^(-2i / rope_dim);
    angles in 64 bits, since a far position's angle has no fraction left in 32."""
    i = torch.arange(0, rope_dim, 2, device=device, dtype=torch.float64)
    angle = torch.arange(max_pos, device=device, dtype=torch.float64)[:, None] * base ** (-i / rope_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def prepare_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor | None, k_pool: torch.Tensor,
                   v_pool: torch.Tensor | None, slots: torch.Tensor, positions: torch.Tensor | None,
                   rope_table: torch.Tensor | None, q_out: torch.Tensor | None, *,
                   q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, norm_from: int = 0,
                   eps: float = 1e-6, interleaved: bool = False, status: torch.Tensor | None = None) -> PreparedCall:
    """Norm, rotation and append of new tokens, checked and packed once.

    q [n, Hq, D], k and v [n, H, D] may be strided rows (slices of one projection).  With ``q_weight`` / ``k_weight``
    (fp32 [D - norm_from]) each vector's columns [norm_from, D) are divided by their root mean square and multiplied
    by the weight; the leading rope_table.shape[1] columns are then rotated by row positions[i] (int32) of the table
    (see ``rope_table``), halves paired, or neighbours with ``interleaved``.  Queries go to q_out [n, Hq, D]
    (contiguous; may be q itself), keys and values to pool slot slots[i] (int64: page * T + row; -1: not written).
    Slots must be distinct.  Calling the result enqueues the kernel and returns status[n] int32: SEQ_BAD_BLOCK where
    a position lies outside the table (nothing written) or a slot outside the pool (only the query written)."""
    dev = _check_pool(k_pool, v_pool)
    pages, T, H, D = k_pool.shape
    _check_rows("k", k, k_pool.dtype, dev, H, D)
    n = k.shape[0]
    if (v is None) != (v_pool is None):
        raise RuntimeError("v must be given exactly when v_pool is")
    if (q is None) != (q_out is None):
        raise RuntimeError("q_out must be given exactly when q is")
    if v is not None:
        _check_rows("v", v, k_pool.dtype, dev, H, D)
    if q is not None:
        _check_rows("q", q, k_pool.dtype, dev, None, D)
        _require_cuda("q_out", q_out, (k_pool.dtype,), dev)
        if q_out.shape != q.shape:
            raise RuntimeError("q_out shape must match q shape")
    if any(t is not None and t.shape[0] != n for t in (q, v)):
        raise RuntimeError("q, k and v must hold the same number of rows")
    _check_vector("slots", slots, n, (torch.int64,), dev)
    R, max_pos = 0, 0
    if rope_table is not None:
        _require_cuda("rope_table", rope_table, (torch.float32,), dev)
        if rope_table.dim() != 2:
            raise RuntimeError("rope_table must have shape [max_pos, rope_dim]")
        max_pos, R = rope_table.shape
        if positions is None:
            raise RuntimeError("a rotation needs positions")
        _check_vector("positions", positions, n, (torch.int32,), dev)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _check_vector(name, w, D - norm_from, (torch.float32,), dev)
    status = _status(status, n, dev)
    in_place = q is not None and q.data_ptr() == q_out.data_ptr() and q.stride() == q_out.stride()
    _check_disjoint([("k_pool", k_pool), ("v_pool", v_pool), ("q_out", q_out), ("status", status)],
                    [("q", None if in_place else q), ("k", k), ("v", v), ("slots", slots), ("positions", positions),
                     ("rope_table", rope_table), ("q_weight", q_weight), ("k_weight", k_weight)])
    rows = lambda t: (0, 0) if t is None else (t.stride(0), t.stride(1))  # noqa: E731
    block = _Append(_ptr(q), k.data_ptr(), _ptr(v), *rows(q), *rows(k), *rows(v), _ptr(q_out), k_pool.data_ptr(),
                    _ptr(v_pool), slots.data_ptr(), _ptr(positions), _ptr(rope_table), _ptr(q_weight), _ptr(k_weight),
                    n, 0 if q is None else q.shape[1], pages, max_pos, capi.geometry(T, H, D, R, v_pool is None),
                    _dtype(k_pool), int(norm_from), int(bool(interleaved)), float(eps))
    keep = (q, k, v, k_pool, v_pool, slots, positions, rope_table, q_out, q_weight, k_weight, status)
    return _OwningCall(_load().ztcp_append_tokens, (block, status.data_ptr()), dev, keep, status, (status,))


def append_tokens(q, k, v, k_pool, v_pool, slots, positions, rope_table, q_out, *, stream=None, **kw) -> torch.Tensor:
    """Norm, rotation and append of new tokens, enqueued on `stream` (default: the current stream); arguments as
    for ``prepare_append``.  Returns status[n] int32 (device)."""
    return _run_once(lambda: prepare_append(q, k, v, k_pool, v_pool, slots, positions, rope_table, q_out, **kw), k_pool, stream)


# ---- eviction ---------------------------------------------------------------------------------------------------
class ColdSelection(NamedTuple):
    """Outputs of ``select_cold_pages`` (device tensors)."""

    cold_blocks: torch.Tensor  # int32 [n * P]: the cold pages' pool blocks, sequence by sequence; -1 behind the last
    cold_index: torch.Tensor   # int32 [n * P]: sequence * P + page of the same pages
    cold_starts: torch.Tensor  # int32 [n + 1]: where each sequence's cold pages begin
    kept_tables: torch.Tensor  # int32 [n, P]: block tables of the pages that stay, -1 behind the last
    kept_mass: torch.Tensor    # fp32 [n, P]: their weight, 0 behind the last
    kept_lens: torch.Tensor    # int32 [n]: tokens that stay
    status: torch.Tensor       # int32 [n]


def prepare_select(mass: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor, cold_blocks: torch.Tensor,
                   cold_index: torch.Tensor, cold_starts: torch.Tensor, kept_tables: torch.Tensor,
                   kept_mass: torch.Tensor, kept_lens: torch.Tensor, *, page_tokens: int, keep: int, sink: int = 1,
                   recent: int = 1, status: torch.Tensor | None = None) -> PreparedCall:
    """Choice of the pages to evict, checked and packed once.

    Sequence b has n = ceil(kv_lens[b] / page_tokens) pages.  Of pages [sink, n - recent), the
    min(n - keep, n - recent - sink) with the least mass (ties: the lower page; a NaN counts as the most) are cold;
    ``recent`` is at least 1, so the last, possibly unfilled page stays.  Outputs as ``ColdSelection``.  Calling the
    result enqueues the kernel and returns the ``ColdSelection``.  A block that several sequences share can be cold
    for more than one of them: whoever owns the pool counts its users before it is freed."""
    _require_cuda("mass", mass, (torch.float32,))
    dev = mass.device
    _require_cuda("block_tables", block_tables, (torch.int32,), dev)
    if mass.dim() != 2 or mass.shape != block_tables.shape:
        raise RuntimeError("mass and block_tables must have the same shape [sequences, pages]")
    n, P = mass.shape
    _check_vector("kv_lens", kv_lens, n, (torch.int32,), dev)
    for name, t, size in (("cold_blocks", cold_blocks, n * P), ("cold_index", cold_index, n * P),
                          ("cold_starts", cold_starts, n + 1), ("kept_lens", kept_lens, n)):
        _check_vector(name, t, size, (torch.int32,), dev)
    for name, t, dtype in (("kept_tables", kept_tables, torch.int32), ("kept_mass", kept_mass, torch.float32)):
        _require_cuda(name, t, (dtype,), dev)
        if t.shape != mass.shape:
            raise RuntimeError(f"{name} must have mass's shape {tuple(mass.shape)}")
    status = _status(status, n, dev)
    outs = ColdSelection(cold_blocks, cold_index, cold_starts, kept_tables, kept_mass, kept_lens, status)
    _check_disjoint(list(zip(outs._fields, outs)),
                    [("mass", mass), ("block_tables", block_tables), ("kv_lens", kv_lens)])
    block = _Selection(mass.data_ptr(), block_tables.data_ptr(), kv_lens.data_ptr(), n, P, int(page_tokens), int(keep),
                       int(sink), int(recent), *(t.data_ptr() for t in outs))
    return _OwningCall(_load().ztcp_select_cold_pages, (block,), dev, (mass, block_tables, kv_lens, *outs), outs, (status,))


def select_cold_pages(mass: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor, *, page_tokens: int,
                      keep: int, sink: int = 1, recent: int = 1, stream=None) -> ColdSelection:
    """Choice of the pages to evict into new tensors, enqueued on `stream` (default: the current stream);
    arguments as for ``prepare_select``.  ``sel.cold_blocks[:int(sel.cold_starts[-1])]`` is the block table that
    ``codec.encode_pages`` takes for the egress of all cold pages."""
    _require_cuda("mass", mass, (torch.float32,))
    if mass.dim() != 2:
        raise RuntimeError("mass and block_tables must have the same shape [sequences, pages]")

    def prepare():
        n, P = mass.shape
        ints = lambda *s: torch.empty(s, dtype=torch.int32, device=mass.device)  # noqa: E731
        return prepare_select(mass, block_tables, kv_lens, ints(n * P), ints(n * P), ints(n + 1), ints(n, P),
                              torch.empty_like(mass), ints(n), page_tokens=page_tokens, keep=keep, sink=sink, recent=recent)

    return _run_once(prepare, mass, stream)
