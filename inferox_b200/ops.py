"""Mirror of src/ops.rs (and the dequantiser, src/gguf/dequant.rs) over the
op-level C ABI. Arguments are CUDA tensors (torch is used only to hold device
memory and streams); every call runs the library's sm_100a kernels.

Shape mismatches raise IfxError("Shape") where the reference panics.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple

import numpy as np
import torch

from ._lib import IfxError, SamplerC, check, lib


def _p(t: torch.Tensor) -> C.c_void_p:
    if not t.is_cuda:
        raise IfxError(24, "expected a CUDA tensor")
    if not t.is_contiguous():
        raise IfxError(24, "expected a contiguous tensor")
    return C.c_void_p(t.data_ptr())


def _s() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need(cond: bool, what: str):
    if not cond:
        raise IfxError(20, what)


def dequantize(ttype: int, data: torch.Tensor, n_out: int) -> torch.Tensor:
    """dequantize_f32 (dequant.rs:10-31): uint8 CUDA bytes -> f32 [n_out]."""
    out = torch.empty(n_out, dtype=torch.float32, device=data.device)
    check(lib.ifx_op_dequantize(ttype, _p(data), data.numel(), _p(out), n_out, _s()), "dequantize")
    return out


def matmul(a, b, m, n, k) -> torch.Tensor:  # ops.rs:15-26
    _need(a.numel() == m * k and b.numel() == k * n, "matmul shape mismatch")
    c = torch.empty(m * n, dtype=torch.float32, device=a.device)
    check(lib.ifx_op_matmul(_p(a), _p(b), _p(c), m, n, k, _s()), "matmul")
    return c


def matmul_t(a, b, m, n, k) -> torch.Tensor:  # ops.rs:33-44
    _need(a.numel() == m * k and b.numel() == n * k, "matmul_t shape mismatch")
    c = torch.empty(m * n, dtype=torch.float32, device=a.device)
    check(lib.ifx_op_matmul_t(_p(a), _p(b), _p(c), m, n, k, _s()), "matmul_t")
    return c


class QMatrix:
    """A quantised [rows, cols] weight uploaded and repacked once."""

    def __init__(self, ttype: int, gguf_bytes: bytes | np.ndarray, rows: int, cols: int,
                 device: int = 0):
        buf = np.frombuffer(bytes(gguf_bytes), np.uint8) if not isinstance(gguf_bytes, np.ndarray) \
            else np.ascontiguousarray(gguf_bytes, np.uint8)
        h = C.c_void_p()
        check(lib.ifx_qmatrix_create(ttype, buf.ctypes.data_as(C.c_void_p), buf.nbytes, rows, cols,
                                     device, C.byref(h)), "qmatrix_create")
        self._h = h
        self.rows, self.cols, self.type = rows, cols, ttype

    def __del__(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            lib.ifx_qmatrix_free(self._h)
            self._h = None


def matmul_t_q(a: torch.Tensor, w: QMatrix, m: int) -> torch.Tensor:
    """C[m, rows] = A[m, cols] W^T with the fused dequant kernels."""
    _need(a.numel() == m * w.cols, "matmul_t_q shape mismatch")
    c = torch.empty(m * w.rows, dtype=torch.float32, device=a.device)
    check(lib.ifx_op_matmul_t_q(_p(a), w._h, _p(c), m, _s()), "matmul_t_q")
    return c


def bench_matmul_t_q(a: torch.Tensor, w: QMatrix, m: int, reps: int = 10) -> float:
    """ms per call of the fused dequant matmul the token loop runs at batch m
    (GEMV at 1, small-batch GEMM up to 32, prefill GEMM above), each launch
    timed alone with the weights coming from HBM."""
    _need(a.numel() == m * w.cols, "bench_matmul_t_q shape mismatch")
    c = torch.empty(m * w.rows, dtype=torch.float32, device=a.device)
    ms = C.c_float(0.0)
    check(lib.ifx_bench_matmul_t_q(_p(a), w._h, _p(c), m, reps, C.byref(ms)), "bench_matmul_t_q")
    return float(ms.value)


def rms_norm(x, w, eps):  # ops.rs:155-168 (in place)
    _need(x.numel() == w.numel(), "RMSNorm weight length mismatch")
    check(lib.ifx_op_rms_norm_rows(_p(x), _p(w), eps, 1, w.numel(), _s()), "rms_norm")
    return x


def rms_norm_rows(x, w, eps, rows):  # ops.rs:173-180 (in place)
    _need(x.numel() == rows * w.numel(), "RMSNorm rows shape mismatch")
    check(lib.ifx_op_rms_norm_rows(_p(x), _p(w), eps, rows, w.numel(), _s()), "rms_norm_rows")
    return x


def silu(x):  # ops.rs:183-187 (in place)
    check(lib.ifx_op_silu(_p(x), x.numel(), _s()), "silu")
    return x


def swiglu(gate, up):  # ops.rs:190-197
    _need(gate.numel() == up.numel(), "SwiGLU gate/up length mismatch")
    out = torch.empty_like(gate)
    check(lib.ifx_op_swiglu(_p(gate), _p(up), _p(out), gate.numel(), _s()), "swiglu")
    return out


def add_in_place(out, b):  # ops.rs:212-217
    _need(out.numel() == b.numel(), "add length mismatch")
    check(lib.ifx_op_add_in_place(_p(out), _p(b), out.numel(), _s()), "add_in_place")
    return out


def softmax_rows(x, rows, cols):  # ops.rs:223-239 (in place)
    _need(x.numel() == rows * cols, "softmax shape mismatch")
    check(lib.ifx_op_softmax_rows(_p(x), rows, cols, _s()), "softmax_rows")
    return x


def embedding_lookup(emb, ids, hidden):  # ops.rs:246-258
    out = torch.empty(ids.numel() * hidden, dtype=torch.float32, device=emb.device)
    check(lib.ifx_op_embedding_lookup(_p(emb), emb.numel(), _p(ids), ids.numel(), hidden, _p(out),
                                      _s()), "embedding_lookup")
    return out


def rope(x, seq_len, n_heads, head_dim, rope_dim, base, pos0=0):  # ops.rs:265-287
    _need(x.numel() == seq_len * n_heads * head_dim, "rope shape mismatch")
    check(lib.ifx_op_rope(_p(x), seq_len, n_heads, head_dim, rope_dim, base, pos0, _s()), "rope")
    return x


def argmax(x) -> int:  # forward.rs:615-622
    out = torch.zeros(1, dtype=torch.int32, device=x.device)
    check(lib.ifx_op_argmax(_p(x), x.numel(), _p(out), _s()), "argmax")
    return int(out.item())


def sample_u(logits, temperature, top_k, top_p, u) -> int:
    """Sampler::sample (sampler.rs:28-73) with the uniform draw supplied."""
    s = SamplerC(temperature, top_k, top_p)
    tok = C.c_uint32()
    check(lib.ifx_op_sample_u(_p(logits), logits.numel(), C.byref(s), float(u), C.byref(tok),
                              _s()), "sample_u")
    return int(tok.value)


# ---- a paged serving step on the device (no counterparts in the reference) --
PAGE_ROWS = 64
_TYPES = {torch.float32: 0, torch.float16: 1}


def _dev(*tensors) -> int:
    """The one CUDA device the tensors are on."""
    d = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != d or d < 0:
            raise IfxError(24, "expected CUDA tensors of one device")
    return d


def _ints(what: str, *tensors):
    for t in tensors:
        if t.dtype is not torch.int32 or not t.is_contiguous():
            raise IfxError(24, f"{what}: expected contiguous int32 tensors")


def _call(dev: int, what: str, fn, *args):
    """fn(*args, stream) on the current stream of device `dev`."""
    if dev == torch._C._cuda_getDevice():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if code:
        check(code, what)


class PageStep(NamedTuple):
    """What pages_extend gives: the sequences' new lengths, the free list's new
    length, the sequences' first new rows [n_seqs + 1], each new row's slot,
    position and sequence [max_tokens] (-1 behind the last), and the status
    (0, or 1 too few free pages, 2 a sequence beyond its table row, 3 more
    rows than max_tokens: nothing was taken)."""

    lens: torch.Tensor
    n_free: torch.Tensor
    q_start: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    seqs: torch.Tensor
    status: torch.Tensor


def pages_extend(lens, add, table, free, n_free, max_tokens: int) -> PageStep:
    """Pages and slots for add[b] new rows behind sequence b's lens[b] rows.
    table [n_seqs, max_pages] takes the new pages, from the end of
    free[:n_free]; all int32. The caller goes on with the returned lens and
    n_free. Nothing is copied to the host: the status is on the device."""
    dev = _dev(lens, add, table, free, n_free)
    _ints("pages_extend", lens, add, table, free, n_free)
    n = lens.numel()
    _need(table.dim() == 2 and table.shape[0] == n and add.numel() == n and n_free.numel() == 1,
          "pages_extend shape mismatch")
    _need(max_tokens >= 0, "pages_extend: negative max_tokens")
    # one allocation: slots, positions, seqs, q_start, lens, n_free, status
    sizes = (max_tokens, max_tokens, max_tokens, n + 1, n, 1, 1)
    slots, positions, seqs, q_start, lens_out, n_free_out, status = torch.empty(
        3 * max_tokens + 2 * n + 3, dtype=torch.int32, device=lens.device).split_with_sizes(sizes)
    q = q_start.data_ptr()  # (an empty part has no address)
    p = q - 12 * max_tokens
    _call(dev, "pages_extend", lib.ifx_op_pages_extend, lens.data_ptr(), add.data_ptr(), n, table.data_ptr(),
          table.shape[1], free.data_ptr(), free.numel(), n_free.data_ptr(), max_tokens, q + 4 * n + 4, q + 8 * n + 4, q,
          p, p + 4 * max_tokens, p + 8 * max_tokens, q + 8 * n + 8)
    return PageStep(lens_out, n_free_out, q_start, slots, positions, seqs, status)


def pages_release(done, lens, table, free, n_free):
    """Sequences with done[b] != 0 give their pages back to the end of
    free[:n_free]; returns (lens, n_free) to go on with."""
    dev = _dev(done, lens, table, free, n_free)
    _ints("pages_release", done, lens, table, free, n_free)
    n = lens.numel()
    _need(table.dim() == 2 and table.shape[0] == n and done.numel() == n and n_free.numel() == 1,
          "pages_release shape mismatch")
    lens_out, n_free_out = torch.empty(n + 1, dtype=torch.int32, device=lens.device).split_with_sizes((n, 1))
    p = n_free_out.data_ptr()
    _call(dev, "pages_release", lib.ifx_op_pages_release, done.data_ptr(), lens.data_ptr(), n, table.data_ptr(),
          table.shape[1], free.data_ptr(), free.numel(), n_free.data_ptr(), p - 4 * n, p)
    return lens_out, n_free_out


@lru_cache(maxsize=None)
def kv4_page_bytes(n_kv_heads: int, head_dim: int) -> int:
    """Bytes of one page (64 rows of keys and values) of the cache in 4 bits."""
    n = lib.ifx_kv4_page_bytes(n_kv_heads, head_dim) if n_kv_heads > 0 and head_dim > 0 else 0
    if not n:
        raise IfxError(26, "kv4: 1 to 1024 kv heads, head_dim a multiple of 32 up to 256")
    return n


@lru_cache(maxsize=None)
def _workspace_bytes(n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    return lib.ifx_kv4_attention_workspace(n_heads, n_kv_heads, head_dim)


def kv4_pages(n_pages: int, n_kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Memory for n_pages pages, uint8 [n_pages, page bytes]."""
    return torch.zeros(n_pages, kv4_page_bytes(n_kv_heads, head_dim), dtype=torch.uint8, device=device)


def _pool(what: str, pages: torch.Tensor, n_kv_heads: int, head_dim: int) -> int:
    if pages.dtype is not torch.uint8 or pages.dim() != 2 or not pages.is_contiguous():
        raise IfxError(24, f"{what}: pages must be a contiguous uint8 tensor [n_pages, page bytes]")
    n, size = pages.shape
    if size != kv4_page_bytes(n_kv_heads, head_dim):
        raise IfxError(20, f"{what}: page bytes mismatch")
    return n


def _rows(what: str, x: torch.Tensor):
    """(rows, heads, head_dim, stride between the rows) of x, whose rows are contiguous."""
    if x.dtype not in _TYPES:
        raise IfxError(26, f"{what}: float32 or float16 rows")
    if x.dim() != 3:
        raise IfxError(20, f"{what}: expected [rows, heads, head_dim]")
    n, h, d = x.shape
    if x.is_contiguous():
        return n, h, d, h * d
    sn, sh, sd = x.stride()
    if (sd != 1 and d != 1) or (sh != d and h != 1):
        raise IfxError(24, f"{what}: a row's heads must be contiguous")
    return n, h, d, sn if n > 1 else h * d


def kv4_store(k, v, slots, pages) -> None:
    """Rows k, v [n, n_kv_heads, head_dim] quantised into the rows slots [n] of
    the pages; a slot outside them (-1) skips its row. The slots differ."""
    dev = _dev(k, v, slots, pages)
    n, g, d, ks = _rows("kv4_store", k)
    vs = _rows("kv4_store", v)[3]
    _need(k.shape == v.shape and k.dtype is v.dtype and slots.numel() == n, "kv4_store shape mismatch")
    _ints("kv4_store", slots)
    np_ = _pool("kv4_store", pages, g, d)
    _call(dev, "kv4_store", lib.ifx_op_kv4_store, _TYPES[k.dtype], k.data_ptr(), ks, v.data_ptr(), vs,
          slots.data_ptr(), n, pages.data_ptr(), np_, g, d)


def kv4_load(slots, pages, n_kv_heads: int, head_dim: int, dtype=torch.float32):
    """The values of the rows slots [n]: (k, v) [n, n_kv_heads, head_dim]; zeros
    for a slot outside the pages."""
    dev = _dev(slots, pages)
    _ints("kv4_load", slots)
    np_ = _pool("kv4_load", pages, n_kv_heads, head_dim)
    if dtype not in _TYPES:
        raise IfxError(26, "kv4_load: float32 or float16 rows")
    n = slots.numel()
    k = torch.empty(n, n_kv_heads, head_dim, dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    _call(dev, "kv4_load", lib.ifx_op_kv4_load, _TYPES[dtype], pages.data_ptr(), np_, n_kv_heads, head_dim,
          slots.data_ptr(), n, k.data_ptr(), v.data_ptr())
    return k, v


def kv4_attention(q, pages, table, kv_len, n_kv_heads: int, q_start=None, scale=None, window: int = 0,
                  out=None, workspace=None) -> torch.Tensor:
    """Causal attention of q [rows, n_heads, head_dim] over the cache in 4 bits.
    Sequence b has kv_len[b] rows in the cache, the query rows' own among
    them, in the pages table[b]; its query rows are q_start[b]:q_start[b + 1],
    or row b when q_start is None. scale: 1 / sqrt(head_dim) when None;
    window > 0: each row sees its last `window` rows. A row that sees nothing
    gives 0; rows of a given `out` that are no sequence's stay as they were,
    those of a fresh one are 0. workspace: uint8 scratch kept by the caller
    (kv4_workspace), for one call at a time."""
    rows, h, d, qs = _rows("kv4_attention", q)
    n = kv_len.numel()
    if n_kv_heads <= 0 or h % n_kv_heads:
        raise IfxError(20, "kv4_attention: query heads must be a multiple of the kv heads")
    np_ = _pool("kv4_attention", pages, n_kv_heads, d)
    _ints("kv4_attention", table, kv_len)
    _need(table.dim() == 2 and table.shape[0] == n, "kv4_attention: table is [n_seqs, max_pages]")
    _need(window >= 0, "kv4_attention: negative window")
    starts = None
    if q_start is None:
        _need(rows == n, "kv4_attention: one row per sequence without q_start")
    else:
        _ints("kv4_attention", q_start)
        _need(q_start.numel() == n + 1, "kv4_attention: q_start is [n_seqs + 1]")
        starts = q_start.data_ptr()
    fresh = out is None
    if fresh:
        out, os = torch.empty((rows, h, d), dtype=q.dtype, device=q.device), h * d
    else:
        _need(out.shape == q.shape and out.dtype is q.dtype, "kv4_attention: out mismatch")
        os = _rows("kv4_attention", out)[3]
    if workspace is None:
        workspace = torch.empty(_workspace_bytes(h, n_kv_heads, d), dtype=torch.uint8, device=q.device)
    elif workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise IfxError(24, "kv4_attention: workspace must be a contiguous uint8 tensor")
    dev = _dev(q, pages, table, kv_len, out, workspace) if q_start is None else _dev(
        q, pages, table, kv_len, out, workspace, q_start)
    _call(dev, "kv4_attention", lib.ifx_op_kv4_attention, _TYPES[q.dtype], q.data_ptr(), qs, rows, pages.data_ptr(),
          np_, table.data_ptr(), table.shape[1], kv_len.data_ptr(), starts, n, h, n_kv_heads, d,
          d ** -0.5 if scale is None else scale, window, out.data_ptr(), os, fresh, workspace.data_ptr(),
          workspace.numel())
    return out


def kv4_workspace(n_heads: int, n_kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Scratch of kv4_attention for these shapes."""
    return torch.empty(_workspace_bytes(n_heads, n_kv_heads, head_dim), dtype=torch.uint8, device=device)


def sample_rows(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of every row of logits [rows, n] (float32), by
    Sampler::sample's rule with min-p beside its filters and the uniform draws
    u [rows] given, a tensor: (tokens int32 [rows], logprobs float32 [rows]).
    Settings are tensors [rows] or one value for all rows. A temperature that
    is not above 0 is greedy; a row whose logits are all masked (-inf, NaN)
    gives token -1."""
    if logits.dtype != torch.float32 or logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise IfxError(24, "sample_rows: logits must be float32 [rows, n] with contiguous rows")
    if not isinstance(u, torch.Tensor):  # (one number would be every row's)
        raise IfxError(24, "sample_rows: u is a float32 tensor, one draw per row")
    rows, n = logits.shape
    at = []
    for x, dt in ((u, torch.float32), (temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32),
                  (min_p, torch.float32)):
        if not isinstance(x, torch.Tensor):
            x = torch.full((rows,), x, dtype=dt, device=logits.device)
        if x.dtype != dt or not x.is_contiguous():
            raise IfxError(24, "sample_rows: settings are contiguous float32 tensors, top_k int32")
        _need(x.numel() == rows, "sample_rows shape mismatch")
        at.append(x)
    dev = _dev(logits, *at)
    token = torch.empty(rows, dtype=torch.int32, device=logits.device)
    logp = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _call(dev, "sample_rows", lib.ifx_op_sample_rows, logits.data_ptr(), logits.stride(0) if rows > 1 else n, rows, n,
          *(x.data_ptr() for x in at), token.data_ptr(), logp.data_ptr())
    return token, logp
