"""Attention over packed prompts, its gradient, and the operators of a paged cache.

The batched companions of quant.decode_attention (raster/dl/attention.clj:197-287,
413-416, one token of one sequence):

  prompt_attention      every token of packed prompts attends its own sequence
  prompt_attention_bwd  its gradient (explicit, like matmul_dx)
  paged_attention       one new token of every sequence: RoPE, append, attention over pages
  pages_append          RoPE of packed prompts' q and k; k and v into the pages
  pages_copy            pages copied in every plane of a cache

Arrays are torch CUDA tensors of the context's device (memory and streams only);
rows may be strided (columns of one product's output), their elements may not. Without
`stream` the current one of the tensors' device is used. Every call goes through the C ABI of
include/rq.h; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from array import array

from ._lib import Pages, Prompt, call
from .quant import Context, _current_stream, _dtype_code, _need, _stream_ptr, _t

__all__ = ["prompt_attention", "prompt_attention_bwd", "paged_attention", "pages_append", "pages_copy"]


def _code(t) -> int:
    _t()  # (fills the table of types)
    return _dtype_code(t)


def _bad_rows(t, ctx: Context, rows, width: int, dtype, what: str):
    _need(t.is_cuda and t.get_device() == ctx.device, f"{what} must be a CUDA tensor of the context's device")
    _need(t.dtype == dtype, f"{what} must be {dtype}")
    raise ValueError(f"{what} must be [{'rows' if rows is None else rows}, {width}] with its rows' elements side by side")


def _rows(t, ctx: Context, rows, width: int, dtype, what: str) -> int:
    """The row stride of t, checked to be [rows, width] (rows None: any number) of
    dtype on the context's device with the elements of a row side by side."""
    shape = t.shape
    if (t.dtype != dtype or t.get_device() != ctx.device or len(shape) != 2 or shape[1] != width
            or (rows is not None and shape[0] != rows)):
        _bad_rows(t, ctx, rows, width, dtype, what)
    s0, s1 = t.stride()
    if s1 != 1 and width != 1:
        _bad_rows(t, ctx, rows, width, dtype, what)
    return s0 if shape[0] > 1 else max(s0, width)  # (of a single row, torch's stride may be anything)


def _i32(t, ctx: Context, n: int, what: str) -> int:
    if t.dtype != _t().int32 or t.get_device() != ctx.device or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 CUDA tensor of {n} elements on the context's device")
    return t.data_ptr()


def _on(stream, t):
    """The raw stream of a call, and a context in which new tensors belong to it."""
    torch = _t()
    if stream is None:
        return _current_stream(t), None
    if isinstance(stream, int):
        s = torch.cuda.ExternalStream(stream, t.device) if stream else torch.cuda.default_stream(t.device)
    else:
        s = stream
    return _stream_ptr(stream), torch.cuda.stream(s)


def _empty(scope, shape, like, dtype=None):
    if scope is not None:
        with scope:
            return like.new_empty(shape, dtype=dtype)
    return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)


def _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal):
    code, dtype, kw = _code(q), q.dtype, n_kv * head_dim
    n = cu.numel()
    _need(n >= 1, "cu must hold batch + 1 row numbers")
    qs = _rows(q, ctx, None, n_q * head_dim, dtype, "q")
    ks = _rows(k, ctx, None, kw, dtype, "k")
    rows, rows_k = q.shape[0], k.shape[0]
    vs = _rows(v, ctx, rows_k, kw, dtype, "v")
    p = Prompt(code, n - 1, rows, rows_k, n_q, n_kv, head_dim, _i32(cu, ctx, n, "cu"),
               None if cu_k is None else _i32(cu_k, ctx, n, "cu_k"), 1 if causal else 0, scale)
    return p, qs, ks, vs


def _check_lse(lse, ctx, n):
    _need(lse.dtype == _t().float32 and lse.get_device() == ctx.device and lse.is_contiguous() and lse.numel() == n,
          "lse must be a contiguous f32 CUDA tensor [n_q, rows] of the context's device")


def prompt_attention(ctx: Context, q, k, v, cu, n_q: int, n_kv: int, head_dim: int, scale: float, causal: bool = True,
                     cu_k=None, out=None, lse=None, stream=None):
    """rq_prompt_attention: q [rows, n_q*head_dim], k and v [rows_k, n_kv*head_dim]
    (f32 or bf16), sequence b in rows cu[b] .. cu[b+1] - 1 (int32 [batch + 1];
    cu_k: the keys', when they differ) -> out [rows, n_q*head_dim]. lse f32
    [n_q, rows] is filled when given (prompt_attention_bwd needs it)."""
    p, qs, ks, vs = _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal)
    raw, scope = _on(stream, q)
    width = n_q * head_dim
    if out is None:
        out, os = _empty(scope, (q.shape[0], width), q), width
    else:
        os = _rows(out, ctx, q.shape[0], width, q.dtype, "out")
    if lse is not None:
        _check_lse(lse, ctx, n_q * q.shape[0])
    call("rq_prompt_attention", ctx.handle, C.byref(p), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
         out.data_ptr(), os, None if lse is None else lse.data_ptr(), raw)
    return out


def prompt_attention_bwd(ctx: Context, dout, q, k, v, out, lse, cu, n_q: int, n_kv: int, head_dim: int, scale: float,
                         causal: bool = True, cu_k=None, dq=None, dk=None, dv=None, stream=None):
    """rq_prompt_attention_bwd: the gradient of prompt_attention for dout, from
    the forward's out and lse -> (dq, dk, dv), written into the given tensors if any."""
    p, qs, ks, vs = _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal)
    qw, kw, rows, rows_k, dtype = n_q * head_dim, n_kv * head_dim, q.shape[0], k.shape[0], q.dtype
    dos = _rows(dout, ctx, rows, qw, dtype, "dout")
    os = _rows(out, ctx, rows, qw, dtype, "out")
    _check_lse(lse, ctx, n_q * rows)
    need = C.c_size_t()
    call("rq_prompt_attention_bwd_work", C.byref(p), C.byref(need))
    raw, scope = _on(stream, q)
    work = _empty(scope, need.value // 4, q, _t().float32)
    dq = _empty(scope, (rows, qw), q) if dq is None else dq
    dk, dv = (_empty(scope, (rows_k, kw), q) if t is None else t for t in (dk, dv))
    dqs = _rows(dq, ctx, rows, qw, dtype, "dq")
    dks, dvs = _rows(dk, ctx, rows_k, kw, dtype, "dk"), _rows(dv, ctx, rows_k, kw, dtype, "dv")
    call("rq_prompt_attention_bwd", ctx.handle, C.byref(p), dout.data_ptr(), dos, q.data_ptr(), qs, k.data_ptr(), ks,
         v.data_ptr(), vs, out.data_ptr(), os, lse.data_ptr(), dq.data_ptr(), dqs, dk.data_ptr(), dks, dv.data_ptr(),
         dvs, work.data_ptr(), need.value, raw)
    return dq, dk, dv


def _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch):
    shape, dev, ts = kpages.shape, ctx.device, table.shape
    if (len(shape) != 3 or shape[2] != n_kv * head_dim or kpages.get_device() != dev or not kpages.is_contiguous()
            or vpages.shape != shape or vpages.dtype != kpages.dtype or vpages.get_device() != dev
            or not vpages.is_contiguous()):
        raise ValueError(f"kpages and vpages must be contiguous CUDA tensors [pages, page_size, {n_kv * head_dim}] of one "
                         "type on the context's device")
    if len(ts) != 2 or ts[0] != batch:
        raise ValueError("table must be [batch, pages of a sequence]")
    n = ts[1]
    return Pages(_code(kpages), kpages.data_ptr(), vpages.data_ptr(), shape[0], shape[1], n_kv, head_dim,
                 _i32(table, ctx, batch * n, "table"), n)


_work_sizes: dict = {}  # rq_paged_attention_work by its arguments


def _paged_work(ctx, batch, n_q, n_kv, head_dim, max_len) -> int:
    key = (ctx.device, batch, n_q, n_kv, head_dim, max_len)
    n = _work_sizes.get(key)
    if n is None:
        need = C.c_size_t()
        call("rq_paged_attention_work", ctx.handle, batch, n_q, n_kv, head_dim, max_len, C.byref(need))
        if len(_work_sizes) >= 4096:
            _work_sizes.clear()
        n = _work_sizes[key] = need.value
    return n


def paged_attention(ctx: Context, q, k, v, kpages, vpages, table, lens, n_q: int, n_kv: int, head_dim: int,
                    theta: float, scale: float, max_len: int | None = None, out=None, stream=None):
    """rq_paged_attention: one new token of each sequence b (rows of q [batch,
    n_q*head_dim], k and v [batch, n_kv*head_dim]) at position lens[b] of its
    pages (kpages, vpages [pages, page_size, n_kv*head_dim], table int32 [batch,
    pages of a sequence]): RoPE, append, attention over rows 0 .. lens[b] -> out
    [batch, n_q*head_dim]. k and v None: nothing appended, rows 0 .. lens[b] - 1. max_len:
    no sequence is longer, the new row included (default: what the table holds)."""
    code, dtype, qw, kw = _code(q), q.dtype, n_q * head_dim, n_kv * head_dim
    qs = _rows(q, ctx, None, qw, dtype, "q")
    batch = q.shape[0]
    _need((k is None) == (v is None), "k and v must both be given, or neither")
    kd = vd = None
    ks = vs = 0
    if k is not None:
        ks, vs = _rows(k, ctx, batch, kw, dtype, "k"), _rows(v, ctx, batch, kw, dtype, "v")
        kd, vd = k.data_ptr(), v.data_ptr()
    pg = _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch)
    if max_len is None:
        max_len = table.shape[1] * kpages.shape[1]
    need = _paged_work(ctx, batch, n_q, n_kv, head_dim, max_len)
    raw, scope = _on(stream, q)
    work = _empty(scope, need // 4, q, _t().float32) if need else None
    if out is None:
        out, os = _empty(scope, (batch, qw), q), qw
    else:
        os = _rows(out, ctx, batch, qw, dtype, "out")
    call("rq_paged_attention", ctx.handle, C.byref(pg), code, q.data_ptr(), qs, kd, ks, vd, vs,
         _i32(lens, ctx, batch, "lens"), batch, n_q, max_len, theta, scale, out.data_ptr(), os,
         work.data_ptr() if need else None, need, raw)
    return out


def pages_append(ctx: Context, q, k, v, kpages, vpages, table, cu, past, n_q: int, n_kv: int, head_dim: int,
                 theta: float, q_out=None, k_out=None, stream=None):
    """rq_pages_append: packed rows (sequence b: cu[b] .. cu[b+1] - 1, at positions
    past[b] and on) of q [rows, n_q*head_dim] and k [rows, n_kv*head_dim] rotated,
    the rotated k and v stored in the pages -> (rotated q, rotated k), written
    into q_out / k_out when given (they may be q and k)."""
    code, dtype, qw, kw = _code(q), q.dtype, n_q * head_dim, n_kv * head_dim
    qs = _rows(q, ctx, None, qw, dtype, "q")
    rows = q.shape[0]
    ks, vs = _rows(k, ctx, rows, kw, dtype, "k"), _rows(v, ctx, rows, kw, dtype, "v")
    batch = cu.numel() - 1
    _need(batch >= 0, "cu must hold batch + 1 row numbers")
    pg = _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch)
    raw, scope = _on(stream, q)
    qos, kos = qw, kw
    if q_out is None:
        q_out = _empty(scope, (rows, qw), q)
    else:
        qos = _rows(q_out, ctx, rows, qw, dtype, "q_out")
    if k_out is None:
        k_out = _empty(scope, (rows, kw), q)
    else:
        kos = _rows(k_out, ctx, rows, kw, dtype, "k_out")
    call("rq_pages_append", ctx.handle, C.byref(pg), code, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
         _i32(cu, ctx, batch + 1, "cu"), _i32(past, ctx, batch, "past"), batch, rows, n_q, theta,
         q_out.data_ptr(), qos, k_out.data_ptr(), kos, raw)
    return q_out, k_out


def pages_copy(ctx: Context, pages, src, dst, stream=None):
    """rq_pages_copy: page src[i] -> page dst[i] in every plane of pages [planes,
    pages, page_size, width] (src, dst host sequences of page numbers, all dst
    different and none of them a src) -> pages."""
    shape = pages.shape
    _need(pages.get_device() == ctx.device and pages.is_contiguous() and len(shape) == 4,
          "pages must be a contiguous CUDA tensor [planes, pages, page_size, width] of the context's device")
    n = len(src)
    _need(len(dst) == n, "src and dst must be equally long")
    page = shape[2] * shape[3] * pages.element_size()
    ids = array("i", src), array("i", dst)  # (OverflowError past 32 bits)
    raw, _ = _on(stream, pages)
    call("rq_pages_copy", ctx.handle, pages.data_ptr(), shape[0], shape[1] * page, shape[1], page,
         ids[0].buffer_info()[0], ids[1].buffer_info()[0], n, raw)
    return pages
