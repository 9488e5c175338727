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

from ._lib import Pages, Prompt, call
from .quant import Context, _current_stream, _dtype_code, _need, _stream_ptr, _t

__all__ = ["prompt_attention", "prompt_attention_bwd", "paged_attention", "pages_append", "pages_copy"]


def _rows(t, ctx: Context, width: int, what: str, dtype=None, rows: int | None = None):
    """t [rows, width] on the context's device, elements of a row side by side -> its row stride."""
    _need(t.is_cuda and t.get_device() == ctx.device, f"{what} must be a CUDA tensor of the context's device")
    _need(t.dim() == 2 and t.shape[1] == width and (t.stride(1) == 1 or t.numel() == 0),
          f"{what} must be [rows, {width}] with its rows' elements side by side")
    _need(dtype is None or t.dtype == dtype, f"{what} has another type")
    _need(rows is None or t.shape[0] == rows, f"{what} must have {rows} rows")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)


def _i32(t, ctx: Context, n: int, what: str):
    _need(t.is_cuda and t.get_device() == ctx.device and t.dtype == _t().int32 and t.is_contiguous()
          and t.numel() == n, f"{what} must be a contiguous int32 CUDA tensor of {n} elements on the context's device")
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


def _empty(scope, *shapes_dtypes, device):
    torch = _t()
    if scope is None:
        return [torch.empty(s, dtype=d, device=device) for s, d in shapes_dtypes]
    with scope:
        return [torch.empty(s, dtype=d, device=device) for s, d in shapes_dtypes]


def _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal):
    _dtype_code(q)
    qw, kw = n_q * head_dim, n_kv * head_dim
    _need(cu.dim() == 1 and cu.numel() >= 1, "cu must hold batch + 1 row numbers")
    batch = cu.numel() - 1
    qs = _rows(q, ctx, qw, "q")
    ks = _rows(k, ctx, kw, "k", q.dtype)
    vs = _rows(v, ctx, kw, "v", q.dtype, k.shape[0])
    p = Prompt(_dtype_code(q), batch, q.shape[0], k.shape[0], n_q, n_kv, head_dim, _i32(cu, ctx, batch + 1, "cu"),
               None if cu_k is None else _i32(cu_k, ctx, batch + 1, "cu_k"), 1 if causal else 0, float(scale))
    return p, qs, ks, vs


def prompt_attention(ctx: Context, q, k, v, cu, n_q: int, n_kv: int, head_dim: int, scale: float, causal: bool = True,
                     cu_k=None, out=None, lse=None, stream=None):
    """rq_prompt_attention: q [rows, n_q*head_dim], k and v [rows_k, n_kv*head_dim]
    (f32 or bf16), sequence b in rows cu[b] .. cu[b+1] - 1 (int32 [batch + 1];
    cu_k: the keys', when they differ) -> out [rows, n_q*head_dim]. lse f32
    [n_q, rows] is filled when given (prompt_attention_bwd needs it)."""
    torch = _t()
    p, qs, ks, vs = _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal)
    raw, scope = _on(stream, q)
    if out is None:
        out, = _empty(scope, (q.shape, q.dtype), device=q.device)
    os = _rows(out, ctx, n_q * head_dim, "out", q.dtype, q.shape[0])
    if lse is not None:
        _need(lse.is_cuda and lse.get_device() == ctx.device and lse.dtype == torch.float32 and lse.is_contiguous()
              and lse.numel() == n_q * q.shape[0], "lse must be a contiguous f32 CUDA tensor [n_q, rows]")
    call("rq_prompt_attention", ctx.handle, C.byref(p), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
         out.data_ptr(), os, None if lse is None else lse.data_ptr(), raw)
    return out


def prompt_attention_bwd(ctx: Context, dout, q, k, v, out, lse, cu, n_q: int, n_kv: int, head_dim: int, scale: float,
                         causal: bool = True, cu_k=None, dq=None, dk=None, dv=None, stream=None):
    """rq_prompt_attention_bwd: the gradient of prompt_attention for dout, from
    the forward's out and lse -> (dq, dk, dv), written into the given tensors if any."""
    torch = _t()
    p, qs, ks, vs = _prompt(ctx, q, k, v, cu, cu_k, n_q, n_kv, head_dim, scale, causal)
    qw, kw, rows, rows_k = n_q * head_dim, n_kv * head_dim, q.shape[0], k.shape[0]
    dos = _rows(dout, ctx, qw, "dout", q.dtype, rows)
    os = _rows(out, ctx, qw, "out", q.dtype, rows)
    _need(lse.is_cuda and lse.get_device() == ctx.device and lse.dtype == torch.float32 and lse.is_contiguous()
          and lse.numel() == n_q * rows, "lse must be the forward's f32 CUDA tensor [n_q, rows]")
    need = C.c_size_t()
    call("rq_prompt_attention_bwd_work", C.byref(p), C.byref(need))
    raw, scope = _on(stream, q)
    new = [((rows, qw), q.dtype)] * (dq is None) + [((rows_k, kw), q.dtype)] * ((dk is None) + (dv is None))
    work, *made = _empty(scope, ((need.value // 4,), torch.float32), *new, device=q.device)
    dq, dk, dv = (made.pop(0) if t is None else t for t in (dq, dk, dv))
    dqs = _rows(dq, ctx, qw, "dq", q.dtype, rows)
    dks, dvs = (_rows(t, ctx, kw, n, q.dtype, rows_k) for t, n in ((dk, "dk"), (dv, "dv")))
    call("rq_prompt_attention_bwd", ctx.handle, C.byref(p), dout.data_ptr(), dos, q.data_ptr(), qs, k.data_ptr(), ks,
         v.data_ptr(), vs, out.data_ptr(), os, lse.data_ptr(), dq.data_ptr(), dqs, dk.data_ptr(), dks, dv.data_ptr(),
         dvs, work.data_ptr(), need.value, raw)
    return dq, dk, dv


def _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch):
    for t, n in ((kpages, "kpages"), (vpages, "vpages")):
        _need(t.is_cuda and t.get_device() == ctx.device and t.is_contiguous() and t.dim() == 3
              and t.shape[2] == n_kv * head_dim,
              f"{n} must be a contiguous CUDA tensor [pages, page_size, n_kv*head_dim] of the context's device")
    _need(vpages.shape == kpages.shape and vpages.dtype == kpages.dtype, "kpages and vpages must be alike")
    _need(table.dim() == 2 and table.shape[0] == batch, "table must be [batch, pages of a sequence]")
    return Pages(_dtype_code(kpages), kpages.data_ptr(), vpages.data_ptr(), kpages.shape[0], kpages.shape[1], n_kv,
                 head_dim, _i32(table, ctx, table.numel(), "table"), table.shape[1])


def paged_attention(ctx: Context, q, k, v, kpages, vpages, table, lens, n_q: int, n_kv: int, head_dim: int,
                    theta: float, scale: float, max_len: int | None = None, out=None, stream=None):
    """rq_paged_attention: one new token of each sequence b (rows of q [batch,
    n_q*head_dim], k and v [batch, n_kv*head_dim]) at position lens[b] of its
    pages (kpages, vpages [pages, page_size, n_kv*head_dim], table int32 [batch,
    pages of a sequence]): RoPE, append, attention over rows 0 .. lens[b] -> out
    [batch, n_q*head_dim]. k and v None: nothing appended, rows 0 .. lens[b] - 1. max_len:
    no sequence is longer, the new row included (default: what the table holds)."""
    torch = _t()
    dt = _dtype_code(q)
    batch, kw = q.shape[0], n_kv * head_dim
    qs = _rows(q, ctx, n_q * head_dim, "q")
    _need((k is None) == (v is None), "k and v must both be given, or neither")
    ks = vs = 0
    if k is not None:
        ks, vs = _rows(k, ctx, kw, "k", q.dtype, batch), _rows(v, ctx, kw, "v", q.dtype, batch)
    pg = _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch)
    if max_len is None:
        max_len = table.shape[1] * kpages.shape[1]
    need = C.c_size_t()
    call("rq_paged_attention_work", ctx.handle, batch, n_q, n_kv, head_dim, max_len, C.byref(need))
    raw, scope = _on(stream, q)
    new = [(q.shape, q.dtype)] * (out is None)
    work, *made = _empty(scope, ((need.value // 4,), torch.float32), *new, device=q.device)
    if out is None:
        out, = made
    os = _rows(out, ctx, n_q * head_dim, "out", q.dtype, batch)
    call("rq_paged_attention", ctx.handle, C.byref(pg), dt, q.data_ptr(), qs, None if k is None else k.data_ptr(), ks,
         None if v is None else v.data_ptr(), vs, _i32(lens, ctx, batch, "lens"), batch, n_q, max_len, float(theta),
         float(scale), out.data_ptr(), os, work.data_ptr() if need.value else None, need.value, raw)
    return out


def pages_append(ctx: Context, q, k, v, kpages, vpages, table, cu, past, n_q: int, n_kv: int, head_dim: int,
                 theta: float, q_out=None, k_out=None, stream=None):
    """rq_pages_append: packed rows (sequence b: cu[b] .. cu[b+1] - 1, at positions
    past[b] and on) of q [rows, n_q*head_dim] and k [rows, n_kv*head_dim] rotated,
    the rotated k and v stored in the pages -> (rotated q, rotated k), written
    into q_out / k_out when given (they may be q and k)."""
    rows, qw, kw = q.shape[0], n_q * head_dim, n_kv * head_dim
    dt = _dtype_code(q)
    qs = _rows(q, ctx, qw, "q")
    ks, vs = _rows(k, ctx, kw, "k", q.dtype, rows), _rows(v, ctx, kw, "v", q.dtype, rows)
    _need(cu.dim() == 1 and cu.numel() >= 1, "cu must hold batch + 1 row numbers")
    batch = cu.numel() - 1
    pg = _pages(ctx, kpages, vpages, table, n_kv, head_dim, batch)
    raw, scope = _on(stream, q)
    made = _empty(scope, *[((rows, qw), q.dtype)] * (q_out is None), *[((rows, kw), q.dtype)] * (k_out is None),
                  device=q.device)
    q_out, k_out = (made.pop(0) if t is None else t for t in (q_out, k_out))
    qos, kos = _rows(q_out, ctx, qw, "q_out", q.dtype, rows), _rows(k_out, ctx, kw, "k_out", q.dtype, rows)
    call("rq_pages_append", ctx.handle, C.byref(pg), dt, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
         _i32(cu, ctx, batch + 1, "cu"), _i32(past, ctx, batch, "past"), batch, rows, n_q, float(theta),
         q_out.data_ptr(), qos, k_out.data_ptr(), kos, raw)
    return q_out, k_out


def pages_copy(ctx: Context, pages, src, dst, stream=None):
    """rq_pages_copy: page src[i] -> page dst[i] in every plane of pages [planes,
    pages, page_size, width] (src, dst host sequences of page numbers, all dst
    different and none of them a src) -> pages."""
    _need(pages.is_cuda and pages.get_device() == ctx.device and pages.is_contiguous() and pages.dim() == 4,
          "pages must be a contiguous CUDA tensor [planes, pages, page_size, width] of the context's device")
    _need(len(src) == len(dst), "src and dst must be equally long")
    n = len(src)
    arr = C.c_int32 * n
    size = pages.element_size()
    page = pages.shape[2] * pages.shape[3] * size
    raw, _ = _on(stream, pages)
    call("rq_pages_copy", ctx.handle, pages.data_ptr(), pages.shape[0], pages.shape[1] * page, pages.shape[1], page,
         arr(*src), arr(*dst), n, raw)
    return pages
