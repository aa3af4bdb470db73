"""Serving many requests from one paged key/value cache: attention of packed prompts,
attention of new tokens over the cache's pages, and a beam search step, through
libmtrtq's C ABI (include/mtrtq.h, which defines the formulas).

The reference decodes one sequence over contiguous caches (KVDecoder,
tools/run_gpt2.cpp:88-191). Lengths, page numbers and scores are read on the device, so
every call can be captured in a CUDA graph (with `out` and `workspace` given).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import check, lib
from .matmulq import Workspace, _stream_ptr

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_workspaces: dict = {}


def _workspace(workspace, device, stream_ptr: int, nbytes: int):
    """The caller's workspace (a Workspace, or a tensor), or one kept for each stream:
    calls that share a workspace must be ordered."""
    if isinstance(workspace, torch.Tensor):
        return workspace
    if workspace is None:
        key = (device.index, stream_ptr)
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = Workspace(device)
    return workspace.get(nbytes)


def _rows(name: str, x: torch.Tensor, heads: int | None, dim: int | None, rows: int | None, dtype=None):
    if x.dim() != 3 or x.dtype not in _DTYPES or not x.is_cuda:
        raise ValueError(f"{name} must be a float32 or bfloat16 CUDA tensor [rows, heads, head_dim]")
    if x.stride(2) != 1 and x.shape[2] > 1:
        raise ValueError(f"{name} must have unit stride along head_dim")
    want = (x.shape[0] if rows is None else rows, x.shape[1] if heads is None else heads,
            x.shape[2] if dim is None else dim)
    if tuple(x.shape) != want or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{name} must be {dtype or 'float32 or bfloat16'} {list(want)}, got {x.dtype} {list(x.shape)}")


def _ints(name: str, x: torch.Tensor, shape, device):
    if x.dtype != torch.int32 or x.device != device or tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must be int32 {list(shape)} on {device}, got {x.dtype} {list(x.shape)} on {x.device}")
    if x.shape and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension")


def _out(out, q, dtype, stream):
    if out is None:
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
        if isinstance(stream, torch.cuda.Stream):
            out.record_stream(stream)
    else:
        _rows("out", out, q.shape[1], q.shape[2], q.shape[0], dtype)
    return out


def _args(q, k, v, out, cu_rows, scale):
    a = _lib.AttentionArgs()
    T, H, D = q.shape
    a.q, a.out, a.cu_rows = q.data_ptr(), out.data_ptr(), cu_rows.data_ptr()
    a.q_row, a.q_head = q.stride(0), q.stride(1)
    a.out_row, a.out_head = out.stride(0), out.stride(1)
    if k is not None:
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.k_row, a.k_head = k.stride(0), k.stride(1)
        a.v_row, a.v_head = v.stride(0), v.stride(1)
    a.rows, a.batch, a.heads, a.head_dim = T, cu_rows.shape[0] - 1, H, D
    a.x_dtype, a.dtype = _DTYPES[q.dtype], _DTYPES[out.dtype]
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    return a


def _attend(fn, where, a, q, workspace, stream):
    with torch.cuda.device(q.device):
        sp = _stream_ptr(stream)
        need = lib().mtrtq_attention_workspace_bytes(ctypes.byref(a))
        if need < 0:
            # the call repeats the check and says what is wrong
            check(fn(ctypes.byref(a), None, 0, sp), where)
        ws = _workspace(workspace, q.device, sp, need)
        check(fn(ctypes.byref(a), ws.data_ptr() if ws is not None else None,
                 ws.numel() * ws.element_size() if ws is not None else 0, sp), where)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                     scale: float | None = None, workspace=None, stream=None) -> torch.Tensor:
    """Causal attention of packed prompts: request b owns rows cu_seqlens[b] to
    cu_seqlens[b+1] - 1 of q [rows, heads, head_dim], k and v [rows, kv_heads,
    head_dim] (views of one projection's rows are fine) and of the result.

    out_dtype: torch.bfloat16 (tensor cores) or torch.float32 (fp32 throughout, f32
    rows only); by default q's. scale defaults to 1 / sqrt(head_dim)."""
    _rows("q", q, None, None, None)
    _rows("k", k, None, q.shape[2], q.shape[0], q.dtype)
    _rows("v", v, k.shape[1], q.shape[2], q.shape[0], q.dtype)
    if cu_seqlens.dim() != 1:
        raise ValueError("cu_seqlens must be int32 [requests + 1]")
    _ints("cu_seqlens", cu_seqlens, cu_seqlens.shape, q.device)
    out = _out(out, q, out_dtype or (out.dtype if out is not None else q.dtype), stream)
    a = _args(q, k, v, out, cu_seqlens, scale)
    a.kv_heads = k.shape[1]
    _attend(lib().mtrtq_prompt_attention, "mtrtq_prompt_attention", a, q, workspace, stream)
    return out


def paged_attention(q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, k_pages: torch.Tensor,
                    v_pages: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, cu_rows: torch.Tensor, *,
                    out: torch.Tensor | None = None, scale: float | None = None, workspace=None,
                    stream=None) -> torch.Tensor:
    """New tokens over a paged cache: row t of request b's m rows (cu_rows[b] to
    cu_rows[b+1] - 1 of q [rows, heads, head_dim]) is its token kv_len[b] - m + t. k and
    v [rows, kv_heads, head_dim] are stored in the pages first (None: they are there
    already), then each row attends to its request's tokens up to its own.

    k_pages, v_pages [pages, kv_heads, page_size, head_dim] (float32, or bfloat16 with
    q, k, v of either type); table int32 [requests, columns] of page numbers; kv_len
    int32 [requests] counts the new tokens too. The result has the cache's type."""
    _rows("q", q, None, None, None)
    if k_pages.dim() != 4 or k_pages.dtype not in _DTYPES or k_pages.device != q.device:
        raise ValueError("k_pages must be float32 or bfloat16 [pages, kv_heads, page_size, head_dim] on q's device")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != q.device:
        raise ValueError("v_pages must be like k_pages")
    P, KV, S, D = k_pages.shape
    if D != q.shape[2]:
        raise ValueError(f"the pages' head_dim is {D}, q's {q.shape[2]}")
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if x.stride(0) != k_pages.stride(0) or P == 0 or not x[0].is_contiguous():
            raise ValueError(f"each page of {name} must be contiguous")
    if (k is None) != (v is None):
        raise ValueError("k and v are given together")
    if k is not None:
        _rows("k", k, KV, D, q.shape[0], q.dtype)
        _rows("v", v, KV, D, q.shape[0], q.dtype)
    if kv_len.dim() != 1 or table.dim() != 2:
        raise ValueError("kv_len must be int32 [requests], table int32 [requests, columns]")
    B = kv_len.shape[0]
    _ints("kv_len", kv_len, (B,), q.device)
    _ints("table", table, (B, table.shape[1]), q.device)
    _ints("cu_rows", cu_rows, (B + 1,), q.device)
    out = _out(out, q, k_pages.dtype, stream)
    a = _args(q, k, v, out, cu_rows, scale)
    a.kv_heads, a.page_size, a.num_pages, a.page_stride = KV, S, P, k_pages.stride(0)
    a.k_pages, a.v_pages, a.kv_len = k_pages.data_ptr(), v_pages.data_ptr(), kv_len.data_ptr()
    a.table, a.table_ld, a.table_width = table.data_ptr(), table.stride(0), table.shape[1]
    _attend(lib().mtrtq_paged_attention, "mtrtq_paged_attention", a, q, workspace, stream)
    return out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, done: torch.Tensor, eos: int = -1, *,
                out: tuple | None = None, workspace=None, stream=None):
    """One beam search step: logits float32 [requests * beams, vocab], scores float32
    and done uint8 [requests, beams]. Returns (scores, parent, token, done), each
    [requests, beams], the best `beams` of scores + log_softmax(logits) over beams and
    vocabulary, best first, ties to the lowest beam and token. A beam that is done
    goes on as the one candidate (itself, eos) with its score; a beam not in use has
    the score -inf. out: the four tensors to write (not the inputs)."""
    if scores.dim() != 2 or scores.dtype != torch.float32 or not scores.is_cuda or not scores.is_contiguous():
        raise ValueError("scores must be a contiguous float32 CUDA tensor [requests, beams]")
    B, W = scores.shape
    dev = scores.device
    if done.dtype != torch.uint8 or done.shape != scores.shape or done.device != dev or not done.is_contiguous():
        raise ValueError("done must be contiguous uint8 [requests, beams]")
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.shape[0] != B * W or logits.device != dev \
            or logits.stride(1) != 1:
        raise ValueError("logits must be float32 [requests * beams, vocab] with unit stride along vocab")
    if out is None:
        out = (torch.empty_like(scores), torch.empty((B, W), dtype=torch.int32, device=dev),
               torch.empty((B, W), dtype=torch.int32, device=dev), torch.empty_like(done))
        if isinstance(stream, torch.cuda.Stream):
            for x in out:
                x.record_stream(stream)
    else:
        for x, t in zip(out, (torch.float32, torch.int32, torch.int32, torch.uint8), strict=True):
            if x.shape != scores.shape or x.dtype != t or x.device != dev or not x.is_contiguous():
                raise ValueError("out is (float32, int32, int32, uint8), each contiguous [requests, beams]")
    V = logits.shape[1]
    with torch.cuda.device(dev):
        sp = _stream_ptr(stream)
        need = lib().mtrtq_beam_workspace_bytes(B, W, V)
        ws = _workspace(workspace, dev, sp, need) if need >= 0 else None
        check(lib().mtrtq_beam_select(logits.data_ptr(), logits.stride(0), scores.data_ptr(), done.data_ptr(), eos, B,
                                      W, V, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
                                      out[3].data_ptr(), ws.data_ptr() if ws is not None else None,
                                      ws.numel() * ws.element_size() if ws is not None else 0, sp),
              "mtrtq_beam_select")
    return out


def beam_reorder(parent: torch.Tensor, table: torch.Tensor, owned: torch.Tensor, kv_len: torch.Tensor,
                 k_pages: torch.Tensor, v_pages: torch.Tensor, *, stream=None) -> None:
    """The beams' cached states follow `parent` int32 [requests, beams], in place: rows
    of table int32 [requests * beams, columns] are taken from the parents' for the
    pages that are full at kv_len int32 [requests] tokens, and from owned (the pages
    only that beam writes) for the others; the tokens of the page being filled are
    copied between owned pages in every layer of k_pages and v_pages [layers, pages,
    kv_heads, page_size, head_dim] (or one layer's, without the first dimension)."""
    if parent.dim() != 2 or kv_len.dim() != 1 or table.dim() != 2:
        raise ValueError("parent must be [requests, beams], table [requests * beams, columns], kv_len [requests]")
    if k_pages.dim() == 4 and v_pages.dim() == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    if k_pages.dim() != 5 or k_pages.dtype not in _DTYPES or not k_pages.is_cuda:
        raise ValueError("k_pages must be a float32 or bfloat16 CUDA tensor [layers, pages, kv_heads, page_size, head_dim]")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device:
        raise ValueError("v_pages must be like k_pages")
    L, P, KV, S, D = k_pages.shape
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if x.stride()[:2] != k_pages.stride()[:2] or 0 in (L, P) or not x[0, 0].is_contiguous():
            raise ValueError(f"each page of {name} must be contiguous")
    B, W = parent.shape
    dev = k_pages.device
    _ints("parent", parent, (B, W), dev)
    if not parent.is_contiguous():
        raise ValueError("parent must be contiguous")
    _ints("table", table, (B * W, table.shape[1]), dev)
    _ints("owned", owned, tuple(table.shape), dev)
    _ints("kv_len", kv_len, (B,), dev)
    with torch.cuda.device(dev):
        check(lib().mtrtq_beam_reorder(parent.data_ptr(), B, W, table.data_ptr(), table.stride(0), owned.data_ptr(),
                                       owned.stride(0), table.shape[1], kv_len.data_ptr(), k_pages.data_ptr(),
                                       v_pages.data_ptr(), L, k_pages.stride(0), k_pages.stride(1), P, KV, S, D,
                                       _DTYPES[k_pages.dtype], _stream_ptr(stream)), "mtrtq_beam_reorder")
