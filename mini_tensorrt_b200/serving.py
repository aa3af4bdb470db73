"""Serving many requests from one paged key/value cache: attention of packed prompts,
attention of new tokens over the cache's pages, and a beam search step, through
libmtrtq's C ABI (include/mtrtq.h, which defines the formulas).

The reference decodes one sequence over contiguous caches (KVDecoder,
tools/run_gpt2.cpp:88-191). Lengths, page numbers and scores are read on the device, so
every call can be captured in a CUDA graph (with `out` and `workspace` given).

`stream` (a torch stream or a raw stream's address; by default the current one) is where a
call runs; results and scratch that the call makes come from that stream's memory. That stream
must have waited for the inputs, and who reads the result elsewhere waits for that stream.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from ._lib import check, lib
from .matmulq import Workspace

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_workspaces: dict = {}
_NO_PAGES = (0, 0, 0, 0, 0, 0, 0, 0, 0)
# mtrtq_attention_args in the order of _lib.AttentionArgs, packed in one call (setting its
# fields one by one takes three times as long)
_pack = struct.Struct("@4P8q2q5if P2P2qiP2qP").pack
assert struct.calcsize("@4P8q2q5if P2P2qiP2qP") == ctypes.sizeof(_lib.AttentionArgs)


def _stream_ptr(stream, index: int) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)
    return stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else int(stream)


def _call(where: str, index: int, *args) -> None:
    """Calls the library with that device current. (These calls are a few microseconds of
    host time, so the device is only switched where it has to be.)"""
    fn = getattr(lib(), where)
    if torch.cuda.current_device() == index:
        check(fn(*args), where)
    else:
        with torch.cuda.device(index):
            check(fn(*args), where)


def _other_stream(stream, stream_ptr: int, index: int):
    """The call's stream as torch's, None if it is the current one."""
    if stream is None or stream_ptr == torch._C._cuda_getCurrentRawStream(index):
        return None
    return stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(stream_ptr, device=index)


def _made_there(other, device, make):
    """What make() allocates, from the memory of `other`, the call's stream, and kept from being
    given out again before the current stream's work with it is done."""
    with torch.cuda.stream(other):
        made = make()
    for x in made:
        x.record_stream(torch.cuda.current_stream(device))
    return made


def _workspace(workspace, device, stream_ptr: int, other, nbytes: int) -> torch.Tensor:
    """The caller's workspace (a Workspace, or a tensor), or one kept for each stream: calls
    that share a workspace must be ordered. What is made here is made and zero-filled on the
    call's stream (other, or the current one); while that is being captured it is the graph's
    (filled by its replays alone), so it is not kept for other calls."""
    if workspace is None:
        key = (device.index, stream_ptr)
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = Workspace(device)
    if not isinstance(workspace, Workspace):
        return workspace
    buf = workspace.buf
    if buf is not None and buf.numel() >= nbytes:
        return buf
    with torch.cuda.stream(other):
        if torch.cuda.is_current_stream_capturing():
            return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return workspace.get(nbytes, other)


def _rows(name: str, x: torch.Tensor, shape, dtype, device):
    """Checks rows of heads; returns their strides."""
    if x.shape != shape or x.dtype is not dtype or x.device != device:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on {device}, got {x.dtype} {list(x.shape)} on {x.device}")
    s = x.stride()
    if s[2] != 1 and shape[2] > 1:
        raise ValueError(f"{name} must have unit stride along head_dim")
    return s


def _ints(name: str, x: torch.Tensor, shape, device):
    if x.dtype != torch.int32 or x.device != device or x.shape != shape:
        raise ValueError(f"{name} must be int32 {list(shape)} on {device}, got {x.dtype} {list(x.shape)} on {x.device}")
    s = x.stride()
    if s[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must have unit stride along its last dimension")
    return s


def _attend(where, q, k, v, out, out_dtype, kv_heads, cu_rows, scale, workspace, stream, pages=_NO_PAGES):
    dtype, device = q.dtype, q.device
    if q.dim() != 3 or dtype not in _DTYPES or device.type != "cuda":
        raise ValueError("q must be a float32 or bfloat16 CUDA tensor [rows, heads, head_dim]")
    if out_dtype not in _DTYPES:
        raise ValueError("the result is float32 or bfloat16")
    shape, index = q.shape, device.index
    T, H, D = shape
    if D == 0:
        raise ValueError("head_dim must be positive")
    qs = _rows("q", q, shape, dtype, device)
    if k is not None:
        kv = (T, kv_heads, D)
        ks, vs = _rows("k", k, kv, dtype, device), _rows("v", v, kv, dtype, device)
        kp, vp = k.data_ptr(), v.data_ptr()
    else:
        ks, vs, kp, vp = (0, 0), (0, 0), 0, 0
    sp = _stream_ptr(stream, index)
    other = _other_stream(stream, sp, index)
    if out is None:
        if other is None:
            out = torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
        else:
            out, = _made_there(other, device, lambda: [torch.empty(shape, dtype=out_dtype, device=device)])
        os = (H * D, D)
    else:
        os = _rows("out", out, shape, out_dtype, device)
    if cu_rows.dim() != 1:
        raise ValueError("the row bounds must be int32 [requests + 1]")
    batch = cu_rows.shape[0] - 1
    _ints("the row bounds", cu_rows, (batch + 1,), device)
    a = _pack(q.data_ptr(), kp, vp, out.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], T, batch, H,
              kv_heads, D, _DTYPES[dtype], _DTYPES[out_dtype], D ** -0.5 if scale is None else scale,
              cu_rows.data_ptr(), *pages)
    need = lib().mtrtq_attention_workspace_bytes(a)
    if need > 0:
        ws = _workspace(workspace, device, sp, other, need)
        _call(where, index, a, ws.data_ptr(), ws.numel() * ws.element_size(), sp)
    else:  # refused by the call too, with the reason
        _call(where, index, a, None, 0, sp)
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                     scale: float | None = None, workspace=None, stream=None) -> torch.Tensor:
    """Causal attention of packed prompts: request b owns rows cu_seqlens[b] to
    cu_seqlens[b+1] - 1 of q [rows, heads, head_dim], k and v [rows, kv_heads,
    head_dim] (views of one projection's rows are fine) and of the result.

    out_dtype: torch.bfloat16 (tensor cores) or torch.float32 (fp32 throughout, f32
    rows only); by default q's. scale defaults to 1 / sqrt(head_dim)."""
    if out_dtype is None:
        out_dtype = q.dtype if out is None else out.dtype
    return _attend("mtrtq_prompt_attention", q, k, v, out, out_dtype, k.shape[1], cu_seqlens, scale, workspace, stream)


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
    if k_pages.dim() != 4 or k_pages.dtype not in _DTYPES or k_pages.device != q.device:
        raise ValueError("k_pages must be float32 or bfloat16 [pages, kv_heads, page_size, head_dim] on q's device")
    shape, s, dtype, device = k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.device
    if v_pages.shape != shape or v_pages.dtype != dtype or v_pages.device != device:
        raise ValueError("v_pages must be like k_pages")
    P, KV, S, D = shape
    # (strides of single heads say nothing)
    if P == 0 or s[1:] != (S * D, D, 1) and not k_pages[0].is_contiguous() or v_pages.stride() != s \
            and (v_pages.stride(0) != s[0] or not v_pages[0].is_contiguous()):
        raise ValueError("pages of k_pages and v_pages must be contiguous, and equally far apart")
    if D != q.shape[-1]:
        raise ValueError(f"the pages' head_dim is {D}, q's {q.shape[-1]}")
    if (k is None) != (v is None):
        raise ValueError("k and v are given together")
    if kv_len.dim() != 1 or table.dim() != 2:
        raise ValueError("kv_len must be int32 [requests], table int32 [requests, columns]")
    B, width = table.shape
    _ints("kv_len", kv_len, (B,), device)
    ld = _ints("table", table, (B, width), device)[0]
    if cu_rows.shape != (B + 1,):
        raise ValueError(f"cu_rows must be int32 [{B + 1}]")
    pages = (k_pages.data_ptr(), v_pages.data_ptr(), s[0], P, S, table.data_ptr(), ld if B > 1 else width, width,
             kv_len.data_ptr())
    return _attend("mtrtq_paged_attention", q, k, v, out, dtype, KV, cu_rows, scale, workspace, stream, pages)


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
            or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must be float32 [requests * beams, vocab] with unit stride along vocab")
    sp = _stream_ptr(stream, dev.index)
    other = _other_stream(stream, sp, dev.index)
    if out is None:
        make = lambda: (torch.empty_like(scores), torch.empty_like(scores, dtype=torch.int32),
                        torch.empty_like(scores, dtype=torch.int32), torch.empty_like(done))
        out = make() if other is None else _made_there(other, dev, make)
    else:
        for x, t in zip(out, (torch.float32, torch.int32, torch.int32, torch.uint8), strict=True):
            if x.shape != scores.shape or x.dtype != t or x.device != dev or not x.is_contiguous():
                raise ValueError("out is (float32, int32, int32, uint8), each contiguous [requests, beams]")
    V = logits.shape[1]
    need = lib().mtrtq_beam_workspace_bytes(B, W, V)
    ws = _workspace(workspace, dev, sp, other, need) if need > 0 else None
    _call("mtrtq_beam_select", dev.index, logits.data_ptr(), logits.stride(0) if B * W > 1 else V, scores.data_ptr(), done.data_ptr(), eos,
          B, W, V, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
          None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel() * ws.element_size(), sp)
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
    s = k_pages.stride()
    if 0 in (L, P) or s[2:] != (S * D, D, 1) and not k_pages[0, 0].is_contiguous() or v_pages.stride() != s \
            and (v_pages.stride()[:2] != s[:2] or not v_pages[0, 0].is_contiguous()):
        raise ValueError("pages of k_pages and v_pages must be contiguous, and equally far apart")
    B, W = parent.shape
    dev = k_pages.device
    if _ints("parent", parent, (B, W), dev)[0] != W and B > 1:
        raise ValueError("parent must be contiguous")
    width = table.shape[1]
    ld = _ints("table", table, (B * W, width), dev)[0]
    ldo = _ints("owned", owned, (B * W, width), dev)[0]
    if B * W == 1:
        ld = ldo = width
    _ints("kv_len", kv_len, (B,), dev)
    _call("mtrtq_beam_reorder", dev.index, parent.data_ptr(), B, W, table.data_ptr(), ld, owned.data_ptr(),
          ldo, width, kv_len.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), L, s[0], s[1], P, KV, S, D,
          _DTYPES[k_pages.dtype], _stream_ptr(stream, dev.index))
