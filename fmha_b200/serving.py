"""Serving with a paged KV cache, on torch tensors: the calls of include/fmha.h
``fmha_rope_append``, ``fmha_paged_decode`` and ``fmha_prompt``.

One step of a server, for a batch of sequences whose new tokens are packed
rows (``cu_seqlens_q``; left out when each sequence has one new token):

  q, k = fmha_rope_append(q, k, v, k_pages, v_pages, table, seqlens, cos, sin,
                          cu_seqlens_q=cu, return_k=True)   # fills the pages
  o = fmha_prompt(q, k, v, cu)                              # whole prompts
  o = fmha_paged_decode(q, k_pages, v_pages, table, seqlens)  # one token each

Pages are ``[num_pages, Hkv, page_size, D]`` tensors of any strides with
adjacent D, so a pool stored token by token is passed as
``pool.transpose(1, 2)``. Head dimension 128 or 256; q, k and v bf16 or fp16;
pages of the same type, or float8_e4m3fn with a scale. The calls run on
torch's current stream of q's device (or ``stream``), allocate their outputs
and workspace there, and raise FmhaError for arguments that they refuse.

The checks are written out flat: a decode step makes these calls once per
layer, and at small batches the host's time is what they cost.
"""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from ._lib import FMHA_ERR_INVALID_ARG, FMHA_ERR_UNSUPPORTED, FMHA_OK, FmhaError

_C = _lib.load()
_append, _decode, _prompt = _C.fmha_rope_append, _C.fmha_paged_decode, _C.fmha_prompt
_pack_append = _lib.packer(_lib.RopeAppendArgs)
_pack_decode = _lib.packer(_lib.PagedDecodeArgs)
_pack_prompt = _lib.packer(_lib.PromptArgs)

_TYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_PAGE_TYPES = {**_TYPES, torch.float8_e4m3fn: _lib.DTYPE_E4M3}


def _refuse(what: str, why: str, status: int = FMHA_ERR_INVALID_ARG):
    raise FmhaError(status, f"{what}: {why}")


def _here(what, q, stream):
    """A context with q's device and the call's stream as torch's current ones, so that what
    the call allocates belongs to that stream; None where they are already."""
    if not q.is_cuda:
        _refuse(what, "q must be a CUDA tensor")
    if stream is None and q.get_device() == torch.cuda.current_device():
        return None
    inside = contextlib.ExitStack()
    inside.enter_context(torch.cuda.device(q.device))
    if stream is not None:
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=q.device)
        inside.enter_context(torch.cuda.stream(stream))
    return inside


def _handle(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The same without building a Stream object, where torch offers it.
_handle = getattr(torch._C, "_cuda_getCurrentRawStream", _handle)


def _rows(what, name, t, tokens, heads, d, dtype, device):
    """Checks a [tokens, heads, d] operand with adjacent heads; its token stride."""
    if t.shape != (tokens, heads, d) or t.dtype != dtype or t.get_device() != device:
        _refuse(what, f"{name} must be {dtype} [{tokens}, {heads}, {d}] on cuda:{device}")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != d and heads > 1):
        _refuse(what, f"{name}'s heads must be adjacent (strides (*, {d}, 1))")
    return s0 if tokens > 1 else heads * d


def _ints(what, name, t, n, device):
    if t.dtype != torch.int32 or t.shape != (n,) or t.get_device() != device or (
            n > 1 and t.stride(0) != 1):
        _refuse(what, f"{name} must be {n} adjacent int32 on cuda:{device}")
    return t.data_ptr()


def _type(what, name, dtype):
    code = _TYPES.get(dtype)
    if code is None:
        _refuse(what, f"{name} must be bf16 or fp16", FMHA_ERR_UNSUPPORTED)
    return code


def _pages(what, k_pages, v_pages, block_table, seqlens_kv, d, device):
    """The cache's struct but for its scales, as a tuple; Hkv; batch."""
    shape, st = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape[3] != d or v_pages.shape != shape:
        _refuse(what, f"k_pages and v_pages must be [num_pages, Hkv, page_size, {d}]")
    if v_pages.stride() != st or st[3] != 1:
        _refuse(what, "k_pages and v_pages must have equal strides and adjacent elements")
    dtype = k_pages.dtype
    code = _PAGE_TYPES.get(dtype)
    if code is None or v_pages.dtype != dtype:
        _refuse(what, "pages must both be bf16, fp16 or float8_e4m3fn", FMHA_ERR_UNSUPPORTED)
    if not (k_pages.get_device() == v_pages.get_device() == block_table.get_device() == device):
        _refuse(what, f"pages and block_table must be on cuda:{device}")
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        _refuse(what, "block_table must be int32 [batch, max_pages]")
    batch, columns = block_table.shape
    row, column = block_table.stride()
    if column != 1 and columns > 1:
        _refuse(what, "block_table's columns must be adjacent")
    return (k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
            _ints(what, "seqlens_kv", seqlens_kv, batch, device), st[0], st[1], st[2], row,
            shape[0], shape[2], columns, code), shape[1], batch


def _done(what, status):
    if status != FMHA_OK:
        raise FmhaError(status, what)


def fmha_rope_append(q, k, v, k_pages, v_pages, block_table, seqlens_kv, cos, sin, *,
                     cu_seqlens_q=None, interleaved=False, k_scale=1.0, v_scale=1.0, q_out=None,
                     k_out=None, return_k=False, stream=None):
    """Rotates the new tokens' q [T,Hq,D] and k [T,Hkv,D] by their positions and writes k and
    v [T,Hkv,D] into the pages. Sequence b's new tokens are rows cu_seqlens_q[b] ..
    cu_seqlens_q[b+1]-1 (row b alone without cu_seqlens_q), its last token has position
    seqlens_kv[b]-1. cos and sin are fp32 [max_position, rotary_dim/2]; None for both rotates
    nothing. Returns the rotated q (in q_out if given; q itself may be given), or with
    return_k or k_out the pair (q, rotated k). Rows behind the last sequence are left as they
    were."""
    what = "fmha_rope_append"
    inside = _here(what, q, stream)
    if inside is not None:
        with inside:
            return fmha_rope_append(q, k, v, k_pages, v_pages, block_table, seqlens_kv, cos, sin,
                                    cu_seqlens_q=cu_seqlens_q, interleaved=interleaved,
                                    k_scale=k_scale, v_scale=v_scale, q_out=q_out, k_out=k_out,
                                    return_k=return_k)
    if q.dim() != 3:
        _refuse(what, "q must be [tokens, heads, head_dim]")
    tokens, hq, d = q.shape
    device, dtype = q.get_device(), q.dtype
    code = _type(what, "q", dtype)
    cache, hkv, batch = _pages(what, k_pages, v_pages, block_table, seqlens_kv, d, device)
    qs = _rows(what, "q", q, tokens, hq, d, dtype, device)
    ks = _rows(what, "k", k, tokens, hkv, d, dtype, device)
    vs = _rows(what, "v", v, tokens, hkv, d, dtype, device)
    cu = cos_p = sin_p = rot = positions = 0
    if cu_seqlens_q is not None:
        cu = _ints(what, "cu_seqlens_q", cu_seqlens_q, batch + 1, device)
    if cos is not None and sin is not None:
        positions, rot = cos.shape if cos.dim() == 2 else (0, 0)
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.shape != (positions, rot) or not t.is_contiguous() or (
                    t.get_device() != device):
                _refuse(what, "cos and sin must be contiguous fp32 [max_position, rotary_dim/2]")
        cos_p, sin_p, rot = cos.data_ptr(), sin.data_ptr(), 2 * rot
    elif cos is not sin:
        _refuse(what, "cos and sin go together")
    if q_out is None:
        q_out, qos = torch.empty_like(q, memory_format=torch.contiguous_format), hq * d
    else:
        qos = _rows(what, "q_out", q_out, tokens, hq, d, dtype, device)
    k_out_p, kos = 0, 0
    if k_out is not None:
        kos, k_out_p = _rows(what, "k_out", k_out, tokens, hkv, d, dtype, device), k_out.data_ptr()
    elif return_k:
        k_out, kos = torch.empty_like(k, memory_format=torch.contiguous_format), hkv * d
        k_out_p = k_out.data_ptr()
    status = _append(_pack_append(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_out_p, cu, cos_p, sin_p, qs,
        ks, vs, qos, kos, *cache, k_scale, v_scale, tokens, batch, hq, hkv, d, rot, positions,
        1 if interleaved else 0, code), _handle(device))
    if status != FMHA_OK:
        _done(what, status)
    return q_out if k_out is None else (q_out, k_out)


def fmha_paged_decode_workspace(num_heads_q: int, num_heads_kv: int, head_dim: int,
                                max_tokens: int) -> int:
    """Bytes of scratch that fmha_paged_decode needs for these heads and a block table with
    room for max_tokens (columns * page_size) tokens of a sequence."""
    n = _C.fmha_paged_decode_workspace(num_heads_q, num_heads_kv, head_dim, max_tokens)
    if n < 0:
        _refuse("fmha_paged_decode_workspace", "unsupported sizes", FMHA_ERR_UNSUPPORTED)
    return n


def _lse(what, lse, rows, heads, device):
    if lse.dtype != torch.float32 or lse.shape != (rows, heads) or lse.get_device() != device or (
            not lse.is_contiguous()):
        _refuse(what, f"lse must be contiguous fp32 [{rows}, {heads}] on cuda:{device}")
    return lse.data_ptr()


def _output(what, q, o, out_dtype, tokens, heads, d, device):
    """The output tensor, its type's code and its token stride."""
    if o is None:
        dtype = out_dtype or torch.float16
        code = _type(what, "out_dtype", dtype)
        return torch.empty_like(q, dtype=dtype, memory_format=torch.contiguous_format), code, heads * d
    if out_dtype is not None and o.dtype != out_dtype:
        _refuse(what, f"o must be {out_dtype}")
    code = _type(what, "o", o.dtype)
    return o, code, _rows(what, "o", o, tokens, heads, d, o.dtype, device)


def fmha_paged_decode(q, k_pages, v_pages, block_table, seqlens_kv, *, softmax_scale=0.0,
                      k_scale=1.0, v_scale=1.0, o=None, out_dtype=None, lse=None, workspace=None,
                      stream=None):
    """Attention of one new token per sequence, q [B,Hq,D], over the cached tokens
    0..seqlens_kv[b]-1. Returns o [B,Hq,D] (fp16, or out_dtype bf16); a fp32 [B,Hq] tensor
    given as lse receives the log-sum-exp of the scaled scores. workspace: a tensor of at
    least fmha_paged_decode_workspace() bytes for callers that keep one (calls that may run
    at the same time need one each); by default one is allocated."""
    what = "fmha_paged_decode"
    inside = _here(what, q, stream)
    if inside is not None:
        with inside:
            return fmha_paged_decode(q, k_pages, v_pages, block_table, seqlens_kv,
                                     softmax_scale=softmax_scale, k_scale=k_scale, v_scale=v_scale,
                                     o=o, out_dtype=out_dtype, lse=lse, workspace=workspace)
    if q.dim() != 3:
        _refuse(what, "q must be [batch, heads, head_dim]")
    b, hq, d = q.shape
    device, dtype = q.get_device(), q.dtype
    code = _type(what, "q", dtype)
    cache, hkv, batch = _pages(what, k_pages, v_pages, block_table, seqlens_kv, d, device)
    if batch != b:
        _refuse(what, "q and block_table must have the same batch")
    qs = _rows(what, "q", q, b, hq, d, dtype, device)
    o, o_code, os = _output(what, q, o, out_dtype, b, hq, d, device)
    lse_p = 0 if lse is None else _lse(what, lse, b, hq, device)
    if workspace is None:
        # -1 for heads that the call refuses: allocate nothing and let it say so.
        need = _C.fmha_paged_decode_workspace(hq, hkv, d, cache[9] * cache[10])
        if need > 0:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        ws, size = (workspace.data_ptr(), need) if need > 0 else (0, 0)
    else:
        if workspace.get_device() != device or not workspace.is_contiguous():
            _refuse(what, f"workspace must be contiguous on cuda:{device}")
        ws, size = workspace.data_ptr(), workspace.nbytes
    status = _decode(_pack_decode(
        q.data_ptr(), o.data_ptr(), lse_p, ws, size, qs, os, *cache, k_scale, v_scale, b, hq, hkv,
        d, code, o_code, softmax_scale), _handle(device))
    if status != FMHA_OK:
        _done(what, status)
    return o


def fmha_prompt(q, k, v, cu_seqlens_q, cu_seqlens_kv=None, *, causal=True, softmax_scale=0.0,
                o=None, out_dtype=None, lse=None, stream=None):
    """Attention over packed prompts: q [Tq,Hq,D], k and v [Tk,Hkv,D], sequence b's rows
    cu_seqlens_q[b] .. cu_seqlens_q[b+1]-1 (keys: cu_seqlens_kv, the same if left out). With
    causal, the last query of a sequence sees all its keys and each earlier one a key less.
    Returns o [Tq,Hq,D] (fp16, or out_dtype bf16); a fp32 [Tq,Hq] tensor given as lse
    receives the log-sum-exp of the scaled scores. Rows behind the last sequence are left as
    they were."""
    what = "fmha_prompt"
    inside = _here(what, q, stream)
    if inside is not None:
        with inside:
            return fmha_prompt(q, k, v, cu_seqlens_q, cu_seqlens_kv, causal=causal,
                               softmax_scale=softmax_scale, o=o, out_dtype=out_dtype, lse=lse)
    if q.dim() != 3 or k.dim() != 3:
        _refuse(what, "q and k must be [tokens, heads, head_dim]")
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    device, dtype = q.get_device(), q.dtype
    code = _type(what, "q", dtype)
    qs = _rows(what, "q", q, tq, hq, d, dtype, device)
    ks = _rows(what, "k", k, tk, hkv, d, dtype, device)
    vs = _rows(what, "v", v, tk, hkv, d, dtype, device)
    batch = cu_seqlens_q.shape[0] - 1
    cu = _ints(what, "cu_seqlens_q", cu_seqlens_q, batch + 1, device)
    cu_kv = 0
    if cu_seqlens_kv is not None:
        cu_kv = _ints(what, "cu_seqlens_kv", cu_seqlens_kv, batch + 1, device)
    o, o_code, os = _output(what, q, o, out_dtype, tq, hq, d, device)
    lse_p = 0 if lse is None else _lse(what, lse, tq, hq, device)
    status = _prompt(_pack_prompt(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse_p, cu, cu_kv, qs, ks, vs, os,
        tq, tk, batch, hq, hkv, d, 1 if causal else 0, code, o_code, softmax_scale),
        _handle(device))
    if status != FMHA_OK:
        _done(what, status)
    return o
