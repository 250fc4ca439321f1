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
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import FMHA_ERR_INVALID_ARG, FMHA_ERR_UNSUPPORTED, FmhaError, PagedCacheStruct, check

_TYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_PAGE_TYPES = dict(_TYPES)
_PAGE_TYPES[torch.float8_e4m3fn] = _lib.DTYPE_E4M3


def _refuse(what: str, why: str, status: int = FMHA_ERR_INVALID_ARG):
    _lib.load()
    raise FmhaError(status, f"{what}: {why}")


def _rows(what, name, t, heads, d, dtype, device):
    """Checks a [tokens, heads, d] operand with adjacent heads; its token stride."""
    if t.dim() != 3 or t.shape[2] != d or (heads and t.shape[1] != heads):
        _refuse(what, f"{name} must be [tokens, {heads or 'heads'}, {d}]")
    if t.dtype != dtype:
        _refuse(what, f"{name} must be {dtype}")
    if t.device != device:
        _refuse(what, f"{name} must be on {device}")
    n, h, _ = t.shape
    s0, s1, s2 = t.stride()
    if s2 != 1 or (h > 1 and s1 != d):
        _refuse(what, f"{name}'s heads must be adjacent (strides (*, {d}, 1))")
    return s0 if n > 1 else h * d


def _ints(what, name, t, n, device):
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != device or (
            n > 1 and t.stride(0) != 1):
        _refuse(what, f"{name} must be {n} adjacent int32 on {device}")
    return t.data_ptr()


def _type(what, name, dtype):
    code = _TYPES.get(dtype)
    if code is None:
        _refuse(what, f"{name} must be bf16 or fp16", FMHA_ERR_UNSUPPORTED)
    return code


def _cache(what, k_pages, v_pages, block_table, seqlens_kv, d, k_scale, v_scale, device):
    """The C struct of the cache, its kv heads and its batch."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or k_pages.shape[3] != d:
        _refuse(what, f"k_pages/v_pages must be [num_pages, Hkv, page_size, {d}]")
    st = k_pages.stride()
    if v_pages.stride() != st or st[3] != 1:
        _refuse(what, "k_pages and v_pages must have equal strides and adjacent elements")
    code = _PAGE_TYPES.get(k_pages.dtype)
    if code is None or v_pages.dtype != k_pages.dtype:
        _refuse(what, "pages must be bf16, fp16 or float8_e4m3fn", FMHA_ERR_UNSUPPORTED)
    if k_pages.device != device or v_pages.device != device or block_table.device != device:
        _refuse(what, f"pages and block_table must be on {device}")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        _refuse(what, "block_table must be int32 [batch, max_pages] with adjacent columns")
    batch, cols = block_table.shape
    lens = _ints(what, "seqlens_kv", seqlens_kv, batch, device)
    n, hkv, size, _ = k_pages.shape
    return PagedCacheStruct(k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), lens,
                            st[0], st[1], st[2], block_table.stride(0), n, size, cols, code,
                            k_scale, v_scale), hkv, batch


class _On:
    """q's device and the call's stream as torch's current ones, so that what the call
    allocates belongs to that stream. Costs nothing where they are current already."""

    def __init__(self, what, q, stream):
        if not q.is_cuda:
            _refuse(what, "q must be a CUDA tensor")
        self.inside = []
        if q.device.index != torch.cuda.current_device():
            self.inside.append(torch.cuda.device(q.device))
        if stream is not None:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device=q.device)
            self.inside.append(torch.cuda.stream(stream))
        self.device = q.device

    def __enter__(self):
        for c in self.inside:
            c.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        for c in reversed(self.inside):
            c.__exit__(*exc)
        return False


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
    with _On(what, q, stream) as handle:
        if q.dim() != 3:
            _refuse(what, "q must be [tokens, heads, head_dim]")
        tokens, hq, d = q.shape
        device, dtype = q.device, q.dtype
        code = _type(what, "q", dtype)
        cache, hkv, batch = _cache(what, k_pages, v_pages, block_table, seqlens_kv, d, k_scale,
                                   v_scale, device)
        qs = _rows(what, "q", q, hq, d, dtype, device)
        ks = _rows(what, "k", k, hkv, d, dtype, device)
        vs = _rows(what, "v", v, hkv, d, dtype, device)
        if k.shape[0] != tokens or v.shape[0] != tokens:
            _refuse(what, "q, k and v must have the same tokens")
        cu = 0
        if cu_seqlens_q is not None:
            cu = _ints(what, "cu_seqlens_q", cu_seqlens_q, batch + 1, device)
        elif tokens != batch:
            _refuse(what, "without cu_seqlens_q there must be one token per sequence")
        if (cos is None) != (sin is None):
            _refuse(what, "cos and sin go together")
        rot = positions = cp = sp = 0
        if cos is not None:
            for t in (cos, sin):
                if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape or (
                        not t.is_contiguous() or t.device != device):
                    _refuse(what, "cos and sin must be contiguous fp32 [max_position, rotary_dim/2]")
            positions, rot = cos.shape[0], 2 * cos.shape[1]
            cp, sp = cos.data_ptr(), sin.data_ptr()
        if q_out is None:
            q_out = torch.empty((tokens, hq, d), dtype=dtype, device=device)
        qos = _rows(what, "q_out", q_out, hq, d, dtype, device)
        if k_out is None and return_k:
            k_out = torch.empty((tokens, hkv, d), dtype=dtype, device=device)
        kos, kp = 0, 0
        if k_out is not None:
            kos, kp = _rows(what, "k_out", k_out, hkv, d, dtype, device), k_out.data_ptr()
        if q_out.shape[0] != tokens or (k_out is not None and k_out.shape[0] != tokens):
            _refuse(what, "q_out and k_out must have as many tokens as q")
        check(_lib.load().fmha_rope_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), kp, ctypes.byref(cache), cu,
            cp, sp, tokens, batch, hq, hkv, d, qs, ks, vs, qos, kos, rot, positions,
            1 if interleaved else 0, code, handle), what)
    return q_out if k_out is None else (q_out, k_out)


def fmha_paged_decode_workspace(num_heads_q: int, num_heads_kv: int, head_dim: int) -> int:
    """Bytes of scratch that fmha_paged_decode needs for these heads."""
    n = _lib.load().fmha_paged_decode_workspace(num_heads_q, num_heads_kv, head_dim)
    if n < 0:
        _refuse("fmha_paged_decode_workspace", "unsupported heads", FMHA_ERR_UNSUPPORTED)
    return n


_workspaces: dict = {}  # (Hq, Hkv, D) -> bytes


def fmha_paged_decode(q, k_pages, v_pages, block_table, seqlens_kv, *, softmax_scale=0.0,
                      k_scale=1.0, v_scale=1.0, o=None, out_dtype=None, lse=None, workspace=None,
                      stream=None):
    """Attention of one new token per sequence, q [B,Hq,D], over the cached tokens
    0..seqlens_kv[b]-1. Returns o [B,Hq,D] (fp16, or out_dtype bf16); a fp32 [B,Hq] tensor
    given as lse receives the log-sum-exp of the scaled scores. workspace: a uint8 tensor of
    at least fmha_paged_decode_workspace() bytes for callers that keep one (calls that may
    run at the same time need one each); by default one is allocated."""
    what = "fmha_paged_decode"
    with _On(what, q, stream) as handle:
        if q.dim() != 3:
            _refuse(what, "q must be [batch, heads, head_dim]")
        b, hq, d = q.shape
        device = q.device
        code = _type(what, "q", q.dtype)
        cache, hkv, batch = _cache(what, k_pages, v_pages, block_table, seqlens_kv, d, k_scale,
                                   v_scale, device)
        if batch != b:
            _refuse(what, "q and block_table must have the same batch")
        qs = _rows(what, "q", q, hq, d, q.dtype, device)
        if o is None:
            o = torch.empty((b, hq, d), dtype=out_dtype or torch.float16, device=device)
        elif out_dtype is not None and o.dtype != out_dtype:
            _refuse(what, f"o must be {out_dtype}")
        os = _rows(what, "o", o, hq, d, o.dtype, device)
        if o.shape[0] != b:
            _refuse(what, "o must have q's batch")
        lp = _lse(what, lse, b, hq, device)
        need = _workspaces.get((hq, hkv, d))
        if need is None:
            need = _workspaces[(hq, hkv, d)] = _lib.load().fmha_paged_decode_workspace(hq, hkv, d)
        if workspace is None:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        elif workspace.device != device or not workspace.is_contiguous():
            _refuse(what, f"workspace must be contiguous on {device}")
        check(_lib.load().fmha_paged_decode(
            q.data_ptr(), ctypes.byref(cache), o.data_ptr(), lp, b, hq, hkv, d, qs, os,
            softmax_scale, code, _type(what, "o", o.dtype), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), handle), what)
    return o


def _lse(what, lse, rows, heads, device):
    if lse is None:
        return 0
    if lse.dtype != torch.float32 or lse.shape != (rows, heads) or lse.device != device or (
            not lse.is_contiguous()):
        _refuse(what, f"lse must be contiguous fp32 [{rows}, {heads}] on {device}")
    return lse.data_ptr()


def fmha_prompt(q, k, v, cu_seqlens_q, cu_seqlens_kv=None, *, causal=True, softmax_scale=0.0,
                o=None, out_dtype=None, lse=None, stream=None):
    """Attention over packed prompts: q [Tq,Hq,D], k and v [Tk,Hkv,D], sequence b's rows
    cu_seqlens_q[b] .. cu_seqlens_q[b+1]-1 (keys: cu_seqlens_kv, the same if left out). With
    causal, the last query of a sequence sees all its keys and each earlier one a key less.
    Returns o [Tq,Hq,D] (fp16, or out_dtype bf16); a fp32 [Tq,Hq] tensor given as lse
    receives the log-sum-exp of the scaled scores. Rows behind the last sequence are left as
    they were."""
    what = "fmha_prompt"
    with _On(what, q, stream) as handle:
        if q.dim() != 3 or k.dim() != 3:
            _refuse(what, "q and k must be [tokens, heads, head_dim]")
        tq, hq, d = q.shape
        tk, hkv, _ = k.shape
        device, dtype = q.device, q.dtype
        code = _type(what, "q", dtype)
        qs = _rows(what, "q", q, hq, d, dtype, device)
        ks = _rows(what, "k", k, hkv, d, dtype, device)
        vs = _rows(what, "v", v, hkv, d, dtype, device)
        if v.shape[0] != tk:
            _refuse(what, "k and v must have the same tokens")
        batch = cu_seqlens_q.shape[0] - 1
        cu = _ints(what, "cu_seqlens_q", cu_seqlens_q, batch + 1, device)
        cu_kv = 0
        if cu_seqlens_kv is not None:
            cu_kv = _ints(what, "cu_seqlens_kv", cu_seqlens_kv, batch + 1, device)
        if o is None:
            o = torch.empty((tq, hq, d), dtype=out_dtype or torch.float16, device=device)
        elif out_dtype is not None and o.dtype != out_dtype:
            _refuse(what, f"o must be {out_dtype}")
        os = _rows(what, "o", o, hq, d, o.dtype, device)
        if o.shape[0] != tq:
            _refuse(what, "o must have q's tokens")
        check(_lib.load().fmha_prompt(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _lse(what, lse, tq, hq, device),
            cu, cu_kv, tq, tk, batch, hq, hkv, d, qs, ks, vs, os, softmax_scale,
            1 if causal else 0, code, _type(what, "o", o.dtype), handle), what)
    return o
