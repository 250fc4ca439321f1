"""What the paged-cache entry points refuse. Every refusal comes before the first CUDA call,
so these run without a GPU."""
import ctypes

import pytest

import fmha_b200
from fmha_b200 import _lib

BF16, FP16, E4M3 = _lib.DTYPE_BF16, _lib.DTYPE_FP16, _lib.DTYPE_E4M3
INVALID, UNSUPPORTED, MISALIGNED, OK = (_lib.FMHA_ERR_INVALID_ARG, _lib.FMHA_ERR_UNSUPPORTED,
                                        _lib.FMHA_ERR_MISALIGNED, _lib.FMHA_OK)
NAN, INF = float("nan"), float("inf")

CACHE = dict(k=1 << 20, v=2 << 20, block_table=64, seqlens_kv=128, page_stride=8 * 16 * 128,
             head_stride=16 * 128, token_stride=128, table_stride=10, num_pages=99, page_size=16,
             max_pages=100, dtype=BF16, k_scale=1.0, v_scale=1.0)
COMMON = dict(batch=3, num_heads_q=32, num_heads_kv=8, head_dim=128, q=16, q_stride=4096, dtype=BF16)
APPEND = dict(COMMON, k=32, v=48, q_out=64, k_out=0, cu_seqlens_q=256, cos_table=512, sin_table=1024,
              total_tokens=7, k_stride=1024, v_stride=1024, q_out_stride=4096, k_out_stride=1024,
              rotary_dim=128, max_position=1000, interleaved=0)
DECODE = dict(COMMON, o=32, lse=64, o_stride=4096, softmax_scale=0.0, o_dtype=FP16, workspace=1 << 12,
              workspace_bytes=1 << 24)
PROMPT = dict(COMMON, batch=2, k=32, v=48, o=64, lse=0, cu_seqlens_q=128, cu_seqlens_kv=0, total_q=9,
              total_kv=9, k_stride=1024, v_stride=1024, o_stride=4096, softmax_scale=0.0, causal=1,
              o_dtype=FP16)


def fill(cls, base, kw):
    a = {**base, **{n: x for n, x in kw.items() if not n.startswith("pages_")}}
    if any(n == "cache" for n, _ in cls._fields_):
        a["cache"] = _lib.PagedCacheStruct(**{**CACHE, **{n[6:]: x for n, x in kw.items()
                                                           if n.startswith("pages_")}})
    return ctypes.byref(cls(**a))


def append(**kw):
    return fmha_b200.load().fmha_rope_append(fill(_lib.RopeAppendArgs, APPEND, kw), None)


def decode(**kw):
    return fmha_b200.load().fmha_paged_decode(fill(_lib.PagedDecodeArgs, DECODE, kw), None)


def prompt(**kw):
    return fmha_b200.load().fmha_prompt(fill(_lib.PromptArgs, PROMPT, kw), None)


HEADS = [
    (dict(num_heads_q=0), INVALID), (dict(num_heads_kv=0), INVALID), (dict(num_heads_q=30), INVALID),
    (dict(head_dim=0), INVALID), (dict(head_dim=64), UNSUPPORTED), (dict(head_dim=192), UNSUPPORTED),
    (dict(batch=-1), INVALID), (dict(dtype=E4M3), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED),
    (dict(q=0), INVALID), (dict(q=24), MISALIGNED), (dict(q_stride=4088), INVALID),
    (dict(q_stride=4100), MISALIGNED),
]
PAGES = [({"pages_" + n: x for n, x in kw.items()}, status) for kw, status in [
    (dict(k=0), INVALID), (dict(v=0), INVALID),
    (dict(block_table=0), INVALID), (dict(seqlens_kv=0), INVALID), (dict(num_pages=0), INVALID),
    (dict(page_size=0), INVALID), (dict(max_pages=0), INVALID), (dict(k=8), MISALIGNED),
    (dict(v=(1 << 20) + 4), MISALIGNED), (dict(block_table=66), MISALIGNED),
    (dict(seqlens_kv=129), MISALIGNED), (dict(dtype=FP16), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED),
    (dict(page_stride=-8), INVALID), (dict(page_stride=4), MISALIGNED),
    (dict(head_stride=120), INVALID), (dict(head_stride=2052), MISALIGNED),
    (dict(token_stride=64), INVALID), (dict(token_stride=132), MISALIGNED),
    (dict(dtype=E4M3, token_stride=136), MISALIGNED), (dict(k_scale=0.5), INVALID),
    (dict(dtype=E4M3, k_scale=0.0), INVALID), (dict(dtype=E4M3, v_scale=-1.0), INVALID),
    (dict(dtype=E4M3, v_scale=1e-40), INVALID), (dict(dtype=E4M3, v_scale=NAN), INVALID), (dict(dtype=E4M3, k_scale=INF), INVALID),
    (dict(table_stride=-1), INVALID),
]]


@pytest.mark.parametrize("kw,status", HEADS + PAGES + [
    (dict(total_tokens=-1), INVALID), (dict(k=0), INVALID), (dict(v=40), MISALIGNED),
    (dict(k_stride=1000), INVALID), (dict(v_stride=1028), MISALIGNED), (dict(q_out=0), INVALID),
    (dict(q_out=72), MISALIGNED), (dict(q_out_stride=8), INVALID), (dict(k_out=80, k_out_stride=1000), INVALID),
    (dict(k_out=88), MISALIGNED), (dict(rotary_dim=24), UNSUPPORTED), (dict(rotary_dim=144), UNSUPPORTED),
    (dict(rotary_dim=-16), INVALID), (dict(cos_table=0), INVALID), (dict(sin_table=0), INVALID),
    (dict(max_position=0), INVALID), (dict(cos_table=520), MISALIGNED), (dict(cu_seqlens_q=258), MISALIGNED),
    (dict(cu_seqlens_q=0), INVALID),                       # one token per sequence, but 7 tokens for 3
    (dict(q_out=16, q_out_stride=4104), INVALID),          # in place with another stride
    (dict(k_out=32, k_out_stride=1032), INVALID),
])
def test_append_refuses(kw, status):
    assert append(**kw) == status


@pytest.mark.parametrize("kw,status", HEADS + PAGES + [
    (dict(o=0), INVALID), (dict(o=36), MISALIGNED), (dict(o_stride=4000), INVALID), (dict(lse=66), MISALIGNED),
    (dict(o_dtype=E4M3), UNSUPPORTED), (dict(softmax_scale=-1.0), INVALID), (dict(softmax_scale=NAN), INVALID),
    (dict(softmax_scale=INF), INVALID), (dict(softmax_scale=3e38), INVALID),
    (dict(workspace=0), INVALID), (dict(workspace=(1 << 12) + 8), MISALIGNED),
    (dict(workspace_bytes=1000), INVALID), (dict(batch=1 << 28), UNSUPPORTED),
])
def test_decode_refuses(kw, status):
    assert decode(**kw) == status


@pytest.mark.parametrize("kw,status", HEADS + [
    (dict(total_q=-1), INVALID), (dict(total_kv=-1), INVALID), (dict(k=0), INVALID), (dict(v=56), MISALIGNED),
    (dict(k_stride=1000), INVALID), (dict(v_stride=1028), MISALIGNED), (dict(o=0), INVALID),
    (dict(o=72), MISALIGNED), (dict(o_stride=4092), INVALID), (dict(lse=2), MISALIGNED),
    (dict(cu_seqlens_q=0), INVALID), (dict(cu_seqlens_q=130), MISALIGNED), (dict(cu_seqlens_kv=131), MISALIGNED),
    (dict(total_kv=10), INVALID), (dict(o_dtype=E4M3), UNSUPPORTED), (dict(softmax_scale=-0.5), INVALID),
    (dict(softmax_scale=NAN), INVALID), (dict(o_stride=1 << 31), UNSUPPORTED),
    (dict(softmax_scale=3e38), INVALID), (dict(o=16), INVALID),
])
def test_prompt_refuses(kw, status):
    assert prompt(**kw) == status


def test_empty_calls_are_no_ops():
    assert append(total_tokens=0, q=0, k=0, v=0, q_out=0) == OK
    assert append(batch=0, total_tokens=0, cu_seqlens_q=0, pages_k=0) == OK
    assert decode(batch=0, q=0, o=0, pages_k=0, workspace=0) == OK
    assert prompt(total_q=0, q=0, o=0) == OK
    assert prompt(batch=0) == OK
    lib = fmha_b200.load()
    assert lib.fmha_rope_append(None, None) == lib.fmha_paged_decode(None, None) == INVALID
    assert lib.fmha_prompt(None, None) == INVALID


def test_workspace_size():
    f = fmha_b200.load().fmha_paged_decode_workspace
    assert f(32, 8, 128, 10000) > 0 and f(32, 8, 256, 10000) > f(32, 8, 128, 10000)
    assert f(32, 8, 128, 1 << 40) == f(32, 8, 128, 10000) and f(32, 8, 128, 16) == 0
    assert f(32, 8, 64, 99) == f(30, 8, 128, 99) == f(0, 1, 128, 99) == f(32, 8, 128, -1) == -1
    with pytest.raises(fmha_b200.FmhaError):
        fmha_b200.fmha_paged_decode_workspace(32, 8, 64, 99)
    # A byte less than it says is refused.
    assert decode(workspace_bytes=f(32, 8, 128, 1600) - 1) == INVALID


STRUCTS = dict(fmha_paged_cache_t=_lib.PagedCacheStruct, fmha_rope_append_args_t=_lib.RopeAppendArgs,
               fmha_paged_decode_args_t=_lib.PagedDecodeArgs, fmha_prompt_args_t=_lib.PromptArgs)


def test_struct_layouts_match_the_header(tmp_path):
    """The ctypes structs are the C structs: offsets printed by a compiled program."""
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines, want = [], []
    for name, cls in STRUCTS.items():
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"fmha.h\"\nint main(void) {\n"
                   + "\n".join(lines) + "\n  return 0;\n}\n")
    subprocess.check_call([cc, "-I" + os.path.join(root, "include"), str(src), "-o", str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want


def test_python_refuses_cpu_tensors():
    import torch
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(fmha_b200.FmhaError):
        fmha_b200.fmha_prompt(q, q, q, cu)
    pool = torch.zeros(4, 4, 16, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(fmha_b200.FmhaError):
        fmha_b200.fmha_paged_decode(q, pool, pool, table, lens)
    with pytest.raises(fmha_b200.FmhaError):
        fmha_b200.fmha_rope_append(q, q, q, pool, pool, table, lens, None, None)
