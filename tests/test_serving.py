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
             max_pages=10, dtype=BF16, k_scale=1.0, v_scale=1.0)


def cache(**kw):
    c = dict(CACHE)
    c.update(kw)
    return ctypes.byref(_lib.PagedCacheStruct(**c))


def split(kw, base):
    return {**base, **{a: b for a, b in kw.items() if a in base}}, \
        {a: b for a, b in kw.items() if a not in base}


def append(**kw):
    a, c = split(kw, dict(q=16, kn=32, vn=48, q_out=64, k_out=0, cu=256, cos=512, sin=1024, tokens=7,
                          batch=3, hq=32, hkv=8, d=128, qs=4096, ks=1024, vs=1024, qos=4096, kos=1024,
                          rot=128, positions=1000, inter=0, type=BF16, struct=True))
    return fmha_b200.load().fmha_rope_append(
        a["q"], a["kn"], a["vn"], a["q_out"], a["k_out"], cache(**c) if a["struct"] else None, a["cu"],
        a["cos"], a["sin"], a["tokens"], a["batch"], a["hq"], a["hkv"], a["d"], a["qs"], a["ks"],
        a["vs"], a["qos"], a["kos"], a["rot"], a["positions"], a["inter"], a["type"], None)


def decode(**kw):
    a, c = split(kw, dict(q=16, o=32, lse=64, batch=3, hq=32, hkv=8, d=128, qs=4096, os=4096, scale=0.0,
                          type=BF16, otype=FP16, ws=1 << 12, bytes=1 << 24, struct=True))
    return fmha_b200.load().fmha_paged_decode(
        a["q"], cache(**c) if a["struct"] else None, a["o"], a["lse"], a["batch"], a["hq"], a["hkv"],
        a["d"], a["qs"], a["os"], a["scale"], a["type"], a["otype"], a["ws"], a["bytes"], None)


def prompt(**kw):
    a = dict(q=16, k=32, v=48, o=64, lse=0, cu=128, cu_kv=0, tq=9, tk=9, batch=2, hq=32, hkv=8, d=128,
             qs=4096, ks=1024, vs=1024, os=4096, scale=0.0, causal=1, type=BF16, otype=FP16)
    a.update(kw)
    return fmha_b200.load().fmha_prompt(
        a["q"], a["k"], a["v"], a["o"], a["lse"], a["cu"], a["cu_kv"], a["tq"], a["tk"], a["batch"],
        a["hq"], a["hkv"], a["d"], a["qs"], a["ks"], a["vs"], a["os"], a["scale"], a["causal"],
        a["type"], a["otype"], None)


HEADS = [
    (dict(hq=0), INVALID), (dict(hkv=0), INVALID), (dict(hq=30), INVALID), (dict(d=0), INVALID),
    (dict(d=64), UNSUPPORTED), (dict(d=192), UNSUPPORTED), (dict(batch=-1), INVALID),
    (dict(type=E4M3), UNSUPPORTED), (dict(type=7), UNSUPPORTED),
    (dict(q=0), INVALID), (dict(q=24), MISALIGNED),
    (dict(qs=4088), INVALID), (dict(qs=4100), MISALIGNED),
]
PAGES = [
    (dict(struct=False), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID),
    (dict(block_table=0), INVALID), (dict(seqlens_kv=0), INVALID), (dict(num_pages=0), INVALID),
    (dict(page_size=0), INVALID), (dict(max_pages=0), INVALID), (dict(k=8), MISALIGNED),
    (dict(v=(1 << 20) + 4), MISALIGNED), (dict(block_table=66), MISALIGNED),
    (dict(seqlens_kv=129), MISALIGNED), (dict(dtype=FP16), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED),
    (dict(page_stride=-8), INVALID), (dict(page_stride=4), MISALIGNED),
    (dict(head_stride=120), INVALID), (dict(head_stride=2052), MISALIGNED),
    (dict(token_stride=64), INVALID), (dict(token_stride=132), MISALIGNED),
    (dict(dtype=E4M3, token_stride=136), MISALIGNED), (dict(k_scale=0.5), INVALID),
    (dict(dtype=E4M3, k_scale=0.0), INVALID), (dict(dtype=E4M3, v_scale=-1.0), INVALID),
    (dict(dtype=E4M3, v_scale=NAN), INVALID), (dict(dtype=E4M3, k_scale=INF), INVALID),
    (dict(table_stride=-1), INVALID),
]


@pytest.mark.parametrize("kw,status", HEADS + PAGES + [
    (dict(tokens=-1), INVALID), (dict(kn=0), INVALID), (dict(vn=40), MISALIGNED), (dict(ks=1000), INVALID),
    (dict(vs=1028), MISALIGNED), (dict(q_out=0), INVALID), (dict(q_out=72), MISALIGNED),
    (dict(qos=8), INVALID), (dict(k_out=80, kos=1000), INVALID), (dict(k_out=88), MISALIGNED),
    (dict(rot=24), UNSUPPORTED), (dict(rot=144), UNSUPPORTED), (dict(rot=-16), INVALID),
    (dict(cos=0), INVALID), (dict(sin=0), INVALID), (dict(positions=0), INVALID),
    (dict(cos=520), MISALIGNED), (dict(cu=258), MISALIGNED),
    (dict(cu=0), INVALID),                       # one token per sequence, but 7 tokens for 3
    (dict(q_out=16, qos=4104), INVALID),         # in place with another stride
    (dict(k_out=32, kos=1032), INVALID),
])
def test_append_refuses(kw, status):
    assert append(**kw) == status


@pytest.mark.parametrize("kw,status", HEADS + PAGES + [
    (dict(o=0), INVALID), (dict(o=36), MISALIGNED), (dict(os=4000), INVALID), (dict(lse=66), MISALIGNED),
    (dict(otype=E4M3), UNSUPPORTED), (dict(scale=-1.0), INVALID), (dict(scale=NAN), INVALID),
    (dict(scale=INF), INVALID), (dict(ws=0), INVALID), (dict(ws=(1 << 12) + 8), MISALIGNED),
    (dict(bytes=1000), INVALID), (dict(batch=1 << 28), UNSUPPORTED),
])
def test_decode_refuses(kw, status):
    assert decode(**kw) == status


@pytest.mark.parametrize("kw,status", HEADS + [
    (dict(tq=-1), INVALID), (dict(tk=-1), INVALID), (dict(k=0), INVALID), (dict(v=56), MISALIGNED),
    (dict(ks=1000), INVALID), (dict(vs=1028), MISALIGNED), (dict(o=0), INVALID), (dict(o=72), MISALIGNED),
    (dict(os=4092), INVALID), (dict(lse=2), MISALIGNED), (dict(cu=0), INVALID), (dict(cu=130), MISALIGNED),
    (dict(cu_kv=131), MISALIGNED), (dict(tk=10), INVALID), (dict(otype=E4M3), UNSUPPORTED),
    (dict(scale=-0.5), INVALID), (dict(scale=NAN), INVALID),
])
def test_prompt_refuses(kw, status):
    assert prompt(**kw) == status


def test_empty_calls_are_no_ops():
    assert append(tokens=0, q=0, kn=0, vn=0, q_out=0) == OK
    assert append(batch=0, tokens=0, cu=0, struct=False) == OK
    assert decode(batch=0, q=0, o=0, struct=False, ws=0) == OK
    assert prompt(tq=0, q=0, o=0) == OK
    assert prompt(batch=0) == OK


def test_workspace_size():
    f = fmha_b200.load().fmha_paged_decode_workspace
    assert f(32, 8, 128) > 0 and f(32, 8, 256) > f(32, 8, 128)
    assert f(32, 8, 64) == f(30, 8, 128) == f(0, 1, 128) == -1
    with pytest.raises(fmha_b200.FmhaError):
        fmha_b200.fmha_paged_decode_workspace(32, 8, 64)
    # A byte less than it says is refused.
    assert decode(bytes=f(32, 8, 128) - 1) == INVALID


def test_struct_layout_matches_the_header(tmp_path):
    """The ctypes struct is the C struct: offsets printed by a compiled program."""
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.PagedCacheStruct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "fmha.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu\\n", offsetof(fmha_paged_cache_t, {n}));\n' for n in names) +
        '  printf("%zu\\n", sizeof(fmha_paged_cache_t));\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.check_call([cc, "-I" + os.path.join(root, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    want = [getattr(_lib.PagedCacheStruct, n).offset for n in names]
    assert got == want + [ctypes.sizeof(_lib.PagedCacheStruct)]


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
