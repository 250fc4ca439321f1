"""fmha_rope_append, fmha_paged_decode and fmha_prompt against their formulas in 64 bits
(serving_ref.py: the reference and the derived error bounds)."""
import math

import pytest
import torch

import fmha_b200
from tests.serving_ref import attend64, check, gather_pages, rotate64, tiny, u

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
SITE_APPEND_POSITION, SITE_APPEND_PAGE, SITE_DECODE_LENGTH, SITE_DECODE_PAGE, SITE_PROMPT_LENGTH = 16, 17, 18, 19, 20


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return i32(cu)


def make_pool(pages, hkv, size, d, dtype, g, order="hnd"):
    shape = (pages, hkv, size, d) if order == "hnd" else (pages, size, hkv, d)
    x = torch.randn(shape, device="cuda", generator=g)
    x = (x * 20).clamp(-448, 448).to(E4M3) if dtype == E4M3 else x.to(dtype)
    return x if order == "hnd" else x.transpose(1, 2)


def make_table(lens, size, g, spare=2, columns=None):
    counts = [-(-n // size) for n in lens]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max([1, columns or 0] + counts)), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, total


def bits(x):
    return x.contiguous().view(torch.uint8)


def error_site():
    """(status, site) of the device error word, which this clears."""
    code = fmha_b200.device_error()
    return (code & 0xff, code >> 8)


# ---------------------------------------------------------------- append


def angles(positions, rot, g):
    a = torch.rand((positions, rot // 2), device="cuda", generator=g, dtype=torch.float64) * 2 * math.pi
    return a.cos().float(), a.sin().float()


def expected_pools(pool, size, table, places, x64, scale):
    """The pool in fp64 with the new rows put in; True where they are."""
    want = pool.float().double() if pool.dtype == E4M3 else pool.double()
    new = torch.zeros(want.shape[0], want.shape[2], dtype=torch.bool, device="cuda")
    for t, (b, pos) in enumerate(places):
        if b < 0:
            continue
        page = int(table[b, pos // size])
        want[page, :, pos % size] = x64[t] / scale
        new[page, pos % size] = True
    return want, new


@pytest.mark.parametrize("dtype,ctype,d,hq,hkv,size,order,rot,inter,new,past", [
    (BF16, BF16, 128, 32, 8, 16, "hnd", 128, False, [1, 1, 1, 1, 1], [0, 15, 16, 31, 700]),
    (BF16, BF16, 128, 8, 8, 16, "nhd", 128, True, [5, 0, 1, 33, 100], [0, 3, 15, 16, 50]),
    (FP16, FP16, 256, 6, 2, 7, "hnd", 64, False, [17, 1, 2], [0, 6, 7]),
    (FP16, FP16, 128, 5, 5, 1, "nhd", 48, True, [3, 4], [0, 9]),
    (BF16, E4M3, 128, 16, 2, 16, "nhd", 128, False, [40, 1], [2, 31]),
    (FP16, E4M3, 256, 9, 3, 32, "hnd", 256, True, [64, 3, 0], [0, 0, 4]),
    (BF16, E4M3, 256, 3, 1, 48, "hnd", 0, False, [12], [100]),
    (BF16, BF16, 256, 71, 1, 64, "hnd", 16, False, [300, 1, 77], [10, 0, 1000]),
])
def test_append(cuda, dtype, ctype, d, hq, hkv, size, order, rot, inter, new, past):
    g = gen(hq * d + size)
    lens = [n + p for n, p in zip(new, past)]
    table, pages = make_table(lens, size, g)
    pk, pv = make_pool(pages, hkv, size, d, ctype, g, order), make_pool(pages, hkv, size, d, ctype, g, order)
    pad = 3  # rows behind the last sequence
    t = sum(new) + pad
    qkv = randn((t, hq + 2 * hkv, d), g, dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cos, sin = angles(max(lens), rot, g) if rot else (None, None)
    ks, vs = (0.05, 0.04) if ctype == E4M3 else (1.0, 1.0)
    before = qkv.clone()
    pk0, pv0 = pk.clone(), pv.clone()
    q_out = torch.full((t, hq, d), 5.0, dtype=dtype, device="cuda")
    k_out = torch.full((t, hkv, d), 5.0, dtype=dtype, device="cuda")
    got = fmha_b200.fmha_rope_append(q, k, v, pk, pv, table, i32(lens), cos, sin, cu_seqlens_q=starts(new),
                                     interleaved=inter, k_scale=ks, v_scale=vs, q_out=q_out, k_out=k_out)
    assert got[0] is q_out and got[1] is k_out
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    assert torch.equal(bits(qkv), bits(before))
    assert bool((q_out[-pad:] == 5.0).all()) and bool((k_out[-pad:] == 5.0).all())

    places = [(b, p + i) for b, (n, p) in enumerate(zip(new, past)) for i in range(n)]
    n = len(places)
    pos = torch.tensor([p for _, p in places], device="cuda")
    c, s = (cos[pos], sin[pos]) if rot else (torch.zeros(n, 0, device="cuda"),) * 2
    for out, x in ((q_out[:n], q[:n]), (k_out[:n], k[:n])):
        want, mag = rotate64(x, c, s, inter)
        check(out, want, u(dtype) * want.abs() + 2.0 ** -22 * mag + tiny(dtype), "rotated")
    k64, kmag = rotate64(k[:n], c, s, inter)
    for pool, pool0, x64, mag, scale, what in ((pk, pk0, k64, kmag, ks, "k pages"),
                                               (pv, pv0, v[:n].double(), v[:n].double().abs() * 0, vs, "v pages")):
        want, put = expected_pools(pool0, size, table, places, x64, scale)
        m64, _ = expected_pools(torch.zeros_like(pool0, dtype=torch.float32), size, table, places, mag, scale)
        if ctype == E4M3:
            want = want.clamp(-448, 448)
        bound = u(ctype) * want.abs() + 2.0 ** -22 * (m64 + want.abs()) + tiny(ctype)
        got = pool.float() if ctype == E4M3 else pool
        at = put[:, None, :, None].expand_as(want)
        check(torch.where(at, got.double(), want), want, bound, what)
        # Every other row is what it was, bit for bit.
        old = ~put[:, None, :, None].expand_as(pool)
        assert torch.equal(pool.contiguous().view(torch.uint8 if ctype == E4M3 else torch.int16)[old],
                           pool0.contiguous().view(torch.uint8 if ctype == E4M3 else torch.int16)[old])
        if what == "v pages" and ctype != E4M3:
            assert torch.equal(torch.where(at, got.double(), want), want)  # values are copied


def decode_step_inputs(g, b=9, hq=8, hkv=2, d=128, size=16, dtype=BF16):
    lens = [1 + 13 * i for i in range(b)]
    table, pages = make_table(lens, size, g)
    return (lens, table, make_pool(pages, hkv, size, d, dtype, g), make_pool(pages, hkv, size, d, dtype, g),
            randn((b, hq, d), g, dtype), randn((b, hkv, d), g, dtype), randn((b, hkv, d), g, dtype))


def test_append_in_place_and_without_offsets(cuda):
    g = gen(3)
    lens, table, pk, pv, q, k, v = decode_step_inputs(g)
    cos, sin = angles(200, 128, g)
    a, b = pk.clone(), pv.clone()
    q1, k1 = fmha_b200.fmha_rope_append(q, k, v, a, b, table, i32(lens), cos, sin, return_k=True,
                                        cu_seqlens_q=starts([1] * len(lens)))
    q2, k2 = q.clone(), k.clone()
    fmha_b200.fmha_rope_append(q2, k2, v, pk, pv, table, i32(lens), cos, sin, q_out=q2, k_out=k2)
    for x, y in ((q1, q2), (k1, k2), (a, pk), (b, pv)):
        assert torch.equal(bits(x), bits(y))


def test_append_saturates_and_keeps_nan(cuda):
    g = gen(4)
    lens, table, _, _, q, k, v = decode_step_inputs(g)
    pk = torch.zeros(int(table.max()) + 3, 2, 16, 128, device="cuda").to(E4M3)
    pv = pk.clone()
    v[0, 0, 0], v[0, 0, 1], v[0, 0, 2], v[0, 0, 3] = 1e30, -1e30, float("nan"), float("inf")
    fmha_b200.fmha_rope_append(q, k, v, pk, pv, table, i32(lens), None, None, k_scale=0.1, v_scale=0.1)
    row = pv[int(table[0, 0]), 0, 0].float()
    assert row[0] == 448 and row[1] == -448 and torch.isnan(row[2]) and row[3] == 448
    assert fmha_b200.device_error() == 0


@pytest.mark.parametrize("what", ["page", "negative page", "length", "past the table", "position", "more new than all"])
def test_append_leaves_out_what_is_impossible(cuda, what):
    g = gen(5)
    lens, table, pk, pv, q, k, v = decode_step_inputs(g)
    cos, sin = angles(200, 128, g)
    cu, bad = None, 4  # sequence 4 is spoiled
    if what == "page":
        table[bad] = pk.shape[0]
    elif what == "negative page":
        table[bad] = -1
    elif what == "length":
        lens[bad] = -5
    elif what == "past the table":
        lens[bad] = table.shape[1] * 16 + 1
        cos, sin = angles(lens[bad] + 5, 128, g)
    elif what == "position":
        cos, sin = cos[:lens[bad] - 1].contiguous(), sin[:lens[bad] - 1].contiguous()
        bad = [b for b in range(9) if lens[b] > cos.shape[0]]
    else:
        cu, lens[bad] = starts([1] * 9), 0
    bad = bad if isinstance(bad, list) else [bad]
    good = [b for b in range(9) if b not in bad]
    pk0 = pk.clone()
    q_out = torch.full_like(q, 5.0)
    fmha_b200.fmha_rope_append(q, k, v, pk, pv, table, i32(lens), cos, sin, q_out=q_out, cu_seqlens_q=cu)
    torch.cuda.synchronize()
    status, site = error_site()
    assert status == fmha_b200.FMHA_ERR_INVALID_ARG
    assert site == (SITE_APPEND_PAGE if "page" in what else SITE_APPEND_POSITION)
    assert fmha_b200.device_error() == 0  # read and cleared
    assert bool((q_out[bad] == 5.0).all())
    changed = (bits(pk) != bits(pk0)).view(pk.shape[0], -1).any(1).nonzero()[:, 0].tolist()
    assert sorted(changed) == sorted(int(table[b, (lens[b] - 1) // 16]) for b in good)
    want, mag = rotate64(q[good], cos[[lens[b] - 1 for b in good]], sin[[lens[b] - 1 for b in good]], False)
    check(q_out[good], want, u(BF16) * want.abs() + 2.0 ** -22 * mag)


# ---------------------------------------------------------------- decode


def decode_case(lens, hq, hkv, d, size, dtype, ctype, order, seed, out=FP16, scale=0.0, spoil=True, columns=None):
    """Runs fmha_paged_decode with NaN in every row of the pages that no sequence holds, and
    checks output and log-sum-exp."""
    g = gen(seed)
    table, pages = make_table(lens, size, g, columns=columns)
    pk, pv = make_pool(pages, hkv, size, d, ctype, g, order), make_pool(pages, hkv, size, d, ctype, g, order)
    if spoil:
        used = torch.zeros(pages, size, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for i in range(-(-n // size)):
                used[int(table[b, i]), : min(size, n - i * size)] = True
        for pool in (pk, pv):
            flat = pool.view(torch.uint8) if ctype == E4M3 else pool
            flat.masked_fill_(~used[:, None, :, None], 0x7f if ctype == E4M3 else float("nan"))
    ks, vs = (0.05, 0.04) if ctype == E4M3 else (1.0, 1.0)
    q = randn((len(lens), hq, d), g, dtype)
    lse = torch.full((len(lens), hq), 99.0, device="cuda")
    o = fmha_b200.fmha_paged_decode(q, pk, pv, table, i32(lens), k_scale=ks, v_scale=vs, out_dtype=out, lse=lse,
                                    softmax_scale=scale)
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    check_decode(q, pk, pv, table, lens, ks, vs, scale or d ** -0.5, o, lse)
    return o


def check_decode(q, pk, pv, table, lens, ks, vs, scale, o, lse=None):
    hkv = pk.shape[1]
    gq = q.shape[1] // hkv
    p_round = 2 * (2.0 ** -16 if q.dtype == BF16 and pk.dtype != E4M3 else 2.0 ** -21)
    for b, n in enumerate(lens):
        k, v = gather_pages(pk, table[b], n), gather_pages(pv, table[b], n)
        for h in range(hkv):
            rows = slice(h * gq, (h + 1) * gq)
            want, bound, wl, bl = attend64(q[b:b + 1, rows], k[h].double() * ks, v[h].double() * vs,
                                           torch.ones(1, n, dtype=torch.bool, device="cuda"), scale, p_round, o.dtype)
            check(o[b:b + 1, rows], want, bound, f"sequence {b} (length {n}) kv head {h}")
            if lse is not None:
                check(lse[b:b + 1, rows], wl, bl + 2.0 ** -22, f"lse of sequence {b}")


@pytest.mark.parametrize("lens", [[0], [1], [137], [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 500], [2] * 40])
@pytest.mark.parametrize("hq,hkv,d,size,dtype,ctype,order", [
    (16, 16, 128, 16, BF16, BF16, "hnd"), (32, 8, 128, 16, BF16, BF16, "nhd"), (16, 2, 256, 64, FP16, FP16, "hnd"),
    (10, 2, 256, 7, BF16, BF16, "nhd"), (9, 1, 128, 1, FP16, FP16, "hnd"), (32, 2, 256, 33, BF16, BF16, "hnd"),
    (20, 1, 128, 16, BF16, BF16, "hnd"), (40, 1, 256, 16, FP16, FP16, "hnd"),
    (16, 8, 128, 16, BF16, E4M3, "hnd"), (6, 2, 256, 5, BF16, E4M3, "nhd"), (16, 1, 128, 32, FP16, E4M3, "nhd"),
    (24, 2, 256, 16, BF16, E4M3, "hnd"),
])
def test_decode(cuda, lens, hq, hkv, d, size, dtype, ctype, order):
    decode_case(lens, hq, hkv, d, size, dtype, ctype, order, seed=len(lens) * d + hq)


@pytest.mark.parametrize("lens,hq,hkv,d,size,dtype,ctype", [
    ([5000, 3, 0, 1234], 8, 2, 128, 16, BF16, BF16),          # few long rows: split and joined
    ([40001], 4, 1, 128, 48, FP16, FP16),                     # one row over every CTA
    ([9000, 12], 10, 2, 256, 16, BF16, BF16),
    ([7777], 16, 1, 256, 64, BF16, E4M3),
    ([20000, 1], 5, 5, 128, 16, BF16, E4M3),
    ([600] * 70 + [0, 1], 12, 4, 128, 16, BF16, BF16),         # units end anywhere in a CTA's range
    ([100 + 37 * i for i in range(60)], 32, 2, 256, 16, FP16, FP16),
    (list(range(300)), 4, 2, 128, 8, BF16, BF16),              # more sequences than threads
])
def test_decode_split_and_joined(cuda, lens, hq, hkv, d, size, dtype, ctype):
    decode_case(lens, hq, hkv, d, size, dtype, ctype, "hnd", seed=len(lens) + hq, out=BF16 if d == 256 else FP16,
                spoil=sum(lens) < 50000)


def test_decode_is_the_same_split_or_whole(cuda):
    """A wide block table (lengths may be long: split) and a narrow one (whole units) agree
    within both kernels' bounds, and each repeats bit for bit."""
    lens = [300, 17, 1, 480, 0]
    a = decode_case(lens, 8, 2, 128, 16, BF16, BF16, "hnd", seed=2)
    b = decode_case(lens, 8, 2, 128, 16, BF16, BF16, "hnd", seed=2, columns=400)
    assert torch.equal(bits(a), bits(decode_case(lens, 8, 2, 128, 16, BF16, BF16, "hnd", seed=2)))
    assert torch.equal(bits(b), bits(decode_case(lens, 8, 2, 128, 16, BF16, BF16, "hnd", seed=2, columns=400)))


def test_decode_scale_strides_and_shared_pages(cuda):
    g = gen(8)
    size, hkv, gq, d = 16, 2, 3, 128
    pool = randn((9, 2, hkv, size, d), g, BF16)          # keys and values in one allocation
    pk, pv = pool[:, 0], pool[:, 1]
    table = i32([[3, 5, 3, 1], [3, 5, 8, 8], [0, 0, 0, 0]])[:, :4]  # a shared prefix, pages met twice
    wide = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    wide[:, :4] = table
    lens = [64, 55, 40]
    q = randn((3, 2 * hkv * gq, d), g, BF16)[:, hkv * gq:]  # rows of a wider tensor
    o = torch.full((3, 2 * hkv * gq, d), 7.0, dtype=FP16, device="cuda")
    fmha_b200.fmha_paged_decode(q, pk, pv, wide[:, :4], i32(lens), softmax_scale=0.3, o=o[:, :hkv * gq])
    torch.cuda.synchronize()
    check_decode(q, pk, pv, table, lens, 1.0, 1.0, 0.3, o[:, :hkv * gq])
    assert bool((o[:, hkv * gq:] == 7.0).all())


def test_decode_offsets_past_32_bits(cuda):
    """Pages more than 2^31 elements into the pool."""
    size, hkv, d = 64, 8, 128
    pages = (1 << 31) // (size * hkv * d) + 40
    pool = torch.empty((pages, hkv, size, d), dtype=BF16, device="cuda")
    g = gen(9)
    use = [pages - 1, 0, pages - 17, 5, pages - 2]
    for i in use:
        pool[i] = randn((hkv, size, d), g, BF16)
    table, lens = i32([use, use[::-1]]), [310, 257]
    q = randn((2, 16, d), g, BF16)
    o = fmha_b200.fmha_paged_decode(q, pool, pool, table, i32(lens))
    check_decode(q, pool, pool, table, lens, 1.0, 1.0, d ** -0.5, o)


def test_decode_longest_sequence(cuda):
    """Lengths up to the last token number are taken or refused, never read out of range: one
    page stands in every place of the table."""
    size, cols = 1 << 20, 2048
    pool = torch.ones((1, 1, size, 128), dtype=BF16, device="cuda")
    table = torch.zeros((2, cols), dtype=torch.int32, device="cuda")
    q = randn((2, 1, 128), gen(10), BF16)
    o = torch.full((2, 1, 128), 7.0, dtype=FP16, device="cuda")
    for n in (2 ** 31 - 1, 2 ** 31 - 63):
        fmha_b200.fmha_paged_decode(q, pool, pool, table, i32([n, 3]), o=o)
        torch.cuda.synchronize()
        assert error_site() == (fmha_b200.FMHA_ERR_INVALID_ARG, SITE_DECODE_LENGTH)
        assert bool((o[0] == 7.0).all()) and bool((o[1] == 1.0).all())
    fmha_b200.fmha_paged_decode(q, pool, pool, table, i32([3 * size + 17, 3]), o=o)
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    assert bool((o - 1.0).abs().max() <= 2.0 ** -10)


@pytest.mark.parametrize("columns", [None, 100])
@pytest.mark.parametrize("d,ctype,gq", [(128, BF16, 2), (256, BF16, 2), (128, E4M3, 2), (128, FP16, 3),
                                        (128, BF16, 16), (256, FP16, 12)])
def test_decode_nonfinite(cuda, d, ctype, gq, columns):
    """NaN and infinities in keys, values and queries reach exactly the rows and columns that
    the formula takes them to."""
    g = gen(11)
    lens, hkv, size = [40, 40, 40, 40, 40, 0], 2, 16
    dtype = BF16 if ctype == E4M3 else ctype
    table, pages = make_table(lens, size, g, columns=columns)
    pk, pv = make_pool(pages, hkv, size, d, dtype, g), make_pool(pages, hkv, size, d, dtype, g)
    q = randn((6, hkv * gq, d), g, dtype)
    at = lambda b, j: (int(table[b, j // size]), j % size)  # noqa: E731
    p, r = at(0, 39)
    pk[p, 0, r, 3] = float("nan")                       # a NaN score
    p, r = at(1, 20)
    pv[p, 1, r, 7] = float("nan") if ctype == E4M3 else float("inf")
    q[2, 0] = float("nan")
    q[3, 1, 5] = float("inf")
    if ctype != E4M3:
        for j in range(40):
            p, r = at(4, j)
            pk[p, 0, r] = 0
            pk[p, 0, r, 1] = -float("inf")
        q[4, 0] = 1.0                                    # every score -inf: 0/0
        q[4, 1] = -1.0                                   # every score +inf
    if ctype == E4M3:
        pk, pv = (x.float().mul(20).clamp(-448, 448).to(E4M3) for x in (pk, pv))
    ks = 0.05 if ctype == E4M3 else 1.0
    o = fmha_b200.fmha_paged_decode(q, pk, pv, table, i32(lens), k_scale=ks, v_scale=ks)
    torch.cuda.synchronize()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[0, :gq] = True
    bad[2, 0] = True
    bad[3, 1] = True
    if ctype == E4M3:
        bad[1, gq:, 7] = True
    else:
        bad[4, :gq] = True  # the other queries meet -inf in every key too
        assert bool(torch.isinf(o[1, gq:, 7]).all())
    assert torch.equal(torch.isnan(o), bad)
    assert bool((o[5] == 0).all())
    good = ~bad
    good[1, gq:, 7] = False
    assert bool(torch.isfinite(o[good]).all())


@pytest.mark.parametrize("columns", [None, 200])
def test_decode_leaves_out_what_is_impossible(cuda, columns):
    g = gen(12)
    lens, hq, hkv, d, size = [50, 60, 70, 33], 8, 2, 128, 16
    table, pages = make_table(lens, size, g, columns=columns)
    pk, pv = make_pool(pages, hkv, size, d, BF16, g), make_pool(pages, hkv, size, d, BF16, g)
    q = randn((4, hq, d), g, BF16)
    for bad_len in (-1, table.shape[1] * size + 1, 2 ** 31 - 1, -2 ** 31):
        given = list(lens)
        given[1] = bad_len
        o = torch.full((4, hq, d), 7.0, dtype=FP16, device="cuda")
        fmha_b200.fmha_paged_decode(q, pk, pv, table, i32(given), o=o)
        torch.cuda.synchronize()
        assert error_site() == (fmha_b200.FMHA_ERR_INVALID_ARG, SITE_DECODE_LENGTH)
        assert bool((o[1] == 7.0).all())
        keep = [0, 2, 3]
        check_decode(q[keep], pk, pv, table[keep], [lens[b] for b in keep], 1.0, 1.0, d ** -0.5, o[keep])
    for page in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        spoiled = table.clone()
        spoiled[2, 1] = page  # tokens 16..31 of sequence 2 are left out
        o = fmha_b200.fmha_paged_decode(q, pk, pv, spoiled, i32(lens))
        torch.cuda.synchronize()
        assert error_site() == (fmha_b200.FMHA_ERR_INVALID_ARG, SITE_DECODE_PAGE)
        keep = [0, 1, 3]
        check_decode(q[keep], pk, pv, table[keep], [lens[b] for b in keep], 1.0, 1.0, d ** -0.5, o[keep])
        seen = torch.ones(1, 70, dtype=torch.bool, device="cuda")
        seen[0, 16:32] = False
        k, v = gather_pages(pk, table[2], 70), gather_pages(pv, table[2], 70)
        want, bound, _, _ = attend64(q[2:3, :4], k[0], v[0], seen, d ** -0.5, 2.0 ** -15, FP16)
        check(o[2:3, :4], want, bound)


def test_decode_streams_graphs_and_workspace(cuda):
    """A captured call follows the lengths in device memory; a second graph with its own
    workspace replays beside it; a side stream's result is the same bits."""
    g = gen(13)
    lens, hq, hkv, d, size = [900, 40, 1500], 8, 2, 128, 16
    table, pages = make_table([2000, 2000, 2000], size, g)
    pk, pv = make_pool(pages, hkv, size, d, BF16, g), make_pool(pages, hkv, size, d, BF16, g)
    q = randn((3, hq, d), g, BF16)
    n = i32(lens)
    args = (q, pk, pv, table, n)
    want = fmha_b200.fmha_paged_decode(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o = fmha_b200.fmha_paged_decode(*args, stream=side)
    side.synchronize()
    assert torch.equal(o, want)
    with torch.cuda.stream(side):
        fmha_b200.fmha_paged_decode(*args)
    torch.cuda.synchronize()
    need = fmha_b200.fmha_paged_decode_workspace(hq, hkv, d, table.shape[1] * size)
    graphs, outs = [], []
    for own in (False, True):
        out = torch.zeros_like(want)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda") if own else None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fmha_b200.fmha_paged_decode(*args, o=out, workspace=ws)
        graphs.append(graph)
        outs.append(out)
    for grown in ([900, 40, 1500], [901, 41, 1501], [2000, 0, 1]):
        n.copy_(i32(grown))
        torch.cuda.synchronize()
        fresh = fmha_b200.fmha_paged_decode(*args)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, (torch.cuda.current_stream(), side)):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        check_decode(q, pk, pv, table, grown, 1.0, 1.0, d ** -0.5, fresh)
        for out in outs:
            assert torch.equal(out, fresh)
    assert fmha_b200.device_error() == 0


# ---------------------------------------------------------------- prompt


def check_prompt(q, k, v, nq, nk, causal, scale, o, lse=None):
    hkv = k.shape[1]
    gq = q.shape[1] // hkv
    # P enters the second product rounded to the operands' type, or, for an fp16 result of
    # bf16 operands, as two bf16 parts.
    p_round = 2 * (2.0 ** -16 if q.dtype == BF16 and o.dtype == FP16 else u(q.dtype))
    at = ak = 0
    for b, (n, m) in enumerate(zip(nq, nk)):
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        seen = (j <= i + (m - n)) if causal else torch.ones(n, m, dtype=torch.bool, device="cuda")
        for h in range(hkv):
            rows = slice(h * gq, (h + 1) * gq)
            want, bound, wl, bl = attend64(q[at:at + n, rows], k[ak:ak + m, h], v[ak:ak + m, h], seen, scale,
                                           p_round, o.dtype)
            check(o[at:at + n, rows], want, bound, f"sequence {b} ({n} of {m}) kv head {h}")
            if lse is not None:
                check(lse[at:at + n, rows], wl, bl + 2.0 ** -22, f"lse of sequence {b}")
        at += n
        ak += m


def prompt_case(nq, nk, hq, hkv, d, dtype, out, causal, seed, scale=0.0, pad=5):
    g = gen(seed)
    q = randn((sum(nq) + pad, hq, d), g, dtype)
    kv = randn((sum(nk) + pad, 2 * hkv, d), g, dtype)
    kv[sum(nk):] = float("nan")  # behind the last sequence
    q[sum(nq):] = float("nan")
    k, v = kv[:, :hkv], kv[:, hkv:]
    o = torch.full((q.shape[0], hq, d), 7.0, dtype=out, device="cuda")
    lse = torch.full((q.shape[0], hq), 7.0, device="cuda")
    fmha_b200.fmha_prompt(q, k, v, starts(nq), starts(nk), causal=causal, o=o, lse=lse, softmax_scale=scale)
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    assert bool((o[sum(nq):] == 7.0).all()) and bool((lse[sum(nq):] == 7.0).all())
    check_prompt(q, k, v, nq, nk, causal, scale or d ** -0.5, o, lse)


@pytest.mark.parametrize("nq", [[1], [100], [0, 1, 63, 64, 65, 127, 128, 129, 300], [257, 2, 512, 31]])
@pytest.mark.parametrize("hq,hkv,d,dtype,out,causal", [
    (2, 2, 128, BF16, FP16, True), (8, 2, 128, BF16, BF16, True), (6, 2, 128, FP16, FP16, False),
    (5, 1, 128, FP16, BF16, True), (16, 1, 128, BF16, BF16, False), (4, 2, 256, BF16, BF16, True),
    (8, 1, 256, FP16, FP16, True), (3, 1, 256, BF16, FP16, False), (32, 1, 128, BF16, FP16, True),
    (64, 1, 256, BF16, BF16, True), (128, 1, 128, BF16, BF16, True), (256, 1, 128, FP16, FP16, True),
])
def test_prompt(cuda, nq, hq, hkv, d, dtype, out, causal):
    prompt_case(nq, nq, hq, hkv, d, dtype, out, causal, seed=sum(nq) + hq)


@pytest.mark.parametrize("nq,nk", [([5, 130, 64], [700, 130, 65]), ([50, 3, 200, 1], [20, 0, 150, 1000]),
                                   ([1, 1, 1], [0, 1, 2000])])
@pytest.mark.parametrize("hq,hkv,d,dtype,out", [(8, 2, 128, BF16, BF16), (4, 4, 256, FP16, FP16), (3, 1, 128, BF16, FP16)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_with_other_keys_than_queries(cuda, nq, nk, hq, hkv, d, dtype, out, causal):
    """Prefixes, and fewer keys than queries: with a causal mask the first rows see nothing."""
    prompt_case(nq, nk, hq, hkv, d, dtype, out, causal, seed=sum(nk) + hq)


@pytest.mark.parametrize("d,dtype,out", [(128, BF16, BF16), (256, FP16, FP16), (128, BF16, FP16)])
def test_prompt_long(cuda, d, dtype, out):
    prompt_case([2500, 1], [2500, 4000], 4, 2, d, dtype, out, True, seed=d)


@pytest.mark.parametrize("b", [300, 40])
def test_prompt_many_sequences(cuda, b):
    """More sequences than the planning warp sorts, empty ones among them."""
    nq = [(7 * i) % 23 if i % 11 else 140 + i for i in range(b)]
    prompt_case(nq, [n + i % 3 for i, n in enumerate(nq)], 4, 2, 128, BF16, BF16, True, seed=b)


@pytest.mark.parametrize("b,d,hq,out", [(257, 128, 4, BF16), (1000, 256, 8, FP16), (8193, 128, 2, FP16)])
def test_prompt_is_the_same_in_one_call_or_many(cuda, b, d, hq, out):
    """Sequences do not depend on their neighbours: bit for bit what calls of 100 give."""
    g = gen(b)
    nq = [(5 * i) % 4 if i % 301 else 400 for i in range(b)]
    q, k, v = (randn((sum(nq), h, d), g, BF16) for h in (hq, 2, 2))
    o = fmha_b200.fmha_prompt(q, k, v, starts(nq), out_dtype=out)
    at = 0
    for i in range(0, b, 100):
        part = nq[i:i + 100]
        rows = slice(at, at + sum(part))
        at += sum(part)
        if sum(part):
            want = fmha_b200.fmha_prompt(q[rows], k[rows], v[rows], starts(part), out_dtype=out)
            assert torch.equal(bits(o[rows]), bits(want)), i
    assert fmha_b200.device_error() == 0


def test_prompt_leaves_out_impossible_ones_of_many(cuda):
    """Offsets that run back or past the rows, among more sequences than are sorted."""
    g = gen(26)
    b, n, hq, d = 600, 3, 4, 128
    q, k, v = (randn((b * n, h, d), g, BF16) for h in (hq, 2, 2))
    want = fmha_b200.fmha_prompt(q[:300], k[:300], v[:300], starts([n] * 100))
    for bad in (-2 ** 31, -1, 0, 2 ** 31 - 1):
        cu = starts([n] * b)
        cu[350:] = bad
        o = torch.full((b * n, hq, d), 7.0, dtype=FP16, device="cuda")
        fmha_b200.fmha_prompt(q, k, v, cu, o=o)
        torch.cuda.synchronize()
        assert error_site() == (fmha_b200.FMHA_ERR_INVALID_ARG, SITE_PROMPT_LENGTH)
        assert torch.equal(bits(o[:300]), bits(want))
        assert bool((o[349 * n:] == 7.0).all())
    assert fmha_b200.device_error() == 0


@pytest.mark.parametrize("d,dtype,out", [(128, BF16, BF16), (128, BF16, FP16), (256, FP16, FP16), (256, BF16, BF16)])
def test_prompt_repeats(cuda, d, dtype, out):
    """Many short and long pieces in a row, on and on: the same bits every time, and no wait
    that runs out."""
    g = gen(d)
    nq = [1, 700, 33, 128, 5, 260, 64, 1025, 17] * 8
    q, k, v = (randn((sum(nq), h, d), g, dtype) for h in (8, 2, 2))
    cu = starts(nq)
    first = fmha_b200.fmha_prompt(q, k, v, cu, out_dtype=out)
    for _ in range(150):
        o = fmha_b200.fmha_prompt(q, k, v, cu, out_dtype=out)
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    assert torch.equal(bits(o), bits(first))


def test_decode_repeats(cuda):
    g = gen(41)
    lens = [1, 700, 33, 0, 5000, 260, 64, 1025, 17] * 6
    table, pages = make_table(lens, 16, g)
    pk, pv = make_pool(pages, 2, 16, 128, BF16, g), make_pool(pages, 2, 16, 128, BF16, g)
    q, n = randn((len(lens), 8, 128), g, BF16), i32(lens)
    first = fmha_b200.fmha_paged_decode(q, pk, pv, table, n)
    for _ in range(150):
        o = fmha_b200.fmha_paged_decode(q, pk, pv, table, n)
    torch.cuda.synchronize()
    assert fmha_b200.device_error() == 0
    assert torch.equal(bits(o), bits(first))


def test_prompt_large_scores(cuda):
    """Scores of hundreds: the running maximum rises late and far, weights underflow."""
    g = gen(21)
    n, d = 700, 128
    q, k, v = (randn((n, 2, d), g, BF16) for _ in range(3))
    k *= torch.linspace(0.01, 8.0, n, device="cuda")[:, None, None].to(BF16)
    o = fmha_b200.fmha_prompt(q, k, v, starts([n]), softmax_scale=1.0, out_dtype=BF16)
    check_prompt(q, k, v, [n], [n], True, 1.0, o)
    o = fmha_b200.fmha_prompt(q, k.flip(0).contiguous(), v, starts([n]), softmax_scale=1.0, out_dtype=BF16)
    check_prompt(q, k.flip(0), v, [n], [n], True, 1.0, o)


def test_prompt_strided_rows(cuda):
    g = gen(22)
    hq, hkv, d, nq = 4, 2, 128, [70, 200]
    qkv = randn((270, hq + 2 * hkv, d), g, BF16)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    wide = torch.full((270, 2 * hq, d), 7.0, dtype=FP16, device="cuda")
    fmha_b200.fmha_prompt(q, k, v, starts(nq), o=wide[:, hq:])
    check_prompt(q, k, v, nq, nq, True, d ** -0.5, wide[:, hq:])
    assert bool((wide[:, :hq] == 7.0).all())


@pytest.mark.parametrize("d", [128, 256])
def test_prompt_nonfinite(cuda, d):
    """NaN and infinities reach the rows that see their token, and only those."""
    g = gen(23)
    n, hq, hkv = 200, 2, 1
    q, k, v = randn((n, hq, d), g, BF16), randn((n, hkv, d), g, BF16), randn((n, hkv, d), g, BF16)
    k[150, 0, 3] = float("nan")
    v[100, 0, 7] = float("inf")
    v[120, 0, 9] = float("nan")
    q[20, 1] = float("nan")
    o = fmha_b200.fmha_prompt(q, k, v, starts([n]))
    torch.cuda.synchronize()
    nan = torch.zeros_like(o, dtype=torch.bool)
    nan[150:] = True
    nan[120:, :, 9] = True
    nan[20, 1] = True
    assert torch.equal(torch.isnan(o), nan)
    inf = torch.zeros_like(nan)
    inf[100:150, :, 7] = True
    assert torch.equal(torch.isinf(o), inf)


def test_prompt_leaves_out_what_is_impossible(cuda):
    g = gen(24)
    hq, hkv, d = 4, 2, 128
    q, k, v = randn((300, hq, d), g, BF16), randn((300, hkv, d), g, BF16), randn((300, hkv, d), g, BF16)
    for cu_q, cu_k, good in (([0, 100, 200, 301], None, [0, 1]), ([0, 100, 200, 300], [0, 100, 90, 300], [0]),
                             ([0, 100, 200, 300], [0, 100, 2 ** 31 - 1, -2 ** 31], [0])):
        o = torch.full((300, hq, d), 7.0, dtype=FP16, device="cuda")
        fmha_b200.fmha_prompt(q, k, v, i32(cu_q), None if cu_k is None else i32(cu_k), o=o)
        torch.cuda.synchronize()
        assert error_site() == (fmha_b200.FMHA_ERR_INVALID_ARG, SITE_PROMPT_LENGTH)
        n = 100 * len(good)
        check_prompt(q[:n], k[:n], v[:n], [100] * len(good), [100] * len(good), True, d ** -0.5, o[:n])
    assert fmha_b200.device_error() == 0


def test_prompt_graph_and_side_stream(cuda):
    g = gen(25)
    q, k, v = (randn((400, 4, 128), g, BF16) for _ in range(3))
    cu = starts([150, 250])
    want = fmha_b200.fmha_prompt(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o = fmha_b200.fmha_prompt(q, k, v, cu, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(o, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fmha_b200.fmha_prompt(q, k, v, cu, o=out)
    cu.copy_(i32([0, 90, 400]))
    graph.replay()
    torch.cuda.synchronize()
    check_prompt(q, k, v, [90, 310], [90, 310], True, 128 ** -0.5, out)


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("ctype", [BF16, E4M3])
def test_serving_run(cuda, ctype):
    """Prompts in one packed pass, then three steps of one token each: every output against
    the formulas on the whole history."""
    g = gen(31)
    hq, hkv, d, size, prompts, steps = 8, 2, 128, 16, [37, 1, 90], 3
    b = len(prompts)
    table, pages = make_table([n + steps for n in prompts], size, g)
    pk, pv = (torch.zeros((pages, hkv, size, d), dtype=BF16, device="cuda").to(ctype) for _ in range(2))
    ks, vs = (0.02, 0.02) if ctype == E4M3 else (1.0, 1.0)
    cos, sin = angles(200, d, g)
    lens, new = i32(prompts), prompts
    for step in range(steps + 1):
        t = sum(new)
        qkv = randn((t, hq + 2 * hkv, d), g, BF16)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        cu = starts(new)
        if step == 0:
            q, k = fmha_b200.fmha_rope_append(q, k, v, pk, pv, table, lens, cos, sin, cu_seqlens_q=cu,
                                              k_scale=ks, v_scale=vs, return_k=True)
            o = fmha_b200.fmha_prompt(q, k, v, cu)
            check_prompt(q, k, v, new, new, True, d ** -0.5, o)
            if ctype == BF16:  # the pages hold what was kept
                for s in range(b):
                    held = gather_pages(pk, table[s], new[s])
                    assert torch.equal(held, k[int(cu[s]):int(cu[s + 1])].float().transpose(0, 1))
        else:
            lens += 1
            q = fmha_b200.fmha_rope_append(q, k, v, pk, pv, table, lens, cos, sin, k_scale=ks, v_scale=vs)
            o = fmha_b200.fmha_paged_decode(q, pk, pv, table, lens, k_scale=ks, v_scale=vs)
            check_decode(q, pk, pv, table, lens.tolist(), ks, vs, d ** -0.5, o)
        new = [1] * b
    assert fmha_b200.device_error() == 0


def test_torch_ops(cuda):
    """torch.ops.fmha_b200.{rope_append,paged_decode,prompt} make the same calls."""
    import fmha_b200.torch_op  # noqa: F401
    g = gen(33)
    ops = torch.ops.fmha_b200
    new, hq, hkv, d, size = [5, 20], 4, 2, 128, 16
    table, pages = make_table(new, size, g)
    pools = [torch.zeros((pages, hkv, size, d), dtype=BF16, device="cuda") for _ in range(4)]
    q, k, v = (randn((25, h, d), g, BF16) for h in (hq, hkv, hkv))
    cos, sin = angles(32, d, g)
    lens, cu = i32(new), starts(new)
    a = ops.rope_append(q, k, v, pools[0], pools[1], table, lens, cos, sin, cu)
    b = fmha_b200.fmha_rope_append(q, k, v, pools[2], pools[3], table, lens, cos, sin, cu_seqlens_q=cu, return_k=True)
    for x, y in ((a[0], b[0]), (a[1], b[1]), (pools[0], pools[2]), (pools[1], pools[3])):
        assert torch.equal(bits(x), bits(y))
    assert torch.equal(ops.prompt(a[0], a[1], v, cu), fmha_b200.fmha_prompt(a[0], a[1], v, cu))
    q1 = a[0][:2].contiguous()
    assert torch.equal(ops.paged_decode(q1, pools[0], pools[1], table, lens),
                       fmha_b200.fmha_paged_decode(q1, pools[0], pools[1], table, lens))
