"""The attention-block operators on the GPU against 64-bit statements of their formulas: rotary positions, the paged
cache append, packed attention with modified scores, paged attention, and a run of them together."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

import attention_block_reference as R
from infinity_b200 import _lib

pytestmark = pytest.mark.gpu
NAN = math.nan


# -- rotary positions ---------------------------------------------------------------------------
def _rope(lib, x, out, d, heads, dim, positions=None, cu=None, start=None):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(lib.b200emb_op_rope(x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), ptr(positions), ptr(cu), ptr(start),
                                   0 if cu is None else len(cu) - 1, x.shape[0], heads, dim, C.byref(d), R.stream()))
    torch.cuda.synchronize()
    return out


ROPES = [
    dict(rot=128), dict(rot=64, layout="interleaved"), dict(rot=32, scaling="linear", factor=4.0),
    dict(rot=128, scaling="ntk", factor=8.0, theta=1e6), dict(rot=64, scaling="bands", factor=8.0, theta=5e5, low=1.0, high=4.0),
    dict(rot=128, layout="interleaved", scaling="yarn", factor=16.0, theta=1e6, low=32.0, high=1.0),
    dict(rot=24, inverse=1), dict(rot=6), dict(rot=6, layout="interleaved"), dict(rot=2), dict(rot=10, layout="interleaved"),
    dict(rot=64, scaling="yarn", factor=4.0, low=32.0, high=1.0, magnitude=1.25, inverse=1),
]


@pytest.mark.parametrize("kw", ROPES, ids=lambda k: "-".join(str(v) for v in k.values()))
@pytest.mark.parametrize("lens", [[1], [3, 0, 130, 1, 17, 0]], ids=str)
def test_rope_packed_positions(lib, kw, lens):
    heads, dim = 5, 128
    d = R.rope_desc(**kw)
    x = R.normal(sum(lens) + kw["rot"], sum(lens), heads * dim)
    start = R.ints([7 * i for i in range(len(lens))])
    out = _rope(lib, x, torch.empty_like(x), d, heads, dim, cu=R.cu_of(lens), start=start)
    pos = torch.cat([torch.arange(n, device="cuda") + 7 * i for i, n in enumerate(lens)])
    want, size = R.rotate(x.view(-1, heads, dim), pos, d)
    R.assert_rotated(out.view(-1, heads, dim), want, size)
    rest = slice(kw["rot"], dim)
    assert torch.equal(out.view(-1, heads, dim)[..., rest], x.view(-1, heads, dim)[..., rest])
    again = x.clone()
    _rope(lib, again, again, d, heads, dim, cu=R.cu_of(lens), start=start)  # in place
    assert torch.equal(again, out)


def test_rope_far_and_negative_positions(lib):
    d = R.rope_desc(64, theta=1e6)
    pos = R.ints([0, 1, -1, 131071, 1_000_003, 2**31 - 1, -2**31])
    x = R.normal(5, 7, 3 * 64)
    out = _rope(lib, x, torch.empty_like(x), d, 3, 64, positions=pos)
    R.assert_rotated(out.view(7, 3, 64), *R.rotate(x.view(7, 3, 64), pos, d))


@pytest.mark.parametrize("dim,shift,stride", [(96, 0, 300), (64, 1, 195), (64, 2, 198), (64, 4, 196), (7, 0, 21)])
def test_rope_strides_and_alignment(lib, dim, shift, stride):
    """Rows at any element offset and stride, heads of odd size; what lies between the rows stays."""
    heads, n = 3, 9
    rot = min(dim // 2 * 2, 48)
    store = R.normal(dim + shift, n * stride + 8)
    x = store[shift:].as_strided((n, heads * dim), (stride, 1))
    for layout in ("half", "interleaved"):
        d = R.rope_desc(rot, layout)
        back = torch.full((n * stride + 8,), 3.0, dtype=R.BF16, device="cuda")
        out = back[shift:].as_strided((n, heads * dim), (stride, 1))
        _rope(lib, x, out, d, heads, dim, positions=torch.arange(n, dtype=torch.int32, device="cuda"))
        R.assert_rotated(out.reshape(n, heads, dim), *R.rotate(x.reshape(n, heads, dim), torch.arange(n, device="cuda"), d))
        out.fill_(3.0)
        assert (back == 3.0).all()


def test_rope_leaves_rows_of_no_sequence(lib):
    x, out = R.normal(1, 10, 64), torch.full((10, 64), 3.0, dtype=R.BF16, device="cuda")
    _rope(lib, x, out, R.rope_desc(64), 1, 64, cu=R.cu_of([2, 4]))
    assert (out[6:] == 3.0).all() and not (out[:6] == 3.0).all()


def test_rope_inverse_is_the_gradient(lib):
    """The transposed rotation of g against central differences of sum(g * rope(x)) in 64 bits, and against the formula."""
    n, dim = 4, 16
    d, back = R.rope_desc(12, "interleaved"), R.rope_desc(12, "interleaved", inverse=1)
    pos = R.ints([0, 3, 50, 1000])
    g = R.normal(2, n, dim)
    got = _rope(lib, g, torch.empty_like(g), back, 1, dim, positions=pos)
    x = R.normal(3, n, dim).double()
    f = lambda x: (R.rotate(x.view(n, 1, dim), pos, d)[0].view(n, dim) * g.double()).sum()  # noqa: E731
    num = torch.zeros_like(x)
    for i in range(n):
        for j in range(dim):
            e = torch.zeros_like(x)
            e[i, j] = 0.5
            num[i, j] = f(x + e) - f(x - e)  # linear in x: exact up to rounding
    _, size = R.rotate(g.view(n, 1, dim), pos, back)
    R.assert_rotated(got.view(n, 1, dim), num.view(n, 1, dim), size + 1e-9)


# -- cache append -------------------------------------------------------------------------------
@pytest.mark.parametrize("page,by_head,dim,pad", [(16, False, 128, 0), (8, True, 64, 0), (24, False, 96, 8), (5, True, 32, 3), (64, True, 128, 0)])
@pytest.mark.parametrize("rope", [None, dict(rot=32, layout="interleaved"), dict(rot=32)], ids=str)
def test_append(lib, page, by_head, dim, pad, rope):
    heads, kv_heads = 6, 2
    new, old = [1, 40, 0, 7, 3], [0, 5, 9, 63, 130]
    kv = [n + o for n, o in zip(new, old)]
    pages = R.Pages(kv, kv_heads, dim, page, by_head, pad=pad)
    before = [pages.k.clone(), pages.v.clone()]
    t = sum(new)
    qkv = R.normal(9, t, (heads + 2 * kv_heads) * dim)
    q_out = torch.empty(t, heads * dim, dtype=R.BF16, device="cuda")
    d = None if rope is None else R.rope_desc(**rope)
    cu = R.cu_of(new)
    R.append(lib, qkv, cu, R.ints(kv), heads, pages, d, q_out)
    x = qkv.view(t, -1, dim)
    turned = x[:, :heads + kv_heads].contiguous()
    pos = torch.cat([torch.arange(n, device="cuda") + o for n, o in zip(new, old)]).to(torch.int32)
    if d is not None:  # the rotation is the operator's own, bit for bit
        turned = _rope(lib, turned.view(t, -1), torch.empty_like(turned).view(t, -1), d, heads + kv_heads, dim, positions=pos).view(t, -1, dim)
    assert torch.equal(q_out.view(t, heads, dim), turned[:, :heads])
    want = R.Pages(kv, kv_heads, dim, page, by_head, pad=pad)
    for i, n in enumerate(new):
        rows = slice(int(cu[i]), int(cu[i]) + n)
        want.put("k", i, pos[rows], turned[rows, heads:])
        want.put("v", i, pos[rows], x[rows, heads + kv_heads:])
    for got, exp, was in ((pages.k, want.k, before[0]), (pages.v, want.v, before[1])):
        assert torch.equal(got.view(torch.int16) if got.is_contiguous() else got.contiguous().view(torch.int16),
                           exp.contiguous().view(torch.int16))
        assert got.isnan().any() and was.isnan().all()
    # without q_out only the cache is written
    again = R.Pages(kv, kv_heads, dim, page, by_head, pad=pad)
    R.append(lib, qkv, cu, R.ints(kv), heads, again, d, None)
    assert torch.equal(again.k.contiguous().view(torch.int16), want.k.contiguous().view(torch.int16))


def test_append_skips_slots_that_do_not_exist(lib):
    """A length below the new tokens', a table that is too short, pages outside the cache: nothing else is written."""
    heads, kv_heads, dim = 2, 1, 32
    pages = R.Pages([16, 16, 16], kv_heads, dim, 8, table_extra=0)
    pages.table[1, 1] = 1 << 20
    pages.table[2, 0] = -1
    kv = R.ints([2, 16, 18])  # first: 3 of 5 tokens are at negative positions; third: two lie past the table
    new = [5, 4, 12]
    qkv, q_out = R.normal(4, 21, 4 * dim), torch.empty(21, heads * dim, dtype=R.BF16, device="cuda")
    R.append(lib, qkv, R.cu_of(new), kv, heads, pages, None, q_out)
    assert torch.equal(q_out, qkv[:, :heads * dim])
    v = qkv[:, 3 * dim:].view(-1, 1, dim)
    want = torch.full_like(pages.v, NAN)
    want[pages.table[0, 0], 0:2] = v[3:5]
    want[pages.table[2, 1], 0:8] = v[9 + 2:9 + 10]  # positions 8 .. 15 of 6 .. 17
    assert torch.equal(pages.v.view(torch.int16), want.view(torch.int16))


# -- packed attention -----------------------------------------------------------------------------
def _slopes(heads):
    return torch.tensor([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], device="cuda")


def _bias(heads, radius, seed=3):
    return torch.randn(heads, 2 * radius + 1, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 2


def _docs(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = [torch.randint(-1, 3, (max(1, n // 20 + 1),), generator=g).repeat_interleave(20)[:n] for n in lens]
    return torch.cat(rows).to(torch.int32).cuda()


MODS = {
    "plain": {}, "causal": dict(causal=1), "cap": dict(cap=30.0), "cap_causal_window": dict(cap=20.0, causal=1, left=37),
    "small_cap": dict(cap=2.0), "scale": dict(scale=0.03), "window": dict(left=5, right=11), "window_zero": dict(left=0, right=0),
    "slopes": dict(slopes=True), "slopes_causal": dict(slopes=True, causal=1), "bias": dict(bias=9), "bias_point": dict(bias=0),
    "bias_wide_causal": dict(bias=1023, causal=1), "prefix": dict(causal=1, prefix=True), "prefix_window": dict(causal=1, left=3, prefix=True),
    "docs": dict(docs=True), "docs_causal_slopes": dict(docs=True, causal=1, slopes=True), "docs_prefix": dict(docs=True, prefix=True, causal=1),
    "all": dict(cap=15.0, bias=40, causal=1, left=100, prefix=True, docs=True),
}
SHAPES = [  # lengths, heads, key heads, head_dim
    ([1], 1, 1, 64), ([24], 12, 12, 64), ([1, 2, 127, 128, 129, 0, 17, 300], 4, 4, 64), ([0, 257, 0, 31], 4, 2, 128), ([70, 5], 7, 1, 128),
    ([33, 140], 6, 3, 32), ([65, 1], 2, 1, 96), ([40], 3, 3, 8), ([150], 10, 2, 80),
]


def _scored_case(lens, heads, kv_heads, dim, mod, seed=0, gain=2.0):
    mod = dict(mod)
    t = sum(lens)
    x = R.normal(seed + t, t, (heads + 2 * kv_heads) * dim)
    x[:, :heads * dim] *= gain * (4 if mod.get("cap") else 1)
    slopes = _slopes(heads) if mod.pop("slopes", False) else None
    radius = mod.pop("bias", None)
    bias = None if radius is None else _bias(heads, radius)
    prefix = R.ints([n // 3 for n in lens]) if mod.pop("prefix", False) else None
    docs = _docs(lens) if mod.pop("docs", False) else None
    return x, mod, slopes, bias, prefix, docs


def _split(x, heads, kv_heads, dim):
    return x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:]


def _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs):
    at = 0
    for i, n in enumerate(lens):
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        dd = None if docs is None else docs[rows]
        want, size = R.attend(q[rows].reshape(n, heads, dim), k[rows].reshape(n, kv_heads, dim), v[rows].reshape(n, kv_heads, dim), 0,
                              scale=mod.get("scale"), cap=mod.get("cap", 0.0), left=mod.get("left", -1),
                              right=0 if mod.get("causal") else mod.get("right", -1), slopes=slopes, bias=bias,
                              prefix=0 if prefix is None else int(prefix[i]), q_docs=dd, k_docs=dd)
        R.assert_attended(out[rows], want, size)


@pytest.mark.parametrize("name", list(MODS))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scored(lib, shape, name):
    lens, heads, kv_heads, dim = shape
    x, mod, slopes, bias, prefix, docs = _scored_case(*shape, MODS[name])
    q, k, v = _split(x, heads, kv_heads, dim)
    o = R.options(slopes=slopes, bias=bias, prefix=prefix, docs=docs, **mod)
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, o)
    _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)
    assert torch.equal(out, R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, o))  # the same bits every time


@pytest.mark.parametrize("shape,name", [(([3000], 2, 2, 64), "slopes"), (([2049, 700], 4, 1, 128), "cap_causal_window"),
                                        (([1500, 1025], 2, 2, 32), "all"), (([2600], 14, 2, 128), "causal"),
                                        (([90] * 60, 12, 12, 64), "plain"), (([4000, 1], 1, 1, 64), "docs"),
                                        (([3100], 2, 2, 64), "prefix_window")], ids=str)
def test_scored_long(lib, shape, name):
    lens, heads, kv_heads, dim = shape
    x, mod, slopes, bias, prefix, docs = _scored_case(*shape, MODS[name])
    q, k, v = _split(x, heads, kv_heads, dim)
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(slopes=slopes, bias=bias, prefix=prefix, docs=docs, **mod))
    _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("mod", [dict(cap=100.0), dict(cap=1e4, causal=1), dict(cap=1e7), dict(cap=2e38), dict(cap=1e-3), dict(cap=1e-42),
                                 dict(cap=1e6, slopes=True), dict(scale=-0.2), dict(scale=-0.1, cap=9.0), dict(scale=-0.3, slopes=True, causal=1),
                                 dict(scale=1e-42, slopes=True)], ids=str)
def test_scored_caps_and_scales_of_any_size(lib, mod, dim):
    lens, heads, kv_heads = [3, 200, 64], 4, 2
    x, mod, slopes, bias, prefix, docs = _scored_case(lens, heads, kv_heads, dim, mod)
    q, k, v = _split(x, heads, kv_heads, dim)
    q[1] = 0.0  # scores of zero
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(slopes=slopes, **mod))
    _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [56.0, 1e3, 1e5, 1e6])
def test_scored_large_caps_at_scores_of_their_size(lib, cap, dim):
    """Scores of a hundredth of the cap up to all of it, keys a few units apart, and values that show each key's weight. The products are exact
    (small whole numbers), so what is left is the arithmetic of cap * tanh(s / cap) in fp32: two roundings of the argument, one unit in the last
    place of tanh, two roundings of cap * log2(e), one of the sum with the reference, 7 * 2^-24 of the score altogether."""
    n, far = 48, [0.01, 0.05, 0.0999, 0.1001, 0.102, 0.11, 0.13, 0.16, 0.2, 0.25, 0.3, 0.35, 0.4, 0.45, 0.5, 0.6, 0.8, 1.0]
    rows = len(far) * 16
    g = torch.Generator().manual_seed(7)
    want_at = torch.tensor(far).repeat_interleave(16) * cap
    q, k = torch.zeros(rows, dim), torch.zeros(rows, dim)
    # s = 128 q0 + q1 + k1: q0 and q1 of the row, k1 of the key
    q[:, 0] = (want_at / 128).floor().clamp(max=255) if cap < 3e4 else (want_at / 128).to(R.BF16).float()
    q[:, 1], q[:, 2] = torch.randint(0, 128, (rows,), generator=g).float() * (cap > 500), 1.0
    k[:, 0], k[:, 1], k[:, 2] = 128.0, 1.0, torch.randint(-3, 4, (rows,), generator=g).float()
    v = torch.eye(dim)[torch.arange(rows) % n]
    q, k, v = (z.to(R.BF16).cuda() for z in (q, k, v))
    # blocks of one document: every query sees the n keys of its own block
    docs = (torch.arange(rows) // n).to(torch.int32).cuda()
    out = R.scored(lib, q, k, v, R.cu_of([rows]), 1, 1, R.options(scale=1.0, cap=cap, docs=docs)).double()
    want, size = R.attend(*(z.view(rows, 1, dim) for z in (q, k, v)), 0, scale=1.0, cap=cap, q_docs=docs, k_docs=docs)
    s = (q.double() @ k.double().T).abs()
    top = (cap * torch.tanh(torch.where(docs[:, None] == docs[None], s, 0.0) / cap)).amax(1)
    off = torch.expm1(2 * 7 * 2.0 ** -24 * top)[:, None]  # of a weight: its own exponent, and those of the sum
    tol = size.view(rows, dim) * (R.HALF_STEP * (1 + off) + off) + want.view(rows, dim) * R.HALF_STEP * (1 + off)
    bad = ((out - want.view(rows, dim)).abs() - tol).amax(1)
    assert torch.isfinite(out).all() and (bad <= 0).all(), [(f, round(b, 4)) for f, b in zip(far, bad.view(-1, 16).amax(1).tolist())]


def test_scored_slopes_that_grow_with_the_distance(lib):
    lens, heads, dim = [1100, 70], 2, 64
    x = R.normal(3, sum(lens), 3 * heads * dim)
    q, k, v = _split(x, heads, heads, dim)
    slopes = torch.tensor([-0.5, -0.0625], device="cuda")
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, heads, R.options(slopes=slopes))
    # biases of up to 550, rounded to fp32 after the slope's log2(e) is: off by at most 3 * 2^-24 * 800 = 1.4e-4 in log2 units
    _check_scored(out, q, k, v, lens, heads, heads, dim, {}, slopes, None, None, None)


@pytest.mark.parametrize("name", ["causal", "slopes", "docs"])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([1, 0, 5, 2, 70, 3] * 260, 2, 1, 64),  # more sequences than the planner keeps at hand
                                                     ([2200, 40], 64, 1, 32),               # and more query tiles
                                                     ([1, 9, 131], 128, 1, 128), ([4, 1], 2304, 24, 8)], ids=["sequences", "tiles", "group", "heads"])
def test_scored_counts_beyond_the_common(lib, lens, heads, kv_heads, dim, name):
    x, mod, slopes, bias, prefix, docs = _scored_case(lens, heads, kv_heads, dim, MODS[name])
    q, k, v = _split(x, heads, kv_heads, dim)
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(slopes=slopes, docs=docs, **mod))
    _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)


@pytest.mark.parametrize("name", ["slopes_prefix", "slopes_prefix_window", "slopes_window", "steep_prefix", "bias_prefix", "cap_prefix", "docs_slopes_prefix"])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([5, 200, 0, 700], 4, 2, 64), ([1500, 90], 7, 1, 128)], ids=["64", "128"])
def test_scored_prefix_with_the_others(lib, lens, heads, kv_heads, dim, name):
    """A prefix is walked before the window: with slopes its keys, the farthest of all, give a row its first reference."""
    mods = {"slopes_prefix": dict(causal=1, slopes=True, prefix=True), "slopes_prefix_window": dict(causal=1, left=40, slopes=True, prefix=True),
            "slopes_window": dict(left=70, right=130, slopes=True), "steep_prefix": dict(causal=1, left=3, slopes=True, prefix=True),
            "bias_prefix": dict(causal=1, left=20, bias=33, prefix=True), "cap_prefix": dict(causal=1, left=20, cap=20.0, prefix=True),
            "docs_slopes_prefix": dict(causal=1, left=90, slopes=True, prefix=True, docs=True)}
    x, mod, slopes, bias, prefix, docs = _scored_case(lens, heads, kv_heads, dim, mods[name])
    if name == "steep_prefix":
        slopes = slopes * 16
    q, k, v = _split(x, heads, kv_heads, dim)
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(slopes=slopes, bias=bias, prefix=prefix, docs=docs, **mod))
    _check_scored(out, q, k, v, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)


def test_scored_options_null_is_plain_attention(lib):
    lens = [30, 61]
    x = R.normal(1, 91, 3 * 2 * 64)
    q, k, v = _split(x, 2, 2, 64)
    out = R.scored(lib, q, k, v, R.cu_of(lens), 2, 2, None)
    _check_scored(out, q, k, v, lens, 2, 2, 64, {}, None, None, None, None)


def test_scored_strided_rows_and_rows_behind_the_last_sequence(lib):
    lens, heads, kv_heads, dim = [50, 77], 4, 2, 64
    t = sum(lens)
    big = torch.full((t + 9, 1000), NAN, dtype=R.BF16, device="cuda")
    q, k, v = big[:, 8:8 + 256], big[:, 400:528], big[:, 600:728]
    for i, z in enumerate((q, k, v)):
        z[:t] = R.normal(i, t, z.shape[1])
    out = torch.full((t + 9, 304), 3.0, dtype=R.BF16, device="cuda")
    R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, None, out=out[:, 16:272])
    _check_scored(out[:t, 16:272], q, k, v, lens, heads, kv_heads, dim, {}, None, None, None, None)
    out[:t, 16:272] = 3.0
    assert (out == 3.0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_scored_not_finite_stays_in_its_sequence(lib, dim):
    """NaN and inf in a neighbour's rows, and in keys that a mask hides, reach nobody else."""
    lens, heads = [37, 21, 130], 2
    x = R.normal(3, sum(lens), 3 * heads * dim)
    x[37:58] = NAN
    x[40, :] = math.inf
    q, k, v = _split(x, heads, heads, dim)
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, heads, None)
    for rows in (slice(0, 37), slice(58, 188)):
        _check_scored(out[rows], q[rows], k[rows], v[rows], [rows.stop - rows.start], heads, heads, dim, {}, None, None, None, None)
    assert out[37:58].isnan().all()
    # a padding token (document -1) whose key is not finite
    x = R.normal(4, 60, 3 * heads * dim)
    q, k, v = _split(x, heads, heads, dim)
    docs = torch.zeros(60, dtype=torch.int32, device="cuda")
    docs[20:25] = -1
    k[20:22], k[22:25] = NAN, math.inf
    out = R.scored(lib, q, k, v, R.cu_of([60]), heads, heads, R.options(docs=docs))
    assert (out[20:25] == 0).all()
    clean = k.clone()
    clean[20:25] = 0
    _check_scored(out, q, clean, v, [60], heads, heads, dim, {}, None, None, None, docs)


def test_scored_bias_of_minus_infinity_and_the_lowest_value(lib):
    lens, heads, dim = [140], 2, 64
    x = R.normal(5, 140, 3 * heads * dim)
    q, k, v = _split(x, heads, heads, dim)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        bias = torch.zeros(heads, 2 * 70 + 1, device="cuda")
        bias[0, 60:] = low  # head 0 looks back by more than 10 only: rows 0 .. 9 see nothing but the masked value
        bias[1, 100:] = low
        out = R.scored(lib, q, k, v, R.cu_of(lens), heads, heads, R.options(bias=bias))
        want, size = R.attend(*(z.reshape(140, heads, dim) for z in (q, k, v)), 0, bias=bias)
        seen = torch.ones(140, heads, dtype=torch.bool, device="cuda")
        seen[:11, 0] = False
        R.assert_attended(out.view(140, heads, dim)[seen], want[seen], size[seen])
        if low == -math.inf:
            assert (out.view(140, heads, dim)[:11, 0] == 0).all()
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -2.41e38])
@pytest.mark.parametrize("lens,heads,kv_heads,radius", [([140], 2, 2, 70), ([1100], 4, 1, 150), ([1100], 2, 2, 600)],
                         ids=["staged", "beyond a table read in place", "in a table read in place"])
@pytest.mark.parametrize("docs", [False, True])
def test_scored_bias_below_the_limit_is_minus_infinity(lib, lens, heads, kv_heads, radius, low, docs):
    """Rows whose visible biases are all below -2.4e38 are zero, and no key with such a bias counts elsewhere: head 0 sees no key ahead of -10, head 1
    none from radius on. Tables of up to 1024 entries of a key head are staged, larger ones are read where they lie."""
    n, dim = lens[0], 64
    x = R.normal(5, n, (heads + 2 * kv_heads) * dim)
    q, k, v = _split(x, heads, kv_heads, dim)
    bias = _bias(heads, radius)
    bias[0, radius - 10:] = low
    bias[1, 2 * radius:] = low
    ids = torch.zeros(n, dtype=torch.int32, device="cuda") if docs else None
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(bias=bias, docs=ids)).view(n, heads, dim)
    bias[bias < -2.4e38] = -math.inf
    want, size = R.attend(q.reshape(n, heads, dim), k.reshape(n, kv_heads, dim), v.reshape(n, kv_heads, dim), 0, bias=bias)
    assert (want[:11, 0] == 0).all() and (out[:11, 0] == 0).all()
    R.assert_attended(out, want, size)


@pytest.mark.parametrize("power", [79, -60])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("mod", [{}, dict(causal=1), dict(slopes=True), dict(bias=9), dict(cap=200.0), dict(docs=True)], ids=str)
def test_scored_values_of_any_magnitude(lib, mod, dim, power):
    """Values as large, and as small, as the header allows without a cap up to 55, with scores that rise by 50 along the row after its first keys, and
    that fall by as much before them: sums that follow a first reference would pass fp32's range."""
    lens, heads, kv_heads = [300], 4, 2
    x, mod, slopes, bias, prefix, docs = _scored_case(lens, heads, kv_heads, dim, mod)
    q, k, v = _split(x, heads, kv_heads, dim)
    x[:, :(heads + kv_heads) * dim] *= 0.05
    q[:, ::dim], k[:, ::dim] = dim ** 0.5, 0.0
    k[100:200, ::dim], k[200:, ::dim] = 25.0, 50.0
    if power < 0:
        k[:100, ::dim] = 50.0  # the first reference is far above all that follows in the rows that do not see these keys
    v[:] = (R.normal(3, 300, kv_heads * dim).float().clamp(-1, 1) * 2.0 ** power).to(R.BF16)
    docs = torch.arange(300, dtype=torch.int32, device="cuda") // 250 if docs is not None else None
    out = R.scored(lib, q, k, v, R.cu_of(lens), heads, kv_heads, R.options(slopes=slopes, bias=bias, docs=docs, **mod))
    scale = 2.0 ** -power  # exact: compared at the values' own scale
    _check_scored(out.double() * scale, q, k, v.double() * scale, lens, heads, kv_heads, dim, mod, slopes, bias, prefix, docs)


@pytest.mark.parametrize("power", [17, -40])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_scored_values_of_any_magnitude_under_a_cap(lib, dim, sign, power):
    """The largest and smallest values that the header allows under a cap, where all scores lie at one end of it, and at both."""
    lens, heads = [500, 70], 2
    for mixed in (False, True):
        x, mod, slopes, bias, prefix, docs = _scored_case(lens, heads, heads, dim, dict(cap=55.0))
        q, k, v = _split(x, heads, heads, dim)
        q[:, ::dim], k[:, ::dim] = 8.0 * dim ** 0.5, sign * 100.0
        if mixed:
            k[::7, ::dim] = -sign * 100.0
        v[:] = (R.normal(3, sum(lens), heads * dim).float().clamp(-1, 1) * 2.0 ** power).to(R.BF16)
        out = R.scored(lib, q, k, v, R.cu_of(lens), heads, heads, R.options(**mod))
        scale = 2.0 ** -power
        _check_scored(out.double() * scale, q, k, v.double() * scale, lens, heads, heads, dim, mod, slopes, bias, prefix, docs)


def test_scored_large_scores(lib):
    """Scores that differ by thousands between keys, growing and falling along the row."""
    lens, heads, dim = [400], 2, 64
    for flip in (False, True):
        x = R.normal(6, 400, 3 * heads * dim, gain=0.05)
        q, k, v = _split(x, heads, heads, dim)
        q[:, ::dim] = 60.0
        ramp = torch.linspace(-200, 200, 400, device="cuda").to(R.BF16)
        k[:, 0], k[:, dim] = (ramp.flip(0) if flip else ramp), ramp
        v[:] = R.normal(7, 400, heads * dim)
        out = R.scored(lib, q, k, v, R.cu_of(lens), heads, heads, None)
        # scores of up to 1500: 64 * 2^-24 * 1500 = 6e-3 at worst, so the bound of the other tests does not hold for p; the two largest
        # keys differ by 1 in k, that is 60 * 1 / 8 = 7.5 in the score: p of all but a run of equal keys is below 6e-4
        want, size = R.attend(*(z.reshape(400, heads, dim) for z in (q, k, v)), 0)
        assert ((out.double().view(400, heads, dim) - want).abs() <= size * (R.HALF_STEP + 2 ** -6) + want.abs() * R.HALF_STEP).all()


# -- paged attention ------------------------------------------------------------------------------
PAGED = [  # new tokens, keys in all, heads, key heads, head_dim, page, by_head
    ([1], [1], 4, 4, 64, 16, False), ([1], [700], 28, 4, 128, 16, False), ([1, 1, 1, 0, 1], [5, 129, 1000, 40, 128], 8, 2, 64, 16, True),
    ([3, 40, 130], [3, 300, 500], 6, 3, 32, 24, False), ([20, 1, 257], [600, 1, 300], 7, 1, 128, 64, True),
    ([5], [77], 3, 1, 96, 8, False), ([64, 64], [64, 200], 4, 4, 128, 128, True), ([9], [260], 2, 2, 8, 40, False),
    ([1] * 40, [3 + 61 * i for i in range(40)], 4, 1, 128, 32, False), ([1], [9000], 16, 1, 64, 16, False),
]
PAGED_MODS = {"causal": {}, "cap_window": dict(cap=20.0, left=50), "slopes": dict(slopes=True), "bias": dict(bias=30), "both_ways": dict(causal=0),
              "prefix": dict(left=7, prefix=True), "window_zero": dict(left=0)}


def _check_paged(out, q, new, kv, heads, pages, mod, slopes=None, bias=None, prefix=None):
    at = 0
    for i, n in enumerate(new):
        if n == 0:
            continue
        want, size = R.attend(q[at:at + n].reshape(n, heads, pages.dim), pages.get("k", i, kv[i]), pages.get("v", i, kv[i]), kv[i] - n,
                              scale=mod.get("scale"), cap=mod.get("cap", 0.0), left=mod.get("left", -1), right=0 if mod.get("causal", 1) else -1,
                              slopes=slopes, bias=bias, prefix=0 if prefix is None else int(prefix[i]))
        R.assert_attended(out[at:at + n], want, size)
        at += n


@pytest.mark.parametrize("name", list(PAGED_MODS))
@pytest.mark.parametrize("case", PAGED, ids=str)
def test_paged(lib, case, name):
    new, kv, heads, kv_heads, dim, page, by_head = case
    mod = dict(PAGED_MODS[name])
    pages = R.Pages(kv, kv_heads, dim, page, by_head, pad=8 if dim == 96 else 0).fill(11)
    q = R.normal(12, sum(new), heads * dim, gain=8.0 if mod.get("cap") else 2.0)
    slopes = _slopes(heads) if mod.pop("slopes", False) else None
    radius = mod.pop("bias", None)
    bias = None if radius is None else _bias(heads, radius)
    prefix = R.ints([n // 2 for n in kv]) if mod.pop("prefix", False) else None
    o = R.options(slopes=slopes, bias=bias, prefix=prefix, **{"causal": 1, **mod})
    out = R.paged(lib, q, R.cu_of(new), R.ints(kv), heads, pages, o)
    _check_paged(out, q, new, kv, heads, pages, mod, slopes, bias, prefix)
    assert torch.equal(out, R.paged(lib, q, R.cu_of(new), R.ints(kv), heads, pages, o))


@pytest.mark.parametrize("left", [-1, 25])
def test_paged_slopes_with_a_prefix(lib, left):
    new, kv, heads, kv_heads, dim = [1, 40, 130], [900, 41, 600], 8, 2, 64
    pages = R.Pages(kv, kv_heads, dim, 16).fill(3)
    q, slopes, prefix = R.normal(12, sum(new), heads * dim, gain=2.0), _slopes(heads), R.ints([300, 0, 599])
    out = R.paged(lib, q, R.cu_of(new), R.ints(kv), heads, pages, R.options(causal=1, left=left, slopes=slopes, prefix=prefix))
    _check_paged(out, q, new, kv, heads, pages, dict(left=left), slopes, None, prefix)


def test_paged_counts_beyond_the_common(lib):
    """More sequences than the planner keeps at hand, most of one new token, some of none."""
    new = [(1, 1, 0, 2)[i % 4] for i in range(1300)]
    kv = [n + (7 * i) % 90 for i, n in enumerate(new)]
    pages = R.Pages(kv, 1, 64, 16, False).fill(4)
    q = R.normal(5, sum(new), 2 * 64, gain=2.0)
    out = R.paged(lib, q, R.cu_of(new), R.ints(kv), 2, pages, R.options(causal=1, cap=20.0))
    _check_paged(out, q, new, kv, 2, pages, dict(cap=20.0))


def test_paged_options_null_is_causal_and_rows_behind_stay(lib):
    new, kv = [4, 2], [40, 2]
    pages = R.Pages(kv, 2, 64, 16).fill(1)
    q = R.normal(2, 9, 4 * 64)
    out = torch.full((9, 4 * 64), 3.0, dtype=R.BF16, device="cuda")
    R.paged(lib, q, R.cu_of(new), R.ints(kv), 4, pages, None, out=out)
    _check_paged(out[:6], q, new, kv, 4, pages, {})
    assert (out[6:] == 3.0).all()


def test_paged_lengths_that_do_not_fit(lib):
    """No key at all, fewer keys than new tokens, more than the table holds, pages that do not exist: zeros, never a fault."""
    heads, dim = 2, 64
    pages = R.Pages([16, 16, 32], 1, dim, 16, table_extra=0).fill(3)
    q = R.normal(4, 9, heads * dim)
    out = R.paged(lib, q, R.cu_of([3, 3, 3]), R.ints([0, 2, 1 << 30]), heads, pages, None)
    assert (out[:3] == 0).all()
    _check_paged(out[4:6], q[4:6], [2], [2], heads, _one(pages, 1, 2), {})
    assert (out[3] == 0).all()  # at position -1
    _check_paged(out[6:9], q[6:9], [3], [32], heads, _one(pages, 2, 32), {})  # cut to the table
    pages.table[2, 1] = 1 << 29  # reads as zeros: keys score 0, values add nothing
    out = R.paged(lib, q, R.cu_of([3, 3, 3]), R.ints([1, 2, 32]), heads, pages, R.options(causal=0))
    k, v = pages.get("k", 2, 16), pages.get("v", 2, 16)
    zero = torch.zeros(16, 1, dim, dtype=R.BF16, device="cuda")
    want, size = R.attend(q[6:9].view(3, heads, dim), torch.cat([k, zero]), torch.cat([v, zero]), 29)
    R.assert_attended(out[6:9], want, size)


def _one(pages, seq, n):
    """The same cache seen as one sequence."""
    one = R.Pages([n], pages.kv_heads, pages.dim, pages.page)
    one.table, one.k, one.v = pages.table[seq:seq + 1], pages.k, pages.v
    return one


def test_paged_offsets_beyond_32_bits(lib):
    """Pages further apart than 2^31 elements."""
    dim, stride = 64, 1_300_000_000
    store = [torch.empty(2 * stride + 16 * dim, dtype=R.BF16, device="cuda") for _ in range(2)]
    pages = R.Pages([40], 1, dim, 16, spare=0, table_extra=0)
    pages.k, pages.v = (s.as_strided((3, 16, 1, dim), (stride, dim, dim, 1)) for s in store)
    pages.k.zero_(), pages.v.zero_()
    qkv = R.normal(5, 40, 4 * dim)
    q_out = torch.empty(40, 2 * dim, dtype=R.BF16, device="cuda")
    R.append(lib, qkv, R.cu_of([40]), R.ints([40]), 2, pages, None, q_out)
    assert torch.equal(pages.get("k", 0)[:, 0], qkv[:, 2 * dim:3 * dim]) and torch.equal(pages.get("v", 0)[:, 0], qkv[:, 3 * dim:])
    out = R.paged(lib, q_out[39:], R.cu_of([1]), R.ints([40]), 2, pages, None)
    _check_paged(out, q_out[39:], [1], [40], 2, pages, {})


# -- in place -------------------------------------------------------------------------------------
@pytest.mark.parametrize("rope", [None, dict(rot=32, layout="interleaved"), dict(rot=6), dict(rot=6, layout="interleaved")], ids=str)
def test_append_turns_queries_in_place(lib, rope):
    heads, kv_heads, dim, kv = 6, 2, 32, [41, 3]
    pages, again = (R.Pages(kv, kv_heads, dim, 16) for _ in range(2))
    qkv, cu = R.normal(9, 44, (heads + 2 * kv_heads) * dim), R.cu_of(kv)
    d = None if rope is None else R.rope_desc(**rope)
    q_out, same = torch.empty(44, heads * dim, dtype=R.BF16, device="cuda"), qkv.clone()
    R.append(lib, qkv, cu, R.ints(kv), heads, pages, d, q_out)
    R.append(lib, same, cu, R.ints(kv), heads, again, d, same)
    assert torch.equal(same[:, :heads * dim], q_out) and torch.equal(same[:, heads * dim:], qkv[:, heads * dim:])
    assert torch.equal(again.k.view(torch.int16), pages.k.view(torch.int16)) and torch.equal(again.v.view(torch.int16), pages.v.view(torch.int16))


@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([300, 1, 70], 4, 2, 64), ([2600], 7, 1, 128), ([40] * 50, 2, 2, 32)], ids=str)
def test_attention_in_place_of_its_queries(lib, lens, heads, kv_heads, dim):
    """Items that several streams share are joined after the last of them has read its queries."""
    t = sum(lens)
    x, cu = R.normal(4, t, (heads + 2 * kv_heads) * dim, gain=1.5), R.cu_of(lens)
    q, k, v = _split(x, heads, kv_heads, dim)
    want = R.scored(lib, q, k, v, cu, heads, kv_heads, R.options(causal=1))
    R.scored(lib, q, k, v, cu, heads, kv_heads, R.options(causal=1), out=q)
    assert torch.equal(q, want)
    new, kv = [1, 3, 130], [1500, 3, 400]
    pages = R.Pages(kv, kv_heads, dim, 16).fill(2)
    q = R.normal(3, sum(new), heads * dim, gain=2.0)
    want = R.paged(lib, q, R.cu_of(new), R.ints(kv), heads, pages, None)
    R.paged(lib, q, R.cu_of(new), R.ints(kv), heads, pages, None, out=q)
    assert torch.equal(q, want)


# -- together, captured, on other streams --------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (7, 1, 128, 24)])
def test_chunks_over_the_cache_match_one_pass(lib, heads, kv_heads, dim, page):
    """Documents fed in chunks (rotate and append, then attend over the cache) give what one pass over the packed batch gives."""
    lens, rope = [190, 33, 300], R.rope_desc(dim // 2, "interleaved", "yarn", factor=4.0, theta=1e4, trained=128, low=32.0, high=1.0)
    t, width = sum(lens), (heads + 2 * kv_heads) * dim
    qkv = R.normal(8, t, width)
    cu = R.cu_of(lens)
    whole = qkv.clone()
    _rope(lib, whole, whole, rope, heads + kv_heads, dim, cu=cu)
    q, k, v = _split(whole, heads, kv_heads, dim)
    o = dict(causal=1, cap=25.0, left=150)
    one_pass = R.scored(lib, q, k, v, cu, heads, kv_heads, R.options(**o))
    pages = R.Pages(lens, kv_heads, dim, page, by_head=True)
    done, chunks = [0] * len(lens), torch.zeros_like(one_pass)
    for step in (1, 100, 1, 64, 300):
        new = [min(step, n - d) for n, d in zip(lens, done)]
        if not any(new):
            break
        rows = torch.cat([torch.arange(int(cu[i]) + d, int(cu[i]) + d + n) for i, (d, n) in enumerate(zip(done, new))]).cuda()
        done = [d + n for d, n in zip(done, new)]
        part, kv = qkv[rows], R.ints(done)
        q_out = torch.empty(len(rows), heads * dim, dtype=R.BF16, device="cuda")
        R.append(lib, part, R.cu_of(new), kv, heads, pages, rope, q_out)
        assert torch.equal(q_out, q[rows])
        chunks[rows] = R.paged(lib, q_out, R.cu_of(new), kv, heads, pages, R.options(**o))
    assert done == lens
    for i, n in enumerate(lens):
        assert torch.equal(pages.get("k", i).reshape(n, -1), k[int(cu[i]):int(cu[i + 1])])
    _check_scored(one_pass, q, k, v, lens, heads, kv_heads, dim, o, None, None, None, None)
    _check_scored(chunks, q, k, v, lens, heads, kv_heads, dim, o, None, None, None, None)


def test_captured_step_follows_the_lengths(lib):
    """One captured decoding step (append, attend) replayed while kv_lens grow in device memory, with a second graph that
    shares the workspace in between."""
    heads, kv_heads, dim, steps = 8, 2, 64, 5
    start = [130, 7, 300]
    pages = R.Pages([n + steps for n in start], kv_heads, dim, 16).fill(21)
    cu, kv = R.cu_of([1, 1, 1]), R.ints(start)
    rope = R.rope_desc(dim)
    qkv = torch.zeros(3, (heads + 2 * kv_heads) * dim, dtype=R.BF16, device="cuda")
    q_out, out = (torch.empty(3, heads * dim, dtype=R.BF16, device="cuda") for _ in range(2))
    other = R.normal(30, 50, 3 * 2 * 64)
    oq, ok, ov = _split(other, 2, 2, 64)
    other_cu, other_out = R.cu_of([50]), torch.empty(50, 2 * 64, dtype=R.BF16, device="cuda")
    n = max(lib.b200emb_attention_workspace_bytes(3, 3, heads, kv_heads, dim), lib.b200emb_attention_workspace_bytes(1, 50, 2, 2, 64))
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    R.scored(lib, oq, ok, ov, other_cu, 2, 2, None, out=other_out, ws=ws)
    want_other = other_out.clone()
    s = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0], stream=s):
        kv += 1
        R.append(lib, qkv, cu, kv, heads, pages, rope, q_out)
        R.paged(lib, q_out, cu, kv, heads, pages, None, out=out, ws=ws)
    with torch.cuda.graph(graphs[1], stream=s):
        R.scored(lib, oq, ok, ov, other_cu, 2, 2, None, out=other_out, ws=ws)
    lens = list(start)
    for i in range(steps):
        qkv.copy_(R.normal(100 + i, *qkv.shape))
        other_out.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        lens = [x + 1 for x in lens]
        assert kv.tolist() == lens
        _check_paged(out, q_out, [1, 1, 1], lens, heads, pages, {})
        assert torch.equal(other_out, want_other)
        _lib.check(lib.b200emb_op_workspace_status(ws.data_ptr(), R.stream()))


FIRST = """
import torch, attention_block_reference as R
from infinity_b200 import _lib
lib = _lib.load()
lens, heads, dim = [40, 9], 2, 64
q, k, v = (R.normal(i, 49, heads * dim) for i in range(3))
cu, out, ws = R.cu_of(lens), torch.empty_like(q), R.workspace(lib, 2, 49, heads, heads, dim)
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    R.scored(lib, q, k, v, cu, heads, heads, R.options(causal=1, cap=20.0), out=out, ws=ws)
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, R.scored(lib, q, k, v, cu, heads, heads, R.options(causal=1, cap=20.0)))
"""


def test_the_first_call_of_a_process_may_be_captured():
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    done = subprocess.run([sys.executable, "-c", FIRST], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("args", ["rope --seqs 3 --len 200 --heads 6 --kv-heads 2", "scored --seqs 3 --len 200 --heads 6 --kv-heads 2 --causal 1 --cap 20",
                                  "scored --seqs 2 --len 150 --heads 4 --slopes 1 --window 40", "paged --seqs 3 --len 300 --new 2 --heads 6 --kv-heads 2",
                                  "paged --seqs 1 --len 90 --new 90 --heads 4 --slopes 1 --page 24 --head-dim 128"])
def test_kernel_case_runs_them(args):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-m", "infinity_b200.kernel_case", *args.split()], cwd=root, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and " ok" in done.stdout, done.stderr


def test_two_streams_with_their_own_workspaces(lib):
    x = [R.normal(i, 700, 3 * 4 * 64) for i in range(2)]
    cu = R.cu_of([400, 300])
    want = [R.scored(lib, *_split(z, 4, 4, 64), cu, 4, 4, None) for z in x]
    ws = [R.workspace(lib, 2, 700, 4, 4, 64) for _ in range(2)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k, v = _split(x[i], 4, 4, 64)
                got[i] = torch.empty(700, 256, dtype=R.BF16, device="cuda")
                _lib.check(lib.b200emb_op_attention_scored(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                                           got[i].data_ptr(), 256, cu.data_ptr(), 2, 700, 4, 4, 64, None, ws[i].data_ptr(),
                                                           ws[i].numel(), s.cuda_stream))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_nothing_to_do(lib):
    x = R.normal(1, 4, 3 * 64)
    q, k, v = _split(x, 1, 1, 64)
    out = torch.full((4, 64), 3.0, dtype=R.BF16, device="cuda")
    R.scored(lib, q, k, v, R.cu_of([0, 0]), 1, 1, None, out=out)  # empty sequences only
    pages = R.Pages([20], 1, 64, 16).fill(1)
    R.paged(lib, q, R.cu_of([0]), R.ints([20]), 1, pages, None, out=out)
    assert (out == 3.0).all()


@pytest.mark.parametrize("n_seqs,n_tokens", [(1, 0), (0, 4), (0, 0)])
@pytest.mark.parametrize("left", [0xFF, 7], ids=["fresh", "of an older call"])
@pytest.mark.parametrize("captured", [False, True])
def test_status_after_a_call_without_rows(lib, n_seqs, n_tokens, left, captured):
    """Neither what a fresh workspace holds nor what an older call left is reported for a call that had nothing to do."""
    x = R.normal(1, 4, 3 * 64)
    q, k, v = _split(x, 1, 1, 64)
    cu, kv, out, pages = R.cu_of([4]), R.ints([20]), torch.full((4, 64), 3.0, dtype=R.BF16, device="cuda"), R.Pages([20], 1, 64, 16).fill(1)
    desc = pages.desc()

    def calls(ws, stream):
        return (lambda: lib.b200emb_op_attention_scored(q.data_ptr(), 192, k.data_ptr(), 192, v.data_ptr(), 192, out.data_ptr(), 64, cu.data_ptr(), n_seqs,
                                                        n_tokens, 1, 1, 64, None, ws.data_ptr(), ws.numel(), stream),
                lambda: lib.b200emb_op_attention_paged(q.data_ptr(), 192, out.data_ptr(), 64, cu.data_ptr(), kv.data_ptr(), n_seqs, n_tokens, 1,
                                                       C.byref(desc), None, ws.data_ptr(), ws.numel(), stream))

    for which in range(2):
        ws = R.workspace(lib, 1, 4, 1, 1, 64)
        ws[:4] = torch.tensor([left, 0, 0, 0] if left == 7 else [left] * 4, dtype=torch.uint8)
        before = ws.clone()
        if captured:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                _lib.check(calls(ws, R.stream())[which]())
            assert torch.equal(ws, before)  # in the graph, not before it
            graph.replay()
            torch.cuda.synchronize()
        else:
            _lib.check(calls(ws, R.stream())[which]())
        _lib.check(lib.b200emb_op_workspace_status(ws.data_ptr(), R.stream()))
        assert torch.equal(ws[4:], before[4:]) and (out == 3.0).all()


AFTER_A_REFUSAL = """
import ctypes as C, torch, attention_block_reference as R
from infinity_b200 import _lib
lib = _lib.load()
x, out = R.normal(1, 6, 64), torch.zeros(6, 64, dtype=R.BF16, device="cuda")
ws, cu, rope = R.workspace(lib, 1, 6, 1, 1, 64, fill=0), R.cu_of([6]), R.rope_desc(64)
torch.cuda.synchronize()
s = torch.cuda.Stream()
graph, rc = torch.cuda.CUDAGraph(), 0
try:
    with torch.cuda.graph(graph, stream=s):
        rc = lib.b200emb_op_workspace_status(ws.data_ptr(), R.stream())  # waits for the stream: refused while it is captured
except Exception as e:
    print("the capture ended:", type(e).__name__)
assert rc == 1, rc  # B200EMB_ERR_CUDA
torch.cuda.synchronize()
_lib.check(lib.b200emb_op_rope(x.data_ptr(), 64, out.data_ptr(), 64, None, cu.data_ptr(), None, 1, 6, 1, 64, C.byref(rope), None))
torch.cuda.synchronize()
R.assert_rotated(out.view(6, 1, 64), *R.rotate(x.view(6, 1, 64), torch.arange(6, device="cuda"), rope))
print("done")
"""


def test_an_error_of_an_earlier_call_is_not_reported_again():
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    done = subprocess.run([sys.executable, "-c", AFTER_A_REFUSAL], env=env, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and "done" in done.stdout, done.stdout + done.stderr
