"""64-bit statements of the attention-block operators (rotary positions, paged cache, attention with modified
scores), written from their formulas, and the call helpers the GPU tests share."""
import ctypes as C
import math

import torch

from infinity_b200 import _lib

BF16 = torch.bfloat16
HALF_STEP = torch.finfo(BF16).eps / 2  # rounding to bf16 moves a value by at most this much of itself


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(lens):
    return ints([0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist())


def normal(seed, *shape, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * gain).to(BF16)


def rope_desc(rot, layout="half", scaling="none", factor=1.0, theta=1e4, trained=2048, low=0.0, high=0.0, magnitude=0.0, inverse=0):
    return _lib.RopeDesc(rot_dim=rot, layout=_lib.ROPE_LAYOUT[layout], scaling=_lib.ROPE_SCALING[scaling], original_max_pos=trained,
                         theta=theta, factor=factor, low=low, high=high, magnitude=magnitude, inverse=inverse)


def frequencies(d):
    """Angle per position of every pair and the factor on cos and sin, in Python floats."""
    r, f = d.rot_dim, d.factor
    out = []
    for i in range(r // 2):
        theta = d.theta * f ** (r / (r - 2)) if d.scaling == 2 else d.theta
        w = theta ** (-2.0 * i / r)
        if d.scaling == 1:
            w /= f
        elif d.scaling == 3:
            turns = d.original_max_pos * w / (2 * math.pi)
            k = 1.0 if turns >= d.high else 0.0 if turns <= d.low else (turns - d.low) / (d.high - d.low)
            w = w * (k + (1 - k) / f)
        elif d.scaling == 4:
            at = [r * math.log(d.original_max_pos / (2 * math.pi * n)) / (2 * math.log(d.theta)) for n in (d.low, d.high)]
            a, b = max(0, math.floor(at[0])), min(r - 1, math.ceil(at[1]))
            k = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            w = w * (1 - k) + w / f * k
        out.append(w)
    m = d.magnitude or (0.1 * math.log(max(f, 1.0)) + 1.0 if d.scaling == 4 else 1.0)
    return out, m


def rotate(x, positions, d):
    """x [n, heads, dim] -> (rotated in float64, what its error is relative to: |u| + |v| of each pair)."""
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    w, m = frequencies(d)
    for p, wp in enumerate(w):
        a = positions.double() * wp
        c, s = (a.cos() * m)[:, None], (a.sin() * m * (-1 if d.inverse else 1))[:, None]
        i, j = (2 * p, 2 * p + 1) if d.layout == 1 else (p, p + d.rot_dim // 2)
        u, v = x[..., i], x[..., j]
        y[..., i], y[..., j] = u * c - v * s, v * c + u * s
        size[..., i] = size[..., j] = (u.abs() + v.abs()) * m
    return y, size


def assert_rotated(got, want, size):
    # one rounding to bf16; cos and sin in fp32 of an angle within pi rounded to fp32: off by at most 2^-23 pi + 2 ulp < 2^-20
    tol = want.abs() * HALF_STEP + size * 2.0 ** -20
    bad = (got.double() - want).abs() - tol
    assert (bad <= 0).all(), bad.max().item()


def attend(q, k, v, q0, scale=None, cap=0.0, left=-1, right=-1, slopes=None, bias=None, prefix=0, q_docs=None, k_docs=None):
    """One sequence: q [n, H, d], k and v [m, Hk, d] -> (o, a) in float64, a = sum p |v| / sum p. Query i is at q0 + i.
    Values of masked keys are never touched."""
    q, k, v = q.double(), k.double(), v.double()
    n, H, d = q.shape
    m, g = k.shape[0], H // k.shape[1]
    s = torch.einsum("nhd,mhd->hnm", q, k.repeat_interleave(g, 1)) * (1 / math.sqrt(d) if scale is None else scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    dist = torch.arange(m, device=q.device)[None] - (torch.arange(n, device=q.device)[:, None] + q0)
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * dist.abs()
    if bias is not None:
        r = (bias.shape[1] - 1) // 2
        s = s + bias.double()[:, dist.clamp(-r, r) + r]
    seen = torch.ones_like(dist, dtype=torch.bool)
    if left >= 0:
        seen &= dist >= -left
    if right >= 0:
        seen &= dist <= right
    seen |= (torch.arange(m, device=q.device) < prefix)[None]
    if q_docs is not None:
        seen &= (q_docs[:, None] == k_docs[None]) & (q_docs >= 0)[:, None]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(s == -math.inf, torch.zeros_like(s), torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    vv = v.repeat_interleave(g, 1)
    used = seen.any(0)  # keys that no row sees may hold anything
    vv = torch.where(used[:, None, None], vv, torch.zeros_like(vv))
    return torch.einsum("hnm,mhd->nhd", p, vv), torch.einsum("hnm,mhd->nhd", p, vv.abs())


def assert_attended(got, want, size):
    # probabilities rounded to bf16 (half a step each, so at most HALF_STEP * sum p |v|), scores in fp32 (below 2^-10 of p for the
    # sizes here: head_dim * 2^-24 * sum |q k| * scale < 6e-4), one rounding of the result
    tol = size * (HALF_STEP + 2.0 ** -10) + want.abs() * HALF_STEP
    bad = (got.double().reshape(want.shape) - want).abs() - tol
    assert torch.isfinite(got).all() and (bad <= 0).all(), bad.max().item()


def workspace(lib, n_seqs, n_tokens, heads, kv_heads, dim, fill=0xFF):
    n = lib.b200emb_attention_workspace_bytes(n_seqs, n_tokens, heads, kv_heads, dim)
    assert n > 0, _lib.last_error()
    return torch.full((n,), fill, dtype=torch.uint8, device="cuda")


def options(causal=0, left=-1, right=-1, cap=0.0, scale=0.0, slopes=None, bias=None, prefix=None, docs=None):
    o = _lib.AttnOpts(scale=scale, cap=cap, causal=causal, window_left=left, window_right=right,
                      bias_radius=0 if bias is None else (bias.shape[1] - 1) // 2)
    for name, t in (("slopes", slopes), ("bias", bias), ("prefix_lens", prefix), ("doc_ids", docs)):
        if t is not None:
            setattr(o, name, t.data_ptr())
    return o


def scored(lib, q, k, v, cu, heads, kv_heads, opts, out=None, ws=None, n_seqs=None):
    """q, k, v: [tokens, heads * dim] tensors whose rows may be strided."""
    t, dim = q.shape[0], q.shape[1] // heads
    out = torch.empty(t, heads * dim, dtype=BF16, device="cuda") if out is None else out
    n_seqs = len(cu) - 1 if n_seqs is None else n_seqs
    ws = workspace(lib, n_seqs, t, heads, kv_heads, dim) if ws is None else ws
    _lib.check(lib.b200emb_op_attention_scored(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                               out.data_ptr(), out.stride(0), cu.data_ptr(), n_seqs, t, heads, kv_heads, dim,
                                               None if opts is None else C.byref(opts), ws.data_ptr(), ws.numel(), stream()))
    _lib.check(lib.b200emb_op_workspace_status(ws.data_ptr(), stream())) if not torch.cuda.is_current_stream_capturing() else None
    return out


class Pages:
    """A paged cache of `kv_lens` keys: pages in shuffled order, table entries that are not used hold nonsense, slots past
    the end of a sequence hold NaN."""

    def __init__(self, kv_lens, kv_heads, dim, page, by_head=False, seed=0, spare=2, pad=0, table_extra=1):
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in kv_lens]
        self.page, self.by_head, self.kv_heads, self.dim, self.kv_lens = page, by_head, kv_heads, dim, list(kv_lens)
        n_pages = sum(used) + spare
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        table = torch.full((len(kv_lens), max(used + [0]) + table_extra), 0x7FFFFFFF, dtype=torch.int32)
        table[::2, -1:] = -5
        at = 0
        for i, n in enumerate(used):
            table[i, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        shape = (n_pages, kv_heads, page, dim + pad) if by_head else (n_pages, page, kv_heads, dim + pad)
        self.k = torch.full(shape, math.nan, dtype=BF16, device="cuda")[..., :dim]
        self.v = torch.full(shape, math.nan, dtype=BF16, device="cuda")[..., :dim]

    def tokens(self, name):
        """[pages, page, heads, dim] view."""
        t = getattr(self, name)
        return t.transpose(1, 2) if self.by_head else t

    def where(self, seq, positions):
        p = positions.long()
        return self.table[seq].long()[p // self.page], p % self.page

    def put(self, name, seq, positions, rows):
        at, off = self.where(seq, positions)
        self.tokens(name)[at, off] = rows

    def get(self, name, seq, n=None):
        n = self.kv_lens[seq] if n is None else n
        at, off = self.where(seq, torch.arange(n, device="cuda"))
        return self.tokens(name)[at, off]

    def fill(self, seed):
        for i, n in enumerate(self.kv_lens):
            if n:
                self.put("k", i, torch.arange(n, device="cuda"), normal(seed + 2 * i, n, self.kv_heads, self.dim))
                self.put("v", i, torch.arange(n, device="cuda"), normal(seed + 2 * i + 1, n, self.kv_heads, self.dim))
        return self

    def desc(self):
        t = self.tokens("k")
        return _lib.KvCache(k=self.k.data_ptr(), v=self.v.data_ptr(), page_table=self.table.data_ptr(), n_pages=t.shape[0],
                            page_size=self.page, n_kv_heads=self.kv_heads, head_dim=self.dim, table_stride=self.table.shape[1],
                            page_stride=t.stride(0), token_stride=t.stride(1), head_stride=t.stride(2))


def paged(lib, q, cu, kv_lens, heads, pages, opts, out=None, ws=None, n_seqs=None):
    t = q.shape[0]
    out = torch.empty(t, heads * pages.dim, dtype=BF16, device="cuda") if out is None else out
    n_seqs = len(cu) - 1 if n_seqs is None else n_seqs
    ws = workspace(lib, n_seqs, t, heads, pages.kv_heads, pages.dim) if ws is None else ws
    desc = pages.desc()
    _lib.check(lib.b200emb_op_attention_paged(q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), cu.data_ptr(),
                                              kv_lens.data_ptr(), n_seqs, t, heads, C.byref(desc),
                                              None if opts is None else C.byref(opts), ws.data_ptr(), ws.numel(), stream()))
    _lib.check(lib.b200emb_op_workspace_status(ws.data_ptr(), stream())) if not torch.cuda.is_current_stream_capturing() else None
    return out


def append(lib, qkv, cu, kv_lens, heads, pages, rope, q_out):
    desc = pages.desc()
    _lib.check(lib.b200emb_op_kv_append(qkv.data_ptr(), qkv.stride(0), cu.data_ptr(), kv_lens.data_ptr(), len(cu) - 1, qkv.shape[0],
                                        heads, None if rope is None else C.byref(rope), None if q_out is None else q_out.data_ptr(),
                                        0 if q_out is None else q_out.stride(0), C.byref(desc), stream()))
