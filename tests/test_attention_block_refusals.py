"""What the attention-block operators refuse, before anything reaches a device: no call here needs a GPU, the pointers
are never followed."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest

from infinity_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent
INVALID, UNSUPPORTED = -1, -2
P = 1 << 20  # an aligned address that nobody reads


def rope(lib, heads=4, dim=64, n_tokens=8, x_stride=256, out_stride=256, x=P, out=2 * P, positions=None, cu=P, n_seqs=2, null=False, **kw):
    d = dict(rot_dim=64, layout=0, scaling=0, original_max_pos=2048, theta=1e4, factor=1.0, low=1.0, high=4.0)
    d.update(kw)
    desc = _lib.RopeDesc(**d)
    return lib.b200emb_op_rope(x, x_stride, out, out_stride, positions, cu, None, n_seqs, n_tokens, heads, dim,
                               None if null else C.byref(desc), None)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=66), dict(rot_dim=258, dim=512, x_stride=2048, out_stride=2048), dict(layout=2),
    dict(scaling=5), dict(scaling=-1), dict(theta=0.0), dict(theta=math.inf), dict(theta=math.nan), dict(scaling=1, factor=0.0),
    dict(scaling=1, factor=math.nan), dict(scaling=2, rot_dim=2, factor=2.0), dict(scaling=3, low=4.0, high=4.0), dict(scaling=3, low=-1.0),
    dict(scaling=3, original_max_pos=0), dict(scaling=4, low=1.0, high=32.0), dict(scaling=4, low=32.0, high=0.0),
    dict(scaling=4, low=32.0, high=1.0, theta=1.0), dict(inverse=2), dict(magnitude=-1.0), dict(magnitude=math.nan),
    dict(reserved=(C.c_int32 * 6)(0, 1, 0, 0, 0, 0)), dict(null=True), dict(x=None), dict(out=None), dict(cu=None), dict(heads=0), dict(dim=0),
    dict(n_tokens=-1), dict(n_seqs=-1), dict(x_stride=255), dict(out_stride=255), dict(out=P, out_stride=512),
], ids=str)
def test_rope_refuses(lib, kw):
    assert rope(lib, **kw) == INVALID and "rope" in _lib.last_error()


def test_rope_with_no_rows_does_nothing(lib):
    assert rope(lib, n_tokens=0, x=None, out=None) == 0
    assert rope(lib, n_seqs=0) == 0


def cache(**kw):
    d = dict(k=P, v=2 * P, page_table=3 * P, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64, table_stride=4,
             page_stride=16 * 128, token_stride=128, head_stride=64)
    d.update(kw)
    return _lib.KvCache(**d)


BAD_CACHES = [dict(k=None), dict(v=None), dict(page_table=None), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(head_dim=0),
              dict(table_stride=0), dict(reserved=1), dict(token_stride=63), dict(head_stride=8), dict(page_stride=8), dict(page_stride=-2048)]


def append(lib, heads=4, n_tokens=8, stride=512, q_out=P, q_stride=256, qkv=P, cu=P, kv=P, n_seqs=2, desc=None, no_cache=False, **kw):
    return lib.b200emb_op_kv_append(qkv, stride, cu, kv, n_seqs, n_tokens, heads, None if desc is None else C.byref(desc), q_out, q_stride,
                                    None if no_cache else C.byref(cache(**kw)), None)


@pytest.mark.parametrize("kw", BAD_CACHES + [dict(no_cache=True), dict(qkv=None), dict(cu=None), dict(kv=None), dict(stride=511), dict(q_stride=255),
                                             dict(heads=0), dict(n_tokens=-1), dict(n_seqs=-1),
                                             dict(desc=_lib.RopeDesc(rot_dim=66, theta=1e4))], ids=str)
def test_append_refuses(lib, kw):
    assert append(lib, **kw) == INVALID and _lib.last_error()


def test_append_refuses_queries_in_place_with_another_stride(lib):
    assert append(lib, qkv=P, q_out=P, stride=512, q_stride=256) == INVALID and "in place" in _lib.last_error()


def test_append_refuses_positions_that_pass_32_bits(lib):
    assert append(lib, table_stride=1 << 28) == UNSUPPORTED


def opts(**kw):
    d = dict(window_left=-1, window_right=-1)
    d.update(kw)
    return _lib.AttnOpts(**d)


BAD_OPTS = [dict(scale=math.nan), dict(scale=math.inf), dict(scale=3e38), dict(scale=-3e38), dict(cap=3e38), dict(cap=-1.0), dict(cap=math.inf), dict(cap=math.nan), dict(causal=2),
            dict(causal=1, window_right=3), dict(slopes=P, bias=P), dict(reserved=(C.c_int32 * 4)(1, 0, 0, 0))]


def scored(lib, q=P, k=P, v=P, out=P, strides=(512, 512, 512, 512), cu=P, n_seqs=2, n_tokens=8, heads=4, kv_heads=2, dim=64, o=None, ws=P, ws_bytes=None):
    if ws_bytes is None:
        ws_bytes = max(0, lib.b200emb_attention_workspace_bytes(n_seqs, n_tokens, heads, kv_heads, dim))
    return lib.b200emb_op_attention_scored(q, strides[0], k, strides[1], v, strides[2], out, strides[3], cu, n_seqs, n_tokens, heads, kv_heads, dim,
                                           None if o is None else C.byref(o), ws, ws_bytes, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu=None), dict(ws=None), dict(ws=P + 16), dict(ws_bytes=8),
                                dict(q=P + 8), dict(out=P + 2), dict(strides=(510, 512, 512, 512)), dict(strides=(248, 512, 512, 512)),
                                dict(strides=(512, 120, 512, 512)), dict(strides=(512, 512, 120, 512)), dict(strides=(512, 512, 512, 248)),
                                dict(n_tokens=-1), dict(n_seqs=-1), dict(heads=0), dict(kv_heads=0), dict(heads=5, kv_heads=2)]
                         + [dict(o=opts(**b)) for b in BAD_OPTS])
def test_scored_refuses(lib, kw):
    assert scored(lib, **kw) == INVALID and "attention" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(dim=4), dict(dim=60), dict(dim=136, strides=(1024,) * 4), dict(heads=130, kv_heads=1),
                                dict(o=opts(bias_radius=1024, bias=P)), dict(o=opts(bias_radius=-1, bias=P)),
                                dict(n_tokens=(1 << 30) + 1)], ids=str)
def test_scored_does_not_cover(lib, kw):
    assert scored(lib, **kw) == UNSUPPORTED


def paged(lib, q=P, out=P, q_stride=256, out_stride=256, cu=P, kv=P, n_seqs=2, n_tokens=8, heads=4, o=None, ws=P, ws_bytes=None, **kw):
    c = cache(**kw)
    if ws_bytes is None:
        ws_bytes = max(0, lib.b200emb_attention_workspace_bytes(n_seqs, n_tokens, heads, c.n_kv_heads, c.head_dim))
    return lib.b200emb_op_attention_paged(q, q_stride, out, out_stride, cu, kv, n_seqs, n_tokens, heads, C.byref(c),
                                          None if o is None else C.byref(o), ws, ws_bytes, None)


@pytest.mark.parametrize("kw", BAD_CACHES + [dict(q=None), dict(out=None), dict(cu=None), dict(kv=None), dict(ws=None), dict(ws_bytes=1), dict(k=P + 8),
                                             dict(token_stride=132), dict(head_stride=68), dict(page_stride=2052), dict(q_stride=248), dict(heads=3),
                                             dict(o=opts(doc_ids=P))] + [dict(o=opts(**b)) for b in BAD_OPTS])
def test_paged_refuses(lib, kw):
    assert paged(lib, **kw) == INVALID and _lib.last_error()


@pytest.mark.parametrize("kw", [dict(page_size=12, page_stride=12 * 128), dict(head_dim=60), dict(table_stride=1 << 28),
                                dict(table_stride=(1 << 26) + 1), dict(n_tokens=(1 << 30) + 1)], ids=str)
def test_paged_does_not_cover(lib, kw):
    assert paged(lib, **kw) == UNSUPPORTED


def test_empty_calls_do_nothing(lib):
    assert scored(lib, n_tokens=0, q=None) == 0 and scored(lib, n_seqs=0) == 0
    assert paged(lib, n_tokens=0, q=None) == 0 and paged(lib, n_seqs=0) == 0
    assert append(lib, n_tokens=0, qkv=None) == 0 and append(lib, n_seqs=0) == 0


def test_workspace_bytes(lib):
    f = lib.b200emb_attention_workspace_bytes
    base = f(4, 100, 8, 2, 64)
    assert base > 0 and base % 256 == 0
    assert f(5, 100, 8, 2, 64) >= base and f(4, 5000, 8, 2, 64) >= base and f(1, 1, 8, 2, 64) <= base
    assert f(4, 100, 8, 3, 64) < 0 and f(4, 100, 8, 2, 60) < 0 and f(-1, 100, 8, 2, 64) < 0
    assert lib.b200emb_op_workspace_status(None, None) == INVALID


def test_struct_layouts_match_the_compiler(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200emb.h"\nint main(){printf("%zu %zu %zu %zu %zu %zu %zu\\n", '
                   'sizeof(b200emb_rope_desc), offsetof(b200emb_rope_desc, inverse), sizeof(b200emb_kv_cache), '
                   'offsetof(b200emb_kv_cache, page_stride), sizeof(b200emb_attn_opts), offsetof(b200emb_attn_opts, slopes), '
                   'offsetof(b200emb_attn_opts, reserved));return 0;}\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [C.sizeof(_lib.RopeDesc), _lib.RopeDesc.inverse.offset, C.sizeof(_lib.KvCache), _lib.KvCache.page_stride.offset,
                   C.sizeof(_lib.AttnOpts), _lib.AttnOpts.slopes.offset, _lib.AttnOpts.reserved.offset]
