"""What the drafted tree's entry points refuse, checked on the host before anything is launched."""
import ctypes

import pytest

import eyebrowse_amd as eb

P, Q = 1 << 20, 2 << 20  # addresses that are never read
F32, F16, E4M3, I8 = (int(t) for t in (eb.DType.F32, eb.DType.F16, eb.DType.F8E4M3, eb.DType.I8))


def refused(status, match, fn, *args):
    st = getattr(eb.lib(), fn)(None, *args)
    msg = eb.lib().eb_last_error().decode()
    assert st == status and match in msg, (st, msg)


def attn(h=4, hkv=2, pos=100, n=8, hd=64, max_seq=200, window=0, q=P, qn=None, kc=P, kn=None, vc=P, dtype=F32, masks=P,
         mn=8, depths=P, dn=8, o=P, on=None, ws=None, wn=0):
    size = max_seq * hkv * hd
    return (q, n * h * hd if qn is None else qn, kc, size if kn is None else kn, vc, size, dtype, masks, mn, depths, dn,
            o, n * h * hd if on is None else on, h, hkv, pos, n, hd, max_seq, 0.1, window, ws, wn, 256)


@pytest.mark.parametrize("status,match,change", [
    (4, "multiple", dict(h=5, on=1 << 20, qn=1 << 20)),
    (4, "positive", dict(hkv=0)),
    (3, "head_dim", dict(hd=6)), (3, "head_dim", dict(hd=136)), (3, "head_dim", dict(hd=264)),
    (3, "head_dim", dict(hd=4, dtype=F16)),
    (3, "nodes", dict(n=257, pos=0, max_seq=300)),
    (4, "max_seq", dict(pos=193)), (4, "max_seq", dict(pos=2 ** 64 - 4)), (4, "max_seq", dict(pos=201)),
    (4, "q holds", dict(qn=8 * 4 * 64 - 1)), (4, "o holds", dict(on=8 * 4 * 64 - 1)),
    (4, "kcache", dict(kn=200 * 2 * 64 - 1)),
    (4, "masks holds", dict(mn=7)), (4, "masks holds", dict(n=33, mn=33, pos=0)),
    (4, "depths", dict(window=5, dn=7)), (4, "depths", dict(window=5, depths=None)),
    (4, "null", dict(q=None)), (4, "null", dict(kc=None)), (4, "null", dict(vc=None)), (4, "null", dict(o=None)),
    (4, "null", dict(masks=None)),
    (3, "aligned", dict(q=P + 4)), (3, "aligned", dict(o=P + 8)), (3, "aligned", dict(kc=P + 4)),
    (3, "aligned", dict(vc=P + 8)), (3, "aligned", dict(masks=P + 2)), (3, "aligned", dict(window=3, depths=P + 1)),
    (3, "f32, f16 or f8e4m3", dict(dtype=I8)), (3, "f32, f16 or f8e4m3", dict(dtype=77)),
    (3, "limits", dict(h=1028, hkv=2)),  # 514 heads per KV head
    (3, "limits", dict(h=32768, hkv=32768, hd=64)), (3, "limits", dict(max_seq=(1 << 27) + 1)),
])
def test_attn_tree(status, match, change):
    refused(status, match, "eb_launch_attn_tree", *attn(**change))


def test_attn_tree_workspace():
    need = eb.attn_tree_workspace_floats(4, 2, 5000, 8, 64, F32)
    assert need > 0 and need % (8 * 4 * 66) == 0
    big = dict(pos=5000, max_seq=6000)
    refused(4, "workspace holds", "eb_launch_attn_tree", *attn(**big, ws=P, wn=need - 1))
    refused(4, "workspace", "eb_launch_attn_tree", *attn(**big, ws=None, wn=need))
    refused(3, "aligned", "eb_launch_attn_tree", *attn(**big, ws=P + 4, wn=need))
    # few keys stay in one workgroup; a shape that is refused needs none
    assert eb.attn_tree_workspace_floats(4, 2, 20, 8, 64, F32) == 0
    for bad in ((5, 2, 5000, 8, 64), (4, 2, 5000, 257, 64), (4, 2, 5000, 0, 64), (4, 2, 5000, 8, 6), (4, 0, 1, 1, 64),
                (4, 2, 2 ** 63, 8, 64)):
        assert eb.attn_tree_workspace_floats(*bad, F32) == 0
    # a window lowers the splits, and never raises them
    assert eb.attn_tree_workspace_floats(32, 8, 32000, 64, 128, I8) > 0


def test_attn_tree_no_nodes():
    assert eb.lib().eb_launch_attn_tree(None, *attn(n=0, q=None, kc=None, vc=None, masks=None, o=None, mn=0)) == 0


def test_attn_tree_i8():
    def call(max_seq=200, hkv=2, hd=64, block=64, codes=None, exps=None, **kw):
        size = max_seq * hkv * hd
        cache = eb.CacheI8(kw.pop("k", P), P, P, P, size if codes is None else codes,
                           -(-max_seq // max(block, 1)) * hkv if exps is None else exps, max_seq, hkv, hd, block)
        a = attn(hkv=hkv, hd=hd, max_seq=max_seq, **kw)
        return (a[0], a[1], ctypes.byref(cache), *a[7:14], *a[15:17], *a[19:])

    refused(3, "block 48", "eb_launch_attn_tree_i8", *call(block=48))
    refused(3, "head_dim 24", "eb_launch_attn_tree_i8", *call(hd=24))
    refused(4, "codes hold", "eb_launch_attn_tree_i8", *call(codes=200 * 2 * 64 - 1))
    refused(4, "exponents hold", "eb_launch_attn_tree_i8", *call(exps=7))
    refused(3, "aligned", "eb_launch_attn_tree_i8", *call(k=P + 4))
    refused(4, "null", "eb_launch_attn_tree_i8", *call(k=None))
    refused(3, "nodes", "eb_launch_attn_tree_i8", *call(n=257, pos=0, max_seq=300))
    refused(4, "max_seq", "eb_launch_attn_tree_i8", *call(pos=193))
    refused(4, "workspace", "eb_launch_attn_tree_i8", *call(pos=5000, max_seq=6000))


def test_plan_and_accept():
    fn = "eb_launch_tree_plan"
    refused(3, "nodes", fn, P, 300, P, 3000, P, 300, 257)
    refused(4, "parents holds", fn, P, 32, P, 66, P, 33, 33)
    refused(4, "masks holds", fn, P, 33, P, 65, P, 33, 33)
    refused(4, "depths holds", fn, P, 33, P, 66, P, 32, 33)
    refused(4, "null", fn, None, 33, P, 66, P, 33, 33)
    refused(4, "null", fn, P, 33, None, 66, P, 33, 33)
    refused(3, "aligned", fn, P, 33, P, 66, P + 2, 33, 33)
    assert eb.lib().eb_launch_tree_plan(None, None, 0, None, 0, None, 0, 0) == 0
    fn = "eb_launch_tree_accept"
    good = [P, 9, P, 9, P, 9, P, 9, P, 9, P, 9]
    for i, name in ((1, "tokens"), (3, "parents"), (5, "sampled"), (7, "path"), (9, "emitted")):
        a = list(good)
        a[i] = 8
        refused(4, f"{name} holds", fn, *a)
    for i in (0, 2, 4, 6, 8, 10):
        a = list(good)
        a[i] = None
        refused(4, "null", fn, *a)
    refused(4, "root", fn, *good[:-1], 0)
    refused(3, "nodes", fn, *[300 if x == 9 else x for x in good[:-1]], 257)


def test_prologue_tree():
    def call(rows=8, h=4, hkv=2, hd=64, pos=10, seq=30, table=30 * 32, depths=P, dn=8, dtype=F32, cos=P):
        return (P, rows * h * hd, P, rows * hkv * hd, P, rows * hkv * hd, rows, h, hkv, hd, None, None, None, 1e-6, cos,
                P if cos else None, table, pos, depths, dn, P, rows * h * hd, P, seq * hkv * hd, P, seq * hkv * hd, seq,
                dtype)

    fn = "eb_launch_attn_prologue_tree"
    refused(4, "depths", fn, *call(depths=None))
    refused(4, "depths holds", fn, *call(dn=7))
    refused(4, "tables", fn, *call(table=18 * 32 - 1))
    refused(4, "max_seq", fn, *call(pos=23))
    refused(3, "f32, f16 or f8e4m3", fn, *call(dtype=I8))
    refused(4, "even", fn, *call(hd=7))
    with pytest.raises(eb.ShapeMismatch):
        eb.launch_attn_prologue_tree(0, *call(dn=7))


def test_null_handles():
    """The handle forms' null arguments: errors, no crashes."""
    l = eb.lib()
    assert l.eb_tree_plan(None, None, None, None, 4) == 6
    assert l.eb_tree_accept(None, None, None, None, None, None, None, 4) == 6
    assert l.eb_attn_tree(None, None, None, None, None, None, None, 4, 2, 0, 1, 64, 8, 0.1, 0) == 6
    assert l.eb_attn_tree_i8(None, None, None, 0, None, None, None, 4, 0, 1, 0.1, 0) == 6
    assert l.eb_attn_prologue_tree(None, None, None, None, None, None, None, None, 1, 4, 2, 64, 0, 8, None, None, None,
                                   1e-6, None, None) == 4
    assert l.eb_kv_compact(None, None, None, None, 4, 0) == 6
    assert l.eb_kv_fork(None, None, None, 4) == 6
    out = ctypes.c_void_p()
    assert l.eb_attention_forward_tree_qkv(None, None, None, None, None, None, None, 0, None, None, 1, 0,
                                           ctypes.byref(out)) == 6
    assert l.eb_attention_forward_tree(None, None, None, None, None, 0, None, None, 1, 0, ctypes.byref(out)) == 6
