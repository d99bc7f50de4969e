"""CPU checks of the quantised operators' refusals: every size, type and pointer is checked before
a launch."""
import ctypes

import pytest

import eyebrowse_amd as eb
from eyebrowse_amd import _lib

P = 1 << 20  # (an address that is aligned and never touched: each call below is refused first)


def err(fn, *args):
    st = fn(*args)
    return st, eb.lib().eb_last_error().decode()


def cache(max_seq=128, hkv=2, hd=64, block=32, **over):
    c = dict(k=P, k_exp=P, v=P, v_exp=P, code_numel=max_seq * hkv * hd, exp_numel=-(-max_seq // max(block, 1)) * hkv,
             max_seq=max_seq, hkv=hkv, hd=hd, block=block)
    c.update(over)
    return _lib.CacheI8(*(c[n] for n, _ in _lib.CacheI8._fields_))


@pytest.mark.parametrize("over,status,word", [
    (dict(hd=24, code_numel=1 << 20), 3, "head_dim"), (dict(hd=40, code_numel=1 << 20), 3, "head_dim"),
    (dict(hd=272, code_numel=1 << 20), 3, "head_dim"), (dict(hd=16), 3, "head_dim"), (dict(hd=0), 3, "head_dim"),
    (dict(block=8), 3, "block"), (dict(block=48), 3, "block"), (dict(block=512), 3, "block"), (dict(block=0), 3, "block"),
    (dict(hkv=0), 4, "head"), (dict(code_numel=128 * 2 * 64 - 1), 4, "codes"), (dict(exp_numel=7), 4, "exponents"),
    (dict(k=None), 4, "null"), (dict(v=None), 4, "null"), (dict(k_exp=None), 4, "null"), (dict(v_exp=None), 4, "null"),
    (dict(k=P + 8), 3, "aligned"), (dict(max_seq=1 << 28, code_numel=1 << 62, exp_numel=1 << 40), 3, "limits"),
    (dict(hkv=1 << 60, code_numel=1 << 62, exp_numel=1 << 62), 3, "limits"),
])
def test_caches(over, status, word):
    l = eb.lib()
    c = ctypes.byref(cache(**over))
    n = 1 << 20
    for st, msg in (err(l.eb_launch_kv_write_i8, None, c, P, P, n, 3, 5), err(l.eb_launch_kv_read_i8, None, c, P, P, n, 3, 5),
                    err(l.eb_launch_attn_decode_i8, None, P, n, None, None, 0, c, P, n, 4, 9, 0.1, 0, None, 0, 256)):
        assert st == status and word in msg, msg
    st, msg = err(l.eb_launch_attn_prefill_chunk_i8, None, P, n, c, P, n, 4, 9, 2, 0.1, 0, None, 0, 256)
    assert st == status and word in msg


def test_rows_and_operands():
    l = eb.lib()
    c = ctypes.byref(cache())
    row = 2 * 64
    for args, status, word in (((P, P, 3 * row, 3, 126), 4, "max_seq"), ((P, P, 3 * row, 3, 1 << 40), 4, "max_seq"),
                               ((P, P, 3 * row - 1, 3, 0), 4, "k/v"), ((None, P, 3 * row, 3, 0), 4, "null"),
                               ((P, None, 3 * row, 3, 0), 4, "null"), ((P + 4, P, 3 * row, 3, 0), 3, "aligned")):
        for fn in (l.eb_launch_kv_write_i8, l.eb_launch_kv_read_i8):
            st, msg = err(fn, None, c, *args)
            assert st == status and word in msg, msg
    assert l.eb_launch_kv_write_i8(None, c, None, None, 0, 0, 128) == 0  # no row: a no-op
    assert l.eb_launch_kv_write_i8(None, None, P, P, row, 1, 0) == 4
    h, q = 4, 4 * 64

    def decode(q_ptr=P, qn=q, kn=None, vn=None, nn=0, o=P, on=q, heads=h, pos=9, ws=None, wsn=0):
        return err(l.eb_launch_attn_decode_i8, None, q_ptr, qn, kn, vn, nn, c, o, on, heads, pos, 0.1, 0, ws, wsn, 256)

    for over, word in ((dict(heads=5), "multiple"), (dict(heads=0), "head"), (dict(pos=128), "max_seq"), (dict(qn=q - 1), "q holds"),
                       (dict(on=q - 1), "o holds"), (dict(q_ptr=None), "null"), (dict(o=None), "null"), (dict(q_ptr=P + 4), "aligned"),
                       (dict(kn=P, vn=None, nn=row), "null"), (dict(kn=P, vn=P, nn=row - 1), "knew"), (dict(kn=P + 8, vn=P, nn=row), "aligned")):
        st, msg = decode(**over)
        assert st in (3, 4) and word in msg, msg
    # a long cache splits its keys, which takes a workspace
    big = ctypes.byref(cache(max_seq=1 << 15))
    need = eb.attn_i8_workspace_floats(4, 2, 64, 20000, 1, 32)
    assert need > 0
    for ws, wsn, word in ((None, 0, "workspace"), (P, need - 1, "workspace"), (None, need, "null"), (P + 4, need, "aligned")):
        st, msg = err(l.eb_launch_attn_decode_i8, None, P, q, None, None, 0, big, P, q, 4, 20000, 0.1, 0, ws, wsn, 256)
        assert word in msg, msg
    st, msg = err(l.eb_launch_attn_prefill_chunk_i8, None, P, 100 * q, big, P, 100 * q, 4, 0, 100, 0.1, 0, None, 0, 256)
    assert st == 4 and "workspace" in msg
    assert l.eb_launch_attn_prefill_chunk_i8(None, None, 0, big, None, 0, 4, 7, 0, 0.1, 0, None, 0, 256) == 0
    assert eb.attn_i8_workspace_floats(5, 2, 64, 0, 1, 32) == 0 and eb.attn_i8_workspace_floats(4, 2, 40, 0, 1, 32) == 0


def test_linear_q4():
    l = eb.lib()
    bytes_ = eb.q4_packed_bytes(256, 10, 64, True)
    assert bytes_ == 2 * (1024 + 16 * 2 * 3) and eb.q4_packed_bytes(256, 10, 64, False) == 2 * (1024 + 16 * 2 * 2)
    assert eb.q4_packed_bytes(200, 10, 64, False) == 0 and eb.q4_packed_bytes(256, 10, 48, False) == 0

    def pack(w=P, words=10 * 32, s=P, sn=10 * 4, z=P, zn=10 * 4, in_f=256, out_f=10, group=64, packed=P, n=bytes_):
        return err(l.eb_launch_q4_pack, None, w, words, s, sn, z, zn, in_f, out_f, group, packed, n)

    def call(a=P, an=256, w=P, n=bytes_, c=P, cn=10, m=1, in_f=256, out_f=10, group=64, zeros=1, ws=None, wsn=0):
        return err(l.eb_launch_linear_q4, None, a, an, w, n, c, cn, m, in_f, out_f, group, zeros, ws, wsn)

    shapes = ((dict(group=16), 3, "group"), (dict(group=256), 3, "group"), (dict(group=0), 3, "group"),
              (dict(in_f=200), 4, "multiple"), (dict(in_f=0), 4, "multiple"), (dict(out_f=1 << 62), 3, "overflows"),
              (dict(in_f=1 << 25), 3, "in_f"), (dict(n=bytes_ - 1), 4, "packed holds"))
    for over, status, word in (*shapes, (dict(words=319), 4, "w holds"), (dict(sn=39), 4, "scales holds"), (dict(zn=39), 4, "zeros holds"),
                               (dict(w=None), 4, "null"), (dict(s=None), 4, "null"), (dict(packed=None), 4, "null"),
                               (dict(packed=P + 8), 3, "aligned"), (dict(w=P + 2), 3, "aligned"), (dict(s=P + 1), 3, "aligned")):
        over = {**over, **(dict(words=1 << 40, sn=1 << 40, zn=1 << 40) if "in_f" in over else {})}
        st, msg = pack(**over)
        assert st == status and word in msg, (over, msg)
    for over, status, word in (*shapes, (dict(an=255), 4, "a holds"), (dict(cn=9), 4, "c holds"), (dict(a=None), 4, "null"),
                               (dict(w=None), 4, "null"), (dict(c=None), 4, "null"), (dict(a=P + 4), 3, "aligned"), (dict(w=P + 4), 3, "aligned"),
                               (dict(m=40, an=40 * 256, cn=400), 4, "workspace")):
        st, msg = call(**over)
        assert st == status and word in msg, (over, msg)
    assert call(m=0, an=0, cn=0)[0] == 0
    assert call(out_f=0, n=0, cn=0, w=None, c=None)[0] == 0
    assert pack(out_f=0, words=0, sn=0, zn=0, n=0, w=None, s=None, packed=None)[0] == 0
    assert eb.linear_q4_workspace_floats(1, 1024) == 0
    assert eb.linear_q4_workspace_floats(100, 1024) >= 100 * 1024


def test_sample():
    l = eb.lib()

    def call(x=P, xn=300, u=P, out=P, rows=3, vocab=100):
        return err(l.eb_launch_sample, None, x, xn, u, out, rows, vocab, None, None, None, None, None, 0)

    for over, status, word in ((dict(xn=299), 4, "logits"), (dict(x=None), 4, "null"), (dict(u=None), 4, "null"), (dict(out=None), 4, "null"),
                               (dict(vocab=0), 4, "vocab"), (dict(), 4, "workspace"), (dict(rows=65536, vocab=2, xn=1 << 17), 3, "rows"), (dict(vocab=(1 << 24) + 1, rows=1, xn=1 << 25), 3, "vocab"),
                               (dict(rows=1 << 40, vocab=1 << 40), 3, "overflows")):
        st, msg = call(**over)
        assert st == status and word in msg, (over, msg)
    assert call(rows=0, xn=0)[0] == 0


def test_handles_refuse_null():
    l = eb.lib()
    out = ctypes.c_void_p()
    assert l.eb_kv_cache_new_i8(None, None, 0, 16, 1, 16, ctypes.byref(out)) == 6
    assert l.eb_attention_new_q4(None, None, ctypes.byref(out)) == 6
    assert l.eb_kv_cache_block(None) == 0 and not l.eb_kv_cache_k_scale(None, 0)
    assert l.eb_sample(None, None, None, None, 1, 1, None, None, None, None) == 6
    assert l.eb_linear_q4(None, None, None, None, 1) == 6
    assert l.eb_kv_write_i8(None, None, 0, None, None, 1, 0) == 6
    d = _lib.AttentionDesc(4, 2, 64, 0.125, 1e-6, None, None, None, 0, None, None, None, None, 256)
    proj = (_lib.Q4Weight * 4)(*[_lib.Q4Weight(None, i, o, 64, 0) for i, o in ((256, 256), (256, 128), (256, 128), (256, 256))])
    assert l.eb_attention_new_q4(ctypes.byref(d), proj, ctypes.byref(out)) == 4
    assert "not a packed" in l.eb_last_error().decode()
    proj[0].in_f = 128
    assert l.eb_attention_new_q4(ctypes.byref(d), proj, ctypes.byref(out)) == 4
    assert "projection 0 is" in l.eb_last_error().decode()
    proj[0].in_f, proj[0].group = 256, 48
    assert l.eb_attention_new_q4(ctypes.byref(d), proj, ctypes.byref(out)) == 3
