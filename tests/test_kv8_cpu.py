"""Host-side checks of the 8-bit KV cache entry points: every refusal, without a device."""
import ctypes as C

import numpy as np
import pytest

import kv8_ref
from smallmind_b200 import _lib as L
from smallmind_b200 import KV8Cache, ShapeError, last_error, lib


def view(k=64, v=64, ks=64, vs=64, seqs=4, tokens=32, n_kv=2, hd=64):
    return L.KV8(k, v, ks, vs, seqs, tokens, n_kv, hd)


P = 4096  # any non-null address: nothing here is dereferenced
BAD_CACHES = [
    (dict(seqs=0), -2), (dict(tokens=0), -2), (dict(n_kv=0), -2), (dict(n_kv=-1), -2), (dict(n_kv=4097), -5),
    (dict(hd=0), -5), (dict(hd=63), -5), (dict(hd=96), -5), (dict(hd=256), -5),
    (dict(k=None), -1), (dict(v=None), -1), (dict(ks=None), -1), (dict(vs=None), -1),
    (dict(k=72), -1), (dict(v=65), -1), (dict(ks=66), -1), (dict(vs=67), -1),
]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(change, code):
    c, ok = view(**change), view()
    f = lib()
    assert f.sm_kv8_write(None, c, P, P, 1 << 20, P, P, 1) == code
    assert f.sm_kv8_read(None, c, P, P, 1, P, P, 1 << 20) == code
    assert f.sm_attention_decode_kv8(None, c, P, 1 << 20, P, P, 1, 1, 4, P) == code
    assert f.sm_attention_shared_kv8(None, ok, 0, 1, c, P, 1 << 20, P, P, 1, 1, 4, P) == code
    assert f.sm_attention_shared_kv8(None, c, 0, 1, ok, P, 1 << 20, P, P, 1, 1, 4, P) == code
    assert "kv8" in last_error()


def test_null_cache_is_refused():
    f = lib()
    assert f.sm_kv8_write(None, None, P, P, 128, P, P, 1) == -1
    assert f.sm_kv8_read(None, None, P, P, 1, P, P, 128) == -1
    assert f.sm_attention_decode_kv8(None, None, P, 256, P, P, 1, 1, 4, P) == -1
    assert f.sm_attention_shared_kv8(None, None, 0, 1, view(), P, 256, P, P, 1, 1, 4, P) == -1
    assert f.sm_attention_shared_kv8(None, view(), 0, 1, None, P, 256, P, P, 1, 1, 4, P) == -1


def test_row_calls_refuse_bad_arguments():
    f, c = lib(), view()
    for call in (lambda **a: f.sm_kv8_write(None, c, P, P, a.get("stride", 128), P, P, a.get("n", 1)),
                 lambda **a: f.sm_kv8_read(None, c, P, P, a.get("n", 1), P, P, a.get("stride", 128))):
        assert call(n=-1) == -2
        assert call(stride=127) == -2
        assert call(stride=-128) == -2
        assert call() == -1 and "null" in last_error()  # the context


@pytest.mark.parametrize("at", range(4))
def test_row_calls_refuse_misaligned_pointers(at):
    """Checked after the context, which therefore has to look like one; nothing of it is used."""
    f, c = lib(), view()
    p = [P] * 4
    p[at] += 2
    assert f.sm_kv8_write(P, c, p[0], p[1], 128, p[2], p[3], 1) == -1 and "misaligned" in last_error()
    assert f.sm_kv8_read(P, c, p[2], p[3], 1, p[0], p[1], 128) == -1 and "misaligned" in last_error()


@pytest.mark.parametrize("name", ["q", "seq", "lens", "out"])
def test_attention_refuses_misaligned_pointers(name):
    a = dict(q=P, seq=P, lens=P, out=P)
    a[name] += 2
    f = lib()
    assert f.sm_attention_decode_kv8(P, view(), a["q"], 256, a["seq"], a["lens"], 32, 1, 4, a["out"]) == -1
    assert "misaligned" in last_error()
    assert f.sm_attention_shared_kv8(P, view(), 0, 1, view(), a["q"], 256, a["seq"], a["lens"], 32, 1, 4,
                                     a["out"]) == -1
    assert "misaligned" in last_error()


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), -2), (dict(n_heads=0), -2), (dict(n_heads=-2), -2), (dict(n_heads=5), -2), (dict(n_heads=34), -5),
    (dict(max_len=-1), -2), (dict(max_len=33), -2), (dict(stride=255), -2), (dict(seq=None, B=5), -2),
    (dict(q=None), -1), (dict(lens=None), -1), (dict(out=None), -1), (dict(q=P + 2), -1), (dict(out=P + 1), -1),
    (dict(), -1),  # only the context is missing
])
def test_attention_refuses_bad_arguments(change, code):
    a = dict(q=P, stride=34 * 64, seq=P, lens=P, max_len=32, B=1, n_heads=4, out=P)
    if "stride" in change:
        a["n_heads"] = 4
    a.update(change)
    f = lib()
    assert f.sm_attention_decode_kv8(None, view(), a["q"], a["stride"], a["seq"], a["lens"], a["max_len"], a["B"],
                                     a["n_heads"], a["out"]) == code
    assert f.sm_attention_shared_kv8(None, view(), 0, 1, view(), a["q"], a["stride"], a["seq"], a["lens"],
                                     a["max_len"], a["B"], a["n_heads"], a["out"]) == code


@pytest.mark.parametrize("prefix,seq,n,code", [
    (dict(n_kv=4), 0, 1, -2), (dict(hd=128), 0, 1, -2), (dict(), -1, 1, -2), (dict(), 4, 1, -2), (dict(), 0, -1, -2),
    (dict(), 0, 33, -2), (dict(tokens=2 ** 31 - 1), 0, 2 ** 31 - 1, -2),  # prefix + own keys past 2^31
])
def test_shared_attention_refuses_bad_prefixes(prefix, seq, n, code):
    assert lib().sm_attention_shared_kv8(None, view(**prefix), seq, n, view(), P, 256, P, P, 32, 1, 4, P) == code


def test_python_class_raises_the_frameworks_errors():
    class NoContext:
        handle = None

    c = KV8Cache(NoContext(), 64, 64, 64, 64, 4, 32, 2, 64)
    with pytest.raises(ShapeError):
        c.write_device(P, P, P, P, -1)
    with pytest.raises(ShapeError):
        c.read_device(P, P, 1, P, P, row_stride=5)
    with pytest.raises(ShapeError):
        c.attention_decode_device(P, P, P, 1, 3, P)
    with pytest.raises(ShapeError):
        c.attention_shared_device(P, c, 9, 1, P, P, 1, 4, P)
    assert (c.max_seqs, c.max_tokens, c.n_kv_heads, c.head_dim) == (4, 32, 2, 64)


def test_struct_matches_the_header():
    assert C.sizeof(L.KV8) == 4 * 8 + 4 * 4
    assert [n for n, _ in L.KV8._fields_] == ["k", "v", "k_scale", "v_scale", "max_seqs", "max_tokens", "n_kv",
                                              "head_dim"]


def test_reference_forms():
    """The tests' own 64-bit forms at values that can be checked by hand."""
    codes, scale = kv8_ref.quantize(np.array([[127.0, 0.5, 1.5, -2.5, -127.0, 0.0]], np.float32))
    assert scale[0] == 1.0 and codes.tolist() == [[127, 0, 2, -2, -127, 0]]
    codes, scale = kv8_ref.quantize(np.array([[0.0, 0.0], [np.inf, 1.0], [1.0, np.nan]], np.float32))
    assert scale[0] == 0 and np.isnan(scale[1:]).all() and not codes.any()
    assert kv8_ref.weight(np.array(0.0)) == 1.0 and kv8_ref.weight(np.array(-1e9)) == kv8_ref.weight(np.array(-87.3))
    assert abs(kv8_ref.weight(np.array(-1.0)) - 7 / 19) < 1e-15
    out, _ = kv8_ref.attend(np.zeros((1, 4)), np.ones((3, 4)), np.arange(12).reshape(3, 4))
    assert np.allclose(out, [[4, 5, 6, 7]])
