"""The operators of drafted tokens over a paged cache without a device: what they refuse, calls without work, and the plain forms themselves."""
import ctypes as C

import numpy as np
import pytest

import paged_oracle as po
from powerinfer_b200 import _lib

lib = _lib.lib
P = 1 << 20                      # a fake, aligned "device pointer": validation never dereferences it
F32, F16 = _lib.PI_TYPE_F32, _lib.PI_TYPE_F16
INVALID, WORKSPACE = 1, 3


def err():
    return lib.pi_last_error().decode()


def cache(**over):
    c = dict(k=P, v=P, table=P, n_layer=2, n_pages=16, n_seq=2, max_pages=8, n_head_kv=4, page=64, head_dim=128)
    c.update(over)
    return _lib.KvPaged(*c.values())


def batch(**over):
    b = dict(q_start=P, seq=None, pos0=P, n=2, T=2, max_new=1)
    b.update(over)
    return _lib.KvBatch(*b.values())


def mask(b=None, parents=P, to=P, words=1, pos=P):
    return lib.pi_tree_mask(C.byref(b or batch()), parents, to, words, pos, None)


def accept(b=None, tokens=P, parents=P, choice=P, path=P, n_path=P, then=P):
    return lib.pi_tree_accept(C.byref(b or batch()), tokens, parents, choice, path, n_path, then, None)


def append(c=None, b=None, layer=0, xtype=F32, k=P, ks=512, v=P, vs=512, q=None, qs=1024, nh=8, qo=1 << 24, qos=1024, pos=P, freqs=P, n_rot=128):
    return lib.pi_kv_append_paged(C.byref(c or cache()), C.byref(b or batch()), layer, xtype, k, ks, v, vs, q, qs, nh, qo, qos, pos, freqs, n_rot, 0, 1.0, None)


def attention(c=None, b=None, layer=0, xtype=F32, q=P, qs=1024, n_head=8, m=P, words=1, max_kv=512, out=1 << 24, outs=1024, ws=1 << 21, wsn=1 << 26):
    return lib.pi_attention_tree(C.byref(c or cache()), C.byref(b or batch()), layer, xtype, q, qs, n_head, m, words, max_kv, 0.1, out, outs, ws, wsn, None)


def keep(c=None, path=P, most=4, n_path=P, pos0=P, n=2):
    return lib.pi_kv_keep_paged(C.byref(c or cache()), path, most, n_path, pos0, None, n, None)


@pytest.mark.parametrize("call,code,needle", [
    (lambda: mask(words=0), INVALID, "words"),
    (lambda: mask(words=65), INVALID, "words"),
    (lambda: mask(parents=None), INVALID, "parents"),
    (lambda: mask(to=None), INVALID, "mask"),
    (lambda: mask(to=P + 4), INVALID, "8-byte"),
    (lambda: mask(batch(pos0=None)), INVALID, "pos0"),
    (lambda: mask(batch(q_start=None)), INVALID, "batch"),
    (lambda: mask(batch(T=5000, max_new=5000)), INVALID, "4096"),
    (lambda: mask(batch(n=-1)), INVALID, "batch"),
    (lambda: accept(tokens=None), INVALID, "tokens"),
    (lambda: accept(path=None), INVALID, "path"),
    (lambda: accept(n_path=None), INVALID, "n_path"),
    (lambda: accept(batch(T=5000, max_new=5000)), INVALID, "4096"),
    (lambda: append(cache(k=None)), INVALID, "null cache"),
    (lambda: append(cache(table=None)), INVALID, "null cache"),
    (lambda: append(cache(v=P + 8)), INVALID, "16-byte"),
    (lambda: append(cache(head_dim=80)), INVALID, "head_dim"),
    (lambda: append(cache(page=24)), INVALID, "page"),
    (lambda: append(cache(n_pages=0)), INVALID, "positive"),
    (lambda: append(cache(max_pages=1 << 25)), INVALID, "2^30"),
    (lambda: append(cache(n_pages=1 << 23)), INVALID, "2^31"),
    (lambda: append(layer=2), INVALID, "layer"),
    (lambda: append(layer=-1), INVALID, "layer"),
    (lambda: append(xtype=2), INVALID, "unknown type"),
    (lambda: append(k=None), INVALID, "k must be"),
    (lambda: append(vs=256), INVALID, "v must be"),
    (lambda: append(n_rot=63), INVALID, "even"),
    (lambda: append(n_rot=130), INVALID, "within"),
    (lambda: append(q=P, freqs=None), INVALID, "frequencies"),
    (lambda: append(q=P, nh=0), INVALID, "n_head"),
    (lambda: append(q=P, qo=P + 64), INVALID, "overlaps"),
    (lambda: append(q=1 << 25, qo=P), INVALID, "overlap q_out"),
    (lambda: append(q=P, qo=None), INVALID, "q_out must be"),
    (lambda: append(b=batch(T=1 << 30, max_new=1 << 30), q=1 << 44, qo=1 << 52, nh=512, qs=65536, qos=65536), INVALID, "too many"),
    (lambda: attention(n_head=6), INVALID, "multiple of n_head_kv"),
    (lambda: attention(layer=7), INVALID, "layer"),
    (lambda: attention(xtype=5), INVALID, "unknown type"),
    (lambda: attention(out=P), INVALID, "different"),
    (lambda: attention(out=P + 4096), INVALID, "different"),
    (lambda: attention(words=0), INVALID, "words"),
    (lambda: attention(words=65), INVALID, "words"),
    (lambda: attention(m=P + 4), INVALID, "8-byte"),
    (lambda: attention(qs=1026), INVALID, "q must be"),
    (lambda: attention(cache(max_pages=64), max_kv=4096, ws=None, wsn=0), WORKSPACE, "workspace"),
    (lambda: attention(cache(max_pages=64), max_kv=4096, ws=(1 << 21) + 8), WORKSPACE, "workspace"),
    (lambda: attention(b=batch(T=1 << 24, max_new=1 << 24)), INVALID, "too many"),
    (lambda: keep(path=None), INVALID, "path"),
    (lambda: keep(pos0=None), INVALID, "pos0"),
    (lambda: keep(n=-1), INVALID, "bad arguments"),
    (lambda: keep(most=-1), INVALID, "bad arguments"),
    (lambda: keep(cache(page=8)), INVALID, "page"),
])
def test_refusals(call, code, needle):
    assert call() == code and needle in err()


@pytest.mark.parametrize("call", [
    lambda: mask(batch(n=0, T=0)), lambda: mask(batch(T=0)), lambda: mask(batch(max_new=0)), lambda: accept(batch(n=0)), lambda: append(b=batch(T=0)), lambda: append(b=batch(n=0)),
    lambda: append(b=batch(max_new=0)), lambda: attention(b=batch(T=0)), lambda: attention(b=batch(n=0)), lambda: keep(n=0), lambda: keep(most=0)])
def test_calls_without_work_launch_nothing(call):
    assert call() == 0


def test_workspace_is_sized_by_the_same_arguments():
    c, b = cache(max_pages=512), batch(T=50, max_new=25)
    one = lib.pi_attention_tree_workspace_bytes(C.byref(c), C.byref(b), F32, 8, 32768)
    assert one > 0
    assert lib.pi_attention_tree_workspace_bytes(C.byref(c), C.byref(batch(T=0)), F32, 8, 32768) == 0
    assert lib.pi_attention_tree_workspace_bytes(C.byref(cache(page=5)), C.byref(b), F32, 8, 32768) == 0 and "page" in err()


@pytest.mark.parametrize("n", [500, 520, 600, 900, 1200])
def test_more_values_than_64_bits_count_are_many(n):
    """n caches of 65535 KV heads of 256, 2^30 slots each: the queries are laid out (F16) as for all large calls."""
    c, b = cache(max_pages=1 << 26, page=16, n_head_kv=65535, head_dim=256, n_pages=1), batch(n=n, T=500, max_new=1)
    assert lib.pi_attention_tree_workspace_bytes(C.byref(c), C.byref(b), F16, 65535 * 32, 1 << 30) >= 500 * 65535 * 32 * 256 * 2


def test_structures_are_packed_as_c_lays_them_out():
    pytest.importorskip("torch")
    from powerinfer_b200 import ggml_ops as g
    raw = g._KV_PAGED.pack(11, 12, 13, 1, 2, 3, 4, 5, 6, 7)
    c = _lib.KvPaged.from_buffer_copy(raw)
    assert [getattr(c, f) for f, _ in c._fields_] == [11, 12, 13, 1, 2, 3, 4, 5, 6, 7]


def test_plain_trees():
    """A tree by hand: 0 -> (1, 2), 1 -> 3, 2 -> (4, 5); 6's parent is itself: it has none."""
    parents = [-1, 0, 0, 1, 2, 2, 6]
    mask_, pos = po.tree_mask(parents, [0, 7], [10], 7, 1)
    assert mask_ == [0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100101, 0b1000000] and pos == [10, 11, 11, 12, 12, 12, 10]
    tokens, choice = [9, 5, 6, 7, 8, 8, 9], [6, 0, 8, 0, 3, 4, 9]
    assert po.tree_accept(tokens, parents, choice, [0, 7], 7) == ([[0, 2, 4]], [3])
    assert po.tree_accept(tokens, parents, choice, [0, 0], 7) == ([[]], [-1])
    assert po.tree_accept(tokens, parents, choice, [0, 7], 3) == ([[0, 2]], [8])


def test_plain_attention_is_a_softmax():
    rng = np.random.default_rng(0)
    c = po.Cache(rng.standard_normal((1, 3, 1, 16, 64)).astype(np.float16), rng.standard_normal((1, 3, 1, 16, 64)).astype(np.float16), np.array([[2, 0]], np.int32))
    q = rng.standard_normal((2, 64)).astype(np.float32)
    out, tol = po.attention(c, 0, q, 1, [0, 2], [17], None, 2, np.array([[0b01], [0b11]]), 0.125, 2.0 ** -24, 0.0)
    k, v = (np.concatenate([x[0, 2, 0], x[0, 0, 0]]).astype(np.float64) for x in (c.k, c.v))
    for t, n in ((0, 18), (1, 19)):
        p = np.exp(0.125 * k[:n] @ q[t].astype(np.float64))
        assert np.allclose(out[t, 0], p @ v[:n] / p.sum(), rtol=1e-12, atol=1e-12) and (tol[t] < 1e-4).all()
