"""The operators of a long context without a device: what they refuse, calls without work, and the frequencies of scaled rotary positions."""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest

from powerinfer_b200 import _lib

lib = _lib.lib
P = 1 << 20                      # a fake, aligned "device pointer": validation never dereferences it
F32, F16 = _lib.PI_TYPE_F32, _lib.PI_TYPE_F16
INVALID, WORKSPACE = 1, 3


def err():
    return lib.pi_last_error().decode()


def cache(**over):
    c = dict(k=P, v=P, k_scale=P, v_scale=P, n_seq=2, n_head_kv=4, n_ctx=256, head_dim=128, block=64)
    c.update(over)
    return _lib.KvQ8(*c.values())


def batch(**over):
    b = dict(q_start=P, seq=None, pos0=P, n=2, T=2, max_new=1)
    b.update(over)
    return _lib.KvBatch(*b.values())


def rope(xtype=F32, q=P, qs=512, nh=4, qo=1 << 24, qos=512, k=None, ks=0, nk=0, ko=None, kos=0, T=2, hd=128, n_rot=128, pos=P, freqs=P):
    return lib.pi_rope_ext(xtype, q, qs, nh, qo, qos, k, ks, nk, ko, kos, T, hd, n_rot, 0, pos, freqs, 1.0, None)


def store(c=None, b=None, xtype=F32, k=P, ks=512, v=P, vs=512, fn="pi_kv_store_q8"):
    return getattr(lib, fn)(C.byref(c or cache()), C.byref(b or batch()), xtype, k, ks, v, vs, None)


def attention(c=None, b=None, xtype=F32, q=P, qs=1024, n_head=8, max_kv=256, out=1 << 24, outs=1024, w_in=None, w_out=None, ws=1 << 21, wsn=1 << 26):
    return lib.pi_attention_q8(C.byref(c or cache()), C.byref(b or batch()), xtype, q, qs, n_head, max_kv, 0.1, out, outs, w_in, w_out, ws, wsn, None)


def evict(c=None, lens=P, n=2, keep=128, sink=4, recent=32, w=P, w_out=None, kept=P):
    return lib.pi_kv_evict_q8(C.byref(c or cache()), lens, None, n, keep, sink, recent, w, w_out, kept, None)


@pytest.mark.parametrize("call,code,needle", [
    (lambda: rope(xtype=2), INVALID, "unknown type"),
    (lambda: rope(hd=12, nh=4, qs=48, qos=48, n_rot=4), INVALID, "multiple of 8"),
    (lambda: rope(n_rot=63), INVALID, "even"),
    (lambda: rope(n_rot=130), INVALID, "within"),
    (lambda: rope(hd=264, qs=2048, qos=2048), INVALID, "256"),
    (lambda: rope(q=P + 4), INVALID, "q must be 16-byte aligned"),
    (lambda: rope(qs=510), INVALID, "q must be"),
    (lambda: rope(qs=514), INVALID, "16 bytes apart"),
    (lambda: rope(qo=P + 2048), INVALID, "overlaps"),
    (lambda: rope(qo=P, qos=1024), INVALID, "overlaps"),
    (lambda: rope(k=P + 512 * 4 * 8, ks=256, nk=2, ko=(1 << 24) + 16, kos=256), INVALID, "each other's"),
    (lambda: rope(k=1 << 24, ks=512, nk=2, ko=1 << 25, kos=256), INVALID, "each other's"),
    (lambda: rope(k=P + 1024, ks=512, nk=2, ko=P, kos=512), INVALID, "each other's"),
    (lambda: rope(nk=2), INVALID, "rope_ext"),
    (lambda: rope(pos=None), INVALID, "positions"),
    (lambda: store(cache(head_dim=80)), INVALID, "head_dim"),
    (lambda: store(cache(block=24)), INVALID, "block"),
    (lambda: store(cache(n_ctx=200)), INVALID, "multiple of block"),
    (lambda: store(cache(k=None)), INVALID, "null cache"),
    (lambda: store(cache(v=P + 8)), INVALID, "16-byte"),
    (lambda: store(b=batch(q_start=None)), INVALID, "batch"),
    (lambda: store(b=batch(n=70000)), INVALID, "batch"),
    (lambda: store(b=batch(T=-1)), INVALID, "batch"),
    (lambda: store(xtype=7), INVALID, "unknown type"),
    (lambda: store(k=None), INVALID, "k must be"),
    (lambda: store(vs=256), INVALID, "v must be"),
    (lambda: store(fn="pi_kv_load_q8", k=None), INVALID, "k must be"),
    (lambda: store(cache(head_dim=80), fn="pi_kv_load_q8"), INVALID, "head_dim"),
    (lambda: attention(n_head=6), INVALID, "multiple of n_head_kv"),
    (lambda: attention(out=P), INVALID, "different"),
    (lambda: attention(out=P + 4096), INVALID, "different"),
    (lambda: attention(out=P - 16), INVALID, "different"),
    (lambda: attention(w_in=P), INVALID, "weights_out"),
    (lambda: attention(qs=1026), INVALID, "q must be"),
    (lambda: attention(cache(n_ctx=4096), max_kv=4096, ws=None, wsn=0), WORKSPACE, "workspace"),
    (lambda: attention(cache(n_ctx=4096), max_kv=4096, ws=(1 << 21) + 8), WORKSPACE, "workspace"),
    (lambda: attention(b=batch(T=1 << 24, max_new=1 << 24)), INVALID, "too many"),
    (lambda: evict(keep=100), INVALID, "multiple of block"),
    (lambda: evict(keep=0), INVALID, "keep"),
    (lambda: evict(keep=512), INVALID, "n_ctx"),
    (lambda: evict(keep=64, sink=40, recent=30), INVALID, "more than keep"),
    (lambda: evict(sink=-1), INVALID, "bad arguments"),
    (lambda: evict(lens=None), INVALID, "needed"),
    (lambda: evict(kept=None), INVALID, "needed"),
    (lambda: evict(cache(n_ctx=1 << 19)), INVALID, "262144"),
    (lambda: evict(w=P, w_out=P + 1024), INVALID, "the same array, or apart"),
    (lambda: attention(w_in=P + 4, w_out=P), INVALID, "the same array, or apart"),
    (lambda: store(fn="pi_kv_load_q8", k=P, v=P), INVALID, "k and v overlap"),
    (lambda: store(fn="pi_kv_load_q8", k=P, ks=768, v=P + 256 * 4, vs=768), INVALID, "k and v overlap"),
    (lambda: store(cache(n_head_kv=65535, n_ctx=1 << 30, block=16), batch(T=1 << 30, max_new=1 << 30), ks=65535 * 128, vs=65535 * 128), INVALID, "too many slots"),
])
def test_bad_arguments_are_refused_before_any_launch(call, code, needle):
    rc = call()
    assert rc == code, (rc, err())
    assert needle in err(), err()


def test_calls_without_work_are_ok():
    assert rope(T=0) == 0
    assert store(b=batch(n=0)) == 0 and store(b=batch(T=0)) == 0 and store(b=batch(max_new=0)) == 0
    assert store(b=batch(n=0), fn="pi_kv_load_q8") == 0
    assert attention(b=batch(n=0)) == 0 and attention(b=batch(T=0)) == 0
    assert evict(n=0) == 0


def workspace(c, b, n_head, max_kv, weights=0):
    return lib.pi_attention_q8_workspace_bytes(C.byref(c), C.byref(b), n_head, max_kv, weights)


def test_workspace_sizes():
    """One split needs nothing; a long range of one sequence is split; weights need a normaliser for each row; a refused call has no size."""
    assert workspace(cache(), batch(), 8, 256) == 0
    assert workspace(cache(n_ctx=32768), batch(n=1, T=1), 8, 32768) > 0
    assert workspace(cache(), batch(), 8, 256, 1) >= 2 * 8 * 4
    assert workspace(cache(), batch(), 6, 256) == 0 and "multiple" in err()


@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("n,new,group", [(1, 1, 8), (50, 1, 8), (37, 1, 1), (3, 20, 4), (2, 1000, 8), (400, 1, 16)])
def test_partial_sums_stay_small(hd, n, new, group):
    """Partial sums are of the last round's items: a few rounds of 444 CTAs of 8 rows, or of 148 of 128, however long the context is."""
    for n_ctx in (4096, 1 << 20):
        got = workspace(cache(n_seq=1, head_dim=hd, n_ctx=n_ctx), batch(n=n, T=n * new, max_new=new), 4 * group, n_ctx)
        assert got <= 4 * 444 * 16 * (hd * 4 + 8) * 3 + 4096


def freqs(n_rot, base=10000.0, scale=1.0, ext=0.0, attn=1.0, fast=32.0, slow=1.0, orig=0, factors=None):
    out, m = np.empty(n_rot // 2), C.c_float()
    f = None if factors is None else np.asarray(factors, np.float32)
    rc = lib.pi_rope_freqs_host(out.ctypes.data, C.addressof(m), n_rot, base, scale, ext, attn, fast, slow, orig, None if f is None else f.ctypes.data)
    assert rc == 0, err()
    return out, m.value


def test_frequencies_unscaled_linear_and_by_factors():
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    f, m = freqs(64)
    assert np.allclose(f, plain, rtol=1e-14) and m == 1.0
    f, m = freqs(64, scale=0.25, attn=1.5)
    assert np.allclose(f, np.array(plain) / 4, rtol=1e-14) and m == 1.5
    by = np.linspace(1, 8, 32).astype(np.float32)
    f, _ = freqs(64, factors=by)
    assert np.allclose(f, plain / by.astype(np.float64), rtol=1e-14)


@pytest.mark.parametrize("n_rot,scale,orig", [(64, 0.25, 2048), (128, 1 / 16, 4096), (32, 0.5, 512)])
def test_frequencies_of_yarn(n_rot, scale, orig):
    """Fast pairs keep their angle, slow ones are stretched, between them there is a ramp; the factor grows with the logarithm of the stretch."""
    f, m = freqs(n_rot, scale=scale, ext=1.0, orig=orig)
    plain, _ = freqs(n_rot)
    turns = orig * plain / (2 * math.pi)
    share = f / plain                                                  # 1: kept, scale: stretched
    assert np.all(np.diff(share) <= 1e-12) and np.all(share >= scale * (1 - 1e-6)) and np.all(share <= 1 + 1e-12)
    lo = max(0, math.floor(n_rot * math.log(orig / (32 * 2 * math.pi)) / (2 * math.log(10000.0))))
    hi = min(n_rot - 1, math.ceil(n_rot * math.log(orig / (2 * math.pi)) / (2 * math.log(10000.0))))
    for i in range(n_rot // 2):
        keep = 1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
        assert share[i] == pytest.approx(keep + (1 - keep) * scale, rel=1e-6), (i, turns[i])
    assert m == pytest.approx(1 + 0.1 * math.log(1 / scale), rel=1e-6)


@pytest.mark.parametrize("bad", [dict(n_rot=63), dict(n_rot=0), dict(n_rot=512), dict(base=1.0), dict(scale=0.0), dict(ext=1.0)])
def test_frequencies_refuse(bad):
    a = dict(n_rot=64, base=10000.0, scale=1.0, ext=0.0)
    a.update(bad)
    out, m = np.empty(256), C.c_float()
    assert lib.pi_rope_freqs_host(out.ctypes.data, C.addressof(m), a["n_rot"], a["base"], a["scale"], a["ext"], 1.0, 32.0, 1.0, 0, None) == INVALID
    assert "rope_freqs" in err()


def test_the_prompt_kernel_gives_tensor_memory_back_when_no_product_is_in_flight():
    """The issuing warp waits for its last products, also after a wait ran out (no look at s_dead); copies on their way land before the CTA ends; the threads that meet
    at a named barrier come to it whatever ran out."""
    text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "pi_attn_q8_tc.cu")).read()
    assert text.count("tc_dealloc(") == 1
    assert re.search(r"tc_commit\(&(\w+)\);[^\n]*\n *for \(int spins = 0; spins < \(1 << 20\) && !mbar_try_wait\(&\1, 0u\); spins\+\+\) \{\}\n *__syncwarp\(\);", text)
    assert "ring_land(s_rfull, i, AT_RAW)" in text
    loop = text[text.index("for (int i = b; i < n_tiles; i += 2)"):text.index("// ================================================================= tiles in, sums out")]
    assert "bar.sync" in loop and not re.search(r"\b(break|return);", re.sub(r"if \([^)]*parts\) break;", "", loop))


def test_the_prompt_kernel_writes_no_numbers_after_any_wait_ran_out():
    """(A wait cannot be made to run out on the device without a broken kernel.)  The warps that make probabilities go on behind a wait that ran out and arrive at the
    barrier that the draining warps wait for, so these look at the flag that the others have set before."""
    text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "pi_attn_q8_tc.cu")).read()
    give_up = text[text.index("auto wait = [&]"):text.index("// ---- codes: keys and values in turn")]
    assert give_up.index("s_dead = 1") < give_up.index("return ok;")
    out = text[text.index("for (int i = max(0, n_tiles - 2); i < n_tiles && ok; i++) drain(i);"):]
    assert "s_dead) sum = __int_as_float(0x7fc00000);" in out[:out.index("p.part")]


def test_the_status_word_of_a_prompt_is_cleared_before_its_launch():
    """No CTA clears what another one may have set by then."""
    text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "pi_attn_q8_tc.cu")).read()
    assert not re.search(r"\*p\.status\s*=", text)
    assert text.index("launch_k(k_attn_q8_clear") < text.index("launch_k(k_attn_q8_tc")


@pytest.mark.parametrize("n_ctx,block", [(128, 96), (96, 64), (160, 64), (100, 64), (0, 64), (128, 0), (128, -64)])
def test_an_empty_cache_has_the_block_that_was_asked_for(n_ctx, block):
    """(128 slots in blocks of 96 made a cache with one block of 128.)"""
    ggml_ops = pytest.importorskip("powerinfer_b200.ggml_ops")
    with pytest.raises(ValueError, match="multiple of block"):
        ggml_ops.KvCacheQ8.empty(1, n_ctx, 1, 64, block)
