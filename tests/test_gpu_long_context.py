"""The operators of a long context against plain ones in 64 bits (long_context_oracle): rotary positions, the KV cache in 8 bits, its
attention with accumulated weights, eviction, and a run of all of them.

Tolerances.  Half a step is u = 2^-24 in FP32 and 2^-11 in FP16.
  rope       cosine and sine: 2 u from the reduced angle and its function, u from the factor; two products and a sum: 3 u of |x0| + |x1|.  With a
             margin of one third 8 u (|x0| + |x1|) mscale, and in FP16 the result's own rounding.
  store      codes and scales are defined by their FP32 steps: equal.
  attention  a query is held to 2^-22 of its row's largest value, sums of hd products are off by at most hd u, the factor of the scores by 3 u:
             with E = scale * max_j sum_d |q_d k_jd| a score is off by at most E (2^-22 + (hd + 3) u), and as E log2(e) is the largest size of an exponent its
             rounding by 2 E u: e_s = E (hd + 10) u in all.  A probability is then off by 2 e_s of itself, 4 u from exp2 (2 ulp),
             4 u from its product with the scale and its two halves, both sums by n u at most.  So an output is off by at most sum_j p_j |v_j| * (2 e_s + (2 n + 16) u); sums on
             the tensor cores are cut, not rounded: twice the u of sums.  The lower half of a probability has no steps below 2^-24 of what it
             is held times, 2^7 or more over the largest scale of values so far, beside which the largest probability is 1 or more: what is left out is
             2^-25 / 2^7 = 2^-32 of the largest value that a block holds, for each slot.  (Peaked softmaxes show it where the one value that counts is 0.)
  weights    the same of the sum of probabilities, over the tokens and heads that it adds.
"""
import numpy as np
import pytest

import long_context_oracle as lc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
TYPES = {"f32": torch.float32, "f16": torch.float16}
NP = {"f32": np.float32, "f16": np.float16}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from powerinfer_b200 import ggml_ops
    return ggml_ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rows(rng, T, n, x="f32"):
    return rng.standard_normal((T, n), dtype=np.float32).astype(NP[x])


# ------------------------------------------------------------------------------------------------ rotary positions

@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("T,heads,heads_kv,hd,n_rot,far", [
    (1, 4, 2, 64, 64, 7), (3, 64, 8, 128, 128, 100000), (5, 3, 1, 96, 42, 1000000), (2, 7, 7, 256, 256, 131072), (17, 8, 8, 192, 2, 500),
    (130, 16, 2, 64, 32, 4096), (1, 2, 1, 8, 8, 3), (4, 1, 1, 24, 16, 2000000), (3, 5, 0, 80, 48, 60000)])
def test_rope_against_64_bits(ops, x, halves, T, heads, heads_kv, hd, n_rot, far):
    rng = np.random.default_rng(T * 1000 + hd + n_rot)
    f = ops.rope_freqs(n_rot, freq_scale=0.125, ext_factor=1.0, n_orig_ctx=2048)
    fh = f.freqs.cpu().numpy()
    pos = np.concatenate([[0], rng.integers(0, far, T - 1)]).astype(np.int32) if T > 1 else np.array([far - 1], np.int32)
    qkv = rows(rng, T, (heads + 2 * heads_kv) * hd, x)
    nq, nk = heads * hd, heads_kv * hd
    on = dev(qkv)
    q, k = ops.rope_ext(on[:, :nq], on[:, nq:nq + nk] if heads_kv else None, ints(pos.tolist()), f, hd, mode=2 if halves else 0)
    for got, host in ((q, qkv[:, :nq]), (k, qkv[:, nq:nq + nk])):
        if got is None:
            continue
        want = lc.rope(host, pos, fh, f.mscale, hd, halves)
        h = np.abs(host.astype(np.float64)).reshape(T, -1, hd)
        pair = h.copy()
        half = n_rot // 2
        i0, i1 = (np.arange(half), np.arange(half) + half) if halves else (np.arange(half) * 2, np.arange(half) * 2 + 1)
        pair[..., i0] = pair[..., i1] = h[..., i0] + h[..., i1]
        tol = 8 * U["f32"] * pair.reshape(T, -1) * f.mscale + (U[x] * np.abs(want) + 2.0 ** -25 if x == "f16" else 0.0)
        assert np.all(np.abs(got.cpu().numpy().astype(np.float64) - want) <= tol)
        assert np.array_equal(got.cpu().numpy().reshape(T, -1, hd)[..., n_rot:], host.reshape(T, -1, hd)[..., n_rot:])     # the others pass
    assert np.array_equal(on.cpu().numpy(), qkv)                       # the inputs are left alone
    before = on.clone()
    q2, k2 = ops.rope_ext(on[:, :nq], on[:, nq:nq + nk] if heads_kv else None, ints(pos.tolist()), f, hd, mode=2 if halves else 0, inplace=True)
    assert torch.equal(q2, q) and (k is None or torch.equal(k2, k)) and torch.equal(on[:, nq + nk:], before[:, nq + nk:])


def test_rope_agrees_with_the_table_form(ops):
    """Positions of a short context: the same rotation as ggml_rope_custom's, whose table is a recurrence in FP32 (off by about 64 u of the angle)."""
    x = torch.randn(9, 4 * 64, device="cuda")
    pos = ints(list(range(9)))
    table = ops.rope_table(16, 64, 10000.0)
    for mode in (0, 2):
        a = ops.ggml_rope_custom(x.view(9, 4, 64), pos, 64, mode, table).reshape(9, -1)
        b, _ = ops.rope_ext(x, None, pos, ops.rope_freqs(64), 64, mode)
        assert (a - b).abs().max().item() <= 9 * 64 * U["f32"] * 6


def test_rope_refuses(ops):
    f = ops.rope_freqs(64)
    q, pos = torch.zeros(2, 128, device="cuda"), ints([0, 1])
    with pytest.raises(ValueError):
        ops.rope_ext(q, torch.zeros(2, 64, device="cuda", dtype=torch.float16), pos, f, 64)
    with pytest.raises(ValueError):
        ops.rope_ext(q, torch.zeros(3, 64, device="cuda"), pos, f, 64)
    with pytest.raises(ValueError):
        ops.rope_ext(q, None, pos.long(), f, 64)
    with pytest.raises(ValueError):
        ops.rope_ext(q.double(), None, pos, f, 64)
    with pytest.raises(ValueError):
        ops.rope_ext(torch.zeros(2, 129, device="cuda")[:, 1:], None, pos, f, 64, inplace=True)
    with pytest.raises(ValueError):
        ops.rope_ext(q, None, pos.cpu(), f, 64)
    a, _ = ops.rope_ext(torch.ones(2, 129, device="cuda")[:, 1:], None, pos, f, 64)         # odd addresses are copied first
    b, _ = ops.rope_ext(torch.ones(2, 128, device="cuda"), None, pos, f, 64)
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ store and load

class Pair:
    """A cache on the device and the oracle's"""

    def __init__(self, ops, n_seq, H, n_ctx, hd, block, fill=None):
        self.ops, self.c = ops, lc.Cache(n_seq, H, n_ctx, hd, block)
        if fill is not None:
            for n in "kv":
                self.c.codes[n][:] = np.clip(np.rint(fill.standard_normal(self.c.codes[n].shape) * 30), -127, 127)
                self.c.scale[n][:] = np.exp(fill.standard_normal(self.c.scale[n].shape) * 0.5) / 30
        self.d = ops.KvCacheQ8(dev(self.c.codes["k"]), dev(self.c.codes["v"]), dev(self.c.scale["k"]), dev(self.c.scale["v"]))

    def store(self, k, v, q_start, pos0, seq=None, max_new=None):
        self.ops.kv_store_q8(self.d, dev(k), dev(v), ints(q_start), ints(pos0), None if seq is None else ints(seq), max_new)
        self.c.store(k, v, q_start, pos0, seq, len(k) if max_new is None else max_new)

    def same(self):
        for n, codes, scale in (("k", self.d.k, self.d.k_scale), ("v", self.d.v, self.d.v_scale)):
            assert np.array_equal(scale.cpu().numpy(), self.c.scale[n])
            assert np.array_equal(codes.cpu().numpy(), self.c.codes[n])


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,block", [(64, 16), (96, 32), (128, 64), (192, 16), (256, 128)])
def test_store_token_by_token_and_in_chunks(ops, x, hd, block):
    """Prompts of different lengths, then single tokens through open blocks whose scale grows; what is behind the new tokens keeps its bits."""
    rng = np.random.default_rng(hd + block)
    p = Pair(ops, 4, 3, 512, hd, block, fill=rng)
    lens = [131, 1, 0, 40]
    start = np.concatenate([[0], np.cumsum(lens)]).tolist()
    T = start[-1]
    k, v = rows(rng, T, 3 * hd, x), rows(rng, T, 3 * hd, x)
    p.store(k, v, start, [0, 5, 9, 300], seq=[2, 0, 3, 1])
    p.same()
    for step in range(6):
        size = 0.5 * 1.7 ** step                                       # every token larger than those before it
        k, v = (rows(rng, 4, 3 * hd, x).astype(np.float32) * size).astype(NP[x]), rows(rng, 4, 3 * hd, x)
        p.store(k, v, [0, 1, 2, 3, 4], [131 + step, 6 + step, step, 340 + step], seq=[2, 0, 3, 1], max_new=1)
        p.same()
    few = rows(rng, 7, 3 * hd, x)
    p.store(few, few, [0, 3, 7], [block - 2, 2 * block - 1], seq=[0, 2], max_new=4)            # across a block's end
    p.same()


def test_store_edges(ops):
    rng = np.random.default_rng(5)
    p = Pair(ops, 3, 2, 128, 64, 32, fill=rng)
    # not finite, zeros, values below the normal numbers, the largest ones
    k = rows(rng, 8, 128)
    k[0, :5], k[1, :64], k[2, 3], k[3] = np.inf, np.nan, -np.inf, 0.0
    k[4], k[5] = 1e-42, np.float32(3.4e38)
    v = np.zeros_like(k)
    v[6], v[7, 64:] = 1e-39, 1e-30
    p.store(k, v, [0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 32, 64, 96, 0, 32, 64, 96], seq=[0, 0, 0, 0, 1, 1, 1, 1])   # (a sequence again: the last of its entries)
    p.same()
    for i in range(8):
        p.store(k[i:i + 1], v[i:i + 1], [0, 1], [16 * i], seq=[i % 3])
        p.same()
    # entries that the cache cannot hold, starts outside the rows, lengths below zero: nothing is touched
    p.store(k, v, [0, 2, 4, 6, 8], [-1, 128, 5, 7], seq=[0, 1, 3, -1])
    p.store(k, v, [5, 2, 20, 3], [0, 0, 0], seq=[0, 1, 2])
    p.same()
    p.store(k, v, [0, 8], [124], seq=[2])                               # runs over the end
    p.same()
    p.store(k, v, [0, 8], [8], seq=[1], max_new=3)                      # more tokens than max_new
    p.same()
    # the same sequence several times, one of the later ones without tokens
    p.store(k, v, [0, 3, 6, 6, 8], [40, 44, 0, 0], seq=[2, 2, 2, 0])
    p.same()


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_load_gives_the_values(ops, x):
    rng = np.random.default_rng(11)
    p = Pair(ops, 3, 5, 256, 96, 16, fill=rng)
    start, pos, seq = [0, 100, 100, 117, 125], [3, 0, 200, -1], [2, 1, 0, 1]
    k, v = ops.kv_load_q8(p.d, ints(start), ints(pos), 140, ints(seq), dtype=TYPES[x])
    for got, n in ((k, "k"), (v, "v")):
        got = got.cpu().numpy().reshape(140, 5, 96)
        for i in (0, 2):
            m = start[i + 1] - start[i]
            want = (p.c.codes[n][seq[i], :, pos[i]:pos[i] + m].astype(np.float32) * np.repeat(p.c.scale[n][seq[i]], 16, 1)[:, pos[i]:pos[i] + m, None]).transpose(1, 0, 2)
            assert np.array_equal(got[start[i]:start[i + 1]], want.astype(NP[x]))
        assert np.all(got[117:125] == 0)                               # an entry without a place in the cache


def test_store_takes_strided_rows_and_refuses_others(ops):
    rng = np.random.default_rng(3)
    a, b = (Pair(ops, 1, 2, 64, 64, 16) for _ in range(2))
    qkv = rows(rng, 9, 6 * 64)
    on = dev(qkv)
    ops.kv_store_q8(a.d, on[:, 128:256], on[:, 256:], ints([0, 9]), ints([2]))
    b.store(qkv[:, 128:256].copy(), qkv[:, 256:].copy(), [0, 9], [2])
    b.same()
    assert torch.equal(a.d.k, b.d.k) and torch.equal(a.d.v_scale, b.d.v_scale)
    odd = dev(np.concatenate([np.zeros((9, 1), np.float32), qkv[:, 128:]], 1))
    ops.kv_store_q8(a.d, odd[:, 1:129], odd[:, 129:], ints([0, 9]), ints([2]))                # odd addresses are copied first
    assert torch.equal(a.d.k, b.d.k)
    with pytest.raises(ValueError):
        ops.kv_store_q8(a.d, on[:, :64], on[:, :64], ints([0, 9]), ints([2]))
    with pytest.raises(ValueError):
        ops.kv_store_q8(a.d, on[:, :128], on[:5, :128], ints([0, 9]), ints([2]))
    with pytest.raises(ValueError):
        ops.kv_store_q8(a.d, on[:, :128], on[:, :128], ints([0]), ints([2]))
    with pytest.raises(ValueError):
        ops.kv_store_q8(a.d, on[:, :128], on[:, :128], torch.tensor([0, 9], device="cuda"), ints([2]))
    with pytest.raises(ValueError):
        ops.KvCacheQ8(a.d.k, a.d.v[..., :32], a.d.k_scale, a.d.v_scale)
    with pytest.raises(ValueError):
        ops.KvCacheQ8(a.d.k.float(), a.d.v, a.d.k_scale, a.d.v_scale)


# ------------------------------------------------------------------------------------------------ attention

def attention_bound(size, terms, most, hd, n, x, want):
    u = U["f32"]
    per_row = 2 * terms * (hd + 10) * 2 * u + (4 * n + 16) * u
    group = size.reshape(size.shape[0], terms.shape[1], -1) * per_row[..., None] + 2.0 ** -32 * most[..., None]
    tol = group.reshape(size.shape) + 1e-30
    return tol + (U["f16"] * (np.abs(want) + tol) + 2.0 ** -25 if x == "f16" else 0.0)


def run_attention(ops, p, rng, q_start, pos0, n_head, x="f32", seq=None, max_new=None, max_kv=None, weights=False, T=None, scale=None, size=1.0, q=None):
    hd, T = p.c.hd, q_start[-1] if T is None else T
    q = (rows(rng, T, n_head * hd, "f32") * np.float32(size)).astype(NP[x]) if q is None else q
    scale_ = 1.0 / np.sqrt(hd) if scale is None else scale
    shape = (p.c.n_seq, p.c.H, p.c.n_ctx)
    w_in = rng.random(shape, dtype=np.float32) if weights else None
    w_want = np.full(shape, 7.0) if weights else None
    w_got = torch.full(shape, 7.0, device="cuda") if weights else None
    fill = np.full((T, n_head * hd), 5.0)
    out = torch.full((T, n_head * hd), 5.0, device="cuda", dtype=TYPES[x])
    got = ops.attention_q8(p.d, dev(q), ints(q_start), ints(pos0), None if seq is None else ints(seq), max_new, max_kv, scale,
                           None if w_in is None else dev(w_in), w_got, out)
    assert got is out
    want, err, terms, most = p.c.attention(q, n_head, scale_, q_start, pos0, seq, T if max_new is None else max_new, w_in, w_want, fill)
    n = max([min(p.c.n_ctx, a + b - c) for a, b, c in zip(pos0, q_start[1:], q_start)] + [1])
    g = got.float().cpu().numpy().astype(np.float64)
    tol = attention_bound(err, terms, most, hd, max(n, 1), x, want)
    off = np.abs(g - want)
    assert np.all(off <= tol), (float(off.max()), float((off / tol).max()), np.unravel_index((off / tol).argmax(), off.shape))
    if weights:
        gw = w_got.cpu().numpy().astype(np.float64)
        wt = np.abs(w_want) * (2 * terms.max() * (hd + 10) * 2 + 4 * n + 4 * T * n_head // p.c.H + 16) * U["f32"]
        assert np.all(np.abs(gw - w_want) <= wt)
    return got


SHAPES = [(64, 16), (96, 32), (128, 64), (128, 16), (192, 32), (256, 128)]


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,block", SHAPES)
@pytest.mark.parametrize("group", [1, 3, 8, 9, 16])
def test_attention_of_single_tokens(ops, x, hd, block, group):
    """Sequences from one slot to some hundreds, in another order than the batch's, with and without weights; rows behind the last entry stay."""
    rng = np.random.default_rng(hd * 10 + group)
    p = Pair(ops, 6, 2, 640, hd, block, fill=rng)
    run_attention(ops, p, rng, [0, 1, 2, 3, 4, 5], [0, 14, 63, 64, 639], 2 * group, x, seq=[4, 0, 5, 1, 2], max_new=1, weights=group == 3, T=7)


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,block", SHAPES)
@pytest.mark.parametrize("group,lens,pos0", [(1, [2, 1, 9], [0, 30, 200]), (8, [1, 5, 0, 3], [10, 0, 7, 255]), (4, [33, 70], [100, 0]), (7, [20], [301])])
def test_attention_of_several_tokens(ops, x, hd, block, group, lens, pos0):
    """Prompts and chunks: every token sees the slots up to its own."""
    rng = np.random.default_rng(hd + group + len(lens))
    p = Pair(ops, 4, 3, 384, hd, block, fill=rng)
    start = np.concatenate([[0], np.cumsum(lens)]).tolist()
    run_attention(ops, p, rng, start, pos0, 3 * group, x, seq=[3, 1, 0, 2][:len(lens)], max_new=max(lens), weights=group != 1, T=start[-1] + 2)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [4095, 4096, 5000])
@pytest.mark.parametrize("max_kv", [None, 1, 300, 100000])
def test_attention_over_split_ranges(ops, hd, n, max_kv):
    """One long sequence and a short one: the range is cut, and joined; the expected length is only an expectation."""
    rng = np.random.default_rng(n + hd)
    p = Pair(ops, 2, 1, 5120, hd, 64, fill=rng)
    run_attention(ops, p, rng, [0, 1, 2], [n - 1, 70], 8, seq=[1, 0], max_kv=max_kv, weights=True)
    run_attention(ops, p, rng, [0, 3], [n - 3], 4, "f16", seq=[1], max_kv=max_kv)


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,lens,pos0,group", [(128, [129, 300, 17], [0, 200, 40], 8), (64, [257, 64], [13, 700], 16), (128, [260], [0], 1), (64, [140], [511], 5)])
def test_attention_of_long_prompts(ops, x, hd, lens, pos0, group):
    rng = np.random.default_rng(hd + lens[0])
    p = Pair(ops, 3, 2, 1024, hd, 32, fill=rng)
    start = np.concatenate([[0], np.cumsum(lens)]).tolist()
    run_attention(ops, p, rng, start, pos0, 2 * group, x, seq=[2, 0, 1][:len(lens)], weights=lens[0] == 260)


def test_attention_with_large_and_small_queries(ops):
    """Peaked and flat softmaxes, and queries beyond what halves hold."""
    rng = np.random.default_rng(8)
    p = Pair(ops, 1, 2, 512, 128, 64, fill=rng)
    for size in (1e-6, 1e-3, 8.0):
        run_attention(ops, p, rng, [0, 1], [500], 8, size=size)
        run_attention(ops, p, rng, [0, 140], [300], 8, size=size)
    run_attention(ops, p, rng, [0, 1], [500], 8, size=1e6, scale=1e-7)
    run_attention(ops, p, rng, [0, 140], [300], 8, size=1e6, scale=1e-7)
    run_attention(ops, p, rng, [0, 1], [500], 8, scale=0.0)
    run_attention(ops, p, rng, [0, 1], [500], 8, scale=-0.1)
    q = np.zeros((2, 8 * 128), np.float32)
    run_attention(ops, p, rng, [0, 2], [37], 8, q=q)


@pytest.mark.parametrize("T", [1, 3, 150])
def test_attention_does_not_see_what_is_masked(ops, T):
    """Scales that are not finite, and any codes, behind a sequence's slots leave no trace; entries that the cache lacks have zeros."""
    rng = np.random.default_rng(T)
    p = Pair(ops, 4, 2, 512, 64, 16, fill=rng)
    n = T + 33
    end = (n + 15) // 16
    for s in (p.c.scale["k"], p.c.scale["v"]):
        s[0, :, end:], s[1, :, end:], s[2], s[3] = np.nan, np.inf, np.nan, -np.inf
    p.d.k_scale.copy_(dev(p.c.scale["k"]))
    p.d.v_scale.copy_(dev(p.c.scale["v"]))
    run_attention(ops, p, rng, [0, T, 2 * T, 3 * T, 4 * T], [33, 33, -1, 512], 16, seq=[1, 0, 2, 3], max_new=T, weights=True)
    run_attention(ops, p, rng, [0, T, 2 * T], [33, 33], 16, seq=[0, 9], max_new=T)
    run_attention(ops, p, rng, [0, T, 2 * T], [33, 33], 16, seq=[-4, 1], max_new=T)
    run_attention(ops, p, rng, [3, T, 90 * T, 1], [33, 33, 33], 4, seq=[1, 0, 0], max_new=T, T=T)             # starts and ends that make no sense


def test_attention_at_the_end_of_the_cache(ops):
    """Tokens whose slots lie behind the cache see nothing, the others everything up to theirs."""
    rng = np.random.default_rng(21)
    p = Pair(ops, 2, 2, 256, 128, 128, fill=rng)
    for T in (5, 150):
        run_attention(ops, p, rng, [0, T], [254], 8, seq=[1], weights=True)
        run_attention(ops, p, rng, [0, T], [256 - T], 8, seq=[1], weights=True)


def test_attention_zero_scales_and_equal_scores(ops):
    """A sequence of zeros: every slot counts the same; blocks of zeros between others."""
    rng = np.random.default_rng(2)
    p = Pair(ops, 2, 1, 256, 64, 16, fill=rng)
    for n in "kv":
        p.c.scale[n][0] = 0
        p.c.scale[n][1, :, ::2] = 0
    p.d.k_scale.copy_(dev(p.c.scale["k"]))
    p.d.v_scale.copy_(dev(p.c.scale["v"]))
    for T in (1, 2, 130):
        run_attention(ops, p, rng, [0, T, 2 * T], [100, 99], 4, max_new=T, weights=True)


def test_attention_values_of_very_different_sizes(ops):
    """Scales of values over twelve orders, rising and falling: sums are held relative to the largest so far."""
    rng = np.random.default_rng(4)
    p = Pair(ops, 2, 2, 512, 128, 16, fill=rng)
    p.c.scale["v"][0] = np.logspace(-9, 3, 32, dtype=np.float32)
    p.c.scale["v"][1] = np.logspace(3, -9, 32, dtype=np.float32)
    p.d.v_scale.copy_(dev(p.c.scale["v"]))
    for T in (1, 140):
        run_attention(ops, p, rng, [0, T, 2 * T], [512 - T, 512 - T], 16, max_new=T)


@pytest.mark.parametrize("T", [1, 140])
def test_attention_values_of_the_smallest_scales(ops, T):
    """Scales of values from the smallest normal number on.  Below 2^-118 probabilities are held times 2^8 over 2^-118, at 2^-126 times 1: what their
    lower halves leave out is 2^-25 of the largest value.  Sums near the smallest numbers are off by half of 2^-149 wherever they are rounded: once a tile
    or warp, once a split, once where they are put out."""
    rng = np.random.default_rng(T)
    p = Pair(ops, 2, 2, 512, 128, 16, fill=rng)
    p.c.scale["v"][0] = 2.0 ** -126
    p.c.scale["v"][1] = 2.0 ** rng.integers(-126, -112, (2, 32)).astype(np.float32)
    p.c.scale["v"][1, :, 0] = 2.0 ** -126
    p.d.v_scale.copy_(dev(p.c.scale["v"]))
    q, start, at, up = rows(rng, 2 * T, 16 * 128), [0, T, 2 * T], [512 - T, 512 - T], 2.0 ** 100
    got = ops.attention_q8(p.d, dev(q), ints(start), ints(at)).cpu().numpy().astype(np.float64) * up
    want, size, terms, most = p.c.attention(q, 16, 128 ** -0.5, start, at)
    tol = attention_bound(size * up, terms, most * up * 2 ** 7, 128, 512, "f32", want) + 32 * 2.0 ** -149 * up
    assert np.all(np.abs(got - want * up) <= tol)


def test_attention_nan_and_inf_stay_in_their_rows(ops):
    """A query that is not a number gives rows of no number, its neighbours' are untouched; so does a scale that a row sees."""
    rng = np.random.default_rng(6)
    p = Pair(ops, 2, 1, 256, 64, 16, fill=rng)
    for T in (1, 140):
        q = rows(rng, 2 * T, 8 * 64)
        clean = ops.attention_q8(p.d, dev(q), ints([0, T, 2 * T]), ints([100, 60]), max_new=T)
        bad = q.copy()
        bad[T // 2, 64 * 3] = np.nan
        bad[T, 64 * 5 + 7] = np.inf
        got = ops.attention_q8(p.d, dev(bad), ints([0, T, 2 * T]), ints([100, 60]), max_new=T)
        hurt = torch.zeros_like(got, dtype=torch.bool)
        hurt[T // 2, 64 * 3:64 * 4] = True
        hurt[T, 64 * 5:64 * 6] = True
        assert torch.isnan(got[hurt]).all() and torch.equal(got[~hurt], clean[~hurt])
    p.d.v_scale[0, 0, 2] = float("nan")
    got = ops.attention_q8(p.d, dev(q), ints([0, 140, 280]), ints([0, 0]), max_new=140)
    seen = torch.arange(140, device="cuda") >= 32
    assert torch.isnan(got[:140][seen]).all() and torch.isfinite(got[:140][~seen]).all() and torch.isfinite(got[140:]).all()


def test_attention_offsets_past_32_bits(ops):
    """A cache of more than 2^31 codes: the last sequence is read where it lies."""
    rng = np.random.default_rng(9)
    n_ctx, H, hd, n_seq = 65536, 8, 128, 33
    assert n_seq * n_ctx * H * hd > 1 << 31
    small = Pair(ops, 1, H, 256, hd, 64, fill=rng)
    k, v = (torch.empty(n_seq, H, n_ctx, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(n_seq, H, n_ctx // 64, device="cuda") for _ in range(2))
    big = ops.KvCacheQ8(k, v, ks, vs)
    at = n_ctx - 256
    new_k, new_v = rows(rng, 200, H * hd), rows(rng, 200, H * hd)
    ops.kv_store_q8(big, dev(new_k), dev(new_v), ints([0, 200]), ints([at]), ints([32]))
    small.store(new_k, new_v, [0, 200], [0])
    assert torch.equal(k[32, :, at:at + 200], small.d.k[0, :, :200])
    got_k, _ = ops.kv_load_q8(big, ints([0, 200]), ints([at]), 200, ints([32]))
    want_k, _ = ops.kv_load_q8(small.d, ints([0, 200]), ints([0]), 200)
    assert torch.equal(got_k, want_k)
    k[32, :, :at], v[32, :, :at] = 0, 0
    ks[32, :, :at // 64], vs[32, :, :at // 64] = 0, 0
    q = dev(rows(rng, 1, H * 8 * hd))
    got = ops.attention_q8(big, q, ints([0, 1]), ints([at + 199]), ints([32]), max_kv=n_ctx)
    # zeros in front: scores of 0 with values of 0, so the sums are those of the 200 slots over a larger normaliser
    lse = []
    for h in range(H):
        kk = torch.from_numpy(small.c.values("k", 0, h, 200)).cuda()
        s = q.double().view(H, 8, hd)[h] @ kk.T / hd ** 0.5
        vv = torch.from_numpy(small.c.values("v", 0, h, 200)).cuda()
        e = torch.exp(s)
        lse.append((e @ vv) / (e.sum(-1, keepdim=True) + at))
    want = torch.stack(lse).reshape(1, -1)
    assert (got - want).abs().max().item() <= 1e-5 * want.abs().max().item()


def test_attention_refuses(ops):
    rng = np.random.default_rng(1)
    p = Pair(ops, 1, 2, 64, 64, 16, fill=rng)
    q, s, z = torch.zeros(1, 256, device="cuda"), ints([0, 1]), ints([3])
    for bad in (dict(q=torch.zeros(1, 250, device="cuda")), dict(q=torch.zeros(1, 192, device="cuda")), dict(q=q.double()), dict(q_start=ints([0])),
                dict(out=torch.zeros(1, 128, device="cuda")), dict(weights_out=torch.zeros(1, 2, 32, device="cuda")), dict(weights_in=torch.zeros(1, 2, 64, device="cuda")),
                dict(pos0=torch.tensor([3], device="cuda")), dict(q=q.cpu()), dict(seq=ints([0, 0])), dict(out=q)):
        a = dict(q=q, q_start=s, pos0=z)
        a.update(bad)
        with pytest.raises((ValueError, RuntimeError)):
            ops.attention_q8(p.d, **a)
    assert ops.attention_q8(p.d, torch.zeros(0, 256, device="cuda"), ints([0, 0]), z).shape == (0, 256)


@pytest.mark.parametrize("hd", [64, 96, 192, 256])
@pytest.mark.parametrize("x", ["f32", "f16"])
def test_weights_where_scores_are_not_kept(ops, hd, x):
    """Scores of 300 tokens and 16 heads with room for 16384 slots are more than the workspace keeps: the keys are read a second time."""
    rng = np.random.default_rng(hd)
    p = Pair(ops, 2, 2, 16384, hd, 32, fill=rng)
    run_attention(ops, p, rng, [0, 290, 300], [41, 7], 16, x, seq=[1, 0], max_kv=400, weights=True)


def test_attention_of_a_prompt_leaves_a_clear_status(ops):
    """Through the C entry, whose workspace is the caller's: full of ones before, the status word says that every wait completed."""
    import ctypes as C
    from powerinfer_b200 import _lib
    rng = np.random.default_rng(5)
    p = Pair(ops, 1, 2, 1024, 128, 64, fill=rng)
    start, at = ints([0, 100]), ints([900])
    q = dev(rows(rng, 100, 8 * 128))
    out = torch.empty_like(q)
    b = _lib.KvBatch(start.data_ptr(), None, at.data_ptr(), 1, 100, 100)
    need = _lib.lib.pi_attention_q8_workspace_bytes(p.d.c, C.byref(b), 8, 1024, 0)
    ws = torch.full((need,), -1, dtype=torch.int8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        assert _lib.lib.pi_attention_q8(p.d.c, C.byref(b), _lib.PI_TYPE_F32, q.data_ptr(), 1024, 8, 1024, 128 ** -0.5, out.data_ptr(), 1024, None, None,
                                        ws.data_ptr(), need, stream) == 0
        assert _lib.lib.pi_op_status(ws.data_ptr(), stream) == 0
    assert torch.equal(out, ops.attention_q8(p.d, q, start, at))


def test_rows_of_heads_and_rows_that_lie_oddly(ops):
    """Three dimensions, a single row of a wider matrix, rows that are no multiple of 16 bytes apart: the same results as contiguous rows."""
    rng = np.random.default_rng(6)
    p = Pair(ops, 2, 2, 64, 64, 16, fill=rng)
    start, at = ints([0, 1, 3]), ints([20, 40])
    q = dev(rows(rng, 3, 4 * 64))
    plain = ops.attention_q8(p.d, q, start, at)
    assert torch.equal(ops.attention_q8(p.d, q.view(3, 4, 64), start, at), plain)
    odd = torch.zeros(3, 4 * 64 + 1, device="cuda")
    odd[:, 1:] = q
    assert torch.equal(ops.attention_q8(p.d, odd[:, 1:], start, at), plain)
    assert torch.equal(ops.attention_q8(p.d, q.t().contiguous().t(), start, at), plain)
    one = ops.attention_q8(p.d, q[:1], ints([0, 1]), ints([20]))
    assert torch.equal(ops.attention_q8(p.d, odd[:1, 1:], ints([0, 1]), ints([20])), one)
    f = ops.rope_freqs(64)
    yq, _ = ops.rope_ext(q, None, ints([5, 6, 7]), f, 64)
    assert torch.equal(ops.rope_ext(odd[:, 1:], None, ints([5, 6, 7]), f, 64)[0], yq)
    assert torch.equal(ops.rope_ext(q.view(3, 4, 64), None, ints([5, 6, 7]), f, 64)[0], yq)
    k, v = q[:, :128], q[:, 128:]
    ops.kv_store_q8(p.d, k.reshape(3, 2, 64), odd[:, 129:], start, at)
    p.c.store(k.cpu().numpy(), v.cpu().numpy(), [0, 1, 3], [20, 40])
    p.same()


# ------------------------------------------------------------------------------------------------ eviction

def run_evict(ops, p, w, lens, keep, n_sink, n_recent, seq=None, in_place=False):
    w_dev, w_want = dev(w), w.copy()
    w_out = w_dev if in_place else torch.full(w.shape, -3.0, device="cuda")
    if not in_place:
        w_want[:] = -3.0
    kept = ops.kv_evict_q8(p.d, w_dev, ints(lens), keep, n_sink, n_recent, None if seq is None else ints(seq), w_out)
    want = p.c.evict(w, lens, keep, n_sink, n_recent, seq, w_want)
    assert np.array_equal(kept.cpu().numpy(), want)
    p.same()
    assert np.array_equal(w_out.cpu().numpy(), w_want, equal_nan=True)
    return kept


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("hd,block,n_ctx,keep,lens,sink,recent", [
    (64, 16, 256, 16, [256, 17, 16, 0], 0, 0), (128, 64, 1024, 128, [1000, 129, 1024, 500], 4, 60), (96, 32, 512, 480, [512, 481, 100, 490], 1, 479),
    (192, 128, 2048, 1024, [2048, 1500, 1025, 1024], 4, 256), (256, 16, 128, 48, [128, 64, 49, 1], 48, 0), (128, 16, 4096, 32, [4096, 33, 4000, 77], 3, 29)])
def test_evict_keeps_the_heaviest(ops, in_place, hd, block, n_ctx, keep, lens, sink, recent):
    rng = np.random.default_rng(hd + keep)
    p = Pair(ops, 5, 3, n_ctx, hd, block, fill=rng)
    w = np.exp(rng.standard_normal((5, 3, n_ctx)) * 2).astype(np.float32)
    run_evict(ops, p, w, lens, keep, sink, recent, seq=[3, 0, 4, 1], in_place=in_place)


def test_evict_ties_zeros_and_what_is_not_finite(ops):
    rng = np.random.default_rng(12)
    p = Pair(ops, 6, 2, 512, 64, 32, fill=rng)
    w = np.zeros((6, 2, 512), np.float32)
    w[0] = rng.integers(0, 3, (2, 512))                                # many equal ones
    w[1] = -0.0                                                        # all equal, zeros of both signs
    w[1, :, ::3] = 0.0
    w[2] = rng.standard_normal((2, 512))                               # below zero too
    w[3] = rng.random((2, 512))
    w[3, :, 100:140], w[3, :, 200] = np.inf, -np.inf
    w[4] = rng.random((2, 512)) * np.float32(1e-41)                    # below the normal numbers
    w[5] = np.float32(3.0)
    for keep in (32, 256):
        run_evict(ops, p, w, [512, 511, 400, 512, 257, 300], keep, 2, 9)
    w[3, :, 50:60] = np.nan                                            # above all others
    run_evict(ops, p, w, [512] * 6, 64, 0, 0)


def test_evict_scales(ops):
    """Blocks take the largest of their rows' scales; zeros and equal scales."""
    rng = np.random.default_rng(13)
    p = Pair(ops, 3, 2, 256, 64, 16, fill=rng)
    p.c.scale["k"][0], p.c.scale["v"][0, :, 1::2] = 0, 0
    p.c.scale["k"][1], p.c.scale["v"][1] = 0.25, np.logspace(-20, 20, 16, dtype=np.float32)
    p.d.k_scale.copy_(dev(p.c.scale["k"]))
    p.d.v_scale.copy_(dev(p.c.scale["v"]))
    run_evict(ops, p, rng.random((3, 2, 256), dtype=np.float32), [256, 256, 200], 64, 4, 16)


def test_evict_entries_that_do_not_count(ops):
    rng = np.random.default_rng(14)
    p = Pair(ops, 3, 1, 128, 64, 16, fill=rng)
    w = rng.random((3, 1, 128), dtype=np.float32)
    run_evict(ops, p, w, [128, 100, 128, 90, 500], 32, 1, 1, seq=[1, 5, 1, -1, 0])             # twice, not there, longer than the cache
    run_evict(ops, p, w, [-5], 32, 1, 1, seq=[2])


def test_evict_long_sequences(ops):
    """More weights than shared memory holds."""
    rng = np.random.default_rng(15)
    n_ctx, keep = 70000 // 128 * 128, 1024
    w = np.exp(rng.standard_normal((1, 2, n_ctx)) * 2).astype(np.float32)
    w[0, 1] = np.round(w[0, 1])
    cache = ops.KvCacheQ8.empty(1, n_ctx, 2, 64, 128)
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(1.0)
    cache.k[..., 0] = (torch.arange(n_ctx, device="cuda") % 251 - 125).to(torch.int8)
    first = cache.k.clone()
    kept = ops.kv_evict_q8(cache, dev(w), ints([n_ctx - 5]), keep, 4, 100).cpu().numpy()
    for h in range(2):
        rank = w[0, h, :n_ctx - 5].astype(np.float64)
        rank[:4] = rank[-100:] = np.inf
        best = np.sort(np.lexsort((np.arange(len(rank)), -rank))[:keep])
        assert np.array_equal(np.sort(kept[0, h]), best)
        stays = kept[0, h] < keep
        assert np.array_equal(kept[0, h][stays], np.flatnonzero(stays)) and np.all(np.diff(kept[0, h][~stays]) > 0)
        assert torch.equal(cache.k[0, h, :keep], first[0, h, torch.from_numpy(kept[0, h]).long().cuda()])
    assert torch.equal(cache.k[:, :, keep:], first[:, :, keep:])


# ------------------------------------------------------------------------------------------------ streams, graphs, a run of all

def test_calls_on_two_streams_and_in_graphs(ops):
    """Two streams at once, and two graphs of the same call replayed in turn with other lengths: no scratch is shared, lengths are read on the device."""
    rng = np.random.default_rng(31)
    n_ctx, hd, H = 4096, 128, 2
    p = Pair(ops, 2, H, n_ctx, hd, 64, fill=rng)
    w_in = torch.rand(2, H, n_ctx, device="cuda")
    qs = [dev(rows(rng, 2, 8 * hd)) for _ in range(2)]
    start, pos = ints([0, 1, 2]), [ints([4000, 900]), ints([100, 4095])]
    plain = [[], []]
    for i in range(2):
        for at in pos:
            w = torch.zeros_like(w_in)
            plain[i].append((ops.attention_q8(p.d, qs[i], start, at, max_new=1, weights_in=w_in, weights_out=w), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for rep in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                w = torch.zeros_like(w_in)
                got.append((i, rep % 2, ops.attention_q8(p.d, qs[i], start, pos[rep % 2], max_new=1, weights_in=w_in, weights_out=w), w))
    torch.cuda.synchronize()
    for i, at, out, w in got:
        assert torch.equal(out, plain[i][at][0]) and torch.equal(w, plain[i][at][1])
    here, graphs, results = pos[0].clone(), [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        w = torch.zeros_like(w_in)
        with torch.cuda.graph(g):
            out = ops.attention_q8(p.d, qs[i], start, here, max_new=1, weights_in=w_in, weights_out=w)
        graphs.append(g)
        results.append((out, w))
    for at in (0, 1, 0, 1):
        here.copy_(pos[at])
        for (out, w) in results:
            w.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(results[i][0], plain[i][at][0]) and torch.equal(results[i][1], plain[i][at][1])


def test_a_step_as_a_graph_on_another_stream(ops):
    """Rotation, store, attention of a prompt and of single tokens, eviction and read-back as one captured step, replayed with other lengths and rows on a
    stream of its own: the same bits as the calls one by one."""
    rng = np.random.default_rng(32)
    H, group, hd, n_ctx, T = 2, 4, 64, 512, 42
    names = ("k", "v", "k_scale", "v_scale")
    a, b = (Pair(ops, 3, H, n_ctx, hd, 16) for _ in range(2))
    f = ops.rope_freqs(hd)
    step = [torch.empty(T, (H * group + 2 * H) * hd, device="cuda"), ints([0] * T), ints([0, 40, 41, 42]), ints([0] * 3), ints([0] * 3)]
    weights = [torch.zeros(3, H, n_ctx, device="cuda") for _ in range(2)]

    def run(c, w):
        qkv, pos, start, at, lens = step
        q, k = ops.rope_ext(qkv[:, :H * group * hd], qkv[:, H * group * hd:H * (group + 1) * hd], pos, f, hd)
        ops.kv_store_q8(c, k, qkv[:, H * (group + 1) * hd:], start, at, max_new=40)
        out = ops.attention_q8(c, q, start, at, max_new=40, weights_in=w, weights_out=w)
        kept = ops.kv_evict_q8(c, w, lens, 128, 2, 16, weights_out=w)
        return (out, kept) + tuple(ops.kv_load_q8(c, start, ints_of_graph, T, max_new=40))

    ints_of_graph = ints([3, 0, 100])
    side = torch.cuda.Stream()
    step[0].copy_(dev(rows(rng, T, step[0].shape[1])))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = run(a.d, weights[0])
    for at in ([0, 7, 200], [40, 8, 201], [80, 9, 128], [120, 511, 128], [128, 128, 128]):
        step[0].copy_(dev(rows(rng, T, step[0].shape[1])))
        step[1].copy_(ints([at[0] + i for i in range(40)] + at[1:]))
        step[3].copy_(ints(at))
        step[4].copy_(ints([at[0] + 40, min(at[1] + 1, n_ctx), at[2] + 1]))
        want = run(b.d, weights[1])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for got, w in zip(captured, want):
            assert torch.equal(got, w)
        assert torch.equal(*weights)
        for n in names:
            assert torch.equal(getattr(a.d, n), getattr(b.d, n))


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_a_run_of_all_operators(ops, x):
    """Two sequences as a server runs them: prompts in chunks, tokens one by one, weights collected, the cache cut to its budget twice; positions go on
    while slots are reused.  The oracle takes the device's own rotated rows, so that codes are equal."""
    rng = np.random.default_rng(77)
    H, group, hd, block, n_ctx, keep, sink, recent = 2, 4, 64, 16, 128, 64, 2, 16
    p = Pair(ops, 2, H, n_ctx, hd, block)
    f = ops.rope_freqs(32, freq_scale=0.25, ext_factor=1.0, n_orig_ctx=64)
    w = torch.zeros(2, H, n_ctx, device="cuda")
    pos, slots = [0, 0], [0, 0]
    for step, news in enumerate([(40, 7), (23, 50), (1, 1), (40, 40), (1, 1), (1, 1), (60, 1), (1, 1)]):
        start = [0, news[0], news[0] + news[1]]
        qkv = dev(rows(rng, start[-1], (H * group + 2 * H) * hd, x))
        at = ints([pos[0] + i for i in range(news[0])] + [pos[1] + i for i in range(news[1])])
        q, k = ops.rope_ext(qkv[:, :H * group * hd], qkv[:, H * group * hd:H * (group + 1) * hd], at, f, hd, mode=2)
        if slots[0] + news[0] > n_ctx or slots[1] + news[1] > n_ctx:
            w_host = w.cpu().numpy()
            kept = ops.kv_evict_q8(p.d, w, ints(slots), keep, sink, recent, weights_out=w)
            want = p.c.evict(w_host, slots, keep, sink, recent, None, w_host)
            assert np.array_equal(kept.cpu().numpy(), want) and np.array_equal(w.cpu().numpy(), w_host)
            p.same()
            slots = [min(s, keep) for s in slots]
        k_host, v_host = k.cpu().numpy(), qkv[:, H * (group + 1) * hd:].cpu().numpy()
        ops.kv_store_q8(p.d, k, qkv[:, H * (group + 1) * hd:], ints(start), ints(slots))
        p.c.store(k_host, v_host, start, slots)
        p.same()
        w_in, w_want = w.cpu().numpy(), w.cpu().numpy().astype(np.float64)
        got = ops.attention_q8(p.d, q, ints(start), ints(slots), max_new=max(news), weights_in=w, weights_out=w)
        want, err, terms, most = p.c.attention(q.cpu().numpy(), H * group, hd ** -0.5, start, slots, w_in=w_in, w_out=w_want)
        assert np.all(np.abs(got.float().cpu().numpy() - want) <= attention_bound(err, terms, most, hd, n_ctx, x, want))
        wt = (np.abs(w_want) + 1) * (2 * terms.max() * (hd + 10) * 2 + 4 * n_ctx + 4 * 60 * group + 16) * U["f32"]
        assert np.all(np.abs(w.cpu().numpy() - w_want) <= wt)
        pos, slots = [pos[0] + news[0], pos[1] + news[1]], [slots[0] + news[0], slots[1] + news[1]]
