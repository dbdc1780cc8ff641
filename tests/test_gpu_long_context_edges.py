"""Calls of the long-context operators that their documentation allows and where they went wrong once, against long_context_oracle or against a call that has to give
the same bits.  Half a step is u = 2^-24 in FP32, 2^-11 in FP16."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_long_context import NP, Pair, U, dev, ints, ops, rows, run_attention, run_evict  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------------------------------ what a row does not see

@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("T,pos0,block", [(3, 95, 6), (140, 101, 14)])
@pytest.mark.parametrize("own,late", [(1.0, 1e12), (2.0 ** -20, 2.0 ** 120), (2.0 ** -20, np.inf), (1.0, np.nan)])
def test_rows_do_not_see_scales_of_later_tokens(ops, x, hd, T, pos0, block, own, late):
    """A block whose scales only the last tokens of a chunk see: the bits of the earlier tokens are those of a cache where that block is ordinary."""
    rng = np.random.default_rng(hd + T)
    p = Pair(ops, 1, 2, 512, hd, 16, fill=rng)
    p.c.scale["v"] *= np.float32(own)
    q = dev(rows(rng, T, 8 * hd, x))
    got = []
    for s in (None, late):
        for n in "kv":
            if s is not None:
                p.c.scale[n][0, :, block] = s
        p.d.k_scale.copy_(dev(p.c.scale["k"]))
        p.d.v_scale.copy_(dev(p.c.scale["v"]))
        got.append(ops.attention_q8(p.d, q, ints([0, T]), ints([pos0])))
    earlier = block * 16 - pos0                                        # tokens that do not see the block
    assert 0 < earlier < T and torch.isfinite(got[0]).all() and (got[0] != 0).any()
    assert torch.equal(got[0][:earlier], got[1][:earlier])
    assert not torch.equal(got[0][earlier:], got[1][earlier:])


def test_prompt_rows_against_64_bits_beside_a_large_later_scale(ops):
    rng = np.random.default_rng(41)
    for hd in (64, 128):
        p = Pair(ops, 1, 2, 512, hd, 16, fill=rng)
        p.c.scale["v"][0, :, 14] = 1e12
        p.d.v_scale.copy_(dev(p.c.scale["v"]))
        run_attention(ops, p, rng, [0, 140], [100], 8)


# ------------------------------------------------------------------------------------------------ queries with one large element

def check_large(ops, p, q, start, pos, n_head, x, max_kv=None):
    """Up to 8 rows a KV head, and any number with head_dim above 128 or where the weights' kernel reads the keys again: a query is whole numbers of which the
    row's largest is 2^30 x 0.99 or more.  A value is off by 2^-30.9 of it at most, products with codes and their sums are exact.  Four sums become one number in FP32
    steps (a sum is 2^22 at most: u of 2^30 each beside u of the score), then come two factors, the product and the difference in the exponent:
        e_s = scale (2^-30.9 max |q| max_j sum_d |k_jd| + 2 u max |q| max_j s_j) + 10 u max_j |s_j|.
    9 to 63 rows: FP16 as they are; FP32 as two halves, off by 2^-22 of the value or 2^-35 of the row's largest; sums are cut, 2 hd u of their terms' sizes at most:
        e_s = scale max_j sum_d |q_d k_jd| (2^-22 + (2 hd + 10) u) + scale 2^-35 max |q| max_j sum_d |k_jd|.
    The rest as in test_gpu_long_context.  Weights are sums of probabilities: 2 e_s + (4 n + 16) u of each, and u for each addition."""
    T, hd, H, group = len(q), p.c.hd, p.c.H, n_head // p.c.H
    scale, u = hd ** -0.5, U["f32"]
    shape = (p.c.n_seq, H, p.c.n_ctx)
    w_got, w_want = torch.zeros(shape, device="cuda"), np.zeros(shape)
    got = ops.attention_q8(p.d, dev(q), ints(start), ints(pos), max_kv=max_kv, weights_out=w_got).float().cpu().numpy().astype(np.float64)
    want, size, _, most = p.c.attention(q, n_head, scale, start, pos, w_out=w_want)
    heads = q.astype(np.float64).reshape(T, n_head, hd)
    e_s, n_max = np.zeros((T, n_head)), 1
    for i, first, n, at, sq in p.c.entries(start, pos, None, T, T):
        end = min(at + n, p.c.n_ctx)
        n_max = max(n_max, end)
        for h in range(H):
            k = p.c.values("k", sq, h, end)
            hs = slice(h * group, (h + 1) * group)
            big = np.abs(heads[first:first + n, hs]).max(-1)
            top = np.abs(np.einsum("tgd,jd->tgj", heads[first:first + n, hs], k)).max(-1)
            sums = np.abs(k).sum(-1).max()
            terms = np.einsum("tgd,jd->tgj", np.abs(heads[first:first + n, hs]), np.abs(k)).max(-1)
            whole = scale * (big * (2.0 ** -30.9 * sums + 2 * u * p.c.scale["k"][sq, h].max()) + 10 * u * top)
            halves = scale * (terms * ((2.0 ** -22 if x == "f32" else 0.0) + (2 * hd + 10) * u) + 2.0 ** -35 * big * sums)
            e_s[first:first + n, hs] = halves if 8 < T * group < 64 and hd <= 128 else whole
    rel = 2 * e_s + (4 * n_max + 16) * u
    tol = (size.reshape(T, n_head, hd) * rel[..., None] + 2.0 ** -32 * most[..., None]).reshape(T, -1) + 1e-30
    if x == "f16":
        tol = tol + U["f16"] * (np.abs(want) + tol) + 2.0 ** -25
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    wt = w_want * (rel.max() + (T * group + 2) * u) + 1e-30
    off = np.abs(w_got.cpu().numpy() - w_want)
    assert np.all(off <= wt), float((off / wt).max())


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("group", [4, 16])
@pytest.mark.parametrize("large", [30.0, 3000.0])
def test_queries_with_one_large_element(ops, x, hd, group, large):
    """A channel that is large in the queries and nothing in the keys: the other elements keep their bits."""
    rng = np.random.default_rng(hd + group)
    p = Pair(ops, 2, 2, 64, hd, 16, fill=rng)
    p.c.codes["k"][..., 5] = 0
    p.d.k.copy_(dev(p.c.codes["k"]))
    q = rng.standard_normal((2, 2 * group, hd)).astype(np.float32)
    q[..., 5] = np.sign(q[..., 5]) * large
    check_large(ops, p, q.reshape(2, -1).astype(NP[x]), [0, 1, 2], [50, 63], 2 * group, x)


@pytest.mark.parametrize("hd", [96, 256])
def test_weights_of_queries_with_one_large_element(ops, hd):
    """Where the keys are read a second time for the weights."""
    rng = np.random.default_rng(hd)
    p = Pair(ops, 1, 1, 16384, hd, 32, fill=rng)
    p.c.codes["k"][..., 5] = 0
    p.d.k.copy_(dev(p.c.codes["k"]))
    T, n_head = 290, 16
    q = rng.standard_normal((T, n_head, hd)).astype(np.float32)
    q[..., 5] = np.sign(q[..., 5]) * 3000
    check_large(ops, p, q.reshape(T, -1), [0, T], [41], n_head, "f32", max_kv=400)


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("T", [1, 3, 140])
@pytest.mark.parametrize("sign", [-1, 1])
def test_infinite_queries_against_keys_of_one_sign(ops, x, hd, T, sign):
    """Scores that are all minus infinity are no mask: their row has no numbers, as a row of plus infinities has."""
    rng = np.random.default_rng(hd + T)
    p = Pair(ops, 1, 2, 256, hd, 16, fill=rng)
    p.c.codes["k"][..., 5] = rng.integers(1, 100, p.c.codes["k"].shape[:-1])
    p.d.k.copy_(dev(p.c.codes["k"]))
    q = rows(rng, T, 8 * hd, x)
    clean = ops.attention_q8(p.d, dev(q), ints([0, T]), ints([40]))
    q[T // 2, 3 * hd + 5] = sign * np.inf
    got = ops.attention_q8(p.d, dev(q), ints([0, T]), ints([40]))
    hurt = torch.zeros_like(got, dtype=torch.bool)
    hurt[T // 2, 3 * hd:4 * hd] = True
    assert torch.isnan(got[hurt]).all() and torch.equal(got[~hurt], clean[~hurt])


# ------------------------------------------------------------------------------------------------ status of a call

@pytest.mark.parametrize("hd,T,n_head,n_ctx,weights", [(128, 1, 16, 16384, False), (128, 1, 16, 256, True), (96, 100, 8, 512, True), (192, 3, 4, 16384, False), (64, 1, 4, 64, False),
                                                       (128, 100, 8, 1024, False)])
def test_status_after_any_call(ops, hd, T, n_head, n_ctx, weights):
    """pi_op_status of a workspace that held anything before: the call's, whichever kernels it took and whether it needed the workspace."""
    from powerinfer_b200 import _lib
    rng = np.random.default_rng(5)
    p = Pair(ops, 1, 2, n_ctx, hd, 64, fill=rng)
    start, at = ints([0, T]), ints([n_ctx - T - 3])
    q = dev(rows(rng, T, n_head * hd))
    out, w = torch.empty_like(q), torch.zeros(1, 2, n_ctx, device="cuda")
    b = _lib.KvBatch(start.data_ptr(), None, at.data_ptr(), 1, T, T)
    need = _lib.lib.pi_attention_q8_workspace_bytes(p.d.c, C.byref(b), n_head, n_ctx, int(weights))
    ws = torch.full((max(need, 256),), -1, dtype=torch.int8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        assert _lib.lib.pi_attention_q8(p.d.c, C.byref(b), _lib.PI_TYPE_F32, q.data_ptr(), n_head * hd, n_head, n_ctx, hd ** -0.5, out.data_ptr(), n_head * hd, None,
                                        w.data_ptr() if weights else None, ws.data_ptr(), ws.numel(), stream) == 0
        assert _lib.lib.pi_op_status(ws.data_ptr(), stream) == 0
    assert torch.equal(out, ops.attention_q8(p.d, q, start, at, weights_out=torch.zeros_like(w) if weights else None))


def test_last_op_status_is_that_of_the_attention(ops):
    """The status word that last_op_status reads is the last operator's: of a prompt's attention, then of another operator."""
    rng = np.random.default_rng(6)
    p = Pair(ops, 1, 2, 1024, 128, 64, fill=rng)
    x = torch.randn(2, 256, device="cuda")
    w = ops.upload_weight(rng.standard_normal((64, 256)).astype(np.float16), ops.PI_TYPE_F16, 64, 256)
    ops.ggml_mul_mat(w, x)
    assert ops.last_op_status() == 0
    q = dev(rows(rng, 100, 8 * 128))
    ops.attention_q8(p.d, q, ints([0, 100]), ints([900]))
    assert ops.last_op_status() == 0
    ops._ws.asked[1][8:12] = torch.tensor([16, 0, 0, 0], dtype=torch.int8, device="cuda")     # as if a wait had run out
    assert ops.last_op_status() == 5
    ops.attention_q8(p.d, q[:1], ints([0, 1]), ints([30]), max_kv=64)
    assert ops.last_op_status() == 0
    ops.attention_q8(p.d, q, ints([0, 100]), ints([900]))
    ops.ggml_mul_mat(w, x)
    assert ops.last_op_status() == 0


# ------------------------------------------------------------------------------------------------ batches

def test_ends_far_below_zero_are_no_tokens(ops):
    """An end so far below its start that the difference does not fit 32 bits."""
    rng = np.random.default_rng(7)
    p = Pair(ops, 2, 2, 128, 64, 16, fill=rng)
    k = rows(rng, 8, 128)
    for end in (-2 ** 31, -2 ** 31 + 4, -1):
        p.store(k, k, [5, end], [0])
        p.same()
        run_attention(ops, p, rng, [5, end], [20], 4, T=8)


# ------------------------------------------------------------------------------------------------ sizes that the other tests do not reach

@pytest.mark.parametrize("in_place", [False, True])
def test_evict_with_more_places_than_the_list_holds(ops, in_place):
    """A budget above 16384 slots: the holes are listed in several turns."""
    rng = np.random.default_rng(15)
    p = Pair(ops, 1, 2, 53248, 64, 128, fill=rng)
    w = np.exp(rng.standard_normal((1, 2, 53248)) * 2).astype(np.float32)
    w[0, 1, :40960] = 0                                                # every place but the first ones and the last ones is a hole
    run_evict(ops, p, w, [53240], 40960, 4, 100, in_place=in_place)


@pytest.mark.parametrize("hd,x", [(64, "f16"), (128, "f32")])
def test_prompt_over_many_parts(ops, hd, x):
    """Few tiles of 128 rows over a long range: more than 8 parts of each are joined."""
    rng = np.random.default_rng(hd)
    p = Pair(ops, 1, 1, 16384, hd, 64, fill=rng)
    run_attention(ops, p, rng, [0, 20], [15990], 8, x)


def test_codes_of_minus_128(ops):
    """The store makes codes of +-127, a caller's own cache may hold -128."""
    rng = np.random.default_rng(18)
    for T, hd in ((1, 128), (3, 96), (140, 64), (140, 128)):
        p = Pair(ops, 1, 2, 256, hd, 16, fill=rng)
        for n, codes in (("k", p.d.k), ("v", p.d.v)):
            p.c.codes[n][rng.random(p.c.codes[n].shape) < 0.3] = -128
            codes.copy_(dev(p.c.codes[n]))
        run_attention(ops, p, rng, [0, T], [100], 8, weights=True)
    run_evict(ops, p, rng.random((1, 2, 256), dtype=np.float32), [256], 64, 2, 9)


@pytest.mark.parametrize("max_kv", [1024, 1000, 300])
def test_weights_of_chunks_of_wide_heads(ops, max_kv):
    """64 rows a KV head of 256 dimensions: scores kept (keys of 16 MB and more are expected), and keys read a second time."""
    rng = np.random.default_rng(21)
    p = Pair(ops, 8, 8, 1024, 256, 64, fill=rng)
    lens = [8, 3, 8, 1, 8, 8, 0, 5]
    start = np.concatenate([[0], np.cumsum(lens)]).tolist()
    run_attention(ops, p, rng, start, [1016, 0, 500, 1023, 1020, 7, 5, 300], 64, seq=[3, 1, 0, 7, 2, 6, 5, 4], max_new=8, max_kv=max_kv, weights=True)


# ------------------------------------------------------------------------------------------------ recent tokens

def test_recent_tokens_stay_where_as_many_slots_go_at_a_time(ops):
    """Evictions of n_recent slots and more keep the n_recent newest tokens, whatever their weights are; what moved has left the end."""
    rng = np.random.default_rng(19)
    keep, recent, n_ctx = 64, 24, 128
    cache = ops.KvCacheQ8.empty(1, n_ctx, 2, 64, 16)
    token = [np.arange(keep) for _ in range(2)]                        # which token a slot holds, for each head
    n = keep
    for more in (24, 40, 24, 64, 30):
        token = [np.concatenate([t, np.arange(n, n + more)]) for t in token]
        n += more
        w = rng.random((1, 2, n_ctx), dtype=np.float32)
        w[:, :, -(n_ctx - keep):] = 0                                  # the new tokens have collected nothing yet
        kept = ops.kv_evict_q8(cache, dev(w), ints([keep + more]), keep, 2, recent).cpu().numpy()
        token = [t[kept[0, h]] for h, t in enumerate(token)]
        for t in token:
            assert set(range(n - recent, n)) <= set(t.tolist())
