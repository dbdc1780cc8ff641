"""Drafted tokens over a paged cache against plain forms in 64 bits (paged_oracle): trees, keys and values into pages with their rotation, attention by
masks, the path that stays, and steps of all of them together.

Tolerances.  Half a step is u = 2^-24 in FP32 and 2^-11 in FP16.
  trees, keep  whole numbers and copies: equal.
  append     cosine and sine: 2 u from the reduced angle and its function, u from the factor; two products and a sum: 3 u of |x0| + |x1|.  With a margin of one third
             8 u (|x0| + |x1|) mscale; keys, values and FP16 queries have their own rounding, 2^-11 of the result, or 2^-25.
  attention  a query is held to 2^-22 of its row's largest value (FP16: as it is), sums of hd products are off by at most hd u, the factor of the scores by 3 u: with
             E = scale * max_j sum_d |q_d k_jd| a score is off by at most E (2^-22 + (hd + 3) u), and as E log2(e) is the largest size of an exponent its rounding by
             2 E u: e_s = E (hd + 10) u in all.  A probability is then off by 2 e_s of itself, 4 u from exp2 (2 ulp), 4 u from its two halves (FP16: 2^-11, one half), both sums by
             n u at most, twice that as sums on the tensor cores are cut: an output by at most sum_j p_j |v_j| (2 e_s + (2 n + 16) u [+ 2^-11]) and
             its own rounding.  A probability has no steps below 2^-24 of what it is held times, 2^8, beside a largest one of 1 or more: 2^-32 of each value over the sum is left out.
"""
import numpy as np
import pytest

import paged_oracle as po

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
NP = {"f32": np.float32, "f16": np.float16}
TY = {"f32": torch.float32, "f16": torch.float16}


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


def pool(rng, n_layer, H, hd, page, lens, spare=2, holes=()):
    """Pools of normal values, a table that hands out pages in no order for sequences of lens slots; holes: (sequence, block) without a page."""
    blocks = [-(-n // page) for n in lens]
    n_pages = sum(blocks) + spare
    k, v = (rng.standard_normal((n_layer, n_pages, H, page, hd), dtype=np.float32).astype(np.float16) for _ in range(2))
    table = np.full((len(lens), max(blocks + [1])), -1, np.int32)
    free = list(rng.permutation(n_pages))
    for i, b in enumerate(blocks):
        for j in range(b):
            table[i, j] = free.pop()
    for i, j in holes:
        table[i, j] = rng.choice([-1, n_pages, 1 << 30])
    return po.Cache(k, v, table)


def on(ops, c):
    return ops.KvCachePaged(dev(c.k), dev(c.v), dev(c.table))


def trees(rng, news, wide=1 << 30):
    return sum(([-1] + [int(rng.integers(max(0, u - wide), u)) for u in range(1, m)] if m else [] for m in news), [])


def starts(news, first=0):
    return [first + sum(news[:i]) for i in range(len(news) + 1)]


def words_of(masks, words):
    out = np.zeros((len(masks), words), np.int64)
    for t, m in enumerate(masks):
        for w in range(words):
            x = (m or 0) >> 64 * w & (1 << 64) - 1
            out[t, w] = x - (1 << 64) if x >> 63 else x
    return out


# ------------------------------------------------------------------------------------------------ trees

@pytest.mark.parametrize("news,wide", [([1], 9), ([25], 9), ([64, 65, 1, 0, 63], 1 << 30), ([129, 2, 300], 4), ([128, 127], 1), ([192] * 5, 1 << 30), ([700, 33], 1), ([4096], 1), ([4095, 1], 50)])
def test_tree_mask(ops, news, wide):
    rng = np.random.default_rng(sum(news) + wide % 97)
    parents, pos0 = trees(rng, news, wide), [int(rng.integers(0, 100000)) for _ in news]
    words = -(-max(news) // 64)
    mask, pos = ops.tree_mask(ints(parents), ints(starts(news)), ints(pos0), max_new=max(news))
    want, want_pos = po.tree_mask(parents, starts(news), pos0, max(news), words)
    assert mask.shape == (sum(news), words) and [po.mask_int(r) for r in mask.cpu().numpy()] == want
    assert pos.cpu().tolist() == want_pos


def test_tree_mask_of_odd_numbers(ops):
    """Parents that are no earlier token, fewer words than tokens, fewer tokens than rows, rows of no entry, entries that do not fit."""
    rng = np.random.default_rng(5)
    T, q_start = 200, [3, 90, 90, 150, 120, 260]
    parents = [int(x) for x in rng.integers(-5, 90, T)]
    for max_new, words in ((100, 2), (100, 1), (70, 2), (200, 4)):
        mask, pos = ops.tree_mask(ints(parents), ints(q_start), ints([7, -3, 0, 9, 2 ** 30]), max_new=max_new, words=words)
        want, want_pos = po.tree_mask(parents, q_start, [7, -3, 0, 9, 2 ** 30], max_new, words)
        got, got_pos = mask.cpu().numpy(), pos.cpu().tolist()
        for t in range(T):
            if want[t] is not None and not (120 <= t < 150):          # (rows of two entries hold either's)
                assert po.mask_int(got[t]) == want[t] and got_pos[t] == want_pos[t], t


@pytest.mark.parametrize("news,vocab", [([1], 3), ([25], 2), ([64, 1, 0, 65], 2), ([192] * 7, 3), ([1000, 30], 1), ([4096], 2)])
def test_tree_accept(ops, news, vocab):
    """A vocabulary of few tokens: siblings are often the same one, and paths long."""
    rng = np.random.default_rng(len(news) + vocab)
    parents, T = trees(rng, news, 3 if vocab == 1 else 1 << 30), sum(news)
    parents = [p if rng.random() < 0.97 else int(rng.integers(-3, 5000)) for p in parents]
    tokens, choice = rng.integers(0, vocab, T).tolist(), rng.integers(0, vocab, T).tolist()
    path, n_path, then = ops.tree_accept(ints(tokens), ints(parents), ints(choice), ints(starts(news)), max_new=max(news))
    want, want_then = po.tree_accept(tokens, parents, choice, starts(news), max(news))
    assert [r[:n] for r, n in zip(path.cpu().tolist(), n_path.cpu().tolist())] == want and then.cpu().tolist() == want_then
    assert all(x == -1 for r, n in zip(path.cpu().tolist(), n_path.cpu().tolist()) for x in r[n:])


def test_no_trees(ops):
    """No entries, entries without tokens, no rows at all, no room for a path."""
    none, z = ints([]), ints([0])
    mask, pos = ops.tree_mask(none, z, none)
    assert mask.shape == (0, 1) and pos.shape == (0,)
    mask, pos = ops.tree_mask(none, ints([0, 0, 0]), ints([5, 6]), max_new=70)
    assert mask.shape == (0, 2)
    for T, most in ((0, 0), (0, 3), (4, 0), (4, 3)):
        t = ints([1] * T)
        path, n_path, then = ops.tree_accept(t, t, t, ints([0, 0, 0, 0]), max_new=most)
        assert path.shape == (3, most) and n_path.tolist() == [0] * 3 and then.tolist() == [-1] * 3 and path.eq(-1).all()


# ------------------------------------------------------------------------------------------------ append

def pair_sums(x, hd, n_rot, halves):
    h = np.abs(x.astype(np.float64)).reshape(x.shape[0], -1, hd)
    pair, half = h.copy(), n_rot // 2
    i0, i1 = (np.arange(half), np.arange(half) + half) if halves else (np.arange(half) * 2, np.arange(half) * 2 + 1)
    pair[..., i0] = pair[..., i1] = h[..., i0] + h[..., i1]
    return pair


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("news,lens,H,group,hd,n_rot,page,far", [
    ([1], [1], 2, 2, 64, 64, 16, 0), ([1] * 5, [40, 1, 17, 16, 64], 8, 8, 128, 128, 64, 0), ([25, 7, 0, 1], [300, 40, 16, 33], 1, 7, 96, 96, 32, 100000),
    ([130], [200], 5, 1, 192, 42, 128, 1000000), ([3, 64], [90, 64], 2, 3, 256, 256, 16, 5), ([17, 2], [17, 100], 4, 2, 64, 2, 16, 70), ([9], [9], 3, 1, 128, 96, 64, 2000000),
    ([700, 77, 1, 133], [900, 80, 100, 133], 8, 8, 64, 64, 16, 0), ([701, 9], [701, 64], 4, 4, 96, 40, 32, 3000), ([211, 214], [300, 214], 8, 7, 128, 128, 64, 5000)])        # (several tokens a CTA)
def test_append(ops, x, halves, news, lens, H, group, hd, n_rot, page, far):
    rng = np.random.default_rng(hd + sum(news) + n_rot)
    n, T, layer = len(news), sum(news), 1
    c = pool(rng, 3, H, hd, page, lens)
    order = rng.permutation(n)                                        # of the sequences in the table
    c.table = c.table[np.argsort(order)]
    q_start, pos0, seq = starts(news), [a - b for a, b in zip(lens, news)], [int(i) for i in order]
    pos = None if far == 0 else rng.integers(0, far + 1, T)
    f = ops.rope_freqs(n_rot, freq_scale=0.25, ext_factor=1.0, n_orig_ctx=2048)
    fh = f.freqs.cpu().numpy()
    nq, nk = H * group * hd, H * hd
    qkv = rows(rng, T, nq + 2 * nk, x)
    there, one = dev(qkv), on(ops, c)
    q = ops.kv_append_paged(one, there[:, nq:nq + nk], there[:, nq + nk:], ints(q_start), ints(pos0), ints(seq), max_new=max(news), q=there[:, :nq],
                            pos=None if pos is None else ints(pos.tolist()), freqs=f, mode=2 if halves else 0, layer=layer)
    kw, vw, wrote = po.append(c, layer, qkv[:, nq:nq + nk], qkv[:, nq + nk:], q_start, pos0, seq, max(news), pos, fh, f.mscale, halves)
    k, v = one.k.cpu().numpy(), one.v.cpu().numpy()
    assert wrote.sum() == T * H
    assert np.array_equal(k[~wrote], c.k[~wrote]) and np.array_equal(v[~wrote], c.v[~wrote])
    assert np.array_equal(v[wrote], vw[wrote].astype(np.float16))     # one rounding
    at = pos if pos is not None else np.concatenate([np.arange(m) + p for m, p in zip(news, pos0)])
    far_pairs = np.zeros_like(kw)
    pairs = pair_sums(qkv[:, nq:nq + nk], hd, n_rot, halves)
    for i in range(n):
        for t in range(news[i]):
            page_, row = c.place(seq[i], pos0[i] + t)
            far_pairs[layer, page_, :, row] = pairs[q_start[i] + t]
    tol = 8 * U["f32"] * far_pairs * f.mscale + U["f16"] * np.abs(kw) + 2.0 ** -25
    assert np.all((np.abs(k - kw) <= tol)[wrote])
    want = po.lc.rope(qkv[:, :nq], at, fh, f.mscale, hd, halves).reshape(T, -1, hd)
    tol = 8 * U["f32"] * pair_sums(qkv[:, :nq], hd, n_rot, halves) * f.mscale + (U[x] * np.abs(want) + 2.0 ** -25 if x == "f16" else 0.0)
    got = q.cpu().numpy().reshape(T, -1, hd)
    assert q.dtype is TY[x] and np.all(np.abs(got.astype(np.float64) - want) <= tol) and np.array_equal(got[..., n_rot:], qkv[:, :nq].reshape(T, -1, hd)[..., n_rot:])
    assert np.array_equal(there.cpu().numpy(), qkv)                   # the inputs are left alone
    # without queries
    two = on(ops, c)
    assert ops.kv_append_paged(two, there[:, nq:nq + nk], there[:, nq + nk:], ints(q_start), ints(pos0), ints(seq), max_new=max(news), pos=None if pos is None else ints(pos.tolist()),
                               freqs=f, mode=2 if halves else 0, layer=layer) is None
    assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v)


def test_append_without_rotation_and_what_the_cache_lacks(ops):
    """Pages that are not there, slots behind the table's end, entries of no sequence, of one sequence twice, without tokens; values that halves do not hold."""
    rng = np.random.default_rng(3)
    c = pool(rng, 1, 2, 64, 16, [64, 64, 40], holes=[(0, 1), (2, 0)])
    news, pos0, seq = [20, 30, 5, 4, 0, 3, 2, 6], [10, 50, 12, 0, 3, -1, 64, 7], [0, 1, 2, 5, 1, 0, 1, 2]
    T = sum(news)
    k, v = rows(rng, T + 2, 128), rows(rng, T + 2, 128) * 1e5         # (infinities as halves)
    v[1, 3], k[2, 0] = np.nan, 1e-9
    q_start = starts(news, 1)
    one = on(ops, c)
    assert ops.kv_append_paged(one, dev(k), dev(v), ints(q_start), ints(pos0), ints(seq), max_new=25) is None
    kw, vw, wrote = po.append(c, 0, k, v, q_start, pos0, seq, 25, None, None, 1.0, False)
    with np.errstate(over="ignore"):
        assert np.array_equal(one.k.cpu().numpy(), kw.astype(np.float16)) and np.array_equal(one.v.cpu().numpy(), vw.astype(np.float16), equal_nan=True)
    assert 0 < wrote.sum() < T * 2


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("news,mode,n_rot", [([3, 2], 0, 64), ([3, 2], 2, 64), ([900, 31], 0, 64), ([900, 31], 2, 64), ([900, 31], 2, 36)])
def test_queries_turned_in_place(ops, x, news, mode, n_rot):
    """q_out may be q where address and stride are the same: the same bits as into another array."""
    from powerinfer_b200._lib import lib
    rng = np.random.default_rng(n_rot + news[0])
    c, T, f = pool(rng, 1, 4, 64, 16, news), sum(news), ops.rope_freqs(n_rot)
    there, one, two = dev(rows(rng, T, (32 + 8) * 64, x)), on(ops, c), on(ops, c)
    q, k, v = there[:, :2048], there[:, 2048:2304], there[:, 2304:]
    q_start, pos0 = ints(starts(news)), ints([0, 0])
    want = ops.kv_append_paged(one, k, v, q_start, pos0, max_new=max(news), q=q, freqs=f, mode=mode)
    b, size, stride = ops._entries(q_start, pos0, None, T, max(news), 0), there.element_size(), there.stride(0)
    assert lib.pi_kv_append_paged(two.c, b, 0, 0 if x == "f32" else 1, k.data_ptr(), stride, v.data_ptr(), stride, q.data_ptr(), stride, 32, q.data_ptr(), stride,
                                  None, f.freqs.data_ptr(), n_rot, 1 if mode else 0, f.mscale, ops._stream()) == 0
    assert size in (2, 4) and torch.equal(q, want) and torch.equal(one.k, two.k) and torch.equal(one.v, two.v)


def test_queries_of_entries_that_are_not_stored_turn_all_the_same(ops):
    c = po.Cache(np.zeros((1, 2, 1, 16, 64), np.float16), np.zeros((1, 2, 1, 16, 64), np.float16), np.array([[0], [-1]], np.int32))
    q, kv, f = torch.randn(4, 128, device="cuda"), torch.randn(4, 64, device="cuda"), ops.rope_freqs(64)
    one, pos = on(ops, c), ints([5, 6, 7, 8])
    got = ops.kv_append_paged(one, kv, kv, ints([0, 1, 2, 4]), ints([0, 0, 15]), ints([0, 7, 0]), max_new=2, q=q, pos=pos, freqs=f)
    want = po.lc.rope(q.cpu().numpy(), [5, 6, 7, 8], f.freqs.cpu().numpy(), 1.0, 64, False)
    assert np.all(np.abs(got.cpu().numpy() - want) <= 8 * U["f32"] * pair_sums(q.cpu().numpy(), 64, 64, False).reshape(4, -1))
    assert torch.equal(one.v[0, 0, 0, 15], kv[2].half()) and not one.v[0, 0, 0, :15].any()


# ------------------------------------------------------------------------------------------------ attention

def attend(ops, c, x, q, n_head, q_start, pos0, seq, max_new, mask, layer=0, max_kv=None, scale=None, out=None):
    return ops.attention_tree(on(ops, c), q if torch.is_tensor(q) else dev(q), ints(q_start), ints(pos0), None if seq is None else ints(seq), max_new=max_new, max_kv=max_kv,
                              mask=None if mask is None else dev(mask), layer=layer, scale=scale, out=out)


def check(got, c, x, q, n_head, q_start, pos0, seq, max_new, mask, layer=0, scale=None):
    hd = c.hd
    want, tol = po.attention(c, layer, q, n_head, q_start, pos0, seq, max_new, mask, hd ** -0.5 if scale is None else scale, U[x], U["f16"] if x == "f16" else 0.0)
    got = got.float().cpu().numpy().astype(np.float64).reshape(want.shape)
    of = ~np.isnan(want)
    bad = ~(np.abs(got - want) <= tol) & of
    assert not bad.any(), (int(bad.sum()), int(of.sum()), float(np.nanmax(np.abs(got - want)[of])), [int(a[0]) for a in np.nonzero(bad)])
    return want


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("news,lens,H,group,hd,page", [
    ([1], [1], 2, 2, 64, 16), ([1], [77], 2, 2, 64, 16), ([1, 1, 1], [300, 16, 1], 4, 1, 128, 64), ([25], [700], 2, 8, 128, 64), ([7, 0, 3, 1], [90, 40, 3, 65], 2, 3, 96, 32),
    ([2, 2], [500, 131], 1, 5, 192, 128), ([33, 5], [33, 800], 1, 2, 256, 16), ([64, 65, 130], [64, 300, 131], 1, 1, 64, 16), ([48, 40], [600, 410], 3, 1, 128, 32),
    ([130], [257], 1, 2, 96, 64), ([16] * 6, [200, 17, 16, 33, 129, 128], 2, 16, 64, 64), ([300], [300], 2, 1, 128, 16), ([20, 9], [1500, 30], 2, 4, 128, 16)])
def test_attention(ops, x, tree, news, lens, H, group, hd, page):
    rng = np.random.default_rng(hd + sum(lens) + group)
    n, T, layer = len(news), sum(news), 1
    c = pool(rng, 2, H, hd, page, lens)
    order = rng.permutation(n)
    c.table = c.table[np.argsort(order)]
    q_start, pos0, seq = starts(news), [a - b for a, b in zip(lens, news)], [int(i) for i in order]
    q = rows(rng, T, H * group * hd, x)
    mask = None
    if tree:
        masks, _ = po.tree_mask(trees(rng, news), q_start, pos0, max(news), -(-max(news) // 64))
        mask = words_of(masks, -(-max(news) // 64))
    got = attend(ops, c, x, q, H * group, q_start, pos0, seq, max(news), mask, layer, max_kv=max(lens))
    check(got, c, x, q, H * group, q_start, pos0, seq, max(news), mask, layer)
    assert ops.last_op_status() == 0
    # the same bits again, and without max_new and max_kv (other parts of the work) within the tolerance
    again = attend(ops, c, x, q, H * group, q_start, pos0, seq, max(news), mask, layer, max_kv=max(lens))
    assert torch.equal(got, again)
    other = attend(ops, c, x, q, H * group, q_start, pos0, seq, None, mask, layer)
    check(other, c, x, q, H * group, q_start, pos0, seq, T, mask, layer)


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,group,m", [(64, 1, 5), (128, 2, 40), (96, 4, 20), (256, 1, 70), (128, 8, 33), (64, 8, 64)])
def test_any_mask(ops, x, hd, group, m):
    """Bits that are no tree's: rows that see nothing, only others, only a later one; no context; bits behind the entry's tokens; fewer words than tokens."""
    rng = np.random.default_rng(m)
    news, lens = [m, m - 2, m], [m, m + 100, m + 15]
    c = pool(rng, 1, 2, hd, 16, lens)
    T = sum(news)
    words = -(-m // 64)
    mask = rng.integers(-2 ** 63, 2 ** 63, (T, words), dtype=np.int64) & rng.integers(-2 ** 63, 2 ** 63, (T, words), dtype=np.int64)
    mask[0] = 0
    mask[3], mask[4], mask[m + 1] = -1, 0, 0
    q_start, pos0 = starts(news), [a - b for a, b in zip(lens, news)]
    q = rows(rng, T, 2 * group * hd, x)
    got = attend(ops, c, x, q, 2 * group, q_start, pos0, None, m, mask)
    want = check(got, c, x, q, 2 * group, q_start, pos0, None, m, mask)
    assert not want[0].any() and not want[4].any() and want[3].any() and want[m + 1].any() and not got[0].any() and not got[4].any()


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,group,m", [(64, 2, 3), (128, 1, 20), (128, 8, 40), (192, 1, 18), (64, 8, 33), (96, 8, 40)])
def test_what_a_row_does_not_see_has_no_part_in_it(ops, x, hd, group, m):
    """Keys and values of other branches, behind the end, and of spare pages that are infinite or no numbers; pages that are not there, in the middle of the context too."""
    rng = np.random.default_rng(hd + m)
    lens = [m + 150, m + 37]
    c = pool(rng, 1, 2, hd, 16, lens, holes=[(0, 2), (0, 5), (1, 0)])
    news, q_start, pos0 = [m, m], [0, m, 2 * m], [150, 37]
    masks, _ = po.tree_mask(trees(rng, news), q_start, pos0, m, 1)
    mask = words_of(masks, 1)
    q = rows(rng, 2 * m, 2 * group * hd, x)
    plain = attend(ops, c, x, q, 2 * group, q_start, pos0, None, m, mask)
    check(plain, c, x, q, 2 * group, q_start, pos0, None, m, mask)
    odd = po.Cache(c.k.copy(), c.v.copy(), c.table)
    used = {odd.place(i, j) for i in range(2) for j in range(lens[i])}
    for p in range(odd.n_pages):
        for r in range(16):
            if (p, r) not in used:
                odd.k[0, p, :, r], odd.v[0, p, :, r] = np.nan, np.nan
    assert torch.equal(plain, attend(ops, odd, x, q, 2 * group, q_start, pos0, None, m, mask))
    # token 2 of each tree: only its descendants see it
    for i in range(2):
        p, r = odd.place(i, pos0[i] + 2)
        odd.k[0, p, :, r, ::3], odd.v[0, p, :, r, 1::2], odd.v[0, p, :, r, ::2] = np.inf, -np.inf, np.nan
    got = attend(ops, odd, x, q, 2 * group, q_start, pos0, None, m, mask)
    blind = [t for t in range(2 * m) if not masks[t] >> 2 & 1]
    g, w = got.view(2 * m, -1), plain.view(2 * m, -1)
    assert len(blind) > m
    assert torch.isfinite(g[blind]).all()
    want, tol = po.attention(c, 0, q, 2 * group, q_start, pos0, None, m, mask, hd ** -0.5, U[x], U["f16"] if x == "f16" else 0.0)
    d = np.abs(g.float().cpu().numpy().astype(np.float64).reshape(want.shape) - want)
    assert np.all(d[blind] <= tol[blind])
    seeing = [t for t in range(2 * m) if t not in blind]
    assert not torch.isfinite(g[seeing]).any()


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd,group,m,context", [(128, 2, 40, 4000), (192, 4, 40, 4000), (256, 2, 40, 4000), (256, 8, 20, 40), (192, 1, 5, 900)])
def test_a_row_with_one_column_that_is_no_number(ops, x, hd, group, m, context):
    """A value of a drafted token that is not finite, in the first or the last column alone: whoever sees it is not finite there, the others are as before."""
    rng = np.random.default_rng(hd + context)
    lens = [context + m, m]
    c = pool(rng, 1, 2, hd, 64, lens)
    news, q_start, pos0 = [m, m], [0, m, 2 * m], [context, 0]
    masks, _ = po.tree_mask(trees(rng, news), q_start, pos0, m, 1)
    mask = words_of(masks, 1)
    q = rows(rng, 2 * m, 2 * group * hd, x)
    want, tol = po.attention(c, 0, q, 2 * group, q_start, pos0, None, m, mask, hd ** -0.5, U[x], U["f16"] if x == "f16" else 0.0)
    seeing = np.array([bool(masks[t] >> 2 & 1) for t in range(2 * m)])
    want, tol = want.reshape(2 * m, 2, group, hd), tol.reshape(2 * m, 2, group, hd)
    for column, value in ((0, np.nan), (hd - 1, np.inf), (hd // 2, -np.inf), (hd // 2 - 1, np.nan)):
        odd = po.Cache(c.k.copy(), c.v.copy(), c.table)
        for i in range(2):
            p, r = odd.place(i, pos0[i] + 2)
            odd.v[0, p, 1, r, column] = value
        got = attend(ops, odd, x, q, 2 * group, q_start, pos0, None, m, mask).float().cpu().numpy().astype(np.float64).reshape(want.shape)
        near = np.abs(got - want) <= tol
        assert near[~seeing].all() and near[:, 0].all() and seeing.any() and not np.isfinite(got[seeing][:, 1, :, column]).any()


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_attention_of_what_the_cache_lacks(ops, x):
    """Entries of no sequence, first slots behind the table, tokens without a slot, rows of no entry, one sequence twice, an end below the start."""
    rng = np.random.default_rng(9)
    c = pool(rng, 1, 2, 128, 16, [64, 64])
    q_start, pos0, seq = [1, 21, 24, 26, 30, 28], [50, 10, 64, 3, 1], [0, 1, 1, 0, 1]
    q = rows(rng, 34, 4 * 128, x)
    for mask in (None, rng.integers(-2 ** 63, 2 ** 63, (34, 1), dtype=np.int64)):
        out = torch.full((34, 512), 7.0, dtype=TY[x], device="cuda")
        got = attend(ops, c, x, q, 4, q_start, pos0, seq, 20, mask, out=out)
        assert got is out
        want = check(got, c, x, q, 4, q_start, pos0, seq, 20, mask)
        none = np.isnan(want).all((1, 2))
        assert none[[0, 30, 31, 32, 33]].all() and bool((out[dev(none)] == 7.0).all())
        assert not want[15:21].any() and not out[15:21].any() and want[1:15].any()
        assert not out[24:26].any()                                   # (its first slot is behind the table's end)
    far = attend(ops, c, x, q, 4, q_start, pos0, [0, 5, -1, 0, 1], 20, None, out=torch.ones(34, 512, dtype=TY[x], device="cuda"))
    assert not far[21:26].any()


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("m,group", [(1, 2), (3, 4), (40, 4)])
def test_scores_of_all_sizes(ops, x, m, group):
    """Large and tiny scales, a channel far above the others, rising scores (every maximum is a new one), equal ones, keys of the largest halves."""
    rng = np.random.default_rng(m)
    c = pool(rng, 1, 2, 64, 32, [m + 400])
    c.k[0, ..., 5] *= 200.0
    q = rows(rng, m, 2 * group * 64, x)
    for scale in (3.0, 1e-6, 0.0, -0.5):
        got = attend(ops, c, x, q, 2 * group, [0, m], [400], None, m, None, scale=scale)
        check(got, c, x, q, 2 * group, [0, m], [400], None, m, None, scale=scale)
    for j in range(400):
        p, r = c.place(0, j)
        c.k[0, p, :, r] = 0
        c.k[0, p, :, r, 0] = 0.25 * j
    q[:, ::64] = 1.0
    got = attend(ops, c, x, q, 2 * group, [0, m], [400], None, m, None, scale=1.0)
    check(got, c, x, q, 2 * group, [0, m], [400], None, m, None, scale=1.0)


def test_rows_that_are_not_finite_are_no_numbers(ops):
    rng = np.random.default_rng(1)
    for m, group in ((2, 2), (40, 4)):
        c = pool(rng, 1, 1, 64, 16, [m + 50])
        for x in ("f32", "f16"):
            q = rows(rng, m, group * 64, x)
            good = attend(ops, c, x, q, group, [0, m], [50], None, m, None)
            q[1, 3] = np.inf
            got = attend(ops, c, x, q, group, [0, m], [50], None, m, None)
            assert torch.isnan(got[1, :64]).all() and torch.equal(got[0], good[0])
        c.k[...] = 0
        c.k[..., 0] = -np.inf                                         # every score is -infinity: no softmax
        q = np.abs(rows(rng, m, group * 64, "f16"))
        assert torch.isnan(attend(ops, c, "f16", q, group, [0, m], [50], None, m, None)).all()


def test_long_contexts_and_parts(ops):
    """One sequence of 20000 slots beside one of 3: parts of it that the short one does not have; more slots than max_kv says."""
    rng = np.random.default_rng(2)
    c = pool(rng, 1, 1, 64, 64, [20000, 3])
    for m, group in ((1, 4), (3, 30)):
        q = rows(rng, 2 * m, group * 64)
        for max_kv in (20000, 1000, 1):
            got = attend(ops, c, "f32", q, group, [0, m, 2 * m], [20000 - m, 3 - m], None, m, None, max_kv=max_kv)
            check(got, c, "f32", q, group, [0, m, 2 * m], [20000 - m, 3 - m], None, m, None)


def test_a_pool_larger_than_32_bits(ops):
    """Pages whose offset in the pool is more than 2^31 halves (and 2^32 bytes)."""
    n_pages, H, page, hd = 2200, 64, 128, 128                         # 2.3e9 halves a pool
    k, v = (torch.zeros(1, n_pages, H, page, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    table = ints([[n_pages - 1, 3, n_pages - 2]])
    big = ops.KvCachePaged(k, v, table)
    small = ops.KvCachePaged.empty(1, 3, 3, H, hd, page)
    small.table.copy_(ints([[0, 1, 2]]))
    kv, q = torch.randn(2, 300, H * hd, device="cuda"), torch.randn(300, H * hd, device="cuda")
    for c in (big, small):
        ops.kv_append_paged(c, kv[0], kv[1], ints([0, 300]), ints([0]))
    assert torch.equal(k[0, n_pages - 1], small.k[0, 0]) and torch.equal(v[0, 3], small.v[0, 1])
    for rows_ in (1, 300):
        a, b = (ops.attention_tree(c, q[:rows_], ints([0, rows_]), ints([300 - rows_])) for c in (big, small))
        assert torch.equal(a, b)
    for c in (big, small):
        ops.kv_keep_paged(c, ints([[0, 2, 5, 90]]), ints([4]), ints([200]))
    assert torch.equal(k[0, n_pages - 1], small.k[0, 0]) and torch.equal(v[0, 3], small.v[0, 1]) and torch.equal(k[0, n_pages - 2], small.k[0, 2])


# ------------------------------------------------------------------------------------------------ the path that stays

@pytest.mark.parametrize("hd,page,n_layer,H,paths,pos0", [
    (128, 64, 3, 2, [[0, 3, 7, 8, 30]], [60]), (64, 16, 2, 3, [[0], [2, 5, 6], [0, 1, 2, 3], [1]], [15, 0, 31, 14]), (96, 32, 1, 5, [[0, 5, 9], list(range(3, 40))], [20, 20]),
    (192, 16, 2, 1, [[0, 1, 4, 9, 16, 25]], [7]), (256, 128, 4, 2, [list(range(1, 60, 2)), [0, 59]], [100, 127]), (64, 64, 1, 1, [list(range(1, 400))], [3])])
def test_keep(ops, hd, page, n_layer, H, paths, pos0):
    rng = np.random.default_rng(hd + page)
    lens = [p + max(r) + 1 for p, r in zip(pos0, paths)]
    c = pool(rng, n_layer, H, hd, page, lens)
    most = max(len(p) for p in paths) + 2
    path = np.array([p + [-1] * (most - len(p)) for p in paths], np.int32)
    n_path = [len(p) for p in paths]
    one = on(ops, c)
    ops.kv_keep_paged(one, dev(path), ints(n_path), ints(pos0))
    k, v = po.keep(c, path, n_path, pos0, None)
    assert np.array_equal(one.k.cpu().numpy(), k) and np.array_equal(one.v.cpu().numpy(), v)


def test_keep_of_odd_paths(ops):
    """Paths that fall, that end early, longer than they say, of no sequence, of one sequence twice, over pages that are not there, past the table's end."""
    rng = np.random.default_rng(4)
    c = pool(rng, 2, 2, 64, 16, [64, 64, 64], holes=[(1, 1), (2, 3)])
    path = np.array([[0, 4, 3, 9, 10], [1, 2, 20, 22, 30], [5, 6, -1, 8, 9], [0, 2, 4, 6, 8], [3, 4, 5, 6, 70], [3, 4, 5, 50, 0x7fffffff], [1, 2, 3, 4, 5]], np.int32)
    n_path, pos0, seq = [5, 5, 5, 5, 5, 9, 0], [3, 5, 40, 7, 60, 0, 0], [0, 1, 2, 9, 0, 2, 1]
    one = on(ops, c)
    ops.kv_keep_paged(one, dev(path), ints(n_path), ints(pos0), ints(seq))
    k, v = po.keep(c, path, n_path, pos0, seq)
    assert np.array_equal(one.k.cpu().numpy(), k) and np.array_equal(one.v.cpu().numpy(), v)
    assert not np.array_equal(k, c.k)
    for bad in (dict(n_path=[0] * 7), dict(pos0=[-1, 64, 1 << 30, 0, 0, 0, 0], n_path=[5, 5, 5, 0, 0, 0, 0])):
        two = on(ops, c)
        ops.kv_keep_paged(two, dev(path), ints(bad["n_path"]), ints(bad.get("pos0", pos0)), ints([0, 1, 2, 0, 0, 0, 0]))
        assert np.array_equal(two.k.cpu().numpy(), c.k) and np.array_equal(two.v.cpu().numpy(), c.v)


# ------------------------------------------------------------------------------------------------ together

class Toy:
    """Two layers of attention with fixed random projections and a vocabulary of 40: enough of a model to decode with."""

    def __init__(self, ops, hd=64, H=2, group=2, vocab=40, n_layer=2, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ops, self.hd, self.H, self.nh, self.n_layer = ops, hd, H, H * group, n_layer
        d = self.nh * hd
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.emb, self.out = r(vocab, d), r(vocab, d)
        self.wq, self.wk, self.wv, self.wo = ([r(n, d) / d ** 0.5 for _ in range(n_layer)] for n in (d, H * hd, H * hd, d))
        self.freqs = ops.rope_freqs(hd)

    def step(self, cache, tokens, q_start, pos0, seq, most, mask=None, pos=None):
        h = self.emb[tokens.long()]
        for l in range(self.n_layer):
            x = h / h.norm(dim=1, keepdim=True) * h.shape[1] ** 0.5
            q = self.ops.kv_append_paged(cache, x @ self.wk[l].T, x @ self.wv[l].T, q_start, pos0, seq, max_new=most, q=x @ self.wq[l].T, pos=pos, freqs=self.freqs, layer=l)
            h = h + self.ops.attention_tree(cache, q, q_start, pos0, seq, max_new=most, mask=mask, layer=l) @ self.wo[l].T
        return h @ self.out.T


def test_speculative_steps_give_the_greedy_tokens(ops):
    """Two sequences decoded token by token, and again in steps of drafted trees, some of whose branches are right: the same tokens, and the same cache rows."""
    torch.backends.cuda.matmul.allow_tf32 = False
    toy, rng, n, steps, prompt = Toy(ops), np.random.default_rng(0), 2, 40, [[3, 7, 1, 9, 30], [5, 5]]

    def fresh():
        c = ops.KvCachePaged.empty(n, 8, 20, toy.H, toy.hd, page=16, n_layer=toy.n_layer)
        c.table.copy_(ints(rng.permutation(20)[:16].reshape(2, 8).tolist()))
        return c

    start = lambda: (ints(sum(prompt, [])), ints([0, 5, 7]), ints([0, 0]), None, 5)
    c = fresh()
    last = toy.step(c, *start()).argmax(1)[[4, 6]].tolist()
    want = [[t] for t in last]
    lens = [5, 2]
    for _ in range(steps):
        last = toy.step(c, ints(last), ints([0, 1, 2]), ints(lens), None, 1).argmax(1).tolist()
        lens = [m + 1 for m in lens]
        for i in range(n):
            want[i].append(last[i])
    plain = c
    c = fresh()
    last = toy.step(c, *start()).argmax(1)[[4, 6]].tolist()
    got, lens, calls, taken = [[t] for t in last], [5, 2], 0, 0
    while min(len(g) for g in got) < steps:
        # a tree for each sequence: the last token, then drafted ones; some follow the right continuation, others are any
        tokens, parents, news = [], [], []
        for i in range(n):
            m = int(rng.integers(1, 14))
            tok, par, deep = [got[i][-1]], [-1], [0]
            for u in range(1, m):
                p = int(rng.integers(max(0, u - 4), u))
                right = len(got[i]) + deep[p]
                tok.append(want[i][right] if rng.random() < 0.7 and right < len(want[i]) else int(rng.integers(0, 40)))
                par.append(p); deep.append(deep[p] + 1)
            tokens += tok; parents += par; news.append(m)
        q_start, pos0, most = ints(starts(news)), ints(lens), max(news)
        tokens, parents = ints(tokens), ints(parents)
        mask, pos = ops.tree_mask(parents, q_start, pos0, max_new=most)
        choice = toy.step(c, tokens, q_start, pos0, None, most, mask, pos).argmax(1).int()
        path, n_path, then = ops.tree_accept(tokens, parents, choice, q_start, max_new=most)
        ops.kv_keep_paged(c, path, n_path, pos0)
        calls += 1
        for i in range(n):
            way = [int(tokens[starts(news)[i] + u]) for u in path[i, 1:int(n_path[i])].tolist()] + [int(then[i])]
            got[i] += way
            taken += len(way)
            lens[i] += int(n_path[i])
        if max(lens) > 60:
            break
    for i in range(n):
        k = min(len(got[i]), len(want[i]))
        assert k > 15 and got[i][:k] == want[i][:k]
    assert taken > 1.5 * n * calls                                    # drafts were taken
    for i in range(n):
        for j in range(min(lens[i], 5 + 15)):
            a, b = (divmod(j, 16) for _ in range(2))
            for x in ("k", "v"):
                p, q = (getattr(o, x)[:, int(o.table[i, a[0]]), :, a[1]].float() for o in (c, plain))
                assert (p - q).abs().max().item() <= 2.0 ** -7 * (1 + q.abs().max().item())


def test_other_streams_and_captured_graphs(ops):
    """The same results from another stream, and from a graph that is captured once and replayed with other inputs in the same places."""
    rng = np.random.default_rng(8)
    lens, news, H, group, hd = [900, 130], [12, 30], 2, 4, 128
    c = pool(rng, 2, H, hd, 64, lens)
    T, q_start, pos0 = 42, ints([0, 12, 42]), ints([888, 100])
    parents = ints(trees(rng, news))
    f = ops.rope_freqs(hd)
    q, k, v = (torch.randn(T, h * hd, device="cuda") for h in (H * group, H, H))
    tokens, choice = ints(rng.integers(0, 3, T).tolist()), ints(rng.integers(0, 3, T).tolist())

    def step(cache):
        mask, pos = ops.tree_mask(parents, q_start, pos0, max_new=30)
        turned = ops.kv_append_paged(cache, k, v, q_start, pos0, max_new=30, q=q, pos=pos, freqs=f, layer=1)
        out = ops.attention_tree(cache, turned, q_start, pos0, max_new=30, mask=mask, layer=1)
        path, n_path, then = ops.tree_accept(tokens, parents, choice, q_start, max_new=30)
        ops.kv_keep_paged(cache, path, n_path, pos0)
        return out, path, n_path, then

    one = on(ops, c)
    want = step(one)
    two, side = on(ops, c), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(two)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(one.k, two.k) and torch.equal(one.v, two.v)
    three = on(ops, c)
    with torch.cuda.stream(side):
        step(three)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(three)
    for seed in range(2):
        torch.manual_seed(seed)
        for t in (q, k, v):
            t.normal_()
        choice.copy_(ints(rng.integers(0, 3, T).tolist()))
        three.k.copy_(dev(c.k)); three.v.copy_(dev(c.v))
        graph.replay()
        four = on(ops, c)
        want = step(four)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured)) and torch.equal(three.k, four.k) and torch.equal(three.v, four.v)


def test_the_same_on_tcgen05_whatever_the_size():
    """Small calls of many rows run with mma.sync: all of the attention's tests again with those on tcgen05."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "pytest", __file__, "-x", "-q", "-p", "no:cacheprovider", "-k", "attention or mask or row or sizes or parts or pool or speculative or streams"],
                       env={**os.environ, "PI_ATTN_TREE_TC": "1"}, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-4000:]


def test_refusals(ops):
    c = ops.KvCachePaged.empty(2, 4, 8, 2, 64, page=16)
    q, kv, start, pos0 = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 128, device="cuda"), ints([0, 1, 2]), ints([0, 0])
    f, par = ops.rope_freqs(64), ints([-1, -1])
    k = c.k
    for bad in (lambda: ops.KvCachePaged(k.float(), c.v, c.table), lambda: ops.KvCachePaged(k, c.v[:, :4], c.table), lambda: ops.KvCachePaged(k, c.v, c.table.long()),
                lambda: ops.KvCachePaged(k, c.v, c.table[0]), lambda: ops.KvCachePaged(k[0, 0], c.v[0, 0], c.table), lambda: ops.KvCachePaged(k.transpose(1, 2), c.v.transpose(1, 2), c.table),
                lambda: ops.KvCachePaged(k, c.v, c.table.cpu()), lambda: ops.tree_mask(par.long(), start, pos0), lambda: ops.tree_mask(par, start[:2], pos0), lambda: ops.tree_mask(par, start, pos0.cpu()),
                lambda: ops.tree_accept(par, par[:1], par, start), lambda: ops.tree_accept(par, par, par.float(), start), lambda: ops.kv_append_paged(c, kv, kv[:1], start, pos0),
                lambda: ops.kv_append_paged(c, kv, kv.half(), start, pos0), lambda: ops.kv_append_paged(c, kv, kv, start, pos0, q=q), lambda: ops.kv_append_paged(c, q, q, start, pos0),
                lambda: ops.kv_append_paged(c, kv, kv, start, pos0, q=q[:, :100], freqs=f), lambda: ops.kv_append_paged(c, kv, kv, start, pos0, pos=pos0[:1]),
                lambda: ops.attention_tree(c, q[:, :100], start, pos0), lambda: ops.attention_tree(c, q, start, pos0, mask=torch.zeros(2, 1, device="cuda")),
                lambda: ops.attention_tree(c, q, start, pos0, mask=torch.zeros(1, 1, dtype=torch.int64, device="cuda")), lambda: ops.attention_tree(c, q, start, pos0, out=q.half()),
                lambda: ops.attention_tree(c, q.cpu(), start, pos0), lambda: ops.attention_tree(c, q.double(), start, pos0), lambda: ops.kv_keep_paged(c, par, par, pos0),
                lambda: ops.kv_keep_paged(c, par.view(2, 1), par, pos0.long()), lambda: ops.kv_keep_paged(c, par.view(2, 1).cpu(), par, pos0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.kv_append_paged(c, kv, kv, start, pos0, layer=1), lambda: ops.attention_tree(c, q, start, pos0, layer=-1), lambda: ops.tree_mask(par, start, pos0, words=100),
                lambda: ops.kv_append_paged(c, kv, kv, start, pos0, freqs=ops.rope_freqs(128)), lambda: ops.attention_tree(c, q[:, :64], start, pos0)):
        with pytest.raises(Exception):
            bad()
    assert ops.attention_tree(c, q, start, pos0).abs().max().item() == 0.0      # (no page is there)
    one = ops.KvCachePaged(c.k[0], c.v[0], c.table)                   # a layer alone
    assert one.n_layer == 1 and ops.attention_tree(one, q[:0], ints([0, 0, 0]), pos0).shape == (0, 256)
