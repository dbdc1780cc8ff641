"""Calls of the operators of drafted tokens over a paged cache where they went wrong once or that the tests beside them do not reach, against paged_oracle.  Half a step is
u = 2^-24 in FP32, 2^-11 in FP16."""
import numpy as np
import pytest

import paged_oracle as po
from test_gpu_paged import TY, U, attend, check, dev, ints, on, ops, pool, rows, starts, trees, words_of  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------------------------------ bits of the probabilities

def norms(got, want):
    """Norms of the error and of what rounding the exact result would leave, over the exact result's."""
    got = got.double().cpu().numpy().reshape(want.shape)
    n = np.linalg.norm(want)
    return np.linalg.norm(got - want) / n, np.linalg.norm(want.astype(np.float16).astype(np.float64) - want) / n


@pytest.mark.parametrize("hd,m,group,slots", [(64, 16, 8, 4096), (96, 16, 8, 4096), (128, 16, 8, 4096), (128, 40, 4, 1500), (64, 1, 8, 4096), (128, 2, 8, 1000), (256, 1, 16, 600), (192, 1, 5, 900)])
def test_f16_rows_have_the_error_of_their_own_rounding(ops, hd, m, group, slots):
    """Results are the roundings of sums with 22 bits of each probability.  Values of both signs: a probability's rounding to 11 bits would leave errors as large as the result's own
    rounding, 1.3 times in all.  Scores are off by less than 2^-17 of a probability here (|s| < 16, hd u of the terms' sizes), as is all else: the rounding itself and 2^-16 beside it."""
    rng = np.random.default_rng(hd + m)
    H = 8
    c = pool(rng, 1, H, hd, 64, [slots])
    q = rows(rng, m, H * group * hd, "f16")
    want, _ = po.attention(c, 0, q, H * group, [0, m], [slots - m], None, m, None, hd ** -0.5, U["f16"], 0.0)
    got = attend(ops, c, "f16", q, H * group, [0, m], [slots - m], None, m, None, max_kv=slots)
    error, rounding = norms(got, want)
    assert error <= 1.02 * rounding + 2.0 ** -16, (error, rounding)


def test_f16_sums_of_many_steps_are_added_with_rounding(ops):
    """9 to 16 rows of a KV head, 2048 steps of a warp (max_kv sets no parts).  Rounded sums are off by some sqrt(2048) u, 3e-6, in no direction, and flip few of the results'
    own roundings; sums that lose their last bits at every step are below by up to 2048 u, 1.2e-4.  Of 1024 results, the mean of what is left behind the exact one's rounding."""
    rng = np.random.default_rng(0)
    slots, hd = 131072, 64
    c = pool(rng, 1, 1, hd, 128, [slots])
    c.v[:] = (rng.uniform(1, 2, hd) * (1 + 0.25 * rng.standard_normal(c.v.shape).clip(-3, 3))).astype(np.float16)
    q = rows(rng, 2, 8 * hd, "f16")
    want, _ = po.attention(c, 0, q, 8, [0, 2], [slots - 2], None, 2, None, hd ** -0.5, U["f16"], 0.0)
    got = attend(ops, c, "f16", q, 8, [0, 2], [slots - 2], None, 2, None, max_kv=1).double().cpu().numpy().reshape(want.shape)
    assert abs(((got - want.astype(np.float16)) / want).mean()) <= 2.0 ** -16


@pytest.mark.parametrize("hd,m,group,slots", [(64, 16, 8, 4096), (96, 16, 8, 4096), (128, 16, 8, 4096), (192, 16, 8, 2000), (256, 16, 8, 2000), (64, 3, 8, 20000), (128, 1, 4, 20000),
                                              (64, 1, 8, 900), (96, 2, 8, 900), (192, 2, 5, 900), (256, 1, 16, 900)])
def test_f32_rows_keep_the_bits_of_both_halves(ops, hd, m, group, slots):
    """The norm of the error, over the result's.  Queries or probabilities of one half alone would leave 2^-12.8 (a score is some units); with both, errors of a query and of a probability are 2^-22
    of it or less, a score of up to 8 is a sum of hd / 16 steps off by 2^-22 at most, 4 of which in the root of their squares are 2^-20, and a probability is off by as much of itself: twice that, and
    as much again for the sums."""
    rng = np.random.default_rng(hd + m)
    H = 8
    c = pool(rng, 1, H, hd, 32, [slots])
    q = rows(rng, m, H * group * hd)
    want, _ = po.attention(c, 0, q, H * group, [0, m], [slots - m], None, m, None, hd ** -0.5, U["f32"], 0.0)
    got = attend(ops, c, "f32", q, H * group, [0, m], [slots - m], None, m, None, max_kv=slots)
    assert norms(got, want)[0] <= 2.0 ** -18


@pytest.mark.parametrize("hd,m", [(192, 16), (256, 16)])
def test_wide_f16_rows_have_the_error_of_their_own_rounding(ops, hd, m):
    test_f16_rows_have_the_error_of_their_own_rounding(ops, hd, m, 8, 2000)


# ------------------------------------------------------------------------------------------------ pieces after pieces

@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
def test_values_of_special_tiles_are_waited_for(ops, x, hd):
    """Contexts of a few tiles, many of them a CTA: the last tile's values are gone over before they are used, and the tile before it may still be on its way.  What lies behind the ends is no
    number, so values that were gone over too early (or another tile's in their place) show."""
    rng = np.random.default_rng(hd)
    n, H, group, m = 24, 8, 8, 5
    lens = [int(v) for v in rng.integers(m + 100, 700, n)]
    c = pool(rng, 1, H, hd, 64, lens, holes=[(3, 1), (5, 0)])
    news, q_start, pos0 = [m] * n, starts([m] * n), [v - m for v in lens]
    masks, _ = po.tree_mask(trees(rng, news), q_start, pos0, m, 1)
    mask = words_of(masks, 1)
    q = rows(rng, n * m, H * group * hd, x)
    odd = po.Cache(np.full_like(c.k, np.nan), np.full_like(c.v, np.nan), c.table)
    for i in range(n):
        for j in range(lens[i]):
            if (at := c.place(i, j)) is not None:
                odd.k[0, at[0], :, at[1]], odd.v[0, at[0], :, at[1]] = c.k[0, at[0], :, at[1]], c.v[0, at[0], :, at[1]]
    for causal in (False, True):
        args = (c, x, q, H * group, q_start, pos0, None, m, None if causal else mask)
        plain = attend(ops, *args, max_kv=max(lens))
        check(plain, *args)
        for _ in range(10):
            assert torch.equal(plain, attend(ops, odd, *args[1:], max_kv=max(lens)))
        assert ops.last_op_status() == 0


@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("n,H,m,group,hd,kv,cut", [
    (20, 16, 5, 8, 128, 700, "whole"), (20, 16, 5, 8, 64, 500, "whole"), (7, 22, 5, 8, 64, 2000, "both"), (5, 30, 5, 8, 96, 2000, "both"), (5, 30, 5, 8, 128, 2000, "both"),
    (5, 16, 5, 8, 192, 2000, "both"), (5, 16, 5, 8, 256, 1500, "whole"), (5, 16, 5, 8, 256, 2000, "both"), (1, 22, 60, 8, 64, 700, "few"), (1, 22, 120, 8, 64, 700, "whole"),
    (40, 8, 1, 8, 128, 1000, "both"), (60, 8, 1, 8, 64, 1500, "both"), (40, 8, 2, 8, 96, 1500, "both"), (20, 8, 2, 8, 192, 1500, "both"), (20, 8, 1, 4, 256, 1000, "both")])
def test_more_items_than_processors(ops, x, n, H, m, group, hd, kv, cut):
    """More pieces of work than CTAs run at once, of unequal lengths; items that are a piece each beside others in parts ("both"); entries without tokens and without a context."""
    from powerinfer_b200 import _lib
    rng = np.random.default_rng(n + hd)
    news = [m if i in (0, 3) else int(v) for i, v in enumerate(rng.integers(0, m + 1, n))]
    lens = [kv if i == 0 else news[i] if i % 5 == 4 else int(v) for i, v in enumerate(rng.integers(m, kv + 1, n))]
    c = pool(rng, 1, H, hd, 32, lens)
    q_start, pos0, T = starts(news), [a - b for a, b in zip(lens, news)], sum(news)
    masks, _ = po.tree_mask(trees(rng, news), q_start, pos0, m, 1)
    q = rows(rng, T, H * group * hd, x)
    # the parts that the workspace has room for, in tiles of rows
    many = m * group > 16
    R, size = 128 if many else 8 if m * group <= 8 else 16, 2 if x == "f16" else 4
    need = _lib.lib.pi_attention_tree_workspace_bytes(on(ops, c).c, ops._entries(ints(q_start), ints(pos0), None, T, m, 0), ops._ROW_TYPES[TY[x]], H * group, kv)
    parts = (need - (256 + T * H * group * (hd * size + (4 if x == "f32" else 0)) if many else min(need, 256))) // ((8 + 4 * hd) * R)
    items = n * H * -(-m * group // R) * (2 if many and hd > 128 else 1)
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert (items > 148) == (cut != "few") and (0 < parts < items // 2 if cut == "both" else parts == 0), (parts, items)
    args = (c, x, q, H * group, q_start, pos0, None, m, None if x == "f32" else words_of(masks, 1))
    got = attend(ops, *args, max_kv=kv)
    check(got, *args)
    assert ops.last_op_status() == 0 and torch.equal(got, attend(ops, *args, max_kv=kv))


# ------------------------------------------------------------------------------------------------ strides

@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("n,m,kv", [(3, 1, 700), (3, 2, 3000), (12, 9, 700), (1, 9, 6000)])
def test_rows_16_bytes_off(ops, x, hd, n, m, kv):
    """Queries and results as columns of wider matrices that begin 16 bytes behind a boundary of 32, rows an odd number of 16 bytes apart: the bits of contiguous ones, and nothing beside them."""
    from powerinfer_b200 import _lib
    rng = np.random.default_rng(hd + m)
    H, group = 4, 8
    lens = [kv] + [int(v) for v in rng.integers(m, kv, n - 1)]
    c, T, width, pad = on(ops, pool(rng, 1, H, hd, 16, lens)), n * m, H * group * hd, 16 // (4 if x == "f32" else 2)
    wide = dev(rows(rng, T, width + 3 * pad, x))
    q = wide[:, pad:pad + width]
    q_start, pos0 = ints(starts([m] * n)), ints([v - m for v in lens])
    want = ops.attention_tree(c, q.contiguous(), q_start, pos0, max_new=m, max_kv=kv)
    assert q.data_ptr() % 32 == 16 and q.stride(0) * q.element_size() % 32 == 16
    assert torch.equal(want, ops.attention_tree(c, q, q_start, pos0, max_new=m, max_kv=kv))
    to = torch.full((T, width + 5 * pad), 7.0, dtype=TY[x], device="cuda")
    b = ops._entries(q_start, pos0, None, T, m, 0)
    need = _lib.lib.pi_attention_tree_workspace_bytes(c.c, b, ops._ROW_TYPES[TY[x]], H * group, kv)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    assert _lib.lib.pi_attention_tree(c.c, b, 0, ops._ROW_TYPES[TY[x]], q.data_ptr(), q.stride(0), H * group, None, 0, kv, hd ** -0.5, to[:, pad:].data_ptr(), to.stride(0), ws.data_ptr(), ws.numel(),
                                      ops._stream()) == 0
    assert torch.equal(to[:, pad:pad + width], want) and (to[:, :pad] == 7).all() and (to[:, pad + width:] == 7).all()
    assert torch.isfinite(want).all() and _lib.lib.pi_op_status(ws.data_ptr(), ops._stream()) == 0


# ------------------------------------------------------------------------------------------------ calls at once

@pytest.mark.parametrize("x", ["f32", "f16"])
def test_two_calls_at_once(ops, x):
    """Steps on two streams at the same time, and two captured graphs of them replayed at the same time: the bits of each alone."""
    steps, want, streams, graphs, captured = [], [], [torch.cuda.Stream() for _ in range(2)], [], []
    for hd, m, kv in ((128, 20, 1500), (256, 9, 900)):
        rng = np.random.default_rng(hd)
        c, H, group = pool(rng, 1, 8, hd, 32, [kv, kv // 2, m]), 8, 8
        pos0, q_start, T = ints([kv - m, kv // 2 - m, 0]), ints(starts([m] * 3)), 3 * m
        masks, _ = po.tree_mask(trees(rng, [m] * 3), starts([m] * 3), [0] * 3, m, 1)
        cache, q, kv_rows, mask, f = on(ops, c), dev(rows(rng, T, H * group * hd, x)), dev(rows(rng, T, H * hd, x)), dev(words_of(masks, 1)), ops.rope_freqs(hd)

        def step(cache=cache, q=q, kv_rows=kv_rows, mask=mask, f=f, pos0=pos0, q_start=q_start, m=m, kv=kv):
            turned = ops.kv_append_paged(cache, kv_rows, kv_rows, q_start, pos0, max_new=m, q=q, freqs=f)
            return [ops.attention_tree(cache, turned, q_start, pos0, max_new=m, max_kv=kv, mask=mask) for _ in range(8)]

        steps.append(step)
        want.append(step()[0])
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, step in zip(streams, steps):
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, g in zip(want, got) for o in g)
    for s, step in zip(streams, steps):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            captured.append(step())
    for _ in range(3):
        for outs in captured:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, g in zip(want, captured) for o in g)


# ------------------------------------------------------------------------------------------------ waits that run out

def test_last_op_status_is_that_of_the_attention(ops):
    """The status word that last_op_status reads is the last operator's: set as if a wait had run out, cleared by the next call."""
    rng = np.random.default_rng(6)
    c = pool(rng, 1, 8, 64, 64, [4096])
    q = rows(rng, 40, 32 * 64)
    attend(ops, c, "f32", q, 32, [0, 40], [4056], None, 40, None)
    assert ops.last_op_status() == 0
    ops._ws.asked[1].view(torch.int32)[2] = 16
    assert ops.last_op_status() == 5
    attend(ops, c, "f32", q, 32, [0, 40], [4056], None, 40, None)
    assert ops.last_op_status() == 0
    attend(ops, c, "f32", q[:1], 32, [0, 1], [50], None, 1, None, max_kv=64)
    assert ops.last_op_status() == 0


def run_out(hd, x):
    """In a process whose waits ask a few times only: statuses, what comes of rows, and calls behind them."""
    from powerinfer_b200 import ggml_ops as g
    rng = np.random.default_rng(hd)
    n, H, group, m = 24, 8, 8, 5
    lens = [int(v) for v in rng.integers(m + 100, 1000, n)]
    c = pool(rng, 1, H, hd, 64, lens)
    q_start, pos0, T = [1 + i * m for i in range(n + 1)], [v - m for v in lens], n * m + 3
    q = dev(rows(rng, T, H * group * hd, x))
    some = range(0, n, 5)                                             # entries whose rows are compared
    exact = [po.attention(c, 0, q[1 + i * m:1 + i * m + m].cpu().numpy(), H * group, [0, m], [pos0[i]], [i], m, None, hd ** -0.5, U[x], U["f16"] if x == "f16" else 0.0) for i in some]
    seen = []
    for max_kv in (max(lens), 6000, max(lens)):
        out = torch.full((T, H * group * hd), 7.0, dtype=TY[x], device="cuda")
        attend(g, c, x, q, H * group, q_start, pos0, None, m, None, max_kv=max_kv, out=out)
        seen.append(g.last_op_status())
        few = attend(g, c, x, q[1:2], H * group, [0, 1], [300], None, 1, None)         # (no bounded waits)
        check(few, c, x, q[1:2].cpu().numpy(), H * group, [0, 1], [300], None, 1, None)
        assert (out[0] == 7).all() and (out[n * m + 1:] == 7).all()   # rows of no entry
        got = out[1:n * m + 1].double().cpu().numpy()
        none = np.isnan(got)                                          # right, or no numbers; none as it was
        assert none.any() == (seen[-1] != 0) and not (got == 7).any()
        for i, (want, tol) in zip(some, exact):
            rows_ = slice(i * m, i * m + m)
            assert np.all((np.abs(got[rows_] - want.reshape(m, -1)) <= tol.reshape(m, -1)) | none[rows_])
    return seen


@pytest.mark.parametrize("tries", [0, 1])
def test_waits_that_run_out_end_with_a_status(ops, tries):
    """PI_ATTN_TREE_TRIES shortens the waits (the first one, for the work in hand, asks once with 0): the kernel ends, reports, rows are right or no numbers, and the
    calls behind it are right."""
    import os
    import subprocess
    import sys
    code = f"import sys; sys.path[:0] = [{os.path.dirname(__file__)!r}, {os.path.dirname(os.path.dirname(__file__))!r}]\nimport test_gpu_paged_edges as t\n" + \
        "print('status', *[s for hd in (64, 96, 128, 192, 256) for x in ('f32', 'f16') for s in t.run_out(hd, x)])"
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PI_ATTN_TREE_TRIES": str(tries)}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "status" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
    seen = [int(v) for v in r.stdout.split("status")[1].split()]
    assert len(seen) == 30 and set(seen) <= {0, 5} and (tries > 0 or set(seen) == {5})
