"""Calls of the long-context operators that their documentation allows and where they went wrong once, against long_context_oracle or against a call that has to give
the same bits.  Half a step is u = 2^-24 in FP32, 2^-11 in FP16."""
import numpy as np
import pytest

from test_gpu_long_context import Pair, dev, ints, ops, rows, run_attention  # noqa: F401

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
