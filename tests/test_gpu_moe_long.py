"""Prompts long enough that a work-group of the experts' down kernel takes several
blocks of 256 columns one after the other: the weights of the next block are on
their way while one is finished, its sums start from zero again and its offsets are
loaded anew. All tokens are compared through their neighbours: a sample in 64 bits,
the others as another order of the same call gives them.

A work-group takes `run` blocks, as many as leave 1536 work-groups; the cases say
how many that are."""
import pytest
import torch

from test_gpu_moe import DEV, Experts, draw_ids, draw_x

pytestmark = pytest.mark.gpu


def _run(hidden, E, entries):
    """Blocks of a work-group (launch_wide in gdn_moe.hip)."""
    blocks, tiles = -(-hidden // 256), entries // 64 + E - E // 2
    run = blocks
    while run > 1 and tiles * -(-blocks // run) < 1536:
        run = (run + 1) // 2
    return run


@pytest.mark.parametrize("hidden,inner,parts,T,k,run", [
    (2048, 128, [4], 12500, 2, 2),      # four runs of two blocks
    (1920, 256, [3, 1], 12500, 2, 2),   # half a block at the end of the last
    (1152, 384, [4], 25000, 2, 3),      # runs of three blocks and of one and a half
    (1280, 512, [5], 25000, 2, 3),      # of three and of two
    (2048, 128, [7, 1], 12500, 8, 8),   # all blocks
    (1664, 128, [8], 13000, 8, 7),      # all of them, the last a half
])
def test_long_prompts_over_several_blocks(gpu, hidden, inner, parts, T, k, run):
    ex = Experts(hidden, inner, parts, seed=hidden + inner)
    assert _run(hidden, ex.E, T * k) == run
    g = torch.Generator().manual_seed(T)
    x, (ids, w) = draw_x(T, T, hidden), draw_ids(T, T, ex.E, k)
    ids[::9, 0] = -1  # some rows of the sum are not there
    out = ex.run(x, ids, w)
    some = torch.randperm(T, generator=g)[:400]
    ref, tol = ex.ref(x[some], ids[some], w[some])
    d = (out[some].double() - ref).abs()
    assert (d <= tol).all(), float((d / tol.clamp_min(1e-30)).max())
    order = torch.randperm(T, generator=g)
    again = ex.run(x[order], ids[order], w[order])
    assert torch.equal(again.view(torch.int16), out[order].view(torch.int16))
    assert out.isfinite().all()
