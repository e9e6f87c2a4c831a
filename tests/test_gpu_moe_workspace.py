"""What a call of the experts asks of its caller's memory."""
import pytest
import torch

import gdn_amd
from test_gpu_moe import BF, DEV, Experts

pytestmark = pytest.mark.gpu


def _layer(hidden, inner, E):
    def mat(n, k):
        return (torch.zeros(E, n, k // 8, device=DEV, dtype=torch.int32),
                torch.zeros(E, n, k // 64, device=DEV, dtype=BF),
                torch.zeros(E, n, k // 64, device=DEV, dtype=BF))
    return gdn_amd.MoE(hidden, inner, [(mat(inner, hidden), mat(inner, hidden), mat(hidden, inner))])


@pytest.mark.parametrize("hidden,inner,E,T,k", [(2048, 512, 257, 16384, 9), (1024, 256, 8, 30000, 2),
                                                (512, 128, 4, 100000, 2)])
def test_long_prompts_reserve_rows_as_they_are_kept(gpu, hidden, inner, E, T, k):
    """Rows between down and the sum are f16 there: two bytes a number, h two, and per row
    the sums' parts and some words. Per token the sums' parts and the maxima of x."""
    row = 2 * hidden + 2 * inner + 6 * max(8, inner // 64) + 64
    token = 6 * max(8, hidden // 64) + 32
    # the largest call that keeps f32 rows is small beside it
    assert _layer(hidden, inner, E).workspace_bytes(T, k) <= 1.1 * (T * k * row + T * token) + (1 << 22)


def test_workspaces_grow_with_the_call_where_the_rows_change(gpu):
    for hidden, inner, E in ((2048, 512, 3), (256, 128, 40), (128, 640, 5), (128, 128, 1)):
        moe, last = _layer(hidden, inner, E), 0
        for n in list(range(1, 200)) + list(range(200, 40000, 61)):
            b = moe.workspace_bytes(n, 1)
            assert b >= last, n
            last = b


@pytest.mark.parametrize("hidden,E", [(2048, 4), (256, 4), (128, 40)])
def test_calls_next_to_where_the_rows_change(gpu, hidden, E):
    """The last call with f32 rows and the first with f16 ones, in memory of exactly the
    size that was asked for, with guards behind it."""
    blocks = -(-hidden // 256)
    first = max(32 * E, 64 * (-(-384 // blocks) - E + E // 2))
    ex = Experts(hidden, 128, [E], seed=3)
    g = torch.Generator().manual_seed(1)
    for T in (first - 1, first):
        x = torch.randn(T, hidden, generator=g).to(BF)
        ids = torch.randint(0, E, (T, 1), generator=g, dtype=torch.int32)
        w = torch.rand(T, 1, generator=g)
        n = ex.moe.workspace_bytes(T, 1)
        mem = torch.full((n + 4096,), 165, device=DEV, dtype=torch.uint8)
        out = torch.empty(T, hidden, device=DEV, dtype=BF)
        ex.moe.forward(x.to(DEV), ids.to(DEV), w.to(DEV), out, mem[:n])
        assert (mem[n:] == 165).all()
        some = torch.randperm(T, generator=g)[:200]
        ref, tol = ex.ref(x[some], ids[some], w[some])
        assert ((out.cpu()[some].double() - ref).abs() <= tol).all()
