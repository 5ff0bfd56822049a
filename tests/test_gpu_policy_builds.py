"""The builds of the policy operators' kernels that small sizes do not take: the feed-forward's larger tiles, several tiles
and several trips a workgroup, long windows whose rows are on no grid, windows without gradients. Tolerances as in
test_gpu_policy."""
import pytest
import torch

import isaac_net_amd as P
from test_gpu_policy import DEV, DT, check_delta, check_norm, close, delta_inputs, ffn_both

pytestmark = pytest.mark.gpu


def tiles(n, t):
    return -(-n // t)


def tile_of(rows, cols):
    """The feed-forward's rule: the largest tile of which a product has one for each of the 256 compute units."""
    return next((t for t in (256, 128) if tiles(rows, t) * tiles(cols, t) >= 256), 64)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("N,D,F,act,gates,dx", [
    (4099, 72, 4104, "silu", 256, 64), (4100, 77, 4101, "relu", 256, 64), (4096, 64, 4096, "gelu", 256, 64),
    (2051, 136, 1032, "gelu", 128, 64), (2048, 128, 1024, "silu", 128, 64), (2050, 65, 1031, "relu", 128, 64),
    (4099, 4104, 72, "silu", 64, 256), (2051, 2064, 136, "gelu", 64, 128), (2051, 2059, 133, "relu", 64, 128),
    (1000, 1032, 1032, "silu", 64, 64), (8200, 512, 1000, "silu", 256, 128)])
def test_ffn_tiles(dt, N, D, F, act, gates, dx):
    """Both projections (2 F columns) and dx (D) by each tile, whole and ragged in every direction, with one step along the
    sum and with several, and with more tiles than compute units; those of the weights by 256 where they have 16 such tiles."""
    assert (tile_of(N, 2 * F), tile_of(N, D + -D % 8)) == (gates, dx)
    a, b = ffn_both(N, D, F, DT[dt], act)
    close("y", a[0], b[0], D)
    for n, x, y, terms in zip(("dx", "dw_gate", "dw_up"), a[1:], b[1:], (F + D, N + D, N + D)):
        close(n, x, y, terms, roundings=3)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,D", [(9001, 64), (9001, 200), (9001, 500), (17001, 512), (2100, 1000), (2100, 1032), (2100, 1071),
                                 (1100, 1536), (1100, 2048), (700, 4000), (600, 8192)])
def test_norm_of_several_rows_a_lane_group(dt, N, D):
    check_norm(N, D, DT[dt])


@pytest.mark.parametrize("gate", ["row", None])
def test_norm_gates_of_several_rows_a_lane_group(gate):
    check_norm(9001, 333, torch.bfloat16, gate=gate)


@pytest.mark.parametrize("B,T,Hk,H,K,V", [(1, 600, 1, 2, 33, 65), (2, 577, 1, 1, 7, 13), (1, 530, 2, 4, 128, 127)])
def test_long_windows_of_rows_on_no_grid(B, T, Hk, H, K, V):
    check_delta(*delta_inputs(B, T, Hk, H, K, V, torch.bfloat16, seed=40, end=0.02))


@pytest.mark.parametrize("dt,B,T", [("f32", 3, 20), ("f32", 60, 90), ("f16", 2, 200), ("bf16", 2, 200), ("bf16", 2, 600)])
def test_window_without_gradients(dt, B, T):
    ins, reset, _, _ = delta_inputs(B, T, 1, 2, 40, 72, DT[dt], seed=41, end=0.02)
    x = [t.to(DEV) for t in ins]
    alone = P.delta_rule(*x, reset=reset.to(DEV))
    trained = P.delta_rule(*(t.requires_grad_(True) for t in x), reset=reset.to(DEV))
    for a, b in zip(alone, trained):
        assert not a.requires_grad and torch.equal(a, b)
