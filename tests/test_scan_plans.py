"""The selective scan where its backward pass cuts a sequence into workgroups of several segments, as it does for the largest
training batches: indexes of segments and workgroups, a last workgroup with fewer segments, segments of more than 16 steps, and the
gradients of initial and final states across them.  Tolerances as in test_gpu_state_space.py."""
import ctypes

import pytest
import torch

import plain_operators as plain
from rnnt_amd import _lib
from test_gpu_state_space import DEV, U, call_scan, lens_for, scan_inputs

# (sequences, steps, channels, states): segments of a sequence, workgroups of a sequence in the backward pass
PLANS = {
    (1500, 90, 3, 8): (3, 2),         # two segments and one
    (1500, 90, 3, 32): (3, 2),
    (1500, 200, 3, 16): (7, 3),       # three, three and one
    (700, 90, 65, 8): (3, 2),         # two groups of channels
    (256, 1500, 2, 16): (32, 16),     # segments of 48 steps
    (128, 300, 3, 16): (10, 10),      # segments of 32 steps, a workgroup each
    (16, 1500, 1024, 16): (32, 16),   # (the shape that these stand for)
}


def plan_of(B, L, D, N):
    """Segments and workgroups per sequence, from the sizes of the workspaces that hold their states and partial sums."""
    lib, n = _lib.load(), ctypes.c_size_t(0)
    round16 = lambda v: (v + 15) & ~15  # noqa: E731

    def size(backward):
        assert lib.rnnt_selective_scan_workspace_size(B, L, D, N, backward, ctypes.byref(n)) == 0
        return n.value

    rows = round16((B * ((L + 15) // 16 * 16) + 1) * 2 * N * 4)
    states = lambda s: 0 if s == 1 else round16(B * s * N * D * 4) + round16(B * s * D * 4)  # noqa: E731
    bc = round16(B * L * ((D + 63) // 64) * 2 * N * 4)
    parts = lambda k: round16(B * k * D * N * 4) + round16(B * k * 2 * D * 4)  # noqa: E731
    most = (L + 15) // 16
    segments, = [s for s in range(1, most + 1) if rows + states(s) == size(0)]
    blocks, = [k for k in range(1, most + 1) if states(segments) + bc + parts(k) == size(1)]
    return segments, blocks


@pytest.mark.parametrize("shape", PLANS)
def test_these_shapes_are_cut_like_that(shape):
    """A retuned plan has to bring other shapes here, with several segments to a workgroup."""
    assert plan_of(*shape) == PLANS[shape]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((1500, 90, 3, 8), torch.float32), ((1500, 90, 3, 32), torch.bfloat16),
                                         ((1500, 200, 3, 16), torch.float32), ((1500, 200, 3, 16), torch.float16),
                                         ((700, 90, 65, 8), torch.float32), ((256, 1500, 2, 16), torch.bfloat16),
                                         ((256, 1500, 2, 16), torch.float32), ((128, 300, 3, 16), torch.float32)])
def test_scan_of_a_large_batch(shape, dtype):
    """Some sequences of every length of the batch against the 64-bit form.  The others get no gradient, so that the parameters' is
    the sum over the chosen ones; with a gradient each, the chosen ones' results are the same bits."""
    B, L, D, N = shape
    a, grads = scan_inputs(B, L, D, N, dtype, seed=L)
    lens = lens_for(True, B, L)
    chosen = sorted({0, 1, 2, 3, B // 2 // 6 * 6 + 4, B // 2 // 6 * 6 + 5, B - 1, (B - 1) // 6 * 6})
    rest = torch.ones(B, dtype=torch.bool)
    rest[chosen] = False
    ref_in = {k: v[chosen].double() if k in ("x", "dt", "B", "C", "z", "init") else v.double() for k, v in a.items()}
    ref_g = {k: v[chosen].double() for k, v in grads.items()}
    past = torch.arange(L)[None] >= lens[:, None]
    for k in ("x", "dt", "z", "B", "C"):
        a[k][past] = float("nan")
    grads["gy"][past] = float("nan")
    only = {k: v.clone() for k, v in grads.items()}
    for v in only.values():
        v[rest] = 0
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    y, state = call_scan(dev, lens)
    leaves = list(dev.values())
    got, every = (dict(zip(dev, torch.autograd.grad([y, state], leaves, [g["gy"].to(DEV), g["gfinal"].to(DEV)], retain_graph=True)))
                  for g in (only, grads))
    lens_l = lens[chosen].tolist()
    ref, mag = (plain.scan(**ref_in, lens=lens_l, **ref_g, magnitude=m) for m in (False, True))
    fwd, bwd = 8 * (L + 1) + N + 32, 16 * (L + 1) + N + 64
    plain.assert_within(y[chosen], ref["y"], fwd * U * mag["y"] + plain.spacing(ref["y"], dtype), "y")
    plain.assert_within(state[chosen], ref["state"], fwd * U * mag["state"] + 1e-40, "state")
    for k, g in got.items():
        n = {"B": D, "C": D}.get(k, len(chosen) * L if k in ("A", "D", "bias") else 0)
        t = torch.float32 if k in ("A", "D", "bias", "init") else dtype
        part = g
        if k not in ("A", "D", "bias"):
            part = g[chosen]
            assert torch.count_nonzero(g[rest.to(DEV)]) == 0 and torch.equal(part, every[k][chosen]), k
        plain.assert_within(part, ref["d" + k], (bwd + n) * U * mag["d" + k] + plain.spacing(ref["d" + k], t), "d" + k)
