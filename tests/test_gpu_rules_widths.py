"""GPU tests of decoding rules on rows at the borders of a workgroup's forms: 512 or 1024 threads to a row, a row to a workgroup or
shared out; the maximum in every part of the row."""
import pytest
import torch

import plain_operators as plain
from test_gpu_rules import check, make, rules_of, DEV

pytestmark = pytest.mark.gpu
# a row of V logits has V / E + 1 pieces of E (4 fp32, 8 16-bit): above 1536 of them 1024 threads take up to 256 rows, and
# rows of more than 16384 - (E - 1) logits are shared out
E = {torch.float32: 4, torch.bfloat16: 8, torch.float16: 8}


def widths(dtype):
    e = E[dtype]
    return [1536 * e - 1, 1536 * e, 8000 * e // 4, 16384 - (e - 1), 16384 - (e - 1) + 1]


CASES = [(dtype, V) for dtype in plain.TYPES for V in widths(dtype)]


@pytest.mark.parametrize("dtype,V", CASES)
def test_against_the_formula(dtype, V):
    for contexts, window in ((1, 1), (2, 3)):            # (an odd V puts the rows off 16 bytes)
        x, r = make(contexts, window, V, 300, dtype, seed=V)
        check(x, r)


@pytest.mark.parametrize("dtype,V", CASES)
def test_the_maximum_in_every_part_of_the_row(dtype, V):
    """One row for every 512th column, the last columns, and a tie of two columns that different waves read: the lower index."""
    import rnnt_amd

    at = sorted({*range(0, V, 512), V - 1, V - 2, V - E[dtype] - 1})
    x, r = make(1, len(at) + 1, V, 200, dtype, seed=1)
    r["history"].clamp_(max=V - 600)                      # (penalised tokens away from the end, and none of the maxima)
    r["history"][torch.isin(r["history"], torch.tensor(at, dtype=torch.int32))] = -1
    r["allowed"][:, at], r["bias"][:, at] = True, 0.0
    x[torch.arange(len(at)), at] = 60.0
    x[-1, at[1:]] = 60.0
    token, logp = rnnt_amd.row_max_logp(x.to(DEV), rules_of(r))
    assert token.tolist() == at + at[1:2]
    check(x, r)


@pytest.mark.parametrize("dtype", plain.TYPES)
def test_rows_above_and_below_the_border_of_threads_agree(dtype):
    """257 rows take 512 threads each, the first 256 of them alone 1024: the same tokens, scores within both sides' rounding."""
    import rnnt_amd

    V = 1600 * E[dtype] + 1
    x, r = make(1, 257, V, 100, dtype, seed=2)
    x, rules = x.to(DEV), rules_of(r)
    many, few = rnnt_amd.row_max_logp(x, rules), rnnt_amd.row_max_logp(x[:256], rules)
    assert torch.equal(many[0][:256], few[0])
    # as in test_gpu_rules: V / 256 additions in a lane and 48 u each side, of sums whose logarithm is a few units
    bound = 2 * (48 + V / 256) * plain.U + 4 * plain.U * few[1].abs()
    assert bool(((many[1][:256] - few[1]).abs() <= bound).all())
