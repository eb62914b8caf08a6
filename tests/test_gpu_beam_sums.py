"""The log of a row's sum on the GPU, seen by itself: a row's best token has the score cum - log sum, and cum is
chosen so close to log sum that the float it is rounded to hides nothing of the difference."""
import math

import numpy as np
import pytest

from test_gpu_beam import DTYPES, on, run_select, torch_dtype

pytestmark = pytest.mark.gpu


def log_sum_error(rows, dtype, device):
    """log sum as the library has it less the true one, for rows [n, vocab] whose largest value is 0 at token 0.  The
    call has them 1024 / n times, so that a row is one slice and its terms are all taken relative to that 0."""
    import torch
    import radx_amd
    logits = torch.from_numpy(rows).to(torch_dtype(dtype)).to(device)
    n, vocab = rows.shape
    x = logits.double().cpu().numpy()
    assert (x[:, 0] == 0).all() and (x[:, 1:] < 0).all()
    true = np.array([math.log(math.fsum(np.exp(row))) if row.size < 1 << 20 else math.log(np.exp(row).sum()) for row in x])
    cum = true.astype(np.float32)
    sel = radx_amd.BeamSelector(1024, 1, vocab, 1)
    logits = logits.expand(1024, vocab) if n == 1 else logits.repeat(1024 // n, 1)
    scores, parents, tokens = run_select(sel, logits, on(np.tile(cum, 1024 // n)[:, None], device), 1)
    sel.close()
    assert (parents == 0).all() and (tokens == 0).all()
    scores = scores.reshape(1024 // n, n)
    assert (scores == scores[0]).all()
    return x, (cum.astype(np.float64) - scores[0]) - true


def test_sum_of_a_leader_over_a_flat_row(device):
    """The row whose sum hangs most on the exponents' accuracy: far from its largest value, and many.  What is off in the
    same direction in every term stays in the sum.  d is exact here (the largest value is 0).  A term is 2^t by the
    hardware, within one unit in the last place (2^-23), of a t that is d log2 e rounded once.  t lies
    between 18 and 21, so the rounding moves a term by at most 2^-20 ln 2 < 7e-7, and the three additions of eight
    terms by at most 3 * 2^-24 < 2e-7, up as often as down: over 2^24 terms, of which none weighs more than
    8 / 2^24 of the sum beside the leader, the mean of such errors is below 1e-8 (Hoeffding: 2 exp(-2 (1e-8)^2 n / (1.4e-6)^2) with n >
    2^21 is below e^-200; for the eights, with n > 2^18 and twice 2e-7, below e^-300).  All else is done in 64 bits.  A
    factor that is log2 e rounded to a float (1.3e-8 of it) would move the sum by 13 times that."""
    rng = np.random.default_rng(1)
    row = np.empty((1, 1 << 24), np.float32)
    row[0] = -13.5 + 2.0 * (rng.random(1 << 24, dtype=np.float32) - 0.5)
    row[0, 0] = 0.0
    _, off = log_sum_error(row, "f32", device)
    print("off by %.3g" % off[0])
    assert abs(off[0]) <= 2.0 ** -23 + 2e-8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 32000, 131072])
def test_sum_of_rows_of_one_distance(device, dtype, vocab):
    """All terms but the first are the same term: nothing averages out.  t = d log2 e is rounded once (half a unit in
    its last place), the term by the hardware (2^-23), and sums of eight equal terms are exact but for the one with the
    leader in it (3 * 2^-24)."""
    distances = -np.array([0.5, 1.375, 2.75, 4.125, 5.625, 7.0, 8.875, 10.25], np.float32)
    rows = np.repeat(distances[:, None], vocab, 1)
    rows[:, 0] = 0.0
    x, off = log_sum_error(rows, dtype, device)
    t = x[:, 1] / math.log(2.0)
    half_unit = 2.0 ** (np.floor(np.log2(-t)) - 24)
    print("off by", off)
    assert np.all(np.abs(off) <= half_unit * math.log(2.0) * (1 + 2.0 ** -20) + 2.0 ** -23 + 3 * 2.0 ** -24)
