"""The operators of a decoder that reads an encoder's states, on the paths that only longer or larger calls take; against the same definitions in 64 bits and
with the same tolerances as in ``test_source_operators_gpu.py``.
"""
import pytest
import torch

from test_source_operators_gpu import DEV, DTYPES, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from marin_b200.kernels import ops as o
    return o


def most_of(values):
    return max([float(v.abs().max()) for v in values if v.numel()] or [1.0])


def climbing(dtype, new, src, step):
    """Scores that move by `step` (a power of two) from every 64 positions to the next: the maximum moves with every block of keys, or never does."""
    case = Case(dtype, 8, 2, 64, 16, new, src, seed=len(src))
    case.q[:, :] = 1.0
    for r, s in enumerate(src):
        at = torch.arange(s, device=DEV)
        case.keys[r] = (0.125 * torch.randn(s, 2, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(r)) + step / 8 * (at // 64)[:, None, None]).to(dtype).double()
        for j in range(-(-s // 16)):
            rows = case.keys[r][16 * j:16 * j + 16]
            case.k[int(case.table[r, j]), :, :rows.shape[0]] = rows.to(dtype).transpose(0, 1)
    return case


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [8.0, -8.0, 0.0])
def test_cross_scores_that_move_with_every_block(ops, dtype, step):
    """Portions of one to fourteen blocks of keys, cut over a cluster (one request) and not (many): every product of weights and values is waited for, whether or not what
    is added up has to be scaled in between.  A score is a sum of 64 terms and ends at 8 * 13 at most: its additions (33 one after the other, in pairs) are off by 2^-24 of what
    they have by then, half of that on average, 33 * 52 * 2^-24 = 1.1e-4 in all, and a product and the exponent's own rounding add 2e-5.  Weights that are off by 1.3e-4 of
    themselves move a mean of values by twice that times the largest value.  bfloat16 adds the rounding of weights and results, 2^-8 each."""
    for src in ([64], [129], [190], [257], [320], [835]):
        for many in (1, 40):
            case = climbing(dtype, [33] * many, src * many, step)
            first = case.run(ops).clone()
            atol = most_of(case.values) * (2 * 1.3e-4 + (0 if dtype == torch.float32 else 2 * 2.0 ** -8))
            torch.testing.assert_close(first.double(), case.want(), rtol=0, atol=atol)
            case.out.zero_()
            assert torch.equal(case.run(ops), first)
    ops.check_device_errors()
