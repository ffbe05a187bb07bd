"""What the operators of a decoder that reads an encoder's states do without a GPU: they refuse, and the table of axes."""
from types import SimpleNamespace

import pytest
import torch

from marin_b200.kernels import ops


def test_axis_sections():
    assert ops.axis_sections([2, 3, 1]) == [0, 0, 1, 1, 1, 2]
    assert ops.axis_sections([2, 3, 1], spread=True) == [0, 1, 2, 0, 1, 1]
    assert ops.axis_sections([4]) == [0, 0, 0, 0]
    assert ops.axis_sections([0, 2]) == [1, 1]
    for bad in ([], [-1, 2]):
        with pytest.raises(ValueError):
            ops.axis_sections(bad)


def test_there_is_no_cpu_path():
    z = torch.zeros(2, 128)
    i = torch.zeros(2, dtype=torch.int32)
    cache = torch.zeros(1, 1, 16, 64)
    ctx = SimpleNamespace(num_requests=1, num_decode=0, max_query_len=2, cu_tokens=i)
    with pytest.raises(ops.KernelError):
        ops.attention_cross(z, cache, cache, z.clone(), ctx, ops.Source(i[None], i, 1), 2, 1, 64, 1.0)
    with pytest.raises(ops.KernelError):
        ops.qk_norm_axes_write(torch.zeros(2, 256), z, None, None, 1e-6, i[None], torch.zeros(32, dtype=torch.int32), torch.zeros(32), 64, False, i, cache, cache, 2, 1, 64)
    with pytest.raises(ops.KernelError):
        ops.page_step(i, i, i[None], i, i[:1], 16, i.clone(), i, i, i, i)
