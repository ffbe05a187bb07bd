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


@pytest.mark.parametrize("dtype,H,K,d,page,kernels", [(torch.bfloat16, 32, 8, 128, 16, {"tc", "decode"}), (torch.bfloat16, 34, 2, 64, 16, {"tc"}), (torch.bfloat16, 8, 2, 64, 256, {"decode"}),
                                                       (torch.bfloat16, 8, 2, 192, 16, set()), (torch.bfloat16, 8, 2, 64, 8, set()), (torch.float32, 32, 8, 128, 16, set())])
def test_jobs_are_the_libraries_that_calls_load(monkeypatch, dtype, H, K, d, page, kernels):
    """What is compiled ahead for a head layout is what its calls ask for, under the same names."""
    asked = {}
    monkeypatch.setattr(ops.build, "load", lambda name, sources, defines=(): asked.__setitem__(name, (list(sources), list(defines))))
    monkeypatch.setattr(ops, "_libraries", {})
    ops._lib("mb_attention_cross")
    for which, supported in (("tc", ops.cross_tc_supported), ("decode", ops.cross_decode_supported)):
        assert supported(dtype, H, K, d, page) == (which in kernels)
        if which in kernels:
            ops._cross_lib(which, d)
    assert {name: (list(sources), list(defines)) for name, (sources, defines) in ops.cross_jobs(dtype, H, K, d, page).items()} == asked
