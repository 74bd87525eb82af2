"""CPU checks of the cache operators beside tests/test_cache_ops_cpu.py: conversions and refusals
that are made before any device work."""

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16, torch.uint32, torch.uint8])
def test_integers_are_cut_to_their_nearest(dtype):
    from mlx_primitives import _lib
    top, low = (1 << 31) - 1, -(1 << 31)
    values = {torch.int32: [low, -1, 5, top], torch.int64: [1 << 32, (1 << 32) + 5, -(1 << 32) + 1, -1, 7, 1 << 62],
              torch.int16: [-3, 300], torch.uint32: [1, (1 << 32) - 1, 1 << 31], torch.uint8: [0, 255]}[dtype]
    t = torch.tensor(values, dtype=torch.int64).to(dtype)
    was = t.clone()
    got = _lib.int32(t, torch.device("cpu"))
    assert got.dtype is torch.int32 and got.tolist() == [min(max(v, low), top) for v in values]
    assert torch.equal(t, was)


def test_tables_and_lengths_as_the_kernels_read_them():
    from mlx_primitives.cache.paged_append import device_ints
    like = torch.zeros(1)
    one = torch.arange(5, dtype=torch.int32)[None]
    for t in (one, one.repeat(3, 1), torch.arange(24, dtype=torch.int32).view(3, 8)[:, :5], one.expand(1, 5)):
        assert device_ints(t, like) is t
    for t in (one.expand(3, 5), torch.arange(10, dtype=torch.int32).as_strided((3, 5), (2, 1)),
              torch.arange(15, dtype=torch.int32).view(5, 3).T, one[0, :1].expand(4)):
        got = device_ints(t, like)
        assert got.is_contiguous() and torch.equal(got, t)
    with pytest.raises(ValueError, match="integers"):
        device_ints(one.float(), like)
