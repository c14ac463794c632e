"""Tables, lengths and positions of other integer types than int32: what does not fit stays out of range."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_values_that_fit_stay(dtype):
    from hbsattn_b200.paged_cache import _int32
    info = torch.iinfo(dtype)
    x = torch.tensor([0, 1, 100, max(info.min, -2 ** 31), min(info.max, 2 ** 31 - 1)], dtype=dtype)
    y = _int32(x)
    assert y.dtype == torch.int32 and y.tolist() == x.tolist()


def test_values_that_do_not_fit_do_not_wrap():
    from hbsattn_b200.paged_cache import _int32
    x = torch.tensor([2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1, -2 ** 32 + 5, torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max])
    top, bottom = 2 ** 31 - 1, -2 ** 31
    assert _int32(x).tolist() == [top, top, bottom, bottom, bottom, top]
