"""The 4-bit cache without a GPU: slots outside the cache in the plain form, and the largest softmax scales."""
import pytest
import torch

from fdl import kv4, lib, ops


def test_plain_rows_outside_the_cache_are_skipped_and_read_as_zeros():
    """As fdl_kv4_append and fdl_kv4_read take them: padding (-1) and slots past the end."""
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn((5, 2 * 128), generator=gen) for _ in range(2))
    slot = torch.tensor([3, -1, 31, 32, 1 << 40])
    cache, want = ops.kv4_cache(32, 2, "cpu"), ops.kv4_cache(32, 2, "cpu")
    kv4.store_rows(cache, slot, k, v)
    kv4.store_rows(want, slot[[0, 2]], k[[0, 2]], v[[0, 2]])
    assert torch.equal(cache, want)
    for got, ref in zip(kv4.load_rows(cache, slot), kv4.load_rows(want, slot[[0, 2]])):
        assert torch.equal(got[[0, 2]], ref) and ref.abs().sum() > 0
        assert (got[[1, 3, 4]] == 0).all()
    before = cache.clone()
    kv4.store_rows(cache, torch.tensor([-1, 32, -16, 99, 40]), k, v)
    assert torch.equal(cache, before)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_softmax_scales_whose_base_2_form_is_infinite_are_refused(scale):
    p = 0x10000  # never read: the calls end before a launch
    with pytest.raises(lib.FdlError, match="softmax_scale"):
        lib.call("fdl_kv4_attention", p, p, 4, 64, 8, 2, 128, p, 1, 2, 5, p, 1, p, 4, 4, scale, p, 0, None,
                 1, 1, None, 0, None)
    with pytest.raises(lib.FdlError, match="softmax_scale"):
        lib.call("fdl_kv4_verify_attention", p, p, p, p, 64, 64, 4, 2, 128, p, 8, p, 1, None, p, 64, scale, p,
                 1, 1, None, 0, None)
