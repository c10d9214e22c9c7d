"""Copies of pages and what goes with them on the host: pools that change between two copies."""

import struct

import pytest
import torch

from test_host_long_lived import FP8, config

from minillm.cache.paged import PagedKVCache


def make_cache():
    return PagedKVCache(config(), 8, "cpu", FP8, block_scales=True)


def shorter(cache):
    cache.k[0] = cache.k[0][:4]


def transposed(cache):
    cache.k[1] = cache.k[1].transpose(1, 2)


def strided(cache):
    cache.v[0] = cache.v[0].as_strided(cache.v[0].shape, (0, *cache.v[0].stride()[1:]))


def of_half_the_bytes(cache):  # the same shape, in the first half of the memory
    like = cache.k[0]
    cache.k[0] = like.view(torch.uint8).flatten()[:like.numel() // 2].view(8, 8, 2, 128)[:4]


def shorter_in_place(cache):
    cache.k[0].data = cache.k[0].data[:4]


def transposed_in_place(cache):
    cache.v[1].transpose_(0, 1)


def shorter_scales(cache):
    cache.v_scale[1] = cache.v_scale[1][:5]


@pytest.mark.parametrize("change", [shorter, transposed, strided, of_half_the_bytes, shorter_in_place, transposed_in_place,
                                    shorter_scales], ids=lambda f: f.__name__)
def test_a_pool_that_changed_at_its_address_is_checked_again(change):
    cache = make_cache()
    cache.check_pages()
    cache.copy_blocks([1], [2])
    change(cache)
    with pytest.raises(ValueError, match="contiguous, of 8 blocks"):
        cache.check_pages()
    with pytest.raises(ValueError, match="contiguous, of 8 blocks"):
        cache.copy_blocks([1], [2])


def test_pages_of_a_pool_in_fewer_bytes_are_packed_again():
    # a pool of another element type where the old one lay: its pages are as long as its own elements make them
    cache = make_cache()
    before = cache._page_tensors()
    cache.k[0] = cache.k[0].view(torch.uint8).flatten()[:8 * 8 * 2 * 128].view(8, 8, 2, 128)
    after = cache._page_tensors()
    sizes = [struct.unpack(f"{x[2]}q", x[1]) for x in (before, after)]
    assert sizes[0][0] == 16 * 2 * 128 and sizes[1][0] == 8 * 2 * 128 and sizes[0][1:] == sizes[1][1:]
    assert struct.unpack("Q", after[0][:8]) == struct.unpack("Q", before[0][:8])


def test_the_number_of_blocks_counts():
    cache = make_cache()
    cache.check_pages()
    cache.num_blocks = 16
    with pytest.raises(ValueError, match="of 16 blocks"):
        cache.check_pages()


def test_pages_the_library_refuses_are_refused_by_the_check(monkeypatch):
    # the library's limit and the check's are one; the check applies it to pools on a GPU
    from minillm import _native
    from minillm.cache import paged

    def copy(nbytes):
        _native.lib().call("mllm_copy_pages", struct.pack("Q", 1 << 20), struct.pack("q", nbytes), 1, 4, struct.pack("q", 0),
                           struct.pack("q", 9), 1, None)

    with pytest.raises(ValueError, match="block 9 is outside"):
        copy(paged.MAX_PAGE_BYTES)
    with pytest.raises(ValueError, match="page too large"):
        copy(paged.MAX_PAGE_BYTES + 1)
    cache = make_cache()
    monkeypatch.setattr(paged, "MAX_PAGE_BYTES", 16 * 2 * 128 - 1)
    cache.check_pages()  # on the host: any size

    class OnGpu(torch.Tensor):
        is_cuda = True

    cache = make_cache()
    cache.k[0] = cache.k[0].as_subclass(OnGpu)
    for call in (cache.check_pages, lambda: cache.copy_blocks([1], [2])):
        with pytest.raises(ValueError, match="too large to copy"):
            call()
    monkeypatch.setattr(paged, "MAX_PAGE_BYTES", 16 * 2 * 128)
    cache.check_pages()
