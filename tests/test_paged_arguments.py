"""Paged caches whose buffers a caller has replaced, and arguments whose strides say nothing: the host's checks, on the CPU."""
import pytest
import torch

from test_paged_cache import E4M3, _cache, _store_args


def _calls(c):
    pages, pos = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    return (lambda: c.store(**_store_args()), lambda: c.load(pos, pages),
            lambda: c.attend(torch.zeros(3, 4, 64, dtype=torch.bfloat16), pos, pages, workspace=torch.zeros(16, dtype=torch.uint8)))


@pytest.mark.parametrize("name,shape", [("v_pages", (6, 16, 2, 64)), ("v_pages", (12, 2, 8, 64)), ("v_pages", (6, 2, 32, 32)), ("k_pages", (6, 16, 2, 64)),
                                        ("k_scale", (6, 16, 2)), ("v_scale", (6, 16, 2)), ("v_scale", (12, 16)), ("k_scale", (192,))])
def test_buffers_of_another_shape_are_refused(name, shape):
    """As many elements in another order: keys, values and scales would be read where they are not."""
    c = _cache(cache_dtype=E4M3)
    setattr(c, name, getattr(c, name).reshape(shape).contiguous())
    for call in _calls(c):
        with pytest.raises(ValueError, match="n_pages, n_heads, page_size"):
            call()


def test_buffers_that_do_not_belong_are_refused():
    c = _cache(cache_dtype=E4M3)
    c.v_scale = None
    for call in _calls(c):
        with pytest.raises(ValueError):
            call()
    c = _cache()
    c.v_scale = torch.zeros(6, 2, 16)
    for call in _calls(c):
        with pytest.raises(ValueError):
            call()
    c = _cache()
    c.k_pages, c.v_pages = (torch.zeros(6, 2, 16 * 64, dtype=torch.bfloat16) for _ in range(2))
    for call in _calls(c):
        with pytest.raises(ValueError):
            call()
