"""What the paged key-value cache refuses, on the CPU: wrong sizes, types and strides, in Python and through the C ABI, and that there is no CPU path."""
import ctypes

import pytest
import torch

E4M3 = torch.float8_e4m3fn


def _cache(**kw):
    from gpt_fast import PagedKVCache
    args = dict(n_pages=6, page_size=16, n_heads=2, head_dim=64, dtype=torch.bfloat16)
    args.update(kw)
    return PagedKVCache(**args)


def test_buffers():
    c = _cache()
    assert c.k_pages.shape == c.v_pages.shape == (6, 2, 16, 64) and c.k_pages.dtype == torch.bfloat16 and c.k_scale is None and c.v_scale is None
    c = _cache(dtype=torch.float16, cache_dtype=E4M3)
    assert c.k_pages.dtype == E4M3 and c.k_scale.shape == (6, 2, 16) and c.k_scale.dtype == torch.float32
    assert set(c.state_dict()) == {"k_pages", "v_pages", "k_scale", "v_scale"}


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(cache_dtype=torch.float16), dict(cache_dtype=torch.float8_e5m2)])
def test_types_that_are_refused(kw):
    with pytest.raises(TypeError):
        _cache(**kw)


@pytest.mark.parametrize("kw", [dict(page_size=0), dict(page_size=12), dict(page_size=8192), dict(head_dim=100), dict(head_dim=264), dict(head_dim=0),
                                dict(n_pages=0), dict(n_heads=0)])
def test_sizes_that_are_refused(kw):
    with pytest.raises(ValueError):
        _cache(**kw)


def _store_args(**kw):
    a = dict(qkv=torch.zeros(3, (4 + 2 * 2) * 64, dtype=torch.bfloat16), table=torch.zeros(50, 32, 2, dtype=torch.bfloat16), input_pos=torch.zeros(3, dtype=torch.int32),
             pages=torch.zeros(3, 2, dtype=torch.int32), n_head=4, sequence=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(qkv=torch.zeros(3, 500, dtype=torch.bfloat16)), dict(qkv=torch.zeros(3, 512, dtype=torch.float16)), dict(qkv=torch.zeros(512, 3, dtype=torch.bfloat16).t()),
    dict(n_head=3), dict(n_head=0), dict(input_pos=torch.zeros(2, dtype=torch.int32)), dict(input_pos=torch.zeros(3)),
    dict(input_pos=torch.zeros(3, 1, dtype=torch.int32)), dict(input_pos=torch.zeros(6, dtype=torch.int32)[::2]), dict(pages=torch.zeros(3, 2, dtype=torch.int64)),
    dict(pages=torch.zeros(3, dtype=torch.int32)), dict(pages=torch.zeros(2, 3, dtype=torch.int32).t()), dict(pages=torch.zeros(2, 2, dtype=torch.int32)),
    dict(pages=torch.zeros(3, 0, dtype=torch.int32)), dict(sequence=torch.zeros(2, dtype=torch.int32)), dict(sequence=torch.zeros(3, dtype=torch.int64)),
    dict(table=torch.zeros(50, 33, 2, dtype=torch.bfloat16)), dict(table=torch.zeros(50, 32, 2, dtype=torch.float16)), dict(table=torch.zeros(50, 64, dtype=torch.bfloat16)),
    dict(table=torch.zeros(50, 0, 2, dtype=torch.bfloat16)), dict(out=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(out=torch.zeros(3, 4, 64))])
def test_store_refuses(kw):
    with pytest.raises(ValueError):
        _cache().store(**_store_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(4, 3, 64, dtype=torch.bfloat16).transpose(0, 1)), dict(q=torch.zeros(3, 0, 64, dtype=torch.bfloat16)), dict(window=-1),
    dict(pages=torch.zeros(4, 2, dtype=torch.int32)), dict(input_pos=torch.zeros(4, dtype=torch.int32)), dict(input_pos=torch.zeros(3, dtype=torch.int16)),
    dict(out=torch.zeros(3, 4, 64)), dict(out=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
    dict(workspace=torch.zeros(16)), dict(window=1 << 62)])
def test_attend_refuses(kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), input_pos=torch.zeros(3, dtype=torch.int32), pages=torch.zeros(3, 2, dtype=torch.int32),
             workspace=torch.zeros(16, dtype=torch.uint8))
    a.update(kw)
    with pytest.raises(ValueError):
        _cache().attend(**a)


@pytest.mark.parametrize("kw", [
    dict(last_pos=torch.zeros(2, dtype=torch.int32)), dict(out=(torch.zeros(3, 2, 32, 64), torch.zeros(3, 2, 32, 64))),
    dict(out=(torch.zeros(3, 2, 32, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 33, 64, dtype=torch.bfloat16))),
    dict(out=(torch.zeros(2, 2, 32, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 32, 64, dtype=torch.bfloat16))),
    dict(out=(torch.zeros(3, 32, 2, 64, dtype=torch.bfloat16).transpose(1, 2),) * 2)])
def test_load_refuses(kw):
    a = dict(last_pos=torch.zeros(3, dtype=torch.int32), pages=torch.zeros(3, 2, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(ValueError):
        _cache().load(**a)


def test_a_cache_that_was_cast_is_refused():
    c = _cache(cache_dtype=E4M3)
    c.k_pages, c.v_pages = c.k_pages.to(torch.bfloat16), c.v_pages.to(torch.bfloat16)
    with pytest.raises(ValueError):
        c.store(**_store_args())
    c = _cache()
    c.k_pages = c.k_pages.to(torch.float16)
    with pytest.raises(ValueError):
        c.store(**_store_args())


def test_no_cpu_path():
    c = _cache(cache_dtype=E4M3)
    for call in (lambda: c.store(**_store_args()), lambda: c.load(torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)),
                 lambda: c.attend(torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32),
                                  workspace=torch.zeros(16, dtype=torch.uint8))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


# The C ABI checks sizes and pointers before it touches a device: addresses that are never read stand in for device memory.
BUF = 1 << 20
ARG, ALIGN, UNSUPPORTED = -1, -2, -3


def _c_store(**kw):
    from gpt_fast import _C
    a = dict(qkv=BUF, rope=BUF, pos=BUF, seq=0, pages=BUF, q=2 * BUF, k=BUF, v=BUF, ks=0, vs=0, stream=0, ld=512, rows=50, pages_ld=2, n_pages=6, tokens=3, dtype=0,
             cache=0, f32=0, rot=64, halves=0, i64=0, n_seq=3, most=2, page=16, n_head=4, n_kv=2, dim=64)
    assert set(kw) <= set(a)
    a.update(kw)
    return _C.lib.lri_rope_paged_store(_C.STORE_CALL.pack(*a.values()))


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), UNSUPPORTED), (dict(cache=1), UNSUPPORTED), (dict(cache=3), ARG), (dict(cache=3, ks=BUF, vs=BUF + 4), ALIGN), (dict(dim=68), UNSUPPORTED),
    (dict(dim=264), UNSUPPORTED), (dict(page=20), UNSUPPORTED), (dict(page=4104), UNSUPPORTED), (dict(n_kv=0), ARG), (dict(n_head=0), ARG), (dict(n_pages=0), UNSUPPORTED),
    (dict(n_pages=1 << 30), UNSUPPORTED), (dict(most=0), ARG), (dict(most=1 << 28, pages_ld=1 << 28), UNSUPPORTED), (dict(pages_ld=1), ARG), (dict(rot=66), ARG),
    (dict(rot=3), ARG), (dict(rot=-2), ARG), (dict(rope=0), ARG), (dict(rows=0), ARG), (dict(tokens=4), ARG), (dict(tokens=-1), ARG), (dict(ld=504), ARG),
    (dict(ld=513), ARG), (dict(qkv=0), ARG), (dict(pos=0), ARG), (dict(q=0), ARG), (dict(k=0), ARG), (dict(v=0), ARG), (dict(pages=0), ARG),
    (dict(qkv=BUF + 8), ALIGN), (dict(q=2 * BUF + 8), ALIGN), (dict(k=BUF + 8), ALIGN), (dict(rope=BUF + 8), ALIGN), (dict(tokens=0, qkv=0), 0), (dict(q=BUF), ARG),
    (dict(q=BUF + 2 * 512 * 2 + 512 * 2 - 16), ARG), (dict(q=BUF - 3 * 256 * 2 + 16), ARG)])
def test_c_store_refuses(kw, status):
    assert _c_store(**kw) == status


def _c_attend(**kw):
    from gpt_fast import _C
    a = dict(q=BUF, k=BUF, v=BUF, ks=0, vs=0, pages=BUF, pos=BUF, out=2 * BUF, ws=BUF, stream=0, n_pages=6, pages_ld=2, window=0, ws_bytes=1 << 30, dtype=0, cache=0, page=16,
             n_seq=3, most=2, i64=0, n_head=4, n_kv=2, dim=64, scale=1.0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _C.lib.lri_paged_attn_decode(_C.ATTN_CALL.pack(*a.values()))


@pytest.mark.parametrize("kw,status", [
    (dict(n_head=3), ARG), (dict(n_head=0), ARG), (dict(window=-1), ARG), (dict(n_seq=-1), ARG), (dict(q=0), ARG), (dict(out=0), ARG), (dict(pos=0), ARG),
    (dict(q=BUF + 8), ALIGN), (dict(out=2 * BUF + 2), ALIGN), (dict(out=BUF), ARG), (dict(out=BUF + 3 * 4 * 64 * 2 - 16), ARG), (dict(dtype=3), UNSUPPORTED), (dict(cache=2), UNSUPPORTED), (dict(cache=3, ks=BUF), ARG),
    (dict(n_seq=0, q=0, out=0), 0)])
def test_c_attend_refuses(kw, status):
    assert _c_attend(**kw) == status


def _c_load(**kw):
    from gpt_fast import _C
    a = dict(k=BUF, v=BUF, ks=0, vs=0, pages=BUF, pos=BUF, k_out=BUF, v_out=2 * BUF, stream=0, n_pages=6, pages_ld=2, rows=32, dtype=0, cache=0, page=16, n_seq=3, most=2, i64=0,
             n_kv=2, dim=64)
    assert set(kw) <= set(a)
    a.update(kw)
    return _C.lib.lri_paged_load(_C.LOAD_CALL.pack(*a.values()))


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), ARG), (dict(rows=1 << 31), ARG), (dict(n_seq=65536), ARG), (dict(pos=0), ARG), (dict(k_out=0), ARG), (dict(v_out=2 * BUF + 8), ALIGN), (dict(v_out=BUF), ARG), (dict(v_out=BUF + 3 * 2 * 32 * 64 * 2 - 16), ARG),
    (dict(n_kv=65536), ARG), (dict(rows=0, k_out=0), 0), (dict(n_seq=0, pos=0), 0)])
def test_c_load_refuses(kw, status):
    assert _c_load(**kw) == status


def test_no_call():
    from gpt_fast import _C
    for f in (_C.lib.lri_rope_paged_store, _C.lib.lri_paged_attn_decode, _C.lib.lri_paged_load):
        assert f(None) == ARG


def test_nothing_to_do():
    """No sequences and no tokens: no launch, whatever the pointers."""
    assert _c_attend(n_seq=0, pages=0, pos=0) == _c_load(n_seq=0, pages=0, k_out=0) == _c_store(tokens=0, n_seq=0, pages=0) == 0


def test_device_messages_name_the_call():
    from gpt_fast import _C
    assert _c_load(rows=-1) < 0 and b"paged_load" in ctypes.string_at(_C.lib.lri_last_error())
