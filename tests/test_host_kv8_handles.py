"""The binding's 8-bit KV cache objects and argument checks, on CPU tensors: nothing here
reaches the device."""
import pytest
import torch

import logicaffeine_amd as lgx


def cache(pages=4, hkv=2, d=64):
    return lgx.KvCacheI8(torch.zeros((pages, hkv, 16, d), dtype=torch.int8), torch.zeros((pages, hkv, d, 16), dtype=torch.int8),
                         torch.zeros((pages, hkv)), torch.zeros((pages, hkv)))


def context():
    """The binding's checks run ahead of the library's, which would refuse this handle."""
    c = lgx.Context.__new__(lgx.Context)
    c.torch, c.dev, c.handle = torch, torch.device("cpu"), None
    return c


@pytest.mark.parametrize("make,name", [
    (cache, "k"), (cache, "v"), (cache, "k_scale"), (cache, "v_scale"), (cache, "num_pages"), (cache, "hkv"), (cache, "d"),
    (lambda: lgx.Rope(torch.ones((9, 32)), torch.zeros((9, 32))), "cos"),
    (lambda: lgx.Rope(torch.ones((9, 32)), torch.zeros((9, 32))), "sin"),
    (lambda: lgx.AttnOpts(slopes=torch.ones(4)), "slopes"), (lgx.AttnOpts, "window"), (lgx.AttnOpts, "softcap"),
    (lgx.AttnOpts, "scale")])
def test_a_handle_refuses_what_it_could_not_take_over(make, name):
    """The calls use the addresses and numbers of the construction: another tensor or
    number put in later would be ignored, and its memory not kept alive."""
    x = make()
    before = getattr(x, name, None)
    with pytest.raises(AttributeError):
        setattr(x, name, torch.ones(4))
    with pytest.raises(AttributeError):
        delattr(x, name)
    assert getattr(x, name, None) is before
    if isinstance(before, torch.Tensor):
        before.fill_(1)                              # the contents stay the caller's
        assert bool((getattr(x, name) == 1).all())


@pytest.mark.parametrize("shape", [(2,), (2, 4, 1), (2, 4, 0), (2, 4, 3)])
def test_a_page_table_is_a_matrix(shape):
    c, kv = context(), cache()
    q, lens, table = torch.zeros((2, 4, 64)), torch.ones(2, dtype=torch.int32), torch.zeros(shape, dtype=torch.int32)
    for call in (lambda: c.gqa_decode_attn_i8(q, kv, table, lens, 64), lambda: c.gqa_prefill_attn_i8(q, kv, table, lens, 1, 64),
                 lambda: c.rope_kv_append_i8(torch.zeros((2, 512)), None, lgx.Rope(torch.ones((9, 32)), torch.zeros((9, 32))), lens,
                                             table, kv),
                 lambda: c.kv_read_i8(kv, table, lens, 3)):
        with pytest.raises(ValueError):
            call()
