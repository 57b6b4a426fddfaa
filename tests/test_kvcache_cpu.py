"""CPU: argument checks of the paged key/value cache's C ABI that come before any GPU work."""
import ctypes as C

import pytest

from veckern_b200 import _native as N


def desc(**kw):
    d = N.KvDesc(device=0, dtype=N.VK_KV_BF16, page_size=16, kv_heads=2, head_dim=64, pages=4, k=4096,
                 k_stride=(C.c_int64 * 3)(2048, 128, 64), v=8192, v_stride=(C.c_int64 * 3)(2048, 128, 64))
    for name, x in kw.items():
        setattr(d, name, x)
    return d


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=7), "dtype"), (dict(page_size=12), "page_size"), (dict(page_size=4), "page_size"),
    (dict(page_size=2048), "page_size"), (dict(head_dim=4), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(head_dim=60), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"), (dict(k=None), "k must"),
    (dict(v=8200), "v must"), (dict(k_stride=(C.c_int64 * 3)(2048, 127, 64)), "k: strides"),
    (dict(v_stride=(C.c_int64 * 3)(-8, 128, 64)), "v: strides")])
def test_create_refuses(kw, msg):
    h = C.c_void_p()
    assert N.lib().vk_kv_create(C.byref(desc(**kw)), C.byref(h)) == N.VK_ERR_INVALID
    assert msg in N.last_error() and not h.value


def test_null_handles_are_refused():
    lib = N.lib()
    bt, at, ev = N.KvBatch(), N.KvAttend(), N.KvEvict()
    s = (C.c_int64 * 2)(64, 64)
    assert lib.vk_kv_create(None, None) == N.VK_ERR_INVALID
    assert lib.vk_kv_append(None, C.byref(bt), None, s, None, s, None) == N.VK_ERR_INVALID
    assert lib.vk_kv_attend(None, C.byref(bt), C.byref(at), None) == N.VK_ERR_INVALID
    assert lib.vk_kv_evict(None, C.byref(bt), C.byref(ev), None) == N.VK_ERR_INVALID
    assert lib.vk_kv_sync(None, None) == N.VK_ERR_INVALID
    assert lib.vk_kv_destroy(None) == N.VK_OK
