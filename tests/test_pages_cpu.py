"""Refusals of the paged store that need no GPU, and its structs in the Rust crate."""
import ctypes as C

import pytest

import kivi_cache as K
from test_rust_sys_binding import _c_struct_fields, _rust_struct_fields


def _refused(variant, **kw):
    with pytest.raises(K.KiviError) as e:
        K.PagesConfig(**kw).sizes()
    assert e.value.variant == variant, e.value
    return e.value


def test_sizes():
    assert K.PagesConfig(num_pages=10, page_size=16, num_kv_heads=3, head_dim=96).sizes() == (10 * 16 * 3 * 192, 0)
    assert K.PagesConfig(bits=8, num_pages=2, page_size=256, head_dim=32).sizes() == (2 * 256 * 32, 2 * 256 * 2)
    assert K.PagesConfig(bits=4, num_pages=2, page_size=64, head_dim=128).sizes() == (2 * 64 * 64, 2 * 64 * 2)


def test_config_refusals():
    assert _refused("InvalidBits", bits=2).a == 2
    _refused("InvalidBits", bits=0)
    _refused("InvalidArgument", bits=16, dtype="f32")
    _refused("InvalidArgument", bits=16, dtype="f64")
    assert _refused("ZeroDimension", num_pages=0).name == "num_pages"
    assert _refused("ZeroDimension", num_kv_heads=0).name == "num_kv_heads"
    for page in (0, 8, 24, 100, 512):
        _refused("Unsupported", page_size=page)
    for dim in (0, 16, 80, 160, 256):
        _refused("Unsupported", head_dim=dim)
    _refused("Unsupported", num_pages=1 << 40)
    _refused("Unsupported", num_pages=1 << 20, page_size=256, num_kv_heads=8)


def test_null_arguments():
    L, err = K.lib(), K._Err()
    c = K.PagesConfig()._c()
    h = C.c_void_p()
    for args in ((None, None, None, None), (16, 0, None, None)):
        assert L.kivi_pages_new(C.byref(c), *args, 0, C.byref(h), C.byref(err)) == 101
    assert L.kivi_pages_new(C.byref(c), 24, 16, None, None, 0, C.byref(h), C.byref(err)) == 101
    assert b"aligned" in err.message
    assert L.kivi_pages_new(None, 16, 16, None, None, 0, C.byref(h), C.byref(err)) == 101
    assert L.kivi_pages_new(C.byref(c), 16, 16, None, None, 0, None, C.byref(err)) == 101
    b = K.PagesBatch(0, 16, 16, 1, 1, batch=1, table_width=0)
    assert L.kivi_pages_write_dev(None, b._ref, 2, 16, 16, 128, 128, None, C.byref(err)) == 101
    assert L.kivi_pages_attention_dev(None, b._ref, 2, 16, 1, 128, 128, 1.0, 0, 0, 16, 128, 128, None, None,
                                      C.byref(err)) == 101
    assert L.kivi_pages_status(None, C.byref(err)) == 101
    L.kivi_pages_free(None)


def test_batches_refused_by_the_python_layer():
    torch = pytest.importorskip("torch")
    i32 = dict(dtype=torch.int32)
    table, cu, kv = torch.zeros(2, 4, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32)
    K.PagesBatch(table, cu, kv, 5, 5)
    for bad in ((table.long(), cu, kv), (table, cu.long(), kv), (table, cu, kv.long()), (table, cu[:2], kv),
                (table[:1], cu, kv), (table.T, cu, kv), (table, cu, kv[:, None])):
        with pytest.raises(K.KiviError):
            K.PagesBatch(*bad, 5, 5)
    with pytest.raises(K.KiviError):
        K.PagesBatch(table, cu, kv, -1, 5)
    with pytest.raises(K.KiviError):
        K.PagesBatch(16, 16, 16, 1, 1)


@pytest.fixture
def store():
    """A handle's Python side on device 0, whose entries may not be reached."""
    def entry(*_):
        raise AssertionError("reached the library")

    s = K.KvPages.__new__(K.KvPages)
    s._h, s.device, s.config, s._heads, s._dim = None, 0, None, 2, 64
    s._write = s._read = s._attention = entry
    return s


def test_memory_of_another_place_is_refused(store):
    """CPU tensors and another device's never become pointers that a kernel follows."""
    torch = pytest.importorskip("torch")
    i32 = dict(dtype=torch.int32)
    here = K.PagesBatch(16, 16, 16, 3, 3, batch=2, table_width=4)
    cpu = K.PagesBatch(torch.zeros(2, 4, **i32), torch.zeros(3, **i32), torch.zeros(2, **i32), 3, 3)
    elsewhere = K.PagesBatch(16, 16, 16, 3, 3, batch=2, table_width=4)
    elsewhere.device = 1
    x, q = torch.zeros(3, 2, 64).bfloat16(), torch.zeros(3, 8, 64).bfloat16()
    at = dict(dtype="bf16")
    calls = [lambda: store.write_dev(here, x, x), lambda: store.read_dev(here, x, x),
             lambda: store.attention_dev(here, q, 8, 0.1, 16, **at), lambda: store.attention_dev(here, 16, 8, 0.1, q, **at),
             lambda: store.attention_dev(here, 16, 8, 0.1, 16, d_lse=torch.zeros(3, 8), **at)]
    for b in (cpu, elsewhere):
        calls += [lambda b=b: store.write_dev(b, 16, 16, **at), lambda b=b: store.read_dev(b, 16, 16, **at),
                  lambda b=b: store.attention_dev(b, 16, 8, 0.1, 16, **at)]
    for call in calls:
        with pytest.raises(K.KiviError) as e:
            call()
        assert e.value.variant == "InvalidArgument" and ("CPU" in e.value.message or "device" in e.value.message)
    with pytest.raises(AssertionError):
        store.write_dev(here, 16, 16, **at)


def test_structs_follow_the_header():
    for name in ("kivi_pages_config", "kivi_pages_batch"):
        assert _c_struct_fields(name) == _rust_struct_fields(name), name
        fields = [f for f, _ in {"kivi_pages_config": K.pages._PagesConfig,
                                 "kivi_pages_batch": K.pages._PagesBatch}[name]._fields_]
        assert fields == _c_struct_fields(name)
