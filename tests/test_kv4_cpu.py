"""The paged 4-bit cache without a GPU: sizes, and what the C entry points refuse on the host before any launch."""
import ctypes as C

import pytest

from vui_b200 import Kv4Cache, _lib


def _cfg(**kw):
    base = dict(n_layers=2, n_heads=16, n_kv_heads=8, head_dim=64, n_blocks=10, block_size=64, max_seqs=4, max_blocks=5)
    base.update(kw)
    return _lib.VuibKv4Config(**base)


def _handle(**kw):
    lib, h = _lib.load(), C.c_void_p()
    assert lib.vuib_kv4_create(C.byref(_cfg(**kw)), C.byref(h)) == 0 and h.value
    return lib, h


def _plan(**kw):
    base = dict(n_seqs=2, n_rows=3, max_new=2, work=4096, cu_rows=4096, row_slot=4096, row_pos=4096, slot_map=4096)
    base.update(kw)
    return C.byref(_lib.VuibKv4Plan(**base))


@pytest.mark.parametrize("bad, status", [
    (dict(head_dim=80), -2), (dict(head_dim=32), -2), (dict(n_kv_heads=0), -2), (dict(n_heads=12), -2), (dict(n_heads=8 * 17), -2),
    (dict(block_size=8), -2), (dict(block_size=48), -2), (dict(block_size=512), -2), (dict(n_layers=0), -3), (dict(n_blocks=0), -3),
    (dict(max_seqs=0), -3), (dict(max_seqs=4097), -3), (dict(max_blocks=0), -3), (dict(max_blocks=1 << 20), -3),
])
def test_create_refuses(bad, status):
    lib, h = _lib.load(), C.c_void_p()
    assert lib.vuib_kv4_create(C.byref(_cfg(**bad)), C.byref(h)) == status and not h.value
    kw = {n: getattr(_cfg(**bad), n) for n, _ in _lib.VuibKv4Config._fields_}
    with pytest.raises(ValueError):
        Kv4Cache(**kw)


@pytest.mark.parametrize("dim, size", [(64, 80), (96, 120), (128, 160)])
def test_pool_bytes(dim, size):
    lib, h = _handle(head_dim=dim)
    n = C.c_size_t()
    assert lib.vuib_kv4_pool_bytes(h, C.byref(n)) == 0
    assert n.value == 2 * 10 * 64 * 8 * size      # layers, blocks, positions, kv heads
    lib.vuib_kv4_destroy(h)


def test_null_and_unbound():
    lib, h = _handle()
    n, p = C.c_size_t(), C.c_void_p(4096)
    assert lib.vuib_kv4_create(None, C.byref(h)) == -1 and lib.vuib_kv4_create(C.byref(_cfg()), None) == -1
    lib, h = _handle()
    assert lib.vuib_kv4_pool_bytes(h, None) == -1 and lib.vuib_kv4_pool_bytes(None, C.byref(n)) == -1
    assert lib.vuib_kv4_reset(h, None) == -4
    assert lib.vuib_kv4_plan(h, _plan(), p, p, None, None) == -4
    assert lib.vuib_kv4_append(h, 0, _plan(), p, 512, p, 512, None) == -4
    assert lib.vuib_kv4_read(h, 0, 1, p, p, p, 512, p, 512, None) == -4
    assert lib.vuib_kv4_attention(h, 0, _plan(), p, 1024, p, 1024, 0.0, None, 0, None) == -4
    assert lib.vuib_kv4_check_flag(h, None) == -4
    assert lib.vuib_kv4_bind(h, None, 0, p, p, p, p, p) == -1
    assert lib.vuib_kv4_bind(h, C.c_void_p(4097), 1 << 30, p, p, p, p, p) == -6
    assert lib.vuib_kv4_bind(h, p, 100, p, p, p, p, p) == -6
    buf = C.create_string_buffer(256)
    assert lib.vuib_kv4_last_error(h, buf, 256) == 0 and b"needed" in buf.value
    for bad, status in ((dict(work=None), -1), (dict(slot_map=None), -1), (dict(n_seqs=0), -3), (dict(n_seqs=5000), -3),
                        (dict(n_rows=-1), -3), (dict(max_new=4), -3), (dict(max_new=-1), -3), (dict(work=4100), -6)):
        assert lib.vuib_kv4_plan(h, _plan(**bad), p, p, None, None) == status
    assert lib.vuib_kv4_plan(h, None, p, p, None, None) == -1
    assert lib.vuib_kv4_launch_count(h) == 0
    assert lib.vuib_kv4_destroy(h) == 0


@pytest.mark.parametrize("name", [n for n, _ in _lib.VuibKv4Config._fields_])
def test_sizes_beyond_32_bits_are_refused(name):
    """Not taken for what 32 bits leave of them."""
    kw = {n: getattr(_cfg(), n) for n, _ in _lib.VuibKv4Config._fields_}
    for more in (2 ** 32, -2 ** 32, 2 ** 40):
        with pytest.raises(ValueError):
            Kv4Cache(**{**kw, name: kw[name] + more})


@pytest.mark.parametrize("device", ["cpu", "cpu:0", "meta"])
def test_other_devices_are_refused(device):
    """With an index they went to the kernels as addresses on the GPU."""
    kw = {n: getattr(_cfg(), n) for n, _ in _lib.VuibKv4Config._fields_}
    with pytest.raises(ValueError, match="CUDA"):
        Kv4Cache(**kw, device=device)
