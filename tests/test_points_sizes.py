"""Which sizes the attention to another sequence takes, as its workspace functions say without a GPU: what its grids and indexes hold, and no less."""
import ctypes as C
import os

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nnv_amd", "libnnvhip.so")
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built (python -m nnv_amd.build)")


def workspaces(**kw):
    """(bytes of the forward pass, of the backward pass); None where the sizes are refused."""
    from nnv_amd import _lib, points
    lib = _lib.load()
    s = dict(type=1, batch=1, queries=1, keys=64, heads=1, kv_heads=1, head=128)
    s.update(kw)
    d, found = points._ATTENTION.pack(*s.values(), 0.125, *[0] * 25), []
    for fn in (lib.nnvhip_cross_attention_workspace, lib.nnvhip_cross_attention_backward_workspace):
        n = C.c_int64()
        try:
            _lib.check(fn(d, C.byref(n)))
            found.append(n.value)
        except ValueError as e:
            assert "too many" in str(e)
            found.append(None)
    return tuple(found)


@pytest.mark.parametrize("type", [0, 1, 2])
def test_many_keys_for_few_rows(type):
    for kw in (dict(batch=64, heads=64, kv_heads=8, keys=65536), dict(batch=256, heads=64, keys=32768), dict(batch=8, heads=64, kv_heads=8, keys=1 << 20),
               dict(heads=8, keys=1 << 26), dict(batch=64, heads=64, kv_heads=64, keys=65536), dict(batch=4096, heads=32, keys=64)):
        forward, backward = workspaces(type=type, **kw)
        rows = kw.get("batch", 1) * kw["heads"]
        assert forward is not None and forward <= 256 * rows * 129 * 4
        assert backward is not None and backward >= 4 * rows


def test_what_grids_and_indexes_do_not_hold():
    for kw in (dict(keys=1 << 31), dict(queries=1 << 31), dict(queries=1 << 30, heads=2), dict(batch=65536), dict(heads=65536),
               dict(batch=65535, heads=65535, kv_heads=65535), dict(batch=65535, queries=1 << 20),
               dict(batch=65535, heads=65535, kv_heads=65535, queries=(1 << 31) - 256, keys=(1 << 31) - 256)):
        assert workspaces(**kw) == (None, None), kw
    # only the backward pass has a block for every tile of keys, and sixteen rows a block
    for kw in (dict(keys=(1 << 31) - 256), dict(batch=4096, keys=1 << 20), dict(batch=65535, queries=1024, heads=8),
               dict(batch=65535, heads=128, kv_heads=128, queries=0, keys=(1 << 31) - 256)):
        forward, backward = workspaces(**kw)
        assert forward is not None and backward is None, kw


def test_rows_of_layer_norm_that_a_grid_does_not_hold():
    """Rows beyond a block's registers take a block of 512 threads each."""
    from nnv_amd import _lib
    lib, n = _lib.load(), C.c_int64()
    for rows, size in (((1 << 23) - 1, 8193), (1 << 30, 8192), ((1 << 31) - 1, 64)):
        _lib.check(lib.nnvhip_layer_norm_backward_workspace(1, rows, size, C.byref(n)))
        assert n.value > 0
    for rows, size in ((1 << 23, 8193), (1 << 31, 64)):
        with pytest.raises(ValueError, match="too many rows"):
            _lib.check(lib.nnvhip_layer_norm_backward_workspace(1, rows, size, C.byref(n)))
