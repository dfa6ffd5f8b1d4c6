"""Pool settings refuse a NULL pool before they touch a device."""
from rmlx_kv import _lib


def test_wait_limit_of_no_pool():
    assert _lib.lib.rmlx_kv_pool_set_wait_limit(None, 1.0) == _lib.E_BAD_ARG
