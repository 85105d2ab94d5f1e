"""Messages of the C ABI's errors name every reason for them."""
from simplical_attn_amd import _lib


def test_a_cache_too_large_for_trees():
    lib = _lib.load()
    message = lib.sa2_strerror(-13)
    assert b"at least 1" in message and b"2^31 - 64" in message
