"""Refusals of the paged operators at the edges of what they allow, which need no GPU."""

from tests.test_paged_host import _L, _params  # noqa: F401


def test_batch_tables_whose_rows_share_memory():
    _lib, L = _L()
    args = [256, 256, 2, 256, 4, 4, 256, 8, 16, 6, 256, 256, 256, 256, 256, None]
    for stride in (3, 1, 0, -3):
        args[4] = stride
        assert L.hyq_paged_batch(*args) == _lib.HYQ_EINVAL, stride
        assert b"share memory" in L.hyq_last_error()


def test_calls_that_no_launch_holds():
    """Refused before the launch: 2^32 threads and more."""
    _lib, L = _L()
    append = [256, 1024, 128, 256, 1024, 128, 0, 256, 1 << 25, 8, 128, 4096, 4096, 32768, 4096, 4096, 4096, 512, 64, 100, 64, None]
    gather = [256, 1 << 25, 8, 128, 4096, 4096, 32768, 4096, 4096, 4096, 512, 64, 100, 64, 0, 256, 256, None]
    for tokens in (1 << 25, 1 << 27, 1 << 40, 1 << 62):
        append[8] = gather[1] = tokens
        assert L.hyq_paged_append(*append) == _lib.HYQ_ENOTSUP and L.hyq_paged_gather(*gather) == _lib.HYQ_ENOTSUP
        assert b"rows" in L.hyq_last_error()
    many = dict(num_requests=1 << 20, num_tokens=1 << 20, kv_repeat=32, kv_heads=8)
    assert L.hyq_paged_attention_workspace_size(_params(_lib, **many)) == 0
    assert L.hyq_paged_attention(_params(_lib, **many), 4096, 1 << 40, None) == _lib.HYQ_ENOTSUP
    assert b"launch" in L.hyq_last_error()
    assert L.hyq_paged_attention_workspace_size(_params(_lib, **{**many, "kv_heads": 4})) > 0
