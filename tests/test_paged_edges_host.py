"""Refusals of the paged operators at the edges of what they allow, which need no GPU."""

from tests.test_paged_host import _L, _params  # noqa: F401


def test_batch_tables_whose_rows_share_memory():
    _lib, L = _L()
    args = [256, 256, 2, 256, 4, 4, 256, 8, 16, 6, 256, 256, 256, 256, 256, None]
    for stride in (3, 1, 0, -3):
        args[4] = stride
        assert L.hyq_paged_batch(*args) == _lib.HYQ_EINVAL, stride
        assert b"share memory" in L.hyq_last_error()
