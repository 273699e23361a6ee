"""What the library asks of its caller for the head's loss."""
from randumb_amd import _lib


def test_workspace_of_a_call_that_keeps_its_logits():
    """Without the piece of logits that a forward call otherwise has in its workspace; where none are kept, what it needs without them."""
    L = _lib.load()
    size = lambda tokens, dim, classes, backward, dtype=_lib.RDB_F32: L.rdb_linear_cross_entropy_workspace_bytes(tokens, dim, classes, dtype, 4096, dim, 4096, dim, backward, 1, 1)  # noqa: E731
    for tokens, dim, classes in ((12, 2048, 47643), (16, 64, 1000), (259, 3136, 96128)):
        kept = 4 * L.rdb_linear_cross_entropy_keeps(tokens, dim, classes, _lib.RDB_F32, dim)
        assert kept == 4 * tokens * classes and size(tokens, dim, classes, 0) - size(tokens, dim, classes, 2) == (kept + 255) // 256 * 256
    for args in ((17, 64, 1000), (2048, 768, 50304)):
        assert size(*args, 0) == size(*args, 2) > 0 and size(*args, 0, _lib.RDB_BF16) == size(*args, 2, _lib.RDB_BF16) > 0
