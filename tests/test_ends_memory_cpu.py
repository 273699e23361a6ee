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


def test_workspace_is_two_pieces_and_copies():
    """Backward: two pieces of G of 512 MB at most (or of 256 classes, the least that there is), fp32 sums of dx, x's copy, the weight's and dW's where their rows are not read or written as they are.
    Forward: 8 bytes for 128 logits, and those copies."""
    L = _lib.load()
    size = lambda dtype, tokens, dim, classes, backward: L.rdb_linear_cross_entropy_workspace_bytes(tokens, dim, classes, dtype, 4096, dim, 4096, dim, backward, 1, 1)  # noqa: E731
    for tokens, dim, classes in ((8192, 256, 50304), (8192, 768, 50304), (4096, 4096, 65536), (4096, 256, 50304), (1025, 999, 10001), (100000, 512, 131072), ((1 << 20) - 37, 16, 769), (5, 64, 1792)):
        wide = (dim + 7) // 8 * 8
        # sums of dx: at most 64 ranges of 16 MB altogether, or 16 where the tokens are that few, or one
        sums = max(16 * tokens * wide * 4 if tokens < 4096 else tokens * wide * 4, 16 << 20)
        copies = tokens * wide * 2 + (2 * classes * wide * 2 if wide != dim else 0) + 32 * tokens + 65536
        piece = min(max(512 << 20, 512 * tokens), 2 * tokens * ((classes + 255) // 256 * 256))
        assert 0 < size(_lib.RDB_BF16, tokens, dim, classes, 1) <= 2 * piece + sums + copies, (tokens, dim, classes)
        parts = 8 * tokens * ((classes + 255) // 256 * 2 if tokens > 64 else 512)
        assert 0 < size(_lib.RDB_BF16, tokens, dim, classes, 0) <= parts + copies, (tokens, dim, classes)
    for tokens, dim, classes in ((2048, 768, 50304), (8192, 768, 50304), (611, 333, 33001)):
        wide = (dim + 7) // 8 * 8
        copies = 6 * (tokens + classes) * wide + 16 * tokens * wide * 4 + 32 * tokens + 65536
        piece = min(512 << 20, 6 * tokens * ((classes + 255) // 256 * 256))
        assert 0 < size(_lib.RDB_F32, tokens, dim, classes, 1) <= 2 * piece + copies, (tokens, dim, classes)
