"""Operands that share memory with what a call writes are refused by their addresses alone (no GPU)."""
import axon_b200 as ax

AT = 1 << 20  # addresses that nothing looks behind


def _refused(status):
    """Whether a call was refused for an overlap; without a GPU every other one ends at its first pointer."""
    return status == ax.Status.ERR_INVALID and b"must not overlap" in ax.lib().axq_last_error()


def test_quantize_f8_padding():
    """The bytes between cols and ld in the last block of 128 columns are set to 0, those of the last row too."""
    L = ax.lib()

    def call(codes, scales, src=AT, rows=1, cols=4, ld=16, block_rows=1):
        return _refused(L.axq_quantize_f8(0, src, codes, ld, scales, rows, cols, block_rows, None))

    c = 2 * AT
    assert call(c, c + 4) and call(c, c + 12) and not call(c, c + 16)
    assert call(c, c + 32 + 8, rows=3) and not call(c, c + 48, rows=3)
    # a row stride beyond the block: what lies behind it is left as it is
    assert call(c, c + 124, ld=256) and not call(c, c + 128, ld=256)
    assert call(c, c + 256 + 124, rows=2, ld=256, block_rows=128)
    assert call(c, 3 * AT, src=c + 8) and not call(c, 3 * AT, src=c + 16) and call(c, 3 * AT, src=3 * AT)
