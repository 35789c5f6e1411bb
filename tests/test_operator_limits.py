"""Sizes that a launch has no lanes for are refused before it (no GPU needed)."""

from miles_amd import _lib

P = 0x1000      # a pointer that no refused call follows


def test_a_launch_has_fewer_than_2_to_the_32_lanes():
    lib = _lib.load()

    def refused(rc):
        return rc == -1 and b"tensor too large" in lib.mq_last_error()

    # the sums of an activation's columns: eight lanes to a column
    assert refused(lib.mq_activation_backward(P, 0, 1 << 29, P, None, 1, P, P, P, 4, 1 << 29, None))
    # 256 lanes restore 4096 16-bit values or 2048 fp32 ones
    assert refused(lib.mq_mxfp8_dequant(P, P, P, 0, (1 << 36) // 64, 64, None))
    assert refused(lib.mq_mxfp8_dequant(P, P, P, 2, (1 << 35) // 64, 64, None))
