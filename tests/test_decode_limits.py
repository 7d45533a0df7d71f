"""The decode step's size limits, where they are decided on the host: nothing
here touches a GPU."""
import s2x


def test_q4_workspace_past_the_int8_gemm():
    """Weights whose scales lie past the int8 GEMM's 31-bit offsets, or whose
    rows of y do, are read as they lie for any number of rows: no workspace."""
    size = s2x.lib.s2x_mul_mat_q4_0_workspace_size
    for m in (257, 1 << 20):
        assert size(1 << 19, 1 << 17, m) == 0  # K * N = 2^36
        assert size(1 << 18, 1 << 17, m) == 0  # 2^35
        assert size((1 << 18) - 32, 1 << 17, m) >= ((1 << 18) - 32) << 17
        assert size(1 << 18, (1 << 17) - 128, m) >= (1 << 18) * ((1 << 17) - 128)
        assert size(1 << 18, (1 << 17) - 127, m) == 0  # (columns count to whole 128)
        assert size(32, 1 << 22, m) == 0
        assert size(32, (1 << 22) - 1, m) >= 32 << 22
