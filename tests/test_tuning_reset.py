"""Tuning overrides of one test do not reach the next (CPU only)."""
import w4a16_hip as hip


def _rows():
    w = hip.W4A16Weights(0x1000, 0x2000, 0x3000, 34816, 5120, 128, 40)
    return hip.linear_max_t(w)


def test_left_behind():
    """Ends as a test does that fails before it restores what it forced."""
    hip.tune_linear(1000)
    assert _rows() == 1000


def test_own_choice():
    assert _rows() == 48   # the measured rule for gate|up
