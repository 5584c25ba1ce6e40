"""The serving operators at their edges, as far as no GPU is needed."""
from mlir_edsl import _native

INVALID = 1


def test_expire_limits():
    L = _native.lib()
    assert L.b200_debug_w4_expire(-1) == INVALID
    assert "negative" in L.b200_last_error().decode()
    assert L.b200_debug_w4_expire(0) == 0
