"""The rows that the fused decode linears take (no launch)."""
import pytest

from epure import _native as N


@pytest.mark.parametrize("k,prologue,epilogue,rows", [
    (2048, N.PRO_RMSNORM, N.EPI_SILU_MUL, 8), (2048, N.PRO_RMSNORM, N.EPI_STORE, 12),
    (512, N.PRO_RMSNORM, N.EPI_SILU_MUL, 11), (512, N.PRO_RMSNORM, N.EPI_STORE, 16),
    (4096, N.PRO_RMSNORM, N.EPI_SILU_MUL, 6), (8192, N.PRO_RMSNORM, N.EPI_STORE, 4),
    (40000, N.PRO_RMSNORM, N.EPI_STORE, 0), (6144, N.PRO_NONE, N.EPI_RESIDUAL, 16),
    (6144, N.PRO_NONE, N.EPI_SILU_MUL, 12)])
def test_most_rows(k, prologue, epilogue, rows):
    """131,072 bytes, 4,096 a row (8,192 for a pair) and the activations within 227 KB; 64 KB of activations."""
    assert N.decode_linear_max_rows(k, prologue, epilogue) == rows


@pytest.mark.parametrize("k,prologue,epilogue", [(0, 0, 0), (-5, 0, 0), (2048, 2, 0), (2048, 0, 3)])
def test_refusals(k, prologue, epilogue):
    with pytest.raises(RuntimeError, match="bad arguments"):
        N.decode_linear_max_rows(k, prologue, epilogue)
