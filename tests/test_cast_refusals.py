"""Casts of types that no tensor holds are refused, also to themselves (no GPU needed)."""
import pytest

from autonomousaicore_amd import _lib
from autonomousaicore_amd._lib import AIC_F32, AIC_U4, AIC_U8, AIC_U16

NOT_IMPLEMENTED = 8
P = 1 << 20


@pytest.mark.parametrize("n", [0, 1, 4096])
@pytest.mark.parametrize("src,dst", [(AIC_U4, AIC_U4), (8, 8), (-1, -1), (AIC_U4, AIC_F32), (AIC_F32, AIC_U4), (AIC_U4, AIC_U8)])
def test_cast_of_no_tensor_type(src, dst, n):
    with pytest.raises(_lib.AicError, match="not implemented") as e:
        _lib.call("aic_hip_cast", P, src, 2 * P, dst, n, None)
    assert e.value.code == NOT_IMPLEMENTED


@pytest.mark.parametrize("t", range(AIC_U16 + 1))
def test_cast_of_nothing_to_itself(t):
    _lib.call("aic_hip_cast", P, t, 2 * P, t, 0, None)
