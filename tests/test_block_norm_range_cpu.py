"""Scales and eps of the norms around a block that f32, in which the kernels hold them, does not have."""
import pytest

from tensoroperations_b200 import abi

torch = pytest.importorskip("torch")
from tensoroperations_b200 import sequence  # noqa: E402


@pytest.mark.parametrize("bad", [dict(scale=1e39), dict(scale=-1e300), dict(eps=1e39), dict(eps=1e-46), dict(eps=5e-324)])
def test_constants_beyond_f32_are_refused(bad):
    with pytest.raises(abi.ToError) as e:
        sequence.BlockNorm("bf16", 64, **bad)
    assert e.value.status == abi.TO_ERR_INVALID_ARGUMENT and "eps" in str(e.value)


@pytest.mark.parametrize("good", [dict(scale=3e38), dict(scale=0.0), dict(scale=-1e-50), dict(eps=0.0), dict(eps=1e-38),
                                  dict(eps=2.0 ** -149), dict(eps=1e38)])
def test_constants_of_f32_are_taken(good):
    sequence.BlockNorm("bf16", 64, **good)
