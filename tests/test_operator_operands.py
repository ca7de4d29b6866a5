"""cvmk_dense_lut_*: operands whose places do not go together.  No device is needed, as in test_operator_refusals."""
import pytest

from test_operator_refusals import dense


@pytest.fixture(scope="module")
def kn(pkg):
    return pkg.kernels


@pytest.mark.parametrize("step", ["ADD_T", "SUB_T", "RSUB_T"])
@pytest.mark.parametrize("of_y,of_operand", [("I8", "I32"), ("I32", "I8")])
def test_an_operand_that_is_the_result_has_its_type(kn, step, of_y, of_operand):
    with pytest.raises(kn.KernelError) as e:
        dense(kn, y_dtype=getattr(kn, of_y), chain_y=[(kn.RSHIFT, 7, 8), (getattr(kn, step), 5 << 20, getattr(kn, of_operand))])
    assert e.value.status == kn.ERR_ARG and "has y's type" in str(e.value)
