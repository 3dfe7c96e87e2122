"""An operator's bank format is the one it was built with: its banks, the pager's fields and the
kernels' entry points all follow from it."""

import pytest

from recap_amd import HostBankOperator, Operator, OperatorConfig
from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation


@pytest.mark.parametrize("cls", [Operator, HostBankOperator])
@pytest.mark.parametrize("given", ["fp16", "int8"])
def test_bank_format_is_fixed(cls, given):
    layout = Layout.from_permutation(hilbert_permutation((4, 8, 8)), text_tokens=7, text_first=False)
    op = cls.build(OperatorConfig(), SparseGeometry.build(layout, 128), n_layers=1, bank_format=given)
    for other in ("int8", "fp16", "int4"):
        with pytest.raises(AttributeError, match="bank_format"):
            op.bank_format = other
        assert op.bank_format == given
    op.alpha_override = 0.5         # other settings stay settable
    op.reset()
    with pytest.raises(AttributeError, match="bank_format"):
        op.bank_format = "int8"
