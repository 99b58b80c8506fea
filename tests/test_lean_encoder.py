"""What the encoder on the training operators says of the dropout that it leaves out (no GPU needed)."""
import warnings

import pytest

KW = dict(vocab=10, hidden=16, layers=1, heads=2, ffn=32, max_seq=8)


def test_left_out_dropout_is_told():
    from cswap_b200.workloads import BertEncoder
    with pytest.warns(UserWarning, match="no dropout on probabilities"):
        BertEncoder(lean=True, **KW)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        BertEncoder(lean=True, dropout=0.0, **KW)
        BertEncoder(**KW)
