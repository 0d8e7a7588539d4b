"""generate()'s draw refuses a vocabulary that it does not take before the state changes. No GPU needed."""
import pytest

from df_ssm_inference import _draw_filters
from dfssm import _C, ops


def test_vocabulary():
    most = ops.MAX_DRAW_VOCAB
    assert _draw_filters(0.8, 5, 1.0, 0.0, 1.0, None, most)
    with pytest.raises(ValueError):
        _draw_filters(0.8, 5, 1.0, 0.0, 1.0, None, most + 1)
    assert not _draw_filters(0.8, 0, 0.9, 0.0, 1.2, None, most + 1)    # dfssm_sample
    f = _C.Filter(0, 0, 0, 0, 1.0, 0, 1.0, 0.0)
    call = lambda vocab: _C.lib().dfssm_sample_filtered(16, 0, vocab, 0, vocab, 16, f, 16, None, None)
    assert call(most) == 0 and call(most + 1) == -2                    # (no rows: nothing is launched)
