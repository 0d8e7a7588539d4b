"""What generate() makes of its filter arguments before anything is launched. No GPU needed."""
import pytest

from df_ssm_inference import _draw_filters


def test_chooses_the_draw():
    assert not _draw_filters(None, 0, 1.0, 0.0, 1.0)
    assert not _draw_filters(0.8, 0, 0.9, 0.0, 1.2)       # dfssm_sample
    assert _draw_filters(0.8, 5, 0.9, 0.0, 1.0)
    assert _draw_filters(0.8, 0, 0.9, 0.1, 1.0)


@pytest.mark.parametrize("args", [(None, 5, 1.0, 0.0, 1.0), (0.0, 5, 1.0, 0.0, 1.0), (float("nan"), 5, 1.0, 0.0, 1.0),
                                  (float("inf"), 5, 1.0, 0.0, 1.0), (0.8, -1, 1.0, 0.0, 1.0),
                                  (0.8, 2**31, 1.0, 0.0, 1.0), (0.8, 0, 1.0, -0.1, 1.0), (0.8, 0, 1.0, 1.1, 1.0),
                                  (0.8, 0, 1.0, float("nan"), 1.0), (0.8, 5, -0.1, 0.0, 1.0),
                                  (0.8, 5, float("nan"), 0.0, 1.0), (0.8, 5, 1.0, 0.0, 1.2)])
def test_refusals(args):
    with pytest.raises(ValueError):
        _draw_filters(*args)


def test_refusals_of_kind():
    with pytest.raises(ValueError):
        _draw_filters(0.8, 5, 1.0, 0.0, 1.0, state_df=object())
    with pytest.raises(TypeError):
        _draw_filters(0.8, 2.5, 1.0, 0.0, 1.0)
