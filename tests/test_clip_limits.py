"""What a clipping handle refuses before a device is looked for, beyond the argument checks of test_adapters_formulas.py."""
import pytest

import streamz_amd as sz


@pytest.mark.parametrize("tensors", [[(1 << 20, 1 << 48)], [(1 << 20, 1 << 47), ((1 << 20) + (1 << 49), 1 << 47)]])
def test_clip_refuses_more_pieces_than_a_launch_can_have(tensors):
    with pytest.raises(sz.StreamzError) as e:
        sz.GradClip(tensors)
    assert e.value.code == -1 and "too many tensors" in str(e.value)
