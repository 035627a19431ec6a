"""CPU checks of what the Python mirror says about arrays without their sizes."""
import pytest

from strict_amd import LogitRules


@pytest.mark.parametrize("arrays,text", [
    (dict(tokens=4096, lengths=8192), "tokens need max_tokens"),
    (dict(bias_starts=4096, bias_tokens=8192, bias_values=12288), "bias_starts needs bias_count"),
    (dict(masks=4096, mask_of=8192), "masks need num_masks")])
def test_arrays_need_sizes(arrays, text):
    with pytest.raises(ValueError, match=text):
        LogitRules(**arrays)


def test_sizes_and_nothing():
    assert LogitRules().struct.tokens is None
    rules = LogitRules(tokens=4096, lengths=8192, max_tokens=0, masks=64, mask_of=128, num_masks=3)
    assert (rules.struct.tokens, rules.struct.max_tokens, rules.struct.bias_count, rules.struct.num_masks) == (4096, 0, 0, 3)
