"""Where 8-bit activations are refused: before anything is allocated."""
import pytest

from hipfm.config import RunConfig
from hipfm.models.deepfm import NativeDeepFM


@pytest.mark.parametrize("kw", [dict(deep_layers=(256, 128, 64)),                    # the fused tower holds these
                                dict(deep_layers=(4096, 4096, 4096), batch_norm=True),
                                dict(deep_layers=(256, 128, 64), batch_norm=True, fused=False)])
def test_only_the_per_layer_tower_without_batch_norm(kw):
    with pytest.raises(ValueError, match="act_dtype=fp8"):
        NativeDeepFM(1000, 4, 8, keep_probs=(0.5, 0.5, 0.5), device="cpu", act_dtype="fp8", **kw)


def test_names():
    with pytest.raises(ValueError, match="act_dtype"):
        NativeDeepFM(1000, 4, 8, device="cpu", act_dtype="e4m3")
    assert RunConfig().act_dtype == "bf16"
    with pytest.raises(ValueError, match="act_dtype"):
        RunConfig(act_dtype="int8").validate()
