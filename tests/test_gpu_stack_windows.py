"""Windows that a stack (``examples/gpt2_stack.py``) is given and attention refuses are refused, not left out."""
import pytest
import torch

from test_gpu_gpt2_stack import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{"window": 0}, {"window": 0, "sinks": 2}, {"window": -1}, {"sinks": 2}, {"window": 4, "sinks": -1}])
def test_refused(kw):
    import latent_weight_lab_amd as lwl

    model = make(**kw)
    lwl.prepare_block_fht_weight_cache(model)
    with torch.no_grad(), pytest.raises(ValueError):
        model(torch.zeros(1, 5, dtype=torch.long, device="cuda"))
    lwl.flush_block_fht_weight_cache(model)
