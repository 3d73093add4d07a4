"""Attention's kernels report offsets and waits in the device's error word: without one a call is refused, not launched
with a null address to report to.  Needs a machine whose device cannot give the word, so one without a GPU."""
import pytest


@pytest.fixture
def no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device gives the word")


@pytest.mark.parametrize("rows", [4, 4000])
def test_no_error_word(jx, no_device, rows):
    size = dict(batch=1, total_q=rows, total_k=rows, heads=4, kv_heads=2, head_dim=8)
    with pytest.raises(jx.JaxRsError, match="error word") as e:
        jx.attention(*range(16, 16 * 8, 16), **size)
    assert e.value.status == jx.JX_ENOMEM
    with pytest.raises(jx.JaxRsError, match="error word") as e:
        jx.attention_bwd(*range(16, 16 * 12, 16), **size)
    assert e.value.status == jx.JX_ENOMEM
