"""The largest scale that the operators over a vocabulary take: beyond it their arithmetic would leave f32."""
import pytest

from test_token_loss_cpu import CALLS, refused


@pytest.mark.parametrize("call", CALLS)
def test_largest_scale(call):
    refused(call(scale=2.0 ** 100), "null context")
    for scale in (1.0001 * 2.0 ** 100, 1e35, 3e38):
        refused(call(scale=scale), "scale must be at most 2^100")
