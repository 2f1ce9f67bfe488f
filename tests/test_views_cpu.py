"""What a view cannot be made of, and what the refusal says."""
import pytest
import torch

import linalg_b200 as lb


def test_refusals_name_their_cause():
    class Backwards:
        """A tensor that steps backwards, as other array packages have them."""

        def __init__(self, t):
            self.t, self.dtype, self.shape = t, t.dtype, t.shape

        def untyped_storage(self):
            return self.t.untyped_storage()

        def storage_offset(self):
            return 3

        def stride(self):
            return (-1,)

    x = torch.zeros(4)
    with pytest.raises(lb.InvalidArgument, match="negative stride"):
        lb.View.of(Backwards(x))
    with pytest.raises(lb.InvalidArgument, match="rank above 8"):
        lb.View.of(torch.zeros([1] * 9))
    with pytest.raises(lb.InvalidArgument, match="unknown element type"):
        lb.View.of(x, 1 << 40)
    for code in ("f32", 1.0):
        with pytest.raises(TypeError, match="element type"):
            lb.View.of(x, code)
    with pytest.raises(TypeError, match="unsupported element type"):
        lb.View.of(x.to(torch.int8))
