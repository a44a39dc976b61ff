"""Sequential with layers that a program defines itself."""
import numpy as np
import pytest

from rgpu_amd import autograd as A
from rgpu_amd import gpu as G

pytestmark = pytest.mark.gpu


def test_a_first_layer_of_its_own_may_have_an_attribute_called_input():
    gpu = G.Gpu(0)

    class Kept:
        """A program's own layer that keeps its last input."""

        def __init__(self):
            self.gpu, self.input = gpu, None

        def forward(self, x):
            self.input = x
            return x.mul(x)

    x = np.arange(6, dtype=np.float32).reshape(2, 3)
    layer = Kept()
    model = A.Sequential([layer])
    for _ in range(2):
        assert np.array_equal(gpu.download(model.predict(x)), x * x)
    layer.w = A.Param(gpu, "W", x)  # a layer with weights is asked for them, as before
    assert np.array_equal(gpu.download(model.predict(x)), x * x)
    gpu.close()
