"""A served model that begins with an Embedding keeps what it was made of: no later change of the model reaches it, and it
holds nothing of the model."""
import gc
import weakref

import numpy as np
import pytest

from rgpu_amd import autograd as A
from rgpu_amd import gpu as G

pytestmark = pytest.mark.gpu


def test_served_embedding_is_apart_from_its_layer():
    gpu = G.Gpu(0)
    rng = np.random.default_rng(2)
    layer = A.Embedding(gpu, 30, 32, scale=2.0, weights=rng.normal(size=(30, 32)))
    model = A.Sequential([layer, A.Dense(gpu, 64, 7, "linear", weights=rng.normal(size=(64, 7)) * 0.2)])
    ids = rng.integers(-1, 30, (20, 2))
    served = A.QuantizedSequential(model)
    before = gpu.download(served.predict(ids))
    layer.scale = 3.0
    gpu.write(layer.w.tensor, np.zeros((30, 32), np.float32))
    assert np.array_equal(gpu.download(served.predict(ids)), before)
    assert np.array_equal(gpu.download(served.predict(A.upload_ids(gpu, ids))), before)
    for wrong in (ids.astype(np.float32), ids[None]):
        with pytest.raises(ValueError):
            served.predict(wrong)
    table = weakref.ref(layer.w.tensor)
    del model, layer
    gc.collect()
    assert table() is None  # the f32 table is free
    assert np.array_equal(gpu.download(served.predict(ids)), before)
    del served
    gpu.close()
