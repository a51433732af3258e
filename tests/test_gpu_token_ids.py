"""Token ids on their way to the device: whole numbers of any type and shape, none at all, and what is refused."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from ferrox_amd import capi
    with capi.Context(0) as c:
        yield c


@pytest.mark.parametrize("ids", [[3, 0, -1], np.array([[1, 2], [3, 4]], np.int32), np.arange(5, dtype=np.uint8), np.arange(12).reshape(3, 4)[:, ::2], [], np.zeros((0, 7))])
def test_ids_come_back(ctx, ids):
    want = np.asarray(ids)
    d = ctx.upload_ids(ids)
    assert d.shape == want.shape and np.array_equal(d.numpy(), want.ravel())
    w = np.arange(20, dtype=np.float32).reshape(5, 4)
    if want.size:  # the pool hands out no empty blocks
        assert ctx.embedding_fwd(ctx.upload(w), d).numpy().shape == want.shape + (4,)


@pytest.mark.parametrize("ids", [[0.7, 1.2], np.ones(3, np.float32), np.array([True, False]), np.array([1 + 0j])])
def test_ids_that_are_no_whole_numbers_are_refused(ctx, ids):
    from ferrox_amd.capi import FerroxHipError
    with pytest.raises(FerroxHipError, match="whole numbers"):
        ctx.upload_ids(ids)
