"""Descriptions of steps and lists of pages for the cache in 8 bits, without a GPU."""
import gc
import weakref

from pytorch_transformers_b200 import kernels as K
from test_q8 import _Ints


def test_a_description_holds_the_tensors_that_it_points_into():
    arrays = [_Ints(0, 3), _Ints(0, 3), _Ints(0, 2), _Ints(0, 2), _Ints(0, 2), _Ints(0, 2, 4)]
    alive = [weakref.ref(a) for a in arrays]
    batch = K.step_batch(*arrays)
    del arrays
    gc.collect()
    assert all(a() is not None for a in alive)      # else their memory is given to the next tensor while the kernels read it
    del batch
    gc.collect()
    assert not any(a() is not None for a in alive)
