"""Descriptions of steps and lists of pages for the cache in 8 bits, without a GPU."""
import gc
import weakref

import numpy as np
import pytest
import torch

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


@pytest.mark.parametrize("bad", [[2 ** 32 + 1], np.array([2 ** 32 + 1]), np.array([2 ** 31], dtype=np.uint32), [-1], [0.7], np.array([1.0]),
                                 torch.tensor([2 ** 40])])
def test_page_numbers_that_are_none_in_32_bits_are_refused(bad):
    # 2^32 + 1 would be page 1
    with pytest.raises(K.KernelError, match="page numbers"):
        K.copy_pages([torch.zeros(1, 4, 4)], bad, [3])
    with pytest.raises(K.KernelError, match="page numbers"):
        K.copy_pages([torch.zeros(1, 4, 4)], [3], bad)


@pytest.mark.parametrize("good", [[0, 2], (2, 0), np.array([0, 2]), np.array([2, 0], dtype=np.uint8), torch.tensor([1, 3]), [], range(3),
                                  np.arange(6, dtype=np.int32)[::2]])
def test_page_numbers_of_other_types(good):
    a = K._page_numbers(good)
    assert a.dtype == np.int32 and a.flags.c_contiguous and a.tolist() == [int(i) for i in good]
