"""Attention over a cache in 8 bits where more than a cluster of blocks shares a row's pages: the parts that join through memory."""
import ctypes

import pytest
import torch

from test_q8_gpu import BF, PAGE, Case, K  # noqa: F401

pytestmark = pytest.mark.gpu


# the rows of parts that no block has written: more splits than asked for by hand, and by the library's own choice behind a wide table
@pytest.mark.parametrize("splits,pages", [(16, 2), (24, 2), (0, 512)])
def test_a_step_without_one_token_each_writes_nothing(K, splits, pages):
    c = Case(1, 2, 64, [10, 20], [2, 0])
    cache, batch = c.device(K)
    before = [t.clone() for t in cache]
    guard = 6
    out = torch.full((2 + guard, 2 * 64), 7.0, dtype=BF, device="cuda")      # two rows of the result, and rows behind it
    L, stream = K.lib(), torch.cuda.current_stream().cuda_stream
    floats = L.ptb_attention_q8_floats(2, 1, 2, 1, 64, splits, pages, 2)
    assert floats > 0      # the parts join through memory
    parts = torch.full((floats,), 3.0, device="cuda")
    code = L.ptb_attention_decode_q8(c.dev["fused"].data_ptr(), *(t.data_ptr() for t in cache), c.pages, out.data_ptr(), ctypes.byref(batch), None,
                                     None, 0, False, None, 2, 1, 64, 0.1, 0, True, splits, pages, parts.data_ptr(), floats,
                                     K.error_flag("cuda").data_ptr(), stream)
    assert code == 0
    with pytest.raises(K.KernelError, match="one token for each"):
        K.check_device_errors("cuda")
    assert bool((out == 7.0).all())
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
