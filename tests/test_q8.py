"""The cache in 8 bits without a GPU: what the Python faces refuse before anything reaches a device, and the plain rule itself."""
import math

import pytest
import torch

import plain_q8 as plain
from pytorch_transformers_b200 import kernels as K


def test_tensors_in_host_memory_are_refused():
    pool, exp = torch.zeros(3, 2, 64, 32).to(K.Q8), torch.zeros(3, 2, dtype=torch.int8)
    cache = (pool, exp, pool.clone(), exp.clone())
    batch = K.StepBatchC(n_tokens=1, n_seqs=1, pages_stride=1)
    fused, q = torch.zeros(1, 2 * 3 * 32).bfloat16(), torch.zeros(1, 2, 32).bfloat16()
    tiles = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(K.KernelError):
        K.split_rotate_store_q8(fused, *cache, batch, 2, 1, 32)
    with pytest.raises(K.KernelError):
        K.attention_decode_q8(fused, *cache, batch, None, None, 2, 1, 32, 0.1)
    with pytest.raises(K.KernelError):
        K.attention_q8(q, *cache, batch, tiles, tiles, 1, 16, None, 2, 0.1)
    with pytest.raises(K.KernelError):
        K.unpack_pages_q8(*cache, tiles)
    with pytest.raises(K.KernelError):
        K.copy_pages([pool], [0], [1])
    with pytest.raises(K.KernelError):
        K.step_batch(tiles, tiles, tiles, tiles, tiles, tiles[None])


def test_head_sizes():
    assert [d for d in range(0, 300) if K.q8_supports(d)] == list(range(16, 257, 16))


@pytest.mark.parametrize("amax,e", [(0.0, -126), (448.0, 0), (448.0001, 1), (449.0, 1), (1.75, -8), (1.7500001, -7), (3.3e38, 119), (2.0 ** -140, -126)])
def test_exponents(amax, e):
    assert plain.exponent(amax) == e


def test_rounding_agrees_with_torch():
    x = torch.cat([torch.randn(20000) * 2.0 ** torch.randint(-12, 9, (20000,)), torch.tensor([0.0, 448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.clamp(-464, 464)
    assert torch.equal(plain.round_e4m3(x).float(), x.to(K.Q8).float())
    assert math.isnan(float(plain.round_e4m3(torch.tensor([math.inf]))[0]))


def test_error_codes_are_nobody_elses():
    # a wait that runs out in another kernel must not read as a page number that is none
    import pathlib
    import re
    used = {}
    for path in (pathlib.Path(K.__file__).parent / "csrc").glob("*.cu*"):
        for code in re.findall(r"error_flag, (\d+)\)", path.read_text()):
            used.setdefault(int(code), set()).add(path.name)
    own = {"attention_q8.cu", "cache_q8.cu"}
    assert {51, 52, 53, 54, 55} <= set(used) and all(used[c] <= own for c in used if used[c] & own)


def test_a_wait_that_ran_out_elsewhere_is_not_called_a_page(monkeypatch):
    monkeypatch.setattr(K, "_error_flags", {torch.device("cpu"): torch.tensor([21], dtype=torch.int32)})
    with pytest.raises(K.KernelError, match="gave up waiting"):
        K.check_device_errors("cpu")


class _Ints:
    """As much of an int32 tensor on a CUDA device as the descriptions of steps look at."""
    dtype, is_cuda = torch.int32, True

    def __init__(self, device, *shape):
        self.device_number, self.shape = device, shape

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device_number

    def numel(self):
        return math.prod(self.shape)

    def data_ptr(self):
        return 256


def test_steps_described_on_two_devices_are_refused():
    arrays = [_Ints(0, 3), _Ints(0, 3), _Ints(0, 2), _Ints(0, 2), _Ints(0, 2), _Ints(0, 2, 4)]
    batch = K.step_batch(*arrays)
    assert (batch.n_tokens, batch.n_seqs, batch.pages_stride) == (3, 2, 4)
    K._check_batch(batch, 0, "here")
    with pytest.raises(K.KernelError, match="device"):
        K._check_batch(batch, 1, "there")
    for i in range(6):
        other = list(arrays)
        other[i] = _Ints(1, *arrays[i].shape)
        with pytest.raises(K.KernelError, match="one device"):
            K.step_batch(*other)
