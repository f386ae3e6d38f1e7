"""The word in which kernels raise errors, where a kernel's first call on a device is one that a graph captures."""
import pytest
import torch

from test_q8_gpu import Case, K  # noqa: F401

pytestmark = pytest.mark.gpu


def test_replays_erase_no_errors(K, monkeypatch):
    c = Case(2, 4, 64, [100, 200], [1, 1], seed=9)
    cache, batch = c.device(K)
    args = (c.dev["fused"], *cache, batch, None, None, 2, 4, 64, c.scale)
    want = K.attention_decode_q8(*args, write_cache=True)      # and whatever else a first call sets up
    torch.cuda.synchronize()
    monkeypatch.setattr(K, "_error_flags", {})
    monkeypatch.setattr(K, "_flag_addresses", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.attention_decode_q8(*args, write_cache=False)
    K.check_device_errors("cuda")      # zero before any replay
    K.error_flag("cuda").fill_(51)
    graph.replay()
    with pytest.raises(K.KernelError, match="a page that the cache does not have"):
        K.check_device_errors("cuda")
    assert torch.equal(out, want)
