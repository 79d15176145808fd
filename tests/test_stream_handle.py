"""The stream of any way to name a device; CPU only."""

from types import SimpleNamespace

import pytest
import torch

from torch2iron_amd import _lib


@pytest.mark.parametrize("device,raw", [(torch.device("cuda", 1), True), (torch.device("cuda"), False), ("cuda:0", False),
                                        (0, False), (None, False)])
def test_stream_handle(monkeypatch, device, raw):
    """A torch device with an index goes to torch's raw accessor, by that index; all else, strings (which have a
    method named index) among them, to torch.cuda.current_stream."""
    def raw_stream(index):
        assert type(index) is int
        return 100 + index

    monkeypatch.setattr(_lib, "_RAW_STREAM", raw_stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=("stream of", d)))
    assert _lib.stream_handle(device) == (100 + device.index if raw else ("stream of", device))


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda:0", "cuda", 0, None, torch.device("cuda:0"), torch.device("cuda")])
def test_stream_handle_on_the_device(gpu, device):
    s = torch.cuda.Stream(gpu)
    with torch.cuda.stream(s):
        assert _lib.stream_handle(device) == s.cuda_stream
