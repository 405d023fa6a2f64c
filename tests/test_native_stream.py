"""stream_ptr takes whatever names a device (no GPU: torch's side is a stand-in)."""
import types

import pytest
import torch

from actkv_open_b200 import _native as N


@pytest.mark.parametrize("raw", [None, lambda index: 70 + index])
@pytest.mark.parametrize("device, index", [(torch.device("cuda", 1), 1), (torch.device("cuda"), 0), ("cuda:1", 1), ("cuda", 0), (1, 1)])
def test_stream_of_every_kind_of_device(device, index, raw, monkeypatch):
    def current_stream(d):
        d = torch.device("cuda", d) if isinstance(d, int) else torch.device(d)
        return types.SimpleNamespace(cuda_stream=70 + (d.index or 0))
    monkeypatch.setattr(N, "_raw_stream", raw)
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    assert N.stream_ptr(device) == 70 + index
