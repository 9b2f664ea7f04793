"""Which stream a launch goes to."""
import types

import pytest
import torch


def test_the_public_call_where_the_address_alone_is_not_to_be_had(monkeypatch):
    from imparo_amd.kernels import ops
    monkeypatch.setattr(ops, "_raw_stream", None, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *device: types.SimpleNamespace(cuda_stream=4711))
    assert ops._stream() == 4711


@pytest.mark.gpu
def test_the_address_is_that_of_the_current_stream():
    from imparo_amd.kernels import ops
    side = torch.cuda.Stream()
    assert ops._stream() == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(side):
        assert ops._stream() == side.cuda_stream
        with ops.on_current_stream():
            assert ops._stream() == side.cuda_stream
    assert ops._stream() == torch.cuda.current_stream().cuda_stream
