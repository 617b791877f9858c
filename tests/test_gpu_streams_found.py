"""The stream that kernels go to is the current one, whichever way this torch offers to ask for it."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offered", [True, False])
def test_the_current_stream(monkeypatch, offered):
    from llmserve_amd.kernels import HipKernels, hip

    if not offered:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(hip, "_current_stream", hip._stream_address())
    for device in ("cuda", "cuda:0"):
        k = HipKernels(torch.bfloat16, torch.device(device))
        assert k._stream == torch.cuda.current_stream().cuda_stream
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            assert k._stream == other.cuda_stream != torch.cuda.default_stream().cuda_stream
            with k.stream_scope():
                assert k._stream == other.cuda_stream
        assert k._stream == torch.cuda.default_stream().cuda_stream
