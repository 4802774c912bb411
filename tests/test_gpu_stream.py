"""The front end hands the library torch's current stream."""

import pytest
import torch

import sdhip


@pytest.mark.gpu
def test_stream_handle_is_the_current_stream(gpu):
    def same():
        return (sdhip.stream_handle().value or 0) == torch.cuda.current_stream().cuda_stream

    assert same()
    for _ in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            assert same() and sdhip.stream_handle().value
    assert same()
