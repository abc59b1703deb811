"""The device status word on a B200: one per device, however the device is named."""

from __future__ import annotations

import pytest
import torch

from vesper_b200 import _lib

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def test_a_device_without_an_index_is_the_current_one() -> None:
    indexed = torch.device("cuda", torch.cuda.current_device())
    assert _lib.status_word(CUDA).data_ptr() == _lib.status_word(indexed).data_ptr()
    for written, read in ((CUDA, indexed), (indexed, CUDA)):
        _lib.status_word(written).fill_(1)
        with pytest.raises(_lib.KernelError, match="status 1"):
            _lib.check_status(read)
        _lib.check_status(written)  # reported once
