"""The device status word's look-up, without a GPU: a device without an index is the current one."""

from __future__ import annotations

import pytest
import torch

from vesper_b200 import _lib


def test_a_device_without_an_index_finds_the_current_one_s_word(monkeypatch: pytest.MonkeyPatch) -> None:
    word = torch.ones(1, dtype=torch.int32)
    monkeypatch.setattr(_lib, "_STATUS", {torch.device("cuda:3"): word})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    assert _lib.status_word(torch.device("cuda")) is word
    with pytest.raises(_lib.KernelError, match="status 1"):
        _lib.check_status(torch.device("cuda"))
    assert int(word) == 0
