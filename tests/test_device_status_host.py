"""The device status word is an ordinary tensor whatever the mode of the first call."""

import torch

from telescope_cache_b200.telescoping_attn import attention


def test_status_word_formed_under_inference_mode(monkeypatch):
    monkeypatch.setattr(attention, "_STATUS", {})
    with torch.inference_mode():
        word = attention.device_status("cpu")
    word.fill_(2)
    assert attention.read_device_status("cpu") == 2
    assert attention.read_device_status("cpu") == 0
