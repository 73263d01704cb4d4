"""Per-device buffers, without a GPU."""

import torch

from online_speculation_b200.ops import workspace


def test_buffers_first_made_in_inference_mode_are_ordinary_tensors(monkeypatch):
    monkeypatch.setattr(workspace, "_buffers", {})
    device = torch.device("cuda", 0)
    with torch.inference_mode():
        word = workspace._get(device, "word", lambda d: torch.ones(1, dtype=torch.int32))
        assert torch.is_inference_mode_enabled()
    assert not word.is_inference()
    word.zero_()
    assert workspace._get(device, "word", None) is word and int(word) == 0
