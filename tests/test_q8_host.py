"""Host side of the 8-bit cache without a GPU: sizes of scratch, refusals of the backend, strides."""
import contextlib
from types import SimpleNamespace

import torch

from rotorquant_vllm.kernels import q8


def test_scratch_is_sized_for_the_tensors_device(monkeypatch):
    """Two GPUs of different sizes: each call's scratch by its own, whichever is current, also once the other's is known."""
    current, cus = [0], [64, 256]

    @contextlib.contextmanager
    def device(dev):
        before, current[0] = current[0], dev
        yield
        current[0] = before

    fake = SimpleNamespace(rq_q8_attention_workspace_bytes=lambda *sizes: cus[current[0]] * 1000)
    monkeypatch.setattr(q8._lib, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", device)
    q8._attention_bytes.cache_clear()
    try:
        for dev in (1, 0, 1, 0):
            assert q8._attention_bytes(dev, 4, 32, 8, 128, 1, 9000) == cus[dev] * 1000
        assert current == [0]
    finally:
        q8._attention_bytes.cache_clear()
