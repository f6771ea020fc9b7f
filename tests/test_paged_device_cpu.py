"""The device that is current while the paged-serving calls ask the library (no GPU: fakes)."""

import types

import pytest

torch = pytest.importorskip("torch")

from decodebench_b200 import ops  # noqa: E402


def test_workspace_size_is_asked_for_the_tensors_device(monkeypatch):
    """The size goes by the SM count of the device that is current when the library is asked, and is kept
    per device: it has to be the tensors' one, whichever is current at the first call."""
    current, asked = [0], []
    dev = types.SimpleNamespace(index=1)

    class Device:
        def __init__(self, d):
            self.to = d.index

        def __enter__(self):
            self.back, current[0] = current[0], self.to

        def __exit__(self, *exc):
            current[0] = self.back

    def answer(status):
        def call(*args):
            asked.append(current[0])
            return status
        return call

    lib = types.SimpleNamespace(dbk_chunk_attention_workspace_bytes=answer(64), dbk_chunk_attention=answer(0))
    fake = lambda *shape, dtype=torch.float16: torch.zeros(*shape, dtype=dtype)  # noqa: E731
    q, cache = fake(3, 2, 128), fake(1, 1, 16, 128)
    i32 = lambda *shape: fake(*shape, dtype=torch.int32)  # noqa: E731
    empty = torch.empty
    monkeypatch.setattr(ops, "_cuda_device", lambda *ts: dev)
    monkeypatch.setattr(ops, "_check_out", lambda out, d: None)
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops, "_stream", lambda d: 0)
    monkeypatch.setattr(ops, "_ws_bytes_cache", {})
    monkeypatch.setattr(ops.N, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    ops.chunk_attention(q, cache, cache, i32(2), i32(1), page_table=i32(1, 1))
    assert asked == [1, 1] and current == [0]
