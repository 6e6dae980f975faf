"""The device error word is read and cleared on the device that was asked for, whatever the current one."""
from types import SimpleNamespace

import pytest
import torch

from zs_b200 import _lib as Z


@pytest.fixture
def cuda(monkeypatch):
    """A machine of four devices, device 0 current, each with a word of its own."""
    state = SimpleNamespace(current=0, words=[0, 0x10, 0, 0x40], clear=[])

    class device:
        def __init__(self, d):
            self.d = state.current if d is None else torch.device(d).index if not isinstance(d, int) else d

        def __enter__(self):
            self.was, state.current = state.current, self.d

        def __exit__(self, *exc):
            state.current = self.was

    def get(out, stream):
        out._obj.value = state.words[state.current]
        return 0 if stream == state.current else 5           # a stream of another device is an error

    def clear(stream):
        state.words[state.current] = 0
        return 0 if stream == state.current else 5

    def current_stream(d=None):
        return SimpleNamespace(cuda_stream=device(d).d)

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    real = Z.lib()
    monkeypatch.setattr(Z, "lib", lambda: SimpleNamespace(zs_device_error_get=get, zs_device_error_clear=clear,
                                                          zs_error_string=real.zs_error_string,
                                                          zs_last_cuda_error=real.zs_last_cuda_error))
    return state


def test_the_word_of_the_device_that_was_asked_for(cuda):
    assert [Z.device_error(f"cuda:{d}") for d in range(4)] == [0, 0x10, 0, 0x40]
    assert Z.device_error() == 0 and Z.device_error(3) == 0x40
    Z.clear_device_error("cuda:3")
    assert cuda.words == [0, 0x10, 0, 0] and cuda.current == 0


def test_a_cache_on_another_device_checks_its_own_word(cuda):
    from zs_b200.paged import PagedKVCache

    c = object.__new__(PagedKVCache)
    c.kv = SimpleNamespace(device=torch.device("cuda:1"))
    with pytest.raises(Z.ZsError, match="out of range"):
        c.check()
    c.check()
    assert cuda.words == [0, 0, 0, 0x40]
