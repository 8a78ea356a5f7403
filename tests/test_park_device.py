"""A parking buffer on another device than the engine's is refused before any
call of the library (no GPU needed: engine and buffer are stand-ins)."""
import pytest

from ssla_rt_b200 import abi
from ssla_rt_b200.engine import SslaEngine


class Buffer:
    is_cuda = True

    def __init__(self, device):
        self.device = device

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device

    def data_ptr(self):
        return 1 << 20

    def numel(self):
        return 4096

    def element_size(self):
        return 1


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or abi.SSLA_OK


@pytest.mark.parametrize("engine_on,buffer_on", [(0, 1), (1, 0), (3, 2), (2, 2), (0, 0)])
@pytest.mark.parametrize("what", ["park", "resume"])
def test_parking_buffer_device(engine_on, buffer_on, what):
    eng = SslaEngine.__new__(SslaEngine)
    eng.device, eng.lib, eng.h = engine_on, Library(), 1
    call = lambda: getattr(eng, what)(Buffer(buffer_on), 0)  # noqa: E731
    if engine_on == buffer_on:
        call()
        assert [n for n, _ in eng.lib.calls] == [f"ssla_engine_{what}"] and eng.lib.calls[0][1][4] == 4096
    else:
        with pytest.raises(ValueError, match="device"):
            call()
        assert not eng.lib.calls
    eng.h = None
