"""CPU: the per-token calls of a layer refuse tensors of another device than the layer's before the library sees a pointer of them.
(No second device is needed: stand-ins say which device they are on, and a library call fails the test.)"""
import pytest
import torch

M, K, N = 4, 32, 8


class On:
    """A CPU tensor that says it lies on a CUDA device."""

    def __init__(self, t, index):
        self._t, self._index = t, index

    is_cuda = True
    device = property(lambda self: torch.device("cuda", self._index))

    def get_device(self):
        return self._index

    def __getattr__(self, name):
        return getattr(self._t, name)


class Reached(Exception):
    pass


@pytest.fixture
def handle(monkeypatch):
    import ltq
    from ltq import layer

    def reached():
        raise Reached

    monkeypatch.setattr(layer, "lib", reached)
    h = object.__new__(ltq.LayerHandle)
    h._h, h.device_index, h.K, h.N, h._row_workspace = None, 0, K, N, 1
    return h


def pieces(**elsewhere):
    at = lambda name: elsewhere.get(name, 0)  # noqa: E731
    return dict(x=On(torch.zeros(M, K, dtype=torch.uint8), at("x")), qparams=On(torch.zeros(M, 8, dtype=torch.uint8), at("qparams")),
                sums=On(torch.zeros(M, dtype=torch.int32), at("sums")), out=On(torch.zeros(M, N), at("out")))


def test_the_stand_ins_reach_the_library(handle):
    with pytest.raises(Reached):
        handle.forward_tokens(**pieces())
    with pytest.raises(Reached):
        handle.set_channel_qparams(On(torch.zeros(N, 8, dtype=torch.uint8), 0), On(torch.zeros(N), 0))


@pytest.mark.parametrize("name", ["x", "qparams", "sums", "out"])
def test_forward_tokens(handle, name):
    with pytest.raises(ValueError):
        handle.forward_tokens(**pieces(**{name: 1}))


def test_all_on_another_device(handle):
    with pytest.raises(ValueError):
        handle.forward_tokens(**pieces(x=1, qparams=1, sums=1, out=1))
    codes = pieces(x=1)
    del codes["out"]   # (made on the layer's device)
    with pytest.raises(ValueError):
        handle.forward_tokens(**codes)


def test_forward_float(handle):
    with pytest.raises(ValueError):
        handle.forward_float(On(torch.zeros(M, K), 1))
    with pytest.raises(ValueError):
        handle.forward_float(On(torch.zeros(M, K), 0), out=On(torch.zeros(M, N), 1))


def test_set_channel_qparams(handle):
    for qparams, bias in ((1, None), (0, 1), (1, 1)):
        with pytest.raises(ValueError):
            handle.set_channel_qparams(On(torch.zeros(N, 8, dtype=torch.uint8), qparams), None if bias is None else On(torch.zeros(N), bias))
