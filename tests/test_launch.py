"""On which device and stream an entry point launches: that of its tensors, whatever the current device is."""
import contextlib
import inspect

import pytest
import torch

import kda355
from kda355 import _lib, decode, latent, pages, prefill, recurrent  # noqa: F401  (`decode` and `prefill` are the functions)


@pytest.fixture
def devices(monkeypatch):
    """Two devices without a GPU: the handle of device i's current stream is 100 + i."""
    now = [0]

    @contextlib.contextmanager
    def on(index):
        before, now[0] = now[0], index
        try:
            yield
        finally:
            now[0] = before

    monkeypatch.setattr(_lib, "_device", lambda: now[0])
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", on)
    return now


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("index", [0, 1])
def test_launch_on_the_tensors_device(devices, current, index):
    devices[0] = current
    seen = []

    def entry(args, stream):
        seen.append((args, stream, devices[0]))
        return -2

    assert _lib.launch(entry, b"x", torch.device("cuda", index)) == -2
    assert seen == [(b"x", 100 + index, index)] and devices[0] == current


def test_device_is_put_back_after_an_error(devices):
    def entry(args, stream):
        raise ValueError

    with pytest.raises(ValueError):
        _lib.launch(entry, b"", torch.device("cuda", 1))
    assert devices[0] == 0


def test_every_entry_point_launches_so():
    """No module of the package takes a stream by itself."""
    for module in (latent, pages, inspect.getmodule(kda355.decode), inspect.getmodule(kda355.prefill), recurrent):
        text = inspect.getsource(module)
        assert "_lib.launch(" in text and "stream(dev" not in text and ".cuda_stream" not in text, module.__name__


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device():
    g = torch.Generator().manual_seed(0)
    latents, pe = torch.randn(40, 512, generator=g).bfloat16(), torch.randn(40, 64, generator=g).bfloat16()
    ql, qp = torch.randn(1, 12, 512, generator=g).bfloat16(), torch.randn(1, 12, 64, generator=g).bfloat16()
    got = []
    for index in (0, 1):
        dev = torch.device("cuda", index)
        cache = torch.zeros(3, 16, 576, dtype=torch.bfloat16, device=dev)
        table, lens = torch.arange(3, dtype=torch.int32, device=dev)[None], torch.tensor([40], dtype=torch.int32, device=dev)
        mass, lse = torch.zeros(1, 48, device=dev), torch.empty(1, 12, device=dev)
        with torch.cuda.device(0):
            kda355.latent_append(latents.to(dev), pe.to(dev), cache, torch.arange(40, device=dev))
            out = kda355.latent_decode(ql.to(dev), qp.to(dev), cache, table, lens, lse=lse)
            kda355.latent_weights(ql.to(dev), qp.to(dev), cache, table, lens, lse, mass)
            refs, free, num = table[0] * 0 + 1, table[0] * 0 - 1, lens * 0
            kda355.evict_tokens([cache], [mass], table, lens, refs, free, num, lens * 0, 20, 4, 16)
            assert torch.cuda.current_device() == 0
        got.append([t.cpu() for t in (out, lse, cache, mass, table, lens, refs, free, num)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
