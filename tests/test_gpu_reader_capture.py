"""A disk reader, or a model with one, that the garbage collector drops while a graph is being captured."""
from __future__ import annotations

import gc
import time

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _captured(dev, middle):
    """x -> 2 x + 1 captured, with middle() between the two kernels; replayed three times beside eager work."""
    x = torch.zeros(1000, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = x * 2
        middle()
        z = y + 1
    for i in range(3):
        x.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((z == 2 * i + 1).all())


def test_reader_dropped_during_capture(dev, tmp_path):
    """The reader and its open read stay until the capture has ended, and go with the next reader's opening."""
    from nurostream_amd.io import reader
    data = np.random.default_rng(3).integers(0, 256, 5 << 20, dtype=np.uint8)
    data.tofile(tmp_path / "blob")
    gc.collect()

    def drop():
        r = reader.DiskReader(tmp_path / "blob", n_workers=2, device=dev, slot_bytes=1 << 20, n_slots=4)
        held = [r, r.submit(4097, 3 << 20)]
        held.append(held)  # a cycle
        while not held[1].done():  # read, but not waited for
            time.sleep(0.001)
        torch.cuda.synchronize()

    gc.disable()
    try:
        drop()
        _captured(dev, gc.collect)
    finally:
        gc.enable()
    kept = list(reader._dropped)
    assert any(isinstance(x, reader.DiskReader) for x in kept)
    with reader.DiskReader(tmp_path / "blob", n_workers=1, device=dev, slot_bytes=1 << 20) as r:
        assert not reader._dropped and all(x._handle is None for x in kept if isinstance(x, reader.DiskReader))
        assert np.array_equal(r.read(1, 999).numpy(), data[1:1000])


def test_model_dropped_during_capture(dev, tmp_path):
    from test_gpu_decode import _tiny_model

    def drop():
        ns, _ = _tiny_model(tmp_path, dev)
        list(ns.generate([3, 4, 5], max_tokens=4))
        ns.itself = ns
        torch.cuda.synchronize()

    gc.collect()
    gc.disable()
    try:
        drop()
        _captured(dev, gc.collect)
    finally:
        gc.enable()
