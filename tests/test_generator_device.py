"""``Generator.beam_search`` leaves the current device as it was: the graph of its steps, whose destruction may
change it, is dropped while the model's device is current."""
import contextlib

import torch


def test_the_graph_is_dropped_on_the_models_device(monkeypatch):
    from atomic_gdn2 import generation
    current, dropped = ["other"], []

    class Graph:
        def replay(self):
            pass

        def __del__(self):
            dropped.append(current[-1])

    @contextlib.contextmanager
    def on(dev):
        current.append(str(dev))
        yield
        current.pop()

    capture = lambda graph, **kw: contextlib.nullcontext()  # noqa: E731
    for name, fake in (("device", on), ("Stream", lambda dev: dev), ("graph", capture), ("CUDAGraph", Graph)):
        monkeypatch.setattr(torch.cuda, name, fake)
    gen = generation.Generator.__new__(generation.Generator)
    gen.device = torch.device("meta")
    cache = generation.Cache([], [])
    gen.prefill = lambda ids: (torch.zeros((1, 5), device="meta"), cache)
    gen._step = lambda tokens, c, rows: (torch.zeros((2, 5), device="meta"), cache)
    z = lambda dt: torch.zeros((1, 2), dtype=dt, device="meta")  # noqa: E731
    monkeypatch.setattr(generation, "beam_step", lambda *a, **kw: generation.BeamStep(z(torch.int64), z(torch.int64), z(torch.float32), None))
    r = gen.beam_search(torch.zeros((1, 3), dtype=torch.int64, device="meta"), 2, 5, graph=True)
    assert r.tokens.shape == (1, 2, 5)
    assert dropped == ["meta"] and current == ["other"]
