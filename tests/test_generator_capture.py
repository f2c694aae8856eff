"""The step that ``Generator.beam_search`` captures: on the model's own device, whatever device is current
(shown without a GPU, by what the capture is asked for), and beside other threads that use the GPU."""
import contextlib
import threading

import pytest
import torch


def _bare(monkeypatch, device):
    """A Generator of no blocks whose step is recorded."""
    from atomic_gdn2 import generation
    seen = {"current": [None]}
    gen = generation.Generator.__new__(generation.Generator)
    gen.device = torch.device(device)

    @contextlib.contextmanager
    def on(dev):
        seen["current"].append(torch.device(dev))
        yield
        seen["current"].pop()

    class Stream:
        def __init__(self, device=None, **kw):
            assert not kw
            self.device = torch.device(device) if device is not None else seen["current"][-1]

    @contextlib.contextmanager
    def capture(graph, pool=None, stream=None, capture_error_mode="global"):
        seen.update(entered_on=seen["current"][-1], stream=stream, mode=capture_error_mode)
        yield

    class Graph:
        def replay(self):
            pass

    for name, fake in (("device", on), ("Stream", Stream), ("graph", capture), ("CUDAGraph", Graph)):
        monkeypatch.setattr(torch.cuda, name, fake)
    monkeypatch.setattr(gen, "_step", lambda tokens, cache, rows: (None, generation.Cache([], [])))
    monkeypatch.setattr(generation, "beam_step", lambda *a, **kw: result())
    result = lambda: generation.BeamStep(torch.zeros((1, 2)), torch.zeros((1, 2)), torch.zeros((1, 2)), None)  # noqa: E731
    return gen, seen, result(), generation.Cache([], [])


def test_capture_is_on_the_models_device(monkeypatch):
    gen, seen, r, cache = _bare(monkeypatch, "cuda:1")
    gen._captured(r, cache, 2, None)
    assert seen["entered_on"] == torch.device("cuda:1")
    assert seen["stream"] is not None and seen["stream"].device == torch.device("cuda:1")


@pytest.mark.gpu
def test_capture_beside_a_thread_that_allocates():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    from atomic_gdn2 import e2e_lm
    from atomic_gdn2.generation import Generator
    gen = Generator(e2e_lm.make_lm(e2e_lm.LMConfig(vocab_size=61, d_model=128, n_heads=2, d_head=64, n_layers=2)), group_size=32)
    ids = torch.arange(18, device="cuda").view(2, 9)
    want = gen.beam_search(ids, 3, 12, graph=False)
    plain, errors, held = gen._step, [], []

    def other():
        try:
            held.append(torch.empty(96 << 20, dtype=torch.uint8, device="cuda"))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    def step(*a, **kw):
        if torch.cuda.is_current_stream_capturing():
            t = threading.Thread(target=other)
            t.start()
            t.join()
        return plain(*a, **kw)

    gen._step = step
    got = gen.beam_search(ids, 3, 12, graph=True)
    assert held and not errors
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.scores, want.scores)
    # and again, with the graph before this one gone
    again = gen.beam_search(ids, 3, 12, graph=True)
    assert torch.equal(again.tokens, want.tokens) and torch.equal(again.scores, want.scores)
