"""The Python path of linear asks for a workspace on the operands' device: how a product is split goes by its CUs, and cards or
partitions of one process may differ in them."""
import contextlib
import types

import torch

from atomic_gdn2 import linear


def test_workspaces_are_asked_for_where_the_kernel_runs(monkeypatch):
    entered, asked = [], []

    @contextlib.contextmanager
    def device(dev):
        entered.append(dev)
        yield
        entered.pop()

    def ask(kind):
        def bytes_of(p):
            asked.append((kind, list(entered)))
            return 64
        return bytes_of

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(linear._lib, "lib", lambda: types.SimpleNamespace(
        gdn2_linear_workspace_bytes=ask("product"), gdn2_linear=lambda *a: 0, gdn2_linear_slope_workspace_bytes=ask("slope"),
        gdn2_linear_slope=lambda *a: 0))
    monkeypatch.setattr(linear._lib, "stream_handle", lambda dev: None)
    x, w, dy = torch.zeros(4, 8), torch.zeros(8, 6), torch.zeros(4, 6)
    linear._product(linear._XW, x, w, 4, 8, 6, dy)
    linear._slope(dy, dy, torch.float32, 1, torch.float32, True)
    here = [torch.device("cpu")]
    assert asked == [("product", here), ("slope", here)]
