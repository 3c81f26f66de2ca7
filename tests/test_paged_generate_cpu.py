"""generate_paged captures and replays its graph on the model's device, whatever device is current."""
import torch

from test_paged_model_cpu import cpu_model, prompts_of  # noqa: F401 (a fixture)


def test_the_graph_belongs_to_the_models_device(cpu_model, monkeypatch):  # noqa: F811
    current, seen = ["other"], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *exc):
            current.pop()

    class Graph:
        def __init__(self, graph=None):
            pass

        def __enter__(self):
            seen.append(("capture", current[-1]))

        def __exit__(self, *exc):
            pass

        def replay(self):
            seen.append(("replay", current[-1]))

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", Graph)
    device = torch.device("cpu")
    outs = cpu_model.generate_paged(prompts_of(3, 5), 4, use_cuda_graph=True)
    assert [len(x) for x in outs] == [7, 9]
    assert seen == [("capture", device), ("replay", device), ("replay", device)] and current == ["other"]
