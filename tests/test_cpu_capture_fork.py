"""The stream that every capture of a step forks one node onto is never the capture's own (torch's pool of streams wraps)."""
import torch


def test_the_fork_is_another_stream(monkeypatch):
    from graphgps_amd import train

    class Stream:
        drawn = 0

        def __init__(self, device=None):
            self.device, self.cuda_stream = device, 1000 + Stream.drawn % 32
            Stream.drawn += 1
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    cur = Stream("cuda:0")
    for _ in range(100):
        side = train._fork_stream(cur)
        assert side.cuda_stream != cur.cuda_stream and side.device == "cuda:0"
