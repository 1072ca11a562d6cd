"""The examples of README.md: what they name exists, and calls that return before their work is done name the stream of the tensors."""
import inspect
import os
import re

import pytest

from juno_b200 import matvec

README = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")


def cache_example():
    with open(README) as f:
        found = [b for b in re.findall(r"```python\n(.*?)```", f.read(), re.S) if "PagedKvCache" in b]
    assert len(found) == 1
    return found[0]


def test_the_cache_example_names_the_stream_of_its_tensors(monkeypatch):
    torch = pytest.importorskip("torch")
    calls, real = [], matvec.PagedKvCache

    class Cache:
        def __init__(self, *args, **kw):
            inspect.signature(real.__init__).bind(self, *args, **kw)

        def __getattr__(self, name):
            def call(*args, **kw):
                calls.append((name, inspect.signature(getattr(real, name)).bind(self, *args, **kw).arguments))
                return 4096
            return call

    here = object()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: here)
    monkeypatch.setattr(matvec, "PagedKvCache", Cache)
    monkeypatch.setattr(matvec.GpuContext, "shared", lambda device: None)
    exec(cache_example(), {name: object() for name in ("layer", "pos", "n", "k", "v", "q", "out")})
    moved = [(name, args) for name, args in calls if "stream" in inspect.signature(getattr(real, name)).parameters]
    assert [name for name, _ in moved] == ["append_device", "attention_device", "evict"]
    assert all(args.get("stream") is here for _, args in moved)
