"""PagedKVCache on the host where a step or a fork fails half way."""
import pytest
import torch

from qwen_image_edit_streamdiffusion_amd import kv_cache
from qwen_image_edit_streamdiffusion_amd.kv_cache import PagedKVCache


def _state(c):
    return c.free_pages, list(c._free), list(c._users), {s: (list(v.pages), v.length) for s, v in c._seqs.items()}


@pytest.mark.parametrize("fails", [1, 2])
def test_fork_whose_copy_fails_holds_nothing(monkeypatch, fails):
    c = PagedKVCache(2, 1, 64, 8, 16, "cpu")
    a = c.add()
    c.step([a], [40])
    before, calls = _state(c), []

    def copy(s, d):
        calls.append(1)
        if len(calls) >= fails:
            raise RuntimeError("no device")
        d.copy_(s)
    monkeypatch.setattr(kv_cache.ops, "copy_batched", copy)
    with pytest.raises(RuntimeError):
        c.fork(a, 37)
    assert _state(c) == before
    f = c.fork(a, 32)  # whole pages: nothing to copy
    assert c.length(f) == 32 and c.free_pages == 5
