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


def test_step_whose_arrays_fail_counts_nothing():
    """No room on the device for the step's arrays."""
    c = PagedKVCache(1, 1, 64, 8, 16, "cpu")
    a, b = c.add(), c.add()
    c.step([a, b], [20, 16])
    before, device = _state(c), c.device

    class Full:
        def __init__(self, left):
            self.left = left

        def __call__(self, values, dtype=None):
            self.left -= 1
            if self.left < 0:
                raise RuntimeError("out of memory")
            return torch.Tensor.new_tensor(torch.empty(0), values, dtype=dtype)
    for left in range(4):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(kv_cache.torch, "tensor", Full(left))
            with pytest.raises(RuntimeError):
                c.step([b, a], [30, 40])
        assert _state(c) == before and c.device is device, left
    st = c.step([b, a], [30, 40])
    assert st.kv_lens.tolist() == [46, 60] and c.free_pages == 1


@pytest.mark.parametrize("new", [[1, -1], [True, 2.5], [2.0, 1]])
def test_step_refuses_counts_that_are_none(new):
    c = PagedKVCache(1, 1, 64, 8, 16, "cpu")
    a, b = c.add(), c.add()
    before = _state(c)
    with pytest.raises((ValueError, TypeError)):
        c.step([a, b], new)
    assert _state(c) == before
    with pytest.raises(KeyError):
        c.step([a, 99], [1, 1])
    assert _state(c) == before
