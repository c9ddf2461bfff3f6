"""The prompt encoder's kept prompts on the host: which rows run, which pages are held and what is answered,
on a model whose k is the tokens themselves and whose hidden states count what the pages hold."""
import pytest
import torch

from qwen_image_edit_streamdiffusion_amd import kv_cache
from qwen_image_edit_streamdiffusion_amd.kv_cache import PagedKVCache

P = 64
IMAGE = 199


def answer(ids):
    """Row i: (i + 1, sum of the first i + 1 tokens, the same weighted by their places)."""
    t = ids.double()
    w = torch.arange(1, len(t) + 1, dtype=torch.float64)
    return torch.stack([w, t.cumsum(0), (t * w).cumsum(0)], 1)


class CountingText:
    """Stands for QwenVLTextModel: tokens (below 200, exact in bf16) are written to the pages and read back."""

    def __init__(self, config):
        self.config, self.device, self.w, self.ran = config, torch.device("cpu"), {}, []
        self.packed_attention = False

    def load_state_dict(self, sd):
        return self

    def new_cache(self, pages, page_size=P):
        return PagedKVCache(1, 1, 8, pages, page_size, "cpu")

    @staticmethod
    def _tokens(t):
        return t[:, 0] if t.is_floating_point() else t

    def extend(self, cache, seqs, tokens, position_ids=None):
        st = cache.step(seqs, [len(t) for t in tokens])
        new = self._tokens(tokens[0]).to(torch.bfloat16)
        cache.k[0, st.slots // cache.page_size, 0, st.slots % cache.page_size, 0] = new
        self.ran.append(len(new))
        n = int(st.kv_lens[0])
        held = cache.k[0, st.page_table[0].long(), 0, :, 0].reshape(-1)[:n]
        return [answer(held)[n - len(new):]]

    def forward_packed(self, prompts, position_ids=None):
        self.ran += [len(p) for p in prompts]
        return [answer(self._tokens(p)) for p in prompts]


@pytest.fixture
def encoder(monkeypatch):
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLEncoder, TextEncoderConfig
    from qwen_image_edit_streamdiffusion_amd.vision import VisionConfig
    monkeypatch.setattr(kv_cache.ops, "copy_batched", lambda s, d: d.copy_(s))
    cfg = TextEncoderConfig(vocab_size=200, hidden_size=256, intermediate_size=512, num_hidden_layers=1,
                            num_attention_heads=2, num_key_value_heads=1)

    def make(size, pages=None):
        enc = QwenVLEncoder(cfg, VisionConfig(depth=1, hidden_size=320, intermediate_size=200, num_heads=4, out_hidden_size=256,
                                              fullatt_block_indexes=(0,)), "cpu", image_token_id=IMAGE,
                            prefix_cache_size=size, prefix_cache_pages=pages)
        enc.text = CountingText(cfg)
        enc._embeds = lambda ids, pv, grid: (ids.float()[:, None].expand(-1, 8), enc._positions(ids, pv, grid))
        return enc
    return make


def _ids(n, seed):
    return torch.randint(0, 190, (n,), generator=torch.Generator().manual_seed(seed))


def _ask(enc, ids, *picture):
    """The rows that ran for a prompt; its answer is checked."""
    at = len(enc.text.ran)
    assert torch.equal(enc(ids, *picture), answer(ids))
    return enc.text.ran[at:]


def test_kept_prompts_are_found(encoder):
    enc = encoder(2)
    a = _ids(300, 0)
    b = torch.cat([a[:200], (a[200:201] + 1) % 190, _ids(59, 1)])
    assert _ask(enc, a) == [300] and _ask(enc, b) == [60] and _ask(enc, a) == [] and _ask(enc, b[:100]) == []


def test_the_callers_ids_may_change_after_the_call(encoder):
    """A tokenizer's buffer is used again for the next prompt."""
    enc = encoder(2)
    ids = _ids(120, 2)
    assert _ask(enc, ids) == [120]
    ids[50:] = (ids[50:] + 7) % 190
    assert _ask(enc, ids) == [70]
    ids[0] = (ids[0] + 1) % 190
    assert _ask(enc, ids) == [120]


def test_other_weights_forget_what_the_old_ones_gave(encoder):
    """Kept prompts and kept pictures both."""
    enc = encoder(2)
    enc.vision.load_state_dict = lambda sd: enc.vision
    enc.vision.forward = lambda pv, grid: torch.full((4, 256), float(len(seen)))
    seen, pv, grid = [], torch.zeros(16, 1176), [(1, 4, 4)]
    assert _ask(enc, _ids(80, 3)) == [80] and enc._vision(pv, grid)[0, 0] == 0
    seen.append(1)
    assert enc._vision(pv, grid)[0, 0] == 0  # the same picture
    enc.load_state_dict({})
    assert enc._vision(pv, grid)[0, 0] == 1
    assert _ask(enc, _ids(80, 3)) == [80]


def _picture(value, grid):
    return torch.full((sum(t * h * w for t, h, w in grid), 1176), value), grid


def test_pictures_are_counted_for_a_kept_prompt_too(encoder):
    """A prompt that lacks a picture's tokens is refused, whatever part of it is kept."""
    enc = encoder(4)
    grid = [(1, 4, 4), (1, 8, 4)]  # 4 and 8 tokens
    pv = _picture(1.0, grid)
    run = lambda n: torch.full((n,), IMAGE)  # noqa: E731
    a, b = _ids(70, 4), _ids(30, 5)
    whole = torch.cat([a, run(4), b, run(8), b])
    assert _ask(enc, whole, *pv) == [len(whole)]
    for ids in (whole[:len(a) + 4 + 5], torch.cat([whole[:len(a) + 4], _ids(9, 6)]), whole[:60], whole[:len(a) + 2],
                whole[:len(a) + 4 + len(b) + 3]):
        with pytest.raises(ValueError):
            enc(ids, *pv)
    with pytest.raises(ValueError):  # image tokens without a picture
        enc(whole, None, None)
    assert _ask(enc, whole, *pv) == [] and _ask(enc, torch.cat([whole[:-3], _ids(9, 6)]), *pv) == [9]
    # other pictures of the same sizes: the text before the first one is shared
    assert _ask(enc, whole, *_picture(2.0, grid)) == [len(whole) - len(a)]
