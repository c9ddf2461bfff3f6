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


def test_a_prompt_that_does_not_fit_beside_what_it_shares_is_kept_instead(encoder):
    """Two prompts of more than half the pool that begin alike: the second one runs whole once, then it is kept."""
    enc = encoder(1)
    a = _ids(1100, 7)
    b = torch.cat([a[:70], _ids(1030, 8)])
    common = int((a != b).nonzero()[0])
    assert enc.prefix_pages == 32 and _ask(enc, a) == [1100] and common >= 70
    assert _ask(enc, b) == [1100]
    assert _ask(enc, b) == [] and _ask(enc, b) == [] and enc.kv.free_pages == 32 - 18
    c = torch.cat([a[:70], _ids(50, 9)])  # beside it there is room for this one
    assert _ask(enc, c) in ([120 - n] for n in range(70, 74))


def test_kept_prompts_beside_it_stay_where_they_fit(encoder):
    """Of three kept prompts only the one that blocks a longer one goes."""
    enc = encoder(4, pages=32)
    small, other, a = _ids(100, 10), _ids(120, 11), _ids(1100, 12)
    assert [_ask(enc, x) for x in (small, other, a)] == [[100], [120], [1100]]
    b = torch.cat([a[:70], _ids(1400, 13)])  # 23 pages: 22 beside a's 18 never fit, 23 beside the two others do
    assert _ask(enc, b) == [1470]
    assert _ask(enc, small) == _ask(enc, other) == _ask(enc, b) == [] and len(enc.prefixes) == 3


def test_a_prompt_longer_than_the_pool_leaves_the_kept_ones(encoder):
    enc = encoder(4)
    kept = [_ids(200 + i, 20 + i) for i in range(4)]
    for x in kept:
        _ask(enc, x)
    free = enc.kv.free_pages
    for long in (_ids(6000, 30), torch.cat([kept[1][:150], _ids(6000, 31)])):
        assert _ask(enc, long) == [len(long)]
        assert enc.kv.free_pages == free and len(enc.prefixes) == 4
    assert [_ask(enc, x) for x in kept] == [[]] * 4


def test_a_call_that_fails_at_its_end_holds_no_pages(encoder):
    """What is shared and the new rows no longer fit into memory together: the new sequence goes."""
    enc = encoder(2)
    a = _ids(300, 40)
    b = torch.cat([a[:192], _ids(100, 41)])
    assert _ask(enc, a) == [300]
    free, kept = enc.kv.free_pages, next(iter(enc.prefixes.values()))
    hidden, kept.hidden = kept.hidden, kept.hidden[:, :2]  # rows that do not go with the new ones
    with pytest.raises(RuntimeError):
        enc(b)
    assert enc.kv.free_pages == free and len(enc.prefixes) == 1
    kept.hidden = hidden
    assert _ask(enc, b) in ([100], [99], [98]) and _ask(enc, a) == []


def test_the_size_may_be_set_after_the_load(encoder):
    """On the encoder that a pipeline holds: pages for that many prompts, as if it had been made so."""
    enc = encoder(0)
    enc.prefix_cache_size = 3
    assert enc.prefix_pages == 16 * 4
    a, b = _ids(900, 50), _ids(800, 51)
    assert [_ask(enc, x) for x in (a, b, a, b)] == [[900], [800], [], []]
    assert encoder(3, pages=5).prefix_pages == 5
