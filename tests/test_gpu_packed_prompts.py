"""The prompt encoder on packed sequences and on a paged cache: several prompts in one pass, new tokens
behind what is kept of a prompt, vs transformers' forward of the same weights (oracle/vl_ref.py).

Tolerance as for the one-prompt form: rel-L2 <= 2e-2 on the last hidden state (every projection
re-rounds to bf16; the oracle stays fp32)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


def _rel(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    return ((a - b).norm() / b.norm()).item()


def _text(seed=0, **kw):
    from oracle import vl_ref as VL
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLTextModel, TextEncoderConfig
    m, sd = VL.tiny_text_model(seed)
    cfg = TextEncoderConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                            num_attention_heads=2, num_key_value_heads=1)
    return m, QwenVLTextModel(cfg, DEV, **kw).load_state_dict(sd)


def test_packed_prompts_vs_transformers():
    from oracle import vl_ref as VL
    m, te = _text()
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (77, 1, 300, 128)]
    got = te.forward_packed(prompts)
    for p, h in zip(prompts, got):
        assert h.shape == (p.numel(), 256) and h.dtype == BF16
        assert _rel(h, VL.text_forward(m, input_ids=p)) <= 2e-2
    # embeddings and 3-D positions among token ids
    emb = (0.5 * torch.randn(90, 256, generator=g)).to(BF16)
    pos = torch.stack([torch.arange(90), torch.arange(90) // 6, torch.arange(90) % 6])
    ids_pos = torch.arange(77).view(1, 77).expand(3, 77)
    a, b = te.forward_packed([emb.to(DEV), prompts[0]], [pos, ids_pos])
    assert _rel(a, VL.text_forward(m, inputs_embeds=emb, position_ids=pos)) <= 2e-2
    assert _rel(b, VL.text_forward(m, input_ids=prompts[0])) <= 2e-2
    assert te.forward_packed([torch.zeros(0, dtype=torch.long)])[0].shape == (0, 256)


def test_packed_attention_switch():
    """``packed_attention`` sends forward the packed way; without it forward stays as it was."""
    from oracle import vl_ref as VL
    m, te = _text(3, packed_attention=True)
    _, old = _text(3)
    ids = torch.randint(0, 1000, (130,), generator=torch.Generator().manual_seed(4))
    want = VL.text_forward(m, input_ids=ids)
    assert _rel(te(ids), want) <= 2e-2 and torch.equal(te(ids), te.forward_packed([ids])[0])
    assert _rel(old(ids), want) <= 2e-2


def test_extend_over_the_cache_vs_transformers():
    """Prompts, then chunks and single tokens of both sequences: every row as in the whole sequence."""
    from oracle import vl_ref as VL
    m, te = _text(1)
    g = torch.Generator().manual_seed(2)
    ids = [torch.randint(0, 1000, (n,), generator=g) for n in (150, 90)]
    want = [VL.text_forward(m, input_ids=i) for i in ids]
    cache = te.new_cache(pages=20, page_size=16)
    seqs = [cache.add(), cache.add()]
    have, rows = [0, 0], [[], []]
    for step in ([100, 33], [1, 1], [17, 30], [0, 1], [32, 25]):
        got = te.extend(cache, seqs, [ids[b][have[b]:have[b] + n] for b, n in enumerate(step)])
        for b, n in enumerate(step):
            rows[b].append(got[b])
            have[b] += n
    assert have == [150, 90] and [cache.length(s) for s in seqs] == have
    for b in range(2):
        assert _rel(torch.cat(rows[b]), want[b]) <= 2e-2
    # a fork in the middle of a page goes another way; the first sequence stays as it was
    other = torch.cat([ids[0][:70], torch.randint(0, 1000, (20,), generator=g)])
    f = cache.fork(seqs[0], 70)
    got = te.extend(cache, [f], [other[70:]])[0]
    assert _rel(got, VL.text_forward(m, input_ids=other)[70:]) <= 2e-2
    more = torch.randint(0, 1000, (3,), generator=g)
    with pytest.raises(ValueError):  # a refused call leaves the sequence as it was
        te.extend(cache, [seqs[0]], [more], [torch.zeros(3, 4, dtype=torch.long)])
    lin, te.lin = te.lin, None  # a forward that fails on its way does, too
    with pytest.raises(AttributeError):
        te.extend(cache, [seqs[0]], [more])
    te.lin = lin
    got = te.extend(cache, [seqs[0]], [more])[0]
    assert _rel(got, VL.text_forward(m, input_ids=torch.cat([ids[0], more]))[150:]) <= 2e-2


def _vision_cfg():
    from qwen_image_edit_streamdiffusion_amd.vision import VisionConfig
    return VisionConfig(depth=4, hidden_size=320, intermediate_size=200, num_heads=4, out_hidden_size=256,
                        fullatt_block_indexes=(1, 3))


def _encoder(seed, **kw):
    from oracle import vl_ref as VL
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLEncoder, TextEncoderConfig
    m, sd = VL.tiny_vl_model(seed)
    enc = QwenVLEncoder(TextEncoderConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                          num_attention_heads=2, num_key_value_heads=1),
                        _vision_cfg(), DEV, image_token_id=990, **kw).load_state_dict(sd)
    return m, sd, enc


@pytest.mark.parametrize("grid", [[(1, 20, 28)], [(1, 16, 16), (1, 8, 12)]])
def test_vision_tower_packed_vs_transformers(grid):
    from oracle import vl_ref as VL
    from qwen_image_edit_streamdiffusion_amd.vision import QwenVLVisionTower
    m, sd = VL.tiny_vl_model(1)
    tower = QwenVLVisionTower(_vision_cfg(), DEV, packed_attention=True).load_state_dict(sd)
    S = sum(t * h * w for t, h, w in grid)
    pv = torch.randn(S, 1176, generator=torch.Generator().manual_seed(S))
    got = tower(pv, grid)
    want = VL.vision_forward(m, pv, torch.tensor(grid))
    assert got.shape == want.shape and _rel(got, want) <= 2e-2


def _prompt(g, tail, image=140):
    return torch.cat([torch.arange(70) + 5, torch.tensor([992]), torch.full((image,), 990), torch.tensor([993]),
                      torch.randint(0, 900, (tail,), generator=g)])


def test_encoder_batch_vs_transformers():
    from oracle import vl_ref as VL
    m, _, enc = _encoder(2, packed_attention=True)
    g = torch.Generator().manual_seed(8)
    grid = torch.tensor([[1, 20, 28]])
    pv = torch.randn(560, 1176, generator=g)
    a, b, c = _prompt(g, 25), _prompt(g, 3), torch.arange(40)
    got = enc.forward_batch([(a, pv, grid), (c, None, None), (b, pv, grid)])
    for h, (ids, x) in zip(got, [(a, pv), (c, None), (b, pv)]):
        want = VL.vl_forward(m, ids, x, grid if x is not None else None)[0]
        assert h.shape == want.shape and _rel(h, want) <= 2e-2


def test_prefix_cache_vs_transformers():
    """A new instruction behind the same template and picture runs only its own tokens; another picture only
    what lies behind the text before it; the kept prompts are evicted in order."""
    from oracle import vl_ref as VL
    m, sd, enc = _encoder(2, prefix_cache_size=2)
    g = torch.Generator().manual_seed(9)
    grid = torch.tensor([[1, 20, 28]])
    pv, pv2 = torch.randn(560, 1176, generator=g), torch.randn(560, 1176, generator=g)
    ran = []
    extend = enc.text.extend
    enc.text.extend = lambda c, s, t, p=None: ran.append(int(t[0].shape[0])) or extend(c, s, t, p)
    a, b = _prompt(g, 25), _prompt(g, 41)
    for ids, x, rows in ((a, pv, 237), (b, pv, 41), (a, pv, 0), (a, pv2, 166), (b, pv, 41)):
        before = len(ran)
        got = enc(ids, x, grid)
        want = VL.vl_forward(m, ids, x, grid)[0]
        assert got.shape == want.shape and _rel(got, want) <= 2e-2
        got.zero_()  # the caller's own rows: what is kept stays as it is
        new = sum(ran[before:])
        if rows == 0:
            assert new == 0
        elif ids is b:  # the common tokens of two random tails may be one or two more
            assert rows - 3 <= new <= rows
        else:
            assert new == rows
    assert len(enc.prefixes) <= 2
    held = enc.kv.num_pages - enc.kv.free_pages
    assert 0 < held <= 2 * (-(-253 // 64))
    enc.load_state_dict(sd)  # other weights: nothing is kept
    assert not enc.prefixes and enc.kv.free_pages == enc.kv.num_pages
    # a prompt longer than the cache still goes through
    m2, _, tiny = _encoder(2, prefix_cache_size=1, prefix_cache_pages=3)
    assert _rel(tiny(a, pv, grid), VL.vl_forward(m2, a, pv, grid)[0]) <= 2e-2 and not tiny.prefixes
    assert _rel(tiny(torch.arange(100)), VL.vl_forward(m2, torch.arange(100))[0]) <= 2e-2 and len(tiny.prefixes) == 1


def test_prompt_hook_batches_prompts():
    """QwenImageEditPromptEncoder on a list of prompts: one pass, padded as before."""
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenImageEditPromptEncoder
    _, _, enc = _encoder(5, packed_attention=True)
    _, _, one = _encoder(5)
    ids = {"long": torch.arange(100) + 3, "short": torch.arange(80) + 7}

    class Proc:
        def __call__(self, text, images=None, return_tensors=None):
            i = ids["long" if "long" in text[0] else "short"]
            return {"input_ids": i.view(1, -1), "attention_mask": torch.ones(1, i.numel(), dtype=torch.long)}

    calls = []
    batch = enc.forward_batch
    enc.forward_batch = lambda p: calls.append(len(p)) or batch(p)
    e, mask = QwenImageEditPromptEncoder(enc, Proc())(["long", "short"])
    w, wmask = QwenImageEditPromptEncoder(one, Proc())(["long", "short"])
    assert calls == [2] and torch.equal(mask, wmask) and e.shape == w.shape == (2, 36, 256)
    assert _rel(e, w) <= 2e-2 and (e[1, 16:] == 0).all()


def test_full_width_layer_packed():
    """Qwen2.5-VL-7B widths, one text layer: two prompts packed and a chunk over the cache."""
    from oracle import vl_ref as VL
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLTextModel, TextEncoderConfig
    m, sd = VL.tiny_text_model(7, hidden=3584, heads=28, kv_heads=4, layers=1, intermediate=18944)
    te = QwenVLTextModel(TextEncoderConfig(vocab_size=1000, hidden_size=3584, intermediate_size=18944, num_hidden_layers=1,
                                           num_attention_heads=28, num_key_value_heads=4), DEV).load_state_dict(sd)
    g = torch.Generator().manual_seed(1)
    a, b = torch.randint(0, 1000, (300,), generator=g), torch.randint(0, 1000, (45,), generator=g)
    wa, wb = VL.text_forward(m, input_ids=a), VL.text_forward(m, input_ids=b)
    ga, gb = te.forward_packed([a, b])
    assert _rel(ga, wa) <= 2e-2 and _rel(gb, wb) <= 2e-2
    cache = te.new_cache(8)
    s = cache.add()
    first = te.extend(cache, [s], [a[:259]])[0]
    rest = te.extend(cache, [s], [a[259:]])[0]
    assert _rel(torch.cat([first, rest]), wa) <= 2e-2
