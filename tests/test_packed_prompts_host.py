"""The packed form of the prompt encoder's language model on the host: what its calls take."""
import pytest
import torch


@pytest.fixture
def model():
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLTextModel, TextEncoderConfig
    te = QwenVLTextModel(TextEncoderConfig(vocab_size=100, hidden_size=256, intermediate_size=512, num_hidden_layers=1,
                                           num_attention_heads=2, num_key_value_heads=1), "cpu", packed_attention=True)
    te.layers = [{}]
    te.seen = []

    def rows(prompts, position_ids, lens, attend):
        te.seen.append([p.tolist() for p in position_ids])
        return torch.zeros(sum(lens), 256)
    te._rows = rows
    return te


def test_positions_of_one_row_serve_all_axes(model):
    """forward takes the positions that its default form takes."""
    ids = torch.arange(5)
    row = torch.tensor([4, 5, 6, 7, 9])
    three = torch.stack([row, row + 1, row + 2])
    for given, want in ((row, [row.tolist()] * 3), (row[None], [row.tolist()] * 3), (three, three.tolist()),
                        (None, [list(range(5))] * 3)):
        model(ids, given)
        assert model.seen[-1] == [want]
    for bad in (row[:4], three[:, :4], three[:2], torch.zeros(1, 3, 5)):
        with pytest.raises(ValueError):
            model(ids, bad)
    with pytest.raises(ValueError):
        model.forward_packed([ids, ids], [row])
    cache = model.new_cache(2)
    s = cache.add()
    with pytest.raises(ValueError):
        model.extend(cache, [s], [ids], [row[:4]])
    assert cache.length(s) == 0


def test_the_encoders_switch_is_its_models():
    """Set after the load, as on the encoder that a pipeline holds: both models and the batch follow."""
    from qwen_image_edit_streamdiffusion_amd.text_encoder import QwenVLEncoder, TextEncoderConfig
    from qwen_image_edit_streamdiffusion_amd.vision import VisionConfig
    make = lambda **kw: QwenVLEncoder(  # noqa: E731
        TextEncoderConfig(vocab_size=100, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=2,
                          num_key_value_heads=1),
        VisionConfig(depth=1, hidden_size=320, intermediate_size=200, num_heads=4, out_hidden_size=256, fullatt_block_indexes=(0,)),
        "cpu", **kw)
    state = lambda e: (e.packed_attention, e.text.packed_attention, e.vision.packed_attention)  # noqa: E731
    enc = make()
    assert state(enc) == (False, False, False)
    enc.packed_attention = True
    assert state(enc) == (True, True, True)
    enc.packed_attention = False
    assert state(enc) == (False, False, False)
    assert state(make(packed_attention=True)) == (True, True, True)
