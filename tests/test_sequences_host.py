"""Host side of the sequence operators: the turns and axes of the rotary layouts against the framework's
own tables, and what the C entry points refuse before any launch."""
import ctypes
import math
import os

import pytest
import torch

from qwen_image_edit_streamdiffusion_amd.rope import axes_turns, rope_angles, section_turns

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from qwen_image_edit_streamdiffusion_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import subprocess
        subprocess.run(["make", "-C", os.path.join(ROOT, "qwen_image_edit_streamdiffusion_amd", "csrc"), "-j8"],
                       check=True, capture_output=True)
    return _lib.load()


def test_turns_are_the_models_angles():
    from qwen_image_edit_streamdiffusion_amd.text_encoder import TextEncoderConfig, mrope_tables
    cfg = TextEncoderConfig(hidden_size=256, num_attention_heads=2, num_key_value_heads=1)
    pos = torch.stack([torch.arange(40), torch.arange(40) * 2 % 17, torch.arange(40) * 3 % 11])
    turns, axis = section_turns(cfg.mrope_section, cfg.rope_theta, "cpu")
    ang = 2 * math.pi * pos.double()[axis.long()].T * turns
    cos, _ = mrope_tables(cfg, pos)
    # bf16 tables of fp32 angles: half a bf16 step, and 2^-24 * 40 rad of the angle
    assert ((ang.cos() - cos[:, :64].double()).abs() <= 2.0 ** -8 + 1e-5).all()
    # the image transformer's axes: the same angles as its tables, 32 bits
    img, txt = rope_angles([(1, 6, 4)], 5)
    turns, axis = axes_turns((16, 56, 56), 10000.0, "cpu")
    hh, ww = torch.arange(6) - 3, torch.arange(4) - 2
    p = torch.stack([torch.zeros(24), hh[:, None].expand(6, 4).reshape(-1), ww.repeat(6)])
    ang = 2 * math.pi * p.double()[axis.long()].T * turns
    assert torch.allclose(ang, img.double(), rtol=1e-6, atol=1e-6)


def test_entry_points_refuse_on_the_host(lib):
    """Null pointers, shapes, strides, alignment: QIE_ERR_INVALID, nothing launched."""
    ok = dict(x=16, ldx=512, out=16, ldo=512, rows=4, heads=4, dh=128, hs=128, pos=16, ldp=4, axes=3, turns=16, axis=16,
              pairs=64)

    def rope(**kw):
        a = {**ok, **kw}
        return lib.qie_rope_axes_bf16(a["x"], a["ldx"], a["out"], a["ldo"], a["rows"], a["heads"], a["dh"], a["hs"],
                                      a["pos"], a["ldp"], a["axes"], a["turns"], a["axis"], a["pairs"], 0, None)
    for kw in (dict(x=None), dict(out=None), dict(pos=None), dict(turns=None), dict(axis=None), dict(rows=-1), dict(heads=0),
               dict(pairs=0), dict(pairs=65), dict(pairs=129, dh=512, hs=512), dict(axes=0), dict(ldp=3), dict(hs=127),
               dict(hs=64), dict(ldx=511), dict(ldx=510), dict(ldo=256), dict(x=18), dict(turns=20)):
        assert rope(**kw) == -1, kw
    assert rope(rows=0) == 0  # nothing to do

    ok2 = dict(x=16, ldx=768, out=16, ldo=512, rows=4, H=4, Hk=1, dh=128, pos=16, ldp=4, axes=3, turns=16, axis=16, pairs=64,
               k=16, v=16, N=2, P=16, ps=2048, hs=2048, ss=128, slots=16)

    def app(**kw):
        a = {**ok2, **kw}
        return lib.qie_rope_append_bf16(a["x"], a["ldx"], a["out"], a["ldo"], a["rows"], a["H"], a["Hk"], a["dh"], a["pos"],
                                        a["ldp"], a["axes"], a["turns"], a["axis"], a["pairs"], 0, a["k"], a["v"], a["N"],
                                        a["P"], a["ps"], a["hs"], a["ss"], a["slots"], None)
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(N=0), dict(P=8), dict(P=24), dict(P=2048), dict(ss=120),
               dict(ss=132), dict(k=24), dict(ldx=760), dict(ldx=772), dict(ldo=500), dict(Hk=0), dict(dh=124, pairs=32)):
        assert app(**kw) == -1, kw

    ok3 = dict(q=16, ldq=512, hsq=128, k=16, v=16, ldk=128, hsk=128, cu=16, B=1, T=4, H=4, Hk=1, dh=128, sc=0.1, out=16,
               ldo=512, hso=128)

    def packed(**kw):
        a = {**ok3, **kw}
        return lib.qie_attention_packed_bf16(a["q"], a["ldq"], a["hsq"], a["k"], a["v"], a["ldk"], a["hsk"], a["cu"], a["B"],
                                             a["T"], a["H"], a["Hk"], a["dh"], 1, a["sc"], a["out"], a["ldo"], a["hso"], None)
    refused = (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(B=0), dict(T=-1), dict(H=0), dict(Hk=0),
               dict(Hk=3), dict(dh=0), dict(dh=136), dict(dh=60), dict(sc=0.0), dict(sc=-1.0), dict(sc=math.inf), dict(sc=65537.0),
               dict(sc=math.nan), dict(q=24), dict(ldq=516), dict(ldk=64), dict(hso=64), dict(T=1 << 30))
    for kw in refused + (dict(cu=None),):
        assert packed(**kw) == -1, kw
    assert packed(T=0) == 0

    ok4 = dict(ok3, N=4, P=16, ps=2048, hsk=2048, table=16, ldt=4096, W=4096, kvl=16, ws=16, wsb=1 << 40)

    def paged(**kw):
        a = {**ok4, **kw}
        return lib.qie_attention_paged_bf16(a["q"], a["ldq"], a["hsq"], a["k"], a["v"], a["N"], a["P"], a["ps"], a["hsk"],
                                            a["ldk"], a["table"], a["ldt"], a["W"], a["kvl"], a["cu"], a["B"], a["T"], a["H"],
                                            a["Hk"], a["dh"], a["sc"], a["out"], a["ldo"], a["hso"], a["ws"], a["wsb"], None)
    for kw in refused + (dict(table=None), dict(kvl=None), dict(cu=None), dict(N=0), dict(P=8), dict(P=48), dict(P=2048),
                         dict(ps=2052), dict(W=0), dict(ldt=4095), dict(W=1 << 27, ldt=1 << 27), dict(ws=None), dict(wsb=64),
                         dict(ws=20)):
        assert paged(**kw) == -1, kw
    n = ctypes.c_int64(-1)
    assert lib.qie_attention_paged_workspace(4, 1, 4, 1, 128, 1, 16, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.qie_attention_paged_workspace(4, 1, 4, 1, 128, 4096, 16, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.qie_attention_paged_workspace(4, 1, 4, 1, 128, 4096, 16, None) == -1


def test_calls_refuse_host_tensors_and_other_objects():
    """The native calls take device tensors only, and say which argument is none."""
    from qwen_image_edit_streamdiffusion_amd import ops
    from qwen_image_edit_streamdiffusion_amd.rope import section_turns
    turns, axis = section_turns((16, 24, 24), 1e6, "cpu")
    x = torch.zeros(4, 768, dtype=torch.bfloat16)
    q, pages = x[:, :512].unflatten(1, (4, 128)), torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16)
    pos, cu = torch.zeros(3, 4, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    for fn in (lambda: ops.rope_axes(x, 0, 4, 128, pos, turns, axis), lambda: ops.attention_packed(q, q, q, cu),
               lambda: ops.rope_append(x, 4, 1, 128, pos, turns, axis, pages, pages, torch.arange(4)),
               lambda: ops.attention_paged(q, pages, pages, pos, cu)):
        with pytest.raises(ValueError):
            fn()
    for fn in (lambda: ops.rope_axes([1.0], 0, 4, 128, pos, turns, axis), lambda: ops.attention_packed(None, q, q, cu),
               lambda: ops.attention_paged(q.numpy, pages, pages, pos, cu)):
        with pytest.raises(TypeError):
            fn()


# ---------------------------------------------------------------------------- the cache's pages
def _cache(pages=8):
    from qwen_image_edit_streamdiffusion_amd.kv_cache import PagedKVCache
    return PagedKVCache(2, 1, 64, pages, 16, "cpu")


def test_paged_cache_steps_and_pages():
    c = _cache()
    a, b = c.add(), c.add()
    st = c.step([a, b], [20, 1])
    assert c.free_pages == 5 and c.length(a) == 20 and c.length(b) == 1
    assert st.kv_lens.tolist() == [20, 1] and st.cu_seqlens.tolist() == [0, 20, 21] and st.page_table.shape == (2, 2)
    t = st.page_table
    want = [int(t[0, i // 16]) * 16 + i % 16 for i in range(20)] + [int(t[1, 0]) * 16]
    assert st.slots.tolist() == want and len(set(want)) == 21
    st2 = c.step([b, a], [0, 12])  # a's second page fills up to its end
    assert c.free_pages == 5 and st2.kv_lens.tolist() == [1, 32] and st2.slots.numel() == 12
    assert st2.slots.tolist() == [int(t[0, 1]) * 16 + i for i in range(4, 16)]
    c.drop(a)
    assert c.free_pages == 7
    with pytest.raises(KeyError):
        c.length(a)


def test_paged_cache_takes_a_step_back():
    c = _cache()
    a, b = c.add(), c.add()
    c.step([a, b], [20, 16])
    before = c.free_pages, list(c._free)
    st = c.step([a, b], [40, 3])
    c.take_back([a, b], [40, 3])
    assert (c.free_pages, c.length(a), c.length(b)) == (before[0], 20, 16)
    again = c.step([a, b], [40, 3])
    assert again.slots.tolist() == st.slots.tolist() and again.page_table.tolist() == st.page_table.tolist()
    with pytest.raises(ValueError):
        c.take_back([b], [20])
    c.fork(a, 48)  # a's third page is shared now
    with pytest.raises(ValueError):
        c.take_back([a], [40])
    assert c.length(a) == 60


def test_paged_cache_shared_pages_and_refusals():
    from qwen_image_edit_streamdiffusion_amd.kv_cache import CacheFull, PagedKVCache
    c = _cache(4)
    a = c.add()
    c.step([a], [40])  # three pages
    f = c.fork(a, 32)  # two of them shared
    assert c.free_pages == 1 and c.length(f) == 32
    with pytest.raises(CacheFull):
        c.step([a, f], [16, 1])
    assert c.length(a) == 40 and c.length(f) == 32 and c.free_pages == 1  # a refused step changes nothing
    st = c.step([f, a], [3, 2])
    assert st.page_table[0, :2].tolist() == st.page_table[1, :2].tolist()
    assert int(st.page_table[0, 2]) != int(st.page_table[1, 2])
    c.drop(a)
    assert c.free_pages == 1  # the shared pages stay with the fork
    c.drop(f)
    assert c.free_pages == 4
    for bad in (lambda: c.fork(c.add(), 1), lambda: c.step([], []), lambda: c.step([1, 1], [1, 1]),
                lambda: PagedKVCache(1, 1, 64, 4, 24, "cpu"), lambda: PagedKVCache(1, 1, 60, 4, 16, "cpu")):
        with pytest.raises((ValueError, KeyError)):
            bad()


def test_paged_cache_takes_back_only_tokens_of_its_own():
    c = _cache()
    a, b = c.add(), c.add()
    c.step([a, b], [28, 5])
    c.step([a], [4])  # a's second page fills up to its end
    f = c.fork(a, 32)  # and is shared
    state = lambda: (c.free_pages, c.length(a), c.length(b), c.length(f))  # noqa: E731
    before = state()
    for bad in (([a], [4]), ([a], [1]), ([b, b], [2, 2]), ([b], [2, 2]), ([b], [-1])):
        with pytest.raises(ValueError):
            c.take_back(*bad)
        assert state() == before, bad  # a refused one changes nothing
    c.take_back([a, b], [0, 5])  # no token of a
    assert (c.length(a), c.length(b), c.free_pages) == (32, 0, 6)
    c.step([f], [3])
    c.take_back([f], [3])  # tokens behind the shared pages
    assert (c.length(f), c.free_pages) == (32, 6)
