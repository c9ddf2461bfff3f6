"""Rotary positions with several axes, the paged cache's write, packed attention and attention over a
paged cache, each vs its formula in 64 bits on the same bf16 inputs.

Tolerances (h = 2^-8, half a bf16 step relative to a value):
  * a rotation: h |want| for its one rounding, and 2^-20 (|x| + |y|) for its fp32 cos, sin (angles
    correct to 2^-24 turns, i.e. 2^-21) and products
  * attention, per element: h |want| for the last rounding; P rounded to bf16 moves every term by at
    most h, i.e. the sum by h sum_j p_j |v_j|; fp32 logits up to 2^6 of 128 products are off by at
    most 2^-12 in all, which moves sum_j p_j |v_j| by 2^-11 at most
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"
H8 = 2.0 ** -8


def _ops():
    from qwen_image_edit_streamdiffusion_amd import ops
    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *s):
    return torch.randn(*s, generator=g).to(BF16)


# ---------------------------------------------------------------------------- formulas
def rope_ref(x, pos, turns, axis, interleaved):
    """x [T, heads, Dh] -> float64 rotated."""
    x = x.double()
    n = turns.numel()
    ang = 2 * math.pi * torch.remainder(pos.double()[axis.long()].T * turns, 1.0)[:, None]
    c, s = ang.cos(), ang.sin()
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = a * c - b * s, b * c + a * s
        mag = out.clone().zero_()
        mag[..., 0:2 * n:2] = mag[..., 1:2 * n:2] = a.abs() + b.abs()
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        out[..., :n], out[..., n:2 * n] = a * c - b * s, b * c + a * s
        mag = out.clone().zero_()
        mag[..., :n] = mag[..., n:2 * n] = a.abs() + b.abs()
    return out, H8 * out.abs() + 2.0 ** -20 * mag


def attn_ref(q, k, v, lim, scale):
    """One sequence: q [n, H, Dh] sees the first lim[i] rows of k, v [K, Hk, Dh] -> (o, tolerance), float64."""
    n, H, Dh = q.shape
    K, Hk = k.shape[:2]
    o, tol = torch.zeros(n, H, Dh, dtype=torch.float64), torch.zeros(n, H, Dh, dtype=torch.float64)
    for h in range(H):
        kk, vv = k[:, h * Hk // H].double(), v[:, h * Hk // H].double()
        for i0 in range(0, n, 512):
            li = lim[i0:i0 + 512]
            m = int(li.max()) if li.numel() else 0
            if m <= 0:
                continue
            s = q[i0:i0 + 512, h].double() @ kk[:m].T * scale
            seen = torch.arange(m)[None] < li[:, None]
            p = torch.exp(s - s.masked_fill(~seen, -1e300).amax(1, keepdim=True)).masked_fill(~seen, 0)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            o[i0:i0 + 512, h] = p @ vv[:m]
            tol[i0:i0 + 512, h] = p @ vv[:m].abs()
    return o, H8 * o.abs() + (H8 + 2.0 ** -11) * tol


def packed_ref(q, k, v, lens, causal, scale=None):
    sc = scale or 1 / math.sqrt(q.shape[-1])
    os_, ts, at = [], [], 0
    for n in lens:
        lim = torch.arange(1, n + 1) if causal else torch.full((n,), n)
        o, t = attn_ref(q[at:at + n], k[at:at + n], v[at:at + n], lim, sc)
        os_.append(o)
        ts.append(t)
        at += n
    return torch.cat(os_), torch.cat(ts)


def _cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


def _check(got, want, tol):
    d = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = (d - tol).max().item() if d.numel() else 0.0
    assert worst <= 0, f"{worst:.3e} over the bound; max error {d.max().item():.3e}"


# ---------------------------------------------------------------------------- rope
PLANS = {"sections": ((16, 24, 24), False), "one": ((64,), False), "grid": ((20, 20), False), "inter": ((8, 28, 28), True),
         "odd": ((9, 9, 18), False), "odd-inter": ((5, 7, 9), True), "wide": ((64, 32, 32), False), "tiny": ((1,), True)}


def _plan(name):
    from qwen_image_edit_streamdiffusion_amd.rope import axes_turns, section_turns
    runs, inter = PLANS[name]
    turns, axis = section_turns(runs, 1e6, "cpu") if name in ("sections", "one") else axes_turns([2 * r for r in runs], 1e4, "cpu")
    return turns, axis, len(runs), inter


@pytest.mark.parametrize("name", list(PLANS))
@pytest.mark.parametrize("T,nh,extra", [(1, 1, 0), (7, 5, 6), (2051, 3, 0)])
def test_rope_axes(name, T, nh, extra):
    """Every layout, in place and into another buffer, with columns that pass through and slots apart."""
    ops = _ops()
    turns, axis, axes, inter = _plan(name)
    Dh = 2 * turns.numel() + extra
    hs = Dh + 2
    g = _gen(T + nh)
    x = _randn(g, T, (nh + 2) * hs)
    pos = torch.randint(-70000, 300000, (axes, T), generator=g, dtype=torch.int32)
    heads = x[:, hs:(nh + 1) * hs].reshape(T, nh, hs)
    want, tol = rope_ref(heads[..., :Dh], pos, turns, axis, inter)
    d = lambda t: t.to(DEV)  # noqa: E731
    xd = d(x)
    out = torch.full((T, nh * hs + 4), 7.0, dtype=BF16, device=DEV)
    r = ops.rope_axes(xd, 1, nh, Dh, d(pos), d(turns), d(axis), interleaved=inter, head_stride=hs, out=out)
    assert r is out and torch.equal(xd.cpu(), x)
    got = out[:, :nh * hs].cpu().reshape(T, nh, hs)
    _check(got[..., :Dh], want, tol)
    assert torch.equal(got[..., 2 * turns.numel():Dh], heads[..., 2 * turns.numel():Dh])
    assert (got[..., Dh:] == 7).all() and (out[:, nh * hs:] == 7).all()
    ops.rope_axes(xd, 1, nh, Dh, d(pos), d(turns), d(axis), interleaved=inter, head_stride=hs)
    got2 = xd.cpu()
    assert torch.equal(got2[:, hs:(nh + 1) * hs].reshape(T, nh, hs)[..., :Dh], got[..., :Dh])
    assert torch.equal(got2[:, :hs], x[:, :hs]) and torch.equal(got2[:, (nh + 1) * hs:], x[:, (nh + 1) * hs:])
    assert torch.equal(got2[:, hs:(nh + 1) * hs].reshape(T, nh, hs)[..., Dh:], heads[..., Dh:])


def test_rope_axes_equals_the_models_own_tables():
    """The language model's 3-D positions: within bf16 tables' rounding of ops.rope_half."""
    ops = _ops()
    from qwen_image_edit_streamdiffusion_amd.text_encoder import TextEncoderConfig, mrope_tables
    from qwen_image_edit_streamdiffusion_amd.rope import section_turns
    cfg = TextEncoderConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2)
    S, g = 70, _gen(2)
    x = _randn(g, S, 9 * 128)
    pos = torch.stack([torch.arange(S), torch.arange(S) // 3, torch.arange(S) % 7])
    cos, sin = mrope_tables(cfg, pos)
    a, b = x.to(DEV), x.to(DEV)
    ops.rope_half(a, 0, 6, 128, cos.to(DEV), sin.to(DEV))
    turns, axis = section_turns(cfg.mrope_section, cfg.rope_theta, DEV)
    ops.rope_axes(b, 0, 6, 128, pos.to(torch.int32).to(DEV), turns, axis)
    x3 = x[:, :768].view(S, 6, 128).float()
    mag = (x3[..., :64].abs() + x3[..., 64:].abs()).repeat(1, 1, 2).view(S, -1)
    # rope_half rounds cos / sin, two products and a sum, rope_axes the sum: at most 4 half steps of |x| + |y|
    assert ((a[:, :768].float().cpu() - b[:, :768].float().cpu()).abs() <= 4 * H8 * mag).all()
    assert torch.equal(a[:, 768:], b[:, 768:])


def _pool(N, Hk, P, Dh, layout="heads", fill=None):
    """Two page pools [N, Hk, P, Dh] of one layout."""
    shape = (N, Hk, P, Dh) if layout == "heads" else (N, P, Hk, Dh)
    ks = [torch.full(shape, float("nan") if fill is None else fill, dtype=BF16, device=DEV) for _ in range(2)]
    return ks if layout == "heads" else [t.transpose(1, 2) for t in ks]


@pytest.mark.parametrize("T,H,Hk,Dh,P,layout,name", [
    (1, 1, 1, 128, 16, "heads", "sections"), (37, 7, 1, 80, 32, "rows", "grid"), (300, 4, 2, 136, 64, "heads", "inter"),
    (2050, 3, 3, 16, 1024, "rows", "tiny"), (129, 28, 4, 128, 16, "rows", "sections")])
def test_rope_append(T, H, Hk, Dh, P, layout, name):
    """q rotated in place or elsewhere; k rotated and v unrotated in their slots; every other slot as it
    was; negative slots and slots past the pool not stored."""
    ops = _ops()
    turns, axis, axes, inter = _plan(name)
    g = _gen(T)
    x = _randn(g, T, (H + 2 * Hk) * Dh + 8)
    pos = torch.randint(0, 40000, (axes, T), generator=g, dtype=torch.int32)
    N = -(-T // P) + 3
    slots = torch.randperm(N * P, generator=g)[:T]
    if T > 10:
        slots[3], slots[5], slots[8] = -1, N * P, 1 << 40
    kp, vp = _pool(N, Hk, P, Dh, layout, 3.0)
    d = lambda t: t.to(DEV)  # noqa: E731
    xd = d(x)
    out = torch.empty(T, H * Dh, dtype=BF16, device=DEV)
    r = ops.rope_append(xd, H, Hk, Dh, d(pos), d(turns), d(axis), kp, vp, d(slots), interleaved=inter, out=out)
    assert r is out and torch.equal(xd.cpu(), x)
    x3 = x[:, :(H + 2 * Hk) * Dh].reshape(T, H + 2 * Hk, Dh)
    want, tol = rope_ref(x3[:, :H + Hk], pos, turns, axis, inter)
    _check(out.view(T, H, Dh), want[:, :H], tol[:, :H])
    keep = (slots >= 0) & (slots < N * P)
    flat = [t.transpose(1, 2).reshape(N * P, Hk, Dh).cpu() for t in (kp, vp)]
    _check(flat[0][slots[keep]], want[keep, H:], tol[keep, H:])
    assert torch.equal(flat[1][slots[keep]], x3[keep, H + Hk:])
    other = torch.ones(N * P, dtype=torch.bool)
    other[slots[keep]] = False
    assert (flat[0][other] == 3).all() and (flat[1][other] == 3).all()
    q = ops.rope_append(xd, H, Hk, Dh, d(pos), d(turns), d(axis), kp, vp, d(slots), interleaved=inter)
    assert q.data_ptr() == xd.data_ptr() and torch.equal(q, out)
    assert torch.equal(xd[:, H * Dh:].cpu(), x[:, H * Dh:])


# ---------------------------------------------------------------------------- packed attention
def _qkv(g, T, H, Hk, Dh, pad=0):
    """q, k, v as columns of one projection's rows."""
    x = _randn(g, T, (H + 2 * Hk) * Dh + pad)
    v3 = lambda a, n: x[:, a * Dh:(a + n) * Dh].view(T, n, Dh) if pad == 0 else x[:, a * Dh:(a + n) * Dh].unflatten(1, (n, Dh))  # noqa: E731
    return x, v3(0, H), v3(H, Hk), v3(H + Hk, Hk)


def _split(xd, H, Hk, Dh):
    f = lambda a, n: xd[:, a * Dh:(a + n) * Dh].unflatten(1, (n, Dh))  # noqa: E731
    return f(0, H), f(H, Hk), f(H + Hk, Hk)


PACKED = [([1], 1, 1, 64), ([0, 5, 0, 64, 65, 0], 4, 2, 64), ([63, 1, 128, 200], 28, 4, 128), ([700], 6, 2, 128),
          ([33, 100], 16, 16, 80), ([129], 28, 1, 72), ([257, 64], 3, 3, 8), ([90, 400, 31], 16, 2, 96),
          ([1] * 70 + [3], 7, 1, 40), ([1100, 2], 8, 8, 128), ([513, 1, 300], 20, 1, 128), ([100], 28, 4, 128),
          ([2600, 1500], 16, 2, 128), ([2600, 1500], 16, 2, 72), ([2600, 1500], 16, 2, 64),
          ([3000, 2500], 16, 2, 128), ([3000, 2500], 16, 2, 72), ([3600], 16, 2, 64), ([30] * 16, 16, 16, 80)]  # 256-row blocks


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,Hk,Dh", PACKED)
def test_attention_packed(lens, H, Hk, Dh, causal):
    ops = _ops()
    T = sum(lens)
    x, q, k, v = _qkv(_gen(T + H), T, H, Hk, Dh, pad=8)
    want, tol = packed_ref(q, k, v, lens, causal)
    qd, kd, vd = _split(x.to(DEV), H, Hk, Dh)
    got = ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV), causal=causal)
    _check(got, want, tol)


def test_attention_packed_long_and_large_logits():
    """A long sequence among short ones; logits far apart, so that the running maximum moves."""
    ops = _ops()
    lens, H, Hk, Dh = [3000, 17, 1], 4, 1, 128
    T, g = sum(lens), _gen(5)
    x, q, k, v = _qkv(g, T, H, Hk, Dh)
    k *= torch.linspace(0.1, 4.0, T)[:, None, None].to(BF16)
    want, tol = packed_ref(q, k, v, lens, True)
    qd, kd, vd = _split(x.to(DEV), H, Hk, Dh)
    _check(ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV)), want, tol)
    want, tol = packed_ref(q, k, v, lens, True, scale=0.01)
    _check(ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV), scale=0.01), want, tol)


@pytest.mark.parametrize("lens,H,Hk", [([70, 130], 6, 2), ([600, 900], 6, 2), ([20, 40], 6, 2), ([150, 2500], 22, 2)])
def test_attention_packed_rows_outside_and_nonfinite_neighbours(lens, H, Hk):
    """Rows behind the last sequence stay as they were; infinities and NaN of another sequence, behind
    the last one, or of a later key do not reach a query that does not see them; one that it sees does."""
    ops = _ops()
    Dh = 128
    T = sum(lens) + 40
    g = _gen(9)
    x, q, k, v = _qkv(g, T, H, Hk, Dh)
    want, tol = packed_ref(q, k, v, lens, True)
    n0, n1 = lens
    x2 = x.clone()
    q2, k2, v2 = _split(x2, H, Hk, Dh)
    x2[n0 + n1:] = float("nan")
    bad = n0 + n1 - 30  # in the second sequence: queries before it are clean
    v2[bad, :, 3] = float("nan")
    v2[bad, :, 4] = float("inf")
    v2[bad + 1, :, 5] = float("-inf")
    k2[bad + 2] = float("nan")
    k2[bad + 3] = float("inf")
    out = torch.full((T, H, Dh), 5.0, dtype=BF16, device=DEV)
    qd, kd, vd = _split(x2.to(DEV), H, Hk, Dh)
    ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV), out=out)
    got = out.cpu()
    assert (got[n0 + n1:] == 5).all()
    _check(got[:bad], want[:bad], tol[:bad])
    # at the bad key: the value itself, where the key has weight
    assert torch.isnan(got[bad, :, 3]).all() and (got[bad, :, 4] == float("inf")).all()
    keep = [d for d in range(Dh) if d not in (3, 4)]
    _check(got[bad][:, keep], want[bad][:, keep], tol[bad][:, keep])
    assert (got[bad + 1, :, 5] == float("-inf")).all() and torch.isnan(got[bad + 2:n0 + n1]).all()


def test_attention_packed_bad_offsets_stay_inside():
    """Offsets past the rows are clamped to them."""
    ops = _ops()
    H, Hk, Dh, T = 4, 2, 64, 100
    x, q, k, v = _qkv(_gen(3), T, H, Hk, Dh)
    want, tol = packed_ref(q, k, v, [40, 60], True)
    qd, kd, vd = _split(x.to(DEV), H, Hk, Dh)
    cu = torch.tensor([-5, 40, 1 << 30], dtype=torch.int32, device=DEV)
    _check(ops.attention_packed(qd, kd, vd, cu), want, tol)


# ---------------------------------------------------------------------------- paged attention
def _paged(g, new, kv, H, Hk, Dh, P, layout="heads", spare=3):
    """A cache with NaN in every unused slot and page, tables with unusable ids behind a sequence's pages."""
    need = [-(-n // P) for n in kv]
    W = max(max(need), 1) + 1
    N = sum(need) + spare
    kp, vp = _pool(N, Hk, P, Dh, layout)
    perm = torch.randperm(N, generator=g)
    table = torch.full((len(kv), W), -7, dtype=torch.int32)
    table[:, -1] = 1 << 30
    ks, vs, at = [], [], 0
    for b, n in enumerate(kv):
        k, v = _randn(g, n, Hk, Dh), _randn(g, n, Hk, Dh)
        ids = perm[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids.to(torch.int32)
        slot = (ids[:, None] * P + torch.arange(P)).reshape(-1)[:n]
        for pool, t in ((kp, k), (vp, v)):
            pool[(slot // P).to(DEV), :, (slot % P).to(DEV)] = t.to(DEV)
        ks.append(k)
        vs.append(v)
    q = _randn(g, sum(new), H, Dh)
    return q, ks, vs, kp, vp, table


def paged_ref(q, ks, vs, new, kv):
    os_, ts, at = [], [], 0
    for n, m, k, v in zip(new, kv, ks, vs):
        lim = (m - n + 1 + torch.arange(n)).clamp(0, m)
        o, t = attn_ref(q[at:at + n], k, v, lim, 1 / math.sqrt(q.shape[-1]))
        os_.append(o)
        ts.append(t)
        at += n
    return torch.cat(os_), torch.cat(ts)


PAGED = [([1], [1], 1, 1, 64, 16, "heads"), ([1, 1, 1], [5, 700, 64], 28, 4, 128, 64, "heads"),
         ([1] * 5, [0, 513, 1, 2000, 512], 7, 1, 128, 16, "rows"), ([41], [309], 28, 4, 128, 64, "rows"),
         ([3, 0, 9], [2, 50, 1300], 6, 2, 80, 32, "heads"), ([300, 17], [300, 1100], 4, 4, 128, 128, "heads"),
         ([64, 130], [64, 5000], 8, 2, 96, 16, "rows"), ([700], [1500], 14, 2, 72, 1024, "heads"),
         ([2] * 67, [40] * 66 + [3000], 20, 1, 128, 64, "heads"), ([600, 900], [5000, 2500], 28, 4, 128, 64, "heads"),
         ([300, 200], [300, 400], 28, 4, 128, 16, "rows"), ([300, 200], [300, 400], 28, 4, 64, 64, "heads"),
         ([8] * 20, [8] * 19 + [3000], 28, 4, 128, 16, "heads"), ([700, 900], [700, 3000], 16, 2, 80, 32, "rows"),
         ([30], [400], 40, 1, 128, 64, "heads"), ([2500], [2500], 16, 2, 64, 16, "heads"),
         # 256-row blocks in equal shares of the work: uneven lengths, none, fewer kept than new, one block cut often
         ([400, 5, 0, 360], [4500, 900, 40, 380], 16, 2, 128, 64, "heads"), ([400, 380], [4500, 4200], 14, 2, 72, 16, "rows"),
         ([900, 300, 1], [5000, 0, 4000], 16, 2, 64, 32, "heads"), ([1000, 40], [1000, 4300], 16, 2, 128, 64, "heads"),
         ([800], [4800], 20, 1, 128, 16, "rows"), ([10] * 70, [70] * 69 + [4200], 64, 1, 64, 16, "heads"),
         ([900, 700], [20, 5000], 24, 3, 96, 128, "heads"),
         # 256-row blocks uncut and in chunks, 64-row ones in chunks, 32-row ones, four waves
         ([2200], [2300], 28, 4, 128, 64, "heads"), ([3600], [3700], 16, 2, 80, 64, "rows"), ([4200], [4300], 16, 2, 64, 16, "heads"),
         ([700, 900], [700, 3000], 16, 2, 128, 16, "heads"), ([60] * 6, [3000] * 5 + [100], 16, 16, 64, 32, "heads"),
         ([60] * 6, [3000] * 5 + [100], 16, 16, 80, 64, "rows"), ([600] * 3, [600, 610, 900], 16, 16, 80, 64, "heads"),
         ([200], [1000], 28, 4, 64, 64, "heads"), ([1] * 70, [40] * 69 + [700], 16, 16, 64, 64, "heads"),
         ([1] * 70, [40] * 69 + [700], 16, 16, 80, 16, "rows"), ([2] * 70, [45] * 69 + [700], 16, 16, 128, 64, "heads"),
         # of one length: whole blocks
         ([500] * 2, [4300] * 2, 24, 4, 128, 64, "heads"), ([400] * 3, [4200] * 3, 16, 4, 64, 64, "rows")]


@pytest.mark.parametrize("new,kv,H,Hk,Dh,P,layout", PAGED)
def test_attention_paged(new, kv, H, Hk, Dh, P, layout):
    ops = _ops()
    g = _gen(sum(kv) + H)
    q, ks, vs, kp, vp, table = _paged(g, new, kv, H, Hk, Dh, P, layout)
    want, tol = paged_ref(q, ks, vs, new, kv)
    kvl = torch.tensor(kv, dtype=torch.int32, device=DEV)
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), kvl, cu_seqlens=_cu(new).to(DEV))
    _check(got, want, tol)
    if all(n == 1 for n in new):
        assert torch.equal(ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), kvl), got)


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [900, 2600, 30]), ([40, 5, 9], [900, 2600, 30]), ([300, 20, 700], [900, 2600, 800])])
def test_attention_paged_rows_do_not_depend_on_other_sequences(new, kv):
    """In calls of one shape a row's bits do not depend on the other sequences' lengths and values."""
    ops = _ops()
    H, Hk, Dh, P = 28, 4, 128, 64
    q, ks, vs, kp, vp, table = _paged(_gen(1), new, kv, H, Hk, Dh, P)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    qd, td, cu = q.to(DEV), table.to(DEV), _cu(new).to(DEV)
    got = ops.attention_paged(qd, kp, vp, td, i32(kv), cu_seqlens=cu)
    q2 = qd.clone()
    q2[:new[0]], q2[new[0] + new[1]:] = 3.0, -1.0
    other = ops.attention_paged(q2, kp, vp, td, i32([new[0], kv[1], new[2]]), cu_seqlens=cu)
    mid = slice(new[0], new[0] + new[1])
    assert torch.equal(other[mid], got[mid]) and not torch.equal(other[:new[0]], got[:new[0]])


@pytest.mark.parametrize("new,kv,H,Hk", [(700, 5000, 28, 4), (60, 100, 28, 4), (7, 2000, 6, 1), (9, 2600, 28, 4), (400, 450, 28, 4), (30, 3000, 40, 1),
                                         (1200, 3000, 28, 4)])
def test_attention_paged_nonfinite_later_keys(new, kv, H, Hk):
    """Infinities and NaN of a later key of the same chunk do not reach the queries before it."""
    ops = _ops()
    Dh, P = 128, 32
    q, ks, vs, kp, vp, table = _paged(_gen(kv), [new], [kv], H, Hk, Dh, P)
    want, tol = paged_ref(q, ks, vs, [new], [kv])
    bad = kv - 3  # query new - 3 and later ones see it
    page, slot = int(table[0, bad // P]), bad % P
    vp[page, :, slot, 5], vp[page, :, slot, 7] = float("nan"), float("-inf")
    nxt = kv - 2
    kp[int(table[0, nxt // P]), :, nxt % P] = float("inf")
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), torch.tensor([kv], dtype=torch.int32, device=DEV),
                              cu_seqlens=_cu([new]).to(DEV)).cpu()
    _check(got[:new - 3], want[:new - 3], tol[:new - 3])
    keep = [d for d in range(Dh) if d not in (5, 7)]
    _check(got[new - 3][:, keep], want[new - 3][:, keep], tol[new - 3][:, keep])
    assert torch.isnan(got[new - 3, :, 5]).all() and (got[new - 3, :, 7] == float("-inf")).all()
    assert not torch.isfinite(got[new - 2:]).all(-1).any()


def test_shared_rows_of_positions_and_tables():
    """expand()ed positions (one row for every axis) and tables (one for every sequence)."""
    ops = _ops()
    turns, axis, axes, _ = _plan("sections")
    d = lambda t: t.to(DEV)  # noqa: E731
    x = _randn(_gen(1), 33, 256)
    row = torch.arange(33, dtype=torch.int32).view(1, 33)
    a = ops.rope_axes(d(x), 0, 2, 128, d(row).expand(3, 33), d(turns), d(axis))
    b = ops.rope_axes(d(x), 0, 2, 128, d(row.repeat(3, 1)), d(turns), d(axis))
    assert torch.equal(a, b)
    q, ks, vs, kp, vp, table = _paged(_gen(2), [1], [100], 4, 2, 128, 16)
    q3 = _randn(_gen(3), 3, 4, 128)
    lens = [100, 57, 3]
    got = ops.attention_paged(d(q3), kp, vp, d(table).expand(3, -1), torch.tensor(lens, dtype=torch.int32, device=DEV))
    for b, n in enumerate(lens):
        want, tol = paged_ref(q3[b:b + 1], [ks[0][:n]], [vs[0][:n]], [1], [n])
        _check(got[b:b + 1], want, tol)
    with pytest.raises(ValueError):  # rows that overlap
        ops.rope_axes(d(x), 0, 2, 128, torch.zeros(40, dtype=torch.int32, device=DEV).as_strided((3, 33), (2, 1)), d(turns), d(axis))


def test_attention_paged_bad_pages_read_as_zeros():
    ops = _ops()
    new, kv, H, Hk, Dh, P = [1, 30], [200, 700], 6, 2, 128, 32
    q, ks, vs, kp, vp, table = _paged(_gen(4), new, kv, H, Hk, Dh, P)
    for b, page, bad in ((0, 2, -1), (1, 0, kp.shape[0]), (1, 9, 2 ** 31 - 1), (1, 21, -2 ** 31)):
        table[b, page] = bad
        ks[b][page * P:(page + 1) * P] = 0
        vs[b][page * P:(page + 1) * P] = 0
    want, tol = paged_ref(q, ks, vs, new, kv)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), i32(kv), cu_seqlens=_cu(new).to(DEV))
    _check(got, want, tol)
    # lengths past the table: clamped to it
    full = ops.attention_paged(q[:1].to(DEV), kp, vp, table[:1, :6].contiguous().to(DEV), i32([1 << 30]))
    want, tol = paged_ref(q[:1], [ks[0][:192]], [vs[0][:192]], [1], [192])
    _check(full, want, tol)


@pytest.mark.parametrize("new,kv,H,Hk", [([2, 1], [70, 40], 4, 2), ([50, 60], [900, 300], 28, 4), ([200, 90], [1500, 100], 28, 4),
                                         ([500, 400], [4400, 600], 28, 4), ([900, 700], [2300, 800], 28, 4)])
def test_attention_paged_bad_offsets_and_lengths_stay_inside(new, kv, H, Hk):
    """Offsets outside the rows are clamped, a negative length is an empty cache: rows that see nothing are 0."""
    ops = _ops()
    q, ks, vs, kp, vp, table = _paged(_gen(31), new, kv, H, Hk, 128, 64)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    want, tol = paged_ref(q, ks, vs, new, kv)
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), i32([kv[0], -3]), cu_seqlens=i32([-7, new[0], 2 ** 31 - 1]))
    _check(got[:new[0]], want[:new[0]], tol[:new[0]])
    assert not got[new[0]:].any()
    # descending offsets: an empty sequence, then all rows
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), i32([5, kv[1]]), cu_seqlens=i32([sum(new), 0, sum(new)]))
    only = slice(sum(new) - new[1], None)
    _check(got[only], want[only], tol[only])


def test_captured_chunk_replays():
    """Many rows over a long table in a graph: replays with other offsets, lengths and q in the same buffers."""
    ops = _ops()
    new, kv, H, Hk, Dh, P = [500, 300, 100], [4500, 3000, 100], 28, 4, 128, 64
    q, ks, vs, kp, vp, table = _paged(_gen(32), new, kv, H, Hk, Dh, P)
    qd, td = q.to(DEV), table.to(DEV)
    cu, lens = _cu(new).to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV)
    ws = torch.empty(ops.attention_paged_workspace_bytes(len(q), 3, H, Hk, Dh, table.shape[1], P), dtype=torch.uint8, device=DEV)
    out = torch.zeros_like(qd)
    run = lambda o, w: ops.attention_paged(qd, kp, vp, td, lens, cu_seqlens=cu, out=o, workspace=w)  # noqa: E731
    run(out, ws)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        run(out, ws)
    for n, k in ((new, kv), ([100, 700, 100], [4500, 3000, 70]), ([900, 0, 0], [4000, 1, 0]), ([1, 1, 1], [3, 2, 1])):
        cu.copy_(_cu(n))
        lens.copy_(torch.tensor(k, dtype=torch.int32))
        qd.neg_()
        ref = torch.zeros_like(qd)
        run(ref, None)
        out.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.isfinite(out).all()


def test_attention_paged_offsets_past_32_bits():
    """A pool of more than 2^31 elements: its last pages."""
    ops = _ops()
    N, Hk, P, Dh, H = 33000, 8, 64, 128, 8  # 2.16e9 elements, 4.3 GB each
    g = _gen(6)
    kp = torch.empty(N, Hk, P, Dh, dtype=BF16, device=DEV)
    vp = torch.empty_like(kp)
    ids = torch.tensor([N - 1, 0, N - 2])
    k, v = _randn(g, 3, Hk, P, Dh), _randn(g, 3, Hk, P, Dh)
    kp[ids.to(DEV)], vp[ids.to(DEV)] = k.to(DEV), v.to(DEV)
    x = _randn(g, 1, (H + 2 * Hk) * Dh)
    slot = (N - 2) * P + 40
    turns, axis, axes, inter = _plan("sections")
    pos = torch.full((3, 1), 168, dtype=torch.int32)
    d = lambda t: t.to(DEV)  # noqa: E731
    out = ops.rope_append(d(x), H, Hk, Dh, d(pos), d(turns), d(axis), kp, vp, torch.tensor([slot], device=DEV))
    k3 = k.transpose(1, 2).reshape(-1, Hk, Dh)[:169].clone()
    v3 = v.transpose(1, 2).reshape(-1, Hk, Dh)[:169].clone()
    k3[168] = kp[N - 2, :, 40].cpu()
    v3[168] = x.view(H + 2 * Hk, Dh)[H + Hk:]
    kw, kt = rope_ref(x.view(1, -1, Dh)[:, :H + Hk], pos, turns, axis, inter)
    _check(k3[168], kw[0, H:], kt[0, H:])
    want, tol = paged_ref(out.view(1, H, Dh).cpu(), [k3], [v3], [1], [169])
    got = ops.attention_paged(out.view(1, H, Dh), kp, vp, ids.to(torch.int32).view(1, 3).to(DEV),
                              torch.tensor([169], dtype=torch.int32, device=DEV))
    _check(got, want, tol)


# ---------------------------------------------------------------------------- together
def _chain_setup(seed=11):
    """Two prompts, then chunks of new tokens: qkv rows as a projection gives them."""
    H, Hk, Dh, P = 28, 4, 128, 16
    g = _gen(seed)
    lens, more = [90, 700], [[1, 1], [17, 3], [1, 1]]
    total = [a + sum(m[b] for m in more) for b, a in enumerate(lens)]
    rows = [_randn(g, n, (H + 2 * Hk) * Dh) for n in total]
    pos = [torch.stack([torch.arange(n), torch.arange(n) // 3, torch.arange(n) % 7]).to(torch.int32) for n in total]
    return H, Hk, Dh, P, lens, more, total, rows, pos


def test_prompt_then_chunks_over_the_cache():
    """rope_append + attention_paged step by step == the whole sequences at once (rope_axes +
    attention_packed), each vs 64 bits; the pages in any order."""
    ops = _ops()
    from qwen_image_edit_streamdiffusion_amd.rope import section_turns
    H, Hk, Dh, P, lens, more, total, rows, pos = _chain_setup()
    turns, axis = section_turns((16, 24, 24), 1e6, DEV)
    d = lambda t: t.to(DEV)  # noqa: E731
    x = torch.cat(rows)
    xd = d(x)
    ops.rope_axes(xd, 0, H + Hk, Dh, d(torch.cat(pos, 1)), turns, axis)
    whole = ops.attention_packed(*_split(xd, H, Hk, Dh), _cu(total).to(DEV))
    rot = xd.cpu()
    want, tol = packed_ref(*_split(rot, H, Hk, Dh), total, True)
    _check(whole, want, tol)
    need = [-(-n // P) for n in total]
    perm = torch.randperm(sum(need), generator=_gen(2))
    W = max(need)
    table = torch.zeros(2, W, dtype=torch.int32)
    table[0, :need[0]], table[1, :need[1]] = perm[:need[0]], perm[need[0]:]
    kp, vp = _pool(sum(need), Hk, P, Dh, "rows")
    have = [0, 0]
    for step in [lens] + more:
        at = [(have[b], have[b] + n) for b, n in enumerate(step)]
        new = d(torch.cat([rows[b][a:e] for b, (a, e) in enumerate(at)]))
        ps = torch.cat([pos[b][:, a:e] for b, (a, e) in enumerate(at)], 1)
        slots = torch.cat([table[b, torch.arange(a, e) // P].long() * P + torch.arange(a, e) % P for b, (a, e) in enumerate(at)])
        q = ops.rope_append(new, H, Hk, Dh, d(ps), turns, axis, kp, vp, d(slots))
        have = [e for _, e in at]
        got = ops.attention_paged(q.unflatten(1, (H, Dh)), kp, vp, d(table), d(torch.tensor(have, dtype=torch.int32)),
                                  cu_seqlens=_cu(step).to(DEV))
        base = [0, total[0]]
        idx = torch.cat([torch.arange(base[b] + a, base[b] + e) for b, (a, e) in enumerate(at)])
        _check(got, want[idx], tol[idx])


def test_captured_steps_replay():
    """A decode step captured into a graph: replays with other tokens, positions, slots and lengths in the
    same buffers, eager work between them; two graphs with workspaces of their own."""
    ops = _ops()
    from qwen_image_edit_streamdiffusion_amd.rope import section_turns
    H, Hk, Dh, P, B, W = 28, 4, 128, 64, 3, 24
    g = _gen(21)
    turns, axis = section_turns((16, 24, 24), 1e6, DEV)
    kp, vp = (t.to(DEV) for t in (_randn(g, B * W, Hk, P, Dh), _randn(g, B * W, Hk, P, Dh)))
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32).to(DEV)
    x = torch.zeros(B, (H + 2 * Hk) * Dh, dtype=BF16, device=DEV)
    pos = torch.zeros(3, B, dtype=torch.int32, device=DEV)
    slots = torch.zeros(B, dtype=torch.int64, device=DEV)
    lens = torch.ones(B, dtype=torch.int32, device=DEV)

    def step(out, ws):
        q = ops.rope_append(x, H, Hk, Dh, pos, turns, axis, kp, vp, slots, out=out)
        return ops.attention_paged(q.view(B, H, Dh), kp, vp, table, lens, workspace=ws)

    nb = ops.attention_paged_workspace_bytes(B, B, H, Hk, Dh, W, P)
    assert nb > 0
    graphs = []
    for _ in range(2):
        q, ws = torch.empty(B, H * Dh, dtype=BF16, device=DEV), torch.empty(nb, dtype=torch.uint8, device=DEV)
        step(q, ws)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = step(q, ws)
        graphs.append((gr, o, q, ws))  # a graph's buffers live as long as it does
    for i, n in enumerate([[1, 600, 1536], [700, 2, 40], [512, 513, 1000]]):
        x.copy_(_randn(g, *x.shape))
        cur = torch.tensor(n)
        pos.copy_((cur - 1).to(torch.int32).expand(3, B))
        lens.copy_(cur)
        at = cur - 1
        slots.copy_(table.cpu()[torch.arange(B), at // P].long() * P + at % P)
        ref = step(torch.empty(B, H * Dh, dtype=BF16, device=DEV), None).clone()
        for gr, o, *_ in graphs:
            o.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, ref)


def test_other_stream():
    ops = _ops()
    lens, H, Hk, Dh = [300, 40], 4, 2, 64
    x, q, k, v = _qkv(_gen(8), sum(lens), H, Hk, Dh)
    qd, kd, vd = _split(x.to(DEV), H, Hk, Dh)
    cu = _cu(lens).to(DEV)
    ref = ops.attention_packed(qd, kd, vd, cu)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.attention_packed(qd, kd, vd, cu)
    st.synchronize()
    assert torch.equal(got, ref)


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [3000, 5, 700]), ([40, 3, 60], [3000, 300, 60]), ([700, 5, 900], [3000, 300, 900]),
                                    ([700, 5, 900], [5000, 300, 900])])
def test_two_streams_and_in_place(new, kv):
    """Two calls at once, each with its own workspace, and a call whose out is q: bitwise the call alone."""
    ops = _ops()
    H, Hk, Dh, P = 28, 4, 128, 64
    q, ks, vs, kp, vp, table = _paged(_gen(21), new, kv, H, Hk, Dh, P)
    qd, td, cu, lens = q.to(DEV), table.to(DEV), _cu(new).to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV)
    q2 = -qd
    run = lambda x, **kw: ops.attention_paged(x, kp, vp, td, lens, cu_seqlens=cu, **kw)  # noqa: E731
    want, want2 = run(qd), run(q2)
    n = ops.attention_paged_workspace_bytes(len(q), len(kv), H, Hk, Dh, table.shape[1], P)
    ws = [torch.empty(max(n, 16), dtype=torch.uint8, device=DEV) for _ in range(2)]
    outs = [torch.empty_like(qd) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, x, o, w in zip(streams, (qd, q2), outs, ws):
            with torch.cuda.stream(s):
                run(x, out=o, workspace=w)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    assert run(q2, out=q2) is q2 and torch.equal(q2, want2)


@pytest.mark.parametrize("lens", [[40, 30], [300, 500, 9], [2600, 1500]])
def test_packed_in_place(lens):
    ops = _ops()
    x, q, k, v = _qkv(_gen(22), sum(lens), 16, 2, 128)
    xd = x.to(DEV)
    qd, kd, vd = _split(xd, 16, 2, 128)
    want = ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV))
    ops.attention_packed(qd, kd, vd, _cu(lens).to(DEV), out=qd)
    assert torch.equal(qd, want) and torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def test_empty_calls():
    ops = _ops()
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    turns, axis, _, _ = _plan("sections")
    turns, axis = turns.to(DEV), axis.to(DEV)
    i32 = torch.int32
    assert ops.rope_axes(z(0, 128), 0, 1, 128, z(3, 0, dt=i32), turns, axis).shape == (0, 128)
    kp, vp = z(2, 1, 16, 128), z(2, 1, 16, 128)
    assert ops.rope_append(z(0, 384), 1, 1, 128, z(3, 0, dt=i32), turns, axis, kp, vp, z(0, dt=torch.int64)).shape == (0, 128)
    assert ops.attention_packed(z(0, 2, 128), z(0, 1, 128), z(0, 1, 128), z(2, dt=i32)).shape == (0, 2, 128)
    got = ops.attention_paged(z(0, 2, 128), kp, vp, z(1, 2, dt=i32), z(1, dt=i32), cu_seqlens=z(2, dt=i32))
    assert got.shape == (0, 2, 128)


def test_refusals():
    ops = _ops()
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    turns, axis = z(64, dt=torch.float64), z(64, dt=i32)
    x, pos, kp, vp, sl = z(4, 512), z(3, 4, dt=i32), z(2, 1, 16, 128), z(2, 1, 16, 128), z(4, dt=i64)
    bad = [lambda: ops.rope_axes(x.float(), 0, 4, 128, pos, turns, axis),
           lambda: ops.rope_axes(x, 1, 4, 128, pos, turns, axis),                    # heads past the row
           lambda: ops.rope_axes(x, 0, 4, 64, pos, turns, axis),                     # 2 pairs > head_dim
           lambda: ops.rope_axes(x, 0, 4, 128, pos[:, :3].contiguous(), turns, axis),
           lambda: ops.rope_axes(x, 0, 4, 128, pos.long(), turns, axis),
           lambda: ops.rope_axes(x, 0, 4, 128, pos, turns.float(), axis),
           lambda: ops.rope_axes(x, 0, 4, 128, pos, turns, axis[:63]),
           lambda: ops.rope_axes(x, 0, 4, 128, pos, turns, axis, out=z(3, 512)),
           lambda: ops.rope_axes(x.cpu(), 0, 4, 128, pos, turns, axis),
           lambda: ops.rope_append(x, 2, 2, 128, pos, turns, axis, kp, vp, sl),      # qkv narrower than its heads
           lambda: ops.rope_append(x, 2, 1, 128, pos, turns, axis, z(2, 2, 16, 128), z(2, 2, 16, 128), sl),
           lambda: ops.rope_append(x, 2, 1, 128, pos, turns, axis, kp, vp, sl.int()),
           lambda: ops.rope_append(x, 2, 1, 128, pos, turns, axis, z(2, 1, 24, 128), z(2, 1, 24, 128), sl),
           lambda: ops.rope_append(x, 2, 1, 128, pos, turns, axis, kp, z(2, 1, 16, 64), sl),
           lambda: ops.rope_append(x, 2, 1, 128, pos, turns, axis, kp, vp, sl, out=z(4, 128))]
    q, k, cu = z(4, 4, 64), z(4, 2, 64), z(3, dt=i32)
    bad += [lambda: ops.attention_packed(q, z(4, 3, 64), z(4, 3, 64), cu),           # 4 heads over 3
            lambda: ops.attention_packed(q, k, z(4, 2, 32), cu), lambda: ops.attention_packed(q, z(5, 2, 64), z(5, 2, 64), cu),
            lambda: ops.attention_packed(z(4, 2, 136), z(4, 2, 136), z(4, 2, 136), cu),
            lambda: ops.attention_packed(z(4, 2, 12), z(4, 2, 12), z(4, 2, 12), cu),
            lambda: ops.attention_packed(q.float(), k, k, cu), lambda: ops.attention_packed(q, k, k, cu.long()),
            lambda: ops.attention_packed(q, k, k, cu[:1]), lambda: ops.attention_packed(q, k, k, cu, scale=0.0),
            lambda: ops.attention_packed(q, k, k, cu, scale=float("nan")),
            lambda: ops.attention_packed(q, k, k, cu, out=z(4, 4, 32)),
            lambda: ops.attention_packed(q, k, k, cu, out=z(1, 4, 64).expand(4, 4, 64)),
            lambda: ops.attention_packed(z(4, 4, 66)[..., 1:65], k, k, cu)]
    q2, t, n = z(2, 4, 128), z(2, 400, dt=i32), z(2, dt=i32)
    bad += [lambda: ops.attention_paged(z(3, 4, 128), kp, vp, t, n), lambda: ops.attention_paged(q2, kp, vp, t.long(), n),
            lambda: ops.attention_paged(q2, kp, vp, t, n[:1]), lambda: ops.attention_paged(q2, kp, vp, t, n, cu_seqlens=n),
            lambda: ops.attention_paged(z(2, 4, 64), kp, vp, t, n), lambda: ops.attention_paged(q2, kp, vp.float(), t, n),
            lambda: ops.attention_paged(q2, kp, vp, t, n, workspace=z(16)), lambda: ops.attention_paged(q2, kp, vp, t.cpu(), n)]
    for i, f in enumerate(bad):
        try:
            f()
        except ValueError:
            continue
        pytest.fail(f"call {i} was not refused")
