"""Attention over sequences where a kernel's own code for rare values runs: infinities and NaN that some rows of a
block see and others do not, and scores far from 0. Every kernel and head width, each vs 64 bits with the
tolerances of test_gpu_sequences.py."""
import math

import pytest
import torch

from test_gpu_sequences import BF16, DEV, _check, _cu, _gen, _ops, _paged, _qkv, _split, packed_ref, paged_ref

pytestmark = pytest.mark.gpu

# (lens, heads, kv_heads): 16-row blocks with eight and four waves, 64-row ones with few and many work-groups, 256-row ones
PACKED = {"16 rows, 8 waves": ([100], 28, 4), "16 rows, 4 waves": ([200], 28, 4), "64 rows": ([300], 28, 4),
          "64 rows, many": ([300] * 10, 28, 4), "256 rows": ([3600], 16, 2)}
# (new, kv, heads, kv_heads)
PAGED = {"16 rows, 8 waves, cut": ([7], [2000], 6, 1), "16 rows, 4 waves": ([2] * 70, [45] * 69 + [700], 16, 16),
         "32 rows": ([200], [1000], 28, 4), "64 rows": ([300, 200], [300, 400], 28, 4),
         "64 rows, many": ([300] * 6 + [280], [300] * 6 + [400], 28, 4), "64 rows, cut": ([60] * 6, [3000] * 5 + [100], 16, 16),
         "256 rows": ([4200], [4300], 16, 2), "256 rows, shares": ([700], [5000], 28, 4)}


@pytest.mark.parametrize("Dh", [64, 80, 128])
@pytest.mark.parametrize("name", list(PACKED))
def test_packed_nonfinite_values_reach_the_rows_that_see_them(name, Dh):
    ops = _ops()
    lens, H, Hk = PACKED[name]
    T = sum(lens)
    x, q, k, v = _qkv(_gen(T + Dh), T, H, Hk, Dh)
    want, tol = packed_ref(q, k, v, lens, True)
    _, _, v2 = _split(x, H, Hk, Dh)
    at, clean, see = 0, [], []
    for n in lens:  # in the middle of a tile, at its end, and in a sequence's last tile
        for bad in (n // 2, n // 2 + 37, n - 5):
            v2[at + bad, :, 3], v2[at + bad, :, 4], v2[at + bad, :, Dh - 1] = float("nan"), float("inf"), float("-inf")
        clean.append(torch.arange(at, at + n // 2))
        see.append(torch.arange(at + n // 2, at + n))
        at += n
    clean, see = torch.cat(clean), torch.cat(see)
    got = ops.attention_packed(*_split(x.to(DEV), H, Hk, Dh), _cu(lens).to(DEV)).cpu()
    _check(got[clean], want[clean], tol[clean])
    rest = [d for d in range(Dh) if d not in (3, 4, Dh - 1)]
    _check(got[see][:, :, rest], want[see][:, :, rest], tol[see][:, :, rest])
    assert torch.isnan(got[see, :, 3]).all()
    assert (got[see, :, 4] == float("inf")).all() and (got[see, :, Dh - 1] == float("-inf")).all()


@pytest.mark.parametrize("Dh", [64, 80, 128])
@pytest.mark.parametrize("name", list(PAGED))
def test_paged_nonfinite_values_reach_the_rows_that_see_them(name, Dh):
    ops = _ops()
    new, kv, H, Hk = PAGED[name]
    P = 32
    q, ks, vs, kp, vp, table = _paged(_gen(sum(kv) + Dh), new, kv, H, Hk, Dh, P)
    want, tol = paged_ref(q, ks, vs, new, kv)
    at, clean, see = 0, [], []
    for b, (n, m) in enumerate(zip(new, kv)):
        seen = n // 2  # the query that first sees the key
        bad = m - n + seen
        page, slot = int(table[b, bad // P]), bad % P
        vp[page, :, slot, 3], vp[page, :, slot, 4], vp[page, :, slot, Dh - 1] = float("nan"), float("inf"), float("-inf")
        clean.append(torch.arange(at, at + seen))
        see.append(torch.arange(at + seen, at + n))
        at += n
    clean, see = torch.cat(clean), torch.cat(see)
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV),
                              cu_seqlens=_cu(new).to(DEV)).cpu()
    _check(got[clean], want[clean], tol[clean])
    rest = [d for d in range(Dh) if d not in (3, 4, Dh - 1)]
    _check(got[see][:, :, rest], want[see][:, :, rest], tol[see][:, :, rest])
    assert torch.isnan(got[see, :, 3]).all()
    assert (got[see, :, 4] == float("inf")).all() and (got[see, :, Dh - 1] == float("-inf")).all()


# ---------------------------------------------------------------------------- scores far from 0
def _far(g, q, k, sign):
    """q and k of one element a row that is not 0, so that every score is one product, exact in 32 bits: sign * 2^103 ..
    2^105 (1e31 .. 4e31), eight values a row, so that several keys share the largest. The others are 2^100 away at least."""
    for t, lead in ((q, sign * 2.0 ** 53), (k, 2.0 ** 50)):
        t.zero_()
        t[..., 1] = lead * (1 + torch.randint(0, 8, t.shape[:-1], generator=g) / 8).to(BF16)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("name", list(PACKED))
def test_packed_scores_far_from_zero(name, sign):
    """A row's weights go by its scores' distances, wherever the scores lie: all of them below -1e30, or above 1e30."""
    ops = _ops()
    lens, H, Hk = PACKED[name]
    g = _gen(sum(lens))
    x, q, k, v = _qkv(g, sum(lens), H, Hk, 128)
    _far(g, q, k, sign)
    want, tol = packed_ref(q, k, v, lens, True)
    _check(ops.attention_packed(*_split(x.to(DEV), H, Hk, 128), _cu(lens).to(DEV)), want, tol)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("name", list(PAGED))
def test_paged_scores_far_from_zero(name, sign):
    ops = _ops()
    new, kv, H, Hk = PAGED[name]
    P, g = 32, _gen(sum(kv))
    q, ks, vs, kp, vp, table = _paged(g, new, kv, H, Hk, 128, P)
    for b, k in enumerate(ks):
        _far(g, q, k, sign)
        slots = torch.arange(len(k))
        kp[table[b, slots // P].long().to(DEV), :, (slots % P).to(DEV)] = k.to(DEV)
    want, tol = paged_ref(q, ks, vs, new, kv)
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV),
                              cu_seqlens=_cu(new).to(DEV))
    _check(got, want, tol)


def test_one_key_gives_its_value_at_any_score_and_scale():
    """Single visible keys: o = v exactly, whatever the score that 32 bits hold."""
    ops = _ops()
    Dh, g = 64, _gen(1)
    v = torch.randn(5, 1, Dh, generator=g).to(BF16)
    for lead, scale in ((2.0 ** 53, None), (2.0 ** 62, None), (1.0, None), (2.0 ** 62, 1e-30), (2.0 ** 53, 65536.0), (1.0, 1e-37)):
        q, k = torch.zeros(5, 1, Dh), torch.zeros(5, 1, Dh)
        q[:, 0, 0] = torch.tensor([-1.0, 1.0, -1.25, 1.75, 0.0]) * lead
        k[:, 0, 0] = 1.5 * lead
        cu = torch.arange(6, dtype=torch.int32)
        d = lambda t: t.to(BF16).to(DEV)  # noqa: E731
        assert torch.equal(ops.attention_packed(d(q), d(k), d(v), cu.to(DEV), scale=scale).cpu(), v), (lead, scale)
        kp, vp = torch.zeros(5, 1, 16, Dh), torch.zeros(5, 1, 16, Dh)
        kp[:, 0, 0], vp[:, 0, 0] = k[:, 0], v[:, 0].float()
        got = ops.attention_paged(d(q), d(kp), d(vp), cu[:5].view(5, 1).to(DEV), torch.ones(5, dtype=torch.int32, device=DEV), scale=scale)
        assert torch.equal(got.cpu(), v), (lead, scale)


def test_scores_past_32_bits():
    """A product past 32 bits is an infinity: of a key that a row sees it has no weight if negative, and a row whose
    visible scores are all -inf is 0, as one that sees none."""
    ops = _ops()
    Dh, g = 64, _gen(2)
    v = torch.randn(4, 1, Dh, generator=g).to(BF16)
    q, k = torch.zeros(4, 1, Dh), torch.zeros(4, 1, Dh)
    q[:, 0, 0] = 2.0 ** 100
    k[:, 0, 0] = torch.tensor([-1.0, -1.0, 2.0 ** -101, -1.0]) * 2.0 ** 100
    d = lambda t: t.to(BF16).to(DEV)  # noqa: E731
    got = ops.attention_packed(d(q), d(k), d(v), torch.tensor([0, 4], dtype=torch.int32, device=DEV)).cpu()
    assert not got[:2].any() and torch.equal(got[2], v[2]) and torch.equal(got[3], v[2])
    assert math.isinf(float(q[0, 0, 0] * k[0, 0, 0]))


def test_one_sequence_that_fills_the_chip_over_a_long_cache():
    """As many 256-row blocks as the chip has places, in equal shares."""
    ops = _ops()
    new, kv, H, Dh, P = [1900], [4200], 32, 64, 64
    q, ks, vs, kp, vp, table = _paged(_gen(5), new, kv, H, H, Dh, P)
    want, tol = paged_ref(q, ks, vs, new, kv)
    got = ops.attention_paged(q.to(DEV), kp, vp, table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV),
                              cu_seqlens=_cu(new).to(DEV))
    _check(got, want, tol)
