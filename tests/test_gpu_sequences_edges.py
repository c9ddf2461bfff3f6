"""Attention over sequences where a kernel's own code for rare values runs: infinities and NaN that some rows of a
block see and others do not. Every kernel and head width, each vs 64 bits with the tolerances of
test_gpu_sequences.py."""
import pytest
import torch

from test_gpu_sequences import DEV, _check, _cu, _gen, _ops, _paged, _qkv, _split, packed_ref, paged_ref

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

