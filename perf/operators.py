"""Cases, plain forms and 64-bit values of the language-model operators beside the prompt encoder:

  rope     ops.rope_axes          rotary positions with several axes on the heads of token rows
  append   ops.rope_append        the same rotation of q and k, with k and v written into a paged cache
  packed   ops.attention_packed   attention over packed sequences of different lengths (causal or full), grouped heads
  paged    ops.attention_paged    attention of the newest tokens of each sequence over a paged cache

A rotation turns pair i of a head by positions[axis[i]] * turns[i] full turns.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16
DEV = "cuda"


def listed():
    return [
        # the prompt encoder's language model, one prompt of an image edit: 28 q and 4 k heads, 3-D sections
        dict(name="rope-prompt", op="rope", tokens=300, heads=32, head_dim=128, slot=128, layout="sections"),
        # the vision tower on one condition picture (28 x 28 patches): 80-wide heads in 128-wide slots, 2 axes
        dict(name="rope-vision", op="rope", tokens=784, heads=32, head_dim=80, slot=128, layout="grid"),
        # the image transformer's q and k heads at 1024^2, two rows of image and text tokens, 3 interleaved axes
        dict(name="rope-video", op="rope", tokens=16816, heads=48, head_dim=128, slot=128, layout="interleaved"),
        # one generated token for each of 16 sequences
        dict(name="append-step", op="append", tokens=16, heads=28, kv_heads=4, head_dim=128, page=64, pages=512),
        # a long chunk of new tokens, not a multiple of anything
        dict(name="append-chunk", op="append", tokens=4099, heads=28, kv_heads=4, head_dim=128, page=16, pages=4096),
        # the vision tower's window blocks of four condition pictures: ragged windows of at most 64 patches
        dict(name="packed-windows", op="packed", seqs=64, longest=64, shortest=16, heads=16, kv_heads=16, head_dim=80,
             causal=False, lens_seed=1),
        # a batch of image-edit prompts
        dict(name="packed-prompts", op="packed", seqs=6, longest=420, shortest=70, heads=28, kv_heads=4, head_dim=128,
             causal=True, lens_seed=2),
        # long documents, one of them a single token, in one pack
        dict(name="packed-long", op="packed", seqs=4, longest=8192, shortest=1, heads=28, kv_heads=4, head_dim=128,
             causal=True, lens_seed=3),
        # a new instruction over a cached template and condition picture
        dict(name="paged-edit", op="paged", seqs=1, new_longest=41, new_shortest=41, kv_longest=309, kv_shortest=309,
             heads=28, kv_heads=4, head_dim=128, page=64, lens_seed=4),
        # one generated token for each of 16 prompts
        dict(name="paged-step", op="paged", seqs=16, new_longest=1, new_shortest=1, kv_longest=600, kv_shortest=70,
             heads=28, kv_heads=4, head_dim=128, page=64, lens_seed=5),
        # the same over long caches: the step that the memory's bandwidth bounds
        dict(name="paged-step-long", op="paged", seqs=48, new_longest=1, new_shortest=1, kv_longest=32768,
             kv_shortest=900, heads=28, kv_heads=4, head_dim=128, page=64, lens_seed=6),
        # chunks of long prompts over what is cached of them, small pages
        dict(name="paged-chunk", op="paged", seqs=3, new_longest=1500, new_shortest=300, kv_longest=24000,
             kv_shortest=5000, heads=28, kv_heads=4, head_dim=128, page=16, lens_seed=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "packed", "paged", "packed", "paged"])
    heads, kv_heads, head_dim = rng.choice([(28, 4, 128), (16, 16, 80), (24, 24, 128), (8, 8, 64), (16, 2, 96),
                                            (12, 4, 64), (20, 1, 128), (14, 2, 72), (32, 8, 128)])
    c = dict(op=op, heads=heads, head_dim=head_dim)
    if op == "rope":
        c.update(tokens=_log(rng, 1, 16000), slot=128 if rng.random() < 0.5 else head_dim,
                 layout=rng.choice(["sections", "grid", "interleaved"]))
    elif op == "append":
        c.update(kv_heads=kv_heads, tokens=_log(rng, 1, 4099), page=rng.choice([16, 32, 64, 128]))
        c["pages"] = -(-c["tokens"] // c["page"]) * 2 + rng.randrange(1, 64)
    elif op == "packed":
        c.update(kv_heads=kv_heads, causal=rng.random() < 0.7, lens_seed=rng.randrange(1 << 30))
        c["longest"] = _log(rng, 1, 6000)
        most = min(64, 7e11 / (4 * heads * head_dim * c["longest"] ** 2 * (0.5 if c["causal"] else 1)))
        c["seqs"] = _log(rng, 1, max(1.0, most))
        c["shortest"] = rng.randrange(0, c["longest"] + 1)
    else:
        step = rng.random() < 0.5
        c.update(kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]), lens_seed=rng.randrange(1 << 30))
        c["new_longest"] = 1 if step else _log(rng, 2, 1400)
        c["new_shortest"] = 1 if step else rng.randrange(0, c["new_longest"] + 1)
        c["kv_longest"] = max(c["new_longest"], _log(rng, 20, 20000))
        c["kv_shortest"] = rng.randrange(c["new_longest"], c["kv_longest"] + 1)
        most = min(40, 5e11 / (4 * heads * head_dim * c["new_longest"] * c["kv_longest"]),
                   48 * 32768 * 4 * 128 / (c["kv_longest"] * kv_heads * head_dim))
        c["seqs"] = _log(rng, 1, max(1.0, most))
    return c


# ---------------------------------------------------------------------------- sizes
def _lens(case, low, high):
    """The sequences' lengths: the longest one, the shortest one, and what lies between."""
    rng = random.Random(case["lens_seed"] * 1000003 + high)
    n = [rng.randint(low, high) for _ in range(case["seqs"])]
    n[rng.randrange(len(n))] = high
    if len(n) > 1:
        n[(n.index(high) + 1) % len(n)] = low
    return n


def _sizes(case):
    """(new tokens, cached tokens with the new ones) of every sequence of a paged case."""
    new = _lens(case, case["new_shortest"], case["new_longest"])
    kv = _lens(case, case["kv_shortest"], case["kv_longest"])
    return new, [max(a, b) for a, b in zip(new, kv)]


def _pairs(new, kv, causal):
    """(query, key) pairs that are looked at, over all sequences."""
    return sum(n * k - (n * (n - 1) // 2 if causal else 0) for n, k in zip(new, kv))


def work(case):
    H, Dh = case["heads"], case["head_dim"]
    if case["op"] == "rope":
        n = case["tokens"] * H * Dh
        return {"bytes": 4 * n + 12 * case["tokens"] + 6 * Dh, "flops": 3 * n + 10 * case["tokens"] * Dh}
    Hk = case["kv_heads"]
    if case["op"] == "append":
        n = case["tokens"] * (H + 2 * Hk) * Dh
        return {"bytes": 4 * n + 20 * case["tokens"] + 6 * Dh,
                "flops": 3 * case["tokens"] * (H + Hk) * Dh + 10 * case["tokens"] * Dh}
    if case["op"] == "packed":
        n = _lens(case, case["shortest"], case["longest"])
        return {"bytes": 4 * sum(n) * (H + Hk) * Dh + 4 * (len(n) + 1),
                "flops": 4 * H * Dh * _pairs(n, n, case["causal"])}
    new, kv = _sizes(case)
    return {"bytes": 4 * sum(new) * H * Dh + 4 * sum(kv) * Hk * Dh + 4 * sum(-(-k // case["page"]) for k in kv) +
            8 * len(kv), "flops": 4 * H * Dh * _pairs(new, kv, True)}


# ---------------------------------------------------------------------------- inputs
def _plan(case):
    """turns [R/2] (64-bit: full turns of a pair for each step of its axis), axis [R/2], interleaved."""
    half = case["head_dim"] // 2
    layout = case.get("layout", "sections")
    if layout == "sections":  # one ladder of frequencies, cut into runs that go by time, height and width
        i = torch.arange(half, dtype=torch.float64)
        turns = 1e6 ** (-i / half) / (2 * math.pi)
        a, b = half // 4, half // 4 + 3 * half // 8
        axis = (torch.arange(half) >= a).int() + (torch.arange(half) >= b).int()
        return turns.to(DEV), axis.to(DEV), False
    # a ladder for each axis: height and width, or time, height and width
    runs = [half - half // 2, half // 2] if layout == "grid" else [half - 2 * (7 * half // 16)] + 2 * [7 * half // 16]
    turns = torch.cat([1e4 ** (-torch.arange(n, dtype=torch.float64) / n) / (2 * math.pi) for n in runs])
    axis = torch.cat([torch.full((n,), k, dtype=torch.int32) for k, n in enumerate(runs)])
    return turns.to(DEV), axis.to(DEV), layout == "interleaved"


def _positions(case, axes, T, g):
    """A prompt's positions: text, a picture's grid, and text far into a long conversation."""
    t = torch.arange(T, device=DEV)
    side = max(1, int(math.sqrt(T / 2)))
    far = int(torch.randint(0, 100000, (1,), generator=g, device=DEV))
    pos = torch.stack([t // (side * side), t % (side * side) // side, t % side])
    pos[1:] -= side // 2  # a picture's grid is centred
    if case.get("layout", "sections") == "sections":
        pos = pos + far
        pos[:, T // 2:] = far + t[T // 2:]
    return pos[3 - axes:].to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32).to(BF16)  # noqa: E731
    H, Dh = case["heads"], case["head_dim"]
    s = {"case": case}
    if case["op"] == "rope":
        T, slot = case["tokens"], case["slot"]
        s["x"] = randn(T, H * slot + 64)  # rows of a packed projection: other columns follow the heads
        s["turns"], s["axis"], s["interleaved"] = _plan(case)
        s["pos"] = _positions(case, 2 if case["layout"] == "grid" else 3, T, g)
        s["out"] = torch.zeros(T, H * slot, device=DEV, dtype=BF16)
        return s
    Hk = case["kv_heads"]
    if case["op"] == "append":
        T, P, N = case["tokens"], case["page"], case["pages"]
        s["qkv"] = randn(T, (H + 2 * Hk) * Dh)
        s["turns"], s["axis"], s["interleaved"] = _plan(case)
        s["pos"] = _positions(case, 3, T, g)
        s["k"], s["v"] = randn(N, Hk, P, Dh), randn(N, Hk, P, Dh)
        # runs of neighbouring slots inside pages that lie anywhere in the pool
        page = torch.randperm(N, generator=g, device=DEV)[:-(-T // P)]
        s["slots"] = (page[:, None] * P + torch.arange(P, device=DEV)).reshape(-1)[:T].contiguous()
        s["out"] = torch.empty(T, H * Dh, device=DEV, dtype=BF16)
        return s
    if case["op"] == "packed":
        n = _lens(case, case["shortest"], case["longest"])
        T = sum(n)
        qkv = randn(T, H + 2 * Hk, Dh)  # q, k and v are columns of one projection
        qkv[:, H:H + Hk] *= 1.5
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        s["longest"] = max(n)
    else:
        n, kv = _sizes(case)
        T, P = sum(n), case["page"]
        need = [-(-x // P) for x in kv]
        N = sum(need) + 7
        s["k"], s["v"] = randn(N, Hk, P, Dh).mul_(1.5), randn(N, Hk, P, Dh)
        pages = torch.randperm(N, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(len(n), max(need), dtype=torch.int32, device=DEV)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = pages[at:at + m]
            at += m
        s["table"], s["kv_lens"] = table, torch.tensor(kv, dtype=torch.int32, device=DEV)
        s["q"] = randn(T, H, Dh)
        s["longest"] = max(n)
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------- plain forms
def _rotate(x, s):
    """x [T, heads, Dh] in 32 bits; the angles of far positions in 64."""
    turn = s["pos"][s["axis"].long()].double().T * s["turns"]  # [T, R/2]
    turn = (turn - turn.round()) * (2 * math.pi)
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]
    x = x.float()
    if s["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _attend(q, k, v, off, n_k, causal):
    """q [B, Hk, G, L, Dh], k and v [B, Hk, K, Dh] in 32 bits; row i of sequence b sees keys < n_k[b], and where
    `causal` keys <= off[b] + i."""
    B, Hk, G, L, Dh = q.shape
    K = k.shape[2]
    s = torch.matmul(q.reshape(B, Hk, G * L, Dh), k.transpose(2, 3).contiguous()).view(B, Hk, G, L, K)
    s.mul_(1.0 / math.sqrt(Dh))
    j, i = torch.arange(K, device=DEV), torch.arange(L, device=DEV)
    seen = (j < n_k[:, None, None]).expand(B, L, K)
    if causal:
        seen = seen & (j <= off[:, None, None] + i[:, None])
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == float("-inf"), torch.zeros_like(m), m)).exp_()
    d = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, Hk, G * L, K), v).view(B, Hk, G, L, Dh)
    return o / torch.where(d == 0, torch.ones_like(d), d)


def _rows(cu, L, T):
    """(row of every sequence's i-th token, whether there is one), both [B, L]."""
    i = torch.arange(L, device=DEV)
    return (cu[:-1, None] + i).clamp_(max=T - 1), i < (cu[1:] - cu[:-1])[:, None]


def _plain_attention(s, k, v, n_k, causal):
    q, cu, L = s["q"], s["cu"].long(), s["longest"]
    T, H, Dh = q.shape
    Hk = k.shape[1]
    rows, there = _rows(cu, L, T)
    qp = q[rows].float().view(-1, L, Hk, H // Hk, Dh).permute(0, 2, 3, 1, 4)
    n_q = cu[1:] - cu[:-1]
    o = _attend(qp, k, v, n_k - n_q, n_k, causal)
    return o.permute(0, 3, 1, 2, 4).reshape(-1, L, H, Dh)[there].to(BF16)


def _plain(s):
    c = s["case"]
    H, Dh = c["heads"], c["head_dim"]
    if c["op"] == "rope":
        x = s["x"][:, :H * c["slot"]].view(-1, H, c["slot"])[..., :Dh]
        return _rotate(x, s).to(BF16)
    if c["op"] == "append":
        Hk, P = c["kv_heads"], c["page"]
        x = s["qkv"].view(-1, H + 2 * Hk, Dh)
        r = _rotate(x[:, :H + Hk], s).to(BF16)
        page, at = s["slots"] // P, s["slots"] % P
        s["k"][page, :, at] = r[:, H:]
        s["v"][page, :, at] = x[:, H + Hk:]
        return {"q": r[:, :H], "k": s["k"], "v": s["v"]}
    if c["op"] == "packed":
        T, L = s["q"].shape[0], s["longest"]
        rows, _ = _rows(s["cu"].long(), L, T)
        k, v = (s[x][rows].float().transpose(1, 2).contiguous() for x in ("k", "v"))
        n = (s["cu"][1:] - s["cu"][:-1]).long()
        return _plain_attention(s, k, v, n, c["causal"])
    t = s["table"].long()
    k, v = (s[x][t].float().transpose(1, 2).reshape(t.shape[0], c["kv_heads"], -1, Dh) for x in ("k", "v"))
    return _plain_attention(s, k, v, s["kv_lens"].long(), True)


# ---------------------------------------------------------------------------- the framework's calls
def _own(s):
    from qwen_image_edit_streamdiffusion_amd import ops
    c = s["case"]
    H, Dh = c["heads"], c["head_dim"]
    if c["op"] == "rope":
        out = ops.rope_axes(s["x"], 0, H, Dh, s["pos"], s["turns"], s["axis"], interleaved=s["interleaved"],
                            head_stride=c["slot"], out=s["out"])
        return out.view(-1, H, c["slot"])[..., :Dh]
    if c["op"] == "append":
        q = ops.rope_append(s["qkv"], H, c["kv_heads"], Dh, s["pos"], s["turns"], s["axis"], s["k"], s["v"],
                            s["slots"], interleaved=s["interleaved"], out=s["out"])
        return {"q": q.view(-1, H, Dh), "k": s["k"], "v": s["v"]}
    if c["op"] == "packed":
        return ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"])
    return ops.attention_paged(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], cu_seqlens=s["cu"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------- 64 bits
def _exact_rope(x, pos, turns, axis, interleaved):
    """Each pair as a complex number times exp(i angle)."""
    ang = 2 * math.pi * torch.remainder(pos.double()[axis.long()] * turns[:, None], 1.0).T[:, None]
    x = x.double()
    n = x.shape[-1] // 2
    z = torch.view_as_complex(x.unflatten(-1, (n, 2)).contiguous()) if interleaved else torch.complex(x[..., :n], x[..., n:])
    z = z * torch.polar(torch.ones_like(ang), ang)
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)


def _exact_rows(q, k, v, causal):
    """One sequence: q [n, H, Dh] are the last n of the K tokens that k and v [K, Hk, Dh] hold."""
    n, H, Dh = q.shape
    K, Hk = k.shape[:2]
    out = torch.empty(n, H, Dh, dtype=torch.float64, device=q.device)
    for h in range(H):
        kk, vv = (x[:, h * Hk // H].double() for x in (k, v))
        for a in range(0, n, 2048):
            s = q[a:a + 2048, h].double() @ kk.T / math.sqrt(Dh)
            if causal:
                s += torch.full_like(s, float("-inf")).triu(K - n + a + 1)
            out[a:a + 2048, h] = torch.softmax(s, -1) @ vv
    return out


def exact(case, seed):
    s = prepare(case, seed)
    H, Dh = case["heads"], case["head_dim"]
    if case["op"] == "rope":
        x = s["x"][:, :H * case["slot"]].unflatten(-1, (H, case["slot"]))[:, :, :Dh]
        return _exact_rope(x, s["pos"], s["turns"], s["axis"], s["interleaved"])
    Hk = case["kv_heads"]
    if case["op"] == "append":
        x = s["qkv"].unflatten(-1, (H + 2 * Hk, Dh))
        r = _exact_rope(x[:, :H + Hk], s["pos"], s["turns"], s["axis"], s["interleaved"])
        k, v = (s[n].double().transpose(1, 2).flatten(0, 1) for n in ("k", "v"))  # [slots, Hk, Dh]
        k[s["slots"]], v[s["slots"]] = r[:, H:], x[:, H + Hk:].double()
        return {"q": r[:, :H], "k": k.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous(),
                "v": v.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous()}
    cu = s["cu"].tolist()
    out = []
    for b, (a, e) in enumerate(zip(cu[:-1], cu[1:])):
        if case["op"] == "packed":
            k, v, causal = s["k"][a:e], s["v"][a:e], case["causal"]
        else:
            n = int(s["kv_lens"][b])
            ids = s["table"][b].long()[:-(-n // case["page"])]
            k, v = (s[x][ids].transpose(1, 2).flatten(0, 1)[:n] for x in ("k", "v"))
            causal = True
        if e > a:
            out.append(_exact_rows(s["q"][a:e], k, v, causal))
    return torch.cat(out) if out else torch.empty(0, H, Dh, dtype=torch.float64, device=DEV)
