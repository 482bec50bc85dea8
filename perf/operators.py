"""Measured cases of the long-video attention operators: rotary positions
(applied to Q and K, or written as the 2x2 matrices that the fused Q/K prologue
reads), the choice of key blocks for each query block from INT8 Q/K, and the
INT8 attention over the chosen blocks.

`run` computes a case in its plain form from elementary torch operations, or,
where `own` is true, with the package's operators.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
QB, KB, D = 128, 64, 128        # query block, key block, channels of a head
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    pkg = str(Path(__file__).resolve().parents[1] / "comfyui-turing-utils_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import comfyui_turing_utils_kernel as kernel

    return kernel


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # One new token of a streamed sequence far from its start: a latency.
        {"name": "rope_token", "op": "rope", "B": 1, "Hq": 32, "Hk": 8, "L": 1, "D": 128,
         "rot": 128, "layout": "NHD", "split_half": True, "axes": 1, "dtype": "bf16",
         "start": 131000, "grad": False},
        # A padded text batch trained through half of each head: forward and gradients.
        {"name": "rope_text_grad", "op": "rope", "B": 3, "Hq": 20, "Hk": 4, "L": 1111, "D": 96,
         "rot": 48, "layout": "HND", "split_half": True, "axes": 1, "dtype": "f32",
         "start": 0, "grad": True},
        # 480p, 81 frames: all heads of a video token grid, gradients of an adapter's training.
        {"name": "rope_480p_grad", "op": "rope", "B": 1, "Hq": 40, "Hk": 40, "L": 32760, "D": 128,
         "rot": 128, "layout": "NHD", "split_half": False, "axes": 3, "dtype": "bf16",
         "start": 0, "grad": True},
        # 720p, 81 frames.
        {"name": "rope_720p", "op": "rope", "B": 1, "Hq": 40, "Hk": 40, "L": 75600, "D": 128,
         "rot": 128, "layout": "NHD", "split_half": False, "axes": 3, "dtype": "bf16",
         "start": 0, "grad": False},
        # The rotation matrices of 512 text tokens.
        {"name": "freqs_text", "op": "freqs", "B": 1, "L": 512, "rot": 64, "axes": 1,
         "dtype": "f32", "start": 0},
        # The rotation matrices of a 720p grid, once for every step and layer.
        {"name": "freqs_720p", "op": "freqs", "B": 1, "L": 75600, "rot": 128, "axes": 3,
         "dtype": "bf16", "start": 0},
        # One query token over a long context with shared key heads.
        {"name": "select_token", "op": "select", "B": 1, "Hq": 32, "Hk": 8, "Lq": 1,
         "Lk": 131071, "keep": 64, "layout": "HND", "lengths": False, "policy": False},
        # A padded batch with text blocks that are always kept and blocks never seen.
        {"name": "select_batch", "op": "select", "B": 3, "Hq": 12, "Hk": 12, "Lq": 4111,
         "Lk": 4623, "keep": 19, "layout": "NHD", "lengths": True, "policy": True},
        # 720p self-attention, a ninth of the key blocks.
        {"name": "select_720p", "op": "select", "B": 1, "Hq": 40, "Hk": 40, "Lq": 75600,
         "Lk": 75600, "keep": 128, "layout": "NHD", "lengths": False, "policy": False},
        # One query token over 64 of its blocks: a latency, split over the keys.
        {"name": "attend_token", "op": "attend", "B": 1, "Hq": 32, "Hk": 8, "Lq": 1,
         "Lk": 131071, "keep": 64, "layout": "HND", "lengths": False, "dtype": "f16",
         "lse": True},
        # A padded batch with shared key heads and ragged lengths.
        {"name": "attend_batch", "op": "attend", "B": 3, "Hq": 20, "Hk": 5, "Lq": 4111,
         "Lk": 4623, "keep": 19, "layout": "HND", "lengths": True, "dtype": "f16",
         "lse": False},
        # 720p self-attention over a ninth of the key blocks.
        {"name": "attend_720p", "op": "attend", "B": 1, "Hq": 40, "Hk": 40, "Lq": 75600,
         "Lk": 75600, "keep": 128, "layout": "NHD", "lengths": False, "dtype": "bf16",
         "lse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "freqs", "select", "select", "attend", "attend"])
    layout = rng.choice(["HND", "NHD"])
    if op in ("rope", "freqs"):
        axes = rng.choice([1, 1, 3])
        head = rng.choice([64, 96, 128])
        rot = rng.choice([r for r in (16, 32, 48, 64, 96, 128) if r <= head])
        L = _log(rng, 1, 75600)
        c = {"op": op, "B": rng.choice([1, 1, 2, 3]) if L < 20000 else 1, "L": L, "rot": rot,
             "axes": axes, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
             "start": rng.choice([0, 0, _log(rng, 1, 1000000)])}
        if op == "rope":
            group = rng.choice([1, 1, 2, 4])
            hk = rng.choice([1, 2, 5, 8, 10])
            c.update(Hq=hk * group, Hk=hk, D=head, layout=layout,
                     split_half=rng.random() < 0.5, grad=rng.random() < 0.4 and L < 33000)
        return c
    group = rng.choice([1, 1, 2, 4])
    hk = rng.choice([1, 2, 5, 8, 10])
    lq = rng.choice([1, _log(rng, 2, 40000), _log(rng, 2, 40000)])
    lk = _log(rng, max(64, min(lq, 4096)), 131072 if lq == 1 else 40000)
    nkb = -(-lk // KB)
    c = {"op": op, "B": rng.choice([1, 1, 2, 3]) if max(lq, lk) < 10000 else 1, "Hq": hk * group,
         "Hk": hk, "Lq": lq, "Lk": lk, "keep": _log(rng, 1, min(nkb, 160)), "layout": layout,
         "lengths": rng.random() < 0.4}
    if op == "select":
        c["policy"] = rng.random() < 0.4
    else:
        c.update(dtype=rng.choice(["bf16", "f16"]), lse=rng.random() < 0.4)
    return c


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _axis_pairs(case):
    """Channel pairs of each axis: time takes what height and width leave over."""
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return None
    side = pairs // 3
    return [pairs - 2 * side, side, side]


def _positions(case, g):
    """Token positions: an index from `start` on, or (frame, row, column) of a
    latent grid; each batch row is shifted by its own amount."""
    B, L = case["B"], case["L"]
    shift = torch.randint(0, 64, (B, 1), generator=g, device=DEV) + case["start"]
    t = torch.arange(L, device=DEV)[None] + shift
    if case["axes"] == 1:
        return t
    width = 52 if L < 40000 else 80
    height = 30 if L < 40000 else 45
    return torch.stack([t // (width * height), (t // width) % height, t % width], dim=-1)


def _inv_freq(case):
    """theta^(-i / pairs) over the pairs of each axis, long contexts slowed by 4."""
    parts = _axis_pairs(case) or [case["rot"] // 2]
    theta = 10000.0 * 4.0
    return torch.cat([theta ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                      for n in parts]).to(DEV)


def _tensor(shape, layout, g):
    """Normal values [B, H, L, D] or [B, L, H, D]."""
    B, H, L, d = shape
    s = (B, H, L, d) if layout == "HND" else (B, L, H, d)
    return torch.randn(s, generator=g, device=DEV)


def _codes(shape, layout, tile, g):
    """INT8 codes and scales of tokens that drift slowly along the sequence, so
    that near tokens are alike and blocks differ: one scale for each `tile`
    tokens, scales [B, H, ceil(L / 64) * 64 / tile]."""
    B, H, L, d = shape
    nt = -(-L // 64) * 64 // tile
    codes = torch.empty((B, H, L, d) if layout == "HND" else (B, L, H, d), dtype=torch.int8,
                        device=DEV)
    scales = torch.zeros((B, H, nt), device=DEV)
    for b in range(B):
        for h in range(H):
            x = torch.zeros((nt * tile, d), device=DEV)
            x[:L] = torch.randn((L, d), generator=g, device=DEV)
            drift = torch.randn((-(-L // 48), d), generator=g, device=DEV) * 0.6
            x[:L] += drift.repeat_interleave(48, dim=0)[:L]
            x = x.view(nt, tile, d)
            s = x.abs().amax(dim=(1, 2)).clamp_min(1e-7) / 127
            c = (x / s[:, None, None]).round().to(torch.int8).view(nt * tile, d)[:L]
            (codes[b, h] if layout == "HND" else codes[b, :, h]).copy_(c)
            scales[b, h] = s
    return codes, scales


def _random_lists(B, H, nqb, nkb, keep, g):
    """`keep` different blocks for each query block, ascending; the last entry of
    every seventh list is left open (-1)."""
    keep = min(keep, nkb)
    out = torch.empty((B, H, nqb, keep), dtype=torch.int32, device=DEV)
    for b in range(B):
        for h in range(H):
            r = torch.rand((nqb, nkb), generator=g, device=DEV)
            out[b, h] = r.argsort(dim=1)[:, :keep].sort(dim=1).values
    if keep > 1:
        out.view(-1, keep)[::7, -1] = -1
    return out


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] in ("rope", "freqs"):
        st["positions"] = _positions(case, g)
        st["inv_freq"] = _inv_freq(case)
        st["axis_pairs"] = _axis_pairs(case)
        st["scale"] = 1.0 if case["axes"] == 3 else 0.1 * math.log(4.0) + 1.0
        if case["op"] == "rope":
            dt = DTYPES[case["dtype"]]
            for n, h in (("q", case["Hq"]), ("k", case["Hk"])):
                shape = (case["B"], h, case["L"], case["D"])
                st[n] = _tensor(shape, case["layout"], g).to(dt).requires_grad_(case["grad"])
                if case["grad"]:
                    st["d" + n] = _tensor(shape, case["layout"], g).to(dt)
        return st
    B, Hq, Hk, Lq, Lk = (case[n] for n in ("B", "Hq", "Hk", "Lq", "Lk"))
    nqb, nkb = -(-Lq // QB), -(-Lk // KB)
    st["q8"], st["qs"] = _codes((B, Hq, Lq, D), case["layout"], 16, g)
    st["k8"], st["ks"] = _codes((B, Hk, Lk, D), case["layout"], 64, g)
    st["lengths"] = None
    if case["lengths"]:
        st["lengths"] = torch.randint(max(1, Lk // 3), Lk + 1, (B,), generator=g, device=DEV,
                                      dtype=torch.int32)
    if case["op"] == "select":
        st["policy"] = None
        if case["policy"]:
            # The last two blocks are text (always kept); some pairs are never seen.
            p = torch.zeros((nqb, nkb), dtype=torch.int8, device=DEV)
            p[torch.rand((nqb, nkb), generator=g, device=DEV) < 0.2] = -1
            p[:, max(0, nkb - 2):] = 1
            st["policy"] = p
        return st
    st["v"] = _tensor((B, Hk, Lk, D), case["layout"], g).to(DTYPES[case["dtype"]])
    st["lists"] = _random_lists(B, Hq, nqb, nkb, case["keep"], g)
    return st


# -------------------------------------------------------------- plain forms --

def _angles(positions, inv_freq, axis_pairs):
    """[B, L, pairs] in 64 bits: far positions lose their phase in 32."""
    p = positions.double()
    if axis_pairs is None:
        return p[..., None] * inv_freq.double()
    idx = torch.repeat_interleave(torch.arange(len(axis_pairs), device=p.device),
                                  torch.tensor(axis_pairs, device=p.device),
                                  output_size=sum(axis_pairs))
    return p[..., idx] * inv_freq.double()


def _rope_plain(x, cos, sin, rot, layout, split_half):
    """Rotates the first `rot` channels of each head; cos, sin [B, L, rot / 2]."""
    if layout == "HND":
        cos, sin = cos[:, None], sin[:, None]
    else:
        cos, sin = cos[:, :, None], sin[:, :, None]
    y = x.float()
    r, rest = y[..., :rot], y[..., rot:]
    if split_half:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def _plain_rope(st):
    c = st["case"]
    ang = _angles(st["positions"], st["inv_freq"], st["axis_pairs"])
    cos = (ang.cos() * st["scale"]).float()
    sin = (ang.sin() * st["scale"]).float()
    with torch.no_grad():
        outs = [_rope_plain(st[n].detach(), cos, sin, c["rot"], c["layout"], c["split_half"])
                for n in ("q", "k")]
        if c["grad"]:
            # The transpose of a rotation is the rotation by the negative angle.
            outs += [_rope_plain(st[n], cos, -sin, c["rot"], c["layout"], c["split_half"])
                     for n in ("dq", "dk")]
    return outs


def _plain_freqs(st):
    ang = _angles(st["positions"], st["inv_freq"], st["axis_pairs"])
    cos, sin = ang.cos() * st["scale"], ang.sin() * st["scale"]
    m = torch.stack([cos, -sin, sin, cos], dim=-1)
    return m.view(*ang.shape[:2], 1, ang.shape[2], 2, 2).to(DTYPES[st["case"]["dtype"]])


def _head(t, layout, b, h):
    return t[b, h] if layout == "HND" else t[b, :, h]


def _plain_select(st):
    """Score = mean query of the query block . mean key of the key block, in 64
    bits since the ranks of near blocks decide; ties go to the lowest block."""
    c = st["case"]
    lay, B, Hq, Hk, Lq, Lk = (c[n] for n in ("layout", "B", "Hq", "Hk", "Lq", "Lk"))
    nqb, nkb = -(-Lq // QB), -(-Lk // KB)
    keep = min(c["keep"], nkb)
    dev = st["q8"].device
    out = torch.empty((B, Hq, nqb, keep), dtype=torch.int32, device=dev)
    start = torch.arange(nkb, device=dev) * KB
    q_count = (Lq - torch.arange(nqb, device=dev) * QB).clamp(max=QB).double()
    for b in range(B):
        length = (torch.tensor(Lk, device=dev) if st["lengths"] is None
                  else st["lengths"][b].long().clamp(0, Lk))
        count = (length - start).clamp(0, KB)
        seen = (torch.arange(nkb * KB, device=dev) < length).view(nkb, KB, 1)
        for hk in range(Hk):
            k = torch.zeros((nkb * KB, D), device=dev)
            k[:Lk] = _head(st["k8"], lay, b, hk)
            ksum = (k.view(nkb, KB, D) * seen).sum(dim=1).double()
            kmean = ksum * (st["ks"][b, hk].double() / count.clamp_min(1).double())[:, None]
            for h in range(hk * (Hq // Hk), (hk + 1) * (Hq // Hk)):
                q = torch.zeros((nqb * QB, D), device=dev)
                q[:Lq] = _head(st["q8"], lay, b, h)
                tiles = q.view(nqb, QB // 16, 16, D).sum(dim=2).double()
                qs = torch.zeros(nqb * 8, device=dev, dtype=torch.float64)
                qs[:st["qs"].size(2)] = st["qs"][b, h]
                qmean = (tiles * qs.view(nqb, 8, 1)).sum(dim=1) / q_count[:, None]
                score = qmean @ kmean.T
                allowed = (count > 0)[None].expand(nqb, nkb)
                if st["policy"] is not None:
                    score = torch.where(st["policy"] == 1, math.inf, score)
                    allowed = allowed & (st["policy"] >= 0)
                score = torch.where(allowed, score, -math.inf)
                best = score.sort(dim=1, descending=True, stable=True).indices[:, :keep]
                best = torch.where(allowed.gather(1, best), best, nkb).sort(dim=1).values
                out[b, h] = torch.where(best == nkb, -1, best)
    return out


def _plain_attend(st):
    """Softmax attention over the listed key blocks of each query block."""
    c = st["case"]
    lay, B, Hq, Hk, Lq, Lk = (c[n] for n in ("layout", "B", "Hq", "Hk", "Lq", "Lk"))
    nqb, nkb = -(-Lq // QB), -(-Lk // KB)
    lists, v = st["lists"], st["v"]
    out = torch.zeros(st["q8"].shape, dtype=v.dtype, device=v.device)
    lse = torch.empty((B, Hq, Lq), device=v.device)
    keep = lists.size(3)
    step = max(1, 20000 // keep)      # query blocks at a time
    for b in range(B):
        length = Lk if st["lengths"] is None else st["lengths"][b]
        for hk in range(Hk):
            k = torch.zeros((nkb * KB, D), device=v.device)
            k[:Lk] = _head(st["k8"], lay, b, hk)
            k = k.view(nkb, KB, D) * st["ks"][b, hk][:, None, None]
            vv = torch.zeros((nkb * KB, D), device=v.device)
            vv[:Lk] = _head(v, lay, b, hk)
            vv = vv.view(nkb, KB, D)
            for h in range(hk * (Hq // Hk), (hk + 1) * (Hq // Hk)):
                q = torch.zeros((nqb * QB, D), device=v.device)
                q[:Lq] = _head(st["q8"], lay, b, h)
                qs = torch.zeros(nqb * 8, device=v.device)
                qs[:st["qs"].size(2)] = st["qs"][b, h]
                q = (q.view(-1, 16, D) * qs[:, None, None]).view(nqb, QB, D)
                for i in range(0, nqb, step):
                    idx = lists[b, h, i:i + step].long()
                    n = idx.size(0)
                    at = idx.clamp_min(0)
                    tok = at[..., None] * KB + torch.arange(KB, device=v.device)
                    ok = ((idx[..., None] >= 0) & (tok < length)).view(n, 1, keep * KB)
                    s = torch.bmm(q[i:i + n], k[at].view(n, keep * KB, D).transpose(1, 2))
                    s = torch.where(ok, s * D ** -0.5, -math.inf)
                    m = s.amax(dim=2, keepdim=True)
                    m = torch.where(m == -math.inf, 0.0, m)
                    p = (s - m).exp_()
                    d = p.sum(dim=2, keepdim=True)
                    o = torch.bmm(p, vv[at].view(n, keep * KB, D)) / torch.where(d > 0, d, 1.0)
                    rows = slice(i * QB, min((i + n) * QB, Lq))
                    size = rows.stop - rows.start
                    _head(out, lay, b, h)[rows] = o.view(-1, D)[:size].to(v.dtype)
                    lse[b, h, rows] = (m + d.log()).view(-1)[:size]
    return [out, lse] if c["lse"] else out


# --------------------------------------------------------------------- run --

def run(state):
    st, c = state, state["case"]
    op = c["op"]
    if not own:
        return {"rope": _plain_rope, "freqs": _plain_freqs, "select": _plain_select,
                "attend": _plain_attend}[op](st)
    kernel = _package()
    if op == "rope":
        q, k = kernel.turing_rope_qk(st["q"], st["k"], st["positions"], st["inv_freq"],
                                     tensor_layout=c["layout"], split_half=c["split_half"],
                                     axis_pairs=st["axis_pairs"], scale=st["scale"])
        if not c["grad"]:
            return [q, k]
        dq, dk = torch.autograd.grad([q, k], [st["q"], st["k"]], [st["dq"], st["dk"]])
        return [q.detach(), k.detach(), dq, dk]
    if op == "freqs":
        return kernel.turing_rope_freqs(st["positions"], st["inv_freq"],
                                        axis_pairs=st["axis_pairs"], scale=st["scale"],
                                        dtype=DTYPES[c["dtype"]])
    sage = kernel.turing_sage
    if op == "select":
        return sage.select_key_blocks(st["q8"], st["qs"], st["k8"], st["ks"], c["keep"],
                                      tensor_layout=c["layout"], key_lengths=st["lengths"],
                                      block_policy=st["policy"])
    result = sage.sparse_sageattn_prequantized(
        st["q8"], st["qs"], st["k8"], st["ks"], st["v"], st["lists"], tensor_layout=c["layout"],
        key_lengths=st["lengths"], return_lse=c["lse"])
    return list(result) if c["lse"] else result


# ------------------------------------------------------------ work and exact --

def work(case):
    op = case["op"]
    if op in ("rope", "freqs"):
        size = 4 if case["dtype"] == "f32" else 2
        tokens = case["B"] * case["L"]
        small = tokens * case["axes"] * 8 + case["rot"] // 2 * 8
        if op == "freqs":
            return {"bytes": tokens * case["rot"] * 2 * size + small,
                    "flops": tokens * case["rot"] // 2 * 2}
        n = tokens * (case["Hq"] + case["Hk"])
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * case["D"] * size + small),
                "flops": passes * n * case["rot"] * 3}
    B, Hq, Hk, Lq, Lk = (case[n] for n in ("B", "Hq", "Hk", "Lq", "Lk"))
    nqb, nkb = -(-Lq // QB), -(-Lk // KB)
    keep = min(case["keep"], nkb)
    q = B * Hq * (Lq * D + -(-Lq // 64) * 16)
    lists = B * Hq * nqb * keep * 4
    if op == "select":
        return {"bytes": q + B * Hk * (Lk * D + nkb * 4) + lists
                + (nqb * nkb if case["policy"] else 0),
                "flops": B * (Hq * Lq + Hk * Lk) * D + 2 * B * Hq * nqb * nkb * D}
    # Keys and values that some list names: at most all of them, at most every list's own.
    keys = B * min(Hk * Lk, Hq * nqb * keep * KB)
    return {"bytes": q + lists + keys * (D + 2 * D) + B * Hq * Lq * D * 2
            + (B * Hq * Lq * 4 if case["lse"] else 0),
            "flops": 4 * B * Hq * Lq * min(keep * KB, Lk) * D}


def _exact_turn(case, x, pos, inv, pairs_of, scale, sign):
    """Rotation as a complex product, one axis at a time."""
    z = x.double()
    if case["layout"] == "HND":
        z = z.transpose(1, 2)
    rot = case["rot"]
    if case["split_half"]:
        w = torch.complex(z[..., :rot // 2], z[..., rot // 2:rot])
    else:
        w = torch.view_as_complex(z[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous())
    lo = 0
    turned = torch.empty_like(w)
    for a, n in enumerate(pairs_of):
        p = (pos if pos.dim() == 2 else pos[..., a]).double()
        phase = p[:, :, None, None] * inv[lo:lo + n] * sign
        turned[..., lo:lo + n] = w[..., lo:lo + n] * torch.polar(
            torch.full_like(phase, scale), phase)
        lo += n
    y = z.clone()
    if case["split_half"]:
        y[..., :rot // 2], y[..., rot // 2:rot] = turned.real, turned.imag
    else:
        y[..., :rot] = torch.view_as_real(turned).flatten(-2)
    return y.transpose(1, 2) if case["layout"] == "HND" else y


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("rope", "freqs"):
        pairs_of = st["axis_pairs"] or [case["rot"] // 2]
        if op == "rope":
            with torch.no_grad():
                args = (st["positions"], st["inv_freq"], pairs_of, st["scale"])
                outs = [_exact_turn(case, st[n], *args, 1.0) for n in ("q", "k")]
                if case["grad"]:
                    outs += [_exact_turn(case, st[n], *args, -1.0) for n in ("dq", "dk")]
            return outs
        m = torch.empty((case["B"], case["L"], 1, case["rot"] // 2, 2, 2), dtype=torch.float64,
                        device=DEV)
        lo = 0
        for a, n in enumerate(pairs_of):
            p = (st["positions"] if case["axes"] == 1 else st["positions"][..., a]).double()
            turn = torch.polar(torch.full((), st["scale"], dtype=torch.float64, device=DEV),
                               p[..., None] * st["inv_freq"][lo:lo + n])
            m[:, :, 0, lo:lo + n, 0, 0] = turn.real
            m[:, :, 0, lo:lo + n, 1, 1] = turn.real
            m[:, :, 0, lo:lo + n, 1, 0] = turn.imag
            m[:, :, 0, lo:lo + n, 0, 1] = -turn.imag
            lo += n
        return m
    lay, B, Hq, Hk, Lq, Lk = (case[n] for n in ("layout", "B", "Hq", "Hk", "Lq", "Lk"))
    nqb, nkb = -(-Lq // QB), -(-Lk // KB)

    def values(codes, scales, tile, b, h):
        x = _head(codes, lay, b, h).double()
        return x * scales[b, h].double().repeat_interleave(tile)[:x.size(0), None]

    if op == "select":
        keep = min(case["keep"], nkb)
        out = torch.full((B, Hq, nqb, keep), -1, dtype=torch.int32, device=DEV)
        for b in range(B):
            length = Lk if st["lengths"] is None else min(int(st["lengths"][b]), Lk)
            blocks = -(-length // KB)
            for h in range(Hq):
                x = values(st["q8"], st["qs"], 16, b, h)
                y = values(st["k8"], st["ks"], 64, b, h * Hk // Hq)
                qm = torch.stack([part.mean(dim=0) for part in x.split(QB)])
                full = length // KB
                km = y[:full * KB].view(full, KB, D).mean(dim=1)
                if blocks > full:
                    km = torch.cat([km, y[full * KB:length].mean(dim=0, keepdim=True)])
                s = (qm[:, None, :] * km[None]).sum(dim=2) if nqb == 1 else qm @ km.T
                never = torch.zeros_like(s, dtype=torch.bool)
                if st["policy"] is not None:
                    s = s.masked_fill(st["policy"][:, :blocks] == 1, math.inf)
                    never = st["policy"][:, :blocks] < 0
                s = s.masked_fill(never, -math.inf)
                # Everything above the keep-th value, then the first of its equals.
                n = min(keep, blocks)
                edge = s.topk(n, dim=1).values[:, -1:]
                above, equal = s > edge, s == edge
                left = n - above.sum(dim=1, keepdim=True)
                chosen = (above | (equal & (equal.cumsum(dim=1) <= left))) & ~never
                where = chosen.cumsum(dim=1) - 1
                qi, kj = chosen.nonzero(as_tuple=True)
                out[b, h, qi, where[qi, kj]] = kj.int()
        return out
    out = torch.zeros(st["q8"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64, device=DEV)
    keep = st["lists"].size(3)
    for b in range(B):
        length = Lk if st["lengths"] is None else int(st["lengths"][b])
        for h in range(Hq):
            x = values(st["q8"], st["qs"], 16, b, h) / math.sqrt(D)
            pad = nkb * KB - Lk
            hk = h * Hk // Hq
            y = torch.nn.functional.pad(values(st["k8"], st["ks"], 64, b, hk), (0, 0, 0, pad))
            z = torch.nn.functional.pad(_head(st["v"], lay, b, hk).double(), (0, 0, 0, pad))
            x = torch.nn.functional.pad(x, (0, 0, 0, nqb * QB - Lq)).view(nqb, QB, D)
            step = max(1, 8000 // keep)
            for i in range(0, nqb, step):
                ids = st["lists"][b, h, i:i + step].long()
                n = ids.size(0)
                tok = (ids.clamp_min(0)[:, :, None] * KB
                       + torch.arange(KB, device=DEV)).view(n, -1)
                hide = (ids < 0).repeat_interleave(KB, dim=1) | (tok >= length)
                s = (x[i:i + n] @ y[tok].transpose(1, 2)).masked_fill(hide[:, None], -math.inf)
                total = torch.logsumexp(s, dim=2)
                p = (s - total[..., None]).exp().nan_to_num(0.0)
                lo, hi = i * QB, min((i + n) * QB, Lq)
                _head(out, lay, b, h)[lo:hi] = (p @ z[tok]).view(-1, D)[:hi - lo]
                lse[b, h, lo:hi] = total.view(-1)[:hi - lo]
    return [out, lse] if case["lse"] else out
