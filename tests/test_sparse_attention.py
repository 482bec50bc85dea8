"""Block-sparse Sage attention: the lists and the attention over them against
64-bit references, as used together, and their refusals.

Bound of one attention output o = sum_j w_j v_j (w = p / d), with h half a step
of V's type and A = sum_j w_j |v_j|:
  * p is rounded to V's type: h A (fp16 also has subnormals: n 2^-25 max |v|,
    the largest p of a row being at least 1);
  * the exponent's factors round three times and its FMA once on logits below 64
    (4 x 64 x 2^-24 ln 2), 2^x to 2^-22, in p and in d: 3e-5 A;
  * up to 4096 products and sums in fp32, in O and in d: 2 x 4096 x 2^-24 A = 5e-4 A;
  * the output's own rounding: h |o|.
The log-sum-exp has the second and third of these, and its own rounding.
"""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, _sage_sparse, turing_sage

gpu = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def to_hnd(t, layout):
    return t if layout == "HND" else t.transpose(1, 2)


def codes(B, H, L, D, tile, layout, seed, gain=1.0, spread=0.0):
    """INT8 codes and one scale per `tile` tokens; spread > 0 varies the scales by
    up to e^spread."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (B, H, L, D), generator=g)
    drift = torch.randint(-40, 41, (B, H, -(-L // 50), D), generator=g)
    q = (q // 3 + drift.repeat_interleave(50, dim=2)[:, :, :L]).clamp(-127, 127).to(torch.int8)
    n = -(-L // 64) * 64 // tile
    s = (torch.rand((B, H, n), generator=g) * spread).exp() * (0.02 * gain)
    q = q if layout == "HND" else q.transpose(1, 2)
    return q.contiguous().cuda(), s.float().cuda()


def dequant(c, s, tile, layout):
    c = to_hnd(c, layout).double()
    return c * s.double().repeat_interleave(tile, dim=2)[:, :, :c.size(2), None]


def lengths_of(key_lengths, B, Lk):
    return [Lk] * B if key_lengths is None else [min(max(int(n), 0), Lk) for n in key_lengths]


def reference(q8, qs, k8, ks, v, lists, layout, key_lengths=None, sm_scale=128 ** -0.5):
    """(o, A, lse) in fp64, one query block at a time, a block once per mention."""
    q, k, vv = dequant(q8, qs, 16, layout), dequant(k8, ks, 64, layout), to_hnd(v, layout)
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    o = torch.zeros_like(q)
    A = torch.zeros_like(q)
    lse = torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths_of(key_lengths, B, Lk)):
        for h in range(Hq):
            hk = h * Hk // Hq
            for i in range(lists.size(2)):
                idx = [j for j in lists[b, h, i].tolist() if 0 <= j and j * 64 < length]
                if not idx:
                    continue
                tok = torch.cat([torch.arange(j * 64, min(j * 64 + 64, length)) for j in idx]).cuda()
                s = q[b, h, i * 128:i * 128 + 128] @ k[b, hk, tok].T * sm_scale
                total = s.logsumexp(dim=1)
                w = (s - total[:, None]).exp()
                x = vv[b, hk, tok].double()
                o[b, h, i * 128:i * 128 + 128] = w @ x
                A[b, h, i * 128:i * 128 + 128] = w @ x.abs()
                lse[b, h, i * 128:i * 128 + 128] = total
    return o, A, lse


def check(out, lse, ref, dtype, keys, layout):
    o, A, want_lse = ref
    h = HALF_STEP[dtype]
    vmax = 6.0  # |v| of normal values
    bound = (h + 5.3e-4) * A + h * o.abs() + (keys * 2.0 ** -25 * vmax if dtype == torch.float16
                                              else 0.0)
    err = (to_hnd(out, layout).double() - o).abs()
    assert (err <= bound).all(), ((err - bound).max().item(), err.max().item())
    if lse is not None:
        assert torch.equal(lse.isinf(), want_lse.isinf())
        d = (lse.double() - want_lse)[~want_lse.isinf()].abs()
        lim = 5.3e-4 + 2.0 ** -22 * want_lse[~want_lse.isinf()].abs()
        assert (d <= lim).all(), d.max().item()


def value(B, H, L, dtype, layout, seed, D=128):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn((B, H, L, D), generator=g)
    return (v if layout == "HND" else v.transpose(1, 2).contiguous()).to(dtype).cuda()


def random_lists(B, H, Lq, Lk, keep, seed, dirty=False):
    nqb, nkb = -(-Lq // 128), -(-Lk // 64)
    g = torch.Generator().manual_seed(seed)
    r = torch.rand((B, H, nqb, nkb), generator=g).argsort(dim=3)[..., :keep].to(torch.int32)
    if dirty:
        # Any order, open places anywhere, blocks past the end, one block twice.
        bad = torch.tensor([-1, nkb, -2 ** 31, 2 ** 31 - 1, nkb + 7], dtype=torch.int64)
        hit = torch.rand(r.shape, generator=g) < 0.3
        r = torch.where(hit, bad[torch.randint(0, 5, r.shape, generator=g)].to(torch.int32), r)
        if keep > 2:
            r[..., 2] = r[..., 0]
        r[:, :, 0] = -1 if nqb > 1 else r[:, :, 0]
    return r.cuda()


SHAPES = [
    # B, Hq, Hk, Lq, Lk, keep
    (1, 1, 1, 1, 1, 1), (1, 3, 1, 1, 4000, 40), (2, 4, 2, 127, 63, 1), (1, 2, 2, 128, 64, 1),
    (1, 2, 1, 129, 65, 2), (2, 2, 2, 300, 1000, 5), (1, 2, 2, 257, 4096, 64),
    (3, 6, 3, 130, 700, 11), (1, 5, 5, 640, 515, 3), (1, 80, 8, 513, 640, 4)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("dirty", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_fp64(dtype, layout, dirty, shape):
    B, Hq, Hk, Lq, Lk, keep = shape
    q8, qs = codes(B, Hq, Lq, 128, 16, layout, 1)
    k8, ks = codes(B, Hk, Lk, 128, 64, layout, 2)
    v = value(B, Hk, Lk, dtype, layout, 3)
    lists = random_lists(B, Hq, Lq, Lk, keep, 4, dirty)
    out, lse = turing_sage.sparse_sageattn_prequantized(
        q8, qs, k8, ks, v, lists, tensor_layout=layout, return_lse=True)
    assert out.shape == q8.shape and out.dtype == dtype
    check(out, lse, reference(q8, qs, k8, ks, v, lists, layout), dtype, keep * 64, layout)
    # The same call gives the same bits; so does an output of the caller's.
    place = torch.full_like(out, float("nan"))
    again = turing_sage.sparse_sageattn_prequantized(
        q8, qs, k8, ks, v, lists, tensor_layout=layout, output=place)
    assert again is place and torch.equal(again, out)
    assert _lib.device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq", [1, 200])
def test_key_lengths_hide_the_padding(dtype, Lq):
    """Padding of NaN and infinity in V and any codes in K is never seen; lengths
    below 0, above Lk, zero, one, on and off a block border."""
    lens = [0, 1, 63, 64, 65, 500, 640, 10 ** 6, -5]
    B, Hq, Hk, Lk = len(lens), 4, 2, 640
    q8, qs = codes(B, Hq, Lq, 128, 16, "HND", 1)
    k8, ks = codes(B, Hk, Lk, 128, 64, "HND", 2)
    v = value(B, Hk, Lk, dtype, "HND", 3)
    key_lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lists = random_lists(B, Hq, Lq, Lk, 10, 5)
    ref = reference(q8, qs, k8, ks, v, lists, "HND", lens)
    for b, n in enumerate(lengths_of(lens, B, Lk)):
        v[b, :, n:] = float("nan")
        v[b, :, n + 1::2] = float("inf")
    out, lse = turing_sage.sparse_sageattn_prequantized(
        q8, qs, k8, ks, v, lists, key_lengths=key_lengths, return_lse=True)
    check(out, lse, ref, dtype, 640, "HND")
    assert (out[0] == 0).all() and (out[-1] == 0).all()


@gpu
@pytest.mark.parametrize("spread,gain", [(0.0, 30.0), (2.0, 1.0), (0.0, 1e-4)])
@pytest.mark.parametrize("Lq", [1, 130])
def test_scales(spread, gain, Lq):
    """Logits up to hundreds (softmax near argmax), blocks of very different scales
    (the reference point moves) and logits near 0.  The exponent's bound grows with
    the logits: 4 x max |logit| x 2^-24 in p and d."""
    q8, qs = codes(1, 2, Lq, 128, 16, "HND", 1, math.sqrt(gain), spread)
    k8, ks = codes(1, 2, 1500, 128, 64, "HND", 2, math.sqrt(gain), spread)
    v = value(1, 2, 1500, torch.bfloat16, "HND", 3)
    lists = random_lists(1, 2, Lq, 1500, 20, 4)
    out, lse = turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v, lists, return_lse=True)
    o, A, want = reference(q8, qs, k8, ks, v, lists, "HND")
    top = (dequant(q8, qs, 16, "HND") @ dequant(k8, ks, 64, "HND").transpose(2, 3)).abs().max()
    grow = 2 * 4 * top.item() * 128 ** -0.5 * 2.0 ** -24
    bound = (2.0 ** -8 + 5.3e-4 + grow) * A + 2.0 ** -8 * o.abs()
    err = (out.double() - o).abs()
    assert (err <= bound).all(), (err - bound).max().item()
    assert ((lse.double() - want).abs() <= 5.3e-4 + grow + 2.0 ** -22 * want.abs()).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq", [1, 200])
@pytest.mark.parametrize("where", ["sm_scale", "query", "key", "both"])
def test_negative_scales(dtype, Lq, where):
    """A negative sm_scale, negative scales of some query tiles (two tiles share a
    warp) or key blocks: the row's largest score is then the smallest integer one.
    Logits of either sign up to tens, as in test_scales."""
    q8, qs = codes(1, 4, Lq, 128, 16, "HND", 1, math.sqrt(30.0))
    k8, ks = codes(1, 2, 1500, 128, 64, "HND", 2, math.sqrt(30.0))
    v = value(1, 2, 1500, dtype, "HND", 3)
    lists = random_lists(1, 4, Lq, 1500, 20, 4)
    sm_scale = 128 ** -0.5
    if where == "sm_scale":
        sm_scale = -sm_scale
    if where in ("query", "both"):
        qs[..., ::2] *= -1
    if where in ("key", "both"):
        ks[..., 1::3] *= -1
    out, lse = turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v, lists,
                                                        sm_scale=sm_scale, return_lse=True)
    o, A, want = reference(q8, qs, k8, ks, v, lists, "HND", sm_scale=sm_scale)
    top = (dequant(q8, qs, 16, "HND") @ dequant(k8, ks, 64, "HND").repeat_interleave(
        2, dim=1).transpose(2, 3)).abs().max().item() * 128 ** -0.5
    grow = 2 * 4 * top * 2.0 ** -24
    bound = (HALF_STEP[dtype] + 5.3e-4 + grow) * A + HALF_STEP[dtype] * o.abs() + (
        20 * 64 * 2.0 ** -25 * 6.0 if dtype == torch.float16 else 0.0)
    err = (out.double() - o).abs()
    assert (err <= bound).all(), (err - bound).max().item()
    assert ((lse.double() - want).abs() <= 5.3e-4 + grow + 2.0 ** -22 * want.abs()).all()


@gpu
def test_small_scores_in_blocks_of_large_scale():
    """Queries whose codes are small beside their tile's largest: the scores are
    small integers times a large factor, exact for every key."""
    q8, qs = codes(1, 1, 128, 128, 16, "HND", 1)
    k8, ks = codes(1, 1, 640, 128, 64, "HND", 2)
    q8 = torch.where(torch.arange(128, device="cuda")[None, None, :, None] % 16 == 0, q8, q8 // 60)
    qs, ks = qs * 20, ks * (1 + torch.arange(10, device="cuda").float() * 0.37)
    v = value(1, 1, 640, torch.float16, "HND", 3)
    lists = random_lists(1, 1, 128, 640, 10, 4)
    out = turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v, lists, sm_scale=1e-3)
    o, A, _ = reference(q8, qs, k8, ks, v, lists, "HND", sm_scale=1e-3)
    small = torch.arange(128, device="cuda") % 16 != 0
    bound = (2.0 ** -11 + 5.3e-4) * A + 2.0 ** -11 * o.abs() + 640 * 2.0 ** -25 * 6
    err = (out.double() - o).abs()
    assert (err <= bound)[:, :, small].all(), (err - bound)[:, :, small].max().item()


@gpu
def test_nan_scales_stay_in_their_rows():
    q8, qs = codes(1, 1, 256, 128, 16, "HND", 1)
    k8, ks = codes(1, 1, 640, 128, 64, "HND", 2)
    v = value(1, 1, 640, torch.bfloat16, "HND", 3)
    lists = torch.tensor([[[[0, 1, 2], [3, 4, 5]]]], dtype=torch.int32, device="cuda")
    qs[0, 0, 2] = float("nan")   # rows 32..47
    ks[0, 0, 4] = float("nan")   # seen by the second query block only
    out = turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v, lists)
    bad = out.isnan().all(dim=3)[0, 0]
    want = torch.zeros(256, dtype=torch.bool, device="cuda")
    want[32:48] = True
    want[128:] = True
    assert torch.equal(bad, want) and torch.equal(out.isnan().any(dim=3)[0, 0], want)


@gpu
def test_strided_values_and_outputs():
    """V as a view of a fused row, an output with gaps; bytes outside stay."""
    B, H, L = 2, 3, 200
    q8, qs = codes(B, H, L, 128, 16, "NHD", 1)
    k8, ks = codes(B, H, L, 128, 64, "NHD", 2)
    g = torch.Generator().manual_seed(3)
    fused = torch.randn((B, L, 3, H, 128), generator=g).to(torch.bfloat16).cuda()
    v = fused[:, :, 2]
    lists = random_lists(B, H, L, L, 3, 4)
    want = turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v.contiguous(), lists,
                                                    tensor_layout="NHD")
    room = torch.full((B, L + 3, H, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    place = room[:, :L, :, :128]
    turing_sage.sparse_sageattn_prequantized(q8, qs, k8, ks, v, lists, tensor_layout="NHD",
                                             output=place)
    assert torch.equal(place, want)
    assert (room[:, L:] == 7).all() and (room[..., 128:] == 7).all()


# ------------------------------------------------------------- block choice --

def choose(q8, qs, k8, ks, keep, layout, key_lengths=None, policy=None):
    """The lists by rank counting in fp64 (a NaN score as -inf)."""
    q, k = dequant(q8, qs, 16, layout), dequant(k8, ks, 64, layout)
    B, Hq, Lq, _ = q.shape
    Hk, Lk = k.shape[1:3]
    nqb, nkb = -(-Lq // 128), -(-Lk // 64)
    keep = min(keep, nkb)
    out = torch.full((B, Hq, nqb, keep), -1, dtype=torch.int32, device=q.device)
    qm = torch.stack([t.mean(dim=2) for t in q.split(128, dim=2)], dim=2)
    order = torch.arange(nkb, device=q.device)
    for b, length in enumerate(lengths_of(key_lengths, B, Lk)):
        n = -(-length // 64)
        if n == 0:
            continue
        km = torch.stack([t.mean(dim=1) for t in k[b, :, :length].split(64, dim=1)], dim=1)
        for h in range(Hq):
            s = (qm[b, h][:, None] * km[h * Hk // Hq][None]).sum(dim=2)
            s = torch.where(s.isnan(), -math.inf, s)
            for i in range(nqb):
                pol = (torch.zeros(n) if policy is None else policy[min(i, len(policy) - 1), :n])
                rank = sorted((j for j in range(n) if pol[j] >= 0),
                              key=lambda j: (pol[j] <= 0, -s[i, j].item() if pol[j] <= 0 else 0, j))
                got = sorted(rank[:keep])
                out[b, h, i, :len(got)] = order[torch.tensor(got, dtype=torch.long)].int()
    return out


@gpu
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES + [(1, 2, 2, 1100, 777, 999)])
def test_choice_matches_fp64(layout, D, shape):
    B, Hq, Hk, Lq, Lk, keep = shape
    q8, qs = codes(B, Hq, Lq, D, 16, layout, 1, spread=1.0)
    k8, ks = codes(B, Hk, Lk, D, 64, layout, 2, spread=1.0)
    got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep, tensor_layout=layout)
    assert torch.equal(got, choose(q8, qs, k8, ks, keep, layout))


@gpu
@pytest.mark.parametrize("rows", [0, 1, 3])
@pytest.mark.parametrize("keep", [1, 4, 11])
def test_choice_lengths_and_policy(rows, keep):
    lens = [0, 1, 64, 65, 511, 700, 9999, -1]
    B, Lq, Lk = len(lens), 300, 700
    q8, qs = codes(B, 4, Lq, 128, 16, "HND", 1)
    k8, ks = codes(B, 2, Lk, 128, 64, "HND", 2)
    policy = None
    if rows:
        g = torch.Generator().manual_seed(rows)
        policy = torch.randint(-1, 2, (rows, 11), generator=g).to(torch.int8)
        policy[0, :3] = torch.tensor([-128, 127, 1], dtype=torch.int8)
        if rows > 1:
            policy[1] = -1       # a query block that sees nothing
            policy[2] = 1
    got = turing_sage.select_key_blocks(
        q8, qs, k8, ks, keep, key_lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"),
        block_policy=None if policy is None else policy.cuda())
    assert torch.equal(got, choose(q8, qs, k8, ks, keep, "HND", lens, policy))


@gpu
@pytest.mark.parametrize("Lk", [70, 640, 100000, 200000])
def test_ties_zeros_and_nan(Lk):
    """Equal scores go to the lowest block: all of them zero (of either sign), pairs
    of equal key blocks, NaN and infinite scales."""
    nkb = -(-Lk // 64)
    keep = min(nkb, 9)
    q8, qs = codes(1, 1, 150, 128, 16, "HND", 1)
    k8, ks = codes(1, 1, Lk, 128, 64, "HND", 2)
    zero = turing_sage.select_key_blocks(q8, qs, torch.zeros_like(k8), ks, keep)
    assert (zero == torch.arange(keep, device="cuda")).all()
    zero = turing_sage.select_key_blocks(q8, qs, torch.zeros_like(k8),
                                         torch.where(torch.arange(nkb, device="cuda") % 2 == 0,
                                                     ks, -ks), keep)
    assert (zero == torch.arange(keep, device="cuda")).all()
    if nkb >= 10:
        even = nkb // 2 * 2
        k2 = k8.clone()
        blocks = k2[:, :, :(Lk // 64) * 64].view(1, 1, Lk // 64, 64, 128)
        blocks[:, :, 1:even:2] = blocks[:, :, 0:even - 1:2][:, :, :blocks[:, :, 1:even:2].size(2)]
        s2 = ks.clone()
        s2[:, :, 1:even:2] = s2[:, :, 0:even:2]
        got = turing_sage.select_key_blocks(q8, qs, k2, s2, keep)
        if Lk < 5000:
            assert torch.equal(got, choose(q8, qs, k2, s2, keep, "HND"))
        odd = got % 2 == 1   # an odd block only beside its equal
        prev = torch.cat([got[..., :1] * 0 - 2, got[..., :-1]], dim=3)
        assert (~odd | (prev == got - 1) | (got >= even)).all()
    s3 = ks.clone()
    s3[0, 0, 0] = float("nan")
    s3[0, 0, -1] = float("inf")
    got = turing_sage.select_key_blocks(q8, qs, k8, s3, keep)
    if Lk < 5000:
        assert torch.equal(got, choose(q8, qs, k8, s3, keep, "HND"))


@gpu
@pytest.mark.parametrize("nkb", [2, 100, 2000])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_one_step_of_fp64_apart(nkb, sign):
    """Channel 0 alone gives every block 127 * 2^33 * 8128, in [2^52, 2^53), where a
    step of fp64 is one; channel 1 adds an integer below 128."""
    q8 = torch.zeros(1, 1, 128, 128, dtype=torch.int8)
    q8[0, 0, 0, 0] = 127 * sign
    q8[0, 0, 16, 1] = 1
    qs = torch.ones(1, 1, 8)
    qs[0, 0, 1] = 2.0 ** -33
    add = torch.randperm(max(nkb, 128), generator=torch.Generator().manual_seed(nkb))[:nkb] % 128
    if nkb == 2:
        add = torch.tensor([2, 3])     # equal but for the last bit
    k8 = torch.zeros(1, 1, nkb, 64, 128, dtype=torch.int8)
    k8[..., 0] = 127
    k8[0, 0, :, 0, 1] = add.to(torch.int8)
    k8 = k8.view(1, 1, nkb * 64, 128).cuda()
    rank = sorted(range(nkb), key=lambda j: (-int(add[j]), j))
    for keep in {1, min(37, nkb - 1), nkb // 2}:
        got = turing_sage.select_key_blocks(q8.cuda(), qs.cuda(), k8,
                                            torch.ones(1, 1, nkb, device="cuda"), keep)
        assert got[0, 0, 0].tolist() == sorted(rank[:keep])


@gpu
@pytest.mark.parametrize("nkb", [40, 500, 2000])
@pytest.mark.parametrize("spread", [20, 31, 34])
def test_scores_that_cancel(nkb, spread):
    """Key sums whose large products cancel to some 2^spread of 2^52, by integers.
    A query channel's mean is written in base 128, a digit to a tile of tokens."""
    g = torch.Generator().manual_seed(nkb + spread)
    rand = lambda lo, hi, n: torch.randint(lo, hi, (n,), generator=g).tolist()
    q = [(1 << 39) + x for x in rand(0, 1 << 37, 1)] + [0, 0] + \
        [-(1 << 39) - x for x in rand(0, 1 << 36, 125)]
    q[1], q[2] = (1 << spread) // 64 + 1, 1
    sums, scores = [], []
    for j in range(nkb):
        S = [0] + rand(-64, 65, 1) + rand(-8000, 8000, 1) + rand(40, 64, 125)
        S[0] = -round(sum(a * b for a, b in zip(q[3:], S[3:])) / q[0])
        # What is left of channel 0's rounding is taken by the others' spread.
        sums.append(S)
        scores.append(sum(a * b for a, b in zip(q, S)))
    q8 = torch.zeros(1, 1, 128, 128, dtype=torch.int8)
    for c, v in enumerate(q):
        u = v + 64 * (128 ** 6 - 1) // 127
        for d in range(6):
            q8[0, 0, 16 * d, c] = (u >> 7 * d) % 128 - 64
    qs = torch.tensor([2.0 ** (7 * d) if d < 6 else 1.0 for d in range(8)]).view(1, 1, 8)
    S = torch.tensor(sums)
    row = torch.arange(64).view(1, 64, 1)
    base = torch.div(S, 64, rounding_mode="floor")[:, None]
    k8 = base + (row < (S - 64 * base[:, 0])[:, None]).long()
    assert k8.abs().max() <= 127 and torch.equal(k8.sum(1), S)
    k8 = k8.to(torch.int8).view(1, 1, nkb * 64, 128).cuda()
    rank = sorted(range(nkb), key=lambda j: (-float(scores[j]), j))
    for keep in (1, nkb // 7, nkb // 2, nkb - 1):
        got = turing_sage.select_key_blocks(q8.cuda(), qs.cuda(), k8,
                                            torch.ones(1, 1, nkb, device="cuda"), keep)
        assert got[0, 0, 0].tolist() == sorted(rank[:keep])


@gpu
@pytest.mark.parametrize("exponents", [(-149, -126), (-130, -100), (60, 127), (-149, 127)])
def test_scales_at_the_ends_of_fp32(exponents):
    q8, qs = codes(1, 2, 300, 128, 16, "HND", 1)
    k8, ks = codes(1, 2, 6400, 128, 64, "HND", 2)
    g = torch.Generator().manual_seed(3)
    power = torch.randint(exponents[0], exponents[1] + 1, ks.shape, generator=g).double()
    ks = torch.exp2(power).float().cuda()
    for keep in (1, 10, 50):
        got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep)
        assert torch.equal(got, choose(q8, qs, k8, ks, keep, "HND"))


@gpu
@pytest.mark.parametrize("Lk", [100000, 131071, 250001])
@pytest.mark.parametrize("keep", [1, 64, 600])
def test_choice_over_long_contexts(Lk, keep):
    q8, qs = codes(1, 2, 130, 128, 16, "HND", 1, spread=0.5)
    k8, ks = codes(1, 1, Lk, 128, 64, "HND", 2, spread=0.5)
    got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep)
    assert torch.equal(got, choose(q8, qs, k8, ks, keep, "HND"))


@gpu
@pytest.mark.parametrize("Lk", [100000, 200000])
def test_nan_and_infinite_scales_over_long_contexts(Lk):
    """Keys beyond the part of a row that the search holds in registers: a NaN score
    comes last and an infinite one first or last, wherever its block lies."""
    q8, qs = codes(1, 1, 150, 128, 16, "HND", 1)
    k8, ks = codes(1, 1, Lk, 128, 64, "HND", 2)
    for at in (0, 1400, -1):
        ks[0, 0, at] = float("nan")
        ks[0, 0, at - 2] = float("inf")
    n = ks.size(2)
    for keep in (1, 9, n - 2):
        got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep)
        assert torch.equal(got, choose(q8, qs, k8, ks, keep, "HND"))


@gpu
def test_choice_reads_views():
    """Codes as views of a fused row (16-byte aligned strides, not contiguous)."""
    g = torch.Generator().manual_seed(1)
    fused = torch.randint(-127, 128, (2, 300, 3, 4, 128), generator=g).to(torch.int8).cuda()
    qs = torch.rand((2, 4, 20), generator=g).cuda()
    ks = torch.rand((2, 4, 5), generator=g).cuda()
    a = turing_sage.select_key_blocks(fused[:, :, 0], qs, fused[:, :, 1], ks, 3,
                                      tensor_layout="NHD")
    b = turing_sage.select_key_blocks(fused[:, :, 0].contiguous(), qs, fused[:, :, 1].contiguous(),
                                      ks, 3, tensor_layout="NHD")
    assert torch.equal(a, b)


@gpu
def test_choice_from_two_threads():
    """Host threads, each on a stream of its own, choose blocks of different lengths:
    another shared memory size of the same kernel."""
    import threading

    lib, cases, errors = _lib.load(), [], []
    for Lk in (6400, 16000, 4160, 17000):
        q8, qs = codes(1, 2, 200, 128, 16, "HND", 1)
        k8, ks = codes(1, 2, Lk, 128, 64, "HND", 2)
        want = turing_sage.select_key_blocks(q8, qs, k8, ks, 7)
        size = ctypes.c_int64(0)
        assert lib.tb_select_key_blocks_workspace(1, 2, 2, 200, Lk, 128, ctypes.byref(size)) == 0
        room = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        strides = (ctypes.c_int64 * 6)(0, 200 * 128, 128, 0, Lk * 128, 128)
        cases.append((Lk, q8, qs, k8, ks, want, torch.zeros_like(want), room, strides,
                      torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(Lk, q8, qs, k8, ks, want, got, room, strides, stream):
        for _ in range(4000):
            if lib.tb_select_key_blocks(
                    q8.data_ptr(), k8.data_ptr(), qs.data_ptr(), ks.data_ptr(), None, None, 0,
                    got.data_ptr(), room.data_ptr(), room.numel(), 1, 2, 2, 200, Lk, 128, 7,
                    strides, stream.cuda_stream) != 0:
                errors.append(_lib.last_error())
                return

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert all(torch.equal(c[6], c[5]) for c in cases)


# ---------------------------------------------------------------- together --

@gpu
@pytest.mark.parametrize("D,layout,smooth", [(128, "HND", False), (64, "NHD", True),
                                             (96, "HND", True)])
def test_all_blocks_give_dense_attention(D, layout, smooth):
    """keep = every block: sageattn of the same codes, up to twice the bound of one."""
    q = value(2, 4, 333, torch.bfloat16, layout, 1, D)
    k, v = (value(2, 2, 450, torch.bfloat16, layout, s, D) for s in (2, 3))
    out = turing_sage.sparse_sageattn(q, k, v, 1000, tensor_layout=layout, smooth_k=smooth)
    dense = turing_sage.sageattn(q, k, v, tensor_layout=layout, smooth_k=smooth)
    assert out.shape == dense.shape == q.shape
    pre = turing_sage.prequantize_sageattn(q, k, v, tensor_layout=layout, smooth_k=smooth)
    lists = torch.arange(8, dtype=torch.int32, device="cuda").expand(2, 4, 3, 8).contiguous()
    o, A, _ = reference(pre.query_int8, pre.query_scale, pre.key_int8, pre.key_scale, pre.value,
                        lists, layout, sm_scale=D ** -0.5)
    o, A = o[..., :D], A[..., :D]
    bound = (2.0 ** -8 + 5.3e-4) * A + 2.0 ** -8 * o.abs()
    assert ((to_hnd(out, layout).double() - o).abs() <= bound).all()
    assert ((to_hnd(dense, layout).double() - o).abs() <= 2 * bound).all()


@gpu
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_rotary_choice_and_attention_together(layout):
    """A video self-attention: rotary positions on Q and K, INT8 codes, the choice
    with text blocks always kept and a padded batch, the attention."""
    import comfyui_turing_utils_kernel as kernel

    B, H, L, keep = 2, 4, 1000, 5
    axis_pairs = [22, 21, 21]
    q, k, v = (value(B, H, L, torch.bfloat16, layout, s) for s in (1, 2, 3))
    inv, scale = kernel.turing_rope_inv_freq(128, axis_pairs=axis_pairs, device="cuda")
    t = torch.arange(L, device="cuda")
    pos = torch.stack([t // 100, (t // 10) % 10, t % 10], dim=-1)
    q, k = kernel.turing_rope_qk(q, k, pos, inv, tensor_layout=layout, axis_pairs=axis_pairs,
                                 scale=scale)
    lens = [L, 700]
    key_lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    policy = torch.zeros((1, 16), dtype=torch.int8, device="cuda")
    policy[0, 3] = 1
    out, lse = turing_sage.sparse_sageattn(q, k, v, keep, tensor_layout=layout,
                                           key_lengths=key_lengths, block_policy=policy,
                                           return_lse=True)
    pre = turing_sage.prequantize_sageattn(q, k, v, tensor_layout=layout)
    args = (pre.query_int8, pre.query_scale, pre.key_int8, pre.key_scale)
    lists = choose(*args, keep, layout, lens, policy.cpu())
    assert torch.equal(lists, turing_sage.select_key_blocks(
        *args, keep, tensor_layout=layout, key_lengths=key_lengths, block_policy=policy))
    assert (lists == 3).any(dim=3).all()
    ref = reference(*args, v, lists, layout, lens)
    check(out, lse, ref, torch.bfloat16, keep * 64, layout)
    # Through the fused RMSNorm + RoPE prologue's codes.
    freqs = kernel.turing_rope_freqs(pos, inv, axis_pairs=axis_pairs, scale=scale)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    qk = turing_sage.prequantize_rms_rope_qk(q, k, w, w, freqs, epsilon=1e-6, rot_dim=128,
                                             tensor_layout=layout)
    pre = turing_sage.prequantize_sageattn_from_qk(qk, v)
    out, lse = turing_sage.sparse_sageattn_from_prequantized(pre, keep, key_lengths=key_lengths,
                                                             return_lse=True)
    args = (pre.query_int8, pre.query_scale, pre.key_int8, pre.key_scale)
    ref = reference(*args, v, choose(*args, keep, layout, lens), layout, lens)
    check(out, lse, ref, torch.bfloat16, keep * 64, layout)


def shifted(n, L, dtype, layout, seed, D=128):
    """Keys whose channels have means far from zero, as smoothing is for."""
    k = value(2, n, L, torch.float32, layout, seed, D)
    g = torch.Generator().manual_seed(seed + 100)
    return (k + 3.0 * torch.randn(D, generator=g).cuda()).to(dtype)


def token_mean(k, layout):
    return to_hnd(k, layout).double().mean(dim=2).float().to(k.dtype)


def mean_scores(pre, mean, layout, sm_scale):
    """sm_scale q . mean and its bound in fp32: 128 products summed."""
    q = dequant(pre.query_int8, pre.query_scale, 16, layout)
    mean = torch.nn.functional.pad(mean, (0, 128 - mean.size(-1))).double()
    mean = mean.repeat_interleave(q.size(1) // mean.size(1), dim=1)[:, :, None]
    return (q * mean).sum(dim=3) * sm_scale, (q * mean).abs().sum(dim=3) * abs(sm_scale) * 132 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout,D,Lq,keep", [("HND", 128, 300, 5), ("NHD", 128, 1, 12),
                                              ("NHD", 96, 130, 1000), ("HND", 64, 1100, 2)])
def test_lse_of_smoothed_keys(dtype, layout, D, Lq, keep):
    """The lse counts the mean that smoothing took off K, row by row; of a row that
    sees no key it stays -inf.  The output and its lists do not change."""
    q = value(2, 4, Lq, dtype, layout, 1, D)
    k, v = shifted(2, 900, dtype, layout, 2, D), value(2, 2, 900, dtype, layout, 3, D)
    lens = [900, 0]
    key_lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kw = dict(key_lengths=key_lengths, return_lse=True)
    out, lse = turing_sage.sparse_sageattn(q, k, v, keep, tensor_layout=layout, smooth_k=True,
                                           **kw)
    pre = turing_sage.prequantize_sageattn(q, k, v, tensor_layout=layout, smooth_k=True)
    lists = turing_sage.select_key_blocks(pre.query_int8, pre.query_scale, pre.key_int8,
                                          pre.key_scale, keep, tensor_layout=layout,
                                          key_lengths=key_lengths)
    codes_ = (pre.query_int8, pre.query_scale, pre.key_int8, pre.key_scale, pre.value)
    o, A, want = reference(*codes_, lists, layout, lens, sm_scale=D ** -0.5)
    check(out, None, (o[..., :D], A[..., :D], want), dtype, 900, layout)
    shift, slack = mean_scores(pre, token_mean(k, layout), layout, D ** -0.5)
    assert (lse[1] == -math.inf).all()
    err = (lse.double() - want - shift).abs()[0]
    lim = (5.3e-4 + 2.0 ** -22 * want.abs() + 2.0 ** -23 * (want + shift).abs() + slack)[0]
    assert shift.abs().max() > 1 and (err <= lim).all(), (err - lim).max().item()
    # The same in parts, and without smoothing as before.
    again = turing_sage.sparse_sageattn_from_prequantized(pre, keep, **kw)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    parts = turing_sage.sparse_sageattn_prequantized(
        *codes_, lists, tensor_layout=layout, sm_scale=D ** -0.5, key_mean=pre.key_mean, **kw)
    assert torch.equal(parts[1], lse)
    plain = turing_sage.sparse_sageattn_prequantized(*codes_, lists, tensor_layout=layout,
                                                     sm_scale=D ** -0.5, **kw)
    assert torch.equal(parts[0], plain[0])
    assert ((plain[1].double() - want).abs()[0] <= 5.3e-4 + 2.0 ** -22 * want.abs()[0]).all()
    assert turing_sage.prequantize_sageattn(q, k, v, tensor_layout=layout).key_mean is None


@gpu
def test_smoothed_halves_join_by_their_lse():
    """Two halves of the keys, each smoothed by its own mean, joined by their lse:
    the attention over all keys.  Joining weights two outputs by e^lse: an lse off by
    e moves their share by at most 2 e, so the output by 2 e (|o1| + |o2|)."""
    q = value(2, 2, 200, torch.bfloat16, "HND", 1)
    parts, scores, values, outs, slacks = [], [], [], [], []
    for seed in (2, 3):
        k, v = shifted(2, 320, torch.bfloat16, "HND", seed), value(2, 2, 320, torch.bfloat16,
                                                                   "HND", seed + 5)
        outs.append(turing_sage.sparse_sageattn(q, k, v, 5, smooth_k=True, return_lse=True))
        pre = turing_sage.prequantize_sageattn(q, k, v, smooth_k=True)
        shift, slack = mean_scores(pre, token_mean(k, "HND"), "HND", 128 ** -0.5)
        s = dequant(pre.query_int8, pre.query_scale, 16, "HND") @ dequant(
            pre.key_int8, pre.key_scale, 64, "HND").transpose(2, 3) * 128 ** -0.5
        scores.append(s + shift[..., None])
        values.append(v.double())
        slacks.append(slack)
    w = torch.cat(scores, dim=3).softmax(dim=3)
    want, A = w @ torch.cat(values, dim=2), w @ torch.cat(values, dim=2).abs()
    lses = torch.stack([x[1].double() for x in outs])
    share = lses.softmax(dim=0)[..., None]
    got = sum(share[i] * outs[i][0].double() for i in range(2))
    e = 5.3e-4 + 2.0 ** -21 * lses.abs().max() + torch.stack(slacks).amax(dim=0)
    size = outs[0][0].double().abs() + outs[1][0].double().abs()
    bound = (2.0 ** -8 + 5.3e-4) * A + 2.0 ** -8 * size + 2 * e[..., None] * size
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max().item()


@gpu
@pytest.mark.parametrize("Lq", [1, 300])
def test_graphs_streams_and_compile(Lq):
    """Two captured calls (each with workspaces of its own) replayed on two streams
    with new inputs, an eager call between them, and the torch.compile leaf."""
    q, k, v = value(1, 4, Lq, torch.bfloat16, "HND", 1), *(
        value(1, 2, 2000, torch.bfloat16, "HND", s) for s in (2, 3))
    news = [[t.clone().normal_(generator=torch.Generator(device="cuda").manual_seed(n))
             for t in (q, k, v)] for n in (1, 2)]
    want = [turing_sage.sparse_sageattn(*n, 12) for n in news]
    graphs, outs, ins = [], [], []
    for _ in range(2):
        ins.append([t.clone() for t in (q, k, v)])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(turing_sage.sparse_sageattn(*ins[-1], 12))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n, (g, i, s) in enumerate(zip(graphs, ins, streams)):
        for a, b in zip(i, news[n]):
            a.copy_(b)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    eager = turing_sage.sparse_sageattn(*news[0], 12)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert torch.equal(eager, want[0])
    f = torch.compile(lambda a, b, c: turing_sage.sparse_sageattn_compiled(a, b, c, 12) * 1,
                      backend="eager", fullgraph=True)
    assert torch.equal(f(*news[0]), want[0])


@gpu
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_keys_shared_by_expansion(layout):
    """K and V of one batch entry and one head seen by all of them (strides of zero)
    give what their copies give."""
    q8, qs = codes(2, 4, 200, 128, 16, layout, 1)
    k8, ks = codes(1, 1, 900, 128, 64, layout, 2)
    v = value(1, 1, 900, torch.bfloat16, layout, 3)
    ks = ks.expand(2, 4, -1)
    shape = (2, 4, 900, 128) if layout == "HND" else (2, 900, 4, 128)
    k8, v = k8.expand(shape), v.expand(shape)
    lists = turing_sage.select_key_blocks(q8, qs, k8, ks, 5, tensor_layout=layout)
    assert torch.equal(lists, turing_sage.select_key_blocks(q8, qs, k8.contiguous(), ks, 5,
                                                            tensor_layout=layout))
    got, want = (turing_sage.sparse_sageattn_prequantized(q8, qs, a, ks, b, lists,
                                                          tensor_layout=layout)
                 for a, b in ((k8, v), (k8.contiguous(), v.contiguous())))
    assert torch.equal(got, want)


@gpu
def test_compiled_leaf_keeps_every_scale():
    q, k, v = (value(1, 2, n, torch.bfloat16, "HND", s) for n, s in ((130, 1), (700, 2), (700, 3)))
    for scale in (None, 0.0, 0.3):
        assert torch.equal(turing_sage.sparse_sageattn_compiled(q, k, v, 4, sm_scale=scale),
                           turing_sage.sparse_sageattn(q, k, v, 4, sm_scale=scale))
    with pytest.raises(ValueError, match="negative"):
        turing_sage.sparse_sageattn_compiled(q, k, v, 4, sm_scale=-0.3)


# --------------------------------------------------------------------- CPU --

class FakeCuda(torch.Tensor):
    """A CPU tensor that claims to be a CUDA tensor: the binding's checks see it;
    nothing is launched because every call below is refused."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.int8):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeCuda)


def good():
    return dict(q_int8=fake(2, 4, 130, 128), q_scale=fake(2, 4, 12, dtype=torch.float32),
                k_int8=fake(2, 2, 200, 128), k_scale=fake(2, 2, 4, dtype=torch.float32))


SHARED = [
    (dict(q_int8=fake(2, 4, 130, 128, dtype=torch.uint8)), "int8"),
    (dict(k_int8=fake(1, 2, 200, 128)), "incompatible"), (dict(k_int8=fake(2, 3, 200, 128)), "divisible"),
    (dict(k_int8=fake(2, 2, 0, 128)), "empty"), (dict(q_int8=fake(2, 0, 130, 128)), "empty"),
    (dict(q_scale=fake(2, 4, 9, dtype=torch.float32)), "query_scale shape"),
    (dict(k_scale=fake(2, 2, 5, dtype=torch.float32)), "key_scale shape"),
    (dict(q_scale=fake(2, 4, 12, dtype=torch.float64)), "float32"),
    (dict(key_lengths=fake(2, dtype=torch.int64)), "key_lengths"),
    (dict(key_lengths=fake(3, dtype=torch.int32)), "key_lengths")]


@pytest.mark.parametrize("change,match", SHARED + [
    (dict(keep=0), "keep"), (dict(keep=-3), "keep"),
    (dict(q_int8=fake(2, 4, 130, 96), k_int8=fake(2, 2, 200, 96)), "head_dim 64 or 128"),
    (dict(block_policy=fake(3, 4)), "block_policy"), (dict(block_policy=fake(2, 3)), "block_policy"),
    (dict(block_policy=fake(2, 4, dtype=torch.bool)), "block_policy")])
def test_choice_refusals(change, match):
    with pytest.raises(RuntimeError, match=match):
        turing_sage.select_key_blocks(**{**good(), "keep": 2, **change})


@pytest.mark.parametrize("change,match", SHARED + [
    (dict(q_int8=fake(2, 4, 130, 64), k_int8=fake(2, 2, 200, 64)), "head_dim 128"),
    (dict(v=fake(2, 2, 199, 128, dtype=torch.float16)), "value must be"),
    (dict(v=fake(2, 2, 200, 128, dtype=torch.float32)), "value must be"),
    (dict(block_index=fake(2, 4, 2, 3, dtype=torch.int64)), "block_index"),
    (dict(block_index=fake(2, 4, 3, 3, dtype=torch.int32)), "block_index"),
    (dict(block_index=fake(2, 2, 2, 3, dtype=torch.int32)), "block_index"),
    (dict(block_index=fake(2, 4, 2, 0, dtype=torch.int32)), "block_index"),
    (dict(output=fake(2, 4, 130, 128, dtype=torch.bfloat16)), "output must match"),
    (dict(output=fake(2, 4, 131, 128, dtype=torch.float16)), "output must match")])
def test_attention_refusals(change, match):
    args = {**good(), "v": fake(2, 2, 200, 128, dtype=torch.float16),
            "block_index": fake(2, 4, 2, 3, dtype=torch.int32), **change}
    with pytest.raises(RuntimeError, match=match):
        turing_sage.sparse_sageattn_prequantized(**args)


def test_other_refusals():
    with pytest.raises(ValueError, match="tensor_layout"):
        turing_sage.select_key_blocks(**good(), keep=1, tensor_layout="BHLD")
    with pytest.raises(ValueError, match="sm_scale"):
        turing_sage.sparse_sageattn_prequantized(
            **good(), v=fake(2, 2, 200, 128, dtype=torch.float16),
            block_index=fake(2, 4, 2, 3, dtype=torch.int32), sm_scale=float("inf"))
    cpu = torch.zeros((1, 1, 8, 128), dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        turing_sage.select_key_blocks(cpu, torch.ones((1, 1, 4)), cpu, torch.ones((1, 1, 1)), 1)
    x = torch.zeros((1, 1, 8, 128), dtype=torch.float16)
    with pytest.raises(ValueError, match="cuda device"):
        turing_sage.sparse_sageattn(x, x, x, 1)
    from comfyui_turing_utils_kernel.turing_sage.core import PrequantizedSageAttention

    causal = PrequantizedSageAttention(cpu, torch.ones((1, 1, 4)), cpu, torch.ones((1, 1, 1)), x,
                                       "HND", 128, True, 1.0)
    with pytest.raises(ValueError, match="causal"):
        turing_sage.sparse_sageattn_from_prequantized(causal, 1)
    turned = PrequantizedSageAttention(cpu, torch.ones((1, 1, 4)), cpu, torch.ones((1, 1, 1)), x,
                                       "HND", 128, False, -1.0)
    with pytest.raises(ValueError, match="negative"):
        turing_sage.sparse_sageattn_from_prequantized(turned, 1)
    with pytest.raises(RuntimeError, match="a place for every element"):
        turing_sage.sparse_sageattn_prequantized(
            **good(), v=fake(2, 2, 200, 128, dtype=torch.float16),
            block_index=fake(2, 4, 2, 3, dtype=torch.int32),
            output=fake(1, 4, 130, 128, dtype=torch.float16).expand(2, 4, 130, 128))


def test_fake_contract():
    q = torch.empty((2, 4, 9, 96), dtype=torch.bfloat16, device="meta")
    k = torch.empty((2, 2, 9, 96), dtype=torch.bfloat16, device="meta")
    out = turing_sage.sparse_sageattn_compiled(q, k, k, 3)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    assert _sage_sparse.QUERY_BLOCK == 128 and _sage_sparse.KEY_BLOCK == 64


def test_c_entry_refusals():
    lib, p, odd = _lib.load(), ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    size = ctypes.c_int64(0)

    def select(q=p, policy=None, rows=0, ws=p, bytes_=1 << 30, B=1, Hq=2, Hk=1, Lq=128, Lk=128,
               D=128, keep=1, strides=(0,) * 6):
        return lib.tb_select_key_blocks(q, p, p, p, None, policy, rows, p, ws, bytes_, B, Hq, Hk, Lq,
                                        Lk, D, keep, (ctypes.c_int64 * 6)(*strides), None)

    for kw, text in ((dict(q=None), "CUDA tensors"), (dict(q=odd), "16-byte"), (dict(D=96), "head_dim"),
                     (dict(Lk=0), "empty"), (dict(Hq=3, Hk=2), "divisible"), (dict(keep=3), "keep"),
                     (dict(keep=0), "keep"), (dict(policy=p, rows=2), "block_policy"),
                     (dict(bytes_=100), "workspace"), (dict(Lk=1572865), "1572864"),
                     (dict(strides=(8,) * 6), "multiples of 16"), (dict(B=1 << 20, Hq=1 << 20), "grid")):
        assert select(**kw) == _lib.TB_ERR_INVALID, kw
        assert text in _lib.last_error(), (kw, _lib.last_error())
    assert lib.tb_select_key_blocks_workspace(1, 2, 1, 129, 65, 128, ctypes.byref(size)) == 0
    assert size.value > 0

    def attend(q=p, v_dtype=0, B=1, Hq=2, Hk=1, Lq=128, Lk=128, D=128, keep=1, sm=1.0,
               strides=(0,) * 12):
        return lib.tb_sparse_attn(q, p, p, v_dtype, p, p, p, p, None, None, None, 0, B, Hq, Hk, Lq,
                                  Lk, D, keep, (ctypes.c_int64 * 12)(*strides), sm, None)

    for kw, text in ((dict(q=None), "CUDA tensors"), (dict(q=odd), "16-byte"), (dict(D=64), "head_dim"),
                     (dict(v_dtype=2), "float16 or bfloat16"), (dict(Lq=0), "empty"),
                     (dict(Lk=0), "empty"), (dict(Hq=3, Hk=2), "divisible"), (dict(keep=0), "block_index"),
                     (dict(sm=float("nan")), "sm_scale"), (dict(B=1 << 20, Hq=1 << 20), "grid"),
                     (dict(strides=(8,) * 12), "multiples of 16"), (dict(strides=(0,) * 6 + (4,) * 6), "V/O")):
        assert attend(**kw) == _lib.TB_ERR_INVALID, kw
        assert text in _lib.last_error(), (kw, _lib.last_error())


@pytest.mark.parametrize("mean", [fake(2, 4, 128, dtype=torch.float16),
                                  fake(2, 2, 64, dtype=torch.float16),
                                  fake(2, 2, 128, dtype=torch.float32),
                                  torch.zeros((2, 2, 128), dtype=torch.float16)])
def test_key_mean_refusals(mean):
    with pytest.raises(RuntimeError, match="key_mean"):
        turing_sage.sparse_sageattn_prequantized(
            **good(), v=fake(2, 2, 200, 128, dtype=torch.float16),
            block_index=fake(2, 4, 2, 3, dtype=torch.int32), key_mean=mean)


def test_lse_of_anchored_keys_is_refused():
    """stabilize_k takes a row off K that the codes do not keep."""
    from comfyui_turing_utils_kernel.turing_sage.core import (PrequantizedQK,
                                                              prequantize_sageattn_from_qk)

    cpu, x = torch.zeros((1, 1, 8, 128), dtype=torch.int8), torch.zeros((1, 1, 8, 128)).half()
    qk = PrequantizedQK(cpu, torch.ones((1, 1, 4)), cpu, torch.ones((1, 1, 1)), "HND", x.dtype,
                        128, True, True)
    with pytest.raises(ValueError, match="stabilize_k"):
        turing_sage.sparse_sageattn_from_prequantized(prequantize_sageattn_from_qk(qk, x), 1,
                                                      return_lse=True)


def test_smoothed_lse_entry_refusals():
    lib, p, odd = _lib.load(), ctypes.c_void_p(4096), ctypes.c_void_p(4100)

    def add(q=p, mean=p, dtype=0, B=1, Hq=2, Hk=1, Lq=128, D=128, sm=1.0, stride=0):
        return lib.tb_smoothed_lse(q, p, mean, dtype, p, B, Hq, Hk, Lq, D,
                                   (ctypes.c_int64 * 3)(*((stride,) * 3)), sm, None)

    for kw, text in ((dict(q=None), "CUDA tensors"), (dict(mean=None), "CUDA tensors"),
                     (dict(q=odd), "16-byte"), (dict(mean=odd), "16-byte"), (dict(D=64), "head_dim"),
                     (dict(dtype=2), "float16 or bfloat16"), (dict(Lq=0), "empty"),
                     (dict(Hk=0), "divisible"), (dict(Hq=3, Hk=2), "divisible"),
                     (dict(sm=float("inf")), "sm_scale"), (dict(stride=8), "multiples of 16"),
                     (dict(B=1 << 20, Hq=1 << 20), "grid")):
        assert add(**kw) == _lib.TB_ERR_INVALID, kw
        assert text in _lib.last_error(), (kw, _lib.last_error())
