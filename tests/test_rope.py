"""Rotary positions: the fp64 formula, gradients, refusals, frequencies.

Bound of one output y = s (x0 cos - x1 sin) in fp32 against fp64: the reduced
angle, quarter turns in [-1/2, 1/2], is rounded once (2^-26 pi / 2 = 0.23e-7), the
polynomials of its sine and cosine are good to 1 ulp of values up to 1 (0.6e-7; 2
are allowed for), the scale, the product and the sum round once each (3 x 0.6e-7):
3.3e-7 s (|x0| + |x1|), 4e-7 allowed; then half a step of the output type.
"""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from comfyui_turing_utils_kernel import _C, _lib

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def angles(positions, inv_freq, axis_pairs):
    p = positions.double().cpu()
    if axis_pairs is None:
        p = p.unsqueeze(-1)
    if p.dim() == 2:
        p = p.unsqueeze(0)
    cols = [p[..., a:a + 1].expand(*p.shape[:-1], n) for a, n in
            enumerate(axis_pairs or [inv_freq.numel()])]
    return torch.cat(cols, dim=-1) * inv_freq.double().cpu()


def formula(x, positions, inv_freq, layout, split_half, axis_pairs, scale, sign=1.0):
    """(y, the bound's s (|x0| + |x1|)) in fp64, channel pair by channel pair."""
    ang = angles(positions, inv_freq, axis_pairs)
    ang = ang.unsqueeze(1 if layout == "HND" else 2) * sign
    x = x.detach().double().cpu()
    y, size = x.clone(), torch.zeros_like(x)
    n = inv_freq.numel()
    for i in range(n):
        a, b = (i, i + n) if split_half else (2 * i, 2 * i + 1)
        c, s = ang[..., i].cos() * scale, ang[..., i].sin() * scale
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = abs(scale) * (x[..., a].abs() + x[..., b].abs())
    return y, size


def check(got, x, *args, **kw):
    want, size = formula(x, *args, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    bound = 4e-7 * size + want.abs() * HALF_STEP[x.dtype] + 2.0 ** -25
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= bound).all(), ((err - bound).max().item(), err.max().item())
    n = 2 * args[1].numel()
    assert torch.equal(got[..., n:].detach().cpu(), x[..., n:].detach().cpu())  # copied channels


def rand(shape, layout, dtype, seed):
    B, H, L, D = shape
    g = torch.Generator().manual_seed(seed)
    return torch.randn((B, H, L, D) if layout == "HND" else (B, L, H, D),
                       generator=g).to(dtype).cuda()


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("split_half", [False, True])
@pytest.mark.parametrize("B,Hq,Hk,L,D,rot", [
    (1, 1, 1, 1, 8, 2), (1, 40, 40, 1, 128, 128), (2, 6, 2, 37, 96, 48), (3, 5, 1, 130, 64, 64),
    (1, 3, 3, 17, 128, 32), (2, 2, 1, 9, 70, 34), (1, 2, 2, 5, 600, 520), (1, 70, 1, 3, 16, 16)])
def test_matches_the_formula(dtype, layout, split_half, B, Hq, Hk, L, D, rot):
    q, k = (rand((B, h, L, D), layout, dtype, 5 + i) for i, h in enumerate((Hq, Hk)))
    inv, scale = kernel.turing_rope_inv_freq(rot, device="cuda")
    pos = torch.arange(L, device="cuda") + 11
    yq, yk = kernel.turing_rope_qk(q, k, pos, inv, tensor_layout=layout, split_half=split_half)
    for x, y in ((q, yq), (k, yk)):
        check(y, x, pos, inv, layout, split_half, None, scale)
    assert torch.equal(kernel.turing_rope(q, pos, inv, tensor_layout=layout,
                                          split_half=split_half), yq)


@gpu
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("axis_pairs", [[16, 24, 24], [64, 0], [1, 2, 3, 58]])
@pytest.mark.parametrize("rows", [0, 1, 2])
def test_axes_position_types_and_rows(ptype, axis_pairs, rows):
    """One row of positions (with and without a batch dimension) or one per batch
    entry, far from zero, negative, and fractional where the type allows."""
    B, H, L = 2, 3, 21
    g = torch.Generator().manual_seed(2)
    shape = ((rows,) if rows else ()) + (L, len(axis_pairs))
    pos = torch.randint(-50, 900000, shape, generator=g)
    pos = (pos.double() + (0.375 if ptype.is_floating_point else 0)).to(ptype).cuda()
    inv, _ = kernel.turing_rope_inv_freq(128, axis_pairs=axis_pairs, device="cuda")
    x = rand((B, H, L, 128), "HND", torch.float32, 3)
    y = kernel.turing_rope(x, pos, inv, axis_pairs=axis_pairs, scale=-1.25)
    check(y, x, pos, inv, "HND", False, axis_pairs, -1.25)


@gpu
@pytest.mark.parametrize("split_half", [False, True])
def test_strides_and_alignment(split_half):
    """Views of a fused QKV row, an odd offset, a head dimension of stride 2 and
    size-one dimensions of any stride give what contiguous copies give."""
    inv, _ = kernel.turing_rope_inv_freq(64, device="cuda")
    g = torch.Generator().manual_seed(1)
    pos = torch.arange(29, device="cuda")
    qkv = torch.randn((2, 29, 3 * 4 * 64), generator=g).to(torch.bfloat16).cuda()
    q, k, _ = qkv.view(2, 29, 3, 4, 64).unbind(2)
    odd = torch.randn(2 * 29 * 4 * 64 + 1, generator=g).to(torch.bfloat16).cuda()[1:].view(
        2, 29, 4, 64)
    wide = torch.randn((2, 29, 4, 128), generator=g).to(torch.bfloat16).cuda()[..., ::2]
    one = torch.randn((2, 29, 4, 64), generator=g).to(torch.bfloat16).cuda().as_strided(
        (1, 29, 1, 64), (7, 256, 13, 1))
    for a, b in ((q, k), (odd, k), (q, wide), (one, one)):
        got = kernel.turing_rope_qk(a, b, pos, inv, tensor_layout="NHD", split_half=split_half)
        want = kernel.turing_rope_qk(a.clone(memory_format=torch.contiguous_format),
                                     b.clone(memory_format=torch.contiguous_format), pos, inv,
                                     tensor_layout="NHD", split_half=split_half)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        check(got[1], b, pos, inv, "NHD", split_half, None, 1.0)


@gpu
def test_empty_and_special_values():
    inv, _ = kernel.turing_rope_inv_freq(64, device="cuda")
    for shape in ((2, 3, 0, 64), (0, 3, 5, 64)):
        x = torch.empty(shape, device="cuda")
        pos = torch.zeros(shape[2], device="cuda")
        assert kernel.turing_rope(x, pos, inv).shape == shape
    # No key heads: the query still turns.
    q, pos = rand((1, 2, 5, 64), "HND", torch.float32, 0), torch.arange(5, device="cuda")
    yq, yk = kernel.turing_rope_qk(q, q[:, :0], pos, inv)
    assert yk.shape == (1, 0, 5, 64)
    check(yq, q, pos, inv, "HND", False, None, 1.0)
    # A NaN stays in its pair; an infinity at angle zero stays in its channel's pair.
    q[0, 0, 3, 6] = float("nan")
    y = kernel.turing_rope(q, pos, inv)
    bad = y.isnan()
    assert bad[0, 0, 3, 6] and bad[0, 0, 3, 7] and bad.sum() == 2


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("split_half", [False, True])
def test_gradients(dtype, split_half):
    """Against the formula's transpose; of one input alone; of an expanded gradient."""
    inv, scale = kernel.turing_rope_inv_freq(32, scaling="yarn", factor=4.0, original_length=64,
                                             device="cuda")
    pos = torch.arange(19, device="cuda") * 3
    q = rand((2, 4, 19, 48), "NHD", dtype, 1).requires_grad_()
    k = rand((2, 2, 19, 48), "NHD", dtype, 2).requires_grad_()
    gq, gk = rand((2, 4, 19, 48), "NHD", dtype, 3), rand((2, 2, 19, 48), "NHD", dtype, 4)
    opts = dict(tensor_layout="NHD", split_half=split_half, scale=scale)
    yq, yk = kernel.turing_rope_qk(q, k, pos, inv, **opts)
    dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
    for d, g in ((dq, gq), (dk, gk)):
        check(d, g, pos, inv, "NHD", split_half, None, scale, sign=-1.0)
    only, = torch.autograd.grad(kernel.turing_rope_qk(q, k.detach(), pos, inv, **opts)[0], q, gq)
    assert torch.equal(only, dq)
    one, = torch.autograd.grad(kernel.turing_rope(k, pos, inv, **opts), k, gk)
    assert torch.equal(one, dk)
    # Only one output reaches the loss, by way of a sum (an expanded gradient).
    yq, yk = kernel.turing_rope_qk(q, k, pos, inv, **opts)
    d, = torch.autograd.grad(yk.sum(), k)
    check(d, torch.ones_like(k), pos, inv, "NHD", split_half, None, scale, sign=-1.0)


@gpu
def test_gradient_against_differences():
    """The directional derivative of a weighted sum of outputs by a central
    difference of the kernel: linear in x, so exact up to rounding (each output
    is off by at most 4e-7 (|x0| + |x1|); 2 x 144 terms of weight |w| <= 5)."""
    inv, _ = kernel.turing_rope_inv_freq(16, device="cuda")
    pos = torch.arange(9, device="cuda") + 5
    x = rand((1, 1, 9, 16), "HND", torch.float32, 1).requires_grad_()
    w, d = (rand((1, 1, 9, 16), "HND", torch.float32, s) for s in (2, 3))
    grad, = torch.autograd.grad(kernel.turing_rope(x, pos, inv, split_half=True), x, w)
    with torch.no_grad():
        f = [(kernel.turing_rope(x + e * d, pos, inv, split_half=True).double() * w).sum()
             for e in (0.5, -0.5)]
    assert abs((f[0] - f[1]) - (grad.double() * d).sum()).item() <= 2 * 144 * 5 * 4e-7 * 10


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,rot,axis_pairs", [(1, 2, None), (7, 6, None), (300, 128, [22, 21, 21]),
                                              (33, 600, [300])])
@pytest.mark.parametrize("batch", [0, 3])
def test_freqs_match_the_formula(dtype, L, rot, axis_pairs, batch):
    g = torch.Generator().manual_seed(4)
    shape = ((batch,) if batch else ()) + (L,) + (() if axis_pairs is None else (len(axis_pairs),))
    pos = torch.randint(0, 100000, shape, generator=g).cuda()
    inv, _ = kernel.turing_rope_inv_freq(rot, axis_pairs=axis_pairs, device="cuda")
    got = kernel.turing_rope_freqs(pos, inv, axis_pairs=axis_pairs, scale=1.5, dtype=dtype)
    ang = angles(pos, inv, axis_pairs)
    c, s = ang.cos() * 1.5, ang.sin() * 1.5
    want = torch.stack([c, -s, s, c], dim=-1).view(max(batch, 1), L, 1, rot // 2, 2, 2)
    assert got.shape == want.shape and got.dtype == dtype
    err = (got.double().cpu() - want).abs()
    assert (err <= 4e-7 * 1.5 + want.abs() * HALF_STEP[dtype]).all(), err.max().item()


@gpu
def test_freqs_feed_the_fused_prologue():
    """turing_rope_freqs -> prequantize_rms_rope_qk gives the codes of the same
    matrices made by torch."""
    from comfyui_turing_utils_kernel import turing_sage

    axis_pairs = [22, 21, 21]
    inv, _ = kernel.turing_rope_inv_freq(128, axis_pairs=axis_pairs, device="cuda")
    t = torch.arange(150, device="cuda")
    pos = torch.stack([t // 50, (t // 10) % 5, t % 10], dim=-1)
    freqs = kernel.turing_rope_freqs(pos, inv, axis_pairs=axis_pairs)
    ang = angles(pos, inv, axis_pairs).cuda()
    want = torch.stack([ang.cos(), -ang.sin(), ang.sin(), ang.cos()], dim=-1).view(
        1, 150, 1, 64, 2, 2).to(torch.bfloat16)
    # Equal but where a value lies within fp32's error of a rounding border.
    assert (freqs != want).float().mean().item() < 1e-3
    q, k = (rand((1, 4, 150, 128), "HND", torch.bfloat16, s) for s in (1, 2))
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    a, b = (turing_sage.prequantize_rms_rope_qk(q, k, w, w, f, epsilon=1e-6, rot_dim=128)
            for f in (freqs, want))
    # A matrix entry one bf16 step off moves a code by at most 2 (127 x 2^-8 x 2 < 1, and rounding).
    assert (a.query_int8.int() - b.query_int8.int()).abs().max() <= 2
    assert (a.key_int8 != b.key_int8).float().mean() < 1e-2


@gpu
def test_streams_graphs_and_compile():
    inv, _ = kernel.turing_rope_inv_freq(64, device="cuda")
    pos = torch.arange(65, device="cuda")
    x = rand((1, 4, 65, 64), "HND", torch.bfloat16, 1)
    want = kernel.turing_rope(x, pos, inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernel.turing_rope(x, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernel.turing_rope(x, pos, inv)
    new = rand((1, 4, 65, 64), "HND", torch.bfloat16, 9)
    x.copy_(new)
    graph.replay()
    assert torch.equal(out, kernel.turing_rope(new, pos, inv))
    f = torch.compile(lambda t: kernel.turing_rope(t, pos, inv) * 2, backend="eager",
                      fullgraph=True)
    assert torch.equal(f(new), kernel.turing_rope(new, pos, inv) * 2)


@gpu
def test_captured_gradients_beside_an_eager_graph():
    """Forward and gradients captured and replayed on new values while an eager
    graph of the same memory lives; that one still gives its own gradients.  (The
    captured leaves are objects of their own: torch refuses to capture a backward
    pass into leaves that a live eager graph holds, whatever the operator.)"""
    inv, _ = kernel.turing_rope_inv_freq(64, device="cuda")
    pos = torch.arange(65, device="cuda")
    q = rand((1, 4, 65, 64), "HND", torch.float32, 1).requires_grad_()
    k = rand((1, 2, 65, 64), "HND", torch.float32, 2).requires_grad_()
    gq, gk = rand((1, 4, 65, 64), "HND", torch.float32, 3), rand((1, 2, 65, 64), "HND",
                                                                 torch.float32, 4)
    eager = kernel.turing_rope_qk(q, k, pos, inv)
    want = torch.autograd.grad(eager, (q, k), (gq, gk), retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    q2, k2 = q.detach().requires_grad_(), k.detach().requires_grad_()
    with torch.cuda.graph(graph):
        out = kernel.turing_rope_qk(q2, k2, pos, inv)
        grads = torch.autograd.grad(out, (q2, k2), (gq, gk))
    new = [rand(tuple(t.shape), "HND", torch.float32, 7 + i) for i, t in enumerate((gq, gk))]
    old = [gq.clone(), gk.clone()]
    gq.copy_(new[0])
    gk.copy_(new[1])
    graph.replay()
    again = torch.autograd.grad(eager, (q, k), tuple(old))
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    expect = torch.autograd.grad(kernel.turing_rope_qk(q, k, pos, inv), (q, k), tuple(new))
    assert torch.equal(grads[0], expect[0]) and torch.equal(grads[1], expect[1])


@gpu
@pytest.mark.parametrize("split_half", [0, 1])
def test_c_entry_in_place(split_half):
    """An output may be its input."""
    inv, _ = kernel.turing_rope_inv_freq(48, device="cuda")
    pos = torch.arange(33, device="cuda")
    for odd in (0, 1):
        x = rand((1, 3, 33, 64), "HND", torch.bfloat16, 1)
        room = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        y = room[odd:odd + x.numel()].view_as(x).copy_(x)
        want = kernel.turing_rope(x, pos, inv, split_half=bool(split_half))
        s = (ctypes.c_int64 * 12)(*((6336, 2112, 64, 0, 0, 0) * 2))
        _lib.call("tb_rope", y.data_ptr(), None, y.data_ptr(), None, pos.data_ptr(), 1, 1,
                  inv.data_ptr(), None, 1, 1, 3, 0, 33, 64, 48, s, split_half, 0,
                  _lib.TB_DTYPE_BF16, 1.0, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(y, want)


def transforms(x, pos, inv):
    """What torch's function transforms, forward-mode differentiation and the tracer
    give for a rotation, against the rotation itself (linear: its tangent is the
    rotated tangent, its gradient the inverse rotation)."""
    import torch.autograd.forward_ad as fwd

    rope = lambda t: kernel.turing_rope(t, pos, inv, split_half=True)  # noqa: E731
    both = lambda t: kernel.turing_rope_qk(t, 2 * t, pos, inv)         # noqa: E731
    y = rope(x)
    many = torch.stack([x, x + 1, -x])
    assert torch.equal(torch.vmap(rope)(many), torch.stack([rope(t) for t in many]))
    assert torch.equal(torch.vmap(both)(many)[1], torch.stack([both(t)[1] for t in many]))
    shifts = torch.stack([pos, pos + 3, pos * 2])
    assert torch.equal(torch.vmap(lambda t, p: kernel.turing_rope(t, p, inv))(many, shifts),
                       torch.stack([kernel.turing_rope(t, p, inv) for t, p in zip(many, shifts)]))
    loss = lambda t: (rope(t) ** 2).sum() / 2                          # noqa: E731
    back = kernel.turing_rope(y, pos, inv, split_half=True, inverse=True)
    assert torch.equal(torch.func.grad(loss)(x), back)
    assert torch.equal(torch.vmap(torch.func.grad(loss))(many)[0], back)
    grads = torch.func.grad(lambda q, k: sum((t ** 2).sum() / 2 for t in
                                             kernel.turing_rope_qk(q, k, pos, inv)),
                            argnums=(0, 1))(x, x + 1)
    leaves = [t.clone().requires_grad_() for t in (x, x + 1)]
    out = kernel.turing_rope_qk(*leaves, pos, inv)
    want = torch.autograd.grad(out, leaves, [t.detach() for t in out])
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    tangent = (x * 3 + 1).detach()
    assert torch.equal(torch.func.jvp(rope, (x,), (tangent,))[1], rope(tangent))
    with fwd.dual_level():
        primal, t = fwd.unpack_dual(rope(fwd.make_dual(x, tangent)))
        assert torch.equal(primal, y) and torch.equal(t, rope(tangent))
        q, k = kernel.turing_rope_qk(fwd.make_dual(x, tangent), x, pos, inv)
        assert torch.equal(fwd.unpack_dual(q).tangent, kernel.turing_rope(tangent, pos, inv))
        assert torch.equal(kernel.turing_rope(x, pos, inv, split_half=True), y)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.ops.turing_utils.rope(fwd.make_dual(x, tangent), pos, inv)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.ops.turing_utils.rope_qk(x, fwd.make_dual(x, tangent), pos, inv)
    second = torch.func.hessian(loss)(x[:1, :1])
    n = x[:1, :1].numel()
    eye = second.reshape(n, n)      # a rotation of scale 1: the identity
    assert (eye - torch.eye(n, dtype=eye.dtype, device=eye.device)).abs().max() <= 4e-6
    traced = torch.jit.trace(rope, (x,))
    assert torch.equal(traced(many[1]), rope(many[1]))
    traced = torch.jit.trace(lambda p: kernel.turing_rope_freqs(p, inv, dtype=torch.float32), (pos,))
    assert torch.equal(traced(pos + 5), kernel.turing_rope_freqs(pos + 5, inv, dtype=torch.float32))


@gpu
@pytest.mark.filterwarnings("ignore")
def test_function_transforms():
    x = rand((2, 3, 5, 8), "HND", torch.float32, 1)
    inv, _ = kernel.turing_rope_inv_freq(8, device="cuda")
    transforms(x, torch.arange(5, device="cuda"), inv)


@gpu
@pytest.mark.parametrize("op", [False, True])
def test_axis_pairs_changed_after_the_call(op):
    """The gradient turns by the axes of the call, whatever becomes of its list."""
    pos = torch.arange(12, device="cuda").view(6, 2)
    inv, _ = kernel.turing_rope_inv_freq(16, device="cuda")
    x, g = (rand((1, 2, 6, 16), "HND", torch.float32, s) for s in (1, 2))
    x.requires_grad_()
    want, = torch.autograd.grad(kernel.turing_rope(x, pos, inv, axis_pairs=[3, 5]), x, g)
    pairs = [3, 5]
    y = (torch.ops.turing_utils.rope if op else kernel.turing_rope)(x, pos, inv, axis_pairs=pairs)
    pairs[:] = [6, 2]
    got, = torch.autograd.grad(y, x, g)
    assert torch.equal(got, want)


# ---------------------------------------------------------------------- CPU --

def test_fake_contracts():
    q = torch.empty((2, 4, 9, 64), dtype=torch.bfloat16, device="meta")
    k = torch.empty((2, 2, 9, 64), dtype=torch.bfloat16, device="meta")
    pos = torch.empty((9, 3), device="meta")
    inv = torch.empty(32, dtype=torch.float64, device="meta")
    yq, yk = kernel.turing_rope_qk(q, k, pos, inv, axis_pairs=[12, 10, 10])
    assert yq.shape == q.shape and yk.shape == k.shape and yk.dtype == torch.bfloat16
    assert kernel.turing_rope(q.transpose(1, 2), pos, inv).is_contiguous()
    f = kernel.turing_rope_freqs(pos, inv, axis_pairs=[12, 10, 10], dtype=torch.float16)
    assert f.shape == (1, 9, 1, 32, 2, 2) and f.dtype == torch.float16


@pytest.mark.filterwarnings("ignore")
def test_function_transforms_without_a_gpu(monkeypatch):
    """The same through the registered ops, the formula in the kernels' place."""
    from comfyui_turing_utils_kernel import ops

    def plain(query, key, positions, inv_freq, layout, split_half, axis_pairs, scale, inverse):
        sign = -1.0 if inverse else 1.0
        outs = []
        for t in (query, key):
            t = None if t is None else t.contiguous()
            assert t is None or t.data_ptr()      # a tensor with memory of its own
            outs.append(None if t is None else formula(t, positions, inv_freq, layout, split_half,
                                                       axis_pairs, scale, sign)[0].to(t.dtype))
        return tuple(outs)

    def matrices(positions, inv_freq, axis_pairs, scale, dtype):
        assert positions.data_ptr()
        ang = angles(positions, inv_freq, axis_pairs)
        c, s = ang.cos() * scale, ang.sin() * scale
        return torch.stack([c, -s, s, c], dim=-1).view(*ang.shape[:2], 1, -1, 2, 2).to(dtype)

    monkeypatch.setattr(ops._C, "turing_rope", plain)
    monkeypatch.setattr(ops._C, "turing_rope_freqs", matrices)
    monkeypatch.setattr(ops, "_require_cuda", lambda *a: None)
    x = torch.randn((2, 3, 5, 8), generator=torch.Generator().manual_seed(1))
    inv, _ = kernel.turing_rope_inv_freq(8)
    transforms(x, torch.arange(5), inv)


def test_inv_freq():
    inv, scale = kernel.turing_rope_inv_freq(8, 10000.0)
    assert scale == 1.0 and inv.dtype == torch.float64
    torch.testing.assert_close(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, _ = kernel.turing_rope_inv_freq(8, scaling="linear", factor=4.0)
    torch.testing.assert_close(lin, inv / 4)
    ntk, _ = kernel.turing_rope_inv_freq(8, scaling="ntk", factor=4.0)
    torch.testing.assert_close(ntk[0], inv[0])
    torch.testing.assert_close(ntk[-1], inv[-1] / 4)
    yarn, scale = kernel.turing_rope_inv_freq(128, scaling="yarn", factor=8.0,
                                              original_length=4096)
    plain, _ = kernel.turing_rope_inv_freq(128)
    turns = plain * 4096 / (2 * torch.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    torch.testing.assert_close(yarn[turns < 0.8], plain[turns < 0.8] / 8)
    assert abs(scale - (0.1 * torch.tensor(8.0).log().item() + 1)) < 1e-6
    axes, _ = kernel.turing_rope_inv_freq(16, axis_pairs=[4, 0, 1, 3])
    torch.testing.assert_close(axes[:4], inv)
    assert axes[4] == 1.0


@pytest.mark.parametrize("rot,theta,length,factor,beta_fast,beta_slow,axis_pairs", [
    (128, 10000.0, 4096, 8.0, 32.0, 1.0, None), (128, 10000.0, 65536, 4.0, 32.0, 1.0, None),
    (128, 10000.0, 131072, 8.0, 32.0, 1.0, None), (16, 10000.0, 32768, 4.0, 32.0, 1.0, None),
    (64, 500000.0, 8192, 2.5, 16.0, 0.5, None), (128, 10000.0, 65536, 4.0, 32.0, 1.0, [22, 21, 21]),
    (2, 10000.0, 4096, 4.0, 32.0, 1.0, None), (128, 100.0, 1 << 24, 4.0, 32.0, 1.0, None)])
def test_yarn_frequencies(rot, theta, length, factor, beta_fast, beta_slow, axis_pairs):
    """The published ramp, pair by pair: its ends are the pairs (of d = 2 n channels)
    that turn beta_fast and beta_slow times, rounded outwards and kept in 0 .. d - 1.
    Where both lie inside, a pair that turns more than beta_slow times is never
    divided by the whole factor."""
    inv, scale = kernel.turing_rope_inv_freq(rot, theta, axis_pairs=axis_pairs, scaling="yarn",
                                             factor=factor, original_length=length,
                                             beta_fast=beta_fast, beta_slow=beta_slow)
    want = []
    for n in axis_pairs or [rot // 2]:
        d = 2 * n

        def pair(turns):
            return d * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), d - 1)
        for i in range(n):
            f = theta ** (-2 * i / d)
            ramp = min(max((i - low) / (high - low if high > low else 1e-3), 0.0), 1.0)
            want.append(f / factor * ramp + f * (1 - ramp))
            if f * length / (2 * math.pi) > beta_slow * 1.001:
                assert want[-1] > f / factor
    torch.testing.assert_close(inv, torch.tensor(want, dtype=torch.float64), rtol=1e-12, atol=0)
    assert scale == 0.1 * math.log(factor) + 1.0


@pytest.mark.parametrize("kw,match", [
    (dict(rot_dim=7), "even"), (dict(rot_dim=8, theta=1.0), "theta"),
    (dict(rot_dim=8, scaling="other"), "scaling"), (dict(rot_dim=8, factor=0.5), "factor"),
    (dict(rot_dim=8, scaling="yarn", factor=2.0), "original_length"),
    (dict(rot_dim=8, axis_pairs=[1, 2]), "axis_pairs"),
    (dict(rot_dim=8, axis_pairs=[5, -1]), "axis_pairs")])
def test_inv_freq_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        kernel.turing_rope_inv_freq(**kw)


def test_cpu_tensors_are_refused():
    x, pos, inv = torch.zeros((1, 2, 3, 8)), torch.arange(3), torch.ones(4, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        kernel.turing_rope(x, pos, inv)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        kernel.turing_rope_qk(x, x, pos, inv)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        kernel.turing_rope_freqs(pos, inv)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _C.turing_rope(x, None, pos, inv)


class FakeCuda(torch.Tensor):
    """A CPU tensor that claims to be a CUDA tensor: the binding's checks see it;
    nothing is launched because every call below is refused."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeCuda)


@pytest.mark.parametrize("change,match", [
    (dict(query=fake(2, 3, 8)), "4D"),
    (dict(query=fake(1, 2, 3, 8, dtype=torch.int8)), "float16, bfloat16, or float32"),
    (dict(key=fake(1, 2, 3, 8, dtype=torch.float16)), "share"),
    (dict(key=fake(1, 2, 4, 8)), "share"), (dict(key=fake(2, 2, 3, 8)), "share"),
    (dict(key=fake(1, 2, 3, 16)), "share"),
    (dict(tensor_layout="DNH"), "tensor_layout"),
    (dict(positions=fake(4, dtype=torch.int64)), "positions must be"),
    (dict(positions=fake(2, 3, dtype=torch.int64)), "positions must be"),
    (dict(positions=fake(3, dtype=torch.int16)), "positions must be int32"),
    (dict(axis_pairs=[2, 2]), "positions must be"),
    (dict(axis_pairs=[2, 1]), "axis_pairs"), (dict(axis_pairs=[5, -1]), "axis_pairs"),
    (dict(axis_pairs=[]), "1 to 4 axes"), (dict(axis_pairs=[1, 1, 1, 1, 0]), "1 to 4 axes"),
    (dict(inv_freq=fake(5, dtype=torch.float64)), "head dimension"),
    (dict(inv_freq=fake(4, dtype=torch.float16)), "inv_freq"),
    (dict(inv_freq=fake(0, dtype=torch.float64)), "inv_freq"),
    (dict(scale=float("inf")), "scale")])
def test_binding_refusals(change, match):
    args = dict(query=fake(1, 2, 3, 8), key=fake(1, 1, 3, 8),
                positions=fake(3, dtype=torch.int64), inv_freq=fake(4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match=match):
        _C.turing_rope(**{**args, **change})


def test_c_entry_refusals():
    lib, p = _lib.load(), ctypes.c_void_p(4096)   # never dereferenced: the checks fail first
    strides = (ctypes.c_int64 * 12)()

    def rope(q=p, k=None, ko=None, hk=0, ptype=1, rows=1, pairs=None, axes=1, B=1, H=1, L=1, D=8,
             rot=8, dtype=0, scale=1.0):
        return lib.tb_rope(q, k, p, ko, p, ptype, rows, p, pairs, axes, B, H, hk, L, D, rot,
                           strides, 0, 0, dtype, scale, None)

    for kw, text in ((dict(q=None), "CUDA tensors"), (dict(k=p), "together"),
                     (dict(k=p, ko=p, hk=0), "together"), (dict(dtype=7), "float16"),
                     (dict(L=0), "positive"), (dict(rot=7), "rot_dim"), (dict(rot=10), "rot_dim"),
                     (dict(ptype=4), "positions"), (dict(rows=2), "positions"),
                     (dict(axes=5), "axes"), (dict(L=1 << 31), "range"),
                     (dict(pairs=(ctypes.c_int32 * 2)(3, 2), axes=2), "axis_pairs"),
                     (dict(scale=float("nan")), "scale")):
        assert rope(**kw) == _lib.TB_ERR_INVALID, kw
        assert text in _lib.last_error(), (kw, _lib.last_error())
    st = lib.tb_rope_freqs(p, 0, 1, p, None, 1, ctypes.c_void_p(4104), 1, 1, 4, 0, 1.0, None)
    assert st == _lib.TB_ERR_INVALID and "16-byte" in _lib.last_error()
    st = lib.tb_rope_freqs(p, 0, 1, p, None, 1, p, 1, 0, 4, 0, 1.0, None)
    assert st == _lib.TB_ERR_INVALID and "positive" in _lib.last_error()
