"""Rotary positions on the GPU against the rotation computed in 64 bits.

Tolerance: the kernel's fp32 arithmetic is off by at most ten units of 2^-24 of (|a| + |b|) f -- the angle's fraction of a
turn rounded once (at most pi 2^-24 rad), cosine and sine within two units in the last place, two products, the factor and
the sum -- plus the 64-bit product position * w on either side (2^-51 of it, in radians); then one rounding to the type."""
import pytest
import torch

from lrqk_b200 import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def exact(x, positions, inv, factor, interleaved, adjoint):
    y, part = x.double().clone(), 2 * inv.numel()
    pos = positions.double()
    if pos.dim() == 1:
        pos = pos[None]
    t = pos[:, None, :, None] * inv
    c, s = torch.cos(t) * factor, torch.sin(t) * (-factor if adjoint else factor)
    ia = torch.arange(0, part, 2, device=x.device) if interleaved else torch.arange(part // 2, device=x.device)
    ib = ia + 1 if interleaved else ia + part // 2
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(y)
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * factor * (10 * 2.0 ** -24 + t.abs() * 2.0 ** -51)
    return y, size


def check(got, x, positions, inv, factor, interleaved, adjoint):
    want, tol = exact(x, positions, inv, factor, interleaved, adjoint)
    half_step = torch.finfo(x.dtype).eps / 2
    allowed = tol + (want.abs() + tol) * half_step
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    assert bool(((got.double() - want).abs() <= allowed).all()), float(((got.double() - want).abs() / allowed.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("adjoint", [False, True])
@pytest.mark.parametrize("b,hq,hk,n,d,part,start", [
    (1, 32, 8, 1, 128, 128, 131071), (4, 8, 2, 1, 64, 64, 0), (2, 7, 1, 33, 128, 64, 5), (1, 3, 3, 257, 64, 48, 1000000),
    (3, 5, 1, 10, 20, 14, 77), (1, 2, 2, 5, 2, 2, 3), (2, 32, 8, 600, 128, 96, 262143), (1, 1, 1, 3, 1024, 1024, 9)])
def test_against_64_bits(dtype, interleaved, adjoint, b, hq, hk, n, d, part, start):
    g = torch.Generator(device="cuda").manual_seed(n * d + part)
    q = torch.randn(b, n, hq, d, generator=g, device="cuda").to(dtype).transpose(1, 2)     # as a projection leaves it
    k = torch.randn(b, hk, n, d, generator=g, device="cuda").to(dtype)
    pos = start + torch.randint(0, 1000, (b, n), generator=g, device="cuda")
    inv, factor = rotary_frequencies(part, 500000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192},
                                     device="cuda")
    q2, k2 = apply_rotary(q, k, pos, inv, factor=factor, interleaved=interleaved, adjoint=adjoint)
    check(q2, q, pos, inv, factor, interleaved, adjoint)
    check(k2, k, pos, inv, factor, interleaved, adjoint)
    assert torch.equal(q2[..., part:], q[..., part:])


def test_position_forms_agree_and_signs_cancel():
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(2, 4, 9, 64, generator=g, device="cuda")
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(100, 109, device="cuda")
    ref = apply_rotary(q, None, pos, inv)
    for p in (pos.int(), pos[None], pos[None].expand(2, 9), pos.repeat(2, 1), pos.repeat_interleave(2)[::2],
              pos.int().repeat(2, 1)):
        assert torch.equal(apply_rotary(q, None, p, inv), ref)
    assert torch.equal(apply_rotary(q, None, -pos, inv), apply_rotary(q, None, pos, inv, adjoint=True))
    far = torch.tensor([2 ** 31 + 7, -2 ** 31 - 9, 2 ** 33, -1, 0, 1, 2 ** 20, -2 ** 20, 12], device="cuda")
    check(apply_rotary(q, None, far, inv), q, far, inv, 1.0, False, False)
    assert torch.equal(apply_rotary(q, None, torch.zeros_like(pos), inv), q)


def test_views_odd_strides_and_unaligned_rows():
    g = torch.Generator(device="cuda").manual_seed(2)
    inv, _ = rotary_frequencies(32, device="cuda")
    wide = torch.randn(2, 3, 11, 41, generator=g, device="cuda").bfloat16()
    pos = torch.arange(11, device="cuda")
    for q in (wide[..., 1:33], wide[..., :32], wide[..., 3:36], wide[:, :, ::2, 5:39], wide.expand(2, 3, 11, 41)[:1].expand(4, 3, 11, 41)[..., :40],
              wide.transpose(2, 3)[..., :, :][:, :, :, :].transpose(2, 3)[..., :36], wide.transpose(1, 3)[..., :3].transpose(1, 3)[..., :34]):
        p = pos[:q.shape[2]]
        check(apply_rotary(q, None, p, inv), q, p, inv, 1.0, False, False)
        check(apply_rotary(q, None, p, inv, interleaved=True) if q.shape[3] % 2 == 0 else q.contiguous(), q, p, inv if q.shape[3] % 2 == 0 else inv[:0],
              1.0, True, False)


@pytest.mark.parametrize("b,n", [(0, 5), (2, 0)])
def test_empty(b, n):
    inv, _ = rotary_frequencies(64, device="cuda")
    q, k = apply_rotary(torch.zeros(b, 4, n, 64, device="cuda"), torch.zeros(b, 2, n, 64, device="cuda"), torch.zeros(1, n, dtype=torch.int64, device="cuda"), inv)
    assert q.shape == (b, 4, n, 64) and k.shape == (b, 2, n, 64)


def test_gradient_is_the_formulas_and_matches_differences():
    g = torch.Generator(device="cuda").manual_seed(3)
    inv, factor = rotary_frequencies(16, 100.0, device="cuda")[0], 1.25
    q = torch.randn(2, 3, 5, 24, generator=g, device="cuda", requires_grad=True)
    k = torch.randn(2, 1, 5, 24, generator=g, device="cuda", requires_grad=True)
    pos = torch.randint(0, 50, (2, 5), generator=g, device="cuda")
    for interleaved in (False, True):
        q2, k2 = apply_rotary(q, k, pos, inv, factor=factor, interleaved=interleaved)
        gq, gk = torch.randn(q2.shape, generator=g, device="cuda"), torch.randn(k2.shape, generator=g, device="cuda")
        dq, dk = torch.autograd.grad([q2, k2], [q, k], [gq, gk])
        check(dq, gq, pos, inv, factor, interleaved, True)
        check(dk, gk, pos, inv, factor, interleaved, True)
        # central difference of a linear map: exact but for rounding.  <g, R(q + h v)> - <g, R(q - h v)> = 2 h <R^T g, v>;
        # both sides sum 720 products of size up to about 16 with errors of some 2^-22 each
        v = torch.randn(q.shape, generator=g, device="cuda")
        with torch.no_grad():
            up, down = apply_rotary(q + v, None, pos, inv, factor=factor, interleaved=interleaved), apply_rotary(q - v, None, pos, inv, factor=factor, interleaved=interleaved)
        diff = float(((up - down).double() / 2 * gq.double()).sum())
        assert abs(diff - float((dq.double() * v.double()).sum())) <= 720 * 16 * 2.0 ** -22
    only = torch.autograd.grad(apply_rotary(q, None, pos, inv).sum(), q)[0]
    check(only, torch.ones_like(q), pos, inv, 1.0, False, True)


def test_other_stream_and_graph():
    g = torch.Generator(device="cuda").manual_seed(4)
    inv, _ = rotary_frequencies(128, device="cuda")
    q, pos = torch.randn(1, 8, 64, 128, generator=g, device="cuda").bfloat16(), torch.arange(64, device="cuda")
    ref = apply_rotary(q, None, pos, inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = apply_rotary(q, None, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(q, None, pos, inv)
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    pos.add_(1000)
    graph.replay()
    assert torch.equal(out, apply_rotary(q, None, pos, inv))


def test_refusals():
    inv, _ = rotary_frequencies(64, device="cuda")
    q, k, pos = torch.zeros(2, 4, 3, 64, device="cuda"), torch.zeros(2, 2, 3, 64, device="cuda"), torch.arange(3, device="cuda")
    bad = [dict(q=q.half()), dict(q=q[0]), dict(k=k.bfloat16()), dict(k=k[:1]), dict(k=k[:, :, :2]), dict(k=k[..., :32]), dict(k=k.cpu()),
           dict(positions=pos.float()), dict(positions=pos[:2]), dict(positions=pos.repeat(3, 1)), dict(positions=pos.cpu()),
           dict(inv_freq=inv.float()), dict(inv_freq=inv.cpu()), dict(inv_freq=inv[:0]), dict(inv_freq=torch.cat((inv, inv[:1]))),
           dict(inv_freq=inv[::2]), dict(factor=float("inf"))]
    for kw in bad:
        args = dict(q=q, k=k, positions=pos, inv_freq=inv)
        args.update(kw)
        with pytest.raises(ValueError):
            apply_rotary(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("inv_freq"), **args)
    from lrqk_b200._lib import LrqkError
    with pytest.raises(LrqkError):
        apply_rotary(torch.zeros(1, 1, 1, 1026, device="cuda"), None, pos[:1], inv)          # a head beyond what the kernel takes
    with pytest.raises(LrqkError):
        apply_rotary(torch.zeros(1, 1, 1, 65, device="cuda"), None, pos[:1], inv, interleaved=True)
