"""flash_rotary on the GPU against the 64-bit form: types, layouts of the pairs, parts of a row, strides, positions, gradients."""
import numpy as np
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def frequencies(fa, rot, **kw):
    return fa.rotary_frequencies(rot, **kw)[0]


def expected(x, positions, inv_freq, interleaved=False, factor=1.0, inverse=False):
    """(result, bound) for x [B,H,N,d] on the CPU, positions [N] or [B,N]"""
    cos, sin = ref.angles(positions.numpy(), inv_freq.numpy())
    if positions.dim() == 2:
        cos, sin = cos[:, None], sin[:, None]
    y = ref.rotate(x, cos, -sin if inverse else sin, interleaved, factor)
    return y, ref.rotate_bound(x, cos, interleaved, factor, x.dtype, y)


def check(y, x, positions, inv_freq, **kw):
    want, bound = expected(x, positions, inv_freq, **kw)
    off = (y.cpu().double() - want).abs() - bound
    assert off.max() <= 0, off.max()
    rot = 2 * inv_freq.numel()
    assert torch.equal(y.cpu()[..., rot:], x[..., rot:])  # behind the part that turns


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# (the last ones at odd sizes: narrow pieces, or element by element)
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (128, 64), (80, 32), (96, 40), (40, 8), (256, 256), (1000, 512), (2, 2), (7, 6), (33, 10), (130, 126)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(fa, dtype, interleaved, d, rot):
    x = normal((2, 3, 37, d), dtype, d + rot)
    positions = torch.arange(5, 42)
    f = frequencies(fa, rot)
    for inverse in (False, True):
        y = fa.flash_rotary(x.cuda(), positions.cuda(), f.cuda(), interleaved=interleaved, factor=1.25, inverse=inverse)
        check(y, x, positions, f, interleaved=interleaved, factor=1.25, inverse=inverse)


@pytest.mark.parametrize("B,H,N", [(1, 1, 1), (1, 32, 1), (3, 5, 1), (1, 1, 4097), (17, 2, 300), (1, 70, 3)])
def test_sizes(fa, B, H, N):
    x = normal((B, H, N, 64), torch.float16, N)
    positions = torch.randint(0, 100000, (B, N), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    f = frequencies(fa, 64)
    check(fa.flash_rotary(x.cuda(), positions.cuda(), f.cuda()), x, positions, f)


@pytest.mark.parametrize("first", [10 ** 6, 2 ** 31 - 40, 2 ** 40, 2 ** 53 - 40])
def test_far_positions(fa, first):
    x = normal((1, 2, 33, 128), torch.float32, 3)
    positions = first + torch.arange(33)
    f = frequencies(fa, 128)
    check(fa.flash_rotary(x.cuda(), positions.cuda(), f.cuda()), x, positions, f)


def test_negative_positions(fa):
    x = normal((1, 2, 33, 128), torch.float32, 4)
    positions = torch.arange(-40, -7, dtype=torch.int32)
    f = frequencies(fa, 128)
    check(fa.flash_rotary(x.cuda(), positions.cuda(), f.cuda()), x, positions, f)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_strides_and_alignment(fa, offset, interleaved):
    """Heads and rows in other orders, pieces of wider rows, bases off 16 bytes, positions with a stride between batches."""
    B, H, N, d = 2, 4, 19, 64
    f = frequencies(fa, d)
    positions = torch.arange(3 * 64).view(3, 64)[:2, 7:7 + N]
    wide = normal((B, N, 3 * H, d + 12), torch.bfloat16, 5)
    x = wide.cuda()[:, :, H:2 * H, offset:offset + d].transpose(1, 2)
    host = wide[:, :, H:2 * H, offset:offset + d].transpose(1, 2)
    y = fa.flash_rotary(x, positions.cuda(), f.cuda(), interleaved=interleaved)
    check(y, host, positions, f, interleaved=interleaved)
    # in place: the same rows, and nothing beside them
    whole = wide.cuda()
    part = whole[:, :, H:2 * H, offset:offset + d].transpose(1, 2)
    z = fa.flash_rotary(part, positions.cuda(), f.cuda(), interleaved=interleaved, out=part)
    assert z.data_ptr() == part.data_ptr() and torch.equal(z, y)
    whole[:, :, H:2 * H, offset:offset + d] = 0
    rest = wide.clone()
    rest[:, :, H:2 * H, offset:offset + d] = 0
    assert torch.equal(whole.cpu(), rest)
    # somewhere else
    out = torch.full((B, H, N, d + 5), 9.0, dtype=torch.bfloat16, device="cuda")
    fa.flash_rotary(x, positions.cuda(), f.cuda(), interleaved=interleaved, out=out[..., :d])
    assert torch.equal(out[..., :d], y) and (out[..., d:] == 9).all()


def test_in_place_part_of_a_row(fa):
    x = normal((2, 3, 21, 80), torch.float16, 6)
    f = frequencies(fa, 48)
    positions = torch.arange(21)
    y = x.cuda()
    fa.flash_rotary(y, positions.cuda(), f.cuda(), out=y)
    check(y, x, positions, f)


def test_tokens(fa):
    x = normal((41, 6, 128), torch.bfloat16, 7)
    positions = torch.arange(41) * 3
    f = frequencies(fa, 128)
    y = fa.flash_rotary(x.cuda(), positions.cuda(), f.cuda())
    check(y.transpose(0, 1)[None], x.transpose(0, 1)[None], positions, f)


def test_broadcast_rows(fa):
    """One row read by every head (stride 0)."""
    x = normal((1, 1, 9, 64), torch.float16, 8)
    positions, f = torch.arange(9), frequencies(fa, 64)
    y = fa.flash_rotary(x.cuda().expand(2, 5, 9, 64), positions.cuda(), f.cuda())
    check(y, x.expand(2, 5, 9, 64), positions, f)


def test_special_values_stay_in_their_pairs(fa):
    x = normal((1, 1, 4, 64), torch.float32, 9)
    x[0, 0, 1, 3], x[0, 0, 2, 40] = float("nan"), float("inf")
    y = fa.flash_rotary(x.cuda(), torch.arange(4).cuda(), frequencies(fa, 64).cuda()).cpu()
    bad = ~torch.isfinite(y)
    assert set(map(tuple, bad.nonzero().tolist())) <= {(0, 0, 1, 3), (0, 0, 1, 35), (0, 0, 2, 8), (0, 0, 2, 40)} and bad.sum() >= 3


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(fa, interleaved):
    """backward() against the transposed map in 64 bits and against differences of the result."""
    B, H, N, d, rot = 2, 3, 11, 40, 32
    f, factor = frequencies(fa, rot, scaling="linear", stretch=4.0), 1.1
    positions = torch.randint(0, 5000, (B, N), generator=torch.Generator().manual_seed(2))
    base, g = normal((B, N, H, d), torch.float32, 10), normal((B, H, N, d), torch.float32, 11)
    leaf = base.cuda().requires_grad_()
    x = leaf.transpose(1, 2)
    y = fa.flash_rotary(x, positions.cuda(), f.cuda(), interleaved=interleaved, factor=factor)
    check(y.detach(), base.transpose(1, 2), positions, f, interleaved=interleaved, factor=factor)
    y.backward(g.cuda())
    want, bound = expected(g, positions, f, interleaved, factor, inverse=True)
    assert ((leaf.grad.cpu().transpose(1, 2).double() - want).abs() <= bound).all()
    # the map is linear: a difference of any size is exact but for the roundings of y, 2^-24 of its elements and those of the sum
    e = normal((B, N, H, d), torch.float32, 12)
    y2 = fa.flash_rotary((base + e).cuda().transpose(1, 2), positions.cuda(), f.cuda(), interleaved=interleaved, factor=factor)
    left = ((y2 - y.detach()).double().cpu() * g.double()).sum()
    right = (leaf.grad.double().cpu() * e.double()).sum()
    size = (y2.double().cpu().abs() + y.detach().double().cpu().abs() + 2).mul(g.double().abs()).sum()
    assert abs(left - right) <= 40 * 2.0 ** -24 * size


def test_gradient_of_a_broadcast_input_and_of_the_gradient(fa):
    f = frequencies(fa, 16).cuda()
    positions = torch.arange(6).cuda()
    leaf = normal((1, 1, 6, 16), torch.float32, 13).cuda().requires_grad_()
    fa.flash_rotary(leaf.expand(3, 2, 6, 16), positions, f).sum().backward()
    one = fa.flash_rotary(torch.ones((1, 1, 6, 16), device="cuda"), positions, f, inverse=True)
    assert torch.allclose(leaf.grad, 6 * one, rtol=0, atol=40 * 2.0 ** -24)
    x = normal((1, 2, 6, 16), torch.float32, 14).cuda().requires_grad_()
    g, = torch.autograd.grad(fa.flash_rotary(x, positions, f).pow(2).sum(), x, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), x)  # a turn keeps lengths: the gradient is 2 x
    assert torch.allclose(g, 2 * x, rtol=0, atol=1e-5) and torch.allclose(gg, torch.full_like(gg, 2.0), rtol=0, atol=1e-5)


def test_stream_and_graph(fa):
    x = normal((1, 8, 65, 128), torch.float16, 15).cuda()
    f, positions = frequencies(fa, 128).cuda(), torch.arange(65).cuda()
    y = fa.flash_rotary(x, positions, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    z = fa.flash_rotary(x, positions, f, stream=side)
    side.synchronize()
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = fa.flash_rotary(x, positions, f)
    for shift in (0, 1000, 7):
        positions.copy_(torch.arange(65) + shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, fa.flash_rotary(x, positions, f))
        torch.cuda.synchronize()


def test_empty(fa):
    f = frequencies(fa, 16).cuda()
    for shape in ((0, 2, 3, 16), (1, 0, 3, 16), (1, 2, 0, 16)):
        assert fa.flash_rotary(torch.empty(shape, device="cuda"), torch.arange(shape[2]).cuda(), f).shape == shape


def test_offsets_past_32_bits(fa):
    """Rows of one tensor more than 2^32 bytes apart."""
    big = torch.empty(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    far = 2 ** 31
    x = big.as_strided((1, 2, 3, 64), (0, far, 64, 1))
    host = normal((1, 2, 3, 64), torch.float16, 16)
    x.copy_(host)
    f, positions = frequencies(fa, 64), torch.arange(3)
    check(fa.flash_rotary(x, positions.cuda(), f.cuda(), out=torch.empty((1, 2, 3, 64), dtype=torch.float16, device="cuda")), host, positions, f)
    fa.flash_rotary(x, positions.cuda(), f.cuda(), out=x)
    check(x, host, positions, f)


def test_frequencies_that_need_a_gradient(fa):
    """A learned inv_freq would get none: refused while gradients are recorded, taken where they are not."""
    x, n, f = torch.randn((1, 2, 3, 16), device="cuda"), torch.arange(3, device="cuda"), torch.rand(8, device="cuda", requires_grad=True)
    for y in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="inv_freq gets no gradient"):
            fa.flash_rotary(y, n, f)
    with pytest.raises(ValueError, match="out must not"):
        fa.flash_rotary(x, n, f.detach(), out=torch.zeros_like(x).requires_grad_())
    with torch.no_grad():
        assert torch.equal(fa.flash_rotary(x, n, f), fa.flash_rotary(x, n, f.detach()))
