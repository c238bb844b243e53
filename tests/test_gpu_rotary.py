"""Rotary positions on the GPU against their definition in 64 bits."""

import math

import pytest
import torch

import strassen_tpu_amd as smx
from test_gpu_parity import DEV, say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    say(f"\n[gpu] {request.node.nodeid}")
    yield
    torch.cuda.synchronize()


def rotate64(x, positions, frequencies, interleaved=False, amplitude=1.0, norm=None, eps=1e-6):
    """The rotated heads, and the sizes that their errors go by: |a| + |b| of each value's pair."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * norm.double()
    half = frequencies.numel()
    angle = positions.double()[:, None] * frequencies.double()
    cos, sin = amplitude * angle.cos()[:, None], amplitude * angle.sin()[:, None]
    out, size = x.clone(), x.abs()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = amplitude * (a.abs() + b.abs())
    return out, size


def check(got, want, size):
    """FP32's part: the angle, less whole quarters, is off by 2^-25 of up to an eighth of a turn (5e-8), sine and cosine by
    two last bits (1.2e-7), amplitude, products and sum by four roundings (2.4e-7), the norm by the squares' sum over up to
    2^10 values (half of 26 roundings), a root, a quotient and two products (1e-6): 2e-6 of the pair in all.
    Then the result's own rounding."""
    half_step = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= half_step * want.abs() + 2e-6 * size + 1e-37).all()


SHAPES = [
    # tokens, heads, dim, rotated, dtype
    (1, 1, 128, 128, torch.bfloat16), (16, 72, 128, 128, torch.bfloat16), (5, 3, 64, 64, torch.float32),
    (33, 10, 256, 64, torch.bfloat16), (7, 5, 80, 80, torch.bfloat16), (7, 5, 80, 80, torch.float32),
    (9, 2, 72, 64, torch.bfloat16), (9, 300, 96, 48, torch.float32),
    # value by value: pairs that are no multiple of eight, odd heads
    (9, 7, 80, 40, torch.bfloat16), (4, 3, 7, 6, torch.float32), (4, 3, 7, 2, torch.bfloat16), (3, 2, 2, 2, torch.bfloat16),
    (3, 2, 1024, 1024, torch.bfloat16), (2, 3, 1000, 999 // 2 * 2, torch.float32),
    # several rows a workgroup
    (2049, 4, 64, 64, torch.bfloat16), (4099, 3, 128, 64, torch.float32),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotated,dtype", SHAPES)
def test_rotary(tokens, heads, dim, rotated, dtype, interleaved):
    g = torch.Generator(device=DEV).manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, device=DEV, generator=g).to(dtype)
    positions = torch.randint(0, 1 << 20, (tokens,), device=DEV, generator=g, dtype=torch.int32)
    frequencies, _ = smx.rotary_frequencies(rotated, 1e4, device=DEV)
    want, size = rotate64(x, positions, frequencies, interleaved)
    kept = x.clone()
    got = smx.rotary(x, positions, frequencies, interleaved=interleaved)
    assert got.dtype == dtype and torch.equal(x, kept)
    check(got, want, size)
    assert torch.equal(got[..., rotated:], x[..., rotated:])
    assert torch.equal(smx.rotary(x, positions.long(), frequencies, interleaved=interleaved), got)
    assert smx.rotary(x, positions, frequencies, interleaved=interleaved, out=x) is x and torch.equal(x, got)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated,dtype,norm_dtype", [
    (128, 128, torch.bfloat16, torch.bfloat16), (64, 32, torch.float32, torch.float32), (512, 512, torch.bfloat16, torch.float32),
    (96, 64, torch.bfloat16, torch.bfloat16), (30, 10, torch.float32, torch.bfloat16), (1024, 16, torch.float32, torch.float64),
    (16, 16, torch.bfloat16, torch.bfloat16)])
def test_rotary_behind_a_norm(dim, rotated, dtype, norm_dtype, interleaved):
    g = torch.Generator(device=DEV).manual_seed(dim)
    x = (3 * torch.randn(37, 9, dim, device=DEV, generator=g)).to(dtype)
    x[3, 2] = 0
    norm = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g)).to(norm_dtype)
    positions = torch.randint(0, 4000, (37,), device=DEV, generator=g)
    frequencies, _ = smx.rotary_frequencies(rotated, device=DEV)
    args = dict(interleaved=interleaved, amplitude=1.25, norm=norm, eps=1e-5)
    want, size = rotate64(x, positions, frequencies, **args)
    check(smx.rotary(x, positions, frequencies, **args), want, size)


@pytest.mark.parametrize("dtype,norm,interleaved", [(torch.bfloat16, False, False), (torch.bfloat16, True, True), (torch.float32, True, False),
                                                    (torch.float32, False, True)])
def test_rotary_of_more_than_the_caches_hold(dtype, norm, interleaved):
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(4111 if dtype == torch.bfloat16 else 2051, 103, 128, device=DEV, generator=g).to(dtype)
    assert 2 * x.numel() * x.element_size() > 200 << 20
    positions = torch.randint(-1, 100000, (x.shape[0],), device=DEV, generator=g)
    positions[7] = -3
    frequencies, _ = smx.rotary_frequencies(64, device=DEV)
    args = dict(interleaved=interleaved, norm=1 + 0.1 * torch.randn(128, device=DEV, generator=g) if norm else None)
    got = smx.rotary(x, positions, frequencies, **args)
    inside = positions >= 0
    check(got[inside], *rotate64(x[inside], positions[inside], frequencies, **args))
    assert got[~inside].eq(0).all()
    assert torch.equal(smx.rotary(x, positions, frequencies, out=x.clone(), **args)[inside], got[inside])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_of_far_positions(dtype):
    """Positions past 2^31, and frequencies of whole turns, where a position's own digits are all that is left."""
    positions = torch.tensor([0, 1, 123456789, 2**31 - 1, 2**31 + 12345, 2**40 + 1], device=DEV)
    x = torch.randn(6, 2, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    turns = torch.arange(32, dtype=torch.float64) / 64  # of a whole turn each position: exact in 64 bits
    got = smx.rotary(x, positions, (turns * (2 * math.pi)).to(DEV))
    # 2^40 positions by a frequency's last bit (2^-53 of up to 2 pi): 8e-4 of a radian
    angle = (positions.cpu().double()[:, None] * turns % 1.0 * (2 * math.pi)).to(DEV)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.double().chunk(2, -1)
    want, size = torch.cat((a * cos - b * sin, b * cos + a * sin), -1), (a.abs() + b.abs()).repeat(1, 1, 2)
    off = positions.double()[:, None, None] * (2 * math.pi) * 2**-53 * 2
    assert ((got.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + (off + 2e-6) * size).all()


def test_rotary_takes_float32_frequencies_as_they_are():
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(50, 3, 64, device=DEV, generator=g)
    positions = torch.randint(0, 200000, (50,), device=DEV, generator=g)
    frequencies = smx.rotary_frequencies(64, device=DEV)[0].float()
    want, size = rotate64(x, positions, frequencies)
    got = smx.rotary(x, positions, frequencies)
    check(got, want, size)
    assert torch.equal(smx.rotary(x, positions, frequencies.double()), got)


def test_rotary_of_views():
    """Columns of a projection, heads outside the tokens, rows of odd distances, repeated rows, strided values."""
    g = torch.Generator(device=DEV).manual_seed(3)
    frequencies, _ = smx.rotary_frequencies(64, device=DEV)
    positions = torch.arange(100, 120, device=DEV, dtype=torch.int32)
    qkv = torch.randn(20, 12, 64, device=DEV, generator=g).to(torch.bfloat16)
    odd = torch.randn(20 * 12 * 67 + 1, device=DEV, generator=g).to(torch.bfloat16)
    views = [qkv[:, :10], qkv[:, 3:4], qkv.transpose(0, 1).contiguous().transpose(0, 1), qkv[:1].expand(20, 12, 64),
             odd[1:].as_strided((20, 12, 64), (12 * 67, 67, 1)), qkv.repeat(1, 1, 2)[..., ::2], qkv[::1, ::3]]
    for x in views:
        want, size = rotate64(x, positions, frequencies)
        check(smx.rotary(x, positions, frequencies), want, size)
    assert torch.equal(smx.rotary(qkv, torch.stack((positions, positions), 1)[:, 0], frequencies), smx.rotary(qkv, positions, frequencies))
    # into columns of a wider tensor, in place among others
    for view in (lambda t: t[:, 2:7], lambda t: t[..., 8:72] if t.shape[-1] > 64 else t[:, ::2]):
        wide = torch.randn(20, 12, 80, device=DEV, generator=g).to(torch.bfloat16)
        x = view(wide)[..., :64]
        kept, want = wide.clone(), smx.rotary(x, positions, frequencies)
        smx.rotary(x, positions, frequencies, out=x)
        assert torch.equal(x, want)
        view(kept)[..., :64].copy_(want)
        assert torch.equal(wide, kept)


@pytest.mark.parametrize("dim,norm", [(64, False), (64, True), (36, False), (36, True)])
def test_rows_of_no_position(dim, norm):
    """Zero in a new result, left as they were in one that is given; their values are not read as numbers."""
    x = torch.randn(30, 4, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)).to(torch.bfloat16)
    positions = torch.arange(30, device=DEV, dtype=torch.int32)
    positions[[0, 7, 29]] = -1
    x[7] = math.nan
    frequencies, _ = smx.rotary_frequencies(dim // 2 * 2, device=DEV)
    args = dict(norm=torch.ones(dim, dtype=torch.bfloat16, device=DEV) if norm else None)
    got = smx.rotary(x, positions, frequencies, **args)
    assert not got[positions < 0].any() and got[positions >= 0].isfinite().all()
    out = torch.full_like(x, 7)
    smx.rotary(x, positions, frequencies, out=out, **args)
    assert (out[positions < 0] == 7).all() and torch.equal(out[positions >= 0], got[positions >= 0])


def test_infinities_stay_in_their_pairs():
    x = torch.randn(4, 3, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).to(torch.bfloat16)
    frequencies, _ = smx.rotary_frequencies(64, device=DEV)
    positions = torch.arange(4, device=DEV)
    want = smx.rotary(x, positions, frequencies)
    x[1, 1, 5], x[2, 0, 40] = math.inf, math.nan
    got = smx.rotary(x, positions, frequencies)
    odd = torch.zeros_like(x, dtype=torch.bool)
    odd[1, 1, [5, 37]] = odd[2, 0, [8, 40]] = True
    assert not got[odd].isfinite().any() and torch.equal(got[~odd], want[~odd])


def test_past_32_bit_offsets():
    """Rows whose offsets pass 2^31 elements and 2^32 bytes."""
    stride = (1 << 31) + 64
    memory = torch.empty(stride + 2 * 128, dtype=torch.bfloat16, device=DEV)
    x = memory.as_strided((2, 2, 128), (stride, 128, 1))
    x.copy_(torch.randn(2, 2, 128, device=DEV))
    frequencies, _ = smx.rotary_frequencies(128, device=DEV)
    positions = torch.tensor([3, 70000], device=DEV)
    want, size = rotate64(x, positions, frequencies)
    check(smx.rotary(x, positions, frequencies), want, size)
    smx.rotary(x, positions, frequencies, out=x)
    check(x, want, size)


def test_nothing_to_rotate_and_other_streams():
    frequencies, _ = smx.rotary_frequencies(64, device=DEV)
    empty = smx.rotary(torch.empty(0, 3, 64, device=DEV), torch.empty(0, device=DEV, dtype=torch.int32), frequencies)
    assert empty.shape == (0, 3, 64)
    x = torch.randn(200, 8, 64, device=DEV)
    positions = torch.arange(200, device=DEV)
    want = smx.rotary(x, positions, frequencies)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [smx.rotary(x, positions + i, frequencies) for i in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want)
    assert torch.equal(got[3], smx.rotary(x, positions + 3, frequencies))


def test_refusals():
    x, positions = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    f, _ = smx.rotary_frequencies(64, device=DEV)
    bad = [
        (dict(x=x.half()), "bf16 or float32"), (dict(x=x[0]), "heads"), (dict(positions=positions[:3]), "positions"),
        (dict(positions=positions.float()), "positions"), (dict(frequencies=f[None]), "frequencies"),
        (dict(frequencies=f.half()), "frequencies"), (dict(frequencies=f.repeat(2)), "frequencies"),
        (dict(frequencies=f[:0]), "frequencies"), (dict(frequencies=f.cpu()), "HIP device"), (dict(norm=torch.ones(32, device=DEV)), "norm"),
        (dict(amplitude=math.inf), "amplitude"), (dict(amplitude=math.nan), "amplitude"), (dict(eps=-1.0), "eps"),
        (dict(out=torch.zeros(4, 2, 64, device=DEV, dtype=torch.bfloat16)), "out"), (dict(out=torch.zeros(4, 64, 2, device=DEV).transpose(1, 2)), "out"),
        (dict(out=torch.zeros(1, 2, 64, device=DEV).expand(4, 2, 64)), "each other"),
        (dict(x=torch.zeros(2, 2, 1025, device=DEV), positions=positions[:2]), "1024"),
        (dict(x=x.requires_grad_(False).clone().requires_grad_()), "gradients"),
    ]
    for change, message in bad:
        args = {"x": x, "positions": positions, "frequencies": f, **change}
        with pytest.raises(ValueError, match=message):
            smx.rotary(args.pop("x"), args.pop("positions"), args.pop("frequencies"), **args)
    rows = torch.zeros(5, 2, 64, device=DEV)
    for a, b in ((rows[:4], rows[1:]), (rows[1:], rows[:4])):
        with pytest.raises(ValueError, match="share no memory"):
            smx.rotary(a, positions, f, out=b)
    with pytest.raises(TypeError, match="tensor"):
        smx.rotary(x, positions, [1.0])
    version = x._version
    smx.rotary(x, positions, f, out=x)
    assert x._version > version
