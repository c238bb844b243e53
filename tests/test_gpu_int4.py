"""4-bit products on the GPU against their definition in 64 bits."""

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


def weight(k, n, group, zeros, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, (k, n), device=DEV, generator=g, dtype=torch.uint8)
    scales = (0.01 * torch.randn(k // group, n, device=DEV, generator=g)).to(torch.bfloat16)
    zero = torch.randint(0, 16, (k // group, n), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
    spread = scales.double().repeat_interleave(group, 0)
    w = (codes.double() - (8 if zero is None else zero.double().repeat_interleave(group, 0))) * spread
    return codes, scales, zero, w, spread.abs(), g


def check(got, x, w, spread, finish=lambda y: y, slope=1.0):
    """One bf16 rounding, and FP32 sums of terms x (16 + code) and x (16 + zero) times the scale, under 62
    |x| scale a weight together: at most 512 additions on the way of any of them (128 in a
    group, the groups of a wave, the waves)."""
    want = finish(x.double() @ w)
    sums = 512 * 2.0 ** -24 * 62 * (x.double().abs() @ spread)
    if sums.shape != want.shape:  # gate and up, each with the other's size as its slope
        gate, up = (x.double() @ w).chunk(2, -1)
        sums = (sums.chunk(2, -1)[0] * 1.1 * up.abs() + sums.chunk(2, -1)[1] * gate.abs())
    assert got.isfinite().all()
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + sums + 1e-30).all()
    assert (got.double() - want).norm() <= (2.0 ** -8 + 1e-4) * want.norm()


# one row to several row blocks; K of one group, of odd numbers of groups, below and past a K tile; N odd
SHAPES = [(1, 32, 1, 32), (1, 128, 16, 128), (3, 96, 33, 32), (16, 192, 40, 64), (17, 5120, 100, 128),
          (33, 1024, 2047, 64), (64, 640, 96, 128), (65, 1056, 250, 32), (130, 384, 31, 128), (2, 25600, 48, 128)]


@pytest.mark.parametrize("m,k,n,group", [(1, 25600, 1024, 128), (16, 5120, 20000, 32), (16, 25600, 512, 64), (61, 5120, 2048, 32)])
def test_int4_gives_the_same_bits_again(m, k, n, group):
    """Weights from memory: nothing is used before it has arrived."""
    codes, scales, zero, w, spread, g = weight(k, n, group, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=group)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    got = smx.int4_matmul(x, laid)
    check(got, x, w, spread)
    other = torch.empty(1 << 28, device=DEV)
    for _ in range(12):
        other.zero_()  # leaves nothing of the weight in the caches
        assert torch.equal(smx.int4_matmul(x, laid), got)


@pytest.mark.parametrize("m,k,n,group", SHAPES)
@pytest.mark.parametrize("zeros", [True, False])
def test_int4_matmul(m, k, n, group, zeros):
    codes, scales, zero, w, spread, g = weight(k, n, group, zeros)
    laid = smx.int4_weight_layout(codes, scales, zero, group=group)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    got = smx.int4_matmul(x, laid)
    check(got, x, w, spread)
    assert torch.equal(smx.int4_matmul(x, laid), got)
    # strided rows, aligned and not, give the same bits
    for pad, offset in ((8, 0), (8, 8), (3, 1)):
        wide = torch.zeros(m, k + pad, dtype=torch.bfloat16, device=DEV)
        view = wide[:, offset:offset + k] if offset + k <= k + pad else wide[:, :k]
        view.copy_(x)
        assert torch.equal(smx.int4_matmul(view, laid), got)


# each way the kernels run: x in LDS in eight and sixteen waves, more than half of LDS, x by wave; streamed
# x of 16, 32 and 64 rows, K whole and in shares
@pytest.mark.parametrize("m,k,n,group,epilogue", [
    (1, 128, 32832, 128, None), (2, 256, 32900, 64, "swiglu"), (1, 8320, 34, 64, "swiglu"), (12, 5120, 70, 128, "residual_add"),
    (16, 5120, 98, 32, "swiglu"), (15, 6016, 100, 64, "residual_add"), (16, 12800, 40, 128, "bias_add"), (9, 12832, 66, 32, "swiglu"),
    (32, 2048, 98, 128, "swiglu"), (31, 12800, 1030, 64, "residual_add"), (32, 512, 96, 128, "swiglu"),
    (61, 6400, 10300, 128, "swiglu"), (64, 25600, 2750, 64, "residual_add"), (128, 5152, 13200, 32, None)])
def test_int4_launches(m, k, n, group, epilogue):
    codes, scales, zero, w, spread, g = weight(k, n, group, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=group, epilogue="swiglu" if epilogue == "swiglu" else None)
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)
    extra = torch.randn(*((n,) if epilogue == "bias_add" else (m, n)), device=DEV, generator=g).to(torch.bfloat16)
    options = {"residual_add": {"residual": extra}, "bias_add": {"bias": extra}}.get(epilogue, {})

    def finish(y):
        if epilogue == "swiglu":
            gate, up = y.chunk(2, -1)
            return gate * torch.sigmoid(gate) * up
        return y + extra.double() if options else y

    got = smx.int4_matmul(x, laid, epilogue=epilogue, **options)
    check(got, x, w, spread, finish)
    assert torch.equal(smx.int4_matmul(x, laid, epilogue=epilogue, **options), got)


def test_int4_matmul_is_exact_on_whole_numbers():
    """Codes, zeros, scales of 1 and whole x: every sum is exact in FP32."""
    codes, _, zero, _, _, g = weight(640, 48, 64, True)
    x = torch.randint(-3, 4, (5, 640), device=DEV, generator=g).to(torch.bfloat16)
    ones = torch.ones(10, 48, dtype=torch.bfloat16, device=DEV)
    want = x.double() @ (codes.double() - zero.double().repeat_interleave(64, 0))
    got = smx.int4_matmul(x, smx.int4_weight_layout(codes, ones, zero, group=64))
    assert torch.equal(got, want.to(torch.bfloat16))


@pytest.mark.parametrize("m,n", [(1, 40), (16, 64), (20, 47), (64, 200)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_int4_residual_and_bias(m, n, dtype):
    codes, scales, zero, w, spread, g = weight(256, n, 128, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=128)
    x = torch.randn(m, 256, device=DEV, generator=g).to(torch.bfloat16)
    residual = torch.randn(m, 2 * n + 1, device=DEV, generator=g).to(dtype)[:, 1::2][:, :n]  # strided columns
    bias = torch.randn(n, device=DEV, generator=g).to(dtype)
    check(smx.int4_matmul(x, laid, epilogue="residual_add", residual=residual), x, w, spread,
          lambda y: y + residual.double())
    check(smx.int4_matmul(x, laid, epilogue="bias_add", bias=bias), x, w, spread, lambda y: y + bias.double())
    shared = residual[:1].expand(m, n)  # one row for all
    check(smx.int4_matmul(x, laid, epilogue="residual_add", residual=shared), x, w, spread,
          lambda y: y + shared.double())


@pytest.mark.parametrize("m,k,n,group", [(1, 128, 2, 128), (4, 320, 34, 64), (16, 512, 128, 32), (61, 1024, 98, 128)])
def test_int4_swiglu(m, k, n, group):
    codes, scales, zero, w, spread, g = weight(k, n, group, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=group, epilogue="swiglu")
    x = torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16)

    def gated(y):
        gate, up = y.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up

    check(smx.int4_matmul(x, laid, epilogue="swiglu"), x, w, spread, gated)


def test_int4_swiglu_of_large_gates():
    """Gates far out on both sides: silu is the gate or zero, never NaN."""
    codes = torch.full((128, 4), 15, dtype=torch.uint8, device=DEV)
    scales = torch.tensor([[100.0, -100.0, 1.0, 1.0]], device=DEV).to(torch.bfloat16)
    laid = smx.int4_weight_layout(codes, scales, group=128, epilogue="swiglu")
    x = torch.ones(1, 128, dtype=torch.bfloat16, device=DEV)
    got = smx.int4_matmul(x, laid, epilogue="swiglu")
    assert got[0, 0] == torch.tensor(700.0 * 128 * 7 * 128).to(torch.bfloat16) and got[0, 1] == 0


@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_quantize(group):
    """Every weight within half a step of its code's value; zeros stay zero; constant and zero groups."""
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randn(384, 50, device=DEV, generator=g) * 0.02
    w[:group, 0], w[:group, 1], w[:group, 2] = 0.0, 0.5, -0.5
    codes, scales, zeros = smx.int4_quantize(w, group)
    spread = scales.double().repeat_interleave(group, 0)
    back = (codes.double() - zeros.double().repeat_interleave(group, 0)) * spread
    # the scale's own rounding (2^-8 of 15 steps) and the zero point's moves the ends by up to half a step more
    assert ((back - w.double()).abs() <= spread * (1 + 15 * 2.0 ** -8) + 1e-12).all()
    assert not back[:group, 0].any()
    x = torch.randn(4, 384, device=DEV, generator=g).to(torch.bfloat16)
    check(smx.int4_matmul(x, smx.int4_weight_layout(codes, scales, zeros, group=group)), x, back, spread)


def test_int4_rows_keep_to_themselves():
    """A NaN or an infinity spoils its own row alone."""
    codes, scales, zero, w, spread, g = weight(256, 40, 64, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=64)
    x = torch.randn(20, 256, device=DEV, generator=g).to(torch.bfloat16)
    clean = smx.int4_matmul(x, laid)
    x[3, 7], x[17, 200] = math.nan, math.inf
    got = smx.int4_matmul(x, laid)
    assert got[3].isnan().all() and got[17].isnan().all()
    keep = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(got[keep], clean[keep])


def test_int4_in_a_graph_and_on_a_stream():
    codes, scales, zero, w, spread, g = weight(1024, 96, 128, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=128)
    x = torch.randn(3, 1024, device=DEV, generator=g).to(torch.bfloat16)
    smx.int4_matmul(x, laid)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = smx.int4_matmul(x, laid)
    for _ in range(3):
        x.copy_(torch.randn(3, 1024, device=DEV, generator=g))
        want = smx.int4_matmul(x, laid)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = smx.int4_matmul(x, laid)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_int4_no_rows():
    codes, scales, zero, *_ = weight(128, 40, 128, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=128)
    assert smx.int4_matmul(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), laid).shape == (0, 40)


def test_int4_refusals():
    codes, scales, zero, *_ = weight(128, 40, 128, True)
    laid = smx.int4_weight_layout(codes, scales, zero, group=128)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    for args, kwargs, message in (
            ((x.float(), laid), {}, "bf16"), ((x[:, :64], laid), {}, "inner"), ((x, laid), {"epilogue": "geglu"}, "epilogue"),
            ((x, laid), {"epilogue": "swiglu"}, "laid out"), ((x, laid), {"epilogue": "residual_add"}, "residual"),
            ((x, laid), {"bias": x[0, :40]}, "bias"), ((x.cpu(), laid), {}, "HIP device"),
            ((x, laid), {"epilogue": "bias_add", "bias": x[0, :41]}, "shape"),
            ((x.clone().requires_grad_(), laid), {}, "gradients")):
        with pytest.raises(ValueError, match=message):
            smx.int4_matmul(*args, **kwargs)
    with pytest.raises(TypeError):
        smx.int4_matmul(x, codes)
