"""Rows in eight bits at inference, against statements in 64 bits: the norm that writes them, the product that reads them, both
layers of an MLP, and a run of all of them."""
import pytest
import torch

from eight_bit_reference import gelu, int8_rows
from swin3d_amd import add_layernorm
from swin3d_amd.eight_bits import Int8Rows, add_norm_int8, checkpointed_linear, checkpointed_mlp, linear_int8, mlp_int8, quantize_rows

pytestmark = pytest.mark.gpu

WIDTHS = [4, 12, 48, 60, 64, 68, 128, 132, 256, 260, 384, 512, 516, 520, 640, 768, 776, 1024, 1028, 1032, 1536, 1544, 2048, 2052, 2056, 2560, 2568, 4096, 4100, 8192]


def _norm(kind, c, gen, eps=1e-5):
    norm = torch.nn.LayerNorm(c, eps=eps, device="cuda") if kind == "layer" else torch.nn.RMSNorm(c, eps=eps, device="cuda")
    with torch.no_grad():
        norm.weight.copy_(1 + 0.3 * torch.randn(c, device="cuda", generator=gen))
        if kind == "layer":
            norm.bias.copy_(0.2 * torch.randn(c, device="cuda", generator=gen))
    return norm.requires_grad_(False)


def _normed(summed, norm):
    s = summed.double()
    if isinstance(norm, torch.nn.LayerNorm):
        s = s - s.mean(1, keepdim=True)
    y = s / torch.sqrt(s.square().mean(1, keepdim=True) + norm.eps)
    y = y if norm.weight is None else y * norm.weight.double()
    return y + norm.bias.double() if isinstance(norm, torch.nn.LayerNorm) and norm.bias is not None else y


def _check_rows(rows, y, off):
    """Rows against float64 rows y, of which the kernel's fp32 ones are `off` [N,1] off at most: half a step of the kernel's scale and that."""
    most = y.abs().amax(1, keepdim=True)
    scales = rows.scales.double().unsqueeze(1)
    assert bool(((scales - most / 127).abs() <= off / 127 + 2.0 ** -23 * most / 127 + 2.0 ** -149).all())
    # (127 / max |y| is rounded, as is the scale: each a 2^-24th of up to 127 steps)
    far = (rows.codes.double() * scales - y).abs()
    assert bool((far <= 0.5 * scales + off + 2.0 ** -22 * most + 2.0 ** -149).all()), float((far - 0.5 * scales - off).max())
    assert int(rows.codes.abs().max()) <= 127 and bool(((rows.codes.abs() == 127).any(1) | (most[:, 0] == 0)).all())


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("kind,residual", [("layer", "fp16"), ("rms", "fp32"), ("layer", None), ("rms", "fp16")])
def test_norm_in_eight_bits(hip_lib, c, kind, residual):
    gen = torch.Generator(device="cuda").manual_seed(c)
    for n in (1, 37):
        x = torch.randn(n, c, device="cuda", generator=gen) * 3 + 0.5
        r = None if residual is None else torch.randn(n, c, device="cuda", generator=gen)
        r = r.half() if residual == "fp16" else r
        norm = _norm(kind, c, gen)
        summed, rows = add_norm_int8(x, r, norm)
        assert torch.equal(summed, x if r is None else x + r.float())
        y = _normed(summed, norm)
        # fp32: a sum over C takes at most 8 + 8 + 32 additions one behind the other, each half a unit of sizes up to C max |s|, so the
        # mean and the root are 2^-24 x 48 off relative to max |s| and to themselves; s - mean, times the root, times gamma, plus beta
        # four roundings more
        s = summed.double()
        rstd = 1 / torch.sqrt((s - (s.mean(1, keepdim=True) if kind == "layer" else 0)).square().mean(1, keepdim=True) + norm.eps)
        off = 2.0 ** -24 * 52 * (y.abs().amax(1, keepdim=True) + 0.5 + s.abs().amax(1, keepdim=True) * rstd * norm.weight.abs().max().double())
        _check_rows(rows, y, off)
        again = add_norm_int8(x, r, norm, inplace=True)
        assert torch.equal(again[0], summed) and again[0] is x and all(torch.equal(a, b) for a, b in zip(again[1], rows))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("c", WIDTHS)
def test_rows_as_they_are(hip_lib, c, dtype):
    gen = torch.Generator(device="cuda").manual_seed(c + 1)
    x = (torch.randn(29, c, device="cuda", generator=gen) * torch.exp(3 * torch.randn(29, 1, device="cuda", generator=gen))).clamp(-60000, 60000).to(dtype)
    x[3] = 0
    rows = quantize_rows(x)
    _check_rows(rows, x.double(), 0.0)
    assert float(rows.scales[3]) == 0 and not rows.codes[3].any()
    for out in (torch.float16, torch.float32):
        assert torch.equal(rows.values(out), (rows.codes.float() * rows.scales.unsqueeze(1)).to(out))


def test_rows_at_the_ends_of_the_types(hip_lib):
    """The smallest numbers and the largest, and rows with NaN and infinity, which stand for NaN beside rows that are as they were."""
    x = torch.ones(9, 64, device="cuda")
    for i, size in enumerate((1e-44, 1e-38, 1e-36, 1e-30, 1e30, 3.4e38)):
        x[i] = torch.linspace(-1, 1, 64, device="cuda") * size
    x[6, 5], x[7, 63], x[8, 0] = float("nan"), float("inf"), -float("inf")
    rows = quantize_rows(x)
    want, _ = int8_rows(x[:6].double())
    # (next to a border the other code may be taken, and a scale of fewer than 24 bits is coarse)
    assert bool(((rows.codes[1:6].double() - want[1:]).abs() <= 1).all()) and bool((rows.codes[:6].abs().amax(1) == 127).all())
    assert rows.scales[6:].isnan().all() and not rows.codes[6:].any()
    assert rows.values(torch.float32)[6:].isnan().all() and rows.values(torch.float32)[:6].isfinite().all()
    half = torch.full((2, 32), 65504.0, device="cuda").half()
    half[1] = 6e-8
    assert torch.equal(quantize_rows(half).codes, torch.full((2, 32), 127, dtype=torch.int8, device="cuda"))
    norm = torch.nn.LayerNorm(64, device="cuda").requires_grad_(False)
    x[:6] = torch.randn(6, 64, device="cuda")
    _, normed = add_norm_int8(x, None, norm)
    assert normed.scales[6:].isnan().all() and normed.scales[:6].isfinite().all()
    y = linear_int8(normed, quantize_rows(torch.randn(16, 64, device="cuda")), torch.randn(16, device="cuda"))
    assert y[6:].isnan().all() and y[:6].isfinite().all()


def test_norms_without_parameters_and_strided_rows(hip_lib):
    gen = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(50, 2 * 96, device="cuda", generator=gen)
    r = torch.randn(96, 50, device="cuda", generator=gen).half().t()
    for norm in (torch.nn.LayerNorm(96, elementwise_affine=False), torch.nn.RMSNorm(96, elementwise_affine=False), torch.nn.LayerNorm(96, bias=False).cuda()):
        norm.requires_grad_(False)
        dense = add_norm_int8(wide[:, 96:].contiguous(), r.contiguous(), norm)
        strided = add_norm_int8(wide[:, 96:], r, norm)
        assert torch.equal(dense[0], strided[0]) and all(torch.equal(a, b) for a, b in zip(dense[1], strided[1]))
        y = _normed(dense[0], _with_eps(norm))
        assert bool(((dense[1].values(torch.float32) - y).abs() <= 0.51 * y.abs().amax(1, keepdim=True) / 127).all())      # half a step


def _with_eps(norm):
    if norm.eps is None:
        norm.eps = torch.finfo(torch.float32).eps
    return norm


def _random_rows(m, k, gen):
    return Int8Rows(torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda", generator=gen), torch.rand(m, device="cuda", generator=gen) * 0.02 + 1e-3)


def _check_product(y, rows, weight, bias, with_gelu):
    z = rows.codes.double() @ weight.codes.double().t() * rows.scales.double().unsqueeze(1) * weight.scales.double()
    size = z.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    # the sum to fp32, the scales' product, its product with the sum and the bias: four halves of a unit.  GELU has a slope of up to 1.13 and is
    # 2.5e-7 off.  Then half a step of fp16, of 2^-24 for its smallest numbers.
    off = 2.0 ** -22 * size
    want = gelu(z) if with_gelu else z
    off = 1.13 * off + 2.0 ** -21 * (1 + size) if with_gelu else off
    off = off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25
    assert bool(((y.double() - want).abs() <= off).all()), float(((y.double() - want).abs() - off).max())


@pytest.mark.parametrize("m,n,k", [
    (1, 8, 16), (1, 640, 2560), (31, 24, 48), (33, 104, 80), (64, 64, 112), (65, 72, 128), (100, 1536, 384), (129, 136, 144),
    (390, 1920, 640), (811, 384, 400), (1000, 200, 4096), (3105, 1152, 384), (12421, 192, 192), (20011, 96, 240), (37499, 320, 1280),
    (66001, 240, 80), (131077, 48, 48),
])
def test_product(hip_lib, m, n, k):
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    rows, weight, bias = _random_rows(m, k, gen), _random_rows(n, k, gen), torch.randn(n, device="cuda", generator=gen)
    weight = Int8Rows(weight.codes, weight.scales * (10.0 / k))
    y = linear_int8(rows, weight, bias)
    assert y.shape == (m, n) and y.dtype == torch.float16
    _check_product(y, rows, weight, bias, False)
    _check_product(linear_int8(rows, weight), rows, weight, None, False)
    _check_product(linear_int8(rows, weight, bias, gelu=True), rows, weight, bias, True)
    assert torch.equal(linear_int8(rows, weight, bias.half()), linear_int8(rows, weight, bias.half().float()))


def test_product_of_the_largest_sums(hip_lib):
    """-128 is no code of these rows, but a sum of 65,536 products of it still fits."""
    for code in (127, -127, -128):
        rows = Int8Rows(torch.full((5, 65536), code, dtype=torch.int8, device="cuda"), torch.full((5,), 2.0 ** -20, device="cuda"))
        weight = Int8Rows(torch.full((8, 65536), code, dtype=torch.int8, device="cuda"), torch.full((8,), 2.0 ** -5, device="cuda"))
        assert torch.equal(linear_int8(rows, weight), torch.full((5, 8), code * code * 65536 * 2.0 ** -25, device="cuda").half())


def test_product_has_the_bits_of_any_tile(hip_lib):
    """Sums of whole numbers: a row's results are the same among few rows and many."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    rows, weight, bias = _random_rows(70000, 96, gen), _random_rows(288, 96, gen), torch.randn(288, device="cuda", generator=gen)
    for gelu_too in (False, True):
        y = linear_int8(rows, weight, bias, gelu=gelu_too)
        for m in (1, 33, 700, 9000):
            assert torch.equal(linear_int8(Int8Rows(rows.codes[:m], rows.scales[:m]), weight, bias, gelu=gelu_too), y[:m])


@pytest.mark.parametrize("m,c,hidden", [(1, 16, 16), (33, 48, 192), (390, 640, 2560), (811, 384, 768), (12421, 192, 768), (60001, 80, 320)])
def test_mlp_is_its_parts(hip_lib, m, c, hidden):
    gen = torch.Generator(device="cuda").manual_seed(m)
    x = quantize_rows(torch.randn(m, c, device="cuda", generator=gen))
    w1, w2 = (quantize_rows(torch.randn(a, b, device="cuda", generator=gen) / b ** 0.5) for a, b in ((hidden, c), (c, hidden)))
    b1, b2 = (torch.randn(a, device="cuda", generator=gen) for a in (hidden, c))
    for bias1, bias2 in ((b1, b2), (None, None)):
        want = linear_int8(quantize_rows(linear_int8(x, w1, bias1, gelu=True)), w2, bias2)
        assert torch.equal(mlp_int8(x, w1, bias1, w2, bias2), want)


# widths in tiles of 32 that are not whole, wavefronts without one in either layer, more of the second layer's than the first's, 32 and 64 rows,
# four wavefronts and eight, the last workgroup of one row, layers apart
@pytest.mark.parametrize("m", [1, 31, 8193, 16385, 16447])
@pytest.mark.parametrize("c,hidden", [(16, 16), (48, 16), (272, 32), (448, 48), (16, 272), (80, 320), (112, 464), (208, 416), (224, 416), (160, 624), (48, 1232),
                                      (48, 1216), (528, 32), (256, 1024)])
def test_mlp_of_any_width(hip_lib, m, c, hidden):
    gen = torch.Generator(device="cuda").manual_seed(m + c)
    x, w1, w2 = (_random_rows(n, k, gen) for n, k in ((m, c), (hidden, c), (c, hidden)))
    b1, b2 = (torch.randn(a, device="cuda", generator=gen) for a in (hidden, c))
    want = linear_int8(quantize_rows(linear_int8(x, w1, b1, gelu=True)), w2, b2)
    assert torch.equal(mlp_int8(x, w1, b1, w2, b2), want)


@pytest.mark.parametrize("m", [70, 8300, 17000])
def test_mlp_of_rows_that_are_not_finite(hip_lib, m):
    """A row whose scale is NaN, one whose hidden layer is beyond fp16 and one of zeros, each among others that stay what they are."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    x, w1, w2 = (_random_rows(n, k, gen) for n, k in ((m, 64), (128, 64), (64, 128)))
    b2 = torch.randn(64, device="cuda", generator=gen)
    clean = mlp_int8(x, w1, None, w2, b2)
    x.scales[5], x.scales[m - 1] = float("nan"), 1e9
    x.codes[40] = 0
    y = mlp_int8(x, w1, None, w2, b2)
    assert y[5].isnan().all() and y[m - 1].isnan().all() and torch.equal(y[40], b2.half())
    same = torch.ones(m, dtype=torch.bool, device="cuda")
    same[[5, 40, m - 1]] = False
    assert clean.isfinite().all() and torch.equal(y[same], clean[same])
    want = linear_int8(quantize_rows(linear_int8(x, w1, None, gelu=True)), w2, b2)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y[same], want[same])


def test_no_rows(hip_lib):
    norm = torch.nn.LayerNorm(48, device="cuda").requires_grad_(False)
    summed, rows = add_norm_int8(torch.empty(0, 48, device="cuda"), torch.empty(0, 48, device="cuda"), norm)
    weight = quantize_rows(torch.randn(16, 48, device="cuda"))
    assert summed.shape == (0, 48) and rows.values().shape == (0, 48) and linear_int8(rows, weight).shape == (0, 16)
    assert mlp_int8(rows, quantize_rows(torch.randn(64, 48, device="cuda")), None, quantize_rows(torch.randn(48, 64, device="cuda")), None).shape == (0, 48)


def _layers(c, hidden, gen):
    return [(quantize_rows(torch.randn(a, b, device="cuda", generator=gen) / b ** 0.5), 0.1 * torch.randn(a, device="cuda", generator=gen))
            for a, b in ((c, c), (hidden, c), (c, hidden))]


def _block(x, layers, norms):
    """What stands around the attention of a block: proj behind the first norm, the second norm, the MLP."""
    (proj, proj_bias), (fc1, b1), (fc2, b2) = layers
    _, rows = add_norm_int8(x, None, norms[0])
    branch = linear_int8(rows, proj, proj_bias)
    summed, rows = add_norm_int8(x, branch, norms[1])
    return summed, mlp_int8(rows, fc1, b1, fc2, b2)


@pytest.mark.parametrize("m,c", [(300, 96), (5003, 192), (20000, 48)])
def test_run_of_a_block(hip_lib, m, c):
    """Norm, product, norm with the branch's sum and MLP in a row, against the same steps in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(c)
    x, layers = torch.randn(m, c, device="cuda", generator=gen), _layers(c, 4 * c, gen)
    norms = [_norm("layer", c, gen), _norm("rms", c, gen)]
    summed, y = _block(x, layers, norms)

    def rounded(v):
        codes, scales = int8_rows(v)
        return codes * scales.unsqueeze(1)

    def dense(v, layer):
        return rounded(v) @ layer[0].values(torch.float32).double().t() + layer[1].double()

    s = x.double() + dense(_normed(x, norms[0]), layers[0]).half().double()
    want = dense(gelu(dense(_normed(s, norms[1]), layers[1])).half().double(), layers[2])
    # Where a number lies next to a border between two codes, or two fp16 numbers, fp32 may take the other one: few of them, a
    # step of a 127th of the row's largest each.  In the mean that is below the rounding of the results to fp16.
    assert float((summed.double() - s).norm() / s.norm()) <= 2.0 ** -12
    assert float((y.double() - want).norm() / want.norm()) <= 2.0 ** -9


def test_captured_and_replayed_on_another_stream(hip_lib):
    gen = torch.Generator(device="cuda").manual_seed(3)
    m, c = 3000, 96
    layers, norms = _layers(c, 384, gen), [_norm("layer", c, gen), _norm("rms", c, gen)]
    inputs = [torch.randn(m, c, device="cuda", generator=gen) for _ in range(3)]
    wants = [_block(x, layers, norms) for x in inputs]
    stream, x = torch.cuda.Stream(), inputs[0].clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _block(x, layers, norms)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _block(x, layers, norms)
    torch.cuda.synchronize()
    for i in (1, 2, 0, 1):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wants[i]))
        _block(inputs[2], layers, norms)


def test_two_streams_at_once(hip_lib):
    gen = torch.Generator(device="cuda").manual_seed(4)
    layers, norms = _layers(96, 384, gen), [_norm("layer", 96, gen), _norm("rms", 96, gen)]
    inputs = [torch.randn(9001, 96, device="cuda", generator=gen) for _ in range(2)]
    wants = [_block(x, layers, norms) for x in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in inputs], [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(_block(inputs[i], layers, norms))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for one in got[i] for a, b in zip(one, wants[i]))


def test_refusals(hip_lib):
    x, norm = torch.randn(4, 48, device="cuda"), torch.nn.LayerNorm(48, device="cuda").requires_grad_(False)
    rows, weight = quantize_rows(x), quantize_rows(torch.randn(16, 48, device="cuda"))
    for bad in (lambda: add_norm_int8(x.half(), None, norm), lambda: add_norm_int8(x[0], None, norm), lambda: add_norm_int8(x[:, :40], None, norm),
                lambda: add_norm_int8(x, x[:3], norm), lambda: add_norm_int8(x, x.cpu(), norm), lambda: add_norm_int8(x, None, torch.nn.Identity()),
                lambda: add_norm_int8(torch.randn(4, 48 * 2, device="cuda")[:, ::2], x, norm, inplace=True),
                lambda: quantize_rows(x.double()), lambda: quantize_rows(torch.randn(4, 6, device="cuda")), lambda: quantize_rows(torch.empty(4, 0, device="cuda")),
                lambda: quantize_rows(torch.empty(1, 8196, device="cuda")),
                lambda: linear_int8(x, weight), lambda: linear_int8(Int8Rows(rows.codes, rows.scales[:3]), weight),
                lambda: linear_int8(rows, quantize_rows(torch.randn(16, 64, device="cuda"))), lambda: linear_int8(rows, weight, torch.zeros(15, device="cuda")),
                lambda: linear_int8(rows, Int8Rows(weight.codes[:12], weight.scales[:12])), lambda: linear_int8(rows, weight, torch.zeros(16)),
                lambda: linear_int8(quantize_rows(torch.randn(4, 40, device="cuda")), quantize_rows(torch.randn(16, 40, device="cuda"))),
                lambda: mlp_int8(rows, weight, None, weight, None), lambda: rows.values(torch.int8)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: add_norm_int8(x.requires_grad_(), None, norm), lambda: add_norm_int8(x.detach(), None, torch.nn.LayerNorm(48, device="cuda")),
                lambda: torch.func.vmap(quantize_rows)(torch.randn(2, 4, 48, device="cuda")),
                lambda: linear_int8(rows, weight, torch.zeros(16, device="cuda", requires_grad=True)),
                lambda: linear_int8(rows, weight, torch.zeros(16, device="cuda", dtype=torch.float16, requires_grad=True)),
                lambda: mlp_int8(rows, weight, None, quantize_rows(torch.randn(48, 16, device="cuda")), torch.zeros(48, device="cuda", requires_grad=True))):
        with pytest.raises((RuntimeError, ValueError)):
            bad()


def test_offsets_beyond_32_bits(hip_lib):
    """Arrays of more than 2^31 numbers: the last rows' results are those of the same rows by themselves."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    c, last = 512, 20000
    m = 2 ** 31 // c + 40001
    x = torch.zeros(m, c, device="cuda")
    x[-last:] = torch.randn(last, c, device="cuda", generator=gen)
    norm = torch.nn.LayerNorm(c, device="cuda").requires_grad_(False)
    summed, rows = add_norm_int8(x, x[:1].half().expand(m, c), norm)
    want_sum, want = add_norm_int8(x[-last:].clone(), None, norm)
    assert torch.equal(summed[-last:], want_sum) and all(torch.equal(a[-last:], b) for a, b in zip(rows, want))
    del x, summed
    weight, bias = _random_rows(64, c, gen), torch.randn(64, device="cuda", generator=gen)
    assert torch.equal(linear_int8(rows, weight, bias)[-last:], linear_int8(want, weight, bias))
    assert torch.equal(rows.values()[-last:], want.values())
    del rows, want
    # more results than 2^31, by each of the kernels for many rows
    for k, n in ((64, 512), (512, 512)):
        rows, weight = _random_rows(m, k, gen), _random_rows(n, k, gen)
        y = linear_int8(rows, weight)
        tail = Int8Rows(rows.codes[-last:].clone(), rows.scales[-last:].clone())
        assert torch.equal(y[-last:], linear_int8(tail, weight))
        del y
    weight2 = _random_rows(512, 64, gen)
    y = mlp_int8(rows, _random_rows(64, 512, torch.Generator(device="cuda").manual_seed(1)), None, weight2, None)
    assert torch.equal(y[-last:], mlp_int8(tail, _random_rows(64, 512, torch.Generator(device="cuda").manual_seed(1)), None, weight2, None))


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norms_whose_parameters_are_not_as_long_as_they_say(hip_lib, kind):
    x = torch.randn(4, 48, device="cuda")
    for name in ("weight", "bias")[:1 if kind == "rms" else 2]:
        for other in (torch.ones(44, device="cuda"), torch.ones(0, device="cuda"), torch.ones(96, device="cuda"), torch.ones(47, device="cuda").half()):
            norm = _norm(kind, 48, torch.Generator(device="cuda").manual_seed(1))
            getattr(norm, name).data = other
            with pytest.raises(ValueError):
                add_norm_int8(x, None, norm)


def test_scales_that_require_a_gradient(hip_lib):
    """Scales are numbers that a program may train.  No call has their gradient: none drops it without a word."""
    rows, w1, w2 = (quantize_rows(torch.randn(n, k, device="cuda")) for n, k in ((4, 48), (64, 48), (48, 64)))
    trained = [Int8Rows(r.codes, r.scales.clone().requires_grad_()) for r in (rows, w1, w2)]
    odd = Int8Rows(w1.codes, torch.randn(128, device="cuda", requires_grad=True)[::2])
    calls = [lambda: trained[0].values(), lambda: linear_int8(trained[0], w1), lambda: linear_int8(rows, trained[1]), lambda: linear_int8(rows, odd),
             lambda: mlp_int8(trained[0], w1, None, w2, None), lambda: mlp_int8(rows, trained[1], None, w2, None), lambda: mlp_int8(rows, w1, None, trained[2], None)]
    for call in calls:
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad():
            assert not call().requires_grad
    with pytest.raises(RuntimeError, match="transform"):
        torch.func.vmap(lambda s: rows.values() * s)(torch.ones(2, device="cuda"))


def test_operands_whose_storage_was_freed(hip_lib):
    """Their null pointers are no sign that there is no bias, weight or residual."""
    def freed(*shape, dtype=torch.float32):
        t = torch.zeros(shape, device="cuda", dtype=dtype)
        t.untyped_storage().resize_(0)
        return t

    x, norm = torch.randn(4, 48, device="cuda"), torch.nn.LayerNorm(48, device="cuda").requires_grad_(False)
    rows, w1, w2 = (quantize_rows(torch.randn(n, k, device="cuda")) for n, k in ((4, 48), (64, 48), (48, 64)))
    emptied = [torch.nn.LayerNorm(48, device="cuda").requires_grad_(False) for _ in range(2)]
    emptied[0].weight.data, emptied[1].bias.data = freed(48), freed(48)
    half, w = x.half(), torch.randn(64, 48, device="cuda")
    for call in (lambda: add_norm_int8(x, freed(4, 48), norm), lambda: add_norm_int8(x, None, emptied[0]), lambda: add_norm_int8(x, None, emptied[1]),
                 lambda: linear_int8(rows, w1, freed(64)), lambda: linear_int8(rows, w1, freed(64, dtype=torch.float16)), lambda: linear_int8(Int8Rows(rows.codes, freed(4)), w1),
                 lambda: mlp_int8(rows, w1, freed(64), w2, None), lambda: mlp_int8(rows, w1, None, w2, freed(48)), lambda: quantize_rows(freed(4, 48)),
                 lambda: checkpointed_linear(half, w, freed(64)), lambda: checkpointed_linear(half, freed(64, 48), None),
                 lambda: checkpointed_mlp(half, w, freed(64), w.t().contiguous(), None), lambda: checkpointed_mlp(half, w, None, w.t().contiguous(), freed(48))):
        with pytest.raises(ValueError, match="without memory"):
            call()


@pytest.mark.parametrize("kind", [torch.nn.LayerNorm, torch.nn.RMSNorm])
def test_norms_with_a_forward_of_their_own(hip_lib, kind):
    """Such as add one to their weight: other norms, which the kernel does not know.  A class that only adds to the parameters is the same norm."""
    class Other(kind):
        def forward(self, x):
            return super().forward(x) + x

    class Same(kind):
        def extra_repr(self):
            return "same"

    x = torch.randn(4, 48, device="cuda")
    norms = [cls(48, device="cuda").requires_grad_(False) for cls in (Other, kind, Same, kind)]
    norms[1].forward = lambda x: x
    for norm in norms[:2]:
        with pytest.raises(ValueError, match="must be a LayerNorm or RMSNorm"):
            add_norm_int8(x, None, norm)
    assert all(torch.equal(a, b) for a, b in zip(add_norm_int8(x, None, norms[2])[1], add_norm_int8(x, None, norms[3])[1]))


@pytest.mark.parametrize("call", [add_norm_int8, add_layernorm])
def test_sum_in_place_is_a_change_that_autograd_sees(hip_lib, call):
    """A graph that has kept x for its backward would compute from the sum otherwise."""
    norm = torch.nn.LayerNorm(48, device="cuda").requires_grad_(False)
    x, residual, w = torch.randn(4, 48, device="cuda"), torch.randn(4, 48, device="cuda"), torch.randn(48, 8, device="cuda", requires_grad=True)
    for inplace, given in ((False, residual), (True, None), (True, residual)):
        y, version = x @ w, x._version
        with torch.no_grad():
            summed, _ = call(x, given, norm, inplace=inplace)
        changed = inplace and given is not None
        assert (summed is x) == (given is None or inplace) and (x._version > version) == changed
        if not changed:
            y.sum().backward()
            continue
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        call(torch.randn(4, 48, device="cuda"), residual, norm, inplace=True)


def test_rows_that_lack_a_part(hip_lib):
    rows, w1, w2 = (quantize_rows(torch.randn(n, k, device="cuda")) for n, k in ((4, 48), (64, 48), (48, 64)))
    lacking = [Int8Rows(r.codes, None) for r in (rows, w1, w2)] + [Int8Rows(None, r.scales) for r in (rows, w1, w2)]
    for i in (0, 3):
        for call in (lambda: lacking[i].values(), lambda: linear_int8(lacking[i], w1), lambda: linear_int8(rows, lacking[i + 1]),
                     lambda: mlp_int8(lacking[i], w1, None, w2, None), lambda: mlp_int8(rows, lacking[i + 1], None, w2, None),
                     lambda: mlp_int8(rows, w1, None, lacking[i + 2], None)):
            with pytest.raises(ValueError):
                call()
