"""Checkpoints in eight bits: their form, and the layers that keep their inputs in it, against statements in whole numbers and 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from eight_bit_reference import GROUP, gelu, gelu_slope, keep, kept
from swin3d_amd.eight_bits import checkpointed_linear, checkpointed_mlp, keep_rows, kept_values

pytestmark = pytest.mark.gpu


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _split(buffer, m, c):
    return buffer[:m * c].view(torch.int8).view(m, c), buffer[m * c:].view(m, c // GROUP)


@pytest.mark.parametrize("m,c", [(1, 16), (3, 48), (257, 80), (1000, 640), (33, 16384)])
def test_form(hip_lib, m, c):
    gen = torch.Generator(device="cuda").manual_seed(m + c)
    x = (_normal(gen, m, c) * torch.exp(4 * _normal(gen, m, 1)) * torch.exp(_normal(gen, c))).clamp(-65504, 65504).half()
    x[0, :16] = 0
    codes, byte = keep(x)
    got = keep_rows(x)
    assert torch.equal(_split(got, m, c)[0].cpu().long(), codes) and torch.equal(_split(got, m, c)[1].cpu().long(), byte)
    assert torch.equal(kept_values(got, c).double(), kept(x))
    # half a step, whose scale is at most an eighth above a 127th of the largest (or 2^-24)
    most = x.double().abs().view(m, -1, GROUP).amax(2, keepdim=True)
    far = (kept(x) - x.double()).abs().view(m, -1, GROUP)
    assert bool((far <= 0.5 * 1.125 * most / 127).logical_or(most >= 60960).logical_or(most < 127 * 2.0 ** -21).all())


def test_every_fp16_number_beside_every_largest(hip_lib):
    """Groups whose largest number takes all scales, and whose others go through all fp16 numbers below it."""
    sizes = torch.arange(1, 0x7c00, dtype=torch.int16, device="cuda").view(torch.float16)
    largest = sizes[torch.linspace(0, sizes.numel() - 1, 1500, device="cuda").long()]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.minimum(sizes[(torch.rand(1500, 1008, device="cuda", generator=gen) * sizes.numel()).long()], largest.unsqueeze(1))
    # ... most of them within a factor of 256 of it, where the codes are not zero
    near = largest.unsqueeze(1).float() * torch.exp2(-8 * torch.rand(1500, 1008, device="cuda", generator=gen))
    x = torch.where(torch.rand(1500, 1008, device="cuda", generator=gen) < 0.8, near.half(), x)
    x = x * torch.where(torch.rand(1500, 1008, device="cuda", generator=gen) < 0.5, -1.0, 1.0).half()
    x[:, ::GROUP] = largest.unsqueeze(1)
    codes, byte = keep(x)
    got = keep_rows(x)
    assert torch.equal(_split(got, 1500, 1008)[0].cpu().long(), codes) and torch.equal(_split(got, 1500, 1008)[1].cpu().long(), byte)
    values = kept_values(got, 1008)
    assert values.isfinite().all() and torch.equal(values.double(), kept(x))


def test_ties_go_to_even(hip_lib):
    """Numbers that lie between two codes of their scale exactly, for every scale of four bits."""
    rows = []
    for four in range(8, 16):
        halves = torch.arange(0, 127, device="cuda", dtype=torch.float64) + 0.5
        ties = halves * four * 2.0 ** -8
        ties = ties[ties == ties.half().double()]
        pad = torch.zeros(-ties.numel() % 15, device="cuda", dtype=torch.float64)
        groups = torch.cat([ties, pad]).view(-1, 15)
        rows.append(torch.cat([torch.full((groups.shape[0], 1), 127 * four * 2.0 ** -8, device="cuda", dtype=torch.float64), groups], 1))
    x = torch.cat(rows)
    assert torch.equal(x.half().double(), x) and x.shape[0] > 8
    codes, byte = keep(x.half())
    got = keep_rows(x.half())
    assert torch.equal(_split(got, *x.shape)[0].cpu().long(), codes) and torch.equal(_split(got, *x.shape)[1].cpu().long(), byte)


def test_what_is_not_finite_spoils_its_group(hip_lib):
    x = torch.ones(3, 64, device="cuda").half()
    x[0, 17], x[1, 0], x[2, 63] = float("nan"), float("inf"), -float("inf")
    values = kept_values(keep_rows(x), 64)
    bad = torch.zeros(3, 64, dtype=torch.bool, device="cuda")
    bad[0, 16:32], bad[1, :16], bad[2, 48:] = True, True, True
    want = kept(torch.ones(3, 64, device="cuda").half())
    assert torch.equal(values.isnan(), bad) and torch.equal(values[~bad].double(), want[~bad])


def _near(got, want, terms, depth, results=torch.float16):
    """got, a sum of `depth` terms rounded in fp32 (each addition off by a unit of the sum's size at most, of a matrix instruction that may
    truncate; roundings of random sign add up as their root), then to its type."""
    off = 2.0 ** -23 * (4 + 2 * depth ** 0.5) * terms
    if results == torch.float16:
        off = off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25
    far = (got.double() - want).abs() - off
    return bool((far <= 0).all()) or float(far.max())


LINEAR = [(1, 16, 16), (63, 48, 48), (257, 64, 640), (811, 1152, 384), (1025, 240, 80), (3105, 384, 1536), (12421, 576, 192), (66001, 144, 48)]


@pytest.mark.parametrize("m,n,k", LINEAR)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_linear(hip_lib, m, n, k, dtype):
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = (_normal(gen, m, k) * torch.exp(_normal(gen, k))).half().requires_grad_()
    w, b = (_normal(gen, n, k) / k ** 0.5).to(dtype).requires_grad_(), _normal(gen, n).to(dtype).requires_grad_()
    dy = _normal(gen, m, n).half()
    y = checkpointed_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd, bd, dyd, kd = x.detach().double(), w.detach().half().double(), b.detach().half().double(), dy.double(), kept(x.detach())
    assert dw.dtype == db.dtype == dtype and dx.dtype == y.dtype == torch.float16
    assert _near(y, xd @ wd.t() + bd, xd.abs() @ wd.abs().t() + bd.abs(), k) is True
    assert _near(dx, dyd @ wd, dyd.abs() @ wd.abs(), n) is True
    assert _near(dw, dyd.t() @ kd, dyd.abs().t() @ kd.abs(), m, dtype) is True
    assert _near(db, dyd.sum(0), dyd.abs().sum(0), m, dtype) is True
    again = torch.autograd.grad(checkpointed_linear(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


def _exact_rows(gen, m, c):
    """fp16 rows that their kept form stands for exactly: whole numbers up to 127 of 2^-6, a 127 in every group."""
    codes = torch.randint(-127, 128, (m, c), device="cuda", generator=gen)
    codes[:, ::GROUP] = 127
    return (codes * 2.0 ** -6).half()


def _mlp(x, w1, b1, w2, b2):
    return gelu(x @ w1.t() + b1) @ w2.t() + b2


# (from 16,384 rows on: both layers in one kernel, for each width that has one, the last rows' wavefronts part full, with one row and empty)
MLP = [(1, 16, 16), (65, 48, 192), (811, 384, 1536), (1025, 80, 160), (12421, 96, 384), (40001, 48, 192), (16385, 64, 32), (16447, 80, 320),
       (20000, 96, 416), (60001, 128, 256), (57345, 160, 640), (49153, 192, 96), (16400, 48, 1024), (16400, 48, 1056)]


@pytest.mark.parametrize("m,c,hidden", MLP)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_mlp(hip_lib, m, c, hidden, dtype):
    """The formulas' gradients.  x and fc1's weight are such that the hidden layer's sums are fp16 numbers, so that what is kept of it is known to
    the bit; what is kept is not what it was."""
    gen = torch.Generator(device="cuda").manual_seed(m + c)
    x = (torch.randint(-15, 16, (m, c), device="cuda", generator=gen) * 0.125).half().requires_grad_()
    w1 = torch.zeros(hidden, c, device="cuda")
    at = torch.randint(0, c, (hidden, 4), device="cuda", generator=gen)
    w1.scatter_(1, at, torch.randint(-3, 4, (hidden, 4), device="cuda", generator=gen).float() * 0.25)
    b1 = torch.randint(-8, 9, (hidden,), device="cuda", generator=gen) * 0.03125
    w2, b2 = _normal(gen, c, hidden) / hidden ** 0.5, _normal(gen, c)
    params = [p.to(dtype).requires_grad_() for p in (w1, b1, w2, b2)]
    dy = _normal(gen, m, c).half()
    y = checkpointed_mlp(x, *params)
    dx, *grads = torch.autograd.grad(y, (x, *params), dy)
    assert all(g.dtype == dtype for g in grads)
    xd, dyd = x.detach().double(), dy.double()
    w1, b1, w2, b2 = (p.detach().half().double() for p in params)
    h = xd @ w1.t() + b1
    assert torch.equal(h.half().double(), h)
    hk, xk = kept(h.half()), kept(x.detach())
    assert not torch.equal(hk, h) or m == 1
    # half a step of fp16 for GELU's rows, whose fp32 is a 2^-20th off at most, and two for those of dh, whose slope is as exact
    eps = 2.0 ** -11
    u, uk = gelu(h), gelu(hk)
    off_u, off_uk = (eps * v.abs() + 2.0 ** -20 for v in (u, uk))
    dhidden = dyd @ w2
    dh = dhidden * gelu_slope(hk)
    off_dh = (2 * eps * dhidden.abs() + 2.0 ** -23 * (4 + 2 * c ** 0.5) * (dyd.abs() @ w2.abs())) * 1.13 + 2.0 ** -20 * dhidden.abs() + 2.0 ** -24

    def near(got, want, terms, depth, off):
        off = off + 2.0 ** -23 * (4 + 2 * depth ** 0.5) * terms
        off = off + eps * (want.abs() + off) + 2.0 ** -25 if got.dtype == torch.float16 else off
        return bool(((got.double() - want).abs() <= off).all())

    assert near(y, u @ w2.t() + b2, u.abs() @ w2.abs().t() + b2.abs(), hidden, off_u @ w2.abs().t())
    assert near(dx, dh @ w1, dh.abs() @ w1.abs(), hidden, off_dh @ w1.abs())
    assert near(grads[0], dh.t() @ xk, dh.abs().t() @ xk.abs(), m, off_dh.t() @ xk.abs())
    assert near(grads[1], dh.sum(0), dh.abs().sum(0), m, off_dh.sum(0))
    assert near(grads[2], dyd.t() @ uk, dyd.abs().t() @ uk.abs(), m, dyd.abs().t() @ off_uk)
    assert near(grads[3], dyd.sum(0), dyd.abs().sum(0), m, 0.0)
    again = torch.autograd.grad(checkpointed_mlp(x, *params), (x, *params), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, *grads)))


@pytest.mark.parametrize("m,c,hidden", [(1, 16, 16), (31, 48, 96), (33, 80, 176), (700, 48, 192), (811, 384, 768), (12421, 96, 384), (16385, 48, 160), (20001, 96, 384),
                                        (57345, 160, 320), (3000, 640, 1280)])
@pytest.mark.parametrize("dx_too", [True, False])
def test_bias_behind_gelu_is_summed_before_rounding(hip_lib, m, c, hidden, dx_too):
    """The hidden layer's gradients are fp16 numbers for the products behind them alone: db1 is the sum of what they are rounded from.  Numbers of which
    each is half a step above an fp16 number all round the same way: db1 of rounded ones is 2^-12 of it off or more, that of the sums an fp32 one's error."""
    gen = torch.Generator(device="cuda").manual_seed(m + c)
    x = torch.zeros(m, c, device="cuda").half().requires_grad_(dx_too)
    b1 = torch.full((hidden,), 12.0, device="cuda")                    # GELU's slope there is 1 to fp32
    # dy w2: 1 + 2^-11 + 2^-13, which fp16 rounds to 1 + 2^-10
    w2 = torch.zeros(c, hidden, device="cuda")
    w2[0], w2[1], w2[2] = 1.0, 2.0 ** -11, 2.0 ** -13
    dy = torch.zeros(m, c, device="cuda").half()
    dy[:, :3] = 1.0
    sign = torch.randint(0, 2, (m, 1), device="cuda", generator=gen) * 2 - 1
    w1, b2 = torch.zeros(hidden, c, device="cuda"), torch.zeros(c, device="cuda")
    params = [p.requires_grad_() for p in (w1, b1, w2, b2)]
    for rows in (dy, dy * sign):
        y = checkpointed_mlp(x, *params)
        db1 = torch.autograd.grad(y, params[1:2] if not dx_too else [x, params[1]], rows)[-1]
        want = (1 + 2.0 ** -11 + 2.0 ** -13) * rows[:, 0].double().sum()
        # sums of some hundred groups of 32 equal numbers, whose roundings are a unit of the sum so far each
        assert bool(((db1.double() - want).abs() <= 2.0 ** -23 * (8 + m / 256) * m ** 0.5 + 2.0 ** -23 * want.abs() * 8).all()), (db1[:3], want)


def test_gradients_against_differences(hip_lib):
    """Where what is kept is what was there, the gradients are those of the layers: against differences in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    m, c, hidden = 40, 32, 64
    x = _exact_rows(gen, m, c)
    w1 = torch.eye(c, device="cuda").repeat(hidden // c, 1)       # the hidden layer's rows are x's, twice
    params = [w1, torch.zeros(hidden, device="cuda"), (_normal(gen, c, hidden) / 8).half().float(), _normal(gen, c).half().float()]
    assert torch.equal(kept_values(keep_rows(x), c), x)
    dy = _normal(gen, m, c).half()
    leaves = [x.clone().requires_grad_(), *(p.clone().requires_grad_() for p in params)]
    grads = torch.autograd.grad(checkpointed_mlp(*leaves), leaves, dy)
    doubles = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        direction = _normal(gen, *g.shape).double()
        step = 1e-5
        ends = [_mlp(*(t + s * step * direction if j == i else t for j, t in enumerate(doubles))) for s in (1, -1)]
        along = float(((ends[0] - ends[1]) * dy.double()).sum() / (2 * step))
        # three roundings to fp16 on the way to a gradient, of random sign along a direction
        assert abs(float((g.double() * direction).sum()) - along) <= 4 * 2.0 ** -11 * float((g.double() * direction).norm()) + 1e-6 * abs(along)
    w, b = (t.clone().requires_grad_() for t in (params[2].t().contiguous(), params[1]))
    xs = leaves[0]
    grads = torch.autograd.grad(checkpointed_linear(xs, w, b), (xs, w, b), F.pad(dy, (0, hidden - c)))
    want = torch.autograd.grad(F.linear(*(doubles_of := [t.detach().double().requires_grad_() for t in (xs, w, b)])), doubles_of, F.pad(dy, (0, hidden - c)).double())
    assert all(float((g.double() - v).norm()) <= 2.0 ** -11 * float(v.norm()) for g, v in zip(grads, want))


@pytest.mark.parametrize("which", range(1, 32, 2))
def test_gradients_that_are_wanted(hip_lib, which):
    """Any of the inputs may need none; those that do get the same gradients, and nothing else is kept."""
    gen = torch.Generator(device="cuda").manual_seed(which)
    tensors = [_normal(gen, 70, 32).half(), _normal(gen, 64, 32) / 6, _normal(gen, 64), _normal(gen, 32, 64) / 8, _normal(gen, 32)]
    dy = _normal(gen, 70, 32).half()
    for flip in (0, 31):
        needs = [bool((which ^ flip) >> i & 1) for i in range(5)]
        if not any(needs):
            continue
        every = [t.clone().requires_grad_() for t in tensors]
        want = torch.autograd.grad(checkpointed_mlp(*every), every, dy)
        some = [t.clone().requires_grad_(need) for t, need in zip(tensors, needs)]
        got = torch.autograd.grad(checkpointed_mlp(*some), [t for t, need in zip(some, needs) if need], dy)
        assert all(torch.equal(g, w) for g, w in zip(got, (w for w, need in zip(want, needs) if need)))
        if any(needs[:3]):
            every, some = ([t[0], t[1], t[2]] for t in (every, some))
            dz = _normal(gen, 70, 64).half()
            want = torch.autograd.grad(checkpointed_linear(*every), every, dz)
            got = torch.autograd.grad(checkpointed_linear(*some), [t for t, need in zip(some, needs) if need], dz)
            assert all(torch.equal(g, w) for g, w in zip(got, (w for w, need in zip(want, needs) if need)))


@pytest.mark.parametrize("m,c,hidden", [(16391, 64, 256), (57347, 160, 320)])
def test_gradients_that_are_wanted_of_many_rows(hip_lib, m, c, hidden):
    """... where both layers are one kernel, which keeps a hidden layer or not, and dx is what its backward is for."""
    gen = torch.Generator(device="cuda").manual_seed(c)
    tensors = [_normal(gen, m, c).half(), _normal(gen, hidden, c) / c ** 0.5, _normal(gen, hidden), _normal(gen, c, hidden) / hidden ** 0.5, _normal(gen, c)]
    dy = _normal(gen, m, c).half()
    with torch.no_grad():
        y = checkpointed_mlp(*tensors)
    want = None
    for needs in ((1, 1, 1, 1, 1), (1, 0, 0, 0, 0), (0, 0, 0, 0, 1), (0, 0, 0, 1, 0), (0, 1, 0, 0, 0), (1, 0, 0, 1, 0)):
        some = [t.clone().requires_grad_(bool(need)) for t, need in zip(tensors, needs)]
        out = checkpointed_mlp(*some)
        assert torch.equal(out, y)
        got = torch.autograd.grad(out, [t for t, need in zip(some, needs) if need], dy)
        if want is None:
            want = got
            continue
        for g, w in zip(got, (w for w, need in zip(want, needs) if need)):
            # without dx the hidden layer's gradient is a product of its own, whose sums have another order: a rounding to fp16 each
            assert torch.equal(g, w) or (not needs[0] and float((g - w).norm()) <= 2.0 ** -11 * float(w.norm()))


@pytest.mark.parametrize("m,n,k,rows", [(70, 144, 48, 48), (5000, 480, 160, 160), (333, 32, 64, 32), (50, 64, 16, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_scaled_rows(hip_lib, m, n, k, rows, dtype):
    """The layer of parameters whose first rows were multiplied by a factor, with the gradients of those that were not."""
    gen, factor = torch.Generator(device="cuda").manual_seed(m), 8 ** -0.5
    x, dy = _normal(gen, m, k).half(), _normal(gen, m, n).half()
    weight, bias = (_normal(gen, n, k) / k ** 0.5).to(dtype), _normal(gen, n).to(dtype)
    scale = torch.ones(n, device="cuda")
    scale[:rows] = torch.tensor(factor)
    given = [t.clone().requires_grad_() for t in (x, weight, bias)]
    y = checkpointed_linear(*given, (rows, factor))
    got = torch.autograd.grad(y, given, dy)
    plain = [t.clone().requires_grad_() for t in (x, weight.float() * scale.unsqueeze(1), bias.float() * scale)]
    want_y = checkpointed_linear(*plain)
    want = list(torch.autograd.grad(want_y, plain, dy))
    want[1], want[2] = (want[1] * scale.unsqueeze(1)).to(dtype), (want[2] * scale).to(dtype)
    assert torch.equal(y, want_y) and all(torch.equal(g, w) for g, w in zip(got, want))
    for bad in ((8, factor), (-16, factor), (n + 16, factor)):
        with pytest.raises(ValueError):
            checkpointed_linear(x, weight, bias, bad)


@pytest.mark.parametrize("m,c,hidden", [(100, 48, 192), (16400, 48, 192), (50000, 160, 640)])
def test_mlp_of_rows_that_are_not_finite(hip_lib, m, c, hidden):
    """A row that is not finite, or whose hidden layer is not, makes its own results and the parameters' gradients NaN, and no other row's."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    params = [_normal(gen, hidden, c) / c ** 0.5, _normal(gen, hidden), _normal(gen, c, hidden) / hidden ** 0.5, _normal(gen, c)]
    x, dy = _normal(gen, m, c).half(), _normal(gen, m, c).half()
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[3, 64, m - 1]] = True
    results = []
    for rows in (x, x.clone()):
        if results:
            rows[3, 5], rows[64, 0], rows[m - 1] = float("nan"), float("inf"), 60000.0
        leaves = [rows.clone().requires_grad_(), *(p.clone().requires_grad_() for p in params)]
        y = checkpointed_mlp(*leaves)
        results.append((y, *torch.autograd.grad(y, leaves, dy)))
    (y, dx, *grads), (bad_y, bad_dx, *bad_grads) = results
    assert torch.equal(y[~bad], bad_y[~bad]) and torch.equal(dx[~bad], bad_dx[~bad]) and y.isfinite().all() and dx.isfinite().all()
    assert bad_y[bad].isnan().all() and bad_dx[bad].isnan().all()
    assert all(g.isnan().all() for g in bad_grads[:1]) and torch.equal(bad_grads[3], grads[3])


def test_without_biases_and_mixed_types(hip_lib):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, dy = _normal(gen, 100, 48).half(), _normal(gen, 100, 48).half()
    w1, w2 = (_normal(gen, 96, 48) / 7).half().requires_grad_(), (_normal(gen, 48, 96) / 10).requires_grad_()
    b1 = torch.zeros(96, device="cuda", requires_grad=True)
    b2 = torch.zeros(48, device="cuda").half().requires_grad_()
    with_zeros = torch.autograd.grad(checkpointed_mlp(x, w1, b1, w2, b2), (w1, w2, b1, b2), dy)
    without = torch.autograd.grad(checkpointed_mlp(x, w1, None, w2, None), (w1, w2), dy)
    assert [g.dtype for g in with_zeros] == [torch.float16, torch.float32, torch.float32, torch.float16]
    assert all(torch.equal(a, b) for a, b in zip(with_zeros, without))
    bias = torch.zeros(96, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(checkpointed_linear(x, w1, bias), (w1, bias), _normal(gen, 100, 96).half())
    assert dw.dtype == torch.float16 and db.dtype == torch.float32
    # strided and shifted operands, broadcast gradients
    wide = _normal(gen, 100, 97).half()
    shifted = wide[:, 1:49].requires_grad_()
    assert torch.equal(checkpointed_linear(shifted, w1, None), checkpointed_linear(shifted.contiguous(), w1, None))
    y = checkpointed_linear(shifted, w1, None)
    assert torch.equal(torch.autograd.grad(y.sum(), w1)[0], torch.autograd.grad(checkpointed_linear(shifted, w1, None), w1, torch.ones_like(y))[0])


def test_no_rows(hip_lib):
    x, w, b = torch.empty(0, 32, device="cuda").half().requires_grad_(), torch.randn(16, 32, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    y = checkpointed_linear(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 16) and not w.grad.any() and not b.grad.any() and x.grad.shape == (0, 32)
    y = checkpointed_mlp(x, w, b, torch.randn(32, 16, device="cuda", requires_grad=True), None)
    y.sum().backward()
    assert y.shape == (0, 32) and kept_values(keep_rows(x), 32).shape == (0, 32)


def test_memory_that_is_kept(hip_lib):
    """1.0625 bytes a number of x, and of x and the hidden layer, beside the weights' copies.  (torch's allocator does not split a block
    for a remainder of up to 1 MiB: at most two blocks are held, and the result's.)"""
    m, c, hidden = 100_000, 96, 384
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = _normal(gen, m, c).half()
    w1, w2 = _normal(gen, hidden, c).requires_grad_(), _normal(gen, c, hidden).requires_grad_()
    for call, numbers, results in ((lambda: checkpointed_linear(x, w1, None), m * c, m * hidden), (lambda: checkpointed_mlp(x, w1, None, w2, None), m * (c + hidden), m * c)):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = call()
        held = torch.cuda.memory_allocated() - before - 2 * results
        assert numbers * 17 // 16 <= held <= numbers * 17 // 16 + 8 * c * hidden + 3 * 2 ** 20
        with torch.no_grad():
            before = torch.cuda.memory_allocated()
            z = call()
            assert torch.cuda.memory_allocated() - before <= 2 * results + 2 ** 20 and torch.equal(z, y)
        del y, z


def test_training_pass_captured(hip_lib):
    gen = torch.Generator(device="cuda").manual_seed(3)
    m, c, hidden = 2000, 96, 384
    values = [(_normal(gen, m, c).half(), _normal(gen, m, c).half()) for _ in range(3)]
    params = [_normal(gen, hidden, c) / 10, _normal(gen, hidden), _normal(gen, c, hidden) / 20, _normal(gen, c)]

    def run(x, dy, leaves):
        y = checkpointed_mlp(x, *leaves)
        return (y.detach(), *torch.autograd.grad(y, (x, *leaves), dy))

    wants = [[t.clone() for t in run(x.clone().requires_grad_(), dy, [p.clone().requires_grad_() for p in params])] for x, dy in values]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [p.clone().requires_grad_() for p in params]
        x, dy = values[0][0].clone().requires_grad_(), values[0][1].clone()
        run(x, dy, leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run(x, dy, leaves)
    torch.cuda.synchronize()
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            x.copy_(values[i][0])
        dy.copy_(values[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wants[i]))


def test_refusals(hip_lib):
    x = torch.randn(4, 32, device="cuda").half()
    w, b = torch.randn(16, 32, device="cuda"), torch.zeros(16, device="cuda")
    back = torch.randn(32, 16, device="cuda")
    for bad in (lambda: checkpointed_linear(x.float(), w, b), lambda: checkpointed_linear(x[0], w, b), lambda: checkpointed_linear(x, w[:, :16], b),
                lambda: checkpointed_linear(x, w[:8], None), lambda: checkpointed_linear(x, w, b[:8]), lambda: checkpointed_linear(x, w.double(), b),
                lambda: checkpointed_linear(x, w.cpu(), b), lambda: checkpointed_linear(x.cpu(), w, b),
                lambda: checkpointed_linear(x[:, :24].contiguous(), w[:, :24].contiguous(), b),
                lambda: checkpointed_mlp(x, w, b, back[:16], None), lambda: checkpointed_mlp(x, w, b, back.t(), None),
                lambda: keep_rows(x.float()), lambda: keep_rows(x[:, :24]), lambda: kept_values(torch.zeros(33, dtype=torch.uint8, device="cuda"), 32),
                lambda: kept_values(torch.zeros(34, dtype=torch.uint8, device="cuda"), 24), lambda: kept_values(x, 32)):
        with pytest.raises(ValueError):
            bad()
    w.requires_grad_()
    dw, = torch.autograd.grad(checkpointed_linear(x, w, b), w, torch.ones(4, 16, device="cuda").half(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), w)


@pytest.mark.parametrize("c,hidden", [(80, 640), (208, 640)])
def test_offsets_beyond_32_bits(hip_lib, c, hidden):
    """A hidden layer of more than 2^31 numbers, in one kernel and in two: the last rows' results are those of the same rows by themselves, and gradients
    of parameters that come of these rows alone theirs."""
    gen = torch.Generator(device="cuda").manual_seed(c)
    m, last = 2 ** 31 // hidden + 40001, 40000
    x, dy = torch.zeros(m, c, device="cuda", dtype=torch.float16), torch.zeros(m, c, device="cuda", dtype=torch.float16)
    x[-last:], dy[-last:] = _normal(gen, last, c).half(), _normal(gen, last, c).half()
    params = [(_normal(gen, hidden, c) / c ** 0.5).requires_grad_(), _normal(gen, hidden).requires_grad_(),
              (_normal(gen, c, hidden) / hidden ** 0.5).requires_grad_(), _normal(gen, c).requires_grad_()]

    def passed(x, dy):
        x = x.requires_grad_()
        y = checkpointed_mlp(x, *params)
        return (y[-last:].clone(), *(g[-last:].clone() if i == 0 else g for i, g in enumerate(torch.autograd.grad(y, [x, *params], dy))))

    got, want = passed(x, dy), passed(x[-last:].detach().clone(), dy[-last:].clone())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # other shares of the rows: the sums of 40,000 products in another order, some of them with zeros in between
    assert all(float((g - w).norm()) <= 2.0 ** -18 * float(w.norm()) for g, w in zip(got[2:], want[2:]))


def test_form_of_more_than_32_bits_of_bytes(hip_lib):
    """Rows whose kept form has more than 2^31 bytes: the last ones' are those of the same rows by themselves, both ways."""
    c, last = 640, 5000
    m = (2 ** 31 // (c + c // GROUP)) + last
    x = torch.zeros(m, c, device="cuda", dtype=torch.float16)
    x[-last:] = _normal(torch.Generator(device="cuda").manual_seed(9), last, c).half()
    got, tail = keep_rows(x), keep_rows(x[-last:].clone())
    assert got.numel() > 2 ** 31
    assert torch.equal(got[(m - last) * c:m * c], tail[:last * c]) and torch.equal(got[-last * (c // GROUP):], tail[last * c:])
    values = kept_values(got, c)
    assert values.shape == x.shape and torch.equal(values[-last:], kept_values(tail, c)) and not values[:-last].any()


def test_factor_that_is_trained(hip_lib):
    """The factor of scaled outputs is a number: one that requires a gradient is refused, not dropped."""
    import numpy as np
    x, w = torch.randn(4, 32, device="cuda").half(), torch.randn(48, 32, device="cuda", requires_grad=True)
    factor = torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        checkpointed_linear(x, w, None, (16, factor))
    want = checkpointed_linear(x, w, None, (16, 0.5))
    with torch.no_grad():
        assert torch.equal(checkpointed_linear(x, w, None, (16, factor)), want)
    assert torch.equal(checkpointed_linear(x, w, None, (np.int64(16), factor.detach())), want)
    for rows in (16.0, torch.tensor(16), "16", None):
        with pytest.raises(ValueError):
            checkpointed_linear(x, w, None, (rows, 0.5))


def test_how_far_the_form_is_off_at_both_ends(hip_lib):
    """Every fp16 size as its group's largest number, beside numbers below it.  A scale s is the smallest of four bits, and of whole 2^-24, that reaches the
    largest number a with 127 codes: s <= 1.125 a / 127 from 8 2^-24 on, less than a / 127 + 2^-24 below, and a number is off by s / 2 at most.  Above 127 512
    = 65,024 s is 576 and codes end at 113, for 65,088: up to 65,504 is 416 off."""
    sizes = torch.arange(0, 0x7c00, dtype=torch.int16, device="cuda").view(torch.float16)
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = (sizes.float().unsqueeze(1) * torch.rand(sizes.numel(), GROUP, device="cuda", generator=gen)).half()
    x[:, 0], x[:, 1] = sizes, -sizes
    x = torch.minimum(x, sizes.unsqueeze(1))
    off = (kept_values(keep_rows(x), GROUP).double() - x.double()).abs()
    most = x.double().abs().amax(1, keepdim=True)
    assert torch.equal(most[:, 0], sizes.double())
    unit = 2.0 ** -24
    bound = 0.5 * torch.where(most > 127 * 8 * unit, 1.125 * most / 127, most / 127 + unit)
    top = most > 65024
    assert int(top.sum()) == 15 and bool((off <= torch.where(top, 416.0, bound)).all())
    assert float(off[top[:, 0]].max()) == 416 and float((off / bound)[~top[:, 0]].max()) > 0.85
    small = (most[:, 0] > 127 * unit) & (most[:, 0] < 254 * unit)      # ... where the scale is a whole 2^-24: up to twice a 254th
    assert float((off / (most / 254))[small].max()) > 1.5
