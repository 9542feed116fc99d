"""Swin blocks with rows in eight bits: at inference the stage's one call against the operators one after the other, in training what is kept
and the gradients that come of it."""
import pytest
import torch

from swin3d_amd import _lib, add_layernorm, encoder, synth
from swin3d_amd.eight_bits import add_norm_int8, linear_int8, mlp_int8, quantize_rows
from swin3d_amd.encoder import eight_bit_checkpoints, eight_bit_inference
from swin3d_amd.sparse_dl.attn.attn_coff import IndexMode, PosEmb, PrecisionMode, SelfAttnAIOFunction, TableDims

pytestmark = pytest.mark.gpu


def _stage(heads, dim, window, mode, voxels, depth=3, seed=5):
    dev = torch.device("cuda")
    scene = synth.make_room((3.0, 3.0, 2.0) if voxels < 10000 else (6.0, 5.0, 2.5), 4, voxels, seed=seed)
    coords = torch.from_numpy(scene.coords).to(dev)
    signals = torch.from_numpy(synth.encoder_inputs(scene)[1].copy()).to(dev)
    torch.manual_seed(1)
    stage = encoder.Stage(heads * dim, depth, heads, window, 4, downsample=False, cRSE="XYZ_RGB_NORM", fp16_mode=mode).to(dev)
    for name, p in stage.named_parameters():
        if "table" in name or "bias" in name:
            torch.nn.init.normal_(p, std=0.1)
    return stage, coords, signals, torch.randn(coords.shape[0], heads * dim, device=dev)


def _run(stage, coords, signals, feats, plan=None):
    with torch.autocast("cuda", dtype=torch.float16):
        return stage(encoder.SparseVoxels(coords, feats, 1), signals, plan)[0].feats


def _one_by_one(stage, feats, args):
    """The blocks of a stage on the operators."""
    pending = None
    for i, block in enumerate(stage.blocks):
        attn, a = block.attn, args[i % len(args)]
        feats, rows = add_norm_int8(feats, pending, block.norm1)
        weight, bias = quantize_rows(attn.qkv.weight), attn.qkv.bias.clone()
        weight.scales[:attn.dim] *= attn.scale
        bias[:attn.dim] *= attn.scale
        qkv = linear_int8(rows, weight, bias).view(-1, 3, attn.num_heads, attn.head_dim)
        tables = [attn._flat_table(kind).half() for kind in ("query", "key", "value")]
        with torch.autocast("cuda", dtype=torch.float16):
            out = SelfAttnAIOFunction.apply(*qkv.unbind(1), *tables, attn.table_sizes, [None, a[3], None, a[4], a[5], a[8]], PosEmb.SEPARATE,
                                            TableDims.D0, IndexMode.INDIRECT, PrecisionMode.HALF_ALL)
        branch = linear_int8(quantize_rows(out.reshape(-1, attn.dim)), quantize_rows(block.attn.proj.weight), block.attn.proj.bias)
        mlp, (m, c), hidden = block.mlp, feats.shape, block.mlp.fc1.out_features
        if m >= 16384 and m >= 192 * c and c in (48, 64, 80, 96, 128, 160, 192) and hidden <= 1024:      # both layers as one kernel in fp16
            feats, normed = add_layernorm(feats, branch, block.norm2)
            params = [p.half() for p in (mlp.fc1.weight, mlp.fc1.bias, mlp.fc2.weight, mlp.fc2.bias)]
            pending = torch.empty(m, c, device="cuda", dtype=torch.float16)
            _lib.check(_lib.lib().s3d_mlp(normed.data_ptr(), *(p.data_ptr() for p in params), pending.data_ptr(), m, c, hidden, _lib.stream(feats.device)), "s3d_mlp")
            continue
        feats, rows = add_norm_int8(feats, branch, block.norm2)
        pending = mlp_int8(rows, quantize_rows(mlp.fc1.weight), mlp.fc1.bias, quantize_rows(mlp.fc2.weight), mlp.fc2.bias)
    return feats + pending.float()


@pytest.mark.parametrize("heads,dim,window,voxels", [(6, 8, 5, 5000), (5, 16, 7, 3000), (1, 16, 5, 7), (6, 8, 5, 40000)])
def test_blocks_at_inference(hip_lib, heads, dim, window, voxels):
    stage, coords, signals, feats = _stage(heads, dim, window, 2, voxels)
    assert voxels != 40000 or coords.shape[0] >= 16384      # (its MLPs run as one kernel)
    stage.eval()
    with torch.no_grad():
        plan = stage.plan(coords, 1, signals)
        before, given = _run(stage, coords, signals, feats, plan), feats.clone()
        assert eight_bit_inference(stage) is stage
        got = _run(stage, coords, signals, feats, plan)
        assert torch.equal(feats, given) and torch.equal(_run(stage, coords, signals, feats, plan), got)
        assert torch.equal(got, _one_by_one(stage, feats, plan[0]))
        # a row's step is a 127th of its largest number, some four times its spread, so a layer's input is off by 1 % of the row's spread, its
        # weight likewise; four layers a block, whose branches are smaller than the stream, of random sign
        assert not torch.equal(got, before) and float((got - before).norm() / before.norm()) < 0.03
        # single blocks, and a stage of which some blocks are in fp16
        single = feats
        for block, a in zip(stage.blocks, (plan[0][i % len(plan[0])] for i in range(3))):
            with torch.autocast("cuda", dtype=torch.float16):
                single = block(single, a)
        assert float((single - got).norm() / got.norm()) < 2.0 ** -10
        stage.blocks[1].eight_bit_rows = False
        mixed = _run(stage, coords, signals, feats, plan)
        assert not torch.equal(mixed, got) and float((mixed - before).norm() / before.norm()) < 0.03
        # a weight that changes is read again; off, the blocks are what they were
        eight_bit_inference(stage)
        stage.blocks[0].mlp.fc1.weight.mul_(1.5)
        changed = _run(stage, coords, signals, feats, plan)
        assert not torch.equal(changed, got) and torch.equal(changed, _one_by_one(stage, feats, plan[0]))
        stage.blocks[0].mlp.fc1.weight.div_(1.5)
        eight_bit_inference(stage, False)
        assert torch.equal(_run(stage, coords, signals, feats, plan), before)


def test_codes_of_weights_on_other_streams_and_in_graphs(hip_lib):
    """Codes are made on the stream that reads them; a graph's are made by its replays, from the parameters of then, and read by nobody else."""
    stage, coords, signals, feats = _stage(6, 8, 5, 2, 3000, depth=2)
    stage.eval()
    eight_bit_inference(stage)
    with torch.no_grad():
        plan = stage.plan(coords, 1, signals)
        want = _run(stage, coords, signals, feats, plan)
        own = stage._s3d_blocks
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            assert torch.equal(_run(stage, coords, signals, feats, plan), want) and stage._s3d_blocks is not own
            stage._s3d_blocks = None
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = _run(stage, coords, signals, feats, plan)
            assert stage._s3d_blocks is None
        torch.cuda.synchronize()
        assert torch.equal(_run(stage, coords, signals, feats, plan), want)      # before the first replay
        for factor in (1.0, 1.5, 1.0):
            stage.blocks[0].mlp.fc1.weight.mul_(factor)
            eager = _run(stage, coords, signals, feats, plan)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, eager) and torch.equal(got, want) == (factor == 1.0 and torch.equal(eager, want))
            stage.blocks[0].mlp.fc1.weight.div_(factor)


def test_without_biases_and_hooks(hip_lib):
    stage, coords, signals, feats = _stage(6, 8, 5, 2, 3000, depth=2)
    stage.eval()
    eight_bit_inference(stage)
    calls = []
    with torch.no_grad():
        plan = stage.plan(coords, 1, signals)
        with_biases = _run(stage, coords, signals, feats, plan)
        handle = stage.blocks[0].mlp.act.register_forward_hook(lambda *_: calls.append(1))
        _run(stage, coords, signals, feats, plan)
        assert calls            # a layer that is watched is called
        handle.remove()
        for block in stage.blocks:
            for layer in (block.attn.qkv, block.attn.proj, block.mlp.fc1, block.mlp.fc2):
                layer.bias.zero_()
        zeros = _run(stage, coords, signals, feats, plan)
        for block in stage.blocks:
            for layer in (block.attn.qkv, block.attn.proj, block.mlp.fc1, block.mlp.fc2):
                layer.bias = None
        assert torch.equal(_run(stage, coords, signals, feats, plan), zeros) and not torch.equal(zeros, with_biases)


def test_widths_that_eight_bits_do_not_come_in(hip_lib):
    stage = encoder.Stage(24, 1, 3, 5, 4, downsample=False, cRSE="XYZ_RGB_NORM", fp16_mode=2)
    for switch in (eight_bit_inference, eight_bit_checkpoints):
        with pytest.raises(ValueError):
            switch(stage)
    assert eight_bit_inference(torch.nn.Linear(3, 3)) is not None


def _gradients(stage, coords, signals, feats, plan):
    x = feats.clone().requires_grad_()
    out = _run(stage, coords, signals, x, plan)
    grad = torch.randn(out.shape, device=out.device, generator=torch.Generator(device="cuda").manual_seed(1))
    named = dict(stage.named_parameters())
    return out.detach(), dict(zip(["x", *named], torch.autograd.grad(out, [x, *named.values()], grad)))


@pytest.mark.parametrize("heads,dim,window,mode,voxels", [(6, 8, 5, 2, 5000), (6, 8, 5, 1, 5000), (5, 16, 7, 1, 3000), (6, 8, 5, 1, 30000)])
def test_blocks_in_training(hip_lib, heads, dim, window, mode, voxels):
    stage, coords, signals, feats = _stage(heads, dim, window, mode, voxels, depth=2)
    plan = stage.plan(coords, 1, signals)
    out, want = _gradients(stage, coords, signals, feats, plan)
    assert eight_bit_checkpoints(stage) is stage
    kept_out, got = _gradients(stage, coords, signals, feats, plan)
    # the forward has the layers' operations in other orders of summation: a rounding to fp16 here and there
    assert float((kept_out - out).norm() / out.norm()) < 2.0 ** -10
    # A kept number is off by half a step at most, by a third of one in the mean: 0.5 % of its group's spread (the largest of sixteen is 1.8 times
    # that, the scale up to an eighth more).  Two blocks add two of these to each of their dense layers.
    for name, g in got.items():
        assert float((g - want[name]).norm()) <= 0.015 * float(want[name].norm()), name
    again = _gradients(stage, coords, signals, feats, plan)[1]
    assert all(torch.equal(again[n], got[n]) for n in got if "table" not in n)
    eight_bit_checkpoints(stage, False)
    back_out, back = _gradients(stage, coords, signals, feats, plan)
    assert torch.equal(back_out, out) and all(torch.equal(back[n], want[n]) for n in want if "table" not in n)


def test_memory_of_a_block_in_training(hip_lib):
    """Some 22 bytes a voxel and channel in place of 36."""
    stage, coords, signals, feats = _stage(6, 8, 5, 1, 60000, depth=4)
    plan = stage.plan(coords, 1, signals)
    held = []
    for on in (False, True):
        eight_bit_checkpoints(stage, on)
        _run(stage, coords, signals, feats.clone().requires_grad_(), plan)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = _run(stage, coords, signals, feats.clone().requires_grad_(), plan)
        held.append((torch.cuda.memory_allocated() - before) / (4 * feats.numel()))
        del out
    assert held[1] < 0.7 * held[0] and 18 < held[1] < 26 and 32 < held[0] < 40, held


def test_a_network_with_both(hip_lib):
    torch.manual_seed(0)
    model = encoder.Swin3DUNet(depths=[2, 2, 2], channels=[16, 32, 64], num_heads=[2, 2, 4], window_sizes=[5, 5, 5], quant_size=4, num_layers=3,
                               num_classes=13, upsample="linear_attn", in_channels=9, cRSE="XYZ_RGB_NORM", fp16_mode=1).cuda()
    eight_bit_checkpoints(eight_bit_inference(model))
    scene = synth.make_room((3.0, 3.0, 2.0), 4, 6000, seed=2)
    feats, signals = (torch.from_numpy(a.copy()).cuda() for a in synth.encoder_inputs(scene))
    voxels = encoder.SparseVoxels(torch.from_numpy(scene.coords).cuda(), feats, 1)
    optimizer = torch.optim.SGD(model.parameters(), lr=1e-3)
    for _ in range(2):
        with torch.autocast("cuda", dtype=torch.float16):
            logits = model(voxels, signals)
        loss = torch.nn.functional.cross_entropy(logits.float(), torch.arange(logits.shape[0], device="cuda") % 13)
        optimizer.zero_grad()
        loss.backward()
        assert all(p.grad is None or p.grad.isfinite().all() for p in model.parameters())
        optimizer.step()
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        got = model(voxels, signals)
        want = eight_bit_inference(model, False)(voxels, signals)
    assert got.isfinite().all() and not torch.equal(got, want) and float((got - want).norm() / want.norm()) < 0.05


def test_blocks_that_cannot_any_more_are_what_they_were(hip_lib):
    """A block that turns to fp16_mode 0 behind the switch runs as without it, to the bit, among others and by itself, and leaves its input alone."""
    stage, coords, signals, feats = _stage(6, 8, 5, 2, 3000)
    stage.eval()
    with torch.no_grad():
        plan = stage.plan(coords, 1, signals)
        for changed in ([0, 1, 2], [1]):
            eight_bit_inference(stage)
            for i in changed:
                stage.blocks[i].attn.fp16_mode = 0
            given, got = feats.clone(), _run(stage, coords, signals, feats, plan)
            assert torch.equal(feats, given)
            for i in changed:
                stage.blocks[i].eight_bit_rows = False
            assert torch.equal(_run(stage, coords, signals, feats, plan), got)
            for block in stage.blocks:
                block.attn.fp16_mode = 2


def test_scale_that_is_trained(hip_lib):
    """A block whose attention's scale is a tensor has its gradient, with the switch as without."""
    stage, coords, signals, feats = _stage(6, 8, 5, 1, 3000, depth=1)
    plan, attn, given = stage.plan(coords, 1, signals), stage.blocks[0].attn, []
    for on in (False, True):
        eight_bit_checkpoints(stage, on)
        attn.scale = torch.tensor(8 ** -0.5, device="cuda", requires_grad=True)
        out = _run(stage, coords, signals, feats, plan)
        grad, = torch.autograd.grad(out.square().sum(), attn.scale)
        given.append((out.detach(), grad))
    assert all(torch.equal(a, b) for a, b in zip(*given)) and float(given[0][1].abs()) > 0
