"""What the dense layers in eight bits refuse, without a device: shapes, types and null pointers at the C entry points, CPU tensors and
other objects at the Python ones; and the statement of the kept form that the GPU tests use."""
import ctypes

import pytest
import torch

from eight_bit_reference import keep, kept, kept_scales
from swin3d_amd import eight_bits, encoder
from swin3d_amd.eight_bits import Int8Rows


def _refused(lib, status, text):
    assert status < 0 and text in lib.s3d_last_error_string().decode()


def test_c_entry_points_refuse(hip_lib):
    lib, one, dtypes = hip_lib, ctypes.c_void_p(16), (ctypes.c_int32 * 4)()
    for n, c in ((-1, 48), (4, 0), (4, 6), (4, 8196), (1 << 31, 48)):
        _refused(lib, lib.s3d_add_norm_int8(one, None, 0, one, one, 1e-5, 0, None, one, one, n, c, None), "s3d_add_norm_int8: N=")
        _refused(lib, lib.s3d_quantize_rows(one, 0, one, one, n, c, None), "s3d_quantize_rows: N=")
        _refused(lib, lib.s3d_int8_values(one, one, one, 0, n, c, None), "s3d_int8_values: N=")
    _refused(lib, lib.s3d_add_norm_int8(one, one, 7, one, one, 1e-5, 0, None, one, one, 4, 48, None), "residual_dtype 7")
    _refused(lib, lib.s3d_quantize_rows(one, 2, one, one, 4, 48, None), "dtype 2")
    _refused(lib, lib.s3d_int8_values(one, one, one, 2, 4, 48, None), "dtype 2")
    _refused(lib, lib.s3d_add_norm_int8(None, None, 0, one, one, 1e-5, 0, None, one, one, 4, 48, None), "null")
    _refused(lib, lib.s3d_quantize_rows(one, 0, None, one, 4, 48, None), "null")
    _refused(lib, lib.s3d_int8_values(one, None, one, 0, 4, 48, None), "null")
    for m, n, k in ((-1, 16, 16), (4, 12, 16), (4, 16, 24), (4, 0, 16), (4, 16, 0), (4, 16, 65552), (1 << 31, 16, 16)):
        _refused(lib, lib.s3d_linear_int8(one, one, one, one, None, one, m, n, k, 0, None), "s3d_linear_int8: M=")
    _refused(lib, lib.s3d_linear_int8(one, None, one, one, None, one, 4, 16, 16, 0, None), "null")
    for m, c, hidden in ((-1, 16, 16), (4, 24, 16), (4, 16, 24), (4, 16, 8208), (4, 8208, 16)):
        _refused(lib, lib.s3d_mlp_int8(*[one] * 9, m, c, hidden, one, 1 << 30, None), "s3d_mlp_int8: M=")
        assert lib.s3d_mlp_int8_workspace_bytes(m, c, hidden) == 0
    _refused(lib, lib.s3d_mlp_int8(*[one] * 9, 4, 640, 2560, one, 16, None), "workspace 16 B")
    # both layers in one kernel: no workspace, but no null pointers
    assert lib.s3d_mlp_int8_workspace_bytes(4, 16, 16) == 0 < lib.s3d_mlp_int8_workspace_bytes(4, 640, 2560)
    _refused(lib, lib.s3d_mlp_int8(None, *[one] * 8, 4, 16, 16, None, 0, None), "null device pointer")
    for m, k in ((-1, 16), (4, 24), (4, 0), (4, 16400)):
        _refused(lib, lib.s3d_keep_rows(one, one, m, k, None), "s3d_keep_rows: M=")
        _refused(lib, lib.s3d_kept_values(one, one, m, k, None), "s3d_kept_values: M=")
        assert lib.s3d_kept_bytes(m, k) == 0
    assert lib.s3d_kept_bytes(100, 48) == 100 * 51
    for m, n, k in ((0, 16, 16), (4, 24, 16), (4, 16, 24), (4, 16, 16400), (4, 16400, 16)):
        _refused(lib, lib.s3d_kept_linear(one, one, 0, None, 0, one, one, one, m, n, k, 0, 1.0, one, 1 << 30, None), "s3d_kept_linear: M=")
        _refused(lib, lib.s3d_kept_linear_grad(one, one, one, one, one, one, 0, m, n, k, 0, 1.0, one, 1 << 30, None), "s3d_kept_linear_grad: M=")
        _refused(lib, lib.s3d_kept_mlp(*[one] * 5, dtypes, *[one] * 5, m, k, n, one, 1 << 30, None), "s3d_kept_mlp: M=")
        _refused(lib, lib.s3d_kept_mlp_grad(*[one] * 10, 0, m, k, n, one, 1 << 30, None), "s3d_kept_mlp_grad: M=")
    _refused(lib, lib.s3d_kept_linear(one, None, 0, None, 0, one, one, one, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_linear(one, one, 2, None, 0, one, one, one, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "dtypes 2")
    _refused(lib, lib.s3d_kept_linear(one, one, 0, one, 5, one, one, one, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "0, 5")
    _refused(lib, lib.s3d_kept_linear(one, one, 0, None, 0, one, one, one, 4, 16, 16, 0, 1.0, one, 8, None), "workspace 8 B")
    for scaled in (-16, 8, 32):
        _refused(lib, lib.s3d_kept_linear(one, one, 0, None, 0, one, one, one, 4, 16, 16, scaled, 1.0, one, 1 << 30, None), "scaled rows")
        _refused(lib, lib.s3d_kept_linear_grad(one, one, one, one, one, one, 0, 4, 16, 16, scaled, 1.0, one, 1 << 30, None), "scaled rows")
    _refused(lib, lib.s3d_kept_linear_grad(one, one, None, one, one, one, 0, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_linear_grad(one, None, one, one, one, one, 0, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_linear_grad(one, one, one, one, one, one, 2, 4, 16, 16, 0, 1.0, one, 1 << 30, None), "grad_dtype 2")
    _refused(lib, lib.s3d_kept_linear_grad(one, one, one, one, one, one, 0, 4, 16, 16, 0, 1.0, one, 8, None), "workspace 8 B")
    _refused(lib, lib.s3d_kept_mlp(one, one, None, None, None, dtypes, *[one] * 5, 4, 16, 16, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_mlp(*[one] * 5, None, *[one] * 5, 4, 16, 16, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_mlp(*[one] * 5, (ctypes.c_int32 * 4)(0, 1, 2, 0), *[one] * 5, 4, 16, 16, one, 1 << 30, None), "dtype 2")
    _refused(lib, lib.s3d_kept_mlp(*[one] * 5, dtypes, *[one] * 5, 4, 16, 16, one, 8, None), "workspace 8 B")
    _refused(lib, lib.s3d_kept_mlp_grad(one, one, one, one, None, one, one, one, one, one, 0, 4, 16, 16, one, 1 << 30, None), "null")
    _refused(lib, lib.s3d_kept_mlp_grad(*[one] * 10, 3, 4, 16, 16, one, 1 << 30, None), "grad_dtype 3")
    _refused(lib, lib.s3d_kept_mlp_grad(*[one] * 10, 0, 4, 16, 16, None, 1 << 30, None), "workspace 0 B")


def test_cpu_tensors_and_other_objects_are_refused():
    x, norm = torch.randn(4, 48), torch.nn.LayerNorm(48)
    rows = Int8Rows(torch.zeros(4, 48, dtype=torch.int8), torch.zeros(4))
    for bad in (lambda: eight_bits.add_norm_int8(x, None, norm), lambda: eight_bits.quantize_rows(x), lambda: eight_bits.linear_int8(rows, rows),
                lambda: eight_bits.mlp_int8(rows, rows, None, rows, None), lambda: rows.values(), lambda: eight_bits.keep_rows(x.half()),
                lambda: eight_bits.kept_values(torch.zeros(51, dtype=torch.uint8), 48), lambda: eight_bits.checkpointed_linear(x.half(), x),
                lambda: eight_bits.checkpointed_mlp(x.half(), x, None, x.t(), None), lambda: eight_bits.quantize_rows([1.0]),
                lambda: eight_bits.linear_int8([1], rows), lambda: eight_bits.add_norm_int8(None, None, norm)):
        with pytest.raises(ValueError):
            bad()


def test_statement_of_the_kept_form():
    """Scales ascend, have four bits, and codes times scales are fp16 numbers."""
    scales = kept_scales()
    assert scales[0] == 0 and scales[1] == 1 and all(a < b for a, b in zip(scales, scales[1:]))
    assert all(s >> max(0, s.bit_length() - 4) << max(0, s.bit_length() - 4) == s for s in scales)
    assert scales[249] == 576 << 24 and 127 * scales[248] < 65504 << 24 <= 127 * scales[249]
    x = torch.randn(200, 64) * torch.exp(5 * torch.randn(200, 1))
    x = x.clamp(-65504, 65504).half()
    x[0], x[1, :32], x[1, 16] = 65504.0, 0.0, 6e-8
    values = kept(x)
    assert torch.equal(values.half().double(), values) and int(keep(x)[0].abs().max()) == 127
    assert torch.equal(values[1, :17], x[1, :17].double())


@pytest.mark.parametrize("name", ["weight", "bias"])
def test_parameters_that_are_not_as_long_as_the_norm_says(name):
    """The kernel reads a number a channel of each, whatever normalized_shape still is."""
    norm, device = torch.nn.LayerNorm(48), torch.device("cpu")
    assert all(a is b for a, b in zip(eight_bits._norm_parameters(norm, False, 48, device), (norm.weight, norm.bias)))
    assert eight_bits._norm_parameters(norm, True, 48, device)[1] is None
    for other in (torch.ones(44), torch.ones(0), torch.ones(96), torch.ones(48, 1)):
        changed = torch.nn.LayerNorm(48)
        getattr(changed, name).data = other
        assert tuple(changed.normalized_shape) == (48,)
        with pytest.raises(ValueError):
            eight_bits._norm_parameters(changed, False, 48, device)


@pytest.mark.parametrize("switch,flag", [(encoder.eight_bit_inference, "eight_bit_rows"), (encoder.eight_bit_checkpoints, "eight_bit_kept")])
def test_switches_refuse_blocks_on_which_they_cannot_act(switch, flag):
    def stage(channels, heads, mode):
        return encoder.Stage(channels, 2, heads, 5, 4, downsample=False, cRSE="XYZ_RGB", fp16_mode=mode)

    for channels, heads, mode in ((48, 6, 0), (48, 12, 2), (64, 1, 1), (24, 3, 2), (48, 3, None), (1040, 65, 2)):
        bad = stage(channels, heads, mode)
        with pytest.raises(ValueError):
            switch(bad)
        assert not any(getattr(b, flag) for b in bad.blocks) and switch(bad, False) is bad
    for channels, heads, mode in ((48, 6, 1), (48, 3, 2), (64, 2, 2)):
        good = stage(channels, heads, mode)
        assert switch(good) is good and all(getattr(b, flag) for b in good.blocks)
        assert switch(good, False) is good and not any(getattr(b, flag) for b in good.blocks)


def test_a_block_adds_what_is_pending_once(monkeypatch):
    """Where the call in eight bits does not apply, the sum that was made for it is the stream of the layers one by one."""
    calls = []
    monkeypatch.setattr(encoder, "swin_blocks", lambda *_, **__: None)

    def add_layernorm(x, residual, norm, inplace=False):
        calls.append((residual is not None, inplace))
        summed = x if residual is None else x + residual
        return summed, norm(summed)

    monkeypatch.setattr(encoder, "add_layernorm", add_layernorm)
    block = encoder.SwinBlock(48, 6, 5, 4, fp16_mode=2)
    monkeypatch.setattr(block.attn, "forward", lambda x, args: 2 * x)
    feats, pending = torch.randn(4, 48), torch.randn(4, 48)
    with torch.no_grad():
        want, want_at_first = block.forward_fused(feats, pending, None), block.forward_fused(feats, None, None)
        assert calls == [(True, False), (True, True), (False, False), (True, False)]
        encoder.eight_bit_inference(block)
        calls.clear()
        got, got_at_first = block.forward_fused(feats, pending, None), block.forward_fused(feats, None, None)
    assert calls == [(False, False), (True, True), (False, False), (True, False)]
    assert all(torch.equal(a, b) for a, b in zip(got + got_at_first, want + want_at_first))


def test_tensors_whose_storage_was_freed():
    for shape in ((48,), (4, 48)):
        t = torch.zeros(shape)
        assert eight_bits._ready(t.device, t) and eight_bits._dense(t) is t
        strided = t[..., ::2]
        t.untyped_storage().resize_(0)
        assert not eight_bits._ready(t.device, t)
        for view in (t, strided):
            with pytest.raises(ValueError, match="without memory"):
                eight_bits._dense(view)
    assert eight_bits._dense(torch.zeros(0, 48)).shape == (0, 48)
