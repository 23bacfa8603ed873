"""FP8QWeight on the CPU: the format against its definition element by element, the layer
against plain products, serialisation, and what is refused before any launch."""

import ctypes

import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from offload_adam_amd import _lib
from offload_adam_amd.qweight import FORMATS, FP8QWeight, quantize_linears

BF16 = torch.bfloat16


def e4m3_values():
    """Every finite magnitude of the format, ascending: s 4.3 bits, bias 7, no infinity."""
    out = [m * 2.0**-9 for m in range(8)]
    out += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return np.array(out[:-1])  # the last pattern is NaN


def encode_by_definition(x, rows, cols):
    """Values held and scales, by searching the table of e4m3 values."""
    x = np.asarray(x, dtype=np.float64)
    table = e4m3_values()
    held, scales = np.empty_like(x), {}
    for r in range(0, x.shape[0], rows):
        for c in range(0, x.shape[1], cols):
            b = x[r:r + rows, c:c + cols]
            mag = np.abs(b[np.isfinite(b)])
            top = mag.max() if mag.size else 0.0
            e = 0
            if top > 0:
                e = -126
                while top > 448 * 2.0**e:
                    e += 1
            v = np.abs(b) / 2.0**e
            i = np.searchsorted(table, v)  # table[i-1] < v <= table[i]
            hi = np.clip(i, 0, len(table) - 1)
            lo = np.clip(i - 1, 0, len(table) - 1)
            dlo, dhi = v - table[lo], table[hi] - v
            pick = np.where(dlo < dhi, lo, np.where(dhi < dlo, hi, np.where(lo % 2 == 0, lo, hi)))
            held[r:r + rows, c:c + cols] = np.where(
                np.isfinite(b), np.sign(b) * table[pick] * 2.0**e, np.nan)
            scales[r // rows, c // cols] = e
    return held, scales


def awkward(rows, cols, seed=0):
    """Blocks of very different magnitude, ties, zeros and values that are not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    scale = torch.randint(-130, 100, (-(-rows // 8), -(-cols // 16)), generator=g).float()
    scale = scale.repeat_interleave(8, 0)[:rows].repeat_interleave(16, 1)[:, :cols]
    x = torch.where(torch.rand(rows, cols, generator=g) < 0.3,
                    torch.randint(-31, 32, (rows, cols), generator=g) / 16.0, x)
    if rows > 8:
        x = x * torch.exp2(scale.double()).float()
    x[0, :16] = 0.0
    x[-1, -1] = float("inf")
    x[-1, -2] = float("nan")
    x[rows // 2, cols // 2] = -float("inf")
    return x


@pytest.mark.parametrize("shape", [(1, 16), (7, 48), (128, 128), (129, 144), (260, 272)])
def test_codes_and_scales_follow_the_definition(shape):
    x = awkward(*shape)
    q = FP8QWeight.from_float(x)
    held, scales = encode_by_definition(x.numpy(), 128, 128)
    got = q.dequantize().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(held))
    assert np.array_equal(np.nan_to_num(got), np.nan_to_num(held))
    bits = q.block_scale.view(torch.uint8).numpy().astype(int) - 127
    assert all(bits[k] == e for k, e in scales.items())


def test_linear_and_its_gradients():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 70, 144, generator=g, dtype=torch.float32).requires_grad_(True)
    w = nn.Parameter(FP8QWeight.from_float(torch.randn(200, 144, generator=g)))
    b = torch.randn(200, generator=g).requires_grad_(True)
    y = F.linear(x, w, b)
    up = torch.randn(3, 70, 200, generator=g)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), up)
    flat, gy = x.detach().reshape(-1, 144), up.reshape(-1, 200)
    held = lambda t, r, c: torch.from_numpy(encode_by_definition(t.numpy(), r, c)[0])  # noqa: E731
    wv = w.detach().dequantize().double()
    want = held(flat, 1, 128) @ wv.T + b.detach().double()
    assert y.shape == (3, 70, 200)
    # fp32 sums of 144 (200, 210) products of a few units each
    assert (y.detach().reshape(-1, 200).double() - want).abs().max() < 210 * 2**-23 * 400
    assert (dx.reshape(-1, 144).double() - held(gy, 1, 128) @ wv).abs().max() < 210 * 2**-23 * 600
    assert (dw.double() - held(gy, 128, 1).T @ held(flat, 128, 1)).abs().max() < 210 * 2**-23 * 600
    assert (db.double() - gy.double().sum(0)).abs().max() < 210 * 2**-23 * 210


def test_checkpointing_with_create_graph():
    g = torch.Generator().manual_seed(8)
    x = torch.randn(4, 64, generator=g).requires_grad_(True)
    w = nn.Parameter(FP8QWeight.from_float(torch.randn(32, 64, generator=g)))
    want = torch.autograd.grad(F.linear(x, w).sum(), (x, w))
    y = checkpoint(F.linear, x, w, use_reentrant=False)
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert torch.equal(dx, want[0])


def test_shapes_on_the_meta_device():
    w = FP8QWeight.from_float(torch.randn(32, 64, device="meta"))
    x = torch.randn(2, 3, 64, device="meta")
    for enabled in (False, True):
        with torch.autocast("cpu", dtype=BF16, enabled=enabled):
            y = F.linear(x, w, torch.zeros(32, device="meta"))
        assert y.shape == (2, 3, 32) and y.dtype == torch.float32 and y.device.type == "meta"


def test_forward_mode_is_refused():
    """A layer that nothing requires a gradient of has no tangents either, as the other
    formats' layers."""
    w = FP8QWeight.from_float(torch.randn(32, 64))
    x, b = torch.randn(4, 64), torch.randn(32)
    plain = F.linear(x, w, b)
    with forward_ad.dual_level():
        assert torch.equal(F.linear(x, w, b), plain)
        for args in ((forward_ad.make_dual(x, torch.ones_like(x)), w, b),
                     (x, w, forward_ad.make_dual(b, torch.ones_like(b)))):
            with pytest.raises(NotImplementedError):
                F.linear(*args)
            with pytest.raises(NotImplementedError), torch.no_grad():
                F.linear(*args)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: F.linear(t, w), (x,), (torch.ones_like(x),))
    assert torch.equal(F.linear(x, w, b), plain)


def test_second_derivatives_are_refused():
    """Also where the incoming gradient is a constant, and where a tangent is taken by
    differentiating twice: neither may come out as zero."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 64, generator=g).requires_grad_(True)
    w = nn.Parameter(FP8QWeight.from_float(torch.randn(32, 64, generator=g)))
    b = torch.randn(32, generator=g).requires_grad_(True)
    up = torch.randn(4, 32, generator=g)
    want = torch.autograd.grad(F.linear(x, w, b), (x, w, b), up)
    got = torch.autograd.grad(F.linear(x, w, b), (x, w, b), up, create_graph=True)
    assert all(torch.equal(i, j) for i, j in zip(want, got))
    y = F.linear(x, w, b).sum()
    dx, dw = torch.autograd.grad(y, (x, w), create_graph=True)
    for penalty, by in ((dx, w), (dw, x), (y + dx.square().sum(), x)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(penalty.sum(), by, retain_graph=True, allow_unused=True)
    for leaves in ((x, w, b), (x, w.detach(), None)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.functional.jvp(lambda t: F.linear(t, *leaves[1:]), (x.detach(),),
                                          (torch.ones_like(x),))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, BF16])
def test_autocast_casts_as_for_a_plain_weight(dtype):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(5, 64, generator=g).to(dtype).requires_grad_(True)
    plain = torch.randn(32, 64, generator=g)
    w = nn.Parameter(FP8QWeight.from_float(plain))
    b = torch.randn(32, generator=g).requires_grad_(True)
    up = torch.randn(5, 32, generator=g).to(BF16)
    with torch.autocast("cpu", dtype=BF16):
        y = F.linear(x, w, b)
        frozen = F.linear(x.detach(), w.detach(), b.detach())
        assert F.linear(x.detach(), plain, b.detach()).dtype == y.dtype == frozen.dtype == BF16
        inside = torch.autograd.grad(y, (x, w, b), up, retain_graph=True)
    got = (y, *torch.autograd.grad(y, (x, w, b), up))
    assert [v.dtype for v in got[1:]] == [dtype, torch.float32, torch.float32]
    # the same as casting by hand: fp32 sums, one rounding
    c, d = x.detach().to(BF16).requires_grad_(True), b.detach().to(BF16).requires_grad_(True)
    want = F.linear(c, w, d)
    want = (want, *torch.autograd.grad(want, (c, w, d), up))
    assert torch.equal(frozen, want[0])
    for i, j in zip(got, want):
        assert torch.equal(i.float(), j.float())
    for i, j in zip(got[1:], inside):
        assert torch.equal(i, j)
    with torch.autocast("cpu", dtype=BF16), pytest.raises(TypeError):
        F.linear(x.detach().double(), w)


def test_state_dict_and_config(tmp_path):
    from safetensors.torch import load_file, save_file

    assert FORMATS["fp8"] is FP8QWeight
    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(256, 130, bias=False), nn.Linear(130, 20)).to(BF16)
    report = quantize_linears(model, FP8QWeight)
    assert report.quantized == ["0"] and report.incompatible[0][0] == "1"  # 130 columns
    sd = model.state_dict()
    assert sd["0.weight"].dtype == torch.float8_e4m3fn
    assert sd["0.weight_scale_inv"].dtype == torch.float32
    save_file({k: v.contiguous() for k, v in sd.items()}, str(tmp_path / "m.safetensors"))
    x = torch.randn(5, 256, dtype=BF16)
    want = model(x)
    other = nn.Sequential(nn.Linear(256, 130, bias=False), nn.Linear(130, 20)).to(BF16)
    quantize_linears(other, FP8QWeight)
    missing, unexpected = other.load_state_dict(load_file(str(tmp_path / "m.safetensors")))
    assert not missing and not unexpected and torch.equal(other(x), want)
    # the checkpoint of a model that was never quantised
    plain = nn.Sequential(nn.Linear(256, 130, bias=False), nn.Linear(130, 20)).to(BF16)
    other.load_state_dict(plain.state_dict())
    assert torch.equal(other[0].weight.data.dequantize(),
                       FP8QWeight.from_float(plain[0].weight.data).dequantize())
    c = FP8QWeight.build_hf_quantization_config(skip_patterns=("lm_head",))
    assert c["quant_method"] == "fp8" and c["weight_block_size"] == [128, 128]
    assert c["modules_to_not_convert"] == ["lm_head"]


def test_checkpoints_with_other_scales_are_encoded_again():
    g = torch.Generator().manual_seed(3)
    codes = torch.randn(150, 160, generator=g).mul(100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ref = FP8QWeight.from_float(torch.zeros(150, 160, dtype=BF16))
    scale = torch.rand(2, 2, generator=g) + 0.3
    got = FP8QWeight.from_plain_state_dict({"weight": codes, "weight_scale_inv": scale}, ref)
    spread = scale.repeat_interleave(128, 0)[:150].repeat_interleave(128, 1)[:, :160]
    value = codes.float() * spread
    assert torch.equal(got.dequantize(torch.float32),
                       FP8QWeight.from_float(value).dequantize(torch.float32))
    # powers of two are taken as they are, whatever the codes reach
    scale = torch.tensor([[0.25, 2.0], [1.0, 2.0**-100]])
    got = FP8QWeight.from_plain_state_dict({"weight": codes, "weight_scale_inv": scale}, ref)
    assert torch.equal(got.weight.view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(got.block_scale.float(), scale)
    with pytest.raises(ValueError, match="reference"):
        FP8QWeight.from_plain_state_dict({"weight": codes, "weight_scale_inv": scale})


def test_layers_without_inputs_stay_plain():
    model = nn.Sequential(nn.Linear(0, 4), nn.Linear(16, 4))
    report = quantize_linears(model, FP8QWeight)
    assert report.quantized == ["1"] and report.incompatible[0][0] == "0"
    assert torch.equal(model[0](torch.zeros(3, 0)), model[0].bias.expand(3, 4))


@pytest.mark.parametrize("name", ["int8", "int4", "nf4", "nvfp4"])
def test_other_formats_take_float8_weights_as_values(name):
    g = torch.Generator().manual_seed(5)
    model = nn.Sequential(nn.Linear(128, 64, bias=False)).to(BF16)
    quantize_linears(model, FORMATS[name])
    values = torch.randn(64, 128, generator=g).to(torch.float8_e4m3fn)
    model.load_state_dict({"0.weight": values})
    want = FORMATS[name].from_float(torch.zeros(64, 128, dtype=BF16))
    want.copy_(values)
    assert torch.equal(model[0].weight.data.dequantize(torch.float32),
                       want.dequantize(torch.float32))


@pytest.mark.parametrize("power", [False, True])
def test_checkpoints_that_do_not_fit_are_refused(power):
    """Scales of finer, coarser or transposed blocks, or that are no scales; codes of another
    type or of an odd width.  A weight of another shape is torch's own size mismatch."""
    g = torch.Generator().manual_seed(4)
    model = nn.Sequential(nn.Linear(256, 384, bias=False)).to(BF16)
    quantize_linears(model, FP8QWeight)
    before = model[0].weight.data.dequantize()
    codes = torch.randn(384, 256, generator=g).mul(50).to(torch.float8_e4m3fn)

    def scales(*grid):
        return torch.full(grid, 0.5) if power else torch.rand(grid, generator=g) + 0.3

    def load(weight, scale):
        return model.load_state_dict({"0.weight": weight, "0.weight_scale_inv": scale})

    for grid in ((6, 4), (1, 1), (2, 3), (3, 1), (6,), ()):
        with pytest.raises(ValueError, match="weight_scale_inv"):
            load(codes, scales(*grid))
    for bad in (float("nan"), float("inf"), -1.0):
        scale = scales(3, 2)
        scale[1, 1] = bad
        with pytest.raises(ValueError, match="weight_scale_inv"):
            load(codes, scale)
    for weight in (codes.view(torch.uint8), codes.to(torch.float8_e5m2), codes[:, :250], codes[0]):
        with pytest.raises(ValueError, match="weight must be"):
            load(codes.view(torch.uint8), scales(3, 2))
        with pytest.raises(ValueError, match="weight must be"):
            FP8QWeight.from_plain_state_dict({"weight": weight, "weight_scale_inv": scales(3, 2)},
                                             model[0].weight.data)
    with pytest.raises(RuntimeError, match="size mismatch"):
        load(codes[:256], scales(2, 2))
    assert torch.equal(model[0].weight.data.dequantize(), before)
    # a block of zeros may come with a scale of zero
    scale = scales(3, 2)
    scale[0, 0] = 0.0
    load(codes, scale)
    assert not model[0].weight.data.dequantize()[:128, :128].any()


def test_refused_arguments():
    w = FP8QWeight.from_float(torch.randn(32, 64))
    x = torch.randn(4, 64)
    assert not FP8QWeight.can_quantize(torch.zeros(8, 24))
    assert not FP8QWeight.can_quantize(torch.zeros(8, 8, 16))
    for args, exc in [((x.double(), w), TypeError), ((x[:, :48], w), ValueError),
                      ((x, w, torch.zeros(31)), ValueError), ((w, w), TypeError),
                      ((x.new_zeros(()), w), ValueError)]:
        with pytest.raises(exc):
            F.linear(*args)
    with pytest.raises(AssertionError):
        FP8QWeight(w.weight, w.block_scale[:, :0], torch.float32)
    with pytest.raises(AssertionError):
        FP8QWeight(w.weight.float(), w.block_scale, torch.float32)
    y = F.linear(x[:0], w)
    assert y.shape == (0, 32)


def test_the_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) // 256 * 256
    ok, odd = ctypes.c_void_p(a), ctypes.c_void_p(a + 1)
    big = ctypes.c_size_t(1 << 40)
    quant = lambda src=ok, dt=1, st=32, r=4, c=32, q=ok, s=ok: lib.oa_quant_fp8(  # noqa: E731
        src, dt, st, r, c, q, s, None)
    assert quant(c=24) == -1 and quant(r=-1) == -1 and quant(dt=5) == -1 and quant(src=None) == -1
    assert quant(q=None) == -1 and quant(s=None) == -1 and quant(st=8) == -1
    assert quant(q=odd) == -2 and quant(src=odd) == -2
    assert quant(r=1 << 40, c=1 << 20, st=1 << 20) == -3
    assert quant(r=0) == 0
    deq = lambda q=ok, s=ok, r=4, c=32, out=ok, dt=1, st=32: lib.oa_dequant_fp8(  # noqa: E731
        q, s, r, c, out, dt, st, None)
    assert deq(c=24) == -1 and deq(dt=9) == -1 and deq(out=None) == -1 and deq(st=16) == -1
    assert deq(out=odd) == -2 and deq(q=odd) == -2

    def fwd(x=ok, ldx=32, dt=1, t=4, q=ok, s=ok, b=None, n=8, k=32, y=ok, ws=ok, wsb=big):
        return lib.oa_fp8_linear_forward(x, ldx, dt, t, q, s, b, n, k, y, ws, wsb, None)

    def bwd(x=ok, ldx=32, dt=1, t=4, q=ok, s=ok, n=8, k=32, ws=ok, wsb=big, g=ok, ldg=8, dx=ok,
            dw=ok, db=ok):
        return lib.oa_fp8_linear_backward(g, ldg, x, ldx, dt, t, q, s, n, k, dx, dw, db, ws, wsb,
                                          None)

    for f in (fwd, bwd):
        assert f(dt=3) == -1 and f(t=0) == -1 and f(n=0) == -1 and f(k=24) == -1 and f(k=0) == -1
        assert f(x=None) == -1 and f(q=None) == -1 and f(s=None) == -1 and f(ws=None) == -1
        assert f(ldx=16) == -1 and f(wsb=ctypes.c_size_t(8)) == -1
        assert f(x=odd) == -2 and f(q=odd) == -2 and f(ws=odd) == -2
        assert f(t=(1 << 22) + 1) == -3 and f(n=(1 << 22) + 1) == -3
    assert fwd(y=None) == -1 and fwd(y=odd) == -2 and fwd(b=odd) == -2
    assert bwd(dx=None, dw=None, db=None) == -1 and bwd(g=None) == -1 and bwd(ldg=4) == -1
    assert bwd(dx=odd) == -2 and bwd(dw=odd) == -2 and bwd(db=odd) == -2
    assert lib.oa_fp8_linear_workspace_bytes(0, 16, 16, 0, 0, 0, 0) == 0
    for sizes in ((1 << 40, 1 << 40, 16), (4, 1 << 62, 16), (4, 16, (1 << 22) + 1)):
        assert lib.oa_fp8_linear_workspace_bytes(*sizes, 0, 0, 0, 0) == 0
        assert lib.oa_fp8_linear_workspace_bytes(*sizes, 1, 1, 1, 1) == 0
