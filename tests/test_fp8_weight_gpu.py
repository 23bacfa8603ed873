"""FP8QWeight's kernels on the GPU: the codec bit for bit against its definition, the
layer's products against 64 bits.

Tolerance of a product of n terms: the codes' values multiply exactly, fp32 sums add at
most 2u (u = 2^-24) of the running magnitude per term in whatever order, and the result is
rounded once by r, half a step of its type:  n 2u sum|a b| + r |y|  (+ fp16's smallest step).
Inside a group of 8 consecutive terms the matrix instruction cuts every product to a
multiple of 2^-13 of the power of two under the group's largest (products of 256 x 256 and
7 x 1 give 65536, of 256 x 256 and 15 x 1 give 65544), which is less than 2^-13 of the
largest product for each of the 7 others:  7 * 2^-13 * sum over groups max|a| max|b|.
"""

import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from test_fp8_weight import awkward, e4m3_values, encode_by_definition

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24


def _bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8)


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.cpu().float()), torch.nan_to_num(b.cpu().float())) and \
        torch.equal(torch.isnan(a.cpu()), torch.isnan(b.cpu()))


# ------------------------------------------------------------------------ codec


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 16), (5, 48), (128, 128), (130, 272), (300, 1040)])
def test_encode_and_decode(shape, dtype):
    from offload_adam_amd.qweight import FP8QWeight

    x = awkward(*shape, seed=sum(shape))
    x = x.clamp(-6e4, 6e4).to(dtype) if dtype == F16 else x.to(dtype)
    x[0, 0], x[-1, -1] = float("nan"), float("inf")
    q = FP8QWeight.from_float(x.cuda())
    cpu = FP8QWeight.from_float(x)
    held, _ = encode_by_definition(x.double().numpy(), 128, 128)
    assert torch.equal(_bits(q.block_scale), _bits(cpu.block_scale))
    got = q.dequantize(F32)
    assert np.array_equal(np.isnan(got.cpu().numpy()), np.isnan(held))
    assert np.array_equal(np.nan_to_num(got.cpu().double().numpy()), np.nan_to_num(held))
    for out in (F32, BF16, F16):
        assert _same(q.dequantize(out), cpu.dequantize(F32).to(out)), out


def test_strided_sources_and_in_place():
    from offload_adam_amd.qweight import FP8QWeight

    g = torch.Generator().manual_seed(0)
    wide = torch.randn(200, 300, generator=g).cuda()
    for name, src in {"unaligned": wide[:, 3:147], "aligned": wide[:, 64:208],
                      "transposed": wide.t()[:144, :160], "rows": wide[::2, :144]}.items():
        want = FP8QWeight.from_float(src.contiguous())
        q = FP8QWeight.from_float(torch.zeros(src.shape, device="cuda"))
        before = q.weight.data_ptr(), q.weight._version
        q.copy_(src)
        assert torch.equal(_bits(q.weight), _bits(want.weight)), name
        assert torch.equal(_bits(q.block_scale), _bits(want.block_scale)), name
        assert q.weight.data_ptr() == before[0] and q.weight._version > before[1]
    with pytest.raises((ValueError, RuntimeError)):
        q.copy_(torch.zeros(3, 16, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("stride, first", [(272, 0), (280, 8), (281, 0), (300, 3)])
def test_the_c_decoder_writes_rows_of_any_stride_and_alignment(stride, first, dtype):
    """Rows that 16-byte stores fit, and rows that take single elements; nothing beside them."""
    from offload_adam_amd import _lib
    from offload_adam_amd.qweight import FP8QWeight

    rows, cols = 131, 272
    q = FP8QWeight.from_float(awkward(rows, cols, seed=2).cuda())
    out = torch.full((rows * stride + 16,), 7.0, dtype=dtype, device="cuda")
    want = out.clone()
    want[first:first + rows * stride].view(rows, stride)[:, :cols] = q.dequantize(dtype)
    code = _lib.load().oa_dequant_fp8(
        q.weight.data_ptr(), q.block_scale.data_ptr(), rows, cols,
        out.data_ptr() + first * out.element_size(), _lib.dtype_code(dtype), stride,
        _lib.current_stream_ptr())
    assert code == 0 and _same(out, want)


def test_state_dict_on_the_gpu():
    from offload_adam_amd.qweight import FP8QWeight, quantize_linears

    g = torch.Generator().manual_seed(1)
    model = nn.Sequential(nn.Linear(272, 200, bias=False)).to(BF16).cuda()
    other = nn.Sequential(nn.Linear(272, 200, bias=False)).to(BF16).cuda()
    for m in (model, other):
        quantize_linears(m, FP8QWeight)
    sd = model.state_dict()
    for checkpoint in (sd, {k: v.cpu() for k, v in sd.items()}):
        other[0].weight.data.copy_(torch.zeros(200, 272, device="cuda"))
        other.load_state_dict(checkpoint)
        assert torch.equal(_bits(other[0].weight.data.weight), _bits(model[0].weight.data.weight))
        assert torch.equal(_bits(other[0].weight.data.block_scale),
                           _bits(model[0].weight.data.block_scale))
    scale = torch.rand(2, 3, generator=g) + 0.3
    codes = torch.randn(200, 272, generator=g).mul(50).to(torch.float8_e4m3fn)
    loaded = []
    for device in ("cpu", "cuda"):
        other.load_state_dict({"0.weight": codes.to(device), "0.weight_scale_inv": scale.to(device)})
        loaded.append(other[0].weight.data.dequantize(F32).cpu())
    spread = scale.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :272]
    want = FP8QWeight.from_float(codes.float() * spread).dequantize(F32)
    assert torch.equal(loaded[0], want) and torch.equal(loaded[1], want)


def test_codec_on_more_than_2_31_elements():
    from offload_adam_amd.qweight import FP8QWeight

    rows, cols = 131_200, 16_400
    x = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(0, 0.02)
    q = FP8QWeight.from_float(x)
    back = q.dequantize()
    for r in (0, 65_472, rows - 128):
        part = FP8QWeight.from_float(x[r - r % 128:r - r % 128 + 128])
        n = part.shape[0]
        assert torch.equal(_bits(q.weight[r - r % 128:r - r % 128 + n]), _bits(part.weight))
        assert torch.equal(back[r - r % 128:r - r % 128 + n], part.dequantize())


# --------------------------------------------------------------------- products


def _held(x, dim):
    """encode_by_definition for blocks of 128 along ``dim``, on the GPU (finite input)."""
    x = x.double()
    if dim == 0:
        return _held(x.t(), 1).t()
    r, c = x.shape
    b = F.pad(x, (0, -c % 128)).reshape(r, -1, 128)
    top = b.abs().amax(2, keepdim=True)
    _, e = torch.frexp(top)  # top < 2^e
    scale = ((e.long() - 9 + 1023) << 52).view(torch.float64)  # 2^(e-9), exactly
    scale = torch.where(top > 448 * scale, 2 * scale, scale)
    scale = torch.where(top == 0, 1.0, scale.clamp_min(2.0**-126))
    table = torch.from_numpy(e4m3_values()).cuda()
    v = b.abs() / scale
    hi = torch.searchsorted(table, v.reshape(r, -1).contiguous()).reshape(v.shape)
    hi = hi.clamp_max(len(table) - 1)
    lo = (hi - 1).clamp_min(0)
    down, up = v - table[lo], table[hi] - v
    pick = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (torch.sign(b) * table[pick] * scale).reshape(r, -1)[:, :c]


def _tops(a):
    """Largest magnitude of every 8 columns."""
    return F.pad(a.abs(), (0, -a.shape[1] % 8)).reshape(a.shape[0], -1, 8).amax(2)


def _close(got, a, b, what, bias=None, codes=True):
    """got against a @ b; ``codes``: computed from 8-bit codes."""
    want = a @ b.contiguous()
    mag = a.abs() @ b.abs().contiguous()
    if bias is not None:
        want = want + bias
        mag = mag + bias.abs()
    r = torch.finfo(got.dtype).eps / 2
    tol = (a.shape[1] + 2) * 2 * U * mag + r * want.abs()
    if codes:
        tol = tol + 7 * 2.0**-13 * (_tops(a) @ _tops(b.t()).t().contiguous())
    if got.dtype == F16:
        tol = tol + 2.0**-25
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all(), what
    assert bool((off <= 0).all()), f"{what}: over by {float(off.max())}"


def _layer(t, k, n, dtype, seed=0, bias=False):
    from offload_adam_amd.qweight import FP8QWeight

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    w = torch.randn(n, k, generator=g) * 0.05 * torch.exp2(torch.randn(n, 1, generator=g))
    gy = torch.randn(t, n, generator=g) * 0.01 * torch.exp2(2 * torch.randn(t, 1, generator=g))
    q = nn.Parameter(FP8QWeight.from_float(w.to(dtype).cuda()))
    b = torch.randn(n, generator=g).to(dtype).cuda().requires_grad_(True) if bias else None
    return x.to(dtype).cuda().requires_grad_(True), q, b, gy.to(dtype).cuda()


SHAPES = [(1, 16, 1), (1, 4096, 300), (3, 48, 5), (24, 2064, 130), (100, 688, 250),
          (128, 128, 128), (129, 144, 257), (300, 1040, 513), (65, 5632, 96), (2049, 272, 640)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_and_its_gradients(shape, dtype):
    t, k, n = shape
    x, q, b, gy = _layer(t, k, n, dtype, seed=t + k + n, bias=True)
    y = F.linear(x, q, b)
    dx, dw, db = torch.autograd.grad(y, (x, q, b), gy)
    assert all(v.dtype == dtype for v in (y, dx, dw, db))
    xv, w = x.detach(), q.detach().dequantize(F32).double()
    _close(y.detach(), _held(xv, 1), w.t(), "y", b.detach().double())
    _close(dx, _held(gy, 1), w, "dx")
    _close(dw, _held(gy, 0).t(), _held(xv, 0), "dw")
    _close(db[None], torch.ones(1, t, dtype=torch.float64, device="cuda"), gy.double(), "db",
           codes=False)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 14336, 70), (1, 144, 4200), (4, 4096, 4117), (7, 2064, 33),
                                   (16, 1024, 300), (16, 1040, 50), (12, 8400, 50), (17, 8400, 70),
                                   (32, 400, 4200), (32, 2064, 19), (33, 2064, 19), (64, 48, 70)])
def test_few_tokens(shape, dtype):
    """Both sides of what decides how few tokens are multiplied: how many, where their codes
    are made, how many waves share a column, whether rows can be read in octets."""
    t, k, n = shape
    x, q, b, _ = _layer(t, k, n, dtype, seed=sum(shape), bias=True)
    x, w = x.detach(), q.detach().dequantize(F32).double()
    y = F.linear(x, q.detach(), b.detach())
    _close(y, _held(x, 1), w.t(), "y", b.detach().double())
    wide = torch.zeros(t, k + 11, dtype=dtype, device="cuda")
    wide[:, 3:3 + k] = x
    assert torch.equal(F.linear(wide[:, 3:3 + k], q.detach(), b.detach()), y)
    if t > 1:
        x[0, -1], x[-1, 0] = float("nan"), float("-inf")
        bad = F.linear(x, q.detach(), b.detach())
        assert torch.isnan(bad[[0, -1]]).all() and torch.equal(bad[1:-1], y[1:-1])


def test_the_bias_gradient_is_the_plain_sum():
    """Infinities and NaN stay in their columns, and stay what they are."""
    x, q, b, gy = _layer(300, 144, 130, BF16, bias=True)
    gy[7, 3], gy[200, 3], gy[8, 40], gy[9, 129] = *2 * [float("inf")], float("-inf"), float("nan")
    db, = torch.autograd.grad(F.linear(x, q, b), b, gy)
    assert db[3] == float("inf") and db[40] == float("-inf") and torch.isnan(db[129])
    keep = torch.ones(130, dtype=torch.bool, device="cuda")
    keep[[3, 40, 129]] = False
    _close(db[None, keep], torch.ones(1, 300, dtype=torch.float64, device="cuda"),
           gy[:, keep].double(), "db", codes=False)


@pytest.mark.parametrize("shape", [(4096, 512, 3200), (3000, 2048, 4000), (4300, 4096, 4001),
                                   (4000, 4304, 4096), (2300, 8000, 4100)])
def test_large_tiles(shape):
    """The last three: more tiles than CUs, those that are over cut along k."""
    t, k, n = shape
    x, q, b, gy = _layer(t, k, n, BF16, seed=4, bias=True)
    y = F.linear(x, q, b)
    dx, dw = torch.autograd.grad(y, (x, q), gy)
    xv, w = x.detach(), q.detach().dequantize(F32).double()
    _close(y.detach(), _held(xv, 1), w.t(), "y", b.detach().double())
    _close(dx, _held(gy, 1), w, "dx")
    _close(dw, _held(gy, 0).t(), _held(xv, 0), "dw")


def test_each_result_alone_gives_the_same_bits():
    x, q, b, gy = _layer(200, 272, 333, BF16, bias=True)
    all3 = torch.autograd.grad(F.linear(x, q, b), (x, q, b), gy)
    for i in range(3):
        leaves = [x.detach(), q.detach(), b.detach()]
        leaves[i] = nn.Parameter(leaves[i]) if i == 1 else leaves[i].clone().requires_grad_(True)
        got, = torch.autograd.grad(F.linear(*leaves), leaves[i], gy)
        assert torch.equal(got, all3[i]), i


def test_strides_and_shapes():
    x, q, b, gy = _layer(60, 144, 130, BF16, bias=True)
    want = F.linear(x.detach(), q, b)
    wide = torch.zeros(60, 200, dtype=BF16, device="cuda")
    cases = {"unaligned slice": (wide[:, 5:149], 1), "aligned slice": (wide[:, 16:160], 1),
             "three dimensions": (torch.zeros(4, 15, 144, dtype=BF16, device="cuda"), 0),
             "transposed": (torch.zeros(144, 60, dtype=BF16, device="cuda").t(), 1),
             "one dimension": (torch.zeros(144, dtype=BF16, device="cuda"), 2)}
    for name, (view, kind) in cases.items():
        src = x.detach()[0] if kind == 2 else x.detach().reshape(view.shape)
        view.copy_(src)
        a = view.detach().requires_grad_(True)
        y = F.linear(a, q, b)
        ref = want[0] if kind == 2 else want.reshape(y.shape)
        assert torch.equal(y, ref), name
        da, dq = torch.autograd.grad(y, (a, q), gy[0] if kind == 2 else gy.reshape(y.shape))
        assert da.shape == a.shape and torch.isfinite(da).all() and dq.shape == (130, 144)
    # a broadcast gradient, as sum().backward() gives
    a = x.detach().requires_grad_(True)
    da, = torch.autograd.grad(F.linear(a, q).sum(), a)
    ones = torch.ones(60, 130, dtype=BF16, device="cuda")
    assert torch.equal(da, torch.autograd.grad(F.linear(a, q), a, ones)[0])


def test_non_finite_elements_stay_in_their_rows():
    x, q, _, _ = _layer(40, 272, 64, BF16)
    want = F.linear(x.detach(), q)
    bad = x.detach().clone()
    bad[3, 5], bad[7, 200] = float("nan"), float("inf")
    y = F.linear(bad, q)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 7]] = False
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[~keep]).all()
    assert F.linear(torch.zeros_like(bad), q).abs().max() == 0
    # a gradient of zeros
    a = x.detach().requires_grad_(True)
    da, dq = torch.autograd.grad(F.linear(a, q), (a, q), torch.zeros_like(want))
    assert not da.any() and not dq.any()


def test_nothing_to_do():
    x, q, b, gy = _layer(4, 144, 130, BF16, bias=True)
    a = x.detach()[:0].requires_grad_(True)
    y = F.linear(a, q, b)
    da, dq, db = torch.autograd.grad(y, (a, q, b), gy[:0])
    assert y.shape == (0, 130) and da.shape == (0, 144)
    assert not dq.any() and not db.any()


def test_autocast_casts_as_for_a_plain_weight():
    x, q, b, gy = _layer(40, 144, 130, F32, bias=True)
    for low in (BF16, F16):
        c, d = x.detach().to(low).requires_grad_(True), b.detach().to(low).requires_grad_(True)
        want = F.linear(c, q, d)
        want = (want, *torch.autograd.grad(want, (c, q, d), gy.to(low)))
        with torch.autocast("cuda", dtype=low):
            y = F.linear(x, q, b)
        got = (y, *torch.autograd.grad(y, (x, q, b), gy.to(low)))
        assert y.dtype == low and all(v.dtype == F32 for v in got[1:])
        assert all(torch.equal(i.float(), j.float()) for i, j in zip(got, want))


def test_gradient_against_differences():
    """The layer is linear in its encoded input: steps that the codes hold exactly."""
    from offload_adam_amd.qweight import FP8QWeight

    g = torch.Generator().manual_seed(0)
    k, n = 128, 96
    x = torch.randint(-6, 7, (50, k), generator=g).float()
    x[:, 0] = 8.0  # no step moves a scale
    q = nn.Parameter(FP8QWeight.from_float(torch.randint(-8, 9, (n, k), generator=g).float().cuda()))
    gy = torch.randint(-8, 9, (50, n), generator=g).float().cuda()
    s = torch.randint(0, 2, (50, k), generator=g).float() * 2 - 1
    s[:, 0] = 0.0
    x, s = x.cuda(), s.cuda()
    a = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(F.linear(a, q), a, gy)
    with torch.no_grad():
        diff = ((F.linear(x + s, q) - F.linear(x - s, q)).double() * gy).sum() / 2
    assert float(diff) == float((dx.double() * s).sum())  # small integers: exact


def test_another_stream_and_graphs():
    layers = [_layer(90, 272, 200, BF16, seed=s, bias=True) for s in range(3)]
    eager = []
    for x, q, b, gy in layers:
        y = F.linear(x, q, b)
        eager.append([y.detach(), *torch.autograd.grad(y, (x, q, b), gy)])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x, q, b, gy = layers[0]
        y = F.linear(x, q, b)
        got = [y.detach(), *torch.autograd.grad(y, (x, q, b), gy)]
    side.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(got, eager[0]))
    del y, got

    graphs = []
    for x, q, b, gy in layers[:2]:
        # leaves of their own: no eager graph of theirs is alive during the capture
        x, b = x.detach().clone().requires_grad_(True), b.detach().clone().requires_grad_(True)
        q = nn.Parameter(q.detach().clone())
        gy = gy.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = F.linear(x, q, b)
            out = [y, *torch.autograd.grad(y, (x, q, b), gy)]
        graphs.append((graph, x, gy, out))
    for _ in range(3):
        for i, (graph, x, gy, out) in enumerate(graphs):
            with torch.no_grad():
                x.copy_(layers[i][0])
                gy.copy_(layers[i][3])
            graph.replay()
        x, q, b, gy = layers[2]
        y = F.linear(x, q, b)
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), eager[2][0])
        for i, (_, _, _, out) in enumerate(graphs):
            assert all(torch.equal(a.detach(), c) for a, c in zip(out, eager[i])), i


# --------------------------------------------------------------------- training


def test_optimizers_re_encode_the_payload():
    from offload_adam_amd import Adam
    from offload_adam_amd.qweight import FP8QWeight, quantize_linears

    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(256, 200), nn.SiLU(), nn.Linear(200, 96)).to(BF16).cuda()
    assert len(quantize_linears(model, FP8QWeight).quantized) == 1  # 200 columns are refused
    opt = Adam(model.parameters(), lr=1e-2, mode="fp32_master", decoupled_weight_decay=True)
    x = torch.randn(64, 256, dtype=BF16, device="cuda")
    w = model[0].weight
    codes = _bits(w.data.weight).clone()
    with pytest.warns(UserWarning):
        for _ in range(2):
            model(x).float().square().mean().backward()
            opt.step()
            opt.zero_grad()
    master = opt.state[w]["master_params"]
    want = FP8QWeight.from_float(master)
    assert torch.equal(_bits(w.data.weight), _bits(want.weight))
    assert torch.equal(_bits(w.data.block_scale), _bits(want.block_scale))
    assert not torch.equal(codes, _bits(w.data.weight))


def test_a_training_step_through_both_operators():
    """Layers on 8-bit codes, the loss behind them, OffloadAdam stepping in the hooks: the
    same gradients as with the logits kept, within what their 16-bit rounding can do, and
    payloads that follow the masters."""
    from offload_adam_amd import OffloadAdam, linear_cross_entropy
    from offload_adam_amd.qweight import FP8QWeight, quantize_linears

    torch.manual_seed(0)
    body = nn.Sequential(nn.Embedding(500, 256), nn.Linear(256, 384), nn.SiLU(),
                         nn.Linear(384, 256)).to(BF16).cuda()
    head = nn.Linear(256, 500, bias=False).to(BF16).cuda()
    model = nn.ModuleList([body, head])
    assert len(quantize_linears(body, FP8QWeight).quantized) == 2
    ids = torch.randint(500, (3, 70), device="cuda")
    target = torch.randint(500, (3, 70), device="cuda")
    target[0, :20] = -100
    hidden = body(ids)
    loss = linear_cross_entropy(hidden, head.weight, target)
    logits = F.linear(hidden, head.weight).float()
    plain = F.cross_entropy(logits.reshape(-1, 500), target.reshape(-1))
    # logits rounded to bf16: half a step of the largest, twice
    assert abs(loss.item() - plain.item()) <= 2 * logits.abs().max().item() * 2.0**-8
    leaves = [p for p in model.parameters()]
    a = torch.autograd.grad(loss, leaves, retain_graph=True)
    assert all(torch.isfinite(v).all() for v in a)
    opt = OffloadAdam(model, lr=1e-3, mode="fp32_master", decoupled_weight_decay=True)
    opt.ready_for_optimizer_step = True
    del hidden, loss, logits, plain
    for _ in range(2):
        linear_cross_entropy(body(ids), head.weight, target).backward()
        opt.step()
        opt.zero_grad()
    torch.cuda.synchronize()
    for layer in (body[1], body[3]):
        master = opt.state[layer.weight]["master_params"].cuda()
        want = FP8QWeight.from_float(master)
        assert torch.equal(_bits(layer.weight.data.weight), _bits(want.weight))


def test_the_decoder_of_the_step_benchmark(monkeypatch, capsys):
    """``bench_e2e.py --qat fp8 --fused-loss``: the loss is that of the logits kept, and the
    step it follows numerically leaves masters, moments and payloads as they have to be."""
    import json
    import sys

    import bench_e2e
    from offload_adam_amd.qweight import FP8QWeight, quantize_linears

    cfg = bench_e2e.MODELS["tiny"]
    ids = torch.randint(0, cfg["vocab"], (1, 200), device="cuda")
    losses = []
    for fused in (False, True):
        model = bench_e2e.build_model(cfg, torch.device("cuda:0"), fused_loss=fused)
        assert quantize_linears(model, FP8QWeight, skip_patterns=("lm_head",)).quantized
        losses.append(float(model(ids).detach()))
    # the same weights; the logits kept are rounded to bf16, here under 4 of magnitude
    assert abs(losses[0] - losses[1]) <= 2 * 4 * 2.0**-8
    del model
    monkeypatch.setattr(sys, "argv", ["bench_e2e.py", "--model", "tiny", "--qat", "fp8",
                                      "--fused-loss", "--check", "--seq", "200", "--steps", "1",
                                      "--grad-accum", "2"])
    bench_e2e.main()
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["check"]["passed"], out["check"]
    assert out["check"]["quantised_tensors"] > 0 and out["qat"]["format"] == "fp8"
