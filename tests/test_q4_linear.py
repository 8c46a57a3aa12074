"""The linear layer with 4-bit weights against plain 64-bit arithmetic on what its codes and scales stand for."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from rustingbrain_b200 import InvalidConfig, InvalidInput, _lib


# ---- refusals: no device needed -------------------------------------------------------------------------------------
def test_arguments_are_checked_before_any_device_work():
    L = _lib.lib()
    size = L.q4_linear_packed_bytes
    # units of 32 outputs and 128 channels: half a byte a code, two bytes a scale
    assert size(1, 32, 32) == 32 * 64 + 32 * 4 * 2
    assert size(2816, 1024, 32) == 2816 * 512 + 2816 * 32 * 2
    assert size(33, 384, 128) == 64 * 192 + 64 * 3 * 2
    for bad in ((0, 32, 32), (4, 0, 32), (4, 33, 32), (4, 64, 16), (4, 64, 128), (4, 96, 64), (-1, 32, 32), (4, 256, 256)):
        assert size(*bad) == 0, bad
    buf = (C.c_float * 256)()
    p = C.c_void_p((C.addressof(buf) + 15) // 16 * 16)
    msg = C.create_string_buffer(128)

    def fwd(x=p, ldx=64, packed=p, y=p, ldy=8, rows=1, d_in=64, d_out=8, group=32, precision=_lib.PRECISION_BF16):
        return L.q4_linear_forward(x, ldx, packed, y, ldy, rows, d_in, d_out, group, precision, None, msg, 128)
    assert fwd(rows=0) == _lib.OK and fwd(rows=0, x=None, y=None) == _lib.OK
    assert fwd(precision=_lib.PRECISION_Q8) == _lib.INVALID_CONFIG
    assert fwd(group=48) == _lib.INVALID_CONFIG and fwd(d_in=48) == _lib.INVALID_CONFIG and fwd(d_out=0) == _lib.INVALID_CONFIG
    off = lambda n: C.c_void_p(p.value + n)
    for bad in (dict(x=None), dict(y=None), dict(packed=None), dict(packed=off(8)), dict(x=off(2)), dict(x=off(8)), dict(y=off(1)), dict(ldx=63),
                dict(ldy=7), dict(rows=-1), dict(rows=2, ldx=68), dict(rows=64 * 65536)):
        assert fwd(**bad) == _lib.INVALID_INPUT and msg.value, bad
    # y on top of x, or on a part of it: x is 64 channels of 128 bytes
    for bad in (dict(y=p), dict(y=off(126)), dict(rows=3, ldx=72, ldy=72, y=off(126)), dict(rows=3, ldx=72, ldy=72, y=off(130)),
                dict(rows=3, ldx=72, ldy=80, y=off(128)), dict(rows=2, ldx=128, ldy=128, y=off(256 + 120)), dict(x=off(16), y=off(14))):
        assert fwd(**bad) == _lib.INVALID_INPUT and b"overlaps" in msg.value, bad
    assert L.q4_linear_pack(None, p, p, 8, 64, 32, None, msg, 128) == _lib.INVALID_INPUT
    assert L.q4_linear_pack(p, None, p, 8, 64, 32, None, msg, 128) == _lib.INVALID_INPUT
    assert L.q4_linear_quantize(None, p, 8, 64, 32, None, msg, 128) == _lib.INVALID_INPUT
    assert L.q4_linear_dequantize(p, None, 8, 64, 32, None, msg, 128) == _lib.INVALID_INPUT
    assert L.q4_linear_quantize(p, p, 8, 64, 48, None, msg, 128) == _lib.INVALID_CONFIG


# ---- against 64 bits ------------------------------------------------------------------------------------------------
def _layer(d_in, d_out, group, seed):
    from rustingbrain_b200.q4_linear import Q4Linear
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (d_out, d_in), device="cuda", generator=g).to(torch.int8)
    scales = (torch.rand(d_out, d_in // group, device="cuda", generator=g) + 0.1).bfloat16()
    layer = Q4Linear(d_in, d_out, group_size=group)
    layer.set_codes(codes, scales)
    return layer, codes.double() * scales.double().repeat_interleave(group, dim=1)


def _check(y, x, w):
    """Codes, scales and activations are exact.  The tensor core adds 16 products and the sum so far, each cut off at 2^-23 of the largest; then
    one f32 rounding (2^-24) per group, and the rounding of y to its type."""
    want = x.double() @ w.t()
    most = x.double().abs() @ w.abs().t()
    tol = want.abs() * torch.finfo(y.dtype).eps / 2 * 1.0001 + most * x.shape[1] * 1.2 * 2.0 ** -23
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() - tol).max())
    if y.dtype == torch.float32 and want.numel() > 64:       # the roundings are many and independent: far below that bound together
        assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -21


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d_in,d_out,group", [
    (1, 32, 1, 32), (1, 96, 17, 32), (2, 64, 16, 64), (3, 128, 33, 128), (8, 1024, 300, 32), (9, 160, 64, 32), (16, 4096, 70, 64), (17, 384, 129, 128),
    (31, 2048, 48, 32), (33, 512, 257, 64), (64, 1024, 512, 128), (64, 96, 2000, 32), (65, 256, 40, 32), (130, 640, 100, 128), (1, 8192, 4099, 64),
    (5, 1408, 512, 32), (12, 2816, 1024, 64), (40, 5632, 96, 128)])
def test_sizes(dtype, rows, d_in, d_out, group):
    layer, w = _layer(d_in, d_out, group, rows + d_in)
    assert torch.equal(layer.weight().double(), w)
    x = torch.randn(rows, d_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    out = torch.full((rows + 2, d_out), 7.0, device="cuda", dtype=dtype)
    y = layer.forward(x, out=out[1:-1])
    _check(y, x, w)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())          # rows around the last one stay as they were
    assert torch.equal(layer.forward(x), y) and torch.equal(layer(x), y)      # the same order of sums every time


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_apart(dtype):
    layer, w = _layer(192, 50, 64, 1)
    wide = torch.full((11, 256), float("nan"), device="cuda", dtype=dtype)
    wide[:, 32:224] = torch.randn(11, 192, device="cuda").to(dtype)
    x = wide[:, 32:224]
    out = torch.zeros(11, 77, device="cuda", dtype=dtype)
    y = layer.forward(x, out=out[:, 3:53])
    _check(y, x, w)
    assert float(out[:, :3].abs().max()) == 0 and float(out[:, 53:].abs().max()) == 0
    one = wide[4:5, 32:224]
    assert torch.equal(layer.forward(one), y[4:5])
    with pytest.raises(InvalidInput):
        layer.forward(wide[:, 33:225])                    # rows off the 16-byte boundary
    with pytest.raises(InvalidInput):
        layer.forward(wide[:, 32:225])
    with pytest.raises(InvalidInput):
        layer.forward(x.half())
    with pytest.raises(InvalidInput):
        layer.forward(x, out=torch.zeros(11, 51, device="cuda", dtype=dtype))
    with pytest.raises(InvalidInput):
        layer.forward(x.cpu())
    with pytest.raises(InvalidInput):
        layer.forward(wide.t()[:192])
    assert layer.forward(x[:0]).shape == (0, 50)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [4, 20, 64])
def test_infinities_and_nan_reach_their_rows_only(dtype, rows):
    layer, w = _layer(256, 40, 32, 5)
    x = torch.randn(rows, 256, device="cuda").to(dtype)
    clean = layer.forward(x)
    x[1, 17], x[2, 200] = float("inf"), float("nan")
    x[3] = 0
    x[3, 5] = torch.finfo(dtype).max / 1024
    y = layer.forward(x)
    ref = x.double() @ w.t()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[4:], clean[4:])
    assert bool(y[2].isnan().all())
    inf = ref[1].isinf()
    assert bool(inf.any()) and torch.equal(y[1][inf].double(), ref[1][inf]) and bool(y[1][~inf].isnan().all())
    assert float(((y[3].double() - ref[3]).abs() / ref[3].abs().clamp(min=1)).max()) <= torch.finfo(dtype).eps


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantisation_is_the_stated_rule(group):
    from rustingbrain_b200.q4_linear import Q4Linear
    d_in, d_out = 3 * 128, 37
    g = np.random.Generator(np.random.Philox(11))
    w = g.standard_normal((d_out, d_in)).astype(np.float32)
    w[3, :group] = 0
    w[4, :group] *= np.float32(1e-30)
    w[5, 2] = 1e30
    layer = Q4Linear(d_in, d_out, group_size=group)
    assert float(layer.weight().abs().max()) == 0
    layer.set_weight(torch.from_numpy(w).cuda())
    top = np.abs(w.reshape(d_out, -1, group)).max(axis=2) / np.float32(7)
    scale = torch.from_numpy(top).bfloat16().float().numpy()
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.clip(np.rint(w.reshape(d_out, -1, group) / scale[:, :, None]), -8, 7)
    code[scale == 0] = 0
    assert np.array_equal(layer.weight().cpu().numpy(), (code * scale[:, :, None]).reshape(d_out, d_in).astype(np.float32))
    w[6, 1], w[7, 0] = np.nan, np.inf
    layer.set_weight(torch.from_numpy(w).cuda())
    back = layer.weight()
    assert bool(back[6:8, :group].isnan().all()) and bool(back[8:].isfinite().all()) and bool(back[6:8, group:].isfinite().all())
    y = layer.forward(torch.ones(1, d_in, device="cuda"))
    assert bool(y[0, 6:8].isnan().all()) and int(y.isnan().sum()) == 2


@pytest.mark.gpu
def test_streams_graphs_and_errors():
    from rustingbrain_b200.q4_linear import Q4Linear
    layer, w = _layer(1024, 1000, 32, 9)
    other, w2 = _layer(960, 64, 64, 10)
    x = torch.randn(3, 1024, device="cuda").bfloat16()
    want = layer.forward(x)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        assert torch.equal(layer.forward(x), want)
    with torch.cuda.graph(graph, stream=side):
        y = layer.forward(x)
        z = other.forward(y[:, 40:])                      # rows of another layer's output, 16-byte aligned
    x.copy_(torch.randn(3, 1024, device="cuda").bfloat16())
    graph.replay()
    torch.cuda.synchronize()
    _check(y, x, w)
    _check(z, y[:, 40:], w2)
    for bad in ((100, 4, 32), (64, 0, 32), (64, 4, 16)):
        with pytest.raises(InvalidConfig):
            Q4Linear(bad[0], bad[1], group_size=bad[2])
    for codes, scales in ((torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.bfloat16)),
                          (torch.zeros(4, 64, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, device="cuda")),
                          (torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(InvalidInput):
            Q4Linear(64, 4).set_codes(codes, scales)
    with pytest.raises(InvalidInput):
        Q4Linear(64, 4).set_weight(torch.zeros(4, 64, device="cuda").bfloat16())


@pytest.mark.gpu
def test_rows_of_x_and_y_side_by_side_in_one_buffer():
    layer, w = _layer(64, 40, 32, 21)
    buf = torch.randn(5, 112, device="cuda", generator=torch.Generator(device="cuda").manual_seed(22)).bfloat16()
    x, y = buf[:, :64], buf[:, 64:104]
    rest = buf[:, 104:].clone()
    want = layer(x)
    layer(x, out=y)
    assert torch.equal(y, want) and torch.equal(buf[:, 104:], rest)
    _check(y, x, w)
    with pytest.raises(InvalidInput, match="overlaps"):
        layer(x, out=buf[:, 60:100])


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 4, 2.0 ** 10, 2.0 ** 17])
def test_an_outlier_whose_codes_are_zero(group, ratio):
    """bf16: a code enters as code + 8, so a channel costs its group accuracy whatever its codes.  A product of the tensor core adds 16 numbers
    and the sum so far, each cut off at 2^-23 of the largest, which is at most 15 times the group's sum of |x|; group / 16 products: 17 * 15 / 16 *
    group * 2^-23, below group * 2^-19, of scale * sum |x|.  That is the header's bound; the mean over channels stays far below it."""
    from rustingbrain_b200.q4_linear import Q4Linear
    g = torch.Generator(device="cuda").manual_seed(31)
    d_in, d_out, rows = 512, 200, 9
    codes = torch.randint(-8, 8, (d_out, d_in), device="cuda", generator=g).to(torch.int8)
    codes[:, 77] = 0
    scales = (torch.rand(d_out, d_in // group, device="cuda", generator=g) + 0.1).bfloat16()
    layer = Q4Linear(d_in, d_out, group_size=group)
    layer.set_codes(codes, scales)
    w = codes.double() * scales.double().repeat_interleave(group, dim=1)
    x = torch.randn(rows, d_in, device="cuda", generator=g).bfloat16()
    x[:, 77] = ratio
    y, want = layer.forward(x), x.double() @ w.t()
    sums = x.double().abs().view(rows, -1, group).sum(2)                        # [rows, groups]
    cut = (sums @ scales.double().t()) * group * 2.0 ** -19
    tol = want.abs() * 2.0 ** -8 + cut + (x.double().abs() @ w.abs().t()) * d_in * 2.0 ** -24
    assert bool(((y.double() - want).abs() <= tol).all())
    # a half step of bf16 and, of outputs of 4.6 * sqrt(512) scales, the outlier's part: 2^-23 of 8 ratio for each of group / 16 products
    rel = float((y.double() - want).norm() / want.norm())
    assert rel <= 2.0 ** -8 + ratio * 8 * 2.0 ** -23 * (group / 16) / (4.6 * 512 ** 0.5) * 2, rel


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,d_in,group", [(torch.float32, 9, 16384, 32), (torch.float32, 16, 16416, 32), (torch.float32, 17, 65536, 128),
                                                   (torch.float32, 1, 65536, 64), (torch.bfloat16, 9, 49152, 32), (torch.bfloat16, 16, 65536, 64),
                                                   (torch.bfloat16, 40, 65536, 128), (torch.bfloat16, 1, 65504, 32)])
def test_rows_of_very_many_channels(dtype, rows, d_in, group):
    """Where fewer than 16 (or 8) rows fit a pass."""
    layer, w = _layer(d_in, 3, group, 32)
    x = torch.randn(rows, d_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(33)).to(dtype)
    out = torch.full((rows + 2, 3), 7.0, device="cuda", dtype=dtype)
    y = layer.forward(x, out=out[1:-1])
    want = x.double() @ w.t()
    most = x.double().abs() @ w.abs().t()
    # as in _check, with the groups' roundings counted as the 2^-24 each that they are: at most one for every 32 channels
    tol = want.abs() * torch.finfo(dtype).eps / 2 * 1.0001 + most * ((17 + 15 * 17) * (group / 16) * 2.0 ** -23 + d_in / 32 * 2.0 ** -24)
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() - tol).max())
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())
    assert torch.equal(layer.forward(x), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d_in", [(4, 256), (20, 1024)])
def test_a_huge_channel_that_no_weight_takes_leaves_the_others_alone(dtype, rows, d_in):
    """Activations of 2^39 to 2^126 in a group whose scales are 0, beside others of 2^-6: the row's result is that of the others."""
    from rustingbrain_b200.q4_linear import Q4Linear
    g = torch.Generator(device="cuda").manual_seed(30)
    codes = torch.randint(-8, 8, (96, d_in), device="cuda", generator=g).to(torch.int8)
    scales = (torch.rand(96, d_in // 32, device="cuda", generator=g) + 0.1).bfloat16()
    scales[:, 1] = 0
    layer = Q4Linear(d_in, 96, group_size=32)
    layer.set_codes(codes, scales)
    w = codes.double() * scales.double().repeat_interleave(32, dim=1)
    x = (torch.randn(rows, d_in, device="cuda", generator=g) * 2.0 ** -6).to(dtype)
    clean = layer.forward(x)
    for r, e in enumerate((38, 39, 60, 126)):
        x[r, 32 + 7 * r] = 1.5 * 2.0 ** e
    y = layer.forward(x)
    _check(y, x, w)
    assert torch.equal(y[4:], clean[4:])
