"""8-bit floating point on the GPU: quantizers and read-back against the definition, bit for bit; the products,
forward, input and weight gradients, against 64 bits within the bound of their sums and roundings; groups
that are empty, tiny, huge or not finite; views, streams, graphs, gradients."""

from __future__ import annotations

import pytest
import torch

from moss_offload import _native, fp8_kernels as fp8

import fp8_model as model
from gpu_util import requires_gpu

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _matrix(rows, cols, dtype, seed=0, gain=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + cols)
    x = torch.randn(rows, cols, device=DEV, generator=g)
    return (x * torch.exp(gain * torch.randn(cols, device=DEV, generator=g))).to(dtype)


def _bytes(scales):
    return scales.contiguous().view(torch.uint8).to(torch.int64)


def _check_rows(values, scales, x):
    want, exponent = model.row_groups(x)
    assert torch.equal(_bytes(scales), exponent + 127)
    assert torch.equal(values[:, : x.shape[1]].double(), want)


# ---- quantizing and reading back -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (2, 128), (77, 144), (128, 64), (129, 272), (300, 1040), (512, 640), (4097, 4128)])
def test_quantizers_give_the_definition(rows, cols, dtype) -> None:
    x = _matrix(rows, cols, dtype)
    x[rows // 2] = 0
    x[:, cols // 2] *= 1e-4
    (rv, rs), (cv, cs) = fp8.fp8_quantize_both(x)
    _check_rows(rv, rs, x)
    _check_rows(cv, cs, x.t())
    assert cv.shape == (cols, -(-rows // 128) * 128) and not cv[:, rows:].float().any()
    alone = fp8.fp8_quantize_rows(x)
    turned = fp8.fp8_quantize_columns(x)
    for one, both in ((alone, (rv, rs)), (turned, (cv, cs))):
        assert torch.equal(one[0].view(torch.uint8), both[0].view(torch.uint8))
        assert torch.equal(_bytes(one[1]), _bytes(both[1]))
    for out in DTYPES:
        assert torch.equal(fp8.fp8_decode(rv, rs, dtype=out), model.read_back(x).to(out))
        assert torch.equal(fp8.fp8_decode(cv, cs, dtype=out, cols=rows), model.read_back(x.t()).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (16, 16), (128, 256), (139, 400), (640, 48)])
def test_weight_blocks_give_the_definition(rows, cols, dtype) -> None:
    w = _matrix(rows, cols, dtype) * 0.02
    values, scales = fp8.fp8_quantize_weight(w)
    want, exponent = model.block_groups(w)
    assert torch.equal(_bytes(scales), exponent + 127) and torch.equal(values.double(), want)
    for out in DTYPES:
        assert torch.equal(fp8.fp8_decode(values, scales, dtype=out), model.decoded(values, scales).to(out))
    arbitrary = scales.float() * 1.37
    back = fp8.fp8_decode(values, arbitrary, dtype=torch.float32)
    assert torch.equal(back, values.float() * model.spread(arbitrary, w.shape))


def test_every_bf16_value_rounds_to_nearest_even() -> None:
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).to(DEV)
    x = bits[torch.isfinite(bits) & (bits.abs() <= 448)]
    x = x[: x.numel() // 127 * 127].view(-1, 127)
    x = torch.cat((x, torch.full_like(x[:, :1], 448.0)), 1).contiguous()  # holds the scale at 1
    values, scales = fp8.fp8_quantize_rows(x)
    assert (_bytes(scales) == 127).all()
    assert torch.equal(values.double(), model.round_e4m3(x.double()))


@pytest.mark.parametrize("form", ["rows", "columns", "weight"])
def test_scale_at_the_edges_of_its_range(form) -> None:
    """Largest magnitudes on and next to 448 x 2^e, subnormal, the smallest and the largest float32."""

    peaks = [448.0, 448.0 * (1 + 2.0**-23), 449.0, 447.0, 224.0, 225.0, 1.75 * 2.0**-118, 1.75 * 2.0**-117, 2.0**-126,
             2.0**-149, 3.4e38, 1.7e38, 1.75 * 2.0**127, 0.0]
    for peak in peaks:
        x = torch.zeros(128, 128, device=DEV)
        x[5, 7] = -peak
        x[3, 7] = x[5, 9] = peak * 0.3
        if form == "weight":
            values, scales = fp8.fp8_quantize_weight(x)
            want, exponent = model.block_groups(x)
        else:
            values, scales = getattr(fp8, f"fp8_quantize_{form}")(x)
            want, exponent = model.row_groups(x if form == "rows" else x.t())
        assert torch.equal(_bytes(scales), exponent + 127), peak
        assert torch.equal(values.double(), want), peak


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_that_are_not_finite_read_back_as_nan(bad, dtype) -> None:
    x = _matrix(200, 272, dtype)
    x[150, 130] = bad
    (rv, rs), (cv, cs) = fp8.fp8_quantize_both(x)
    back, turned = fp8.fp8_decode(rv, rs), fp8.fp8_decode(cv, cs, cols=200).t()
    want = torch.zeros(200, 272, dtype=torch.bool, device=DEV)
    want[150, 128:256] = True
    assert torch.equal(back.isnan(), want)
    want = torch.zeros(200, 272, dtype=torch.bool, device=DEV)
    want[128:200, 130] = True
    assert torch.equal(turned.isnan(), want)
    w = _matrix(272, 272, dtype)
    w[200, 17] = bad
    block = fp8.fp8_decode(*fp8.fp8_quantize_weight(w)).isnan()
    want = torch.zeros(272, 272, dtype=torch.bool, device=DEV)
    want[128:256, :128] = True
    assert torch.equal(block, want)


def test_views_are_read_where_they_lie() -> None:
    base = _matrix(260, 3 * 160 + 8, torch.bfloat16)
    views = [base[:, 160:320], base[1::3, :144], base[:, 4:148], base[:144, :16].t(), base[:1].expand(40, -1)[:, :64],
             base[:256, :480].view(4, 64, 480)[1:3], base[::5, 488 - 16 :]]
    for view in views:
        values, scales = fp8.fp8_quantize_rows(view)
        assert values.shape == view.shape
        flat = view.reshape(-1, view.shape[-1])
        _check_rows(values.view(flat.shape), scales, flat)
        _check_rows(*fp8.fp8_quantize_columns(view), flat.t())


def test_no_rows() -> None:
    x = torch.empty(0, 256, dtype=torch.bfloat16, device=DEV)
    (rv, rs), (cv, cs) = fp8.fp8_quantize_both(x)
    assert rv.shape == (0, 256) and rs.shape == (0, 2) and cv.shape == (256, 0) and cs.shape == (256, 0)
    assert fp8.fp8_decode(rv, rs).shape == (0, 256)
    weight, scale = fp8.fp8_quantize_weight(_matrix(64, 256, torch.float32))
    assert fp8.fp8_linear_forward(x, weight, scale).shape == (0, 64)
    assert fp8.fp8_linear_backward(x[:, :64], weight, scale).shape == (0, 256)
    gradient = fp8.fp8_weight_gradient(x[:, :64], x)
    assert gradient.shape == (64, 256) and not gradient.any()


# ---- products --------------------------------------------------------------------------------------

# rows from one token up; features that end inside a group, a tile, a reduction step
SHAPES = [(1, 16, 16), (1, 3072, 512), (3, 128, 128), (16, 1040, 272), (17, 512, 3136), (32, 2048, 64), (33, 144, 400),
          (64, 640, 640), (65, 1152, 144), (130, 272, 1040), (256, 384, 256), (300, 1552, 528), (515, 912, 1296),
          (1100, 256, 2064), (2050, 1296, 784)]


def _weight_of(out_features, in_features, kind, seed=0):
    weight, scale = fp8.fp8_quantize_weight(0.02 * _matrix(out_features, in_features, torch.float32, seed, gain=0.3))
    if kind == "float32":
        g = torch.Generator(device="cuda").manual_seed(seed)
        scale = scale.float() * (1 + torch.rand(scale.shape, device=DEV, generator=g))
    return weight, scale


def _within(got, exact, a, b) -> None:
    assert got.shape == exact.shape
    worst = ((got.double() - exact).abs() / model.product_bound(got.dtype, a, b, exact)).max()
    assert worst <= 1, float(worst)


@pytest.mark.parametrize("kind", ["power", "float32"])
@pytest.mark.parametrize("rows,in_features,out_features", SHAPES)
def test_forward_matches_64_bits(rows, in_features, out_features, kind) -> None:
    weight, scale = _weight_of(out_features, in_features, kind, seed=rows)
    b = model.decoded(weight, scale).t().contiguous()
    for dtype in DTYPES:
        tokens = _matrix(rows, in_features, dtype, seed=1)
        bias = _matrix(1, out_features, dtype, seed=2)[0]
        a = model.read_back(tokens)
        exact = a @ b
        got = fp8.fp8_linear_forward(tokens, weight, scale)
        assert got.dtype == dtype
        _within(got, exact, a, b)
        one = torch.ones(rows, 1, device=DEV, dtype=torch.float64)
        _within(fp8.fp8_linear_forward(tokens, weight, scale, bias), exact + bias.double(), torch.cat((a, one), 1),
                torch.cat((b, bias.double()[None]), 0))
        again = fp8.fp8_linear_forward(fp8.fp8_quantize_rows(tokens), weight, scale, dtype=dtype)
        assert torch.equal(again, got)


@pytest.mark.parametrize("kind", ["power", "float32"])
@pytest.mark.parametrize("rows,in_features,out_features", SHAPES)
def test_input_gradient_matches_64_bits(rows, in_features, out_features, kind) -> None:
    weight, scale = _weight_of(out_features, in_features, kind, seed=rows)
    b = model.decoded(weight, scale)
    for dtype in DTYPES:
        gradient = _matrix(rows, out_features, dtype, seed=3)
        a = model.read_back(gradient)
        got = fp8.fp8_linear_backward(gradient, weight, scale)
        assert got.dtype == dtype
        _within(got, a @ b, a, b)
        again = fp8.fp8_linear_backward(fp8.fp8_quantize_rows(gradient), weight, scale, dtype=dtype)
        assert torch.equal(again, got)


@pytest.mark.parametrize("rows,in_features,out_features", SHAPES)
def test_weight_gradient_matches_64_bits(rows, in_features, out_features) -> None:
    for dtype, out in ((torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.float16)):
        gradient, tokens = _matrix(rows, out_features, dtype, seed=4), _matrix(rows, in_features, dtype, seed=5)
        a, b = model.read_back(gradient.t()), model.read_back(tokens.t()).t().contiguous()
        got = fp8.fp8_weight_gradient(gradient, tokens, dtype=out)
        assert got.dtype == out
        _within(got, a @ b, a, b)
        pairs = fp8.fp8_quantize_columns(gradient), fp8.fp8_quantize_columns(tokens)
        assert torch.equal(fp8.fp8_weight_gradient(*pairs, rows=rows, dtype=out), got)


@pytest.mark.parametrize("kind", ["power", "float32"])
def test_calls_in_two_launches_match_64_bits(kind) -> None:
    """Rows past whole rounds of large tiles go to a second launch, its reduction split."""

    rows, in_features, out_features = 17792 - 5, 6144, 3072 - 16
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    plan = fp8.product_plan(rows, out_features, in_features, cus, float_scales=kind == "float32")
    assert len(plan) == 2
    weight, scale = _weight_of(out_features, in_features, kind, seed=3)
    tokens = _matrix(rows, in_features, torch.bfloat16, seed=1)
    bias = _matrix(1, out_features, torch.bfloat16, seed=2)[0]
    got = fp8.fp8_linear_forward(tokens, weight, scale, bias)
    b = model.decoded(weight, scale).t().contiguous()
    one = torch.ones(512, 1, device=DEV, dtype=torch.float64)
    edge = plan[0]["rows"]
    for part in (slice(0, 512), slice(edge - 256, edge + 256), slice(rows - 512, rows)):
        a = model.read_back(tokens[part])
        _within(got[part], a @ b + bias.double(), torch.cat((a, one), 1), torch.cat((b, bias.double()[None]), 0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_hot_operands_place_every_element(dtype) -> None:
    """The identity through the product reads the weight back, each element in its place, both ways."""

    for features, width in ((272, 400), (1040, 144)):
        weight, scale = _weight_of(width, features, "power", seed=7)
        whole = fp8.fp8_decode(weight, scale, dtype=dtype)
        eye = torch.eye(features, dtype=dtype, device=DEV)
        assert torch.equal(fp8.fp8_linear_forward(eye, weight, scale), whole.t())
        eye = torch.eye(width, dtype=dtype, device=DEV)
        assert torch.equal(fp8.fp8_linear_backward(eye, weight, scale), whole)
        x = model.read_back(_matrix(features, width, torch.float32).t()).t().to(dtype)
        eye = torch.eye(features, dtype=dtype, device=DEV)
        assert torch.equal(fp8.fp8_weight_gradient(eye, x, dtype=dtype), x.contiguous())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_not_finite_groups_reach_the_outputs_that_read_them(rows, dtype) -> None:
    weight, scale = _weight_of(272, 400, "power")
    tokens = _matrix(rows, 400, dtype)
    clean = fp8.fp8_linear_forward(tokens, weight, scale)
    tokens[rows - 1, 140] = float("nan")
    got = fp8.fp8_linear_forward(tokens, weight, scale)
    assert got[rows - 1].isnan().all() and torch.equal(got[: rows - 1], clean[: rows - 1])
    bad = scale.clone()
    bad.view(torch.uint8)[1, 2] = 255  # features 128 to 255, reduction 256 to 383
    got = fp8.fp8_linear_forward(_matrix(rows, 400, dtype), weight, bad)
    assert got[:, 128:256].isnan().all()
    assert torch.equal(got[:, :128], clean[:, :128]) and torch.equal(got[:, 256:], clean[:, 256:])
    back = fp8.fp8_linear_backward(_matrix(rows, 272, dtype), weight, bad)
    assert back[:, 256:384].isnan().all() and not back[:, :256].isnan().any() and not back[:, 384:].isnan().any()
    arbitrary = scale.float()
    arbitrary[0, 0] = float("inf")
    got = fp8.fp8_linear_forward(_matrix(rows, 400, dtype), weight, arbitrary)
    assert not got[:, :128].isfinite().any() and got[:, 128:].isfinite().all()


def test_scales_far_apart_stay_apart() -> None:
    """Rows and groups of very different size: each is read under its own scale."""

    weight, scale = _weight_of(256, 512, "power")
    tokens = _matrix(96, 512, torch.float32)
    tokens *= torch.exp2(torch.randint(-40, 40, (96, 4), device=DEV).float()).repeat_interleave(128, 1)
    a, b = model.read_back(tokens), model.decoded(weight, scale).t().contiguous()
    _within(fp8.fp8_linear_forward(tokens, weight, scale), a @ b, a, b)
    _within(fp8.fp8_linear_forward(tokens, weight, scale, dtype=torch.bfloat16), a @ b, a, b)


def test_operands_that_are_views_buffers_and_leading_shapes() -> None:
    weight, scale = _weight_of(144, 272, "power")
    fused = _matrix(2 * 50, 3 * 272, torch.bfloat16).view(2, 50, 3 * 272)
    for view in (fused[..., 272:544], fused[:, ::7, :272], fused[..., 8:280], fused[0, 0, :272]):
        want = fp8.fp8_linear_forward(view.contiguous(), weight, scale)
        got = fp8.fp8_linear_forward(view, weight, scale)
        assert got.shape == (*view.shape[:-1], 144) and torch.equal(got, want)
    tokens = fused[..., :272].reshape(100, 272)
    out = torch.full((100, 144), float("nan"), dtype=torch.bfloat16, device=DEV)
    assert fp8.fp8_linear_forward(tokens, weight, scale, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, fp8.fp8_linear_forward(tokens, weight, scale))
    values, scales = fp8.fp8_quantize_rows(tokens)
    loose = (values, scales.view(torch.uint8).clone().view(torch.float8_e8m0fnu))  # three bytes a row
    assert torch.equal(fp8.fp8_linear_forward(loose, weight, scale), out)


def test_the_same_call_gives_the_same_bits_on_any_stream() -> None:
    weight, scale = _weight_of(1040, 1552, "power")
    tokens, gradient = _matrix(333, 1552, torch.bfloat16), _matrix(333, 1040, torch.bfloat16)

    def calls():
        return [fp8.fp8_linear_forward(tokens, weight, scale), fp8.fp8_linear_backward(gradient, weight, scale),
                fp8.fp8_weight_gradient(gradient, tokens)]

    want = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [calls() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for each in got:
        assert all(torch.equal(a, b) for a, b in zip(each, want))


def test_calls_replay_from_a_graph() -> None:
    weight, scale = _weight_of(528, 1040, "power")
    tokens, gradient = _matrix(40, 1040, torch.bfloat16), _matrix(40, 528, torch.bfloat16)

    def calls():
        return (fp8.fp8_linear_forward(tokens, weight, scale), fp8.fp8_linear_backward(gradient, weight, scale),
                fp8.fp8_weight_gradient(gradient, tokens))

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for seed in range(3):
        tokens.copy_(_matrix(40, 1040, torch.bfloat16, seed=seed + 20))
        gradient.copy_(_matrix(40, 528, torch.bfloat16, seed=seed + 30))
        want = calls()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- gradients -------------------------------------------------------------------------------------


def _on_grid(rows, cols, seed):
    """Whole numbers up to 14 with a 14 in every group: e4m3 holds them and their neighbours exactly."""

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-6, 7, (rows, cols), device=DEV, generator=g).float()
    x[::16, :] = 14.0
    x[:, ::16] = 14.0
    return x


@pytest.mark.parametrize("trained", [False, True])
def test_gradients_are_the_formulas(trained) -> None:
    tokens = _matrix(2 * 75, 272, torch.bfloat16).view(2, 75, 272).requires_grad_()
    master = (0.02 * _matrix(144, 272, torch.float32)).requires_grad_()
    bias = _matrix(1, 144, torch.bfloat16)[0].requires_grad_()
    weight, scale = fp8.fp8_quantize_weight(master.detach())
    y = fp8.fp8_linear(tokens, master, None, bias) if trained else fp8.fp8_linear(tokens, weight, scale, bias)
    assert torch.equal(y, fp8.fp8_linear_forward(tokens.detach(), weight, scale, bias.detach()))
    gradient = _matrix(2 * 75, 144, torch.bfloat16, seed=9).view(2, 75, 144)
    wanted = [tokens, bias, *([master] if trained else [])]
    got = torch.autograd.grad(y, wanted, gradient)
    flat = gradient.view(150, 144)
    assert torch.equal(got[0], fp8.fp8_linear_backward(gradient, weight, scale))
    assert torch.allclose(got[1].double(), flat.double().sum(0), rtol=2.0**-8, atol=1e-4)
    if trained:
        want = fp8.fp8_weight_gradient(flat, tokens.detach().view(150, 272), dtype=torch.float32)
        assert got[2].dtype == master.dtype and torch.equal(got[2], want)


def test_gradients_are_the_differences() -> None:
    """On operands that 8 bits hold exactly, a step of one more keeps them exact, and the loss is linear in
    each: its central difference is the gradient to the last fp32 bit or so."""

    tokens, master, probe = _on_grid(32, 48, 1), _on_grid(64, 48, 2), _on_grid(32, 64, 3)
    leaves = [tokens.clone().requires_grad_(), master.clone().requires_grad_()]
    loss = (fp8.fp8_linear(leaves[0], leaves[1]) * probe).double().sum()
    grads = torch.autograd.grad(loss, leaves)

    def at(t, w):
        return float((fp8.fp8_linear(t, w).double() * probe.double()).sum())

    for which, (i, j) in [(0, (3, 5)), (0, (31, 47)), (0, (17, 2)), (1, (1, 1)), (1, (63, 46)), (1, (40, 7))]:
        values = []
        for step in (1.0, -1.0):
            moved = [tokens.clone(), master.clone()]
            moved[which][i, j] += step
            values.append(at(*moved))
        assert float(grads[which][i, j]) == pytest.approx((values[0] - values[1]) / 2, rel=1e-5)


def test_frozen_weight_saves_only_its_own_buffers() -> None:
    weight, scale = _weight_of(144, 272, "power")
    tokens = _matrix(64, 272, torch.bfloat16).requires_grad_()
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.data_ptr()) or t, lambda t: t):
        fp8.fp8_linear(tokens, weight, scale)
    assert set(saved) == {weight.data_ptr(), scale.data_ptr()}


def test_calls_that_kernels_cannot_take_raise_on_the_device() -> None:
    weight, scale = _weight_of(144, 272, "power")
    tokens = _matrix(8, 272, torch.bfloat16)
    cases = [
        lambda: fp8.fp8_linear_forward(tokens.requires_grad_(), weight, scale),
        lambda: fp8.fp8_linear_forward(tokens.detach(), weight.cpu(), scale.cpu()),
        lambda: fp8.fp8_linear_forward(tokens.detach(), weight, scale[:1]),
        lambda: fp8.fp8_linear_forward(tokens.detach(), weight, scale, out=torch.empty(8, 144, device=DEV)),
        lambda: fp8.fp8_linear_forward(tokens.detach(), weight, scale, bias=torch.ones(1, device=DEV)),
        lambda: fp8.fp8_linear_backward(tokens.detach(), weight, scale),
        lambda: fp8.fp8_weight_gradient(tokens.detach(), tokens.detach()[:4]),
    ]
    for case in cases:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            case()
    lib = _native.load()
    x = tokens.detach()
    y = torch.empty(8, 144, dtype=torch.bfloat16, device=DEV)
    status = lib.mo_fp8_linear_forward(x.data_ptr(), 0, 1, 8, 272, 272, weight.data_ptr(), scale.data_ptr(), 0, 144, 0,
                                       y.data_ptr(), 1, 0, 0, 0)
    assert status == _native.MO_E_INVALID and b"workspace" in lib.mo_last_error()
