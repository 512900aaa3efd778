"""``fp8_linear`` under autograd on the CPU: the library's calls are taken by a stand-in that computes nothing, so
what is checked is which calls are made, what they are given, and what autograd makes of them."""

from __future__ import annotations

from collections import Counter

import pytest
import torch

from moss_offload import _native, fp8_kernels as fp8


class _Library:
    """Every entry point: counts the call and keeps its last arguments."""

    def __init__(self):
        self.calls, self.last = Counter(), {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] += 1
            self.last[name] = args
            return 256 if name.endswith("_bytes") else 0

        return call


@pytest.fixture
def library(monkeypatch):
    library = _Library()
    monkeypatch.setattr(fp8._native, "load", lambda: library)
    monkeypatch.setattr(fp8, "_elsewhere", lambda tensor: False)
    monkeypatch.setattr(fp8, "_stream", lambda tensor: 0)
    fp8._workspace_bytes.cache_clear()
    yield library
    fp8._workspace_bytes.cache_clear()


def _operands(*lead, dtype=torch.float32):
    return torch.zeros(*lead, 144, dtype=dtype).requires_grad_(), torch.zeros(32, 144).requires_grad_()


# ---- second derivatives ---------------------------------------------------------------------------


def test_a_graph_through_a_trained_weights_backward_is_refused(library) -> None:
    """The incoming gradient of a sum needs no graph, but the tokens' gradient depends on the weight: a penalty on
    it would lose its term in the weight's gradient."""

    for wanted in (0, 1, (0, 1)):
        leaves = _operands(5)
        y = fp8.fp8_linear(*leaves)
        inputs = [leaves[i] for i in (wanted if isinstance(wanted, tuple) else (wanted,))]
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(y.sum(), inputs, create_graph=True)
    tokens, master = _operands(5)
    with pytest.raises(RuntimeError):
        fp8.fp8_linear(tokens, master).square().sum().backward(create_graph=True)


def test_first_derivatives_and_constant_ones_are_not(library) -> None:
    tokens, master = _operands(5)
    grads = torch.autograd.grad(fp8.fp8_linear(tokens, master).sum(), [tokens, master])
    assert [g.shape for g in grads] == [tokens.shape, master.shape]
    # nothing that the gradient depends on wants one
    (grad,) = torch.autograd.grad(fp8.fp8_linear(tokens, master.detach()).sum(), [tokens], create_graph=True)
    assert not grad.requires_grad
    (grad,) = torch.autograd.grad(fp8.fp8_linear(tokens.detach(), master).sum(), [master], create_graph=True)
    assert not grad.requires_grad


# ---- a frozen weight ------------------------------------------------------------------------------


def _frozen():
    return torch.zeros(32, 144).to(torch.float8_e4m3fn), torch.ones(1, 2)


def test_a_frozen_weight_or_scale_that_wants_a_gradient_is_refused(library) -> None:
    """Both go to the kernels by address: a learnable scale would get no gradient."""

    weight, scale = _frozen()
    tokens, gradient = torch.zeros(4, 144), torch.zeros(4, 32)
    learnt = scale.clone().requires_grad_()
    calls = [
        (fp8.fp8_linear_forward, (tokens, weight, learnt)),
        (fp8.fp8_linear_backward, (gradient, weight, learnt)),
        (fp8.fp8_linear, (tokens, weight, learnt)),
        (fp8.fp8_linear, (tokens.clone().requires_grad_(), weight, learnt)),
        (fp8.fp8_linear, (tokens, weight, (2 * learnt))),
        (fp8.fp8_linear, (tokens, weight.clone().requires_grad_(), scale)),
        (fp8.fp8_linear_forward, (tokens, weight.clone().requires_grad_(), scale)),
    ]
    for call, operands in calls:
        with pytest.raises(RuntimeError, match="graph"):
            call(*operands)
    assert not library.calls
    with torch.no_grad():  # no graph is wanted
        fp8.fp8_linear(tokens, weight, learnt)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(scale, torch.ones_like(scale))
        with pytest.raises(RuntimeError, match="graph"):
            fp8.fp8_linear_forward(tokens, weight, dual)


def test_a_frozen_weight_gives_the_tokens_their_gradient(library) -> None:
    weight, scale = _frozen()
    tokens = torch.zeros(4, 144).requires_grad_()
    (grad,) = torch.autograd.grad(fp8.fp8_linear(tokens, weight, scale).sum(), [tokens])
    assert grad.shape == tokens.shape and library.calls["mo_fp8_linear_backward"] == 1


# ---- no tokens ------------------------------------------------------------------------------------


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
@pytest.mark.parametrize("trained", [False, True])
def test_no_tokens_have_gradients_without_a_launch(library, lead, trained) -> None:
    tokens, master = _operands(*lead)
    bias = torch.zeros(32).requires_grad_()
    operands = (tokens, master, None, bias) if trained else (tokens, *_frozen(), bias)
    y = fp8.fp8_linear(*operands)
    assert y.shape == (*lead, 32)
    wanted = [tokens, bias, *([master] if trained else [])]
    grads = torch.autograd.grad(y.sum(), wanted)
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    assert not any(g.any() for g in grads)
    assert not [name for name in library.calls if "linear" in name or "gradient" in name]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_tokens_weight_gradient_of_pairs_is_zero(library, dtype) -> None:
    pairs = [fp8.fp8_quantize_columns(torch.zeros(0, features)) for features in (32, 144)]
    out = torch.ones(32, 144, dtype=dtype)
    got = fp8.fp8_weight_gradient(*pairs, rows=0, dtype=dtype, out=out)
    assert got.data_ptr() == out.data_ptr() and not out.any()


# ---- a vector of tokens ---------------------------------------------------------------------------


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("trained", [False, True])
def test_a_vector_of_tokens_is_one_row(library, trained, biased) -> None:
    tokens, master = _operands()
    bias = torch.zeros(32).requires_grad_() if biased else None
    operands = (tokens, master, None, bias) if trained else (tokens, *_frozen(), bias)
    y = fp8.fp8_linear(*operands)
    assert y.shape == (32,)
    wanted = [tokens, *([bias] if biased else []), *([master] if trained else [])]
    grads = torch.autograd.grad(y.sum(), wanted)
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    if biased:
        assert torch.equal(grads[1], torch.ones(32))
    assert library.last["mo_fp8_linear_backward"][3] == 1
    assert not trained or library.last["mo_fp8_weight_gradient"][8] == 1


def test_a_vectors_pair_is_taken_and_read_back(library) -> None:
    pair = fp8.fp8_quantize_rows(torch.zeros(144))
    assert pair[0].shape == (144,) and pair[1].shape == (1, 2)
    assert fp8.fp8_linear_forward(pair, *_frozen()).shape == (32,)
    assert fp8.fp8_decode(*pair).shape == (144,)


# ---- without a graph ------------------------------------------------------------------------------


def test_evaluation_on_a_trained_weight_makes_no_columns(library) -> None:
    """The transposed copy is the weight gradient's alone."""

    tokens, master = _operands(5)
    bias = torch.zeros(32).requires_grad_()
    for mode in (torch.no_grad, torch.inference_mode):
        library.calls.clear()
        with mode():
            y = fp8.fp8_linear(tokens, master, None, bias)
        assert y.shape == (5, 32) and not y.requires_grad
        assert library.calls["mo_fp8_linear_forward"] == library.calls["mo_fp8_quantize_weight"] == 1
        assert not library.calls["mo_fp8_quantize"]
    with torch.enable_grad():
        fp8.fp8_linear(tokens, master, None, bias)
    assert library.calls["mo_fp8_quantize"] == 1 and library.last["mo_fp8_quantize"][7]


# ---- workspaces -----------------------------------------------------------------------------------


def test_a_workspace_that_could_not_be_sized_is_asked_for_again(library) -> None:
    weight, scale = _frozen()
    tokens = torch.zeros(4, 144)
    answers = [_native.MO_FP8_NO_SIZE, 4096]
    library.mo_fp8_workspace_bytes = lambda *args: answers.pop(0)
    library.mo_last_error = lambda: b"no device"
    with pytest.raises(_native.EngineError, match="no device"):
        fp8.fp8_linear_forward(tokens, weight, scale)
    assert not library.calls["mo_fp8_linear_forward"]
    for _ in range(2):  # and kept then
        fp8.fp8_linear_forward(tokens, weight, scale)
        assert library.last["mo_fp8_linear_forward"][14] == 4096
    assert not answers


@pytest.mark.skipif(torch.cuda.is_available(), reason="asks a library without a device")
def test_the_library_tells_a_failure_from_no_room() -> None:
    lib = _native.load()
    assert lib.mo_fp8_workspace_bytes(_native.MO_FP8_FORWARD, 4, 144, 32, 1, 0, 1) == _native.MO_FP8_NO_SIZE
    assert lib.mo_last_error()
    for sizes in ((4, 144, 1 << 21), (4, 1 << 21, 32), (4, 0, 32), (1 << 31, 144, 32)):
        assert lib.mo_fp8_workspace_bytes(_native.MO_FP8_FORWARD, *sizes, 0, 0, 1) == 0


# ---- biases ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_bias_goes_to_the_kernel_unrounded(library, dtype, bias_dtype) -> None:
    weight, scale = _frozen()
    bias = torch.ones(32, dtype=bias_dtype)
    fp8.fp8_linear_forward(torch.zeros(4, 144, dtype=dtype), weight, scale, bias)
    address, kinds = (library.last["mo_fp8_linear_forward"][i] for i in (10, 12))
    assert kinds & 0xFF == _native.DTYPE_CODES[dtype]
    if bias_dtype == dtype:
        assert address == bias.data_ptr()
    assert bool(kinds & _native.MO_FP8_BIAS_F32) == (bias_dtype != dtype or bias_dtype == torch.float32)


def test_the_library_takes_a_float32_bias_by_its_alignment() -> None:
    lib = _native.load()
    for kinds, bias, message in [(1, 4098, None), (1 | _native.MO_FP8_BIAS_F32, 4098, b"bias"), (1, 4097, b"bias"),
                                 (1 | _native.MO_FP8_BIAS_F32, 4100, None), (7 | _native.MO_FP8_BIAS_F32, 4096, b"type")]:
        # one that passes ends at the device or at the workspace of no bytes
        call = [4096, 0, 1, 4, 64, 64, 4096, 4096, 0, 32, bias, 4096, kinds, 4096, 0, 0]
        status = lib.mo_fp8_linear_forward(*call)
        assert status != 0
        assert (message in lib.mo_last_error()) if message else (b"bias" not in lib.mo_last_error()), (kinds, bias)


# ---- reading back ---------------------------------------------------------------------------------


def test_values_whose_rows_overlap_are_copied_to_be_read_back(library) -> None:
    """The kernel takes rows a row's length apart or more."""

    row = torch.zeros(1, 144).to(torch.float8_e4m3fn)
    windows = torch.zeros(400).to(torch.float8_e4m3fn).as_strided((4, 144), (16, 1))
    for values in (row.expand(4, -1), windows, row.expand(2, 3, 144).flatten(0, 1)):
        scales = torch.ones(values.shape[0], 2)
        assert fp8.fp8_decode(values, scales).shape == values.shape
        assert library.last["mo_fp8_decode"][1] == 144
    apart = torch.zeros(4, 160).to(torch.float8_e4m3fn)[:, :144]
    fp8.fp8_decode(apart, torch.ones(4, 2))
    assert library.last["mo_fp8_decode"][:2] == (apart.data_ptr(), 160)
