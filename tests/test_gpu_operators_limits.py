"""The linear operators where their arithmetic ends: infinities, the activations' tails and long sums.

Tolerances, derived before the first run.  One f32 operation is off by at most 2^-24 relative, expf and
__fdividef by 2 ulps (2^-22), and below f32's smallest normal value by whole steps of 2^-149.  A tensor core
adds 16 products to its accumulator with an error of at most 2^-23 of the sum, so sums of one sign in
segments of 512 columns are within 32 * 2^-23, and every f32 addition that joins them adds 2^-24.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    r = WideMoeRuntime.compile_with_fused_gate_up(0)
    r.set_stream(torch.cuda.current_stream())
    yield r
    r.close()


def uniform(shape, seed, dtype, low, high):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda").uniform_(low, high, generator=g).to(dtype)


def of_bias(rt, values, act, width=1):
    """The activation of these f32 values: zero products, the values as the bias."""
    x = torch.zeros((width, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros((values.numel(), 64), dtype=torch.bfloat16, device="cuda")
    got = rt.linear(x, w, bias=values, activation=act, out_dtype=torch.float32, asynchronous=True).output
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("width", [1, 40])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_an_infinite_sum_stays_infinite(rt, act, width):
    # from 25 on every activation is the value itself, to f32, and far below zero it is zero
    v = torch.tensor([25.0, math.inf, 3.4e38, 1e19, 0.0, -1e19, -3.4e38], device="cuda")
    got = of_bias(rt, v, act, width)
    assert torch.equal(got, (v if act == "none" else v.clamp_min(0)).expand(width, -1))
    assert rt.error_flags() & 32  # an infinity is reported


@pytest.mark.parametrize("act,low,high", [("silu", -110.0, -60.0), ("gelu_tanh", -11.0, -8.0), ("gelu", -15.0, -10.0)])
def test_activation_tails_keep_their_digits(rt, act, low, high):
    v = torch.linspace(low, high, 4001, device="cuda")
    d = v.double()
    if act == "silu":
        ref, rel = d * torch.exp(d) / (1 + torch.exp(d)), torch.zeros_like(d)
    elif act == "gelu_tanh":
        # the exponent is six f32 roundings from the value: |u| times their relative error
        u = 2 * math.sqrt(2 / math.pi) * (d + 0.044715 * d ** 3)
        ref, rel = d * torch.exp(u) / (1 + torch.exp(u)), u.abs() * 6 * 2.0 ** -24
    else:
        # the exponent is -v^2 log2(e) / 2 after three roundings, constant included; the polynomial is 6.6e-8 off
        # and takes eleven roundings in its last steps' size
        ref, rel = 0.5 * d * torch.erfc(-d / math.sqrt(2)), d * d / 2 * 3 * 2.0 ** -24 + 12 * 2.0 ** -24 + 1e-7
    # exp, a product, a quotient, and the sum below it; then whole steps, which the value multiplies
    bound = (rel + 6 * 2.0 ** -23) * ref.abs() + (2 * d.abs() + 4) * 2.0 ** -149
    got = of_bias(rt, v, act)[0].double()
    over = (got - ref).abs() - bound
    at = int(over.argmax())
    assert over.max().item() <= 0, f"{act} of {v[at].item()}: {got[at].item()}, not {ref[at].item()}"


def long_product(x, w):
    """x W^T in 64 bits, in pieces of the columns."""
    got = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
    for k in range(0, x.shape[1], 1 << 16):
        got += x[:, k:k + (1 << 16)].double() @ w[:, k:k + (1 << 16)].double().t()
    return got


@pytest.mark.parametrize("width", [1, 8, 9, 16])
@pytest.mark.parametrize("rows,cols", [(8, 1 << 20), (2400, 65536), (600, 16384 + 8), (40, 8192)])
def test_long_f32_sums_of_few_tokens_keep_their_digits(rt, width, rows, cols):
    # sums of one sign: nothing cancels, so the error of the sum is the output's
    x, w = uniform((width, cols), 1, torch.bfloat16, 0.5, 1.0), uniform((rows, cols), 2, torch.bfloat16, 0.5, 1.0)
    ref = long_product(x, w)
    got = rt.linear(x, w, out_dtype=torch.float32).output.double()
    # eight warps at least share the columns; joining them and up to eight splits is 16 additions
    bound = 32 * 2.0 ** -23 + (cols / 512 / 8 + 16) * 2.0 ** -24
    assert ((got - ref).abs() / ref).max().item() <= bound


@pytest.mark.parametrize("dtype,cols", [("f16", 1 << 18), ("f16", 16384), ("bf16", 1 << 19), ("bf16", 131072)])
def test_long_16_bit_sums_of_many_tokens_keep_their_digits(rt, dtype, cols):
    # off by the one rounding and by a quarter of it at most
    t = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    x, w = uniform((136, cols), 3, t, 0.5, 1.0), uniform((136, cols), 4, t, 2.0 ** -6, 2.0 ** -5)
    ref = long_product(x, w)
    got = rt.linear(x, w).output.double()
    half = torch.finfo(t).eps / 2
    assert ((got - ref).abs() / ref).max().item() <= half * 1.25
