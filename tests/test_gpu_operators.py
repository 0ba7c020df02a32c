"""The residual-norm-quantize operator, the 16-bit linear layer and the FP8
linear layer on codes, against their definitions in 64 bits.

Tolerances, derived before the first run.  One rounding to a type T is off by
at most eps(T) / 2 relative.  The norm's sum of squares is a chain of at most
32 + 5 + 16 f32 additions (threads, warp, CTA), so its root is within
53 / 2 * 2^-24 < 1.6e-6, and the five f32 operations after it add 3e-7: 2e-6.
A linear layer adds K products in steps of 16 (f32, truncation allowed:
2^-23 each), within (K / 16 + 16) 2^-23 sum|x w|; the activations are evaluated
to a few f32 ulps and their slopes are at most 1.13.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NORM_TOL = 2e-6


@pytest.fixture(scope="module")
def rt():
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    r = WideMoeRuntime.compile_with_fused_gate_up(0)
    r.set_stream(torch.cuda.current_stream())
    yield r
    r.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def wide(t, pad, fill=0.0):
    """The same values in rows of a wider buffer; (view, buffer)."""
    buf = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device=t.device)
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]], buf


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, ref, dtype, rel, slack=0.0):
    """|got - ref| <= rounding to dtype + rel |ref| + slack (elementwise)."""
    d = (got.double() - ref).abs()
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype)
    bound = (half_step(dtype) + rel) * (ref.abs() + slack) + slack + tiny
    worst = (d - bound).max().item() if d.numel() else -1.0
    assert worst <= 0, f"off by {worst:.3e} over the bound (largest difference {d.max().item():.3e})"


# ------------------------------------------------------------------ norm
def norm_reference(x, r, w, eps):
    s = (x.float() + r.float()).to(x.dtype) if r is not None else x
    v = s.double()
    y = v / (v.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    return s, y


def check_codes(codes, scales, y):
    rows, hidden = y.shape
    groups = -(-hidden // 128)
    full = torch.zeros((rows, groups * 128), dtype=torch.float64, device=y.device)
    full[:, :hidden] = y
    full = full.view(rows, groups, 128)
    ref = full.abs().amax(-1).clamp_min(1e-10) / 448.0
    assert ((scales.double() - ref).abs() <= (NORM_TOL + 2.0 ** -23) * ref).all()
    q = (full / ref[..., None]).view(rows, -1)[:, :hidden]
    d = (codes.view(torch.float8_e4m3fn).double() - q).abs()
    exponent = torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6)))
    half = 2.0 ** (exponent - 4)  # half a step of three mantissa bits, half of 2^-9 below 2^-6
    assert (d <= half + 3 * NORM_TOL * q.abs()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (1, 4096), (5, 128), (33, 200), (7, 2048), (2, 2056), (9, 5003),
                                         (4, 8192), (3, 16384), (2, 16383), (1500, 256)])
def test_norm_matches_its_definition(rt, rows, hidden, dtype):
    t = TYPES[dtype]
    x, r = randn((rows, hidden), 1, t, 3.0), randn((rows, hidden), 2, t, 3.0)
    w = randn((hidden,), 3, torch.bfloat16) + 1
    s, y = norm_reference(x, r, w, 1e-5)
    got = rt.add_rms_norm(x, w, 1e-5, residual=r, want_codes=True)
    assert torch.equal(got.sum, s)
    close(got.y, y, t, NORM_TOL)
    check_codes(got.codes, got.scales, y)
    # the same, asked for one at a time
    assert torch.equal(rt.add_rms_norm(x, w, 1e-5, residual=r).y, got.y)
    alone = rt.add_rms_norm(s, w, 1e-5, want_y=False, want_codes=True)
    assert alone.sum is None and alone.y is None
    assert torch.equal(alone.codes, got.codes) and torch.equal(alone.scales, got.scales)
    close(rt.add_rms_norm(x, w, 1e-5, residual=r, out_dtype=torch.float32).y, y, torch.float32, NORM_TOL)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,hidden,residual", [(4001, 512, True), (2500, 4096, True), (2500, 4096, False),
                                                  (700, 8192, True), (400, 16384, False), (300, 16384, True),
                                                  (2500, 1000, True), (2500, 1024, False)])
def test_norm_over_many_rows(rt, rows, hidden, residual, dtype):
    # several rows per CTA, in place over the stream
    t = TYPES[dtype]
    x, _ = wide(randn((rows, hidden), 13, t, 3.0), 8)
    r = randn((rows, hidden), 14, t, 3.0) if residual else None
    w = randn((hidden,), 15) + 1
    s, y = norm_reference(x, r, w, 1e-5)
    got = rt.add_rms_norm(x, w, 1e-5, residual=r, want_codes=True, in_place=residual)
    if residual:
        assert torch.equal(r, s)
    close(got.y, y, t, NORM_TOL)
    check_codes(got.codes, got.scales, y)


@pytest.mark.parametrize("wtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_norm_strides_and_weight_types(rt, pad, wtype):
    x, _ = wide(randn((13, 384), 4, torch.bfloat16), pad)
    r, buf = wide(randn((13, 384), 5, torch.bfloat16), pad + 8, 7.0)
    w = randn((384,), 6, TYPES[wtype]) + 1
    s, y = norm_reference(x, r, w, 1e-6)
    got = rt.add_rms_norm(x, w, 1e-6, residual=r, want_codes=True, in_place=True)
    assert got.sum is r and torch.equal(r, s)
    assert (buf[:, 384:] == 7.0).all()  # what lies between the rows stays
    close(got.y, y, torch.bfloat16, NORM_TOL)
    check_codes(got.codes, got.scales, y)


def test_norm_vector_and_element_paths_agree_with_an_offset_view(rt):
    flat = randn((5 * 512 + 1,), 7, torch.bfloat16)
    a, b = flat[:-1].view(5, 512), flat[1:].view(5, 512)  # b starts two bytes off a vector boundary
    w = torch.ones(512, device="cuda")
    for t in (a, b):
        _, y = norm_reference(t, None, w, 1e-5)
        got = rt.add_rms_norm(t, w, 1e-5, want_codes=True)
        close(got.y, y, torch.bfloat16, NORM_TOL)
        check_codes(got.codes, got.scales, y)


def test_norm_extremes(rt):
    w = torch.ones(256, device="cuda")
    # a row of zeros, squares beyond f32, squares below f32, one loud channel
    x = torch.zeros((5, 256), device="cuda")
    x[1] = randn((256,), 8) * 1e30
    x[2] = randn((256,), 9) * 1e-30
    x[3, 17] = 3e38
    x[4] = 1.0
    _, y = norm_reference(x, None, w, 1e-5)
    got = rt.add_rms_norm(x, w, 1e-5, want_codes=True)
    close(got.y, y, torch.float32, NORM_TOL)
    assert (got.codes[0] == 0).all() and (got.y[0] == 0).all()
    assert torch.allclose(got.scales[0].double(), torch.full((2,), 1e-10 / 448, dtype=torch.float64, device="cuda"))


def test_norm_matches_the_reference_norm_and_quantizer(rt):
    # pw_rms_norm rounds to bf16 between the products: two bf16 roundings apart
    x = randn((17, 1024), 10, torch.bfloat16)
    w = (randn((1024,), 11) + 1).to(torch.bfloat16)
    staged, _ = rt.rms_norm(x.float(), w, 1e-5)
    once = rt.add_rms_norm(x, w, 1e-5, out_dtype=torch.float32, want_codes=True)
    assert ((staged - once.y).abs() <= 2.01 * 2.0 ** -8 * once.y.abs()).all()
    # the codes are the quantizer's codes of the f32 output, bit for bit
    codes, scales = rt.quantize(once.y)
    assert torch.equal(codes, once.codes) and torch.equal(scales, once.scales)


def test_norm_flags_bad_rows_and_keeps_the_others(rt):
    from mimo_prismwing_b200.runtime import PrismwingError
    w = torch.ones(512, device="cuda")
    x = randn((6, 512), 12, torch.bfloat16)
    good = rt.add_rms_norm(x, w, 1e-5, want_codes=True)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[2, 5] = bad
        with pytest.raises(PrismwingError) as e:
            rt.add_rms_norm(z, w, 1e-5)
        assert e.value.kind == "nonfinite"
        a = rt.add_rms_norm(z, w, 1e-5, want_codes=True, asynchronous=True)
        torch.cuda.synchronize()
        assert rt.error_flags() & 2
        keep = torch.tensor([0, 1, 3, 4, 5], device="cuda")
        assert torch.equal(a.y[keep], good.y[keep]) and torch.equal(a.codes[keep], good.codes[keep])
    # an output beyond f16
    z = torch.zeros((1, 512), dtype=torch.float16, device="cuda")
    z[0, 0] = 1.0
    with pytest.raises(PrismwingError) as e:
        rt.add_rms_norm(z, torch.full((512,), 6e4, device="cuda"), 1e-5)
    assert e.value.kind == "nonfinite"


# ------------------------------------------------------------------ linear
# (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)): the left side loses its digits to cancellation for u < -1, even in
# 64 bits (2^-53 absolute is 2e-6 relative at u = -11); so does 1 + erf in the normal distribution function
ACTS = {"none": lambda v: v, "relu": lambda v: v.clamp_min(0), "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2)),
        "gelu_tanh": lambda v: v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
        "silu": lambda v: v * torch.sigmoid(v)}


def linear_reference(x, w, bias, act, res):
    v = x.double() @ w.double().t()
    if bias is not None:
        v = v + bias.double()
    v = ACTS[act](v)
    return v + res.double() if res is not None else v


def linear_slack(x, w, bias):
    k = x.shape[1]
    size = x.double().abs() @ w.double().abs().t() + (bias.double().abs() if bias is not None else 0)
    return 1.13 * (k / 16 + 16) * 2.0 ** -23 * size


SHAPES = [(1, 128, 64), (1, 1, 1), (1, 4096, 512), (2, 130, 72), (3, 77, 1003), (8, 256, 2048), (9, 1000, 136),
          (16, 384, 4096), (17, 129, 320), (31, 64, 64), (33, 512, 100), (64, 200, 1024), (65, 300, 64), (100, 136, 1000),
          (128, 128, 128), (129, 257, 65), (257, 640, 448), (300, 1000, 1003), (1000, 384, 512)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("width,rows,cols", SHAPES)
def test_linear_sums_are_exact_on_small_integers(rt, width, rows, cols, dtype):
    # products and sums of small integers are exact in f32: every index error shows
    t = TYPES[dtype]
    x, _ = wide(torch.randint(-4, 5, (width, cols), generator=gen(20), device="cuda").to(t), -cols % 8 + 8, float("nan"))
    w, _ = wide(torch.randint(-4, 5, (rows, cols), generator=gen(21), device="cuda").to(t), -cols % 8, float("nan"))
    out, buf = wide(torch.zeros((width, rows), device="cuda"), 5, 9.0)
    got = rt.linear(x, w, out_dtype=torch.float32, out=out)
    assert got.output is out
    assert torch.equal(out.double(), x.double() @ w.double().t())
    assert (buf[:, rows:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("width,rows,cols", [(1500, 2600, 64), (700, 4100, 72), (1500, 3001, 1003), (1030, 5130, 456),
                                             (2048, 4096, 1856), (129, 9500, 128), (200, 1000, 1003), (300, 600, 1992),
                                             (131, 256, 1536), (517, 4096, 520), (140, 200, 60)])
def test_wide_linear_sums_are_exact_on_small_integers(rt, width, rows, cols, dtype):
    # sums of products of -1, 0 and 1 stay below 2048: exact in f16 too
    t = TYPES[dtype]
    x, _ = wide(torch.randint(-1, 2, (width, cols), generator=gen(31), device="cuda").to(t), -cols % 8 + 8, float("nan"))
    w, _ = wide(torch.randint(-1, 2, (rows, cols), generator=gen(32), device="cuda").to(t), -cols % 8, float("nan"))
    out, buf = wide(torch.zeros((width, rows), device="cuda", dtype=torch.float16), 3, 9.0)
    rt.linear(x, w, out=out)
    assert torch.equal(out.float(), x.float() @ w.float().t())
    assert (buf[:, rows:] == 9.0).all()


@pytest.mark.parametrize("width,rows,cols", [(40, 300, 4096), (64, 1000, 1000), (100, 4096, 8192), (77, 5001, 1003),
                                             (200, 130, 16384), (300, 512, 640)])
def test_linear_f32_keeps_its_digits(rt, width, rows, cols):
    # sums in segments of at most 512 columns (32 steps, 2^-23 each at worst), joined in f32: the relative error of
    # the whole output stays below 32 2^-23 and the joins' K / 512 2^-24
    x, w = randn((width, cols), 33, torch.bfloat16), randn((rows, cols), 34, torch.bfloat16, cols ** -0.5)
    w, _ = wide(w, -cols % 8)
    ref = x.double() @ w.double().t()
    got = rt.linear(x, w, out_dtype=torch.float32).output.double()
    assert ((got - ref).norm() / ref.norm()).item() <= 32 * 2.0 ** -23 + cols / 512 * 2.0 ** -24


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("width,rows,cols", [(1, 520, 1024), (5, 130, 200), (40, 257, 512), (200, 300, 776),
                                             (520, 260, 1024)])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "bf16")])
def test_linear_epilogue_matches_its_definition(rt, width, rows, cols, act, dtype, out):
    t, o = TYPES[dtype], TYPES[out]
    x, w = randn((width, cols), 22, t), randn((rows, cols), 23, t, 2 * cols ** -0.5)
    bias, res = randn((rows,), 24, o), randn((width, rows), 25, o, 3.0)
    slack = linear_slack(x, w, bias)
    for b, r in ((bias, res), (None, res), (bias, None)):
        ref = linear_reference(x, w, b, act, r)
        got = rt.linear(x, w, bias=b, activation=act, residual=r, out_dtype=o).output
        assert got.dtype == o
        # f32 evaluation of the activation and the two additions
        close(got, ref, o, 1e-6, slack + 1e-6 * (3 + (r.double().abs() if r is not None else 0)))


def test_linear_activations_far_from_zero(rt):
    # one product per output: the activation alone, from -30 to 30 and at the ends
    v = torch.cat([torch.linspace(-30, 30, 509, device="cuda"), torch.tensor([0.0, -1e4, 1e4], device="cuda")])
    v = v.to(torch.float16)
    x = torch.ones((1, 8), dtype=torch.float16, device="cuda")
    w = torch.zeros((512, 8), dtype=torch.float16, device="cuda")
    w[:, 3] = v
    for act, f in ACTS.items():
        got = rt.linear(x, w, activation=act, out_dtype=torch.float32).output[0].double()
        ref = f(v.double())
        # a few ulps of f32; exp(-v)'s argument carries |v| 2^-24 into the tail's relative error
        over = (got - ref).abs() - (2e-6 * (1 + v.double().abs().clamp_max(100)) * ref.abs() + 1e-30)
        at = int(over.argmax())
        assert over.max().item() <= 0, f"{act} of {v[at].item()}: {got[at].item()}, not {ref[at].item()}"


def test_linear_in_place_residual_f32_rows_and_unaligned_rows(rt):
    x, w = randn((37, 512), 26, torch.bfloat16), randn((260, 512), 27, torch.bfloat16, 0.05)
    h = randn((37, 260), 28, torch.bfloat16)
    ref = rt.linear(x, w, residual=h.clone()).output
    got = rt.linear(x, w, residual=h, out=h)
    assert got.output is h and torch.equal(h, ref)
    # f32 rows of bf16 values, as the other calls return them, are exact
    assert torch.equal(rt.linear(x.float(), w, out_dtype=torch.bfloat16).output, rt.linear(x, w).output)
    # rows off the 16-byte boundary are copied first
    odd, _ = wide(x, 3)
    assert torch.equal(rt.linear(odd, w).output, rt.linear(x, w).output)
    flat = torch.cat([torch.zeros(1, dtype=torch.bfloat16, device="cuda"), x.flatten()])
    assert torch.equal(rt.linear(flat[1:].view(37, 512), w).output, rt.linear(x, w).output)


@pytest.mark.parametrize("width", [1, 8, 16, 50, 200])
def test_linear_tokens_do_not_mix(rt, width):
    # a bad token leaves the others alone, and each is as it is alone
    from mimo_prismwing_b200.runtime import PrismwingError
    x, w = randn((width, 712), 29, torch.bfloat16), randn((333, 712), 30, torch.bfloat16, 0.05)
    good = rt.linear(x, w).output
    z = x.clone()
    z[0, 100] = float("nan")
    with pytest.raises(PrismwingError) as e:
        rt.linear(z, w)
    assert e.value.kind == "nonfinite"
    got = rt.linear(z, w, asynchronous=True).output
    torch.cuda.synchronize()
    assert rt.error_flags() & 32
    assert torch.equal(got[1:], good[1:]) and torch.isnan(got[0]).all()


def test_linear_overflow_of_the_output_type(rt):
    from mimo_prismwing_b200.runtime import PrismwingError
    x = torch.full((2, 64), 200.0, dtype=torch.float16, device="cuda")
    w = torch.full((8, 64), 200.0, dtype=torch.float16, device="cuda")
    assert (rt.linear(x, w, out_dtype=torch.float32).output == 64 * 4e4).all()
    with pytest.raises(PrismwingError):
        rt.linear(x, w)


# ------------------------------------------------------------------ FP8
def fp8_case(width, rows, cols, seed):
    from mimo_prismwing_b200 import synth
    from mimo_prismwing_b200.runtime import WideProjectionBinding
    w = randn((rows // 128, 128, cols // 128, 128), seed, scale=cols ** -0.5)
    scale = w.abs().amax((1, 3)) / 448
    codes = (w / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, cols)
    return randn((width, cols), seed + 1), WideProjectionBinding(codes.contiguous(), scale.contiguous())


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("width", [1, 3, 8, 9, 16, 17, 31, 32, 100, 129, 300, 1500])
def test_fp8_codes_match_fp8_linear(rt, width, layout):
    # two f32 evaluations of the same sum: each within linear_slack of it.  sum |x w| comes from the same
    # projection of the magnitudes.
    from mimo_prismwing_b200.runtime import WideProjectionBinding
    rows, scale_rows = [(640, 5), (13568, 108), (14848, 116)][layout]
    cols = 1024 if layout == 0 else 4096
    x = randn((width, cols), 40)
    w = torch.randint(0, 256, (rows, cols), generator=gen(41), device="cuda", dtype=torch.uint8)
    w[(w & 0x7f) == 0x7f] = 0x30
    b = WideProjectionBinding(w, randn((scale_rows, cols // 128), 42).abs() * 1e-3)
    codes, scales = rt.quantize(x)
    ref = rt.execute_fp8_linear(x, b, layout=layout, f32_output=True).output.double()
    size = rt.execute_fp8_linear(x.abs(), WideProjectionBinding(w & 0x7f, b.scale), layout=layout, f32_output=True).output
    got = rt.fp8_linear_codes(codes, scales, b, layout=layout).output.double()
    assert ((got - ref).abs() <= 2 * (cols / 16 + 16) * 2.0 ** -23 * 1.001 * size.double()).all()


@pytest.mark.parametrize("width", [1, 7, 13, 33, 64, 128, 140, 256, 300, 600])
@pytest.mark.parametrize("rows,cols", [(128, 128), (384, 640), (256, 4096), (9600, 256), (4096, 2048), (4864, 384)])
def test_fp8_sums_are_exact_on_small_integers(rt, width, rows, cols):
    # codes of small integers, scales powers of two: every sum is exact in f32, every index error shows
    from mimo_prismwing_b200.runtime import WideProjectionBinding
    x = torch.randint(-3, 4, (width, cols), generator=gen(43), device="cuda").float()
    w = torch.randint(-3, 4, (rows, cols), generator=gen(44), device="cuda").float()
    xs = 2.0 ** torch.randint(-1, 2, (width, cols // 128), generator=gen(45), device="cuda").float()
    ws = 2.0 ** torch.randint(-1, 2, (rows // 128, cols // 128), generator=gen(46), device="cuda").float()
    b = WideProjectionBinding(w.to(torch.float8_e4m3fn).view(torch.uint8), ws)
    out, buf = wide(torch.zeros((width, rows), device="cuda"), 5, 9.0)
    rt.fp8_linear_codes(x.to(torch.float8_e4m3fn).view(torch.uint8), xs, b, out=out)
    ref = (x.double() * xs.double().repeat_interleave(128, 1)) @ \
        (w.double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)).t()
    assert torch.equal(out.double(), ref)
    assert (buf[:, rows:] == 9.0).all()


@pytest.mark.parametrize("width", [16, 31, 128, 300, 1030])
@pytest.mark.parametrize("rows,cols", [(128, 128), (4864, 384), (19200, 256)])
@pytest.mark.parametrize("out,res", [("f32", "f32"), ("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f32"), ("f32", "f16")])
def test_fp8_residual_and_output_boxes(rt, width, rows, cols, out, res):
    # small integers again, so that one rounding is all there is: many tiles per CTA,
    # residuals of the output's element size and of the other, packed, strided and in place
    from mimo_prismwing_b200.runtime import WideProjectionBinding
    x = torch.randint(-3, 4, (width, cols), generator=gen(246), device="cuda").float()
    w = torch.randint(-3, 4, (rows, cols), generator=gen(247), device="cuda").float()
    r = torch.randint(-99, 100, (width, rows), generator=gen(248), device="cuda").to(TYPES[res])
    bias = torch.randint(-9, 10, (rows,), generator=gen(249), device="cuda").float()
    b = WideProjectionBinding(w.to(torch.float8_e4m3fn).view(torch.uint8), torch.ones(rows // 128, cols // 128, device="cuda"))
    codes, scales = x.to(torch.float8_e4m3fn).view(torch.uint8), torch.ones(width, cols // 128, device="cuda")
    ref = (x.double() @ w.double().t() + bias.double() + r.double()).to(TYPES[out])
    kw = dict(bias=bias, out_dtype=TYPES[out])
    assert torch.equal(rt.fp8_linear_codes(codes, scales, b, residual=r, **kw).output, ref)
    assert torch.equal(rt.fp8_linear_codes(codes, scales, b, residual=wide(r, 16)[0], **kw).output, ref)
    assert torch.equal(rt.fp8_linear_codes(codes, scales, b, residual=wide(r, 3)[0], **kw).output, ref)
    if out == res:
        rt.fp8_linear_codes(codes, scales, b, residual=r, out=r, **kw)
        assert torch.equal(r, ref)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("width,rows,cols", [(1, 256, 128), (8, 4096, 2048), (5, 128, 4096), (20, 384, 384), (32, 256, 1024),
                                             (203, 640, 512), (260, 128, 128)])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
def test_fp8_epilogue_matches_its_definition(rt, width, rows, cols, act, out):
    o = TYPES[out]
    x, b = fp8_case(width, rows, cols, 50)
    codes, scales = rt.quantize(x)
    bias = randn((rows,), 52, o)
    res, _ = wide(randn((width, rows), 53, o, 3.0), 0 if width == 32 else 3)
    y, buf = wide(torch.zeros((width, rows), dtype=o, device="cuda"), 0 if width == 32 else 1, 5.0)
    xd = codes.view(torch.float8_e4m3fn).double() * scales.double().repeat_interleave(128, 1)
    wd = b.weight.view(torch.float8_e4m3fn).double() * b.scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    slack = linear_slack(xd, wd, bias)
    for bb, r in ((bias, res), (None, res), (bias, None)):
        ref = linear_reference(xd, wd, bb, act, r)
        got = rt.fp8_linear_codes(codes, scales, b, bias=bb, activation=act, residual=r, out_dtype=o, out=y).output
        close(got, ref, o, 1e-6, slack + 1e-6 * (3 + (r.double().abs() if r is not None else 0)))
        assert (buf[:, rows:] == 5.0).all()
    # onto the stream itself
    rt.fp8_linear_codes(codes, scales, b, bias=bias, activation=act, residual=res, out=res)
    close(res, linear_reference(xd, wd, bias, act, randn((width, rows), 53, o, 3.0)), o, 1e-6,
          slack + 1e-6 * (3 + res.double().abs()))


def test_fp8_codes_over_many_tokens(rt):
    x, b = fp8_case(6144 + 70, 256, 128, 54)
    codes, scales = rt.quantize(x)
    ref = rt.execute_fp8_linear(x, b, f32_output=True).output
    # one block: one product, one promotion
    assert torch.equal(rt.fp8_linear_codes(codes, scales, b).output, ref)


# ------------------------------------------------------------------ together
def chain(rt, h, x, wo, norm, b, bias, asynchronous):
    """Attention output projection onto the stream, norm into codes, FP8 projection: a layer's half."""
    attn = rt.linear(x, wo, residual=h, asynchronous=asynchronous).output
    n = rt.add_rms_norm(attn, norm, 1e-5, want_y=False, want_codes=True, asynchronous=asynchronous)
    out = rt.fp8_linear_codes(n.codes, n.scales, b, bias=bias, activation="silu", out_dtype=torch.bfloat16,
                              asynchronous=asynchronous).output
    return attn, n, out


@pytest.mark.parametrize("width", [1, 8, 40, 260])
def test_chain_matches_its_definition_eager_streamed_and_captured(rt, width):
    hid, inner = 512, 768
    h, x = randn((width, hid), 60, torch.bfloat16, 2.0), randn((width, 1024), 61, torch.bfloat16)
    wo, norm = randn((hid, 1024), 62, torch.bfloat16, 1 / 32), randn((hid,), 63, torch.bfloat16, 0.1) + 1
    _, b = fp8_case(1, inner, hid, 64)
    bias = randn((inner,), 65, torch.bfloat16)
    attn, n, out = chain(rt, h, x, wo, norm, b, bias, False)
    close(attn, linear_reference(x, wo, None, "none", h), torch.bfloat16, 1e-6,
          linear_slack(x, wo, None) + 1e-6 * (3 + h.double().abs()))
    _, y = norm_reference(attn, None, norm, 1e-5)
    check_codes(n.codes, n.scales, y)
    xd = n.codes.view(torch.float8_e4m3fn).double() * n.scales.double().repeat_interleave(128, 1)
    wd = b.weight.view(torch.float8_e4m3fn).double() * b.scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    close(out, linear_reference(xd, wd, bias, "silu", None), torch.bfloat16, 1e-6, linear_slack(xd, wd, bias) + 3e-6)

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    rt.set_stream(side)
    try:
        with torch.cuda.stream(side):
            again = chain(rt, h, x, wo, norm, b, bias, True)
            side.synchronize()
            assert torch.equal(again[0], attn) and torch.equal(again[2], out)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                captured = chain(rt, h, x, wo, norm, b, bias, True)
            for seed in (66, 67):  # new inputs in the captured buffers
                x.copy_(randn(tuple(x.shape), seed, torch.bfloat16))
                side.synchronize()
                g.replay()
                side.synchronize()
                eager = chain(rt, h, x, wo, norm, b, bias, True)
                side.synchronize()
                assert torch.equal(captured[0], eager[0]) and torch.equal(captured[2], eager[2])
                assert torch.equal(captured[1].codes, eager[1].codes)
            assert rt.error_flags() == 0
    finally:
        torch.cuda.synchronize()
        rt.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("width", [3, 70])
def test_host_rows(rt, width):
    h, x = randn((width, 256), 70, torch.bfloat16), randn((width, 200), 71, torch.bfloat16)
    w, norm = randn((256, 200), 72, torch.bfloat16, 0.07), torch.ones(256, device="cuda")
    _, b = fp8_case(1, 128, 256, 73)
    bias = randn((128,), 74)
    want = rt.linear(x, w, residual=h, out_dtype=torch.float32).output
    got = rt.linear(x.cpu(), w, residual=h.cpu(), out_dtype=torch.float32)
    assert not got.output.is_cuda and torch.equal(got.output, want.cpu())
    assert torch.equal(rt.linear(x.float().cpu().numpy(), w, residual=h.cpu()).output, want.cpu())
    dev = rt.add_rms_norm(h, norm, residual=h, want_codes=True)
    cpu = rt.add_rms_norm(h.cpu(), norm, residual=h.cpu(), want_codes=True)
    for a, c in zip((dev.sum, dev.y, dev.codes, dev.scales), (cpu.sum, cpu.y, cpu.codes, cpu.scales)):
        assert torch.equal(a.cpu(), c)
    want = rt.fp8_linear_codes(dev.codes, dev.scales, b, bias=bias, activation="gelu").output
    assert torch.equal(rt.fp8_linear_codes(cpu.codes, cpu.scales, b, bias=bias, activation="gelu").output, want.cpu())


def test_default_stream_is_ordered_with_torch(rt):
    # set_stream(torch's default stream) runs the calls on that very stream
    w = randn((4096, 1024), 75, torch.bfloat16, 0.03)
    x = randn((64, 1024), 76, torch.bfloat16)
    want = rt.linear(x, w).output
    for _ in range(20):
        z = torch.zeros_like(x)
        z.copy_(x)
        got = rt.linear(z, w, asynchronous=True).output
        z.zero_()
        assert torch.equal(got, want)


# ------------------------------------------------------------------ refusals
def test_refusals(rt):
    from mimo_prismwing_b200.runtime import PrismwingError
    x, w = randn((4, 64), 80, torch.bfloat16), randn((32, 64), 81, torch.bfloat16)
    n = torch.ones(64, device="cuda")

    def refused(f, kind):
        with pytest.raises(PrismwingError) as e:
            f()
        assert e.value.kind == kind, str(e.value)

    refused(lambda: rt.linear(x[:0], w), "shape")
    refused(lambda: rt.linear(x, w.float()), "argument")
    refused(lambda: rt.linear(x.half(), w), "argument")
    refused(lambda: rt.linear(x, w[:, :63].contiguous()), "shape")
    refused(lambda: rt.linear(x[:, :63], w[:, :63].contiguous()), "unsupported")  # weight rows off 16 bytes
    refused(lambda: rt.linear(x, w.cpu()), "argument")
    refused(lambda: rt.linear(x.expand(4, 64)[:1].expand(4, 64), w), "argument")
    refused(lambda: rt.linear(x, w, activation="swish"), "argument")
    refused(lambda: rt.linear(x, w, bias=torch.ones(31, device="cuda")), "argument")
    refused(lambda: rt.linear(x, w, residual=torch.ones(4, 31, device="cuda")), "shape")
    buf = torch.zeros((5, 32), dtype=torch.bfloat16, device="cuda")
    refused(lambda: rt.linear(x, w, residual=buf[:4], out=buf[1:]), "argument")
    refused(lambda: rt.linear(x, w, out=x[:, :32]), "argument")
    refused(lambda: rt.linear(x.cpu(), w, asynchronous=True), "argument")
    refused(lambda: rt.add_rms_norm(x[:0], n), "shape")
    refused(lambda: rt.add_rms_norm(x, n, 0.0), "argument")
    refused(lambda: rt.add_rms_norm(x, n, float("nan")), "argument")
    refused(lambda: rt.add_rms_norm(x, n, want_y=False), "argument")
    refused(lambda: rt.add_rms_norm(x, n[:63]), "argument")
    refused(lambda: rt.add_rms_norm(x, n, residual=x.float()), "argument")
    refused(lambda: rt.add_rms_norm(x, n, residual=x[:3]), "shape")
    refused(lambda: rt.add_rms_norm(x, n, out_dtype=torch.float16), "argument")
    refused(lambda: rt.add_rms_norm(torch.ones((1, 16385), device="cuda"), torch.ones(16385, device="cuda")), "shape")
    y, b = fp8_case(4, 128, 128, 82)
    codes, scales = rt.quantize(y)
    refused(lambda: rt.fp8_linear_codes(codes, scales[:, :0], b), "shape")
    refused(lambda: rt.fp8_linear_codes(codes[:0], scales[:0], b), "shape")
    refused(lambda: rt.fp8_linear_codes(codes.view(torch.int8), scales, b), "argument")
    refused(lambda: rt.fp8_linear_codes(codes, scales.cpu(), b), "argument")
    refused(lambda: rt.fp8_linear_codes(codes, scales, b, layout=7), "argument")
    from mimo_prismwing_b200.runtime import WideProjectionBinding
    refused(lambda: rt.add_rms_norm(x, n, 1e-31), "argument")
    skew = torch.zeros(128 * 128 + 1, dtype=torch.uint8, device="cuda")[1:].view(128, 128)
    refused(lambda: rt.fp8_linear_codes(codes, scales, WideProjectionBinding(skew, b.scale)), "unsupported")
    flat = torch.zeros(4 * 128 + 1, dtype=torch.uint8, device="cuda")
    refused(lambda: rt.fp8_linear_codes(flat[1:].view(4, 128), scales, b), "unsupported")


def test_columns_of_one_buffer_are_not_overlapping(rt):
    # q and its residual side by side in one buffer: same rows, other columns
    x, w = randn((6, 64), 83, torch.bfloat16), randn((32, 64), 84, torch.bfloat16)
    buf = randn((6, 96), 85, torch.bfloat16)
    want = rt.linear(x, w, residual=buf[:, :32].clone()).output
    rt.linear(x, w, residual=buf[:, :32], out=buf[:, 40:72])
    assert torch.equal(buf[:, 40:72], want)


# ------------------------------------------------------------------ streams, graphs, neighbours
class Layer:
    """Buffers of one decoder-like layer that a call chain runs over again and again, in place."""

    def __init__(self, width, seed):
        self.h, self.x = randn((width, 512), seed, torch.bfloat16, 2.0), randn((width, 1024), seed + 1, torch.bfloat16)
        self.wo = randn((512, 1024), seed + 2, torch.bfloat16, 1 / 32)
        self.up = randn((768, 512), seed + 3, torch.bfloat16, 1 / 23)
        self.down = randn((512, 768), seed + 4, torch.bfloat16, 1 / 64)
        self.norm = randn((512,), seed + 5, torch.bfloat16, 0.1) + 1
        _, self.b = fp8_case(1, 512, 512, seed + 6)

    def run(self, rt, wait):
        """Each call takes what the one before it wrote; all over h but the last."""
        def step(r):
            if wait:
                torch.cuda.synchronize()
            return r
        for _ in range(3):
            step(rt.linear(self.x, self.wo, residual=self.h, out=self.h, asynchronous=True))
            n = step(rt.add_rms_norm(self.h, self.norm, asynchronous=True))
            m = step(rt.linear(n.y, self.up, activation="silu", asynchronous=True))
            d = step(rt.linear(m.output, self.down, asynchronous=True))
            n = step(rt.add_rms_norm(d.output, self.norm, residual=self.h, in_place=True, want_codes=True, asynchronous=True))
            out = step(rt.fp8_linear_codes(n.codes, n.scales, self.b, residual=self.h, out=self.h, asynchronous=True))
        return out.output


@pytest.mark.parametrize("width", [1, 12, 40, 100, 300])
def test_two_runtimes_on_two_streams_at_once(width):
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    layers = [Layer(width, 200), Layer(width, 210)]
    rts = [WideMoeRuntime.compile_with_fused_gate_up(0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    try:
        want, start = [], [layer.h.clone() for layer in layers]
        torch.cuda.synchronize()
        for rt, s, layer in zip(rts, streams, layers):
            rt.set_stream(s)
            with torch.cuda.stream(s):
                want.append(layer.run(rt, True).clone())
        torch.cuda.synchronize()
        for _ in range(3):
            for layer, h in zip(layers, start):
                layer.h.copy_(h)
            torch.cuda.synchronize()
            for rt, s, layer in zip(rts, streams, layers):
                with torch.cuda.stream(s):
                    layer.run(rt, False)
            torch.cuda.synchronize()
            for layer, w in zip(layers, want):
                assert torch.equal(layer.h, w)
        # both captured, replayed at once; inputs in place, so each replay starts over
        graphs = []
        for rt, s, layer in zip(rts, streams, layers):
            with torch.cuda.stream(s):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    layer.run(rt, False)
                graphs.append(g)
        for _ in range(3):
            for layer, h in zip(layers, start):
                layer.h.copy_(h)
            torch.cuda.synchronize()
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for layer, w in zip(layers, want):
                assert torch.equal(layer.h, w)
        assert all(rt.error_flags() == 0 for rt in rts)
    finally:
        torch.cuda.synchronize()
        for rt in rts:
            rt.close()


@pytest.mark.parametrize("width", [1, 12, 40, 100, 300])
def test_first_call_of_a_runtime_may_be_captured(width):
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    layer = Layer(width, 220)
    start = layer.h.clone()
    rt, s = WideMoeRuntime.compile_with_fused_gate_up(0), torch.cuda.Stream()
    try:
        rt.set_stream(s)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                layer.run(rt, False)
            g.replay()
            s.synchronize()
            got = layer.h.clone()
            layer.h.copy_(start)
            layer.run(rt, False)
            s.synchronize()
        assert torch.equal(layer.h, got) and not torch.equal(got, start)
    finally:
        torch.cuda.synchronize()
        rt.close()


@pytest.mark.parametrize("width", [1, 12, 40, 100, 300])
def test_linear_leaves_what_is_not_its_own(rt, width):
    # NaN between the rows of x and the weight is not read into a sum, and what
    # lies between and behind the output's rows stays
    nan, guard = float("nan"), 7.0
    x, xb = wide(randn((width, 392), 230, torch.bfloat16), 8, nan)
    w, wb = wide(randn((200, 392), 231, torch.bfloat16, 0.05), 24, nan)
    want = rt.linear(x.contiguous(), w.contiguous()).output
    buf = torch.full((width + 2, 200 + 9), guard, dtype=torch.bfloat16, device="cuda")
    rt.linear(x, w, out=buf[1:-1, 3:203])
    assert torch.equal(buf[1:-1, 3:203], want)
    buf[1:-1, 3:203] = guard
    assert (buf == guard).all()
    assert torch.isnan(xb[:, 392:]).all() and torch.isnan(wb[:, 392:]).all()


@pytest.mark.parametrize("width", [1, 12, 40, 100, 300])
def test_fp8_leaves_what_is_not_its_own(rt, width):
    x, b = fp8_case(width, 384, 512, 232)
    codes, scales = rt.quantize(x)
    want = rt.fp8_linear_codes(codes, scales, b).output
    # the rows behind the last token hold NaN codes and scales
    more = torch.full((width + 130, 512), 0x7F, dtype=torch.uint8, device="cuda")
    some = torch.full((width + 130, 4), float("nan"), device="cuda")
    more[:width], some[:width] = codes, scales
    buf = torch.full((width + 2, 384 + 9), 7.0, device="cuda")
    rt.fp8_linear_codes(more[:width], some[:width], b, out=buf[1:-1, 3:387])
    assert torch.equal(buf[1:-1, 3:387], want)
    buf[1:-1, 3:387] = 7.0
    assert (buf == 7.0).all()
    # rows that start at 16-byte boundaries leave by another way
    for out, cols in ((torch.float32, 4), (torch.bfloat16, 8), (torch.float16, 16)):
        buf = torch.full((width + 2, 384 + 32), 7.0, dtype=out, device="cuda")
        rt.fp8_linear_codes(more[:width], some[:width], b, out=buf[1:-1, cols:cols + 384])
        assert torch.equal(buf[1:-1, cols:cols + 384], want.to(out))
        buf[1:-1, cols:cols + 384] = 7.0
        assert (buf == 7.0).all()


@pytest.mark.parametrize("rows,hidden", [(1, 512), (5, 513), (3000, 512), (3000, 520)])
def test_norm_over_its_input_and_beside_its_neighbours(rt, rows, hidden):
    # through the C call: y may be x itself
    from mimo_prismwing_b200.runtime import Norm, Rows, MEM_DEVICE
    w = randn((hidden,), 233) + 1
    x = randn((rows, hidden), 234, torch.bfloat16, 3.0)
    want = rt.add_rms_norm(x, w, 1e-5, want_codes=True)
    buf = torch.full((rows + 2, hidden + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    v = buf[1:-1, 8:8 + hidden]
    v.copy_(x)
    codes = torch.full((rows + 1, hidden), 9, dtype=torch.uint8, device="cuda")
    groups = -(-hidden // 128)
    scales = torch.full((rows + 1, groups), 9.0, device="cuda")
    torch.cuda.synchronize()
    at = Rows(v.data_ptr(), v.stride(0), 1, 0)
    norm = Norm(w.data_ptr(), hidden, 0, 1e-5)
    assert rt._L.pw_add_rms_norm(rt._rt, ctypes.addressof(norm), ctypes.addressof(at), None, rows, None,
                                 ctypes.addressof(at), codes.data_ptr(), scales.data_ptr(), MEM_DEVICE, None) == 0
    assert torch.equal(v, want.y)
    assert torch.equal(codes[:rows], want.codes) and torch.equal(scales[:rows], want.scales)
    assert (codes[rows] == 9).all() and (scales[rows] == 9).all()
    v.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("width", [1, 40, 300])
def test_graphs_that_convert_x_share_nothing(width):
    # two graphs of one runtime over float32 and unaligned rows, replayed at once
    # after a larger call has moved the runtime's own memory
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    rt, streams = WideMoeRuntime.compile_with_fused_gate_up(0), [torch.cuda.Stream() for _ in range(2)]
    w = [randn((512, 1024), 240 + i, torch.bfloat16, 0.03) for i in range(2)]
    x = [randn((width, 1024), 242 + i, torch.bfloat16).float() for i in range(2)]
    odd = [wide(t.bfloat16(), 3)[0] for t in x]
    try:
        outs, graphs = [], []
        torch.cuda.synchronize()
        for s, wi, xi, oi in zip(streams, w, x, odd):
            rt.set_stream(s)
            with torch.cuda.stream(s):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    outs.append([rt.linear(t, wi, out_dtype=torch.bfloat16, asynchronous=True).output
                                 for t in (xi, oi, xi, oi)])
                graphs.append(g)
        rt.set_stream(torch.cuda.current_stream())
        rt.linear(randn((3000, 4096), 244), randn((64, 4096), 245, torch.bfloat16))
        want = [rt.linear(xi.bfloat16(), wi).output for wi, xi in zip(w, x)]
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for got, ref in zip(outs, want):
                for y in got:
                    assert torch.equal(y, ref)
                    y.zero_()
            torch.cuda.synchronize()
    finally:
        torch.cuda.synchronize()
        rt.close()
