"""The norm and linear operators on streams that change between calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def off_boundary(x):
    """The same rows, not at 16-byte boundaries."""
    buf = torch.zeros((x.shape[0], x.shape[1] + 3), dtype=x.dtype, device=x.device)
    buf[:, :-3] = x
    return buf[:, :-3]


@pytest.mark.parametrize("widths", [(1, 1), (900, 3), (300, 1100), (1100, 1100)])
def test_converted_rows_on_two_streams_of_one_runtime(widths):
    # float32 and unaligned x are copied first: calls that are not waited for, on two streams in turn, the second
    # pair of widths growing the memory of the copies between them
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    rt, streams = WideMoeRuntime.compile_with_fused_gate_up(0), [torch.cuda.Stream() for _ in range(2)]
    try:
        w = [randn((4096, 2048), 1 + i, 0.02) for i in range(2)]
        x = [randn((t, 2048), 3 + i) for i, t in enumerate(widths)]
        want = [rt.linear(xi, wi).output for xi, wi in zip(x, w)]
        forms = [[xi.float(), off_boundary(xi)] for xi in x]
        out = [[torch.empty_like(y) for _ in range(6)] for y in want]
        torch.cuda.synchronize()
        for _ in range(10):
            for i in range(6):
                for s, wi, form, o in zip(streams, w, forms, out):
                    rt.set_stream(s)
                    rt.linear(form[i % 2], wi, out=o[i], asynchronous=True)
            torch.cuda.synchronize()
            for o, y in zip(out, want):
                for got in o:
                    assert torch.equal(got, y)
                    got.zero_()
            torch.cuda.synchronize()
        assert rt.error_flags() == 0
    finally:
        torch.cuda.synchronize()
        rt.close()
