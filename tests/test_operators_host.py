"""Host-side checks of the norm and linear operators: descriptor layouts,
the clean failure of every entry point on a null runtime, and the Python
wrapper's refusals, none of which reaches the library."""
import ctypes
import re

import pytest
import torch


def test_descriptor_layouts_match_the_header():
    from mimo_prismwing_b200 import _lib
    from mimo_prismwing_b200 import runtime as R
    assert [f[0] for f in R.Rows._fields_] == ["data", "stride", "dtype", "reserved"]
    assert [f[0] for f in R.Dense._fields_] == ["weight", "stride", "rows", "cols", "dtype", "reserved"]
    assert [f[0] for f in R.Epilogue._fields_] == ["bias", "bias_dtype", "activation", "residual"]
    assert (ctypes.sizeof(R.Rows), ctypes.sizeof(R.Dense), ctypes.sizeof(R.Epilogue)) == (24, 32, 40)
    # the calls pack them by format
    W = R.WideMoeRuntime
    assert W._NORM_ARGS.size == ctypes.sizeof(R.Norm) + 4 * 24 == 120
    assert W._LINEAR_ARGS.size == 32 + 24 + 40 + 24 and W._CODES_ARGS.size == 40 + 24
    text = open(_lib.HEADER).read()

    def value(name):
        return int(re.search(r"#define %s (\d+)u" % name, text).group(1))

    for dtype, name in ((torch.float32, "F32"), (torch.bfloat16, "BF16"), (torch.float16, "F16")):
        assert R.DTYPES[dtype] == value("PW_DTYPE_" + name) == value("PW_NORM_" + name)
    for name, code in R.ACTIVATIONS.items():
        assert value("PW_ACT_" + name.upper()) == code


def test_null_runtime_fails_cleanly():
    import mimo_prismwing_b200 as m
    L = m.load()
    assert L.pw_add_rms_norm(None, None, None, None, 1, None, None, None, None, 0, None) == -1
    assert L.pw_linear(None, None, None, 1, None, None, 0, None) == -1
    assert L.pw_fp8_linear_codes(None, None, 0, None, None, 1, None, None, 0, None) == -1


@pytest.fixture
def rt():
    # no device here: a runtime object without a handle, for checks before the call
    import mimo_prismwing_b200 as m
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    r = WideMoeRuntime.__new__(WideMoeRuntime)
    r._L, r._rt, r.device, r._banks, r._bank_refs = m.load(), None, 0, [], []
    r._init_args()
    return r


def test_wrapper_refuses_before_the_call(rt):
    from mimo_prismwing_b200.runtime import PrismwingError
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    w = torch.zeros((32, 64), dtype=torch.bfloat16)

    def refused(f, match):
        with pytest.raises(PrismwingError, match=match):
            f()

    refused(lambda: rt.linear(x, w), "weight is on cpu")
    refused(lambda: rt.linear(x.to(torch.int32), w), "x must be float32")
    refused(lambda: rt.linear(x[0], w), "x must be 2-D")
    refused(lambda: rt.linear(x.t(), w), "contiguous rows")
    refused(lambda: rt.linear(x[:1].expand(4, 64), w), "contiguous rows")
    refused(lambda: rt.add_rms_norm(x, torch.ones(64)), "norm weight must be a contiguous")
    refused(lambda: rt.add_rms_norm(x, torch.ones(64, dtype=torch.float64)), "not torch.float64")
    refused(lambda: rt.fp8_linear_codes(x, torch.zeros((4, 1)), None), "codes must be uint8")
    refused(lambda: rt.fp8_linear_codes(torch.zeros((64, 4), dtype=torch.uint8).t(), torch.zeros((4, 1)), None),
            "contiguous")


def test_packed_descriptors_are_the_structures(rt):
    # a recording library on host tensors: what the calls pack is what the structures hold
    from mimo_prismwing_b200 import runtime as R
    seen = {}

    class Fake:
        def __getattr__(self, name):
            def call(_, *args):
                seen[name] = args
                return 0
            return call

    def at(kind, address):
        s = kind.from_address(address)
        return tuple(getattr(s, f) for f, *_ in kind._fields_ if f not in ("residual",))

    rt._L, rt.device = Fake(), -1
    buf = torch.zeros((3, 80), dtype=torch.bfloat16)
    x, w, h = buf[:, :64], torch.zeros((32, 64), dtype=torch.bfloat16), torch.zeros((3, 32))
    bias = torch.zeros(32, dtype=torch.float16)
    out = rt.linear(x, w, bias=bias, activation="silu", residual=h, out_dtype=torch.float32).output
    a = seen["pw_linear"]
    assert at(R.Dense, a[0]) == (w.data_ptr(), 64, 32, 64, 1, 0) and a[2] == 3
    assert at(R.Rows, a[1]) == (x.data_ptr(), 80, 1, 0)
    assert at(R.Epilogue, a[3]) == (bias.data_ptr(), 2, 4)
    assert at(R.Rows, a[3] + R.Epilogue.residual.offset) == (h.data_ptr(), 32, 0, 0)
    assert at(R.Rows, a[4]) == (out.data_ptr(), 32, 0, 0)
    n, r = torch.ones(64), torch.zeros((3, 64), dtype=torch.bfloat16)
    got = rt.add_rms_norm(x, n, 0.25, residual=r, want_codes=True, out_dtype=torch.float32)
    a = seen["pw_add_rms_norm"]
    assert at(R.Norm, a[0]) == (n.data_ptr(), 64, 0, 0.25) and a[3] == 3
    assert at(R.Rows, a[1]) == (x.data_ptr(), 80, 1, 0) and at(R.Rows, a[2]) == (r.data_ptr(), 64, 1, 0)
    assert at(R.Rows, a[4]) == (got.sum.data_ptr(), 64, 1, 0) and at(R.Rows, a[5]) == (got.y.data_ptr(), 64, 0, 0)
    assert a[6:8] == (got.codes.data_ptr(), got.scales.data_ptr())
    got = rt.add_rms_norm(x, n, want_y=False, want_codes=True)
    a = seen["pw_add_rms_norm"]
    assert a[2] is None and a[4] is None and a[5] is None and got.sum is None and got.y is None
    rt._L, rt.device = None, 0


def test_set_stream_names_torchs_default_stream(rt):
    # torch's default stream has handle 0, which the C ABI takes for the runtime's own stream
    class Fake:
        def __init__(self):
            self.seen = []

        def pw_set_stream(self, _, handle):
            self.seen.append(handle.value)
            return 0

    class Stream:
        def __init__(self, handle):
            self.cuda_stream = handle

    rt._L = Fake()
    rt.set_stream(None)
    rt.set_stream(Stream(0))
    rt.set_stream(Stream(1234))
    assert rt._L.seen == [None, 1, 1234]
    rt._L = None
