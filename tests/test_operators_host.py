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


def test_binding_fills_the_structures():
    # the compiled binding over recording entry points, on host tensors: the same
    # descriptors, and None for what it does not take
    from mimo_prismwing_b200 import _lib
    from mimo_prismwing_b200 import runtime as R
    vp, u32 = ctypes.c_void_p, ctypes.c_uint32
    seen, status = {}, [0]

    def at(kind, address):
        s = kind.from_address(address)
        return tuple(getattr(s, f) for f, *_ in kind._fields_ if f not in ("residual",))

    def rows(address):
        return at(R.Rows, address) if address else None

    def norm(rt, n, x, r, t, s, y, codes, scales, mem, stats):
        seen["norm"] = (rt, at(R.Norm, n), rows(x), rows(r), t, rows(s), rows(y), codes, scales, mem, stats)
        return status[0]

    def linear(rt, w, x, width, ep, y, mem, stats):
        seen["linear"] = (rt, at(R.Dense, w), rows(x), width, at(R.Epilogue, ep), rows(ep + R.Epilogue.residual.offset),
                          rows(y), mem, stats)
        return status[0]

    def codes(rt, w, layout, c, s, width, ep, y, mem, stats):
        seen["codes"] = (rt, at(R.Fp8Tensor, w), layout, c, s, width, at(R.Epilogue, ep),
                         rows(ep + R.Epilogue.residual.offset), rows(y), mem, stats)
        return status[0]

    types = [[vp, vp, vp, vp, u32, vp, vp, vp, vp, u32, vp], [vp, vp, vp, u32, vp, vp, u32, vp],
             [vp, vp, u32, vp, vp, u32, vp, vp, u32, vp]]
    entry = [ctypes.CFUNCTYPE(ctypes.c_int, *t)(f) for t, f in zip(types, (norm, linear, codes))]
    c = _lib.binding().Calls(77, -1, *[ctypes.cast(f, vp).value for f in entry])
    ASYNC = R.MEM_DEVICE | R.MEM_ASYNC
    buf = torch.zeros((3, 80), dtype=torch.bfloat16)
    x, w, h = buf[:, :64], torch.zeros((32, 64), dtype=torch.bfloat16), torch.zeros((3, 32))
    bias = torch.zeros(32, dtype=torch.float16)
    out = c.linear(x, w, bias, 4, h, torch.float32, None)
    assert out.shape == (3, 32) and out.dtype == torch.float32
    assert seen["linear"] == (77, (w.data_ptr(), 64, 32, 64, 1, 0), (x.data_ptr(), 80, 1, 0), 3, (bias.data_ptr(), 2, 4),
                              (h.data_ptr(), 32, 0, 0), (out.data_ptr(), 32, 0, 0), ASYNC, None)
    assert c.linear(x, w, None, 0, h, None, h) is h and seen["linear"][6] == (h.data_ptr(), 32, 0, 0)
    assert c.linear(x[:1], torch.nn.Parameter(w), None, 0, None, None, None).dtype == torch.bfloat16
    assert seen["linear"][2] == (x.data_ptr(), 0, 1, 0) and seen["linear"][5] == (None, 0, 0, 0)
    for bad in ((x[0], w, None, 0, None, None, None), (x, w.to(torch.float64), None, 0, None, None, None),
                (x[:1].expand(3, 64), w, None, 0, None, None, None), (x.t(), w, None, 0, None, None, None),
                (x, w[:, :63], None, 0, None, None, None), (x, w, bias[:31], 0, None, None, None),
                (x, w, None, None, None, None, None), (x, w, None, 0, h[:2], None, None),
                (x, w, None, 0, None, torch.int32, None), (x, w, None, 0, None, "float32", None),
                (x, w, None, 0, None, None, h[:, :31]), ([1], w, None, 0, None, None, None),
                (x.to_sparse(), w, None, 0, None, None, None), (x.to("meta"), w, None, 0, None, None, None), (x, w)):
        seen.clear()
        assert c.linear(*bad) is None and not seen
    n, r = torch.ones(64), torch.zeros((3, 64), dtype=torch.bfloat16)
    s, y, q, g = c.add_rms_norm(x, n, 0.25, r, True, True, torch.float32, False)
    assert seen["norm"] == (77, (n.data_ptr(), 64, 0, 0.25), (x.data_ptr(), 80, 1, 0), (r.data_ptr(), 64, 1, 0), 3,
                            (s.data_ptr(), 64, 1, 0), (y.data_ptr(), 64, 0, 0), q.data_ptr(), g.data_ptr(), ASYNC, None)
    assert (s.dtype, y.dtype, q.dtype, g.dtype) == (torch.bfloat16, torch.float32, torch.uint8, torch.float32)
    assert q.shape == (3, 64) and g.shape == (3, 1)
    s, y, q, g = c.add_rms_norm(x, n, 0.25, r, False, True, None, True)
    assert s is r and y is None and seen["norm"][5] == (r.data_ptr(), 64, 1, 0) and seen["norm"][6] is None
    s, y, q, g = c.add_rms_norm(x, n, 0.25, None, True, False, None, False)
    assert s is None and q is None and g is None and seen["norm"][3] is None and seen["norm"][7] is None
    for bad in ((x, n[:63], 0.25, r, True, True, None, False), (x, n, 1, r, True, True, None, False),
                (x, n, 0.25, r.float(), True, True, None, False), (x, n, 0.25, r[:2], True, True, None, False)):
        seen.clear()
        assert c.add_rms_norm(*bad) is None and not seen
    cd, sc = torch.zeros((3, 128), dtype=torch.uint8), torch.zeros((3, 1))
    fw, fs = torch.zeros((256, 128), dtype=torch.uint8), torch.zeros((2, 1))
    out = c.fp8_linear_codes(cd, sc, fw, fs, 0, None, 0, None, torch.float16, None)
    assert out.dtype == torch.float16
    assert seen["codes"] == (77, (fw.data_ptr(), fs.data_ptr(), 256, 128, 2, 1), 0, cd.data_ptr(), sc.data_ptr(), 3,
                             (None, 0, 0), (None, 0, 0, 0), (out.data_ptr(), 256, 2, 0), ASYNC, None)
    for bad in ((cd.to(torch.int8), sc, fw, fs), (cd, sc[:2], fw, fs), (cd, sc, fw[:, :64], fs), (cd[:, ::2], sc, fw, fs)):
        seen.clear()
        assert c.fp8_linear_codes(*bad, 0, None, 0, None, torch.float16, None) is None and not seen
    status[0] = -3
    assert c.linear(x, w, None, 0, None, None, None) == -3
    assert c.add_rms_norm(x, n, 0.25, None, True, False, None, False) == -3
    assert c.fp8_linear_codes(cd, sc, fw, fs, 0, None, 0, None, torch.float16, None) == -3


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
