"""CPU: the refusals of the 8-bit integer operators' C ABI (every argument is checked before the
first HIP call) and of their Python binding."""
import pytest

from hcrag_amd import _lib

torch = pytest.importorskip("torch")

P = 1 << 20            # stands for a device address: never read, every call here is refused or empty
F16, BF16, F32 = _lib.HCR_F16, _lib.HCR_BF16, _lib.HCR_F32


def quant(x=P, xt=F16, ldx=64, rows=4, cols=64, act=0, q=P, ldq=64, scale=P):
    return _lib.lib().hcr_quant_rows_device(x, xt, ldx, rows, cols, act, q, ldq, scale, None)


def norm(x=P, xt=F16, ldx=64, r=P, rt=F32, ldr=64, rows=4, cols=64, kind=0, w=P, b=P, eps=1e-6, s=P,
         lds=64, y=P, yt=F16, ldy=64, q=P, ldq=64, scale=P):
    args = _lib.NORM_QUANT_ARGS.pack(x or 0, ldx, r or 0, ldr, w or 0, b or 0, s or 0, lds, y or 0, ldy, q or 0, ldq,
                                     scale or 0, rows, cols, xt, rt, yt, kind, eps)
    return _lib.lib().hcr_norm_quant_rows_device(args, None)


def dequant(q=P, ldq=64, scale=P, rows=4, cols=64, out=P, ot=F16, ldo=64):
    return _lib.lib().hcr_dequant_rows_device(q, ldq, scale, rows, cols, out, ot, ldo, None)


def linear(x=P, ldx=64, sx=P, rows=4, w=P, ldw=64, sw=P, features=8, depth=64, b=P, out=P, ot=F16, ldo=8):
    return _lib.lib().hcr_int8_linear_device(x, ldx, sx, rows, w, ldw, sw, features, depth, b, out, ot, ldo, None)


BAD = [
    (quant, dict(rows=-1)), (quant, dict(rows=(1 << 30) + 1)), (quant, dict(cols=0)), (quant, dict(cols=32769, ldx=40000, ldq=40000)),
    (quant, dict(act=2)), (quant, dict(xt=3)), (quant, dict(x=None)), (quant, dict(q=None)), (quant, dict(scale=None)),
    (quant, dict(ldx=63)), (quant, dict(ldq=48)), (quant, dict(ldq=72)), (quant, dict(q=P + 8)), (quant, dict(x=P + 1)),
    (quant, dict(x=P + 2, xt=F32)), (quant, dict(scale=P + 2)),
    (norm, dict(kind=2)), (norm, dict(eps=-1e-6)), (norm, dict(eps=float("nan"))), (norm, dict(w=None)), (norm, dict(r=None)),
    (norm, dict(rt=5)), (norm, dict(yt=-1)), (norm, dict(ldr=60)), (norm, dict(lds=60)), (norm, dict(ldy=60)),
    (norm, dict(b=P + 1)), (norm, dict(s=P + 2)), (norm, dict(y=P + 1)), (norm, dict(cols=40000, ldx=40000)), (norm, dict(ldq=65)),
    (dequant, dict(cols=131072, ldq=131072, ldo=131072)), (dequant, dict(out=None)), (dequant, dict(ldo=63)), (dequant, dict(ot=4)),
    (dequant, dict(q=P + 4)), (dequant, dict(rows=1 << 30, cols=65536, ldq=65536, ldo=65536)),
    (linear, dict(depth=0)), (linear, dict(depth=131072, ldx=131072, ldw=131072)), (linear, dict(features=-1)),
    (linear, dict(features=(1 << 30) + 1)), (linear, dict(rows=-5)), (linear, dict(ldx=56)), (linear, dict(ldw=48)),
    (linear, dict(x=P + 15)), (linear, dict(w=P + 1)), (linear, dict(ldo=7)), (linear, dict(ot=7)), (linear, dict(out=P + 1)),
    (linear, dict(sx=None)), (linear, dict(sw=None)), (linear, dict(out=None)), (linear, dict(b=P + 2)), (linear, dict(sx=P + 1)),
    (linear, dict(rows=1 << 30, features=1 << 30, ldo=1 << 30)),
]


@pytest.mark.parametrize("call,wrong", BAD, ids=lambda v: getattr(v, "__name__", None) or ",".join(map(str, v)))
def test_bad_arguments_are_refused(call, wrong):
    assert call(**wrong) == _lib.HCR_EINVAL
    assert _lib.lib().hcr_last_error()


# buffers of their own: what is in one place twice is what the case says
X, R, S, Y, Q, O = (P * (2 + i) for i in range(6))
OWN = {quant: dict(x=X, q=Q), norm: dict(x=X, r=R, s=S, y=Y, q=Q), dequant: dict(q=Q, out=O),
       linear: dict(x=X, w=Q, out=O)}
ALIASED = [
    (quant, dict(q=X)), (dequant, dict(out=Q)), (linear, dict(out=X)), (linear, dict(out=Q)),
    (norm, dict(s=R, lds=128)), (norm, dict(y=X, yt=BF16)), (norm, dict(y=X, ldy=128)), (norm, dict(y=R, yt=F16)),
    (norm, dict(y=R, yt=F32, ldy=128)), (norm, dict(s=X)), (norm, dict(s=Y)), (norm, dict(s=R, y=R, yt=F32)),
    (norm, dict(q=X)), (norm, dict(q=R)), (norm, dict(q=S)), (norm, dict(q=Y)),
]


@pytest.mark.parametrize("call,wrong", ALIASED, ids=lambda v: getattr(v, "__name__", None) or ",".join(v))
def test_outputs_in_the_place_of_operands_are_refused(call, wrong):
    assert call(**{**OWN[call], **wrong}) == _lib.HCR_EINVAL
    assert b"overlap" in _lib.lib().hcr_last_error() or b"buffer of" in _lib.lib().hcr_last_error()


@pytest.mark.parametrize("call,name", [(quant, "cols"), (norm, "cols"), (dequant, "cols"), (linear, "depth"), (linear, "features")])
def test_sizes_past_32_bits_are_refused_not_cut(call, name):
    far = 1 << 33
    strides = {quant: ("ldx", "ldq"), norm: ("ldx", "ldr", "lds", "ldy", "ldq"), dequant: ("ldq", "ldo"),
               linear: ("ldx", "ldw", "ldo")}[call]
    assert call(**{**OWN[call], name: (1 << 32) + 8, **{k: far for k in strides}}) == _lib.HCR_EINVAL


def test_packed_arguments_are_the_struct():
    import ctypes

    class Args(ctypes.Structure):                 # hcr_norm_quant_args, include/hcrag.h
        _fields_ = [(n, ctypes.c_void_p if n in ("x", "r", "w", "b", "s", "y", "q", "scale") else ctypes.c_int64)
                    for n in "x ldx r ldr w b s lds y ldy q ldq scale rows cols".split()] + [
            (n, ctypes.c_int32) for n in ("xt", "rt", "yt", "kind")] + [("eps", ctypes.c_float)]

    values = [*range(1, 16), 1, 2, 0, 1, 0.5]
    packed = _lib.NORM_QUANT_ARGS.pack(*values)
    assert len(packed) == ctypes.sizeof(Args)
    a = Args.from_buffer_copy(packed)
    assert [getattr(a, n) for n, _ in Args._fields_] == values
    assert _lib.lib().hcr_norm_quant_rows_device(None, None) == _lib.HCR_EINVAL


def test_nothing_to_do_is_ok():
    assert quant(rows=0, x=None, q=None, scale=None) == 0
    assert norm(rows=0, x=None, w=None, q=None, scale=None) == 0
    assert dequant(rows=0, q=None, scale=None, out=None) == 0
    assert linear(rows=0, x=None, out=None) == 0
    assert linear(features=0, w=None, out=None) == 0


def test_python_refuses_host_tensors_and_others():
    import hcrag_amd
    x = torch.randn(4, 32)
    with pytest.raises(ValueError, match="device tensor"):
        hcrag_amd.quantize_rows(x)
    with pytest.raises(ValueError, match="torch tensor"):
        hcrag_amd.quantize_rows([[1.0]])
    with pytest.raises(ValueError, match="device tensor"):
        hcrag_amd.norm_quantize(x, torch.ones(32))
    with pytest.raises(ValueError, match="device tensor"):
        hcrag_amd.Int8Rows(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError, match="Int8Rows"):
        hcrag_amd.int8_linear(x, x)
